"""How chromofold_amd.kvselect, and kv's sealing, make their calls (streams, tensors they make and hold, arguments beside a
kept descriptor), without a GPU: stand-ins for streams, and checks that are made before a call reaches one."""
import contextlib
import os

import pytest
import torch

from chromofold_amd import _abi as A
from chromofold_amd import kv, kvselect as ks

pytestmark = pytest.mark.skipif(not os.path.exists(A.LIB_PATH), reason="libchromofold.so not built")


class Streams:
    """Stand-ins for the current stream and a second one: what is made, called and waited for, and on which."""

    def __init__(self, monkeypatch):
        self.log = []
        self.main, self.side = self.Stream("main", self.log), self.Stream("side", self.log)
        self.now = self.main
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.now)
        monkeypatch.setattr(torch.cuda, "stream", self.on)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.log.append(("kept", s.name)))

    class Stream:
        device = torch.device("cpu")

        def __init__(self, name, log):
            self.name, self.log = name, log

        def wait_stream(self, other):
            self.log.append(("wait", self.name, other.name))

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def watch(self, monkeypatch, module, name):
        inner = getattr(module, name)

        def call(*args, **kw):
            self.log.append((name, self.now.name))
            return inner(*args, **kw)
        monkeypatch.setattr(module, name, call)


def test_bounds_of_works_on_its_stream(monkeypatch):
    # the records' zeros, the groups' pages and counts and the bounds in the order of one stream, behind the keys'
    st = Streams(monkeypatch)
    monkeypatch.setattr(ks, "key_bounds", lambda k, f, c, out, stream=None: out)
    for module, name in ((ks, "empty_bounds"), (ks, "key_bounds"), (torch, "arange"), (torch, "clamp")):
        st.watch(monkeypatch, module, name)
    ks.bounds_of(torch.zeros(2, 1, 80, 64), stream=st.side)
    assert st.log[:2] == [("wait", "side", "main"), ("kept", "side")]
    assert {x[0] for x in st.log[2:]} == {"empty_bounds", "key_bounds", "arange", "clamp"}
    assert all(x[1] == "side" for x in st.log[2:]) and st.now is st.main
    st.log.clear()
    ks.bounds_of(torch.zeros(2, 1, 80, 64))
    ks.bounds_of(torch.zeros(2, 1, 80, 64), stream=st.main)
    assert all(x[1] == "main" and x[0] != "wait" for x in st.log)
    st.side.device = torch.device("cuda:0")
    with pytest.raises(ValueError):
        ks.bounds_of(torch.zeros(2, 1, 80, 64), stream=st.side)


class Encoder:
    """Stand-in for the library around one sealing call: notes the stream that is the current one and the call's."""

    def __init__(self, streams, lib):
        self.streams, self.lib = streams, lib

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def cf_kv_encode_groups_async(self, *args):
        self.streams.log.append(("encode", args[-1]))
        return A.CF_OK


def test_sealing_fills_its_results_on_its_stream(monkeypatch):
    st = Streams(monkeypatch)
    lib = Encoder(st, A.lib())
    monkeypatch.setattr(A, "lib", lambda: lib)
    st.main.cuda_stream, st.side.cuda_stream = 1, 2
    for name in ("empty", "zeros", "full"):
        st.watch(monkeypatch, torch, name)
    x = torch.ones(4, 16, 64)
    first, counts, pool = torch.tensor([0]), torch.tensor([4], dtype=torch.int32), torch.ones(1 << 16, dtype=torch.uint8)
    for stream, on in ((None, ("main", 1)), (st.side, ("side", 2))):
        st.log.clear()
        kv.encode_groups_device(kv.CODEC_INT8, x, x, 64, None, first, counts, pool, stream=stream)
        assert {y[0] for y in st.log} == {"empty", "zeros", "full", "encode"}
        assert all(y[1] == (on[1] if y[0] == "encode" else on[0]) for y in st.log), st.log


def test_seal_device_orders_its_two_streams(monkeypatch):
    # what it makes is there before the encoder runs on the other stream, which has run before anything is read or let go of
    st = Streams(monkeypatch)

    def encode(*args, **kw):
        st.log.append(("encode", args[12].name if args[12] else None))
        return kv.DeviceEncodeResult(torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int64),
                                     torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(kv, "encode_groups_device", encode)
    for name in ("arange", "clamp", "empty", "full"):
        st.watch(monkeypatch, torch, name)
    x = torch.zeros(2, 1, 80, 64)
    kv.seal_device(kv.CODEC_INT8, x, x, None, stream=st.side)
    log = [y for y in st.log if y[0] in ("encode", "wait", "kept")]
    assert log == [("wait", "side", "main"), ("encode", "side"), ("wait", "main", "side"), ("kept", "main")]
    assert [y[0] for y in st.log].index("wait") > max(i for i, y in enumerate(st.log) if y[0] in ("arange", "clamp", "empty"))
    assert all(y[1] == "main" for y in st.log if y[0] in ("arange", "clamp", "empty", "full"))
    st.log.clear()
    kv.seal_device(kv.CODEC_INT8, x, x, None)
    assert not any(y[0] == "wait" for y in st.log)
