"""How chromofold_amd.kvselect makes its calls (streams, tensors it makes and holds, arguments beside a kept descriptor),
without a GPU: stand-ins for streams, and checks that are made before a call reaches one."""
import contextlib
import os

import pytest
import torch

from chromofold_amd import _abi as A
from chromofold_amd import kvselect as ks

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
