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


# ---------------------------------------------------------------------------------------------------- kept descriptors
S, H, M, D, K = 2, 3, 5, 64, 4


def z(*shape, t=torch.int32):
    return torch.zeros(*shape, dtype=t)


class Kept:
    """A cache of S sequences, its bounds and a step's tensors, and the three operators' calls with descriptors of them."""

    def __init__(self):
        self.kvb = kv.BatchedKv(kv.CODEC_INT8, S, H, D, M, z(64, t=torch.uint8), z(S, H, M), z(S), None)
        self.b, self.to_b = ks.empty_bounds(S, H, M, D, "cpu"), ks.empty_bounds(S, H, M, D, "cpu")
        f = torch.float32
        self.q, self.out, self.pos, self.units = z(S, 2 * H, D, t=f), z(S, 2 * H, D, t=f), z(S), z(S, H, K)
        self.w, self.w2 = z(S, H, M, t=f), z(S, H, M, t=f)
        self.to = ks.Evicted(z(S, H, M), z(S), z(S, H, M, t=f), self.to_b, z(S, H, M))

    def select(self, desc=None, **kw):
        a = {"kvb": self.kvb, "bounds": self.b, "queries": self.q, "query_pos": self.pos, "units": self.units}
        number = {"unit_groups": 2, "keep_first": 2, "keep_last": 1} if desc is None else {}
        return (ks.select_desc if desc is None else ks.select)(**{**a, **number, **kw}, **({"desc": desc} if desc else {}))

    def attention(self, desc=None, **kw):
        a = {"kvb": self.kvb, "queries": self.q, "output": self.out, "query_pos": self.pos, "softmax_scale": 0.1}
        more = {"units": self.units, "unit_groups": 2, "weights": self.w, "weights_out": self.w2, "decay": 0.9, "splits": 3}
        return (ks.attention_desc if desc is None else ks.attention)(**{**a, **(more if desc is None else {}), **kw},
                                                                     **({"desc": desc} if desc else {}))

    def evict(self, desc=None, **kw):
        a = {"kvb": self.kvb, "weights": self.w, "budget_units": 2}
        more = {"out": self.to, "bounds": self.b, "unit_groups": 2, "keep_first": 0, "keep_last": 2}
        return (ks.evict_desc if desc is None else ks.evict)(**{**a, **(more if desc is None else {}), **kw},
                                                             **({"desc": desc} if desc else {}))


@pytest.fixture
def made(monkeypatch):
    """Calls get as far as the library, which notes them."""
    calls = []
    monkeypatch.setattr(ks, "_raw_stream", lambda device, stream: 0)
    monkeypatch.setattr(ks, "_for_stream", lambda d, *rest: d)
    monkeypatch.setattr(ks, "_with_workspace", lambda *args: None)
    monkeypatch.setattr(ks, "_call", lambda name, *rest: calls.append(name))
    k = Kept()
    k.calls = calls
    return k


def other(t):
    return torch.zeros_like(t)


def test_attention_checks_the_pool_and_the_tables(made):
    u8 = torch.uint8
    k, enough = made, 2 * H * kv.TABLE_BYTES

    def cache(codec=kv.CODEC_INT8, pool=z(64, t=u8), tables=None):
        k.kvb = kv.BatchedKv(codec, S, H, D, M, pool, z(S, H, M), z(S), tables)
        return k.attention()
    cache()
    cache(kv.CODEC_RANS_HYBRID, tables=z(enough, t=u8))
    cache(kv.CODEC_RANS_HYBRID, tables=z(2 * H, kv.TABLE_BYTES, t=u8))
    cache(tables=z(1))  # not read
    cache(pool=z(4, 16, t=u8))
    rans = lambda tables: cache(kv.CODEC_RANS_HYBRID, tables=tables)  # noqa: E731
    for bad in (lambda: cache(pool=z(16)), lambda: cache(pool=z(128, t=u8)[::2]),
                lambda: cache(pool=torch.empty(64, dtype=u8, device="meta")), lambda: rans(z(enough // 4)),
                lambda: rans(z(enough - 1, t=u8)), lambda: rans(z(2 * enough, t=u8)[::2]),
                lambda: rans(torch.empty(enough, dtype=u8, device="meta"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(A.CfError):
        rans(None)


def test_a_kept_descriptor_takes_its_own_arguments(made):
    k = made
    sd, ad, ed = k.select(), k.attention(), k.evict()
    assert k.select(sd) is k.units
    assert k.select(sd, bounds=None, queries=None, query_pos=None, units=None) is k.units
    k.select(sd, units=k.units.view(S, H, K), unit_groups=2, keep_first=2)
    k.attention(ad)
    k.attention(ad, units=k.units, weights=k.w, weights_out=k.w2, decay=0.9, splits=3, unit_groups=2)
    k.attention(ad, softmax_scale=float(torch.tensor(0.1)))  # the same as float32
    k.attention(ad, queries=None, output=None, query_pos=None, softmax_scale=None)
    k.evict(ed)
    k.evict(ed, weights=None, budget_units=None)
    k.evict(ed, out=k.to, bounds=k.b, unit_groups=2, keep_first=0, keep_last=2)
    assert k.calls == ["cf_kv_select_groups_async"] * 3 + ["cf_kv_paged_attention_selected_async"] * 4 + [
        "cf_kv_evict_groups_async"] * 3


def test_a_kept_descriptor_refuses_other_arguments(made):
    k = made
    sd, ad, ed = k.select(), k.attention(), k.evict()
    cache = lambda **kw: kv.BatchedKv(**{**{f: getattr(k.kvb, f) for f in ("codec", "seq_count", "kv_heads", "head_dim",  # noqa
                                                                          "max_groups", "pool", "group_offsets", "seq_tokens",
                                                                          "tables")}, **kw})
    bad = [
        lambda: k.select(sd, queries=other(k.q)), lambda: k.select(sd, query_pos=other(k.pos)),
        lambda: k.select(sd, units=other(k.units)), lambda: k.select(sd, bounds=k.to_b), lambda: k.select(sd, unit_groups=3),
        lambda: k.select(sd, kvb=cache(seq_tokens=z(S))), lambda: k.select(sd, keep_first=3), lambda: k.select(sd, keep_last=2),
        lambda: k.select(sd, units=k.units[:, :, :2]),
        lambda: k.attention(ad, queries=other(k.q)), lambda: k.attention(ad, output=other(k.out)),
        lambda: k.attention(ad, query_pos=other(k.pos)), lambda: k.attention(ad, softmax_scale=0.2),
        lambda: k.attention(ad, units=other(k.units)), lambda: k.attention(ad, weights=k.w2),
        lambda: k.attention(ad, weights_out=k.w), lambda: k.attention(ad, decay=0.5), lambda: k.attention(ad, splits=1),
        lambda: k.attention(ad, kvb=cache(pool=z(64, t=torch.uint8))),
        lambda: k.attention(ad, kvb=cache(group_offsets=z(S, H, M))),
        lambda: k.attention(ad, kvb=cache(tables=z(64, t=torch.uint8))),
        lambda: k.evict(ed, weights=k.w2), lambda: k.evict(ed, budget_units=3), lambda: k.evict(ed, bounds=k.to_b),
        lambda: k.evict(ed, out=ks.Evicted(z(S, H, M), k.to.seq_tokens)), lambda: k.evict(ed, kvb=cache(seq_tokens=z(S))),
        lambda: k.evict(ed, keep_last=3),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="the descriptor"):
            call()
    assert not k.calls


def test_a_kept_descriptor_holds_what_it_points_at(made):
    # tensors of a cache whose fields are given others live as long as the descriptor
    import weakref
    k = made
    refs = [weakref.ref(t) for t in (k.kvb.pool, k.kvb.group_offsets, k.kvb.seq_tokens, k.b.codes, k.to.weights)]
    descs = [k.select(), k.attention(), k.evict()]
    k.kvb.pool, k.kvb.group_offsets, k.kvb.seq_tokens = z(64, t=torch.uint8), z(S, H, M), z(S)
    k.b.codes, k.to.weights = None, None
    assert all(r() is not None for r in refs)
    with pytest.raises(ValueError, match="the descriptor"):
        k.attention(descs[1])
    descs.clear()
    assert all(r() is None for r in refs)
