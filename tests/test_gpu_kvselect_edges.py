"""The operators of chromofold/kv_select.h, and the batched decode whose group body they share, where values, masks and
streams are out of the ordinary (plain forms and tolerances: kvselect_helpers.py)."""
import numpy as np
import pytest

import kvselect_helpers as R
import test_gpu_kvselect as T
from kv_helpers import make_seqs
from test_gpu_kvselect import dev, down, u32, up  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- streams
def test_bounds_of_on_another_stream(dev):
    # keys that the current stream is still making when the call is issued, and a transposed view of them
    import torch
    from chromofold_amd import kvselect as ks
    k = np.random.default_rng(1).standard_normal((2, 3, 208, 64)).astype(np.float32)
    codes, scales = R.bounds_ref([k[s, h, 64 * g: 64 * g + 64] for s in range(2) for h in range(3) for g in range(4)])
    host, side = up(dev, k), torch.cuda.Stream(dev)
    for form in range(4):
        busy = torch.ones(4096, 4096, device=dev)
        for _ in range(4):
            busy = busy @ busy * 1e-4
        keys = host * 1.0 if form % 2 else (host.transpose(0, 1) * 1.0).transpose(0, 1)
        b = ks.bounds_of(keys, stream=side)
        del keys
        side.synchronize()
        assert np.array_equal(down(b.scales).ravel(), scales) and np.array_equal(down(b.codes).reshape(codes.shape), codes)


def test_seal_device_on_another_stream(dev):
    import torch
    from chromofold_amd import kv
    rng = np.random.default_rng(2)
    k, v = (rng.standard_normal((2, 3, 208, 64)).astype(np.float32) for _ in range(2))
    tables = np.concatenate([kv.build_table(x[0, h].reshape(-1, 16, 64)) for h in range(3) for x in (k, v)])
    want = kv.seal_device(kv.CODEC_RANS_HYBRID, up(dev, k), up(dev, v), up(dev, tables))
    q, pos = up(dev, rng.standard_normal((2, 6, 64)).astype(np.float32)), up(dev, np.array([207, 100], np.uint32))
    ref, out = torch.empty_like(q), torch.empty_like(q)
    want.attention(q, ref, pos, 0.125)
    host, side = (up(dev, k), up(dev, v)), torch.cuda.Stream(dev)
    for _ in range(3):
        busy = torch.ones(4096, 4096, device=dev)
        for _ in range(4):
            busy = busy @ busy * 1e-4
        got = kv.seal_device(kv.CODEC_RANS_HYBRID, host[0] * 1.0, host[1] * 1.0, up(dev, tables), stream=side)
        assert torch.equal(got.group_offsets, want.group_offsets) and got.pool.numel() == want.pool.numel()
        got.attention(q, out, pos, 0.125)
        assert torch.equal(out, ref)


def test_every_stream_has_a_workspace(dev, monkeypatch):
    """Calls of one descriptor on several streams, which may overlap: on its own stream it brings its workspace, on every other
    one a copy with one that is that call's. A selection of two launches and an attention of split rows; results as on one
    stream."""
    import torch
    from chromofold_amd import kvselect as ks
    rng = np.random.default_rng(9)
    S, H, M, D = 2, 2, 1100, 128
    codes, scales = T._records(rng, S, H, M, D)
    c = T.Case(dev, [64 * 40, 64 * 33 + 1], H, 4, D, 62)
    b = ks.KeyBounds(up(dev, codes), up(dev, scales))
    long = T._cache(dev, S, H, D, M, [64 * M, 64 * M - 70])
    q, pos, q2 = up(dev, c.q), up(dev, np.array(c.pos, np.uint32)), up(dev, rng.standard_normal((S, 2 * H, D)).astype(np.float32))
    far = up(dev, np.array([64 * M - 1, 64 * M - 1], np.uint32))
    units, out, w = torch.empty(S, H, 70, dtype=torch.int32, device=dev), torch.empty_like(q), torch.empty(S, H, c.M, device=dev)
    own = torch.cuda.Stream(dev)
    own.wait_stream(torch.cuda.current_stream(dev))
    sd = ks.select_desc(long, b, q2, far, units, stream=own)
    ad = ks.attention_desc(c.kvb, q, out, pos, c.scale, weights_out=w, splits=4, stream=own)
    assert sd.workspace and ad.workspace
    used, inner = [], ks._for_stream

    def for_stream(d, cls, device, stream, s):
        got = inner(d, cls, device, stream, s)
        used.append((d, got, s))
        return got
    monkeypatch.setattr(ks, "_for_stream", for_stream)

    def calls(stream):
        ks.select(long, b, q2, far, units, desc=sd, stream=stream)
        ks.attention(c.kvb, q, out, pos, c.scale, desc=ad, stream=stream)
    calls(own)
    own.synchronize()
    want = [x.clone() for x in (units, out, w)]
    assert np.array_equal(u32(units), R.select_ref(down(q2), codes, scales, [64 * M, 64 * M - 70], [64 * M - 1] * 2, 2, 1, 70, 1, 1))
    c.compare(R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, 4, c.scale, None, 1, c.M), down(out).astype(np.float64),
              down(w).astype(np.float64))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    for st in streams + [None, own]:
        calls(st)
    torch.cuda.synchronize()
    for a, e in zip((units, out, w), want):
        assert torch.equal(a, e)
    assert [got is d for d, got, _ in used] == [True, True] + [False] * 8 + [True, True]
    for d in (sd, ad):
        mine = [got for x, got, _ in used if x is d]
        for got in mine:
            assert got.workspace_bytes == d.workspace_bytes and (got is d or got.workspace_tensor is not d.workspace_tensor)
        held = {got.workspace for got in mine}  # `used` keeps all of them: none was reused
        assert len(held) == 5
        assert all(got is d or got.workspace_stream == s for x, got, s in used if x is d)


# ---------------------------------------------------------------------------------------------------- key bounds
@pytest.mark.parametrize("D", [128, 64])
def test_bounds_bound_every_finite_group(dev, D):
    """Groups from the least subnormal key to the largest finite one, whole and cut: scale times code is never inside the keys
    by more than the quotient's and the scale's rounding, 2^-23 of the scale's 127 steps, and a scale of 0 means zeros."""
    from chromofold_amd import kvselect as ks
    rng = np.random.default_rng(D)
    least = np.float64(2.0 ** -149)
    tops = [least * n for n in (1, 2, 63, 64, 100, 126, 127, 128, 180, 190, 191, 254, 300, 1000, 12345, 127 * 2 ** 23 - 1)]
    tops += [127 * 2.0 ** -126, 2.0 ** -126, 1e-20, 1.0, 3.3e38]
    groups = []
    for top in tops:
        k = (rng.uniform(-1, 1, (64, D)) * top).astype(np.float32)
        k[rng.integers(64), rng.integers(D)] = np.float32(top)
        k[rng.integers(64), rng.integers(D)] = -np.float32(top)
        groups.append(k)
    keys, n = np.concatenate(groups).reshape(-1, 16, D), len(groups)
    out = ks.empty_bounds(1, 1, n, D, dev)
    ks.key_bounds(up(dev, keys), up(dev, 4 * np.arange(n, dtype=np.int64)), up(dev, np.full(n, 4, np.uint32)), out)
    codes, scales = down(out.codes)[0, 0].astype(np.float64), down(out.scales)[0, 0].astype(np.float64)
    for k, c, s in zip(groups, codes, scales):
        k, slack = k.astype(np.float64), 2.0 ** -23 * 127 * s
        assert (c[:D] * s >= k.max(0) - slack).all() and (c[D:] * s >= -k.min(0) - slack).all(), (np.abs(k).max(), s)
        assert (c[:D] * s <= k.max(0) + s + slack).all() and (c[D:] * s <= -k.min(0) + s + slack).all()
        assert s > 0


# ---------------------------------------------------------------------------------------------------- V scales
def cache(monkeypatch, dev, lens, H, gqa, D, seed, codec=1, edit=None, **how):
    """A Case whose data `edit(data)` may change before it is sealed (coded pools as chain pairs)."""
    def seqs(*args, **kw):
        data = make_seqs(*args, **kw)
        if edit:
            edit(data)
        return data
    monkeypatch.setattr(T, "make_seqs", seqs)
    return T.Case(dev, lens, H, gqa, D, seed, codec=codec, **how)


def set_v_scales(c, s, h, g, scales):
    """Writes the V scales of the pages of group g into its header (64-byte header: fp32 x 4 at 48), and the reference's."""
    o = 16 * int(c.kvb.host_offsets[s, h, g])
    old = down(c.kvb.pool[o + 48: o + 64]).view(np.float32)
    new = np.array(scales, np.float32)
    c.kvb.pool[o + 48: o + 64] = up(c.dev, new.view(np.uint8))
    for p in range(4):
        t = slice(64 * g + 16 * p, 64 * g + 16 * p + 16)
        c.v[s][h][t] *= float(new[p]) / float(old[p])


def attend(c, call, splits):
    """The rows' results from the call that can select groups, or from the batched one."""
    import torch
    if call == "selected":
        return c.run(splits=splits)[0]
    out = torch.full(c.q.shape, float("nan"), device=c.dev)
    c.kvb.attention(up(c.dev, c.q), out, up(c.dev, np.array(c.pos, np.uint32)), c.scale, splits=splits)
    return down(out).astype(np.float64)


CALLS = [(1, "selected", 1), (1, "selected", 4), (1, "selected", 8), (1, "selected", 16), (2, "selected", 1), (2, "selected", 4),
         (1, "batched", 1), (1, "batched", 4), (2, "batched", 1), (2, "batched", 4)]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, call, gqa", CALLS)
def test_v_scales_that_fall_in_steps(dev, monkeypatch, codec, call, gqa, D):
    """V scales down from 2^30 to 2^-110 in steps of less than 2^60, again and again in each wavefront's groups: sums of the
    large ones stay finite, whatever unit the small ones ask for, and what a later group brings back up is not lost."""
    steps = [30, -25, -80, -110, -110]
    c = cache(monkeypatch, dev, [64 * 40, 64 * 40 - 7], 1, gqa, D, 201, codec)
    for s in range(2):
        for g in range(40):
            set_v_scales(c, s, 0, g, [2.0 ** steps[g % 5]] * 4)
    o, _, mag, big, low = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, gqa, c.scale, None, 1, c.M)
    tol = R.tolerance(big, D)[..., None] * mag + 2.0 ** -23 * np.abs(o) + low
    for splits in (1, 2):
        out = attend(c, call, splits)
        assert np.isfinite(out).all(), splits
        assert (np.abs(out - o) <= tol).all(), splits


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, call, gqa", [c for c in CALLS if c[:2] != (1, "batched")])
def test_small_v_behind_large_v_of_no_weight(dev, monkeypatch, codec, call, gqa, D):
    """Each wavefront's first groups have V scales of 2^20, 2^-30 and 2^-60 and scores so low (150 below the others', in log2
    units 200 or more) that the rest, with V scales of 2^-95 and less, are all of the output: they are held in units that
    follow them, not the sums that have faded. (Not for the batched call of an INT8 pool: its K operands are symbols + 1024,
    whose sums over D / 4 instructions of each of two parts may be off by 2 D / 4 * 2^-24 * 1280 sum |x| of the queries x, here
    0.3 in a score, so that no bound on its outputs would tell.)"""
    exps = [20, -30, -60, -95, -100, -95, -101, -95, -97, -99]
    n = len(exps)
    away = np.array([g % n < 3 for g in range(4 * n)])

    def edit(data):
        for k, _ in data:
            k *= np.float32(0.02)
            k[..., 0] = np.where(np.repeat(away, 64), -8.0, 8.0)
    c = cache(monkeypatch, dev, [64 * 4 * n], 1, gqa, D, 202, codec, edit)
    for g in range(4 * n):
        set_v_scales(c, 0, 0, g, [2.0 ** exps[g % n]] * 4)
    c.q[:, :, 0], c.scale = 1.0, 10.0
    o, _, mag, big, _ = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, gqa, c.scale, None, 1, c.M)
    # weights of the groups with V scales of 2^-95 may be held in units up to 8 binades above their own: 2^-25 of a unit
    # 2^(-95 + 1 - 15 + 8) each, times a symbol, over a sum of weights that is at least 1
    floor = 2.0 ** (-25 - 95 + 1 - 15 + 8) * 128 * c.lens[0]
    for splits in (1, 2):
        out = attend(c, call, splits)
        assert (np.abs(out - o) <= R.tolerance(big, D)[..., None] * mag + 2.0 ** -23 * np.abs(o) + floor).all(), splits
        assert (np.abs(o) > 2 * floor).mean() > 0.9


ZERO_CALLS = [c for c in CALLS if c[1] == "selected"]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, call, gqa", ZERO_CALLS)
@pytest.mark.parametrize("exp", [-20, -30, -44, 10])
def test_pages_of_zeros_beside_small_v(dev, monkeypatch, codec, call, gqa, D, exp):
    """Pages whose V are all 0, or whose tokens before the query are, among pages of V around 2^exp: whatever scale they have
    (the encoders write 1; 2^25 and 0 too), the others keep their bits."""
    lens, pos = [640, 390, 64, 700], [639, 389, 63, 64 * 10 + 16 * 2 + 4]

    def edit(data):
        rng = np.random.default_rng(7)
        for s, (_, v) in enumerate(data):
            v *= np.float32(2.0 ** exp)
            for h in range(2):
                for page in range(-(-lens[s] // 16)):
                    if rng.random() < 0.4 and s != 2 or s == 2 and page in (0, 3):
                        v[h, 16 * page: 16 * page + 16] = 0.0
        data[3][1][:, 640: 640 + 37] = 0.0   # of the query's page only what lies behind it, and far larger
        data[3][1][:, 640 + 16: 640 + 32] = np.float32(2.0 ** exp)
        data[3][1][:, 640 + 37:] = 1.0
    c = cache(monkeypatch, dev, lens, 2, gqa, D, 205, codec, edit, pos=pos)
    for h in (0, 1):
        zero = [p for p in range(40) if not c.v[0][h][16 * p: 16 * p + 16].any()]
        for p, scale in zip(zero, [2.0 ** 25, 0.0] * 20):
            o = 16 * int(c.kvb.host_offsets[0, h, p // 4]) + 48 + 4 * (p % 4)
            c.kvb.pool[o: o + 4] = up(dev, np.array([scale], np.float32).view(np.uint8))
    o, _, mag, big, _ = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, gqa, c.scale, None, 1, c.M)
    # as kvselect_helpers.weight_floor, from the pages that hold something: scales of 2^exp / 127 to 6 times that
    low = np.zeros(o.shape)
    for s in range(4):
        for h in (0, 1):
            low[s, h * gqa: (h + 1) * gqa] = 2.0 ** -39 * 6 * np.abs(c.v[s][h][: pos[s] + 1]).sum(0)
    tol = R.tolerance(big, D)[..., None] * mag + 2.0 ** -23 * np.abs(o) + low
    for splits in (0, 1, 3):
        out = attend(c, call, splits)
        assert (np.abs(out - o) <= tol).all(), splits


# ---------------------------------------------------------------------------------------------------- what is not visible
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, call, gqa", CALLS)
def test_scales_behind_the_query(dev, monkeypatch, codec, call, gqa, D):
    """Pages of a row's last group that the query must not see, with V scales of infinity and NaN (as of a sealed page that
    holds them) and K scales of NaN: outputs and weights as without them. Row 1: raw groups in a coded pool. Row 2: the last
    page is cut, and its pages behind the query are absent."""
    c = cache(monkeypatch, dev, [320, 320, 261], 2, gqa, D, 203, codec, pos=[269, 269, 260],
              **({"raw_groups": {1: 5}} if codec == 2 else {}))
    bad = np.array([np.nan, np.inf, -np.inf], np.float32)
    for s in (0, 1):
        for h in (0, 1):
            o = 16 * int(c.kvb.host_offsets[s, h, 4])
            c.kvb.pool[o + 52: o + 64] = up(dev, np.roll(bad, h).view(np.uint8))
            c.kvb.pool[o + 36: o + 48] = up(dev, np.full(3, np.nan, np.float32).view(np.uint8))
    ref = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, gqa, c.scale, None, 1, c.M)
    o, w, mag, big, low = ref
    for splits in (0, 1, 3):
        out = attend(c, call, splits)
        assert np.isfinite(out).all(), splits
        if call == "selected":
            c.compare(ref, *c.run(splits=splits))
        else:  # the batched call's bar (its scores are not held as finely)
            assert (np.abs(out - o).max(2) <= 1e-3 * np.abs(o).max(2)).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, call, gqa", CALLS)
def test_small_v_beside_absent_pages(dev, monkeypatch, codec, call, gqa, D):
    # V of 2^-112 and pages that are not there, whose scale of 1 is 2^128 in these units
    c = cache(monkeypatch, dev, [69, 5, 300], 1, gqa, D, 204, codec, v_mult=[[2.0 ** -112]] * 3)
    o, _, mag, big, low = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, gqa, c.scale, None, 1, c.M)
    for splits in (0, 1):
        out = attend(c, call, splits)
        assert np.isfinite(out).all()
        assert (np.abs(out - o).max(2) <= 1e-3 * np.abs(o).max(2)).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("codec, gqa", [(1, 1), (1, 4), (1, 7), (1, 16), (2, 1), (2, 4)])
def test_scores_of_minus_infinity(dev, monkeypatch, codec, gqa, D):
    """K scales of +inf with products below 0 in all pages (row 0), in some of them (1), in none (2), and in all but with one
    query head whose products are above 0 (3); row 4 has no tokens. Heads whose scores are all -inf are NaN, and so are the
    weights of their groups; others are as if those tokens were not there."""
    def edit(data):
        for k, _ in data:
            k[:] = 0.0
            k[..., 0] = 1.0
    lens = [300, 300, 300, 300, 0]
    c = cache(monkeypatch, dev, lens, 2, gqa, D, 206, codec, edit, **({"raw_groups": {1: 2}} if codec == 2 else {}))
    gone = {0: range(19), 1: [0, 1, 2, 3, 9, 14], 2: [], 3: range(19)}
    inf = up(dev, np.array([np.inf], np.float32).view(np.uint8))
    for s, pages in gone.items():
        for h in (0, 1):
            for p in pages:
                o = 16 * int(c.kvb.host_offsets[s, h, p // 4]) + 32 + 4 * (p % 4)
                c.kvb.pool[o: o + 4] = inf
    c.q[:] = 0.0
    c.q[:, :, 0] = -1.0
    if gqa > 1:
        c.q[3, 1, 0] = 0.5  # inf - inf
    left = [[x.copy() for x in c.k[1]], [x.copy() for x in c.v[1]]]
    keep = ~np.isin(np.arange(300) // 16, gone[1])
    listed = np.tile(np.arange(5 if codec == 1 else 3, dtype=np.uint32), (5, 2, 1))
    for units, unit in ((None, 1), (listed, codec)):  # (a coded pool's chain pairs)
        for splits in (0, 1, 3):
            out, w = c.run(units, unit, weights=None, splits=splits)
            assert np.isnan(out[[0, 3]]).all() and np.isnan(w[[0, 3]]).all(), splits
            assert np.isfinite(out[[1, 2, 4]]).all() and np.isfinite(w[[1, 2, 4]]).all(), splits
            assert (out[4] == 0).all() and (w[4] == 0).all()
            for h in (0, 1):  # equal scores: means over the tokens that are left, 1 / n of the weight each
                v, g = left[1][h][keep], np.bincount(np.arange(300)[keep] // 64, minlength=c.M)
                bound = (R.tolerance(1.0 / np.sqrt(D), D) + 2.0 ** -23) * np.abs(v).mean(0) + R.weight_floor(left[1][h], np.arange(300))
                assert (np.abs(out[1, h * gqa: (h + 1) * gqa] - v.mean(0)) <= bound).all()
                assert (np.abs(w[1, h] - gqa * g / keep.sum()) <= R.tolerance(1.0 / np.sqrt(D), D) * gqa * g / keep.sum()).all()


def test_many_rows_of_minus_infinity(dev, monkeypatch):
    # the cut into stretches over several rows: every third row's K scales are +inf, every seventh row is empty
    def edit(data):
        for k, _ in data:
            k[:] = 1.0
    rng = np.random.default_rng(8)
    S, M = 600, 60
    lens = [0 if s % 7 == 3 else int(x) for s, x in enumerate(rng.integers(1, 300, S))]
    lens[300] = 64 * M
    c = cache(monkeypatch, dev, lens, 1, 4, 64, 207, 1, edit)
    inf = up(dev, np.full(4, np.inf, np.float32).view(np.uint8))
    for s in range(0, S, 3):
        for g in range(-(-lens[s] // 64)):
            o = 16 * int(c.kvb.host_offsets[s, 0, g])
            c.kvb.pool[o + 32: o + 48] = inf
    c.q[:] = -1.0
    out, w = c.run()
    none = np.array(lens) == 0
    low = (np.arange(S) % 3 == 0) & ~none
    assert np.isnan(out[low]).all() and (out[none] == 0).all() and np.isfinite(out[~low]).all()
    for s in np.flatnonzero(low):
        n = -(-lens[s] // 64)
        assert np.isnan(w[s, 0, :n]).all() and (w[s, 0, n:] == 0).all()
    assert np.isfinite(w[~low]).all()


# ---------------------------------------------------------------------------------------------------- a shared prefix
def cascade(dev, S, H, gqa, shared, seed, exps, away=(), pos=None, edit=None):
    """The cascade entry point over a raw prefix of `shared` groups whose V are 2^exps[g] (keys of the groups `away` along -8,
    others along +8 on one channel if there are any), and own tokens like the last of them; query positions `pos` (the last
    token), and what edit(kvb) makes of the sealed cache. Returns what came out, the reference, its sums of p |v| and the
    bound on a weight's relative error."""
    import torch
    from chromofold_amd import kv
    D, n = 128, 64 * shared
    rng = np.random.default_rng(seed)
    T = n + 5
    exp = np.repeat(np.array(list(exps) + [exps[-1]], np.float32), 64)[:T]
    k0 = rng.standard_normal((H, n, D)).astype(np.float32)
    v0 = rng.standard_normal((H, n, D)).astype(np.float32) * np.exp2(exp[:n])[:, None]
    data = []
    for _ in range(S):
        k1, v1 = (rng.standard_normal((H, 5, D)).astype(np.float32) for _ in range(2))
        data.append((np.concatenate([k0, k1], 1), np.concatenate([v0, v1 * np.exp2(exp[n:])[:, None]], 1)))
    q = rng.standard_normal((S, H * gqa, D)).astype(np.float32)
    scale = D ** -0.5
    if len(away):
        scale, q[:, :, 0] = 10.0, 1.0
        side = np.repeat(np.array([-8.0 if g in away else 8.0 for g in range(shared + 1)], np.float32), 64)[:T]
        for k, _ in data:
            k *= np.float32(0.02)
            k[..., 0] = side
    tables = np.concatenate([kv.build_table(x[h][:128].reshape(-1, 16, D)) for h in range(H) for x in (k0, v0 + 1)])
    kvb = kv.build_batched(kv.CODEC_RANS_HYBRID, lambda s: data[s], S, H, np.full(S, T), D, tables, dev,
                           shared={s: (0, shared) for s in range(1, S)}, raw_groups={0: shared}, keep_host=True)
    if edit:
        edit(kvb)
    pos = np.full(S, T - 1, np.uint32) if pos is None else np.array(pos, np.uint32)
    out = torch.full(q.shape, float("nan"), device=dev)
    kvb.attention(up(dev, q), out, up(dev, pos), scale, splits=1, shared_groups=shared)

    def dequant(x):
        x = torch.from_numpy(np.pad(x, ((0, 0), (0, -T % 16), (0, 0)))).view(H, -1, 16, D)
        m = x.abs().amax(dim=(2, 3), keepdim=True)
        s = torch.where(m == 0, torch.ones_like(m), m / 127.0)
        return (torch.round(x / s).double() * s.double()).view(H, -1, D)[:, :T]
    want, mag, big = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for s in range(S):
        k, v = (dequant(x)[:, : int(pos[s]) + 1] for x in data[s])
        x = torch.from_numpy(q[s]).double().view(H, gqa, D)
        p = torch.softmax(torch.matmul(x, k.transpose(1, 2)) * scale, -1)
        want[s], mag[s] = (torch.matmul(p, y).view(H * gqa, D).numpy() for y in (v, v.abs()))
        big = max(big, float(torch.matmul(x.abs(), k.abs().transpose(1, 2)).max()) * scale)
    # a weight's relative error is its score's absolute one: operands of 22 bits and float32 sums, 2^-21 of sum |q k|, and
    # about 2^-20 for exp, the weights' own parts and the merge; twice that for numerator and sum
    return down(out).astype(np.float64), want, mag, 2 * (2.0 ** -21 * big + 2.0 ** -20)


@pytest.mark.parametrize("gqa", [1, 4])
def test_cascade_v_scales_that_fall_in_steps(dev, gqa):
    # the prefix splits of 240 sequences behind 25 groups of 8 heads hold 5 groups (cu_count / 120 of them)
    out, want, mag, e = cascade(dev, 240, 8, gqa, 25, 301, [30, -25, -80, -110, -110] * 5)
    assert np.isfinite(out).all()
    assert (np.abs(out - want) <= e * mag + 2.0 ** -39 * 2.0 ** 33 / 127 * 25 * 64).all()


@pytest.mark.parametrize("gqa", [1, 4])
def test_cascade_small_v_behind_large_v_of_no_weight(dev, gqa):
    out, want, mag, e = cascade(dev, 240, 8, gqa, 25, 302, [20, -30, -60, -95, -100] * 5, [g for g in range(25) if g % 5 < 3])
    # the units of the groups that count: 2^-92 / 127 at most, so 2^(-98 - 14); each weight 2^-25 of it off, times a symbol
    floor = 2.0 ** (-25 - 98 - 14) * 128 * 25 * 64
    assert (np.abs(out - want) <= e * mag + floor).all()
    assert (np.abs(want) > 2 * floor).mean() > 0.9


@pytest.mark.parametrize("gqa", [1, 4])
def test_cascade_scales_behind_the_query(dev, gqa):
    """Queries that end inside the shared prefix, all of them before the pages whose scales are infinite or NaN; then two
    that see them, whose rows alone are NaN."""
    def edit(kvb):
        for h in range(2):
            o = 16 * int(kvb.host_offsets[0, h, 6])
            kvb.pool[o + 56: o + 64] = up(dev, np.array([np.nan, np.inf], np.float32).view(np.uint8))
            kvb.pool[o + 40: o + 48] = up(dev, np.full(2, np.nan, np.float32).view(np.uint8))
    pos = [64 * 6 + 31, 64 * 6 + 3, 64 * 6, 64 * 5 + 40, 64 * 2 + 7] * 4
    out, want, mag, e = cascade(dev, 20, 2, gqa, 10, 303, [0] * 10, pos=pos, edit=edit)
    assert np.isfinite(out).all()
    assert (np.abs(out - want) <= e * mag + 2.0 ** -39 * 8 / 127 * 127 * 640).all()
    pos[7], pos[12] = 64 * 6 + 32, 64 * 10 - 1
    out, _, _, _ = cascade(dev, 20, 2, gqa, 10, 303, [0] * 10, pos=pos, edit=edit)
    nan = np.isnan(out).all(2)
    assert nan[[7, 12]].all() and np.isfinite(out[[i for i in range(20) if i not in (7, 12)]]).all()
