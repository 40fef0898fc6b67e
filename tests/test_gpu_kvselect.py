"""The operators of chromofold/kv_select.h on the GPU against their plain 64-bit forms (kvselect_helpers.py): bounds, scores
and selections bit for bit, evicted tables exactly, attention within the bound that kvselect_helpers.tolerance derives."""
import numpy as np
import pytest

import kvselect_helpers as R
from kv_helpers import decoded_pages, make_seqs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def up(dev, a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    return torch.from_numpy(a).to(dev)


def down(t):
    return t.cpu().numpy()


def u32(t):
    return down(t).view(np.uint32)


# ---------------------------------------------------------------------------------------------------- key bounds
def _bound_groups(D, seed):
    rng = np.random.default_rng(seed)
    groups, tokens = [], []
    for i, counts in enumerate([[16, 16, 16, 16], [1], [16, 3], [16, 16, 16, 15], [5, 7, 1, 2], [16, 16, 9], [16] * 4, [2]]):
        k = rng.standard_normal((sum(counts), D)).astype(np.float32) * np.float32(10.0 ** (i - 4))
        groups.append(k)
        tokens.append(counts)
    groups[1] = np.zeros_like(groups[1])
    groups[3][:, : D // 2] = np.abs(groups[3][:, : D // 2])       # channels of one sign
    groups[3][7, 5] = 2.5 * np.abs(groups[3]).max()               # one key far out
    groups[4][2, 1], groups[5][40, D - 1], groups[7][1, 0] = np.nan, np.inf, -np.inf
    groups.append(np.full((3, D), 1e-42, np.float32))             # subnormal
    tokens.append([3])
    groups.append(np.full((16, D), 3.0e38, np.float32))
    tokens.append([16])
    return groups, tokens


@pytest.mark.parametrize("D", [128, 64])
def test_bounds(dev, D):
    import torch
    from chromofold_amd import kvselect as ks
    groups, tokens = _bound_groups(D, D)
    order = np.random.default_rng(1).permutation(len(groups))
    pages, first, counts, tc = [np.full((2, 16, D), np.nan, np.float32)], [], [], [99, 99]
    for k, c in zip(groups, tokens):
        first.append(sum(p.shape[0] for p in pages))
        counts.append(len(c))
        at = 0
        for n in c:
            page = np.full((1, 16, D), np.nan, np.float32)  # rows behind a page's tokens hold anything
            page[0, :n] = k[at: at + n]
            at += n
            pages.append(page)
            tc.append(n)
    slots = 2 * order.astype(np.int64) + 1
    out = ks.KeyBounds(torch.full((1, 1, 2 * len(groups) + 1, 2 * D), 99, dtype=torch.int8, device=dev),
                       torch.full((1, 1, 2 * len(groups) + 1), -7.0, device=dev))
    slots[2] = 1 << 40  # behind the records: skipped
    ks.key_bounds(up(dev, np.concatenate(pages)), up(dev, np.array(first, np.int64)), up(dev, np.array(counts, np.uint32)), out,
                  token_counts=up(dev, np.array(tc, np.uint32)), slots=up(dev, slots))
    codes, scales = R.bounds_ref(groups)
    got_c, got_s = down(out.codes)[0, 0], down(out.scales)[0, 0]
    want_c, want_s = np.full_like(got_c, 99), np.full_like(got_s, -7.0)
    for i, s in enumerate(slots):
        if s < got_s.size:
            want_c[s], want_s[s] = codes[i], scales[i]
    assert np.array_equal(got_s, want_s)
    assert np.array_equal(got_c, want_c)


def test_bounds_bad_counts(dev):
    # page and token counts out of their range: not read, the record of a group that must be looked at
    from chromofold_amd import kvselect as ks
    pages = np.random.default_rng(3).standard_normal((8, 16, 64)).astype(np.float32)
    out = ks.empty_bounds(1, 1, 6, 64, dev)
    ks.key_bounds(up(dev, pages), up(dev, np.array([0, 1 << 50, 2, 3, 4, 4], np.int64)),
                  up(dev, np.array([0, 5, 2, 1, 0xFFFFFFFF, 4], np.uint32)), out,
                  token_counts=up(dev, np.array([16, 16, 16, 17, 16, 16, 16, 0], np.uint32)))
    assert np.isinf(down(out.scales)).all() and (down(out.codes) == 127).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("T", [16, 64, 80, 208, 1024])
def test_bounds_of_dense_keys(dev, D, T):
    from chromofold_amd import kvselect as ks
    k = np.random.default_rng(T + D).standard_normal((3, 2, T, D)).astype(np.float32)
    b = ks.bounds_of(up(dev, k))
    codes, scales = R.bounds_ref([k[s, h, 64 * g: 64 * g + 64] for s in range(3) for h in range(2) for g in range(-(-T // 64))])
    assert np.array_equal(down(b.scales).ravel(), scales)
    assert np.array_equal(down(b.codes).reshape(codes.shape), codes)
    # they bound the keys, up to the scale's rounding
    hi = down(b.codes)[..., :D].astype(np.float64) * down(b.scales)[..., None]
    for g in range(-(-T // 64)):
        assert (k[:, :, 64 * g: 64 * g + 64].max(2) <= hi[:, :, g] * (1 + 2.0 ** -23) + 1e-45).all()


# ---------------------------------------------------------------------------------------------------- selection
def _records(rng, S, H, M, D, spread=1.0):
    codes = rng.integers(-127, 128, (S, H, M, 2 * D)).astype(np.int8)
    return codes, (spread * rng.random((S, H, M)) + 0.01).astype(np.float32)


def _cache(dev, S, H, D, M, tokens):
    import torch
    from chromofold_amd import kv
    return kv.BatchedKv(kv.CODEC_INT8, S, H, D, M, torch.zeros(16, dtype=torch.uint8, device=dev),
                        torch.zeros(S, H, M, dtype=torch.int32, device=dev), up(dev, np.array(tokens, np.uint32)), None)


def _select(dev, codes, scales, q, tokens, pos, unit, max_units, first, last):
    import torch
    from chromofold_amd import kvselect as ks
    S, H, M, D2 = codes.shape
    kvb = _cache(dev, S, H, D2 // 2, M, tokens)
    units = torch.full((S, H, max_units), 12345, dtype=torch.int32, device=dev)
    ks.select(kvb, ks.KeyBounds(up(dev, codes), up(dev, scales)), up(dev, q), up(dev, np.array(pos, np.uint32)), units,
              unit_groups=unit, keep_first=first, keep_last=last)
    return u32(units)


LENS = [0, 1, 63, 64, 65, 640, 1000, 4097, 8191]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("gqa, unit, max_units, first, last", [
    (4, 1, 16, 1, 1), (1, 1, 1, 0, 0), (7, 2, 9, 2, 3), (16, 1, 40, 0, 5), (3, 2, 1, 1, 0), (5, 1, 7, 3, 4), (8, 2, 300, 1, 1)])
def test_select(dev, D, gqa, unit, max_units, first, last):
    rng = np.random.default_rng(100 * D + gqa)
    S, H, M = len(LENS), 3, 131
    codes, scales = _records(rng, S, H, M, D)
    q = rng.standard_normal((S, H * gqa, D)).astype(np.float32)
    pos = [max(0, t - 1) for t in LENS]
    pos[6], pos[8] = 500, 0xFFFFFFFF
    got = _select(dev, codes, scales, q, LENS, pos, unit, max_units, first, last)
    assert np.array_equal(got, R.select_ref(q, codes, scales, LENS, pos, gqa, unit, max_units, first, last))


def test_select_tokens_past_the_table(dev):
    rng = np.random.default_rng(5)
    codes, scales = _records(rng, 2, 1, 20, 64)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    t = [0xFFFFFFFF, 64 * 20 + 1]
    got = _select(dev, codes, scales, q, t, [0xFFFFFFFF] * 2, 1, 6, 1, 1)
    assert np.array_equal(got, R.select_ref(q, codes, scales, t, [0xFFFFFFFF] * 2, 2, 1, 6, 1, 1))


@pytest.mark.parametrize("unit", [1, 2])
def test_select_equal_scores_take_the_lower_index(dev, unit):
    rng = np.random.default_rng(6)
    codes, scales = _records(rng, 1, 2, 700, 128)
    codes[:, :, 1::3], scales[:, :, 1::3] = codes[:, :, 1:2], scales[:, :, 1:2]  # a third of the groups are one
    codes[:, 1], scales[:, 1] = codes[:, 1, :1], scales[:, 1, :1]               # one head: all of them
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    for k in (3, 64, 150):
        got = _select(dev, codes, scales, q, [64 * 700], [64 * 700 - 1], unit, k, 1, 1)
        assert np.array_equal(got, R.select_ref(q, codes, scales, [64 * 700], [64 * 700 - 1], 2, unit, k, 1, 1)), k


def test_select_extreme_values(dev):
    # scales of 0, +inf (a group with a NaN), subnormal and huge; queries of 0, with a NaN, an infinity, huge and tiny ones
    rng = np.random.default_rng(7)
    S, M = 7, 90
    codes, scales = _records(rng, S, 1, M, 64)
    scales[:, :, 3], scales[:, :, 5], scales[:, :, 7], scales[:, :, 9] = 0.0, np.inf, 1e-41, 3e38
    codes[:, :, 5] = 127
    codes[:, :, 3] = 0
    q = rng.standard_normal((S, 3, 64)).astype(np.float32)
    q[1] = 0
    q[2, 1, 5] = np.nan
    q[3, 0, 2] = np.inf
    q[4] *= np.float32(1e37)
    q[5] *= np.float32(1e-40)
    q[6, :, 0] = np.nan, np.inf, -np.inf
    t = [64 * M] * S
    pos = [x - 1 for x in t]
    got = _select(dev, codes, scales, q, t, pos, 1, 11, 1, 2)
    assert np.array_equal(got, R.select_ref(q, codes, scales, t, pos, 3, 1, 11, 1, 2))
    assert (got[:, 0] == 5).any(1)[[0, 1, 2, 4]].all()


@pytest.mark.parametrize("M, unit, S", [(2048, 1, 2), (16384, 2, 1), (40000, 1, 1)])
def test_select_long(dev, M, unit, S):
    # contexts of 131k, 1M and 2.6M tokens; scores within a few binades, within one, and far apart
    rng = np.random.default_rng(M)
    codes, scales = _records(rng, S, 2, M, 64)
    scales[:, 1] = np.exp2(rng.uniform(-60, 60, (S, M))).astype(np.float32)
    q = rng.standard_normal((S, 8, 64)).astype(np.float32)
    t = [64 * M - 37 - 999 * s for s in range(S)]
    pos = [x - 1 for x in t]
    for k in (5, 257, 1500):
        got = _select(dev, codes, scales, q, t, pos, unit, k, 1, 3)
        assert np.array_equal(got, R.select_ref(q, codes, scales, t, pos, 4, unit, k, 1, 3)), k


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("S, H, M, unit, k", [(9, 29, 200, 1, 17),   # more rows than CUs, short: 256 threads a row
                                              (9, 29, 300, 2, 30),   # more rows than CUs: 512
                                              (9, 8, 1100, 1, 101),  # longer rows: 1024
                                              (9, 8, 2200, 2, 300), (9, 29, 4100, 1, 64),  # more units than 512 threads take
                                              (9, 1, 1030, 1, 64)])  # few rows: two launches at D = 128
def test_select_workgroup_sizes(dev, D, S, H, M, unit, k):
    rng = np.random.default_rng(M + D)
    codes, scales = _records(rng, S, H, M, D)
    codes[4, :, 50:], scales[4, :, 50:] = 127, np.inf  # records behind a row's length would rank first
    q = rng.standard_normal((S, 2 * H, D)).astype(np.float32)
    t = [64 * M, 0, 1, 64 * M - 65, 64 * 50, 64 * k + 1, 64 * (M // 2) - 3, 64 * M - 1, 64 * 129]
    pos = [max(0, x - 1) for x in t]
    got = _select(dev, codes, scales, q, t, pos, unit, k, 1, 2)
    assert np.array_equal(got, R.select_ref(q, codes, scales, t, pos, 2, unit, k, 1, 2))


# ---------------------------------------------------------------------------------------------------- attention
class Case:
    """An INT8 (or rANS) cache of given lengths, its dequantised K and V in 64 bits, queries and positions."""

    def __init__(self, dev, lens, H, gqa, D, seed, pos=None, codec=1, raw_groups=None, **how):
        from chromofold_amd import kv
        self.dev, self.lens, self.H, self.gqa, self.D = dev, lens, H, gqa, D
        data = make_seqs([max(t, 1) for t in lens], H, D, seed, **how)
        tables = None
        if codec == 2:
            longest = int(np.argmax(lens))
            tables = np.concatenate([kv.build_table(x[h][: x.shape[1] // 16 * 16].reshape(-1, 16, D)[:32]) for h in range(H)
                                     for x in data[longest]])
        self.kvb = kv.build_batched(codec, lambda s: data[s], len(lens), H, np.array([max(t, 1) for t in lens]), D, tables, dev,
                                    keep_host=True, raw_groups=raw_groups)
        self.kvb.seq_tokens.copy_(up(dev, np.array(lens, np.uint32)))
        self.k, self.v = [], []
        for s, t in enumerate(lens):
            rows = [decoded_pages(self.kvb, s, h, max(t, 1)) for h in range(H)]
            self.k.append([np.concatenate([p[1] for p in r]).astype(np.float64) for r in rows])
            self.v.append([np.concatenate([p[2] for p in r]).astype(np.float64) for r in rows])
        rng = np.random.default_rng(seed + 1)
        self.q = rng.standard_normal((len(lens), H * gqa, D)).astype(np.float32)
        self.pos = [max(0, t - 1) for t in lens] if pos is None else pos
        self.M, self.scale = self.kvb.max_groups, float(1 / np.sqrt(D))
        self.rng = rng

    def lists(self, max_units, unit=1, density=0.5):
        """Ascending units of each row, some of them behind what is visible."""
        out = np.full((len(self.lens), self.H, max_units), R.NO_UNIT, np.uint32)
        m = -(-self.M // unit)
        for s in range(len(self.lens)):
            for h in range(self.H):
                at = np.flatnonzero(self.rng.random(m) < density)[:max_units]
                out[s, h, : at.size] = at
        return out

    def run(self, units=None, unit=1, weights=None, want=True, decay=0.75, splits=0, stream=None):
        import torch
        from chromofold_amd import kvselect as ks
        q = up(self.dev, self.q)
        out = torch.full_like(q, float("nan"))
        w = torch.full((len(self.lens), self.H, self.M), float("nan"), device=self.dev) if want else None
        ks.attention(self.kvb, q, out, up(self.dev, np.array(self.pos, np.uint32)), self.scale,
                     None if units is None else up(self.dev, units), unit, None if weights is None else up(self.dev, weights), w,
                     decay, splits, stream)
        return down(out).astype(np.float64), None if w is None else down(w).astype(np.float64)

    def check(self, units=None, unit=1, weights=None, want=True, decay=0.75, splits=(0,)):
        ref = R.attend_ref(self.q, self.k, self.v, self.lens, self.pos, self.gqa, self.scale, units, unit, self.M, weights, decay)
        for sp in splits:
            self.compare(ref, *self.run(units, unit, weights, want, decay, sp))
        return ref

    def compare(self, ref, out, w):
        o, rw, mag, big, low = ref
        tol = R.tolerance(big, self.D)
        bad = np.abs(out - o) > tol[..., None] * mag + 2.0 ** -23 * np.abs(o) + low
        assert not bad.any(), (np.argwhere(bad)[:3], out[bad][:3], o[bad][:3], mag[bad][:3])
        if w is not None:
            wt = tol.reshape(len(self.lens), self.H, self.gqa).max(2)[..., None]
            bad = np.abs(w - rw) > wt * rw + 4 * 2.0 ** -24 * np.abs(rw) + 1e-37
            assert not bad.any(), (np.argwhere(bad)[:3], w[bad][:3], rw[bad][:3])


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("gqa", [1, 2, 3, 4, 5, 7, 8, 12, 16])
def test_attention_head_counts(dev, D, gqa):
    c = Case(dev, [1, 17, 64, 300, 1029], 2, gqa, D, 10 * gqa + D)
    c.check(splits=(0, 1, 3))
    c.check(c.lists(6), weights=c.rng.random((5, 2, c.M)).astype(np.float32))


@pytest.mark.parametrize("D", [128, 64])
def test_attention_lengths_and_masks(dev, D):
    # empty, one token, page and group edges, query positions inside the context and on its first token
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 1000, 0, 2100]
    pos = [0, 0, 14, 3, 16, 62, 0xFFFFFFFF, 64, 100, 63, 0, 77, 1500]
    c = Case(dev, lens, 2, 4, D, 31 + D, pos)
    for splits in (0, 1, 2, 50):
        ref = c.check(weights=c.rng.random((len(lens), 2, c.M)).astype(np.float32), splits=(splits,))
    assert (ref[0][0] == 0).all()
    for unit in (1, 2):
        c.check(c.lists(9, unit), unit, splits=(0, 1, 4))
    out, w = c.run(np.full((len(lens), 2, 3), R.NO_UNIT, np.uint32))
    assert (out == 0).all() and (w == 0).all()


def test_attention_many_groups_per_wavefront(dev):
    # more slots than the 64 a wavefront looks up at once, with one workgroup per row
    c = Case(dev, [64 * 300 + 5, 64 * 299], 1, 4, 64, 5)
    c.check(splits=(1, 2), weights=c.rng.random((2, 1, c.M)).astype(np.float32))
    c.check(c.lists(290, 1, 0.95), splits=(1,))


@pytest.mark.parametrize("S, H, D, gqa, longest", [(300, 2, 128, 4, 4096), (700, 1, 64, 7, 3300), (1030, 1, 64, 2, 2600)])
@pytest.mark.parametrize("unit", [0, 1, 2])
def test_attention_many_ragged_sequences(dev, S, H, D, gqa, longest, unit):
    """Lengths from nothing to long ones side by side, most rows shorter than a wavefront's stretch of the slots: stretches
    over several rows, rows over several stretches, empty rows inside and at both ends of them (1030 sequences: too many
    for stretches, the splits behind them)."""
    rng = np.random.default_rng(S + unit)
    lens = rng.integers(0, 150, S)
    lens[rng.random(S) < 0.3] = 0
    lens[[0, -1]] = 0
    lens[S // 2] = longest
    lens[S // 3] = 700
    c = Case(dev, [int(t) for t in lens], H, gqa, D, S)
    w = rng.random((S, H, c.M)).astype(np.float32)
    if unit == 0:
        c.check(weights=w)
        c.check(want=False)
    else:
        c.check(c.lists(-(-c.M // unit), unit, 0.6), unit, weights=w)


def test_attention_broken_lists_among_ragged_sequences(dev):
    # entries that do not ascend, in rows that lie in one stretch, across stretches, without a visible unit listed before them
    rng = np.random.default_rng(3)
    S, M = 600, 64
    lens = [int(x) for x in rng.integers(1, 300, S)]
    lens[100], lens[101], lens[400] = 64 * M, 64 * M, 64 * M
    c = Case(dev, lens, 1, 4, 64, 71)
    lists = np.full((S, 1, M), R.NO_UNIT, np.uint32)
    for s in range(S):
        n = -(-lens[s] // 64)
        lists[s, 0, :n] = np.arange(n)
    bad = [100, 400, 7, 250]
    lists[100, 0, 63] = 10
    lists[400, 0, 30] = 60
    for s in (7, 250):
        lens_s = -(-lens[s] // 64)
        lists[s, 0, :2] = [1, 0] if lens_s > 1 else [0, 0]
        if lens_s < 2:
            bad.remove(s)  # one unit can be listed: its entry is all that is read
    out, _ = c.run(lists)
    ok = np.ones(S, bool)
    ok[bad] = False
    assert np.isnan(out[bad]).all() and np.isfinite(out[ok]).all()
    ref = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, c.gqa, c.scale, lists, 1, c.M)
    tol = R.tolerance(ref[3], c.D)
    assert (np.abs(out - ref[0]) <= tol[..., None] * ref[2] + 2.0 ** -23 * np.abs(ref[0]) + ref[4])[ok].all()


def test_attention_weights_forms(dev):
    import torch
    from chromofold_amd import kvselect as ks
    c = Case(dev, [500, 0, 130], 2, 3, 128, 8)
    w0 = c.rng.random((3, 2, c.M)).astype(np.float32)
    lists = c.lists(5)
    c.check(lists, weights=None)
    c.check(lists, want=False)
    ref = c.check(lists, weights=w0, decay=1.0)
    c.check(lists, weights=w0, decay=0.0)
    w = up(dev, w0)  # in place
    out = torch.empty(c.q.shape, device=dev)
    ks.attention(c.kvb, up(dev, c.q), out, up(dev, np.array(c.pos, np.uint32)), c.scale, up(dev, lists), 1, w, w, 1.0)
    c.compare(ref, down(out).astype(np.float64), down(w).astype(np.float64))


def test_attention_magnitudes(dev):
    # whole heads of small or huge V, pages of one group 2^20 apart, huge and tiny queries, keys with outlier channels
    mult = [[1e-2, 1e7], [1e-5, 1e3], [1.0, 1e-30]]
    Case(dev, [700, 640, 130], 2, 4, 128, 41, v_mult=mult).check(splits=(0, 1))
    Case(dev, [700, 640, 130], 2, 4, 64, 42, page_spread=20).check(splits=(0, 1))
    Case(dev, [700, 640, 130], 2, 4, 128, 43, scale_spread=True).check(splits=(0, 1))
    for f in (1e-20, 1e-3, 3e3):
        c = Case(dev, [700, 300], 2, 4, 128, 44)
        c.q *= np.float32(f)
        c.scale /= f if f > 1 else 1.0
        c.check()


def test_attention_near_cancelling_values(dev):
    Case(dev, [1024, 512], 2, 4, 128, 45, cancel=1 / 64).check()


def test_attention_nan_stays_in_its_rows(dev):
    # a query of one head, a page's K scale, and a masked page's scales
    import torch
    c = Case(dev, [200, 200, 200], 2, 4, 128, 46, pos=[199, 199, 99])
    c.q[0, 1, 5] = np.nan
    step = 16 * int(c.kvb.host_offsets[1, 1, 2])
    c.kvb.pool[step + 32: step + 36] = torch.tensor([0, 0, 192, 127], dtype=torch.uint8, device=dev)
    masked = 16 * int(c.kvb.host_offsets[2, 0, 1])
    c.kvb.pool[masked + 32 + 12: masked + 48] = torch.tensor([0, 0, 192, 127], dtype=torch.uint8, device=dev)  # tokens 112 ..
    c.kvb.pool[masked + 48 + 12: masked + 64] = torch.tensor([0, 0, 128, 127], dtype=torch.uint8, device=dev)
    out, w = c.run()
    nan = np.isnan(out).all(2)
    assert nan[0].tolist() == [False, True] + [False] * 6
    assert nan[1].tolist() == [False] * 4 + [True] * 4
    assert not np.isnan(out[2]).any() and not np.isnan(w[2]).any()
    q = c.q.copy()
    c.q[0, 1, 5] = 0
    ref = R.attend_ref(c.q, c.k, c.v, c.lens, c.pos, c.gqa, c.scale, None, 1, c.M, None, 0.75)
    keep = ~np.isnan(q).any(2) & ~nan
    tol = R.tolerance(ref[3], c.D)
    assert (np.abs(out - ref[0]) <= tol[..., None] * ref[2] + 1e-7 * np.abs(ref[0]))[keep].all()


@pytest.mark.parametrize("rows", [[3, 3, 5], [5, 4, 6], [0, 2, 1], [1, R.NO_UNIT, 2]])
def test_attention_lists_that_do_not_ascend(dev, rows):
    c = Case(dev, [640, 640], 2, 4, 128, 47)
    lists = np.full((2, 2, 4), R.NO_UNIT, np.uint32)
    lists[:, :, :3] = [0, 2, 5]
    lists[1, 0, :3] = rows
    for splits in (0, 1, 4):
        out, w = c.run(lists, splits=splits)
        assert np.isnan(out[1, :4]).all() and np.isfinite(out[0]).all() and np.isfinite(out[1, 4:]).all()
        assert np.isfinite(w[0]).all() and np.isnan(w[1, 0]).any()


def test_attention_blobs_that_are_no_int8_groups(dev):
    import torch
    c = Case(dev, [640, 640, 640], 1, 4, 128, 48)
    for s, (at, value) in enumerate([(0, 2), (20, 64)]):
        o = 16 * int(c.kvb.host_offsets[s, 0, 4])
        c.kvb.pool[o + at] = torch.tensor(value, dtype=torch.uint8, device=dev)
    out, _ = c.run()
    assert np.isnan(out[:2]).all() and np.isfinite(out[2]).all()
    lists = np.full((3, 1, 2), R.NO_UNIT, np.uint32)
    lists[..., 0] = 3  # not listed: not looked at
    assert np.isfinite(c.run(lists)[0]).all()


def test_attention_pool_past_32_bits(dev):
    # blobs behind the first 4 GiB, and behind the first 2^31 sixteen-byte steps' sign bit
    import torch
    c = Case(dev, [400, 130], 2, 2, 64, 49)
    ref = c.check()
    size = c.kvb.pool.numel()
    for at in ((5 << 30) + 16, (1 << 35) + 48):
        pool = torch.empty(at + size, dtype=torch.uint8, device=dev)
        pool[at:] = c.kvb.pool[-size:]
        small, off = c.kvb.pool, c.kvb.group_offsets.clone()
        c.kvb.pool = pool
        c.kvb.group_offsets += at // 16 if at // 16 < 2 ** 31 else at // 16 - 2 ** 32
        c.compare(ref, *c.run())
        c.kvb.pool, c.kvb.group_offsets = small, off
        del pool
        torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------------- coded pools
def coded(dev, lens, H, gqa, D, seed, chained, pos=None, raw=None, **how):
    """A RANS_HYBRID cache sealed with chain pairs (as build_batched does) or with groups of their own."""
    from chromofold_amd import kv
    flags = kv.pair_flags
    if not chained:
        kv.pair_flags = lambda g, first_coded=0: np.zeros(np.asarray(g).size, np.uint8)
    try:
        return Case(dev, lens, H, gqa, D, seed, pos, codec=2, raw_groups=raw, **how)
    finally:
        kv.pair_flags = flags


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("gqa", [1, 3, 4])
def test_coded_pairs(dev, D, gqa):
    lens = [0, 1, 17, 64, 65, 130, 1000, 2100, 0]
    pos = [0, 0, 16, 63, 20, 129, 640, 2099, 5]
    c = coded(dev, lens, 2, gqa, D, 80 + gqa, True, pos, raw={6: 3})
    w = c.rng.random((len(lens), 2, c.M)).astype(np.float32)
    c.check(weights=w, splits=(0, 1, 3, 17))
    c.check(c.lists(17, 2), 2, weights=w, splits=(0, 1, 4))
    c.check(c.lists(5, 2), 2, want=False)


@pytest.mark.parametrize("D", [128, 64])
def test_coded_groups_of_their_own(dev, D):
    lens = [1, 64, 200, 1500, 4200]
    c = coded(dev, lens, 2, 4, D, 90, False)
    c.check(weights=c.rng.random((5, 2, c.M)).astype(np.float32), splits=(0, 2))
    for unit in (1, 2):
        c.check(c.lists(20, unit), unit, weights=c.rng.random((5, 2, c.M)).astype(np.float32), splits=(0, 1, 5))


def test_coded_magnitudes_and_long_lists(dev):
    coded(dev, [700, 640, 130], 2, 4, 128, 41, True, v_mult=[[1e-2, 1e7], [1e-5, 1e3], [1.0, 1e-30]]).check(splits=(0, 1))
    c = coded(dev, [64 * 150, 64 * 149 + 1], 1, 4, 64, 91, True)  # more than 64 slots a wavefront
    c.check(splits=(1,), weights=c.rng.random((2, 1, c.M)).astype(np.float32))
    c.check(c.lists(70, 2, 0.95), 2, splits=(1,))


def test_coded_groups_that_continue_a_chain_are_not_single_units(dev):
    c = coded(dev, [640, 640, 640], 2, 4, 128, 92, True)
    lists = np.full((3, 2, 3), R.NO_UNIT, np.uint32)
    lists[:, :, :2] = [0, 4]      # even groups begin their chains
    lists[1, 0, :2] = [0, 3]      # an odd one on its own
    lists[2, 1, :2] = [4, 5]      # a pair, but as two units
    out, w = c.run(lists)
    assert np.isnan(out[1, :4]).all() and np.isnan(out[2, 4:]).all()
    assert np.isfinite(out[0]).all() and np.isfinite(out[1, 4:]).all() and np.isfinite(out[2, :4]).all()
    out, _ = c.run(np.where(lists == R.NO_UNIT, R.NO_UNIT, [[[0, 1, 0]]]).astype(np.uint32), 2)
    assert np.isfinite(out).all()


# ---------------------------------------------------------------------------------------------------- eviction
def _evict_ref(x, tokens, unit, budget, first, last, M):
    got = {"dropped": np.full(x["offsets"].shape, R.NO_UNIT, np.uint32), "tokens": np.array(tokens, np.int64), "at": {}}
    for s, t in enumerate(tokens):
        t = min(t, 64 * M)
        n = -(-t // 64)
        m = -(-n // unit)
        k = min(m, budget)
        got["tokens"][s] = t - 64 * unit * (m - k)
        for h in range(x["offsets"].shape[1]):
            w = np.zeros(m * unit, np.float32)
            w[:n] = x["weights"][s, h, :n]
            w = w.reshape(m, unit)
            w = w[:, 0] if unit == 1 else np.where(np.arange(m) * 2 + 1 < n, w[:, 0] + w[:, 1], w[:, 0])
            units = R.pick_ref(w, m, k, first, last)
            at = (units[:, None] * unit + np.arange(unit)).ravel()
            at = at[at < n]
            got["at"][s, h] = at
            gone = np.setdiff1d(np.arange(n), at)
            got["dropped"][s, h, : gone.size] = x["offsets"][s, h, gone]
    return got


def _evict(dev, x, tokens, unit, budget, first, last, D, place, records=True):
    import torch
    from chromofold_amd import kv, kvselect as ks
    S, H, M = x["offsets"].shape
    off, tok, w = up(dev, x["offsets"]), up(dev, np.array(tokens, np.uint32)), up(dev, x["weights"])
    kvb = kv.BatchedKv(kv.CODEC_INT8, S, H, D, M, torch.zeros(16, dtype=torch.uint8, device=dev), off, tok, None)
    b = ks.KeyBounds(up(dev, x["codes"]), up(dev, x["scales"])) if records else None
    dropped = torch.full((S, H, M), 5, dtype=torch.int32, device=dev)
    # place: which outputs are the inputs of their kind (True: all)
    same = {"offsets", "tokens", "weights", "records"} if place is True else set() if place is False else {place}
    other = lambda t, name: t if name in same else torch.full_like(t, 77)
    to = ks.Evicted(other(off, "offsets"), other(tok, "tokens"), other(w, "weights"),
                    ks.KeyBounds(other(b.codes, "records"), other(b.scales, "records")) if records else None, dropped)
    ks.evict(kvb, w, budget, to, bounds=b, unit_groups=unit, keep_first=first, keep_last=last)
    ref = _evict_ref(x, tokens, unit, budget, first, last, M)
    assert np.array_equal(down(to.seq_tokens).view(np.uint32), ref["tokens"])
    assert np.array_equal(u32(to.dropped), ref["dropped"])
    go, gw = u32(to.group_offsets), down(to.weights)
    for (s, h), at in ref["at"].items():
        n = at.size
        assert np.array_equal(go[s, h, :n], x["offsets"][s, h, at])
        assert np.array_equal(go[s, h, n:], x["offsets"][s, h, n:] if "offsets" in same else np.full(M - n, 77))
        assert np.array_equal(gw[s, h, :n], x["weights"][s, h, at], equal_nan=True) and (gw[s, h, n:] == 0).all()
        if records:
            gc, gs = down(to.bounds.codes)[s, h], down(to.bounds.scales)[s, h]
            assert np.array_equal(gc[:n], x["codes"][s, h, at]) and np.array_equal(gs[:n], x["scales"][s, h, at])
            assert np.array_equal(gc[n:], x["codes"][s, h, n:] if "records" in same else np.full_like(gc[n:], 77))
            assert np.array_equal(gs[n:], x["scales"][s, h, n:] if "records" in same else np.full_like(gs[n:], 77))


def _tables(rng, S, H, M, D):
    x = {"offsets": rng.integers(0, 2 ** 32 - 1, (S, H, M), dtype=np.uint32),
         "weights": np.exp(rng.standard_normal((S, H, M))).astype(np.float32)}
    x["codes"], x["scales"] = _records(rng, S, H, M, D)
    return x


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("unit, budget, first, last", [(1, 8, 1, 2), (1, 1, 0, 1), (2, 5, 2, 1), (2, 33, 0, 33), (1, 300, 4, 9),
                                                       (1, 400, 1, 1), (2, 270, 1, 2)])
def test_evict(dev, place, unit, budget, first, last):
    rng = np.random.default_rng(budget + 10 * unit)
    tokens = [0, 1, 64, 513, 576, 1000, 64 * 301, 64 * 599 + 3, 64 * 600, 64 * 600 + 7]
    x = _tables(rng, len(tokens), 2, 600, 64)
    x["weights"][:, :, ::3] = 0.0  # ties
    _evict(dev, x, tokens, unit, budget, first, last, 64, place)


@pytest.mark.parametrize("D, records", [(128, True), (128, False), (64, False)])
def test_evict_record_sizes(dev, D, records):
    x = _tables(np.random.default_rng(D), 3, 3, 700, D)
    _evict(dev, x, [64 * 700, 64 * 650 - 1, 64], 1, 520, 3, 20, D, True, records)
    _evict(dev, x, [64 * 700, 64 * 650 - 1, 64], 2, 299, 3, 20, D, False, records)


def test_evict_weights_out_of_the_ordinary(dev):
    # NaN ranks first, infinities, negative weights, -0 equals 0, subnormals
    x = _tables(np.random.default_rng(9), 4, 2, 50, 64)
    w = x["weights"]
    w[0, 0, [7, 30]], w[0, 1, [3, 4]] = np.nan, [np.inf, -np.inf]
    w[1] = -w[1]
    w[2, :, ::2], w[2, :, 1::2] = 0.0, -0.0
    w[3] = np.float32(1e-44) * np.arange(50)
    for place in (False, True):
        _evict(dev, x, [3200, 3200, 3190, 3000], 1, 9, 1, 1, 64, place)
        _evict(dev, x, [3200, 3200, 3190, 3000], 2, 4, 1, 1, 64, place)


def test_evict_long(dev):
    x = _tables(np.random.default_rng(10), 1, 2, 20000, 64)
    _evict(dev, x, [64 * 20000 - 5], 1, 12345, 10, 100, 64, True)
    _evict(dev, x, [64 * 20000 - 5], 1, 12345, 10, 100, 64, False)
    _evict(dev, x, [64 * 20000 - 5], 2, 5001, 10, 100, 64, False)


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("H, M, unit, budget", [(2, 500, 1, 301), (2, 1000, 2, 120), (65, 260, 1, 100), (65, 1030, 2, 99)])
def test_evict_workgroup_sizes(dev, place, D, H, M, unit, budget):
    x = _tables(np.random.default_rng(M + H), 4, H, M, D)
    _evict(dev, x, [64 * M, 64 * M - 70, 64 * (budget * unit + 1) - 3, 640], unit, budget, 2, 5, D, place)


@pytest.mark.parametrize("place", ["offsets", "tokens", "weights", "records"])
@pytest.mark.parametrize("S, H, M, unit, budget", [(1, 1, 3000, 1, 1500), (3, 2, 2500, 2, 701), (5, 3, 90, 1, 41),
                                                   (16, 8, 300, 1, 130), (20, 13, 70, 2, 20)])
def test_evict_some_arrays_in_place(dev, place, S, H, M, unit, budget):
    # few rows are moved by several workgroups each, unless one of them reads what another one writes
    rng = np.random.default_rng(S + M)
    x = _tables(rng, S, H, M, 128)
    tokens = [64 * M - int(v) for v in rng.integers(0, 64 * (M // 3), S)]
    _evict(dev, x, tokens, unit, budget, 1, 2, 128, place)


# ---------------------------------------------------------------------------------------------------- together
def _tensors(dev, *arrays):
    return [up(dev, a) for a in arrays]


def test_steps_select_attend_evict(dev):
    """A cache that is read in part and cut back while it is used: bounds while sealing, then steps of selection, attention
    with accumulating weights, an eviction in place, and further steps over the smaller tables, which the other entry point
    reads too."""
    import torch
    from chromofold_amd import kv, kvselect as ks
    S, H, gqa, D, T, K = 3, 2, 4, 128, 64 * 40, 12
    rng = np.random.default_rng(77)
    key = rng.standard_normal((S, H, T, D)).astype(np.float32)
    val = rng.standard_normal((S, H, T, D)).astype(np.float32)
    dk, dv = _tensors(dev, key, val)
    kvb = kv.seal_device(kv.CODEC_INT8, dk, dv, None)
    b = ks.bounds_of(dk)
    M = kvb.max_groups
    pool = down(kvb.pool)
    import oracle as O
    offs = u32(kvb.group_offsets)
    deq = {}
    for s in range(S):
        for h in range(H):
            run = O.kv_decode_run([pool[int(o) * 16:][:65536] for o in offs[s, h]], None, h, D)
            for g, (k_, v_, ksc, vsc, _) in enumerate(run):
                deq[s, h, g] = ((k_.reshape(64, D).astype(np.float64) - 128) * np.repeat(ksc, 16)[:, None],
                                (v_.reshape(64, D).astype(np.float64) - 128) * np.repeat(vsc, 16)[:, None])
    held = [[list(range(M)) for _ in range(H)] for _ in range(S)]  # which original groups each table holds
    codes, scales = R.bounds_ref([key[s, h, 64 * g: 64 * g + 64] for s in range(S) for h in range(H) for g in range(M)])
    codes, scales = codes.reshape(S, H, M, -1), scales.reshape(S, H, M)
    weights = torch.zeros(S, H, M, device=dev)
    want_w = np.zeros((S, H, M))
    units = torch.empty(S, H, K, dtype=torch.int32, device=dev)
    out = torch.empty(S, H * gqa, D, device=dev)
    sc = 1 / np.sqrt(D)
    for step in range(6):
        n = len(held[0][0])
        tokens = [64 * n] * S
        pos = up(dev, np.array([t - 1 for t in tokens], np.uint32))
        q = rng.standard_normal((S, H * gqa, D)).astype(np.float32)
        dq = up(dev, q)
        ks.select(kvb, b, dq, pos, units, keep_first=1, keep_last=2)
        want = R.select_ref(q, np.stack([[codes[s, h][held[s][h]] for h in range(H)] for s in range(S)]),
                            np.stack([[scales[s, h][held[s][h]] for h in range(H)] for s in range(S)]), tokens,
                            [t - 1 for t in tokens], gqa, 1, K, 1, 2)
        assert np.array_equal(u32(units), want)
        ks.attention(kvb, dq, out, pos, sc, units, 1, weights, weights, 0.9)
        k = [[np.concatenate([deq[s, h, g][0] for g in held[s][h]]) for h in range(H)] for s in range(S)]
        v = [[np.concatenate([deq[s, h, g][1] for g in held[s][h]]) for h in range(H)] for s in range(S)]
        o, w, mag, big, _ = R.attend_ref(q, k, v, tokens, [t - 1 for t in tokens], gqa, sc, want, 1, M, want_w, 0.9)
        tol = R.tolerance(big, D)
        assert (np.abs(down(out) - o) <= tol[..., None] * mag + 2.0 ** -23 * np.abs(o)).all()
        assert np.allclose(down(weights), w, rtol=2 * tol.max() * (step + 1), atol=1e-30)
        want_w = down(weights).astype(np.float64)
        if step == 2:
            ks.evict(kvb, weights, 25, bounds=b, keep_first=1, keep_last=2)
            for s in range(S):
                for h in range(H):
                    at = R.pick_ref(want_w[s, h].astype(np.float32), n, 25, 1, 2)
                    held[s][h] = [held[s][h][i] for i in at]
                    want_w[s, h] = np.concatenate([want_w[s, h][at], np.zeros(M - 25)])
            assert np.array_equal(down(weights), want_w) and (down(kvb.seq_tokens) == 64 * 25).all()
    # everything that is left, through this entry point and the batched one
    ks.attention(kvb, dq, out, pos, sc)
    full = down(out)
    o, _, mag, big, _ = R.attend_ref(q, k, v, tokens, [t - 1 for t in tokens], gqa, sc, None, 1, M)
    assert (np.abs(full - o) <= R.tolerance(big, D)[..., None] * mag + 2.0 ** -23 * np.abs(o)).all()
    kvb.attention(dq, out, pos, sc)
    assert np.abs(down(out) - full).max() <= 1e-3 * np.abs(full).max()


@pytest.mark.parametrize("chained", [True, False])
def test_coded_cache_after_an_eviction(dev, chained):
    """A rANS cache cut back by its attention weights, as chain pairs or as groups of their own, and what both attention
    calls and a selection make of the tables that remain; ragged sequences, one below the budget, one with a cut last page."""
    import torch
    from chromofold_amd import kvselect as ks
    unit = 2 if chained else 1
    lens = [64 * 41, 64 * 30 + 21, 300, 64 * 44 + 1]
    c = coded(dev, lens, 2, 4, 128, 95, chained)
    S, H, M = len(lens), 2, c.M
    q, w, out = up(dev, c.q), torch.zeros(S, H, M, device=dev), torch.empty(c.q.shape, device=dev)
    pos = up(dev, np.array(c.pos, np.uint32))
    ks.attention(c.kvb, q, out, pos, c.scale, weights=w, weights_out=w)
    weights = down(w)
    dropped = torch.empty(S, H, M, dtype=torch.int32, device=dev)
    budget = 20 // unit
    ks.evict(c.kvb, w, budget, ks.Evicted(c.kvb.group_offsets, c.kvb.seq_tokens, w, None, dropped), unit_groups=unit,
             keep_first=1, keep_last=2)
    tokens, kept = [], {}
    for s, t in enumerate(lens):
        n = -(-t // 64)
        m = -(-n // unit)
        k = min(m, budget)
        tokens.append(t - 64 * unit * (m - k))
        for h in range(H):
            x = np.zeros(m * unit, np.float32)
            x[:n] = weights[s, h, :n]
            units = R.pick_ref(x.reshape(m, unit).sum(1, dtype=np.float32), m, k, 1, 2)
            at = (units[:, None] * unit + np.arange(unit)).ravel()
            kept[s, h] = at[at < n]
    assert down(c.kvb.seq_tokens).tolist() == tokens
    assert (u32(dropped)[0] != R.NO_UNIT).sum(1).tolist() == [41 - len(kept[0, 0]), 41 - len(kept[0, 1])]
    pick = lambda x, s, h: np.concatenate([x[s][h][64 * g: 64 * g + 64] for g in kept[s, h]])  # noqa: E731
    k = [[pick(c.k, s, h) for h in range(H)] for s in range(S)]
    v = [[pick(c.v, s, h) for h in range(H)] for s in range(S)]
    at = [t - 1 for t in tokens]
    pos.copy_(up(dev, np.array(at, np.uint32)))
    o, _, mag, big, low = R.attend_ref(c.q, k, v, tokens, at, 4, c.scale, None, 1, M)
    bound = R.tolerance(big, 128)[..., None] * mag + 2.0 ** -23 * np.abs(o) + low
    ks.attention(c.kvb, q, out, pos, c.scale)
    assert (np.abs(down(out) - o) <= bound).all()
    c.kvb.attention(q, out, pos, c.scale)
    from kv_helpers import head_err
    assert head_err(down(out), o) <= 1e-3
    lists = np.full((S, H, 3), R.NO_UNIT, np.uint32)
    lists[:, :, :2] = [0, 2]
    o, _, mag, big, low = R.attend_ref(c.q, k, v, tokens, at, 4, c.scale, lists, unit, M)
    ks.attention(c.kvb, q, out, pos, c.scale, up(dev, lists), unit)
    assert (np.abs(down(out) - o) <= R.tolerance(big, 128)[..., None] * mag + 2.0 ** -23 * np.abs(o) + low).all()


def test_a_step_in_a_graph(dev):
    """Selection, attention with weights in place and eviction captured into a graph and replayed with eager work between
    the replays: every replay gives what the eager calls give on the same inputs."""
    import torch
    from chromofold_amd import kvselect as ks
    c = Case(dev, [64 * 30, 64 * 12 + 5, 0], 2, 4, 128, 60)
    S, H, M, K = 3, 2, c.M, 6
    k = [np.concatenate([x, np.zeros((64 * M - x.shape[0], c.D))]) for s in range(S) for x in c.k[s]]
    codes, scales = R.bounds_ref([x[64 * g: 64 * g + 64].astype(np.float32) for x in k for g in range(M)])
    b = ks.KeyBounds(up(dev, codes.reshape(S, H, M, -1)), up(dev, scales.reshape(S, H, M)))
    q, pos = up(dev, c.q), up(dev, np.array(c.pos, np.uint32))
    units = torch.empty(S, H, K, dtype=torch.int32, device=dev)
    out, w, w2 = torch.empty_like(q), torch.zeros(S, H, M, device=dev), torch.zeros(S, H, M, device=dev)
    to = ks.Evicted(torch.zeros_like(c.kvb.group_offsets), torch.zeros_like(c.kvb.seq_tokens), torch.zeros_like(w),
                    ks.KeyBounds(torch.zeros_like(b.codes), torch.zeros_like(b.scales)), torch.zeros_like(c.kvb.group_offsets))

    def step(weights):
        ks.select(c.kvb, b, q, pos, units)
        ks.attention(c.kvb, q, out, pos, c.scale, units, 1, weights, weights, 0.5)
        ks.evict(c.kvb, weights, 10, to, bounds=b)

    def results():
        torch.cuda.synchronize()
        return [x.clone() for x in (units, out, to.group_offsets, to.seq_tokens, to.weights, to.bounds.codes, to.dropped)]

    step(w2)  # modules loaded before the capture
    torch.cuda.synchronize()
    w2.zero_()
    side = torch.cuda.Stream(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        step(w)
        graph.capture_end()
    rng = np.random.default_rng(61)
    for _ in range(4):
        q.copy_(up(dev, rng.standard_normal(c.q.shape).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        got = results()
        (torch.randn(1 << 20, device=dev) ** 2).sum().item()
        step(w2)
        for a, e in zip(got, results()):
            assert torch.equal(a, e)
        assert torch.equal(w, w2)


@pytest.mark.parametrize("S, H, longest", [(300, 2, 4096), (260, 2, 500)])
def test_attention_of_ragged_batches_in_a_graph(dev, S, H, longest):
    """The cuts by device-side lengths in a graph: replays follow the lengths, positions and lists of the moment, with eager
    calls (their own workspaces) between them."""
    import torch
    from chromofold_amd import kvselect as ks
    rng = np.random.default_rng(S)
    lens = [int(x) for x in rng.integers(1, 200, S)]
    lens[7] = longest
    c = Case(dev, lens, H, 4, 64, 63)
    q, pos, w = up(dev, c.q), up(dev, np.array(c.pos, np.uint32)), torch.rand(S, H, c.M, device=dev)
    out, w_out, out2, w_out2 = torch.empty_like(q), torch.empty_like(w), torch.empty_like(q), torch.empty_like(w)
    units = up(dev, c.lists(c.M, 1, 0.7))

    def call(o, wo, u):
        ks.attention(c.kvb, q, o, pos, c.scale, u, 1, w, wo, 0.5)

    for u in (None, units):
        call(out2, w_out2, u)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
        with torch.cuda.stream(side):
            graph.capture_begin()
            call(out, w_out, u)
            graph.capture_end()
        for k in range(4):
            cut = rng.integers(0, np.array(lens) + 1).astype(np.uint32)
            cut[7] = longest - 100 * k
            c.kvb.seq_tokens.copy_(up(dev, cut))
            pos.copy_(up(dev, rng.integers(0, np.array(lens) + 50).astype(np.uint32)))
            units.copy_(up(dev, c.lists(c.M, 1, 0.3 + 0.2 * k)))
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            (torch.randn(1 << 20, device=dev) ** 2).sum().item()
            call(out2, w_out2, u)
            torch.cuda.synchronize()
            assert torch.equal(out, out2) and torch.equal(w_out, w_out2) and torch.isfinite(out).all()


def test_two_streams_with_one_descriptor(dev):
    import torch
    from chromofold_amd import kvselect as ks
    c = Case(dev, [64 * 40] * 4, 2, 4, 64, 62)
    k = [x for s in range(4) for x in c.k[s]]
    codes, scales = R.bounds_ref([x[64 * g: 64 * g + 64].astype(np.float32) for x in k for g in range(c.M)])
    b = ks.KeyBounds(up(dev, codes.reshape(4, 2, c.M, -1)), up(dev, scales.reshape(4, 2, c.M)))
    q, pos = up(dev, c.q), up(dev, np.array(c.pos, np.uint32))
    units, out, w = torch.empty(4, 2, 9, dtype=torch.int32, device=dev), torch.empty_like(q), torch.empty(4, 2, c.M, device=dev)
    sd = ks.select_desc(c.kvb, b, q, pos, units)
    ad = ks.attention_desc(c.kvb, q, out, pos, c.scale, units=units, weights_out=w)
    ks.select(c.kvb, b, q, pos, units, desc=sd)
    ks.attention(c.kvb, q, out, pos, c.scale, desc=ad)
    torch.cuda.synchronize()
    want = [x.clone() for x in (units, out, w)]
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    for _ in range(10):
        for st in streams:
            ks.select(c.kvb, b, q, pos, units, desc=sd, stream=st)
            ks.attention(c.kvb, q, out, pos, c.scale, desc=ad, stream=st)
    torch.cuda.synchronize()
    for a, e in zip((units, out, w), want):
        assert torch.equal(a, e)
