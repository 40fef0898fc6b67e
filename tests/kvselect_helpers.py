"""Plain 64-bit (numpy) forms of the operators of chromofold/kv_select.h for the tests, and their inputs."""
from __future__ import annotations

import numpy as np

NO_UNIT = 0xFFFFFFFF


def bounds_ref(groups):
    """groups: list of [tokens, D] fp32 arrays -> codes [n, 2D] int8, scales [n] fp32 (IEEE fp32 quotients)."""
    codes, scales = [], []
    for k in groups:
        if not np.isfinite(k).all():
            codes.append(np.full(2 * k.shape[1], 127, np.int8))
            scales.append(np.float32(np.inf))
            continue
        s = np.float32(np.abs(k).max() / np.float32(127))
        hi, lo = k.max(0), -k.min(0)
        with np.errstate(all="ignore"):
            c = np.concatenate([np.ceil(hi / s), np.ceil(lo / s)]) if s else np.zeros(2 * k.shape[1], np.float32)
        codes.append(np.clip(c, -127, 127).astype(np.int8))
        scales.append(s)
    return np.array(codes), np.array(scales, np.float32)


def visible_tokens(tokens, pos, max_groups):
    return min(int(tokens), int(pos) + 1, 64 * max_groups)


def scores_ref(q, codes, scales):
    """q [gqa, D] fp32, codes [n, 2D], scales [n] -> fp32 scores [n] (whole numbers exact in 64 bits, two fp32 roundings)."""
    D = q.shape[1]
    with np.errstate(all="ignore"):
        step = (np.fmax.reduce(np.abs(q), 1) / np.float32(127)).astype(np.float32)
        r = q / step[:, None]
        a = np.clip(np.rint(np.where(np.isnan(r), 0, r)), -127, 127).astype(np.int64)
        dot = np.maximum(a, 0) @ codes[:, :D].T.astype(np.int64) + np.maximum(-a, 0) @ codes[:, D:].T.astype(np.int64)
        per_head = step[:, None] * dot.astype(np.float32)
        best = np.fmax.reduce(np.concatenate([per_head, np.full((1, dot.shape[1]), -np.inf, np.float32)]), 0)
        return (best * scales).astype(np.float32)


def pick_ref(values, n, k, first, last):
    """The k of n entries that stay: first and last ones, then the largest (NaN above all, ties to the lower index)."""
    if n <= k:
        return np.arange(n)
    forced = set(range(first)) | set(range(n - last, n))
    v = np.where(np.isnan(values), np.inf, values).astype(np.float64)
    nan = np.isnan(values)
    order = sorted((i for i in range(n) if i not in forced), key=lambda i: (not nan[i], -v[i], i))
    return np.sort(np.array(sorted(forced) + order[: k - len(forced)], np.int64))


def select_ref(q, codes, scales, tokens, pos, gqa, unit, max_units, first, last):
    S, H, M = scales.shape
    out = np.full((S, H, max_units), NO_UNIT, np.uint32)
    for s in range(S):
        vis = visible_tokens(tokens[s], pos[s], M)
        n = -(-vis // 64)
        m = -(-n // unit)
        for h in range(H):
            if not n:
                continue
            sc = scores_ref(q[s, h * gqa:(h + 1) * gqa], codes[s, h, :n], scales[s, h, :n])
            sc = np.concatenate([sc, np.full(m * unit - n, -np.inf, np.float32)]).reshape(m, unit)
            best = np.where(np.isnan(sc).any(1), np.nan, sc.max(1))
            at = pick_ref(best, m, min(m, max_units), first, last)
            out[s, h, : at.size] = at
    return out


def attend_ref(q, k, v, tokens, pos, gqa, scale, units, unit, max_groups, weights=None, decay=1.0):
    """q [S, QH, D]; k, v: per (s, h) dequantised float64 [T, D]; units [S, H, max_units] u32 or None. Returns output,
    weights, and for the tolerances per output element sum_t p |v|, per row the largest sum_d |scale q k|, and per output
    element the error that weights below f16's range make (see weight_floor)."""
    S, QH, D = q.shape
    H = QH // gqa
    out, mag, low = np.zeros((S, QH, D)), np.zeros((S, QH, D)), np.zeros((S, QH, D))
    big = np.zeros((S, QH))
    w = np.zeros((S, H, max_groups)) if weights is None else decay * weights.astype(np.float64)
    for s in range(S):
        vis = visible_tokens(tokens[s], pos[s], max_groups)
        for h in range(H):
            t = np.arange(vis)
            if units is not None:
                t = t[np.isin(t // (64 * unit), units[s, h])]
            if not t.size:
                continue
            kk, vv = k[s][h][t], v[s][h][t]
            low[s, h * gqa: (h + 1) * gqa] = weight_floor(v[s][h], t)
            for g in range(gqa):
                x = q[s, h * gqa + g].astype(np.float64)
                sc = kk @ x * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[s, h * gqa + g] = p @ vv
                mag[s, h * gqa + g] = p @ np.abs(vv)
                big[s, h * gqa + g] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                np.add.at(w[s, h], t // 64, p)
    return out, w, mag, big, low


def weight_floor(v, t):
    """What weights too small for f16 leave out of an output. A weight p vs (vs: its page's V scale, p <= 1 relative to the
    running maximum) is held as two f16 in units of 2^e, e = exponent of the group's largest vs - 15, or of an earlier
    group's larger one, so 2^e <= 2^-14 max vs. The second f16 is off by at most half the least step of f16, 2^-25 (the
    relative part of its error is in tolerance()); its product with a symbol, summed over the tokens, over a sum of p that
    is at least 1: 2^-39 max vs sum_t |symbol|."""
    pages = np.concatenate([v, np.zeros((-v.shape[0] % 16, v.shape[1]))]).reshape(-1, 16, v.shape[1])
    vs = np.abs(pages).max((1, 2)) / 127
    vs = np.where(vs == 0, 1.0, vs)  # a page of zeros has scale 1
    return 2.0 ** -39 * vs[np.unique(t // 16)].max() * (np.abs(v[t]) / vs[t // 16][:, None]).sum(0)


def tolerance(big, D):
    """Bound on the relative error of a softmax weight p, from big = the row's largest sum_d |scale q k|.
      score     q in two f16 parts, the rest of it at most half a step of the second: 2^-22 of |q|; products of f16 are exact
                in fp32; 2 D / 32 accumulations of 32 exact products, each rounded to 2^-24 of a sum that is at most `big`
                (within an accumulation as much again): 4 D / 32 * 2^-24; unit factor, page scale, log2 e and their
                products: 6 * 2^-24 of the score
      weight    exp2 of a difference of the score and the running maximum (each at most big, in units of log2 e): 2^-24 * 2
                big; 2^-23 of itself by the instruction; again when states are joined, at most 3 joins: 3 * (2^-23 + 2^-23 big)
      P.V       the weight in two f16 parts 2^-22, with the V scale 2^-24, and sums as above 4 * 2 * 2^-24 per group, taken
                up by the joins' 2^-22
    numerator and denominator both err: twice."""
    e = big * (2.0 ** -22 + (4 * D / 32 + 6 + 2 + 6) * 2.0 ** -24) + 8 * 2.0 ** -22
    return 2 * e
