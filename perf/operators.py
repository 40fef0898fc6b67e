"""The operators of a decode step that attends only a part of its 8-bit paged cache, as calls to be timed and compared:

  bounds   cf_kv_key_bounds_async                  per 64-token group and KV head, the largest and smallest key of each
                                                   channel as 8-bit codes with one scale
  select   cf_kv_select_groups_async               per (sequence, KV head), the groups whose bound on q.k is largest
  attend   cf_kv_paged_attention_selected_async    attention over the selected groups (or all of them) of an INT8 pool,
                                                   and the groups' accumulated attention weight
  evict    cf_kv_evict_groups_async                drops the groups of least accumulated weight from the page tables

`run` computes them in elementary torch operations in 32 bits, or, where `own` is set, through the library.
Group tables, lengths and selections are u32 bit patterns in int32 tensors, as everywhere in this package."""
import math

import numpy as np
import torch

own = False

GROUP, PAGE, NONE = 64, 16, -1  # tokens of a group and of a page; the entry behind a selection's last (0xFFFFFFFF)
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    llama = {"H": 8, "gqa": 4, "D": 128}  # Llama-3-8B layer shape: 32 query heads, 8 KV heads, head_dim 128
    return [
        # one decode step seals one group per KV head of one sequence: latency
        {"name": "bounds_step", "op": "bounds", "S": 1, "H": 8, "D": 128, "lo": 64, "hi": 64},
        # the prompts of a ragged batch sealed at once, groups and pages cut short
        {"name": "bounds_prompts", "op": "bounds", "S": 12, "H": 8, "D": 128, "lo": 333, "hi": 8191},
        # one sequence at 4k tokens: latency
        {"name": "select_one_4k", "op": "select", **llama, "S": 1, "lo": 4096, "hi": 4096, "units": 16, "unit": 1, "first": 1, "last": 1},
        # a serving batch at up to 32k tokens, one slot of the batch empty
        {"name": "select_batch_32k", "op": "select", **llama, "S": 32, "lo": 2048, "hi": 32768, "units": 64, "unit": 1, "first": 1, "last": 2, "padded": True},
        # few long contexts, chain pairs of a coded pool as units
        {"name": "select_4x131k", "op": "select", **llama, "S": 4, "lo": 131072, "hi": 131072, "units": 96, "unit": 2, "first": 1, "last": 1},
        # one sequence attends 32 of its groups: latency
        {"name": "attend_one", "op": "attend", **llama, "S": 1, "lo": 8192, "hi": 8192, "units": 32, "unit": 1, "weights": True},
        # the serving batch's step over 64 groups of each head, weights kept for eviction
        {"name": "attend_batch", "op": "attend", **llama, "S": 32, "lo": 3000, "hi": 32768, "units": 64, "unit": 1, "weights": True, "padded": True},
        # 14 query heads over 2 KV heads of 64 dims, whole ragged caches of a larger batch
        {"name": "attend_hd64_ragged", "op": "attend", "H": 2, "gqa": 7, "D": 64, "S": 48, "lo": 150, "hi": 8000, "units": 0, "unit": 1, "weights": True},
        # the full caches of the batch at 32k tokens: bandwidth
        {"name": "attend_all_32k", "op": "attend", **llama, "S": 32, "lo": 32768, "hi": 32768, "units": 0, "unit": 1, "weights": True},
        # one sequence has run over its budget by one group: latency
        {"name": "evict_one", "op": "evict", "S": 1, "H": 8, "D": 128, "lo": 4160, "hi": 4160, "budget": 64, "unit": 1, "first": 1, "last": 2},
        # a batch cut back to half of its cache, some sequences below the budget already
        {"name": "evict_batch", "op": "evict", "S": 32, "H": 8, "D": 128, "lo": 8000, "hi": 32768, "budget": 256, "unit": 1, "first": 2, "last": 8},
        # long contexts of a pool of chain pairs
        {"name": "evict_4x131k", "op": "evict", "S": 4, "H": 8, "D": 128, "lo": 100001, "hi": 131072, "budget": 512, "unit": 2, "first": 1, "last": 4},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bounds", "select", "attend", "evict"])
    c = {"op": op, "D": rng.choice([64, 128]), "H": rng.choice([1, 2, 3, 4, 5, 8]), "S": _spread(rng, 1, 48)}
    most = {"bounds": 1 << 18, "select": 1 << 20, "attend": 1 << 19, "evict": 1 << 20}[op]
    # a selection needs more groups than it takes
    c["hi"] = min(_spread(rng, 1024 if op == "select" else 1, 131072), max(1, most // c["S"]))
    c["lo"] = max(1, int(c["hi"] * rng.uniform(0.05, 1.0)))
    if op == "bounds":
        return c
    c["unit"] = rng.choice([1, 1, 2])
    n = -(-c["hi"] // (GROUP * c["unit"]))
    if op == "evict":
        c["first"], c["last"] = rng.choice([0, 1, 2]), rng.choice([1, 2, 5])
        c["budget"] = c["first"] + c["last"] + int(n * rng.uniform(0.1, 0.9))
        return c
    c["gqa"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    c["padded"] = rng.random() < 0.3
    if op == "select":
        c["first"], c["last"] = rng.choice([0, 1, 2]), rng.choice([0, 1, 3])
        c["units"] = min(n - 1, c["first"] + c["last"] + _spread(rng, 1, max(2, n // 2)))
    else:
        c["units"] = rng.choice([0, max(1, int(n * rng.uniform(0.05, 0.7)))])
        c["weights"] = rng.random() < 0.7
    return c


def _lens(c):
    """Tokens of each sequence: spread over [lo, hi], the longest among them, the last one empty in a padded batch."""
    S = c["S"]
    t = [c["hi"] - (c["hi"] - c["lo"]) * ((7 * i) % S) // max(1, S - 1) for i in range(S)]
    if c.get("padded") and S > 1:
        t[-1] = 0
    return t


def _groups(c):
    return [-(-t // GROUP) for t in _lens(c)]


def _max_groups(c):
    return max(_groups(c))


def _attended(c):
    """Groups attended per KV head of each sequence."""
    if not c["units"]:
        return _groups(c)
    return [min(g, c["units"] * c["unit"]) for g in _groups(c)]


def work(c):
    S, H, D, n = c["S"], c["H"], c["D"], sum(_groups(c))
    record = 2 * D + 4  # codes and scale of one group
    if c["op"] == "bounds":
        tokens = H * sum(_lens(c))
        return {"bytes": 4 * D * tokens + H * n * (record + 16), "flops": 2 * D * tokens}
    if c["op"] == "select":
        q, most = 4 * H * c["gqa"] * D * S, min(c["units"], -(-_max_groups(c) // c["unit"]))
        return {"bytes": H * n * record + q + 4 * S * H * most + 8 * S, "flops": 4 * D * c["gqa"] * H * n}
    if c["op"] == "attend":
        g, q = H * sum(_attended(c)), 4 * H * c["gqa"] * D * S
        return {"bytes": g * (64 + 2 * GROUP * D + 4 + (4 if c["units"] else 0)) + 2 * q + (8 * H * n if c["weights"] else 0) + 8 * S,
                "flops": 4 * D * GROUP * c["gqa"] * g}
    kept = [min(g, c["unit"] * c["budget"]) for g in _groups(c)]
    return {"bytes": H * (4 * n + sum(kept) * (2 * record + 4 + 4 + 4) + 4 * sum(a - b for a, b in zip(_groups(c), kept))) + 8 * S,
            "flops": H * n}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _u32(values):
    return torch.tensor(values, dtype=torch.int64, device=DEV).to(torch.int32)


def _keys(g, H, T, D):
    """Keys [H, T, D] of one sequence: noise around a direction that holds for 256 tokens, channels of unequal size."""
    topic = torch.randn(H, -(-T // 256), D, generator=g, device=DEV).repeat_interleave(256, 1)[:, :T]
    size = torch.exp(0.4 * torch.randn(H, 1, D, generator=g, device=DEV))
    return (topic + torch.randn(H, T, D, generator=g, device=DEV)) * size


def _queries(c, g, like=None):
    q = torch.randn(c["S"], c["H"], c["gqa"], c["D"], generator=g, device=DEV)
    if like is not None:
        q = 0.7 * q + 0.6 * like[:, :, None]
    return q.reshape(c["S"], c["H"] * c["gqa"], c["D"])


def _positions(c):
    """Query positions: the last token of each sequence; in batches the second sequence asks from inside its context."""
    t = _lens(c)
    p = [max(0, x - 1) for x in t]
    if c["S"] > 2:
        p[1] = max(0, t[1] - 1 - t[1] // 3)
    return p


def _codes_of(keys, T):
    """The 8-bit bounds of keys [H, T, D] in groups: codes [H, groups, 2D] int8 and scales [H, groups]."""
    H, _, D = keys.shape
    n = -(-T // GROUP)
    pad = n * GROUP - T
    k = torch.cat([keys, keys[:, -1:].expand(H, pad, D)], 1).view(H, n, GROUP, D)
    hi, lo = k.amax(2), k.amin(2)
    scale = (torch.maximum(hi, -lo).amax(2).double() / 127).float()
    hi = torch.ceil((hi.double() / scale[..., None].double()).float()).clamp(-127, 127)
    lo = torch.ceil((-lo.double() / scale[..., None].double()).float()).clamp(-127, 127)
    return torch.cat([hi, lo], 2).to(torch.int8), scale


def _quantised(x):
    """x [H, T, D], T a multiple of 16, as int8 values with a scale per page: [H, T, D] int8, [H, T / 16]."""
    H, T, D = x.shape
    p = x.view(H, T // PAGE, PAGE * D)
    s = (p.abs().amax(2).double() / 127).float()
    s = torch.where(s == 0, torch.ones_like(s), s)
    return torch.round(p / s[..., None]).clamp(-128, 127).to(torch.int8).view(H, T, D), s


def _sequence(c, seed, s):
    """Symbols and scales of sequence s (K, K scales, V, V scales; tokens padded to whole groups with zeros), and the
    mean key of each head."""
    T, H, D = _lens(c)[s], c["H"], c["D"]
    g = _gen(seed * 1000003 + s)
    n = -(-T // GROUP)
    K = torch.zeros(H, n * GROUP, D, device=DEV)
    V = torch.zeros(H, n * GROUP, D, device=DEV)
    K[:, :T] = 0.35 * _keys(g, H, T, D)
    V[:, :T] = torch.randn(H, T, D, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(H, T, 1, generator=g, device=DEV))
    return *_quantised(K), *_quantised(V), K[:, T // 2 : T // 2 + 1].mean(1)


def _packed(c, kq, ks, vq, vs, T):
    """INT8 group blobs [H, groups, 64 + 128 D] (u8) of one sequence (layout: chromofold/kv_codec_ext.h)."""
    H, D = c["H"], c["D"]
    n = kq.shape[1] // GROUP
    head = torch.zeros(H, n, 64, dtype=torch.uint8, device=DEV)
    left = (T - GROUP * torch.arange(n, device=DEV)[:, None] - PAGE * torch.arange(4, device=DEV)[None]).clamp(0, PAGE)
    head[..., 0] = 1  # INT8
    head[..., 12:20] = left.to(torch.int16).view(torch.uint8).view(1, n, 8)
    head[..., 20] = D
    head[..., 22] = (left > 0).sum(1).to(torch.uint8)
    head[..., 32:48] = ks.reshape(H, n, 4).contiguous().view(torch.uint8)
    head[..., 48:64] = vs.reshape(H, n, 4).contiguous().view(torch.uint8)
    k = (kq.to(torch.int16) + 128).to(torch.uint8).view(H, n, GROUP, D // 4, 4).permute(0, 1, 3, 2, 4)
    v = (vq.to(torch.int16) + 128).to(torch.uint8).view(H, n, 4, 4, 4, D // 16, 16).permute(0, 1, 3, 5, 2, 6, 4)
    return torch.cat([head, k.reshape(H, n, -1), v.reshape(H, n, -1)], 2)


def _chosen(c, seed, s):
    """Units of sequence s to attend, per head [H, units]: ascending, first and last among them, none behind the visible."""
    visible = min(_lens(c)[s], _positions(c)[s] + 1)
    n = -(-visible // (GROUP * c["unit"]))
    k = min(n, c["units"])
    key = torch.rand(c["H"], n, generator=_gen(seed * 999983 + s), device=DEV)
    if n:
        key[:, [0, -1]] = 2.0
    at = key.topk(k, 1).indices.sort(1).values
    return torch.cat([at, torch.full((c["H"], c["units"] - k), NONE, device=DEV)], 1).to(torch.int32)


def _page_tables(c, seed):
    """Offsets [S, H, max_groups] of a pool's blobs in no order, as after a while of serving."""
    S, H, M = c["S"], c["H"], _max_groups(c)
    step = (64 + 2 * GROUP * c["D"]) // 16
    off = torch.randperm(S * H * M, generator=_gen(seed + 5), device=DEV).view(S, H, M) * step
    have = torch.arange(M, device=DEV)[None, None] < torch.tensor(_groups(c), device=DEV)[:, None, None]
    return (off * have).to(torch.int32)


def _evict_inputs(c, seed):
    S, H, M, g = c["S"], c["H"], _max_groups(c), _gen(seed)
    have = torch.arange(M, device=DEV)[None, None] < torch.tensor(_groups(c), device=DEV)[:, None, None]
    w = torch.exp(2 * torch.randn(S, H, M, generator=g, device=DEV)) * (torch.rand(S, H, M, generator=g, device=DEV) > 0.3)
    codes = torch.randint(-127, 128, (S, H, M, 2 * c["D"]), generator=g, device=DEV, dtype=torch.int8)
    return {"offsets": _page_tables(c, seed), "tokens": _u32(_lens(c)), "weights": w * have, "codes": codes,
            "scales": torch.rand(S, H, M, generator=g, device=DEV) + 0.01}


def prepare(case, seed):
    c, st = case, {"case": case}
    S, H, D, M = c["S"], c["H"], c["D"], _max_groups(c)
    if c["op"] == "evict":
        return {**st, **_evict_inputs(c, seed)}
    if c["op"] == "bounds":
        pages, first, counts, tokens, slots = [], [], [], [], []
        at = 0
        for s, T in enumerate(_lens(c)):
            n = -(-T // PAGE)
            k = torch.zeros(H, n * PAGE, D, device=DEV)
            k[:, :T] = _keys(_gen(seed * 1000003 + s), H, T, D)
            pages.append(k.view(H * n, PAGE, D))
            for h in range(H):
                tokens += [PAGE] * (n - 1) + [T - PAGE * (n - 1)]
                for g in range(-(-n // 4)):
                    first.append(at + h * n + 4 * g)
                    counts.append(min(4, n - 4 * g))
                    slots.append((s * H + h) * M + g)
            at += H * n
        return {**st, "keys": torch.cat(pages), "first": torch.tensor(first, device=DEV), "counts": _u32(counts),
                "tokens": _u32(tokens), "slots": torch.tensor(slots, device=DEV)}
    st["tokens"], st["pos"] = _u32(_lens(c)), _u32(_positions(c))
    if c["op"] == "select":
        codes = torch.zeros(S, H, M, 2 * D, dtype=torch.int8, device=DEV)
        scales = torch.zeros(S, H, M, device=DEV)
        like = torch.zeros(S, H, D, device=DEV)
        for s, T in enumerate(_lens(c)):
            if T:
                k = _keys(_gen(seed * 1000003 + s), H, T, D)
                codes[s, :, : -(-T // GROUP)], scales[s, :, : -(-T // GROUP)] = _codes_of(k, T)
                like[s] = k[:, T // 2]
        return {**st, "codes": codes, "scales": scales, "queries": _queries(c, _gen(seed), like)}
    # attend
    at = _page_tables(c, seed)
    step = 64 + 2 * GROUP * D
    pool = torch.zeros(S * H * M * step, dtype=torch.uint8, device=DEV)
    like = torch.zeros(S, H, D, device=DEV)
    for s, T in enumerate(_lens(c)):
        if T:
            *kv, like[s] = _sequence(c, seed, s)
            n = -(-T // GROUP)
            pool.view(-1, step)[at[s, :, :n].long().reshape(-1) // (step // 16)] = _packed(c, *kv, T).view(H * n, step)
    units = torch.stack([_chosen(c, seed, s) for s in range(S)]) if c["units"] else None
    w = torch.rand(S, H, M, generator=_gen(seed + 9), device=DEV) if c["weights"] else None
    return {**st, "pool": pool, "offsets": at, "queries": _queries(c, _gen(seed), like), "units": units, "weights": w,
            "scale": 1 / math.sqrt(D), "decay": 0.95}


# ------------------------------------------------------------------------------------------------ plain forms
def _largest(key, forced, n, k):
    """Of n [..., 1] leading entries of key [..., m] the k [..., 1] largest, those of `forced` before all others, ties to
    the lowest index: their indices ascending [..., m], the rest set to m."""
    m = key.shape[-1]
    i = torch.arange(m, device=key.device)
    key = torch.where(forced, torch.full_like(key, math.inf), key).masked_fill(i >= n, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    return torch.where((i < k) & (i < n), order, torch.full_like(order, m)).sort(-1).values


def _forced(m, n, first, last):
    i = torch.arange(m, device=DEV)
    return (i < first) | ((i >= n - last) & (i < n))


def _plain_bounds(st):
    c, keys = st["case"], st["keys"]
    page = st["first"][:, None] + torch.arange(4, device=DEV)
    there = (torch.arange(4, device=DEV) < st["counts"][:, None])
    page = torch.where(there, page, torch.zeros_like(page))
    seen = there[..., None] & (torch.arange(PAGE, device=DEV) < st["tokens"][page][..., None])
    k = keys[page]
    hi = k.masked_fill(~seen[..., None], -math.inf).amax((1, 2))
    lo = (-k).masked_fill(~seen[..., None], -math.inf).amax((1, 2))
    scale = (torch.maximum(hi, lo).amax(1).double() / 127).float()
    code = torch.ceil(torch.cat([hi, lo], 1) / scale[:, None]).clamp(-127, 127).to(torch.int8)
    rows = c["S"] * c["H"] * _max_groups(c)
    codes = torch.zeros(rows, 2 * c["D"], dtype=torch.int8, device=DEV)
    scales = torch.zeros(rows, device=DEV)
    codes[st["slots"]], scales[st["slots"]] = code, scale
    shape = (c["S"], c["H"], _max_groups(c))
    return {"codes": codes.view(*shape, -1), "scales": scales.view(shape)}


def _plain_select(st):
    c = st["case"]
    S, H, G, D, M, u = c["S"], c["H"], c["gqa"], c["D"], _max_groups(c), c["unit"]
    q = st["queries"].view(S, H, G, D)
    qs = (q.abs().amax(-1, keepdim=True).double() / 127).float()
    code = torch.round(q / torch.where(qs == 0, torch.ones_like(qs), qs)).clamp(-127, 127)
    part = torch.cat([code.clamp(min=0), (-code).clamp(min=0)], -1)
    dot = torch.matmul(part, st["codes"].float().transpose(2, 3).contiguous())  # whole numbers below 2^24: exact
    score = (dot * qs).amax(2) * st["scales"]
    visible = torch.minimum(st["tokens"], st["pos"] + 1)[:, None, None]
    score = score.masked_fill(torch.arange(M, device=DEV) * GROUP >= visible, -math.inf)
    m = -(-M // u)
    score = torch.nn.functional.pad(score, (0, m * u - M), value=-math.inf).view(S, H, m, u).amax(-1)
    n = (visible + GROUP * u - 1) // (GROUP * u)
    at = _largest(score, _forced(m, n, c["first"], c["last"]), n, torch.clamp(n, max=c["units"]))
    at = torch.nn.functional.pad(at, (0, max(0, c["units"] - m)), value=m)[..., : c["units"]]
    return {"units": torch.where(at == m, torch.full_like(at, NONE), at).to(torch.int32)}


def _plain_attend(st):
    c = st["case"]
    S, H, G, D, M, u = c["S"], c["H"], c["gqa"], c["D"], _max_groups(c), c["unit"]
    if st["units"] is None:
        group = torch.arange(M, device=DEV).expand(S, H, M)
    else:
        t = st["units"].long()
        group = torch.where(t >= 0, t * u, torch.full_like(t, M + 1))[..., None] + torch.arange(u, device=DEV)
        group = group.reshape(S, H, -1)
    n = group.shape[2]
    off = torch.gather(st["offsets"].long(), 2, group.clamp(max=M - 1))
    step = 64 + 2 * GROUP * D
    blob = st["pool"].view(-1, step)[off * 16 // step]
    scale = blob[..., 32:64].contiguous().view(torch.float32)
    ks, vs = scale[..., :4].repeat_interleave(PAGE, -1), scale[..., 4:].repeat_interleave(PAGE, -1)
    size = blob[..., 12:20].contiguous().view(torch.int16).int().repeat_interleave(PAGE, -1)
    k = blob[..., 64 : 64 + GROUP * D].reshape(S, H, n, D // 4, GROUP, 4).permute(0, 1, 3, 5, 2, 4).reshape(S, H, D, n * GROUP)
    lane = torch.arange(GROUP, device=DEV)
    visible = torch.minimum(st["tokens"], st["pos"] + 1)[:, None, None, None]
    seen = (group[..., None] * GROUP + lane < visible) & (lane % PAGE < size) & (group[..., None] < M)
    seen = seen.view(S, H, 1, n * GROUP)
    score = torch.matmul(st["queries"].view(S, H, G, D), k.float() - 128) * (ks.view(S, H, 1, -1) * st["scale"])
    del k
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del score
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = blob[..., 64 + GROUP * D :].reshape(S, H, n, 4, D // 16, 4, 16, 4).permute(0, 1, 2, 5, 3, 7, 4, 6).reshape(S, H, n * GROUP, D)
    del blob
    out = {"output": torch.matmul(p * vs.view(S, H, 1, -1), v.float() - 128).view(S, H * G, D)}
    if st["weights"] is not None:
        w = p.view(S, H, G, n, GROUP).sum((2, 4))
        total = torch.zeros(S, H, M + 1, device=DEV).scatter_add_(2, group.clamp(max=M), w)[..., :M]
        out["weights"] = st["weights"] * st["decay"] + total
    return out


def _plain_evict(st):
    c = st["case"]
    S, H, M, u, D = c["S"], c["H"], _max_groups(c), c["unit"], c["D"]
    tokens = st["tokens"].long()[:, None, None]
    groups = (tokens + GROUP - 1) // GROUP
    units = (groups + u - 1) // u
    kept = torch.clamp(units, max=c["budget"])
    m = -(-M // u)
    here = torch.arange(M, device=DEV) < groups
    w = torch.nn.functional.pad(st["weights"] * here, (0, m * u - M)).view(S, H, m, u).sum(-1)
    at = _largest(w, _forced(m, units, c["first"], c["last"]), units.expand(S, H, 1), kept)
    pick = torch.where(at < m, at * u, torch.full_like(at, m * u))[..., None] + torch.arange(u, device=DEV)
    pick = torch.nn.functional.pad(pick.reshape(S, H, m * u).clamp(max=m * u), (0, 1), value=m * u)[..., :M]
    ok = pick < groups
    src = torch.where(ok, pick, torch.zeros_like(pick))

    def moved(x):
        return torch.gather(x, 2, src).masked_fill(~ok, 0)

    codes = torch.gather(st["codes"], 2, src[..., None].expand(S, H, M, 2 * D)).masked_fill(~ok[..., None], 0)
    stays = torch.zeros(S, H, M + 1, dtype=torch.bool, device=DEV).scatter_(2, torch.where(ok, pick, torch.full_like(pick, M)), True)
    gone = (~stays[..., :M]) & here
    order = torch.sort((~gone).to(torch.int8), dim=-1, stable=True).indices
    dropped = torch.gather(torch.where(gone, st["offsets"], torch.full_like(st["offsets"], NONE)), 2, order)
    left = torch.where(units > kept, tokens - GROUP * u * (units - kept), tokens)
    return {"offsets": moved(st["offsets"]), "weights": moved(st["weights"]), "scales": moved(st["scales"]), "codes": codes,
            "dropped": dropped, "tokens": left.view(S).to(torch.int32)}


# ------------------------------------------------------------------------------------------------ the library's
def _own_bounds(st):
    from chromofold_amd import kvselect
    c = st["case"]
    if "out" not in st:  # a serving program keeps its bounds beside its page tables
        st["out"] = kvselect.empty_bounds(c["S"], c["H"], _max_groups(c), c["D"], DEV)
    kvselect.key_bounds(st["keys"], st["first"], st["counts"], st["out"], token_counts=st["tokens"], slots=st["slots"])
    return {"codes": st["out"].codes, "scales": st["out"].scales}


def _cache(st):
    from chromofold_amd import kv
    c = st["case"]
    pool = st["pool"] if "pool" in st else torch.empty(16, dtype=torch.uint8, device=DEV)
    offsets = st["offsets"] if "offsets" in st else torch.zeros(c["S"], c["H"], _max_groups(c), dtype=torch.int32, device=DEV)
    return kv.BatchedKv(kv.CODEC_INT8, c["S"], c["H"], c["D"], _max_groups(c), pool, offsets, st["tokens"], None)


def _own_select(st):
    from chromofold_amd import kvselect
    c = st["case"]
    if "kept" not in st:  # the cache, the selection's memory and the descriptor, made once by a serving program
        kvb, b = _cache(st), kvselect.KeyBounds(st["codes"], st["scales"])
        units = torch.empty(c["S"], c["H"], c["units"], dtype=torch.int32, device=DEV)
        st["kept"] = kvb, b, units, kvselect.select_desc(kvb, b, st["queries"], st["pos"], units, unit_groups=c["unit"],
                                                         keep_first=c["first"], keep_last=c["last"])
    kvb, b, units, desc = st["kept"]
    kvselect.select(kvb, b, st["queries"], st["pos"], units, desc=desc)
    return {"units": units}


def _own_attend(st):
    from chromofold_amd import kvselect
    c = st["case"]
    if "kept" not in st:
        kvb, out = _cache(st), torch.empty_like(st["queries"])
        w = torch.empty_like(st["weights"]) if c["weights"] else None
        st["kept"] = kvb, out, w, kvselect.attention_desc(kvb, st["queries"], out, st["pos"], st["scale"], units=st["units"],
                                                          unit_groups=c["unit"], weights=st["weights"], weights_out=w, decay=st["decay"])
    kvb, out, w, desc = st["kept"]
    kvselect.attention(kvb, st["queries"], out, st["pos"], st["scale"], desc=desc)
    return {"output": out, "weights": w} if c["weights"] else {"output": out}


def _own_evict(st):
    from chromofold_amd import kvselect
    c = st["case"]
    if "kept" not in st:
        kvb, b = _cache(st), kvselect.KeyBounds(st["codes"], st["scales"])
        to = kvselect.Evicted(torch.zeros_like(st["offsets"]), torch.zeros_like(st["tokens"]), torch.zeros_like(st["weights"]),
                              kvselect.KeyBounds(torch.zeros_like(st["codes"]), torch.zeros_like(st["scales"])),
                              torch.zeros_like(st["offsets"]))
        st["kept"] = kvb, to, kvselect.evict_desc(kvb, st["weights"], c["budget"], to, bounds=b, unit_groups=c["unit"],
                                                  keep_first=c["first"], keep_last=c["last"])
    kvb, to, desc = st["kept"]
    kvselect.evict(kvb, st["weights"], c["budget"], to, desc=desc)
    return {"offsets": to.group_offsets, "weights": to.weights, "scales": to.bounds.scales, "codes": to.bounds.codes,
            "dropped": to.dropped, "tokens": to.seq_tokens}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"bounds": _own_bounds, "select": _own_select, "attend": _own_attend, "evict": _own_evict}[op](state)
    return {"bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend, "evict": _plain_evict}[op](state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _pick(values, n, k, first, last):
    """Ascending indices of the k of n values (numpy, 64 bits) that stay."""
    free = [i for i in range(first, max(first, n - last))]
    forced = [i for i in range(n) if i < first or i >= n - last]
    if len(forced) >= k:
        return np.array(forced[:k] if n > k else forced, np.int64)
    v = values[free]
    best = np.lexsort((np.arange(len(free)), -v))[: k - len(forced)]
    return np.sort(np.concatenate([np.array(forced, np.int64), np.array(free, np.int64)[best]]))


def _exact_bounds(c, st):
    shape = (c["S"], c["H"], _max_groups(c))
    codes = np.zeros((*shape, 2 * c["D"]), np.int8)
    scales = np.zeros(shape)
    keys = st["keys"].double().cpu().numpy()
    at = 0
    for s, T in enumerate(_lens(c)):
        n = -(-T // PAGE)
        k = keys[at : at + c["H"] * n].reshape(c["H"], n * PAGE, c["D"])[:, :T]
        at += c["H"] * n
        for g in range(-(-T // GROUP)):
            part = k[:, GROUP * g : GROUP * (g + 1)]
            top = np.abs(part).max((1, 2)) / 127
            scales[s, :, g] = top
            held = top.astype(np.float32).astype(np.float64)[:, None]  # the codes count steps of the scale as it is held
            for x, to in ((part.max(1), slice(0, c["D"])), (-part.min(1), slice(c["D"], None))):
                codes[s, :, g, to] = np.clip(np.ceil((x / held).astype(np.float32)), -127, 127)
    return {"codes": codes, "scales": scales}


def _exact_select(c, st):
    S, H, G, D, u = c["S"], c["H"], c["gqa"], c["D"], c["unit"]
    q = st["queries"].double().view(S, H, G, D)
    got = np.full((S, H, c["units"]), NONE, np.int32)
    for s in range(S):
        visible = min(_lens(c)[s], _positions(c)[s] + 1)
        n = -(-visible // GROUP)
        if not n:
            continue
        step = (q[s].abs().amax(-1) / 127).float().double()
        a = torch.round((q[s] / step[..., None]).float().double()).clamp(-127, 127)
        hi, low = st["codes"][s, :, :n, :D].double(), -st["codes"][s, :, :n, D:].double()
        # a score is held in 32 bits: the whole number times the query's step, rounded, then times the group's, rounded
        best = torch.stack([((torch.maximum(a[:, g, None] * hi, a[:, g, None] * low).sum(-1) * step[:, g, None]).float().double()
                             * st["scales"][s, :, :n].double()).float().double() for g in range(G)]).amax(0).cpu().numpy()
        m = -(-n // u)
        best = np.concatenate([best, np.full((H, m * u - n), -np.inf)], 1).reshape(H, m, u).max(2)
        for h in range(H):
            at = _pick(best[h], m, min(m, c["units"]), c["first"], c["last"])
            got[s, h, : len(at)] = at
    return {"units": got}


def _exact_attend(c, st, seed):
    S, H, G, D, M, u = c["S"], c["H"], c["gqa"], c["D"], _max_groups(c), c["unit"]
    out = torch.zeros(S, H, G, D, dtype=torch.float64, device=DEV)
    w = None if st["weights"] is None else st["weights"].double() * st["decay"]
    q = st["queries"].double().view(S, H, G, D)
    for s, T in enumerate(_lens(c)):
        visible = min(T, _positions(c)[s] + 1)
        if not visible:
            continue
        kq, ks, vq, vs, _ = _sequence(c, seed, s)
        for h in range(H):
            tok = torch.arange(visible, device=DEV)
            if st["units"] is not None:
                listed_units = st["units"][s, h].long()
                tok = tok[torch.isin(tok // (GROUP * u), listed_units[listed_units >= 0])]
            k = kq[h, tok].double() * ks[h, tok // PAGE].double()[:, None]
            v = vq[h, tok].double() * vs[h, tok // PAGE].double()[:, None]
            p = torch.softmax((q[s, h] @ k.t().contiguous()) * st["scale"], -1)
            out[s, h] = p @ v
            if w is not None:
                w[s, h].index_add_(0, tok // GROUP, p.sum(0))
    return {"output": out.view(S, H * G, D)} if w is None else {"output": out.view(S, H * G, D), "weights": w}


def _exact_evict(c, st):
    S, H, M, u = c["S"], c["H"], _max_groups(c), c["unit"]
    x = {k: st[k].cpu().numpy() for k in ("offsets", "weights", "scales", "codes")}
    got = {k: np.zeros(v.shape, np.float64 if v.dtype == np.float32 else v.dtype) for k, v in x.items()}
    got["dropped"] = np.full((S, H, M), NONE, np.int32)
    got["tokens"] = np.array(_lens(c), np.int32)
    for s, T in enumerate(_lens(c)):
        n = -(-T // GROUP)
        m = -(-n // u)
        k = min(m, c["budget"])
        got["tokens"][s] = T - GROUP * u * (m - k)
        for h in range(H):
            w = np.zeros(m * u)
            w[:n] = x["weights"][s, h, :n]
            w = w.reshape(m, u).sum(1).astype(np.float32).astype(np.float64)  # a unit's weight is held in 32 bits
            units = _pick(w, m, k, c["first"], c["last"])
            at = (units[:, None] * u + np.arange(u)).reshape(-1)
            at = at[at < n]
            for name in x:
                got[name][s, h, : len(at)] = x[name][s, h, at]
            gone = np.setdiff1d(np.arange(n), at)
            got["dropped"][s, h, : len(gone)] = x["offsets"][s, h, gone]
    return got


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "bounds":
        return _exact_bounds(case, st)
    if case["op"] == "select":
        return _exact_select(case, st)
    return _exact_attend(case, st, seed) if case["op"] == "attend" else _exact_evict(case, st)
