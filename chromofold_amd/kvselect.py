"""Reading and keeping only a part of a batched cache (include/chromofold/kv_select.h) over kv.BatchedKv:

  key_bounds   an 8-bit bound on the keys of every group, made while sealing        cf_kv_key_bounds_async
  select       per (sequence, KV head), the groups a query's scores can be largest  cf_kv_select_groups_async
  attention    attention over selected groups or all, and the groups' weight        cf_kv_paged_attention_selected_async
  evict        the groups of least accumulated weight leave the page tables         cf_kv_evict_groups_async

u32 arrays are int32 tensors of the same bits; -1 is CF_KV_NO_UNIT. The *_desc functions make a descriptor to be kept for
repeated calls (and as long as a graph captured with it); it holds the tensors it points at. What a call is given beside one
has to be what the descriptor was made of: other tensors or numbers are refused (None and defaults are not looked at)."""
from __future__ import annotations

import contextlib
import ctypes as C
from dataclasses import dataclass

import torch

from . import _abi as A
from . import kv

SELECT_ABI_VERSION = 1
NO_UNIT = -1


class cf_kv_select_desc(C.Structure):
    _fields_ = [("struct_size", A.U32), ("abi_version", A.U32), ("seq_count", A.U32), ("kv_head_count", A.U32),
                ("query_head_count", A.U32), ("head_dim", A.U32), ("max_groups", A.U32), ("unit_groups", A.U32),
                ("max_units", A.U32), ("keep_first", A.U32), ("keep_last", A.U32), ("reserved", A.U32),
                ("codes", A.P), ("scales", A.P), ("seq_tokens", A.P), ("query_pos", A.P), ("queries", A.P),
                ("units", A.P), ("workspace", A.P), ("workspace_bytes", A.U64)]


class cf_kv_selection(C.Structure):
    _fields_ = [("struct_size", A.U32), ("abi_version", A.U32), ("unit_groups", A.U32), ("max_units", A.U32),
                ("units", A.P), ("weights_in", A.P), ("weights_out", A.P), ("decay", A.F32), ("reserved", A.U32)]


class cf_kv_evict_desc(C.Structure):
    _fields_ = [("struct_size", A.U32), ("abi_version", A.U32), ("seq_count", A.U32), ("kv_head_count", A.U32),
                ("head_dim", A.U32), ("max_groups", A.U32), ("unit_groups", A.U32), ("budget_units", A.U32),
                ("keep_first", A.U32), ("keep_last", A.U32), ("group_offsets", A.P), ("seq_tokens", A.P),
                ("weights", A.P), ("codes", A.P), ("scales", A.P), ("group_offsets_out", A.P), ("seq_tokens_out", A.P),
                ("weights_out", A.P), ("codes_out", A.P), ("scales_out", A.P), ("dropped", A.P)]


A.declare("cf_kv_key_bounds_async", A.I32, [A.P, A.U64, A.P, A.P, A.P, A.U32, A.P, A.P, A.P, A.U64, A.P])
A.declare("cf_kv_validate_select_desc", A.I32, [A.P])
A.declare("cf_kv_select_workspace_bytes", A.U64, [A.P])
A.declare("cf_kv_select_groups_async", A.I32, [A.P, A.P])
A.declare("cf_kv_validate_selection", A.I32, [A.P, A.P])
A.declare("cf_kv_selected_workspace_bytes", A.U64, [A.P, A.P])
A.declare("cf_kv_paged_attention_selected_async", A.I32, [A.P, A.P, A.P])
A.declare("cf_kv_validate_evict_desc", A.I32, [A.P])
A.declare("cf_kv_evict_groups_async", A.I32, [A.P, A.P])


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    """The C calls see addresses only: what a tensor has to be is checked here."""
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on {device} is needed, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _raw_stream(device: torch.device, stream) -> int:
    """Handle of `stream` (default: the device's current stream), which has to belong to the tensors' device."""
    if stream is None:
        # torch.cuda.current_stream(device).cuda_stream without the Stream object, whose making takes 2 us of a 7 us call
        return torch._C._cuda_getCurrentRawStream(device.index)
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    return stream.cuda_stream


def _call(name: str, device: torch.device, s: int, *args) -> None:
    """One asynchronous C call with the tensors' device as the current one."""
    fn = getattr(A.lib(), name)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            A.check(fn(*args, s), name)
    else:
        A.check(fn(*args, s), name)


def _on_device(device: torch.device, fn, *args):
    """A host-side call (validation, workspace sizes) with the tensors' device as the current one: sizes go by its CUs."""
    if device.type != "cuda" or device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


@contextlib.contextmanager
def _working_on(stream, device: torch.device, *inputs: torch.Tensor):
    """Makes `stream` (None: no change) the current one, behind what the current one has been given, so that tensors made
    here are filled and let go of in the order of the work on it; the inputs' memory is kept for it."""
    if stream is not None and stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    if stream is None or stream == torch.cuda.current_stream(device):
        yield
        return
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        for t in inputs:
            t.record_stream(stream)
        yield


def _with_workspace(desc, need: int, device: torch.device, stream) -> None:
    """Gives the descriptor a workspace for calls on `stream`, allocated for that stream."""
    if need:
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        with torch.cuda.device(device):
            kv._give_workspace(desc, need, device, stream if stream is not None else torch.cuda.current_stream(device))


def _kept(d, tensors: tuple, numbers: tuple, defaults: tuple) -> None:
    """Refuses a call whose arguments are not those of the descriptor it brings: the call would read and write the
    descriptor's. tensors in the order of d.held, from the first on; numbers in that of d.numbers."""
    for t, h in zip(tensors, d.held):
        if t is not h and t is not None and (h is None or t.data_ptr() != h.data_ptr() or t.shape != h.shape):
            raise ValueError(f"a tensor of shape {tuple(t.shape)} is not the descriptor's: make a descriptor for it")
    for x, n, default in zip(numbers, d.numbers, defaults):
        if x != n and x != default and not (isinstance(n, float) and C.c_float(x).value == C.c_float(n).value):
            raise ValueError(f"{x} is not the descriptor's {n}: make a descriptor for it")


def _for_stream(d, cls, device: torch.device, stream, s: int):
    """The descriptor, or a copy with a workspace of its own where it was made for another stream than s."""
    if d.workspace and d.workspace_stream != s:
        copy = cls.from_buffer_copy(d)
        _with_workspace(copy, d.workspace_bytes, device, stream)
        return copy
    return d


# ---------------------------------------------------------------------------------------------------- key bounds
@dataclass
class KeyBounds:
    """codes int8 [seq_count, kv_heads, max_groups, 2 D] (upper, negated lower), scales fp32 [seq_count, kv_heads, max_groups]."""
    codes: torch.Tensor
    scales: torch.Tensor


_NO_BOUNDS = KeyBounds(None, None)


def empty_bounds(seq_count: int, kv_heads: int, max_groups: int, head_dim: int, device="cuda") -> KeyBounds:
    """Records of groups without tokens, to be filled as groups are sealed."""
    return KeyBounds(torch.zeros(seq_count, kv_heads, max_groups, 2 * head_dim, dtype=torch.int8, device=device),
                     torch.zeros(seq_count, kv_heads, max_groups, dtype=torch.float32, device=device))


def key_bounds(keys: torch.Tensor, first_page: torch.Tensor, page_counts: torch.Tensor, out: KeyBounds,
               token_counts: torch.Tensor | None = None, slots: torch.Tensor | None = None, stream=None) -> KeyBounds:
    """Bounds of the groups that kv.encode_groups_device seals from the same arguments: keys fp32 [n_pages, 16, D],
    first_page int64, page_counts / token_counts int32, slots int64: the index of each group's record in `out`, the first
    three dims of out.codes taken as one (default: the groups' order)."""
    dev, D, n = keys.device, keys.shape[-1], first_page.numel()
    _need(keys, "keys", torch.float32, (keys.shape[0], kv.PAGE_TOKENS, D), dev)
    _need(first_page, "first_page", torch.int64, (n,), dev)
    _need(page_counts, "page_counts", torch.int32, (n,), dev)
    if token_counts is not None:
        _need(token_counts, "token_counts", torch.int32, (keys.shape[0],), dev)
    if slots is not None:
        _need(slots, "slots", torch.int64, (n,), dev)
    rows = out.scales.shape
    _need(out.scales, "out.scales", torch.float32, rows, dev)
    _need(out.codes, "out.codes", torch.int8, (*rows, 2 * D), dev)
    if n:
        _call("cf_kv_key_bounds_async", dev, _raw_stream(dev, stream), keys.data_ptr(), n, first_page.data_ptr(),
              page_counts.data_ptr(), _ptr(token_counts), D, _ptr(slots), out.codes.data_ptr(), out.scales.data_ptr(),
              out.scales.numel())
    return out


def bounds_of(keys: torch.Tensor, stream=None) -> KeyBounds:
    """Bounds of dense keys [seq_count, kv_heads, T, D] (T a multiple of 16), group for group what kv.seal_device makes of
    them. Made on `stream` (default: the current one) behind what the current stream has been given so far."""
    S, H, T, D = keys.shape
    if T % kv.PAGE_TOKENS:
        raise ValueError("T must be a multiple of 16, as for kv.seal_device")
    dev, pages = keys.device, T // kv.PAGE_TOKENS
    groups = -(-pages // kv.GROUP_PAGES)
    with _working_on(stream, dev, keys):
        out = empty_bounds(S, H, groups, D, dev)
        g = torch.arange(S * H * groups, device=dev)
        first = (g // groups) * pages + (g % groups) * kv.GROUP_PAGES
        counts = torch.clamp(pages - (g % groups) * kv.GROUP_PAGES, max=kv.GROUP_PAGES).to(torch.int32)
        return key_bounds(keys.reshape(-1, kv.PAGE_TOKENS, D), first, counts, out, stream=stream)


# ---------------------------------------------------------------------------------------------------- selection
def _check_cache(kvb: kv.BatchedKv) -> tuple:
    dev, shape = kvb.group_offsets.device, (kvb.seq_count, kvb.kv_heads, kvb.max_groups)
    _need(kvb.group_offsets, "group_offsets", torch.int32, shape, dev)
    _need(kvb.seq_tokens, "seq_tokens", torch.int32, shape[:1], dev)
    return dev, shape


def _check_blobs(kvb: kv.BatchedKv, dev) -> None:
    """The pool, and the tables where it is coded: two of each KV head."""
    _need(kvb.pool, "pool", torch.uint8, kvb.pool.shape, dev)
    if kvb.codec == kv.CODEC_RANS_HYBRID and kvb.tables is not None:
        _need(kvb.tables, "tables", torch.uint8, kvb.tables.shape, dev)
        if kvb.tables.numel() < 2 * kvb.kv_heads * kv.TABLE_BYTES:
            raise ValueError(f"tables: {2 * kvb.kv_heads} of {kv.TABLE_BYTES} bytes are needed, got {kvb.tables.numel()} bytes")


def _check_bounds(b: KeyBounds, name: str, shape: tuple, D: int, dev) -> KeyBounds:
    _need(b.codes, name + ".codes", torch.int8, (*shape, 2 * D), dev)
    _need(b.scales, name + ".scales", torch.float32, shape, dev)
    return b


def select_desc(kvb: kv.BatchedKv, bounds: KeyBounds, queries: torch.Tensor, query_pos: torch.Tensor, units: torch.Tensor,
                unit_groups: int = 1, keep_first: int = 1, keep_last: int = 1, stream=None) -> cf_kv_select_desc:
    """Descriptor for select(), with a workspace of its own for calls on `stream`."""
    dev, shape = _check_cache(kvb)
    S, H, M = shape
    _check_bounds(bounds, "bounds", shape, kvb.head_dim, dev)
    _need(queries, "queries", torch.float32, (S, queries.shape[1], kvb.head_dim), dev)
    _need(query_pos, "query_pos", torch.int32, (S,), dev)
    _need(units, "units", torch.int32, (S, H, units.shape[-1]), dev)
    d = cf_kv_select_desc(C.sizeof(cf_kv_select_desc), SELECT_ABI_VERSION, S, H, queries.shape[1], kvb.head_dim, M, unit_groups,
                          units.shape[2], keep_first, keep_last, 0, bounds.codes.data_ptr(), bounds.scales.data_ptr(),
                          kvb.seq_tokens.data_ptr(), query_pos.data_ptr(), queries.data_ptr(), units.data_ptr())
    d.held = (bounds.codes, bounds.scales, kvb.seq_tokens, query_pos, queries, units)
    d.numbers = (unit_groups, keep_first, keep_last)
    A.check(A.lib().cf_kv_validate_select_desc(C.byref(d)), "cf_kv_validate_select_desc")
    _with_workspace(d, int(_on_device(dev, A.lib().cf_kv_select_workspace_bytes, C.byref(d))), dev, stream)
    return d


def select(kvb: kv.BatchedKv, bounds: KeyBounds, queries: torch.Tensor, query_pos: torch.Tensor, units: torch.Tensor,
           unit_groups: int = 1, keep_first: int = 1, keep_last: int = 1, stream=None,
           desc: cf_kv_select_desc | None = None) -> torch.Tensor:
    """Fills units int32 [seq_count, kv_heads, max_units] with the units of each row whose bound on the scores of `queries`
    [seq_count, query_heads, D] is largest, the first keep_first and the last keep_last always, ascending, then NO_UNIT."""
    if desc is not None:
        d, b = desc, bounds if bounds is not None else _NO_BOUNDS
        _kept(d, (b.codes, b.scales, kvb.seq_tokens, query_pos, queries, units), (unit_groups, keep_first, keep_last), (1, 1, 1))
    else:
        d = select_desc(kvb, bounds, queries, query_pos, units, unit_groups, keep_first, keep_last, stream)
    dev = kvb.group_offsets.device
    s = _raw_stream(dev, stream)
    _call("cf_kv_select_groups_async", dev, s, C.byref(_for_stream(d, cf_kv_select_desc, dev, stream, s)))
    return d.held[5]


# ---------------------------------------------------------------------------------------------------- attention
def attention_desc(kvb: kv.BatchedKv, queries: torch.Tensor, output: torch.Tensor, query_pos: torch.Tensor,
                   softmax_scale: float, units: torch.Tensor | None = None, unit_groups: int = 1,
                   weights: torch.Tensor | None = None, weights_out: torch.Tensor | None = None, decay: float = 1.0,
                   splits: int = 0, stream=None) -> kv.cf_kv_batched_desc:
    """Descriptor for attention() (the batched one, its `selection` beside it), with a workspace for calls on `stream`."""
    dev, shape = _check_cache(kvb)
    _check_blobs(kvb, dev)
    S, H, M = shape
    q = (S, queries.shape[1], kvb.head_dim)
    _need(queries, "queries", torch.float32, q, dev)
    _need(output, "output", torch.float32, q, dev)
    _need(query_pos, "query_pos", torch.int32, (S,), dev)
    if units is not None:
        _need(units, "units", torch.int32, (S, H, units.shape[-1]), dev)
        if units.numel() == 0:  # its address would be NULL, which stands for all groups
            raise ValueError("units lists nothing: at least one entry a row is needed")
    if weights is not None:
        _need(weights, "weights", torch.float32, shape, dev)
    if weights_out is not None:
        _need(weights_out, "weights_out", torch.float32, shape, dev)
    d = kv.cf_kv_batched_desc(C.sizeof(kv.cf_kv_batched_desc), kv.EXT_ABI_VERSION, kvb.codec, S, H, queries.shape[1],
                              kvb.head_dim, M, kvb.pool.data_ptr(), kvb.group_offsets.data_ptr(), kvb.seq_tokens.data_ptr(),
                              query_pos.data_ptr(), _ptr(kvb.tables), queries.data_ptr(), output.data_ptr(), softmax_scale,
                              splits)
    d.selection = cf_kv_selection(C.sizeof(cf_kv_selection), SELECT_ABI_VERSION, unit_groups,
                                  0 if units is None else units.shape[2], _ptr(units), _ptr(weights), _ptr(weights_out), decay)
    d.held = (kvb.pool, kvb.group_offsets, kvb.seq_tokens, kvb.tables, queries, output, query_pos, units, weights, weights_out)
    d.numbers = (float(softmax_scale), unit_groups, float(decay), splits)
    A.check(A.lib().cf_kv_validate_selection(C.byref(d), C.byref(d.selection)), "cf_kv_validate_selection")
    need = _on_device(dev, A.lib().cf_kv_selected_workspace_bytes, C.byref(d), C.byref(d.selection))
    _with_workspace(d, int(need), dev, stream)
    return d


def attention(kvb: kv.BatchedKv, queries: torch.Tensor, output: torch.Tensor, query_pos: torch.Tensor, softmax_scale: float,
              units: torch.Tensor | None = None, unit_groups: int = 1, weights: torch.Tensor | None = None,
              weights_out: torch.Tensor | None = None, decay: float = 1.0, splits: int = 0, stream=None,
              desc: kv.cf_kv_batched_desc | None = None) -> None:
    """kvb.attention over the units listed by select() (None: all groups). weights_out fp32 [seq_count, kv_heads, max_groups]
    (optional; may be `weights`) becomes decay * weights (None: 0) + each group's share of the softmax weight, summed over
    the KV head's query heads."""
    dev = kvb.group_offsets.device
    if desc is not None:
        d = desc
        _kept(d, (kvb.pool, kvb.group_offsets, kvb.seq_tokens, kvb.tables, queries, output, query_pos, units, weights,
                  weights_out), (softmax_scale, unit_groups, decay, splits), (None, 1, 1.0, 0))
    else:
        d = attention_desc(kvb, queries, output, query_pos, softmax_scale, units, unit_groups, weights, weights_out, decay,
                           splits, stream)
    s = _raw_stream(dev, stream)
    _call("cf_kv_paged_attention_selected_async", dev, s, C.byref(_for_stream(d, kv.cf_kv_batched_desc, dev, stream, s)),
          C.byref(d.selection))


# ---------------------------------------------------------------------------------------------------- eviction
@dataclass
class Evicted:
    """Where eviction writes: the page tables and lengths that remain, the weights (None: not wanted) and bounds (None)
    of their groups, and the offsets of the groups that went (None: not wanted)."""
    group_offsets: torch.Tensor
    seq_tokens: torch.Tensor
    weights: torch.Tensor | None = None
    bounds: KeyBounds | None = None
    dropped: torch.Tensor | None = None


def _evicted(kvb: kv.BatchedKv, weights: torch.Tensor, out: Evicted | None, bounds: KeyBounds | None) -> tuple:
    """The tensors of an eviction, None for those that are not there."""
    o, b = out if out is not None else _NO_OUT, bounds if bounds is not None else _NO_BOUNDS
    r = o.bounds if o.bounds is not None else _NO_BOUNDS
    return (kvb.group_offsets, kvb.seq_tokens, weights, o.group_offsets, o.seq_tokens, o.weights, o.dropped, b.codes, b.scales,
            r.codes, r.scales)


_NO_OUT = Evicted(None, None)


def evict_desc(kvb: kv.BatchedKv, weights: torch.Tensor, budget_units: int, out: Evicted | None = None,
               bounds: KeyBounds | None = None, unit_groups: int = 1, keep_first: int = 1,
               keep_last: int = 1) -> cf_kv_evict_desc:
    dev, shape = _check_cache(kvb)
    S, H, M = shape
    _need(weights, "weights", torch.float32, shape, dev)
    if out is None:
        out = Evicted(kvb.group_offsets, kvb.seq_tokens, weights, bounds)
    _need(out.group_offsets, "out.group_offsets", torch.int32, shape, dev)
    _need(out.seq_tokens, "out.seq_tokens", torch.int32, (S,), dev)
    if out.weights is not None:
        _need(out.weights, "out.weights", torch.float32, shape, dev)
    if out.dropped is not None:
        _need(out.dropped, "out.dropped", torch.int32, shape, dev)
    if (bounds is None) != (out.bounds is None):
        raise ValueError("bounds and out.bounds go together")
    rec = (None,) * 4
    if bounds is not None:
        _check_bounds(bounds, "bounds", shape, kvb.head_dim, dev)
        _check_bounds(out.bounds, "out.bounds", shape, kvb.head_dim, dev)
        rec = (bounds.codes.data_ptr(), bounds.scales.data_ptr(), out.bounds.codes.data_ptr(), out.bounds.scales.data_ptr())
    d = cf_kv_evict_desc(C.sizeof(cf_kv_evict_desc), SELECT_ABI_VERSION, S, H, kvb.head_dim, M, unit_groups, budget_units,
                         keep_first, keep_last, kvb.group_offsets.data_ptr(), kvb.seq_tokens.data_ptr(), weights.data_ptr(),
                         rec[0], rec[1], out.group_offsets.data_ptr(), out.seq_tokens.data_ptr(), _ptr(out.weights), rec[2],
                         rec[3], _ptr(out.dropped))
    d.held = _evicted(kvb, weights, out, bounds)
    d.numbers = (budget_units, unit_groups, keep_first, keep_last)
    A.check(A.lib().cf_kv_validate_evict_desc(C.byref(d)), "cf_kv_validate_evict_desc")
    return d


def evict(kvb: kv.BatchedKv, weights: torch.Tensor, budget_units: int, out: Evicted | None = None,
          bounds: KeyBounds | None = None, unit_groups: int = 1, keep_first: int = 1, keep_last: int = 1, stream=None,
          desc: cf_kv_evict_desc | None = None) -> None:
    """Cuts every sequence with more than budget_units units back to that many per KV head: the first keep_first, the last
    keep_last, then those of the largest accumulated `weights`. out=None evicts in place: kvb's tables and lengths, weights
    and bounds."""
    if desc is not None:
        d = desc
        _kept(d, _evicted(kvb, weights, out, bounds), (budget_units, unit_groups, keep_first, keep_last), (None, 1, 1, 1))
    else:
        d = evict_desc(kvb, weights, budget_units, out, bounds, unit_groups, keep_first, keep_last)
    dev = kvb.group_offsets.device
    _call("cf_kv_evict_groups_async", dev, _raw_stream(dev, stream), C.byref(d))
