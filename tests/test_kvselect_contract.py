"""chromofold/kv_select.h without a GPU: C99 header, struct sizes against the ctypes mirrors, and every argument that the
calls refuse on the host."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from chromofold_amd import _abi as A
from chromofold_amd import kv, kvselect as ks

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(A.LIB_PATH), reason="libchromofold.so not built")
OK, INV, UNS = A.CF_OK, A.CF_ERR_INVALID_ARGUMENT, A.CF_ERR_UNSUPPORTED
P = 0x10000  # an aligned address that the host checks never follow


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_header_is_c_and_sizes_match(tmp_path):
    src = tmp_path / "a.c"
    src.write_text('#include <stdio.h>\n#include "chromofold/kv_select.h"\nint main(void) {'
                   'printf("%zu %zu %zu\\n", sizeof(cf_kv_select_desc), sizeof(cf_kv_selection), sizeof(cf_kv_evict_desc));'
                   "return 0;}\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(tmp_path / "a")], check=True, timeout=60)
    out = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, timeout=60).stdout
    assert [int(x) for x in re.findall(r"\d+", out)] == [C.sizeof(x) for x in (ks.cf_kv_select_desc, ks.cf_kv_selection,
                                                                               ks.cf_kv_evict_desc)]


def select_desc(**change):
    d = ks.cf_kv_select_desc(C.sizeof(ks.cf_kv_select_desc), 1, 2, 4, 16, 128, 100, 1, 8, 1, 1, 0, P, P, P, P, P, P, P, 1 << 30)
    for k, v in change.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change, want", [
    ({}, OK), ({"struct_size": 8}, INV), ({"abi_version": 2}, INV), ({"codes": None}, INV), ({"scales": None}, INV),
    ({"seq_tokens": None}, INV), ({"query_pos": None}, INV), ({"queries": None}, INV), ({"units": None}, INV),
    ({"seq_count": 0}, INV), ({"kv_head_count": 0}, INV), ({"query_head_count": 0}, INV), ({"query_head_count": 15}, INV),
    ({"max_groups": 0}, INV), ({"max_units": 0}, INV), ({"codes": P + 8}, INV), ({"unit_groups": 0}, INV),
    ({"unit_groups": 2}, OK), ({"unit_groups": 3}, INV), ({"keep_first": 9}, INV), ({"keep_last": 8}, INV),
    ({"keep_first": 0xFFFFFFFF, "keep_last": 2}, INV), ({"keep_first": 0, "keep_last": 0}, OK),
    ({"keep_first": 4, "keep_last": 4}, OK), ({"head_dim": 64}, OK), ({"head_dim": 96}, UNS), ({"query_head_count": 64}, OK),
    ({"query_head_count": 68}, UNS), ({"seq_count": 65536}, UNS), ({"kv_head_count": 65536, "query_head_count": 65536}, UNS),
    ({"max_groups": 1 << 25}, UNS), ({"max_groups": (1 << 25) - 1}, OK), ({"max_units": 1000}, OK),
])
def test_select_refusals(change, want):
    L, d = A.lib(), select_desc(**change)
    assert L.cf_kv_validate_select_desc(C.byref(d)) == want
    if want != OK:
        assert L.cf_kv_select_groups_async(C.byref(d), None) == want
        assert L.cf_kv_select_workspace_bytes(C.byref(d)) == 0


def test_select_workspace_is_checked():
    L, d = A.lib(), select_desc()
    need = L.cf_kv_select_workspace_bytes(C.byref(d))
    if need:
        for change in ({"workspace": None}, {"workspace_bytes": need - 1}, {"workspace": P + 4}):
            assert L.cf_kv_select_groups_async(C.byref(select_desc(**change)), None) == INV
    assert L.cf_kv_validate_select_desc(None) == INV
    assert L.cf_kv_select_groups_async(None, None) == INV


def attention_args(desc=None, sel=None):
    d = kv.cf_kv_batched_desc(C.sizeof(kv.cf_kv_batched_desc), kv.EXT_ABI_VERSION, kv.CODEC_INT8, 2, 4, 16, 128, 100, P, P, P,
                              P, P, P, P, 0.1, 0, P, 1 << 40)
    s = ks.cf_kv_selection(C.sizeof(ks.cf_kv_selection), 1, 1, 8, P, P, P, 0.9)
    for x, change in ((d, desc), (s, sel)):
        for k, v in (change or {}).items():
            setattr(x, k, v)
    return d, s


@pytest.mark.parametrize("desc, sel, want", [
    ({}, {}, OK), ({}, {"struct_size": 4}, INV), ({}, {"abi_version": 0}, INV), ({}, {"units": None, "unit_groups": 7}, OK),
    ({}, {"max_units": 0}, INV), ({}, {"unit_groups": 0}, INV), ({}, {"unit_groups": 2}, OK), ({}, {"unit_groups": 4}, INV),
    ({}, {"weights_in": None}, OK), ({}, {"weights_in": None, "weights_out": None}, OK), ({}, {"weights_out": None}, INV),
    ({}, {"decay": float("nan")}, INV), ({}, {"decay": float("inf")}, INV), ({}, {"max_units": 1 << 25}, UNS),
    ({"struct_size": 0}, {}, INV), ({"pool": None}, {}, INV), ({"pool": P + 8}, {}, INV), ({"output": None}, {}, INV),
    ({"query_head_count": 64}, {}, OK), ({"query_head_count": 68}, {}, UNS), ({"query_head_count": 17}, {}, INV),
    ({"query_head_count": 64, "head_dim": 80}, {}, UNS), ({"head_dim": 64}, {}, OK), ({"head_dim": 32}, {}, UNS),
    ({"query_head_count": 64, "queries": None}, {}, INV), ({"query_head_count": 64, "seq_count": 65536}, {}, UNS),
    ({"max_groups": 0}, {}, INV), ({"max_groups": 1 << 25}, {}, UNS), ({"softmax_scale": float("inf")}, {}, INV),
    ({"codec": 3}, {}, UNS), ({"codec": kv.CODEC_RANS_HYBRID, "query_head_count": 20}, {}, UNS),
    ({"codec": kv.CODEC_RANS_HYBRID, "tables": None}, {}, INV),
])
def test_attention_refusals(desc, sel, want):
    L = A.lib()
    d, s = attention_args(desc, sel)
    assert L.cf_kv_validate_selection(C.byref(d), C.byref(s)) == want
    if want != OK:
        assert L.cf_kv_paged_attention_selected_async(C.byref(d), C.byref(s), None) == want
        assert L.cf_kv_selected_workspace_bytes(C.byref(d), C.byref(s)) == 0


def test_attention_workspace_is_checked():
    L = A.lib()
    d, s = attention_args()
    need = L.cf_kv_selected_workspace_bytes(C.byref(d), C.byref(s))
    assert need > 0
    for change in ({"workspace": None}, {"workspace_bytes": need - 1}, {"workspace": P + 8}):
        d2, _ = attention_args(change)
        assert L.cf_kv_paged_attention_selected_async(C.byref(d2), C.byref(s), None) == INV
    assert L.cf_kv_paged_attention_selected_async(C.byref(d), None, None) == INV
    assert L.cf_kv_paged_attention_selected_async(None, C.byref(s), None) == INV


def evict_desc(**change):
    d = ks.cf_kv_evict_desc(C.sizeof(ks.cf_kv_evict_desc), 1, 2, 4, 128, 100, 1, 8, 1, 1, P, P, P, P, P, P, P, P, P, P, P)
    for k, v in change.items():
        setattr(d, k, v)
    return d


NO_RECORDS = {"codes": None, "scales": None, "codes_out": None, "scales_out": None}


@pytest.mark.parametrize("change, want", [
    ({}, OK), (NO_RECORDS, OK), ({"weights_out": None, "dropped": None}, OK), ({"struct_size": 0}, INV),
    ({"abi_version": 9}, INV), ({"group_offsets": None}, INV), ({"seq_tokens": None}, INV), ({"weights": None}, INV),
    ({"group_offsets_out": None}, INV), ({"seq_tokens_out": None}, INV), ({"seq_count": 0}, INV), ({"kv_head_count": 0}, INV),
    ({"max_groups": 0}, INV), ({"budget_units": 0}, INV), ({"unit_groups": 3}, INV), ({"unit_groups": 2}, OK),
    ({"keep_last": 0}, INV), ({"keep_first": 8}, INV), ({"keep_first": 7}, OK), ({"keep_last": 9}, INV),
    ({"codes": None}, INV), ({"scales_out": None}, INV), ({"codes": P + 4}, INV), ({"codes_out": P + 4}, INV),
    ({"head_dim": 256}, UNS), ({"head_dim": 64}, OK), ({"seq_count": 65536}, UNS), ({"kv_head_count": 65536}, UNS),
    ({"max_groups": 1 << 25}, UNS), ({"max_groups": (1 << 25) - 1}, OK),
])
def test_evict_refusals(change, want):
    L, d = A.lib(), evict_desc(**change)
    assert L.cf_kv_validate_evict_desc(C.byref(d)) == want
    if want != OK:
        assert L.cf_kv_evict_groups_async(C.byref(d), None) == want
    assert L.cf_kv_validate_evict_desc(None) == INV


@pytest.mark.parametrize("change, want", [
    ({"keys": None}, INV), ({"keys": P + 4}, INV), ({"first": None}, INV), ({"counts": None}, INV), ({"codes": None}, INV),
    ({"codes": P + 4}, INV), ({"scales": None}, INV), ({"n": 0}, INV), ({"D": 96}, UNS), ({"D": 0}, UNS),
])
def test_bounds_refusals(change, want):
    a = {"keys": P, "n": 4, "first": P, "counts": P, "tokens": None, "D": 128, "slots": None, "codes": P, "scales": P}
    a.update(change)
    assert A.lib().cf_kv_key_bounds_async(a["keys"], a["n"], a["first"], a["counts"], a["tokens"], a["D"], a["slots"], a["codes"],
                                          a["scales"], 4, None) == want


def test_binding_checks_tensors():
    import torch
    S, H, M, D = 2, 2, 5, 64
    z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t)  # noqa: E731
    kvb = kv.BatchedKv(kv.CODEC_INT8, S, H, D, M, z(64, t=torch.uint8), z(S, H, M), z(S), None)
    b = ks.empty_bounds(S, H, M, D, "cpu")
    q, w = z(S, H * 2, D, t=torch.float32), z(S, H, M, t=torch.float32)
    bad = [
        lambda: ks.select_desc(kvb, b, q.double(), z(S), z(S, H, 3)),
        lambda: ks.select_desc(kvb, b, q, z(S + 1), z(S, H, 3)),
        lambda: ks.select_desc(kvb, b, q, z(S), z(S, H + 1, 3)),
        lambda: ks.select_desc(kvb, ks.empty_bounds(S, H, M, 128, "cpu"), q, z(S), z(S, H, 3)),
        lambda: ks.select_desc(kvb, b, q.transpose(0, 1).contiguous().transpose(0, 1), z(S), z(S, H, 3)),
        lambda: ks.attention_desc(kvb, q, q[:1], z(S), 1.0),
        lambda: ks.attention_desc(kvb, q, q, z(S), 1.0, weights_out=w[:, :, :4]),
        lambda: ks.attention_desc(kvb, q, q, z(S), 1.0, units=z(S, 1, 3)),
        lambda: ks.attention_desc(kvb, q, q, z(S), 1.0, units=z(S, H, 0)),
        lambda: ks.evict_desc(kvb, w[:1], 2),
        lambda: ks.evict_desc(kvb, w, 2, ks.Evicted(z(S, H, M), z(S), w, b), bounds=None),
        lambda: ks.evict_desc(kvb, w, 2, ks.Evicted(z(S, H, M), z(S + 1))),
        lambda: ks.key_bounds(z(3, 16, D, t=torch.float32), z(1, t=torch.int64), z(1), ks.empty_bounds(S, H, M, 128, "cpu")),
        lambda: ks.key_bounds(z(3, 15, D, t=torch.float32), z(1, t=torch.int64), z(1), b),
        lambda: ks.bounds_of(z(1, 1, 17, D, t=torch.float32)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(A.CfError):
        ks.evict_desc(kvb, w, 2, keep_last=0)
    with pytest.raises(A.CfError):
        ks.attention_desc(kvb, q, q, z(S), float("nan"))
