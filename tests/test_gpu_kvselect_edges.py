"""The operators of chromofold/kv_select.h, and the batched decode whose group body they share, where values, masks and
streams are out of the ordinary (plain forms and tolerances: kvselect_helpers.py)."""
import numpy as np
import pytest

import kvselect_helpers as R
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
