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
