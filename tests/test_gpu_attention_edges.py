"""qmm_paged_attention where roundings and launch choices could show."""
import numpy as np
import pytest

import qmm_hip
from attn_ref import Batch, queries, run_attention
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,new", [(200, 60), (200, 2), (3000, 60), (3000, 1)])
def test_scales_of_hidden_cells(ctx, D, n, new):
    """8-bit: what scale a cell has that no row sees changes no bit of any row."""
    window, got = 20, []
    for hidden in (0.0, 0.1, 0.3, 0.7, 5.0, 3e38, np.inf, np.nan):
        b = Batch([(n, new)], 1, D, 16, True, seed=D)
        p, t = b.cells(0)
        seen = n - new - window + 1  # the first token of any row's window
        b.vs[p, :, t] *= np.float32(2.0 ** -20)  # (weights with few bits: a change of their exponent shows)
        b.vs[p[:seen], :, t[:seen]] = hidden
        say(f"hidden scale {hidden} n={n} new={new} D={D}")
        b.upload(ctx, new, n)
        got.append(run_attention(ctx, b, queries(b, 4), 4, D ** -0.5, window, out_type=qmm_hip.TYPE_F32))
        b.free()
        assert np.isfinite(got[-1]).all() and (got[-1] != 0).any()
        assert np.array_equal(got[0].view(np.uint32), got[-1].view(np.uint32)), f"hidden scales of {hidden} reached a row"
