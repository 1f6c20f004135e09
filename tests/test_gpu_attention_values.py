"""Values at the edges of what the attention kernels can hold, against 64 bits: non-finite values of kept keys, masks of
single tokens, scales and scores of extreme size, small weights, wide integer ids.  Bounds: ``_attention_ref``."""

import math

import pytest
import torch

import kvblockmass_b200 as kb
from test_gpu_cached_attention import Case, _check, _tree

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _put(c, cache, b, slot, col, value):
    cache[int(c.table[b, slot // c.page]), slot % c.page, :, col] = value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,D", [(2, 4, 64), (13, 4, 128), (20, 8, 64), (5, 4, 192), (40, 8, 64)])
def test_nan_before_the_drafts(cuda_device, dtype, T, Hq, D):
    """A NaN in the v of a slot shortly before the drafted tokens, which all of them keep, reaches every row."""
    c = Case([T + 15, T + 77, 300, 401], 16, Hq, 2, D, T, dtype, cuda_device, seed=T)
    for b, n in enumerate(c.lens):
        for col, back in ((1, 1), (2, 7), (3, 15)):
            _put(c, c.v, b, n - T - back, col, math.nan)
    tree = _tree(4, T, T, cuda_device)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    _check(c, out, lse, tree)
    assert bool(torch.isnan(out[..., 1:4]).all()) and bool(torch.isfinite(out[..., 4:]).all())
