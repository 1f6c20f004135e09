"""Host-only checks of the attention entry points' scale and integer arguments (no GPU)."""

import ctypes

import pytest
import torch

from kvblockmass_b200 import _lib
from kvblockmass_b200.ops import _to_int32
from test_attention_host import _cached, _prompt


@pytest.mark.parametrize("scale,code", [(1e300, _lib.KVBM_ERR_SHAPE), (-1e300, _lib.KVBM_ERR_SHAPE),
                                        (3.5e38, _lib.KVBM_ERR_SHAPE), (3.4e38, _lib.KVBM_OK), (-3.4e38, _lib.KVBM_OK),
                                        (1e-300, _lib.KVBM_OK), (0.0, _lib.KVBM_OK)])
def test_scales_are_those_of_float32(scale, code):
    for make, call in ((_prompt, "kvbm_validate_attention"), (_cached, "kvbm_validate_cached_attention")):
        a = make()
        a.scale = scale
        assert getattr(_lib.load(), call)(ctypes.byref(a)) == code


def test_wide_integers_keep_to_the_ends_of_int32():
    low, high = -2 ** 31, 2 ** 31 - 1
    t = torch.tensor([2 ** 32, 2 ** 32 + 3, -2 ** 32, high, low, high + 1, low - 1, 7, -1])
    assert _to_int32(t, t.device).tolist() == [high, high, low, high, low, high, low, 7, -1]
    assert _to_int32(t.view(3, 3).T, t.device).tolist() == [[high, high, low], [high, low, 7], [low, high, -1]]
    for dtype in (torch.int32, torch.int16, torch.uint8):
        assert _to_int32(torch.tensor([5, 0], dtype=dtype), t.device).tolist() == [5, 0]
