"""Host-only checks of the attention entry points' scale (no GPU)."""

import ctypes

import pytest

from kvblockmass_b200 import _lib
from test_attention_host import _cached, _prompt


@pytest.mark.parametrize("scale,code", [(1e300, _lib.KVBM_ERR_SHAPE), (-1e300, _lib.KVBM_ERR_SHAPE),
                                        (3.5e38, _lib.KVBM_ERR_SHAPE), (3.4e38, _lib.KVBM_OK), (-3.4e38, _lib.KVBM_OK),
                                        (1e-300, _lib.KVBM_OK), (0.0, _lib.KVBM_OK)])
def test_scales_are_those_of_float32(scale, code):
    for make, call in ((_prompt, "kvbm_validate_attention"), (_cached, "kvbm_validate_cached_attention")):
        a = make()
        a.scale = scale
        assert getattr(_lib.load(), call)(ctypes.byref(a)) == code
