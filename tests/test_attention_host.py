"""Host-only argument checks of the attention and eviction entry points (no GPU)."""

import ctypes
import math

import pytest
import torch

from kvblockmass_b200 import _lib
from _attention_ref import cached_keep, check, evict_rows, prompt_keep, softmax_rows


def _prompt():
    a = _lib.AttentionArgs()
    a.q = a.k = a.v = a.out = a.lse = 4096
    for i, s in enumerate((8 * 100 * 64, 100 * 64, 64, 1)):
        a.q_stride[i] = a.k_stride[i] = a.v_stride[i] = a.out_stride[i] = s
    a.dtype, a.B, a.Hq, a.Hkv, a.N, a.D = _lib.KVBM_BF16, 2, 8, 2, 100, 64
    a.scale = 0.125
    return a


def _cached():
    a = _lib.CachedArgs()
    a.q = a.k_cache = a.v_cache = a.out = a.lse = a.seq_lens = a.block_table = 4096
    for i in range(4):
        a.q_stride[i] = a.k_stride[i] = a.v_stride[i] = a.out_stride[i] = 64
    a.dtype, a.B, a.Hq, a.Hkv, a.T, a.D = _lib.KVBM_F16, 2, 8, 2, 1, 64
    a.num_pages, a.page_size, a.max_pages = 50, 16, 20
    a.scale = 0.125
    return a


def _evict():
    a = _lib.EvictArgs()
    a.k_cache = a.v_cache = a.k_out = a.v_out = a.seq_lens = a.block_table = 4096
    a.weights = a.seq_lens_out = a.kept_out = 4096
    a.dtype, a.B, a.Hkv, a.D = _lib.KVBM_F32, 2, 2, 64
    a.num_pages, a.page_size, a.max_pages = 50, 16, 20
    a.weight_heads, a.budget, a.n_sinks, a.recency, a.capacity = 2, 40, 4, 32, 40
    return a


def _bad(make, call, code, **fields):
    a = make()
    for k, v in fields.items():
        setattr(a, k, v)
    assert getattr(_lib.load(), call)(ctypes.byref(a)) == code, fields


@pytest.mark.parametrize("code,fields", [
    (_lib.KVBM_OK, {}),
    (_lib.KVBM_ERR_DTYPE, {"dtype": _lib.KVBM_F64}),
    (_lib.KVBM_ERR_DTYPE, {"dtype": 9}),
    (_lib.KVBM_ERR_SHAPE, {"N": 0}),
    (_lib.KVBM_ERR_SHAPE, {"N": (1 << 28) + 1}),
    (_lib.KVBM_ERR_SHAPE, {"B": 8192}),
    (_lib.KVBM_ERR_GQA, {"Hkv": 3}),
    (_lib.KVBM_ERR_HEAD_DIM, {"D": 257}),
    (_lib.KVBM_ERR_SHAPE, {"seq_lens": 4096, "cu_seqlens": 4096}),
    (_lib.KVBM_ERR_SHAPE, {"cu_seqlens": 4096, "total_tokens": -1}),
    (_lib.KVBM_ERR_SHAPE, {"scale": math.nan}),
    (_lib.KVBM_ERR_SHAPE, {"scale": math.inf}),
    (_lib.KVBM_ERR_NULL, {"v": None}),
    (_lib.KVBM_ERR_NULL, {"lse": None}),
])
def test_prompt_checks(code, fields):
    _bad(_prompt, "kvbm_validate_attention", code, **fields)


@pytest.mark.parametrize("code,fields", [
    (_lib.KVBM_OK, {}),
    (_lib.KVBM_OK, {"T": 64}),
    (_lib.KVBM_OK, {"weights": 4096, "weights_out": 4096}),
    (_lib.KVBM_ERR_SHAPE, {"T": 65}),
    (_lib.KVBM_ERR_SHAPE, {"T": 0}),
    (_lib.KVBM_ERR_DTYPE, {"dtype": _lib.KVBM_F64}),
    (_lib.KVBM_ERR_GQA, {"Hkv": 5}),
    (_lib.KVBM_ERR_HEAD_DIM, {"D": 300}),
    (_lib.KVBM_ERR_SHAPE, {"max_pages": 1 << 25}),
    (_lib.KVBM_OK, {"block_table": None}),
    (_lib.KVBM_ERR_SHAPE, {"block_table": None, "max_pages": 26}),
    (_lib.KVBM_ERR_SHAPE, {"T": 2, "weights": 4096, "weights_out": 4096}),
    (_lib.KVBM_ERR_NULL, {"weights": 4096}),
    (_lib.KVBM_ERR_NULL, {"seq_lens": None}),
])
def test_cached_checks(code, fields):
    _bad(_cached, "kvbm_validate_cached_attention", code, **fields)


@pytest.mark.parametrize("code,fields", [
    (_lib.KVBM_OK, {}),
    (_lib.KVBM_OK, {"dtype": _lib.KVBM_F64, "weight_heads": 1}),
    (_lib.KVBM_ERR_SHAPE, {"weight_heads": 3}),
    (_lib.KVBM_ERR_SHAPE, {"budget": 35}),
    (_lib.KVBM_ERR_SHAPE, {"budget": 0, "n_sinks": 0, "recency": 0}),
    (_lib.KVBM_ERR_SHAPE, {"n_sinks": -1}),
    (_lib.KVBM_ERR_SHAPE, {"capacity": 39}),
    (_lib.KVBM_ERR_SHAPE, {"block_table": None, "max_pages": 26}),
    (_lib.KVBM_ERR_NULL, {"kept_out": None}),
])
def test_evict_checks(code, fields):
    _bad(_evict, "kvbm_validate_evict", code, **fields)


def test_null_and_no_device():
    lib = _lib.load()
    assert lib.kvbm_validate_attention(None) == _lib.KVBM_ERR_NULL
    assert lib.kvbm_validate_cached_attention(None) == _lib.KVBM_ERR_NULL
    assert lib.kvbm_validate_evict(None) == _lib.KVBM_ERR_NULL
    assert lib.kvbm_cached_attention_workspace_bytes(ctypes.byref(_cached())) > 0
    if not torch.cuda.is_available():
        assert lib.kvbm_attention(ctypes.byref(_prompt()), None) in (_lib.KVBM_ERR_CUDA, _lib.KVBM_ERR_DEVICE)
        assert lib.kvbm_evict_cache(ctypes.byref(_evict()), None) in (_lib.KVBM_ERR_CUDA, _lib.KVBM_ERR_DEVICE)


def test_python_refuses_cpu_tensors():
    import kvblockmass_b200 as kb

    q = torch.zeros(1, 2, 8, 64)
    with pytest.raises(ValueError):
        kb.attention_b200(q, q, q)
    with pytest.raises(ValueError):
        kb.attention_cached(q, q, q, None, torch.tensor([8]))
    with pytest.raises(ValueError):
        kb.evict_cache(q, q, None, torch.tensor([8]), torch.zeros(1, 8), 4)


def test_the_restatement_itself():
    """softmax_rows against torch's softmax, its handling of dropped NaN, and a planted mistake that the bound catches."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(20, 16, generator=g) for _ in range(3))
    keep = prompt_keep(20, True, None, "cpu")
    out, lse, p, ot, lt, _ = softmax_rows(q, k, v, keep, 0.25)
    x = (q.double() @ k.double().T * 0.25).masked_fill(~keep, -math.inf)
    assert torch.allclose(out, torch.softmax(x, -1) @ v.double())
    assert torch.allclose(lse, torch.logsumexp(x, -1))
    check(out.float(), out, ot, "out")
    with pytest.raises(AssertionError):
        check(out.float() * (1 + 1e-2), out, ot, "scaled")
    v2 = v.clone()
    v2[7, 3] = math.nan
    out2, *_ = softmax_rows(q, k, v2, keep, 0.25)
    assert torch.equal(out2[:7], out[:7]) and bool(torch.isnan(out2[7:, 3]).all())
    tree = cached_keep(5, 3, None, "cpu")
    assert tree.tolist() == [[1, 1, 1, 0, 0], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1]]
    assert evict_rows([5.0, 1.0, 3.0, 3.0, 3.0, 0.0], 6, 4, 1, 1) == [0, 2, 3, 5]
