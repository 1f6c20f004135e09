"""Eviction from a paged cache by accumulated attention weight, on the GPU.

``evict_cache`` keeps, per sequence (and per kv head, when the weights are), the
first tokens, the latest ones and the heaviest of those between, and moves their
keys and values into a compact cache that ``attention_cached`` reads on from.
The weights are those ``attention_cached(..., weights=)`` accumulates, or any
per-token mass (``block_mass_b200(..., block_size=1, per_sequence=True)`` of a
prompt).  Where ``design_from_mass`` draws a random design from block mass,
this choice is deterministic and per token.  ``kvbm_evict_cache`` in
``include/kvbm.h``.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from .attention import _I4, _check_out, _fail, _int32_on, _no_overlap, _on_device, _per_key, _table
from .ops import _DTYPES

__all__ = ["EvictedCache", "evict_cache"]


@dataclass
class EvictedCache:
    """A compact cache: sequence ``b`` is the first ``seq_lens[b]`` slots of page ``b``."""

    k: torch.Tensor         # [B, capacity, H_kv, D]
    v: torch.Tensor         # [B, capacity, H_kv, D]
    seq_lens: torch.Tensor  # [B] int32
    kept: torch.Tensor      # [B, H_w, budget] int32: the slots kept, ascending, -1 past the new length
    weights: torch.Tensor   # [B, H_w, budget] float32: their weights, 0 past the new length


def evict_cache(k_cache, v_cache, block_table, seq_lens, weights, budget, *, n_sinks=4, recency=32, capacity=None,
                out=None):
    """Cut every sequence's cache down to ``budget`` tokens.

    ``k_cache``, ``v_cache``, ``block_table`` and ``seq_lens`` as
    ``attention_cached`` takes them; ``weights`` float32 ``[B, H_kv, max_pages *
    page_size]``, or ``[B, 1, ...]`` / ``[B, ...]`` for one choice for all
    heads.  A sequence of at most ``budget`` tokens keeps them all; otherwise
    its first ``n_sinks`` and last ``recency`` tokens stay, and those of the
    highest weights between them (equal weights: the lower slot; NaN counts as
    -inf).  Order is kept.  The result's caches have ``capacity`` slots per
    sequence (default ``budget``), zeros past the new length; ``out=(k, v)``
    gives the memory instead (``[B, capacity, H_kv, D]``, not overlapping the
    inputs), whose slots past the new length are left as they were.

    Decoding over the result needs ``capacity > budget``: token ``u`` of the
    next call goes to slot ``seq_lens[b] + u`` of sequence ``b``, which differs
    between sequences shorter and longer than ``budget``, and a length past
    ``capacity`` would be clamped.
    """
    if not all(isinstance(t, torch.Tensor) for t in (k_cache, v_cache)):
        raise TypeError("evict_cache: k_cache and v_cache must be torch tensors")
    if not k_cache.is_cuda:
        raise ValueError("evict_cache needs CUDA tensors (there is no CPU path)")
    dev = k_cache.device
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or v_cache.device != dev:
        raise ValueError(f"both caches must be [num_pages, page_size, H_kv, D] of one dtype and device, got "
                         f"{tuple(k_cache.shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")
    if k_cache.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {k_cache.dtype}; expected float32, bfloat16, float16 or float64")
    num_pages, page_size, Hkv, D = k_cache.shape
    lens = _int32_on(seq_lens, dev, "seq_lens")
    B = lens.shape[0]
    if B == 0 or Hkv == 0 or D == 0:
        raise ValueError("evict_cache needs at least one sequence, kv head and element")
    table, max_pages = _table(block_table, B, k_cache, k_cache)
    budget, n_sinks, recency = int(budget), int(n_sinks), int(recency)
    if budget < 1 or n_sinks < 0 or recency < 0 or n_sinks + recency > budget:
        raise ValueError(f"budget={budget} must be >= 1 and hold n_sinks={n_sinks} + recency={recency} tokens")
    w, wb, wh = _per_key("weights", weights, B, Hkv, max_pages * page_size, dev)
    if w.shape[0] != B:
        raise ValueError(f"weights must have B={B} rows, got {w.shape[0]}")
    Hw = w.shape[1]
    if out is None:
        cap = budget if capacity is None else int(capacity)
        if cap < budget:
            raise ValueError(f"capacity={cap} < budget={budget}")
        # a head's slots one after another: the next reader streams them
        ko = k_cache.new_empty((B, Hkv, cap, D)).transpose(1, 2)
        vo = k_cache.new_empty((B, Hkv, cap, D)).transpose(1, 2)
    else:
        ko, vo = out
        if not isinstance(ko, torch.Tensor) or ko.dim() != 4:
            raise ValueError("out must be a pair of [B, capacity, H_kv, D] tensors")
        cap = ko.shape[1]
        if cap < budget or (capacity is not None and cap != int(capacity)):
            raise ValueError(f"out holds {cap} slots per sequence, budget={budget}, capacity={capacity}")
        for name, t in (("out k", ko), ("out v", vo)):
            _check_out(name, t, (B, cap, Hkv, D), k_cache.dtype, dev)
            _no_overlap(name, t, {"k_cache": k_cache, "v_cache": v_cache, "weights": w, "block_table": table,
                                  "seq_lens": lens})
        _no_overlap("out v", vo, {"out k": ko})
    a = _lib.EvictArgs()
    a.k_cache, a.v_cache, a.k_out, a.v_out = k_cache.data_ptr(), v_cache.data_ptr(), ko.data_ptr(), vo.data_ptr()
    a.k_stride, a.v_stride = _I4(*k_cache.stride()), _I4(*v_cache.stride())
    a.k_out_stride, a.v_out_stride = _I4(*ko.stride()), _I4(*vo.stride())
    a.dtype = _DTYPES[k_cache.dtype]
    a.B, a.Hkv, a.D = B, Hkv, D
    a.num_pages, a.page_size, a.max_pages = num_pages, page_size, max_pages
    if table is not None:
        a.block_table, a.block_table_stride = table.data_ptr(), table.stride(0)
    a.seq_lens = lens.data_ptr()
    a.weights, a.weights_bstride, a.weights_hstride, a.weight_heads = w.data_ptr(), wb, wh, Hw
    a.budget, a.n_sinks, a.recency, a.capacity, a.zero_tail = budget, n_sinks, recency, cap, int(out is None)
    kept = w.new_empty((B, Hw, budget), dtype=torch.int32)
    wout = w.new_empty((B, Hw, budget))
    new_lens = w.new_empty((B,), dtype=torch.int32)
    a.kept_out, a.weights_out, a.seq_lens_out = kept.data_ptr(), wout.data_ptr(), new_lens.data_ptr()
    code = _on_device(dev, lambda stream: _lib.load().kvbm_evict_cache(ctypes.byref(a), stream))
    if code != _lib.KVBM_OK:
        _fail(code, "evict_cache")
    return EvictedCache(k=ko, v=vo, seq_lens=new_lens, kept=kept, weights=wout)
