"""Attention on the B200 next to the block mass: whole prompts, and one token or
a tree of drafted tokens over a paged cache.

* ``attention_b200`` / ``attention_varlen``: the attention output of a prompt
  and its row log-sum-exp.  The log-sum-exp is what ``block_mass_b200(...,
  lse=)`` and ``block_mass_varlen(..., lse=)`` take, so that the mass of a
  prompt costs no second pass over the row statistics.
* ``attention_cached``: decoding over ``[num_pages, page_size, H_kv, D]`` key
  and value caches and a block table (``block_mass_paged``'s layout), or over
  the caches ``evict_cache`` returns.  For one token it accumulates the weight
  of every key, which ``evict_cache`` chooses by; ``log_offsets`` are those of
  ``design_from_mass(..., with_log_offsets=True)``.

All three run hand-written kernels behind the C ABI (``kvbm_attention``,
``kvbm_cached_attention`` in ``include/kvbm.h``) on the current stream of the
inputs' device; there is no CPU path and no gradient.  bfloat16, float16 and
float32, ``D <= 256``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DTYPES, _VALUE_ERRORS, _as_mask, _to_int32

__all__ = ["attention_b200", "attention_varlen", "attention_cached", "cached_attention_workspace_bytes"]

MAX_TREE_TOKENS = 64


def _fail(code: int, what: str):
    msg = f"{what}: kvbm error {code}: {_lib.status_string(code)}"
    raise ValueError(msg) if code in _VALUE_ERRORS else RuntimeError(msg)


_I3, _I4 = ctypes.c_int64 * 3, ctypes.c_int64 * 4
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


# The current stream's handle by device index, without building a Stream object
# where this torch has the function (2 us of a call that runs for 15).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on_device(dev: torch.device, call):
    """``call(stream)`` with ``dev`` current, on its current stream."""
    index = dev.index
    if torch.cuda.current_device() == index:
        return call(_raw_stream(index))
    with torch.cuda.device(dev):
        return call(_raw_stream(index))


def _int32_on(t: torch.Tensor, dev, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != 1:
        raise ValueError(f"{name} must be a 1-D integer tensor")
    if t.dtype == torch.int32 and t.device == dev and t.is_contiguous():
        return t
    if t.dtype.is_floating_point or t.dtype == torch.bool:
        raise ValueError(f"{name} must hold integers, got {t.dtype}")
    return _to_int32(t, dev).contiguous()


def _same(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, q on {like.device}")
    if t.dtype != like.dtype:
        raise ValueError(f"{name} dtype {t.dtype} != q dtype {like.dtype}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and one-past-last byte a strided tensor can touch."""
    p = t.data_ptr()
    if t.is_contiguous():
        return (p, p + t.nbytes)
    if t.numel() == 0:
        return (0, 0)
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return (p, p + (last + 1) * t.element_size())


def _no_overlap(name: str, t: torch.Tensor, others: dict) -> None:
    """``others``: the tensors the kernels use besides ``t`` (absent ones, None, and copies made for the call pass)."""
    a0, a1 = _span(t)
    for other, o in others.items():
        if o is None:
            continue
        b0, b1 = _span(o)
        if a0 < b1 and b0 < a1:
            raise ValueError(f"{name} overlaps {other}: the kernels write it while they read the inputs")


def _check_out(name: str, t: torch.Tensor, shape, dtype, device) -> None:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on {device}")
    if not t.is_contiguous() and any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} has expanded (stride 0) dimensions")


def _check_qkv(q, k, v, what):
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError(f"{what}: q, k and v must be torch tensors")
    if not q.is_cuda:
        raise ValueError(f"{what} needs CUDA tensors (there is no CPU path)")
    if q.dtype not in _FLOATS:
        raise ValueError(f"unsupported dtype {q.dtype}; expected float32, bfloat16 or float16")
    _same("k", k, q)
    _same("v", v, q)


def _heads(Hq: int, Hkv: int) -> None:
    if Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"GQA requires H_q % H_kv == 0, got H_q={Hq}, H_kv={Hkv}")


def _key_mask(attn_mask, B: int, N: int, dev):
    """A contiguous bool key mask [B|1, 1, N], or None."""
    if attn_mask is None:
        return None
    m = _as_mask(attn_mask, dev)
    if m.dim() == 1:
        m = m.reshape(1, 1, -1)
    if m.dim() != 3 or m.shape[0] not in (1, B) or m.shape[1] != 1 or m.shape[2] != N:
        raise ValueError(f"attn_mask must be a key mask [N] or [B|1, 1, N] with N={N}, got {tuple(m.shape)}")
    return m.contiguous()


def _prompt(q, k, v, dims, strides, mask, causal, scale, out, out_strides, lse, lse_strides, fill, lens=None,
            cu=None, total=0):
    B, Hq, Hkv, N, D = dims
    dev = q.device
    a = _lib.AttentionArgs()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_stride, a.k_stride, a.v_stride = _I4(*strides[0]), _I4(*strides[1]), _I4(*strides[2])
    a.out_stride, a.lse_stride = _I4(*out_strides), _I3(*lse_strides)
    a.dtype = _DTYPES[q.dtype]
    a.B, a.Hq, a.Hkv, a.N, a.D = B, Hq, Hkv, N, D
    if mask is not None:
        a.key_mask, a.key_mask_bstride = mask.data_ptr(), (mask.stride(0) if mask.shape[0] > 1 else 0)
    a.scale = float(1.0 / D ** 0.5 if scale is None else scale)
    a.causal = int(bool(causal))
    if lens is not None:
        a.seq_lens = lens.data_ptr()
    if cu is not None:
        a.cu_seqlens, a.total_tokens = cu.data_ptr(), total
    a.fill_outside = int(fill)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    code = _on_device(dev, lambda stream: _lib.load().kvbm_attention(ctypes.byref(a), stream))
    if code != _lib.KVBM_OK:
        _fail(code, "attention")


def attention_b200(q, k, v, attn_mask=None, causal=False, scale=None, *, seq_lens=None, out=None, lse_out=None):
    """Attention over whole prompts: ``(out [B, H_q, N, D], lse [B, H_q, N])``.

    ``q [B, H_q, N, D]``, ``k`` and ``v [B, H_kv, N, D]`` of one dtype (any
    strides); ``out`` has it too, ``lse`` (natural log) is float32.
    ``attn_mask``: a key mask ``[N]`` or ``[B|1, 1, N]`` (True = keep); with
    ``causal`` a key must also not lie behind its query.  ``seq_lens [B]``:
    sequence ``b`` is its first ``seq_lens[b]`` positions (clamped into ``[0,
    N]``). A row that keeps no key gets ``out`` 0 and ``lse`` -inf, and so do
    rows past a sequence's end, unless ``out=`` or ``lse_out=`` is given: those
    rows of both are then left as they were. What masked keys and rows past the
    end hold (NaN included) reaches no result; a non-finite value of a kept key
    makes its column of ``out`` non-finite.  At most 65535 heads in all (``B *
    H_q``) and 2^28 positions.
    """
    _check_qkv(q, k, v, "attention_b200")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v must be 4-D [B, H, N, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Hq, N, D = q.shape
    if k.shape[0] != B or tuple(k.shape[2:]) != (N, D) or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    _heads(Hq, k.shape[1])
    lens = None
    if seq_lens is not None:
        lens = _int32_on(seq_lens, q.device, "seq_lens")
        if lens.shape[0] != B:
            raise ValueError(f"seq_lens must have B={B} entries, got {lens.shape[0]}")
    mask = _key_mask(attn_mask, B, N, q.device)
    ins = {"q": q, "k": k, "v": v, "seq_lens": lens, "attn_mask": mask}
    fill = out is None and lse_out is None
    if out is None:
        out = torch.empty_like(q) if fill or lens is None else torch.zeros_like(q)
        if any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_out("out", out, q.shape, q.dtype, q.device)
        _no_overlap("out", out, ins)
    if lse_out is None:
        lse_out = q.new_empty((B, Hq, N), dtype=torch.float32) if fill or lens is None else \
            torch.full((B, Hq, N), float("-inf"), dtype=torch.float32, device=q.device)
    else:
        _check_out("lse_out", lse_out, (B, Hq, N), torch.float32, q.device)
        _no_overlap("lse_out", lse_out, {**ins, "out": out})
    _prompt(q, k, v, (B, Hq, k.shape[1], N, D), (q.stride(), k.stride(), v.stride()), mask, causal, scale, out,
            out.stride(), lse_out, lse_out.stride(), fill, lens=lens)
    return out, lse_out


def attention_varlen(q, k, v, cu_seqlens, max_seqlen=None, causal=False, scale=None, *, out=None, lse_out=None):
    """Attention of a packed batch: ``(out [T, H_q, D], lse [H_q, T])``.

    ``q [T, H_q, D]``, ``k`` and ``v [T, H_kv, D]``; sequence ``b`` is rows
    ``[cu_seqlens[b], cu_seqlens[b + 1])`` and attends to itself alone
    (``cu_seqlens`` must not decrease: a row that two sequences name holds the
    result of either).  At most 65535 heads in all (``B * H_q``).
    ``max_seqlen`` (host int; read from ``cu_seqlens`` when omitted, which
    synchronises): the longest sequence; rows past a sequence's first
    ``max_seqlen`` count as outside it.  ``lse`` has the layout
    ``block_mass_varlen(..., lse=)`` takes.  Rows of no sequence are treated as
    the rows past a sequence's end in ``attention_b200``.
    """
    _check_qkv(q, k, v, "attention_varlen")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"packed q, k and v must be 3-D [T, H, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    T, Hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    Hkv = k.shape[1]
    _heads(Hq, Hkv)
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
        raise ValueError("cu_seqlens must be [B + 1] with B >= 1")
    if max_seqlen is None:
        cu_h = cu_seqlens.detach().to("cpu", torch.int64)
        max_seqlen = int((cu_h[1:] - cu_h[:-1]).max())
    cu = _int32_on(cu_seqlens, q.device, "cu_seqlens")
    ins = {"q": q, "k": k, "v": v, "cu_seqlens": cu}
    fill = out is None and lse_out is None
    if out is None:
        out = q.new_empty((T, Hq, D)) if fill else q.new_zeros((T, Hq, D))
    else:
        _check_out("out", out, q.shape, q.dtype, q.device)
        _no_overlap("out", out, ins)
    if lse_out is None:
        lse_out = q.new_empty((Hq, T), dtype=torch.float32) if fill else \
            torch.full((Hq, T), float("-inf"), dtype=torch.float32, device=q.device)
    else:
        _check_out("lse_out", lse_out, (Hq, T), torch.float32, q.device)
        _no_overlap("lse_out", lse_out, {**ins, "out": out})
    _prompt(q, k, v, (cu.shape[0] - 1, Hq, Hkv, max(int(max_seqlen), 1), D),
            tuple((0, t.stride(1), t.stride(0), t.stride(2)) for t in (q, k, v)), None, causal, scale, out,
            (0, out.stride(1), out.stride(0), out.stride(2)), lse_out, (0, lse_out.stride(0), lse_out.stride(1)), fill,
            cu=cu, total=T)
    return out, lse_out


def _table(block_table, B, k_cache, q):
    """(int32 table or None, max_pages) of a paged call."""
    num_pages, page_size = k_cache.shape[:2]
    if num_pages == 0 or page_size == 0:
        raise ValueError("k_cache has no pages")
    if block_table is None:
        if num_pages % B != 0:
            raise ValueError(f"without a block_table the cache holds B={B} runs of pages, got {num_pages} pages")
        return None, num_pages // B
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be a tensor [B={B}, max_pages]")
    if block_table.dtype.is_floating_point or block_table.dtype == torch.bool:
        raise ValueError(f"block_table must hold integer page ids, got {block_table.dtype}")
    if block_table.device != q.device:
        raise ValueError("q, the caches and block_table must be on one device")
    if block_table.shape[1] == 0:
        raise ValueError("block_table names no pages")
    t = block_table if block_table.dtype == torch.int32 else _to_int32(block_table, block_table.device)
    return (t if t.stride(1) == 1 else t.contiguous()), t.shape[1]


def _per_key(name, t, B, Hkv, L, dev, writable=False):
    """A float32 [B|1, Hkv|1, L] per-key array with unit stride: (tensor, batch stride, head stride)."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev:
        raise ValueError(f"{name} must be a float32 tensor on {dev}")
    if t.shape == (B, Hkv, L):  # the usual case
        st = t.stride()
        if st[2] == 1 and (B == 1 or st[0] > 0) and (Hkv == 1 or st[1] > 0):
            return t, st[0], st[1]
    if t.dim() == 2:
        t = t.unsqueeze(1)
    ok = t.dim() == 3 and t.shape[2] == L
    if writable:
        ok = ok and t.shape[:2] == (B, Hkv)
    else:
        ok = ok and t.shape[0] in (1, B) and t.shape[1] in (1, Hkv)
    if not ok:
        raise ValueError(f"{name} must be [B{'' if writable else '|1'}, H_kv{'' if writable else '|1'}, "
                         f"max_pages * page_size] = [{B}, {Hkv}, {L}], got {tuple(t.shape)}")
    if t.stride(2) != 1 and L > 1:
        if writable:
            raise ValueError(f"{name} must have unit stride over the keys")
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def _cached_args(q, k_cache, v_cache, block_table, seq_lens, tree_mask, log_offsets, weights, weights_out, scale, out,
                 lse_out):
    _check_qkv(q, k_cache, v_cache, "attention_cached")
    if q.dim() != 4 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"q must be [B, H_q, T, D] and both caches [num_pages, page_size, H_kv, D], got "
                         f"{tuple(q.shape)}, {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    B, Hq, T, D = q.shape
    num_pages, page_size, Hkv, Dk = k_cache.shape
    if Dk != D:
        raise ValueError(f"cache head dim {Dk} != q head dim {D}")
    _heads(Hq, Hkv)
    if B == 0 or T == 0:
        raise ValueError("q must hold at least one token")
    if T > MAX_TREE_TOKENS:
        raise ValueError(f"at most {MAX_TREE_TOKENS} tokens per sequence and call, got {T}")
    table, max_pages = _table(block_table, B, k_cache, q)
    lens = _int32_on(seq_lens, q.device, "seq_lens")
    if lens.shape[0] != B:
        raise ValueError(f"seq_lens must have B={B} entries, got {lens.shape[0]}")
    L = max_pages * page_size
    a = _lib.CachedArgs()
    keep = [q, k_cache, v_cache, table, lens]
    a.q, a.k_cache, a.v_cache = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.q_stride, a.k_stride, a.v_stride = _I4(*q.stride()), _I4(*k_cache.stride()), _I4(*v_cache.stride())
    a.dtype = _DTYPES[q.dtype]
    a.B, a.Hq, a.Hkv, a.T, a.D = B, Hq, Hkv, T, D
    a.num_pages, a.page_size, a.max_pages = num_pages, page_size, max_pages
    if table is not None:
        a.block_table, a.block_table_stride = table.data_ptr(), table.stride(0)
    a.seq_lens = lens.data_ptr()
    m = t = None
    if tree_mask is not None:
        m = _as_mask(tree_mask, q.device)
        if m.dim() == 2:
            m = m.unsqueeze(0)
        if m.dim() != 3 or m.shape[0] not in (1, B) or tuple(m.shape[1:]) != (T, T):
            raise ValueError(f"tree_mask must be [T, T] or [B|1, T, T] with T={T}, got {tuple(m.shape)}")
        if m.stride(2) != 1:
            m = m.contiguous()
        a.tree_mask, a.tree_mask_rstride = m.data_ptr(), m.stride(1)
        a.tree_mask_bstride = m.stride(0) if m.shape[0] > 1 else 0
        keep.append(m)
    if log_offsets is not None:
        t, a.log_offsets_bstride, a.log_offsets_hstride = _per_key("log_offsets", log_offsets, B, Hkv, L, q.device)
        a.log_offsets = t.data_ptr()
        keep.append(t)
    if weights is None and weights_out is not None:
        raise ValueError("weights_out needs weights")
    if weights is not None:
        if T != 1:
            raise ValueError("weights are accumulated for single tokens (T == 1): a drafted token may yet be rejected")
        if weights_out is None:
            weights_out = weights
        wo, a.weights_out_bstride, a.weights_out_hstride = _per_key("weights_out", weights_out, B, Hkv, L, q.device, True)
        _check_out("weights_out", wo, wo.shape, wo.dtype, wo.device)
        ins = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "block_table": table, "seq_lens": lens, "tree_mask": m,
               "log_offsets": t}
        if weights is weights_out:
            a.weights, a.weights_bstride, a.weights_hstride = wo.data_ptr(), a.weights_out_bstride, a.weights_out_hstride
        else:
            w, a.weights_bstride, a.weights_hstride = _per_key("weights", weights, B, Hkv, L, q.device)
            if w.shape[:2] != (B, Hkv):
                raise ValueError(f"weights must be [{B}, {Hkv}, {L}], got {tuple(w.shape)}")
            a.weights = w.data_ptr()
            if a.weights != wo.data_ptr() or w.stride() != wo.stride():
                ins["weights"] = w
            keep.append(w)
        a.weights_out = wo.data_ptr()
        _no_overlap("weights_out", wo, ins)
        keep.append(wo)
    a.scale = float(1.0 / D ** 0.5 if scale is None else scale)
    if out is not None or lse_out is not None:
        ins = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "block_table": table, "seq_lens": lens, "tree_mask": m,
               "log_offsets": t, "weights": weights, "weights_out": weights_out}
    if out is None:
        out = q.new_empty((B, Hq, T, D))
    else:
        _check_out("out", out, q.shape, q.dtype, q.device)
        _no_overlap("out", out, ins)
    if lse_out is None:
        lse_out = q.new_empty((B, Hq, T), dtype=torch.float32)
    else:
        _check_out("lse_out", lse_out, (B, Hq, T), torch.float32, q.device)
        _no_overlap("lse_out", lse_out, {**ins, "out": out})
    a.out, a.lse = out.data_ptr(), lse_out.data_ptr()
    a.out_stride, a.lse_stride = _I4(*out.stride()), _I3(*lse_out.stride())
    return a, keep, out, lse_out, weights_out


def cached_attention_workspace_bytes(q, k_cache, v_cache, block_table, seq_lens, **kwargs) -> int:
    """Workspace bytes of the ``attention_cached`` call with the same arguments."""
    args = dict(tree_mask=None, log_offsets=None, weights=None, weights_out=None, scale=None, out=None, lse_out=None)
    args.update(kwargs)
    a, keep, *_ = _cached_args(q, k_cache, v_cache, block_table, seq_lens, **args)
    n = int(_on_device(q.device, lambda _: _lib.load().kvbm_cached_attention_workspace_bytes(ctypes.byref(a))))
    del keep
    return n


def attention_cached(q, k_cache, v_cache, block_table, seq_lens, *, tree_mask=None, log_offsets=None, weights=None,
                     weights_out=None, scale=None, out=None, lse_out=None, workspace=None):
    """Attention of ``T`` tokens per sequence over a paged cache: ``(out, lse)``,
    with ``weights`` ``(out, lse, weights_out)``.

    ``q [B, H_q, T, D]`` (``T <= 64``); ``k_cache`` and ``v_cache [num_pages,
    page_size, H_kv, D]`` (any strides, the dtype of ``q``); ``block_table [B,
    max_pages]`` of page ids, or None when page ``b * max_pages + i`` is page
    ``i`` of sequence ``b``.  ``seq_lens [B]``: the cached tokens of each
    sequence, these ``T`` among them: token ``u`` sits in slot
    ``seq_lens[b] - T + u``, and its k and v are in the cache already.  A
    sequence of length 0 gives ``out`` 0 and ``lse`` -inf; lengths outside ``[0,
    max_pages * page_size]`` are clamped into it.

    Every token attends to the slots before the ``T`` tokens; among them token
    ``t`` attends to ``u`` where ``tree_mask [T, T]`` or ``[B|1, T, T]`` holds
    (None: ``u <= t``).  ``log_offsets [B|1, H_kv|1, max_pages * page_size]``
    (float32; a ``[B, L]`` array serves every head) are added to the scores;
    -inf drops a key.  Only the ``T`` tokens' rows may differ in the keys they
    keep, and what a dropped key holds reaches no result.

    ``weights [B, H_kv, max_pages * page_size]`` (float32, ``T == 1``): the
    softmax weight of every key, summed over the heads of its group, is added
    to it, into ``weights_out`` if given, else in place; slots past a
    sequence's end are not touched.  The call then holds ``B * H_q * max_pages
    * page_size`` float32 scores in its workspace, whatever the lengths.

    A page id outside ``[0, num_pages)`` is not read (its keys count as zero
    vectors); ``check_device_errors()`` reports it.  ``workspace`` (uint8,
    ``cached_attention_workspace_bytes``) lets callers reuse memory; calls
    that may run at the same time need one each.
    """
    a, keep, out, lse_out, weights_out = _cached_args(q, k_cache, v_cache, block_table, seq_lens, tree_mask,
                                                      log_offsets, weights, weights_out, scale, out, lse_out)
    dev = q.device
    lib = _lib.load()

    def launch(stream):
        need = lib.kvbm_cached_attention_workspace_bytes(ctypes.byref(a))
        ws = workspace
        if ws is None:
            ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
        elif ws.device != dev or ws.dtype != torch.uint8 or not ws.is_contiguous() or ws.numel() < need:
            raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on {dev}")
        return lib.kvbm_cached_attention(ctypes.byref(a), ws.data_ptr(), ws.numel(), stream)

    code = _on_device(dev, launch)
    del keep
    if code != _lib.KVBM_OK:
        _fail(code, "attention_cached")
    return (out, lse_out) if weights is None else (out, lse_out, weights_out)
