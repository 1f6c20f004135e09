"""Plain 64-bit restatements of the attention and eviction operators, with error bounds.

The bounds count what the kernels round, with u the half step of the inputs' type:

* a score is a sum of D products in float32 (any order) times a rounded scale,
  plus an offset: it is off by at most ds = (D + 8) 2^-24 S, S = scale sum |q k| + |offset|;
* a weight exp(s - lse) is then off by 2 ds plus 2^-18 (the float32 exponential
  and its polynomial form, and the rounding of its argument) plus the float32 sum of n terms kept in blocks of
  at least 16, (n / 16 + 64) 2^-24; all relative;
* the tensor-core kernels round each weight to the inputs' type (u, relative)
  before the product with v, and the output is rounded once (u, relative).
"""

from __future__ import annotations

import math

import torch

F64 = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def softmax_rows(q, k, v, keep, scale, off=None, dtype=torch.float32):
    """One head: q [R, D], k/v [N, D], keep [R, N], off [N] or None, all as given.

    Returns out, lse, p and the bounds (out_tol, lse_tol, p_tol)."""
    D, n = q.shape[1], k.shape[0]
    qd = q.to(F64)
    some = keep.any(0)  # keys that some row keeps: only their values count
    kd = torch.where(some[:, None], k.to(F64), 0.0)
    vd = torch.where(some[:, None], v.to(F64), 0.0)
    x = qd @ kd.T * scale
    S = qd.abs() @ kd.abs().T * abs(scale)
    if off is not None:
        offd = torch.where(some, off.to(F64), 0.0)
        x = x + offd
        S = S + offd.abs()
    x = torch.where(keep, x, -math.inf)
    top = x.amax(1, keepdim=True)
    base = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(x - base)
    total = e.sum(1, keepdim=True)
    alive = total > 0
    p = torch.where(alive, e / total, 0.0)
    lse = torch.where(alive, base + total.log(), -math.inf)[:, 0]
    # a row may keep keys that another drops: products of dropped pairs count as nothing
    out = torch.zeros(q.shape[0], D, dtype=F64, device=q.device)
    mass = torch.zeros_like(out)
    finite = torch.isfinite(vd)
    out += p @ torch.where(finite, vd, 0.0)
    mass += p @ torch.where(finite, vd, 0.0).abs()
    if not bool(finite.all()):
        for j in range(n):
            if not bool(finite[j].all()):
                add = torch.where(finite[j], 0.0, vd[j])
                out = torch.where(keep[:, j:j + 1] & ~finite[j], out + add, out)
    ds = (D + 8) * 2.0 ** -24 * torch.where(keep, S, 0.0).amax(1)
    rel = 2 * ds + 2.0 ** -18 + (n / 16 + 64) * 2.0 ** -24
    u = half_step(dtype)
    pu = u if dtype != torch.float32 else 0.0
    out_tol = u * out.abs() + (rel[:, None] + pu) * (1 + 2 * u) * mass + 1e-30
    lse_tol = rel + 2.0 ** -23 * lse.abs()
    p_tol = rel[:, None] * p + 1e-30
    return out, lse, p, out_tol, lse_tol, p_tol


def check(got, want, tol, what):
    """Every element within its bound; non-finite ones equal."""
    got = got.to(F64)
    odd = ~torch.isfinite(want)
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert bool((got[inf] == want[inf]).all()), f"{what}: infinities differ"
    d = torch.where(odd, 0.0, (got - want).abs())
    t = torch.where(odd, 1.0, tol)
    bad = ~(d <= t)
    if bool(bad.any()):
        i = int((d / t).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst at {i}: got "
                             f"{got.flatten()[i].item()}, want {want.flatten()[i].item()}, "
                             f"bound {t.flatten()[i].item()}")


def prompt_keep(n, causal, mask, device):
    at = torch.arange(n, device=device)
    keep = torch.ones(n, n, dtype=torch.bool, device=device)
    if causal:
        keep &= at[None, :] <= at[:, None]
    if mask is not None:
        keep &= mask[None, :n]
    return keep


def cached_keep(n, T, tree, device):
    """[T, n]: the slots each of the T tokens keeps."""
    at = torch.arange(n, device=device)
    draft = at - (n - T)
    if tree is None:
        tree = torch.ones(T, T, dtype=torch.bool, device=device).tril()
    seen = tree[:, draft.clamp(0, T - 1)]
    return (draft < 0)[None, :] | seen


def evict_rows(w, n, budget, n_sinks, recency):
    """Slots kept of a row of n weights (list)."""
    if n <= budget:
        return list(range(n))
    key = [(-math.inf if x != x else x) for x in w[:n]]
    free = sorted(range(n_sinks, n - recency), key=lambda i: (-key[i], i))
    return sorted([*range(n_sinks), *free[:budget - n_sinks - recency], *range(n - recency, n)])
