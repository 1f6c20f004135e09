"""Values at the edges of what the attention kernels can hold, against 64 bits: non-finite values of kept keys, masks of
single tokens, scales and scores of extreme size, small weights, wide integer ids.  Bounds: ``_attention_ref``."""

import ctypes
import math

import pytest
import torch

import kvblockmass_b200 as kb
from kvblockmass_b200 import _lib
from _attention_ref import F64, cached_keep, check, evict_rows, half_step, softmax_rows
from test_gpu_attention import _check_dense, _inputs
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (80, 2, 64), (4, 1, 192)])
@pytest.mark.parametrize("weights", [False, True])
def test_tree_mask_of_a_single_token(cuda_device, dtype, Hq, Hkv, D, weights):
    """With one token the mask's one entry says whether it keeps its own slot; a dropped slot may hold anything."""
    c = Case([1, 1, 2, 64, 65, 65, 200, 0], 16, Hq, Hkv, D, 1, dtype, cuda_device, seed=D)
    tree = torch.tensor([0, 1, 0, 0, 0, 1, 0, 1], dtype=torch.bool, device=cuda_device).view(8, 1, 1)
    for b, n in enumerate(c.lens):
        if n and not bool(tree[b, 0, 0]):
            _put(c, c.k, b, n - 1, slice(None), math.nan)
            _put(c, c.v, b, n - 1, slice(0, None, 2), math.nan)
            _put(c, c.v, b, n - 1, slice(1, None, 2), math.inf)
    kw = {}
    if weights:
        kw["weights"] = torch.rand(8, Hkv, c.L, device=cuda_device)
        kw["weights_out"] = torch.full_like(kw["weights"], 3.0)
    got = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree, **kw)
    _check(c, got[0], got[1], tree, weights=kw.get("weights"), wout=kw.get("weights_out"))
    assert bool((got[0][0] == 0).all()) and bool((got[1][0] == -math.inf).all())
    all_on = torch.ones(1, 1, dtype=torch.bool, device=cuda_device)
    d = Case([1, 64, 200], 16, Hq, Hkv, D, 1, dtype, cuda_device, seed=D)
    a = kb.attention_cached(d.q, d.k, d.v, d.table, d.seq_lens, tree_mask=all_on)
    b = kb.attention_cached(d.q, d.k, d.v, d.table, d.seq_lens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,D", [(1, 8, 64), (1, 8, 128), (1, 4, 192), (3, 8, 64), (13, 4, 128), (40, 8, 64)])
@pytest.mark.parametrize("lens", [[1, 64, 65, 200], [5003]])
def test_infinite_values_of_kept_keys(cuda_device, dtype, T, Hq, D, lens):
    """Infinities in the v of kept keys: one of a sign gives it, both signs and a NaN give NaN; every other column is
    finite; those of dropped keys reach nothing."""
    lens = [n + T - 1 for n in lens]
    c = Case(lens, 16, Hq, 2, D, T, dtype, cuda_device, seed=T + D)
    off = torch.zeros(len(lens), 1, c.L, device=cuda_device)
    for b, n in enumerate(lens):
        last = max(n - T, 0)  # kept by every token
        _put(c, c.v, b, last, 1, math.inf)
        _put(c, c.v, b, last, 2, -math.inf)
        _put(c, c.v, b, last // 2, 2, -math.inf)
        if last > 3:
            _put(c, c.v, b, 0, 3, math.inf)
            _put(c, c.v, b, last, 3, -math.inf)
            _put(c, c.v, b, 1, 4, math.nan)
            _put(c, c.v, b, 2, slice(5, None, 2), math.inf)
            off[b, 0, 2] = -math.inf
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off)
    _check(c, out, lse, off=off)
    assert bool((out[..., 1] == math.inf).all()) and bool((out[..., 2] == -math.inf).all())
    if T == 1:
        w = torch.zeros(len(lens), 2, c.L, device=cuda_device)
        a = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off, weights=w)
        assert torch.equal(a[0].isnan(), out.isnan()) and torch.equal(a[0].nan_to_num(), out.nan_to_num())
        assert bool(torch.isfinite(w).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_outside_float32(cuda_device, dtype):
    """A scale below float32's smallest value is 0 (equal weights); one above its largest is refused."""
    q, k, v = _inputs(1, 2, 1, 200, 64, dtype, 21, cuda_device)
    for scale in (1e-60, -1e-60):
        out, lse = kb.attention_b200(q, k, v, causal=True, scale=scale)
        _check_dense(q, k, v, out, lse, True, scale=scale)
    for T in (1, 12, 40):
        c = Case([200, T, 77], 16, 8, 2, 64, T, dtype, cuda_device, seed=29)
        off = torch.rand(3, 2, c.L, device=cuda_device)
        for scale in (1e-60, -1e-60):
            for o in (None, off):
                out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, scale=scale, log_offsets=o)
                _check(c, out, lse, scale=scale, off=o)
        for scale in (1e60, -1e60):
            with pytest.raises(ValueError):
                kb.attention_b200(q, k, v, scale=scale)
            with pytest.raises(ValueError):
                kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("big,small", [(22528.0, 22400.0), (352.0, 350.0)])
def test_scores_past_float32_steps(cuda_device, dtype, big, small):
    """Scores of 3e10 (and 5e8), whose float32 steps are 2048 and 32: the highest ones, which are equal, share the
    weight, and nothing overflows.  Every product and sum here is exact in float32, so the weights are 1 / count:
    rounded once (2 u of the mass), as the sums, and the result once (u).  The lse is the score: the scale, its
    product, and with a maximum in base 2 the two factors and their products, 2^-24 each."""
    dev, D = cuda_device, 64
    u = half_step(dtype)

    def close(out, lse, v, keep, what):
        p = keep.double() / keep.sum(1, keepdim=True)
        check(out, p @ v.double(), (2 * u + 2.0 ** -18) * (p @ v.double().abs()) + u * (p @ v.double()).abs(), what)
        top = 20480.0 * big * 64
        want = torch.full((keep.shape[0],), top, dtype=F64, device=dev) + keep.sum(1).double().log()
        check(lse, want, 6 * 2.0 ** -24 * want, what)

    def rows(n):
        t = torch.full((n, D), big, device=dev)
        t[1::2] = small
        return t.to(dtype)

    N = 300
    v = torch.randn(1, 1, N, D, device=dev).to(dtype)
    q = torch.full((1, 1, N, D), 20480.0, device=dev).to(dtype)
    even = (torch.arange(N, device=dev) % 2 == 0)[None]
    out, lse = kb.attention_b200(q, rows(N)[None, None], v, causal=True, scale=1.0)
    close(out[0, 0], lse[0, 0], v[0, 0], even & torch.ones(N, N, dtype=torch.bool, device=dev).tril(), "prompt")
    for T in (1, 7, 40):
        c = Case([N], N, 2, 1, D, T, dtype, dev, spare=0)
        c.q.fill_(20480.0)
        c.k[0, :, 0] = rows(N)
        for off in (None, torch.zeros(1, 1, N, device=dev)):
            out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, scale=1.0, log_offsets=off)
            for h in range(2):
                close(out[0, h], lse[0, h], c.v[0, :, 0], even & cached_keep(N, T, None, dev), f"T={T}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [12.0, 17.5, 20.0])
def test_many_small_weights(cuda_device, dtype, gap):
    """One key `gap` nats above n equal ones.  Their weights, n exp(-gap) together, are summed at the rounding of each
    to the type (u) or, fp16, to its subnormal step of 2^-25 at 2^7 times the weight: n 2^-32 of the values in all."""
    dev, D = cuda_device, 64
    u = half_step(dtype)

    def close(out, n, what):
        p = n * math.exp(-gap) / (1 + n * math.exp(-gap))
        sub = n * 2.0 ** -32 if dtype == torch.float16 else 0.0
        want = torch.full(out.shape, p, dtype=F64, device=dev)
        # scores are exact but for the scale and the exponential's argument and value: 2^-18 relative; sums (n / 16 + 64) 2^-24
        tol = (2 * u + 2.0 ** -18 + 2 * gap * 2.0 ** -24 + (n / 16 + 64) * 2.0 ** -24) * p + sub + 1e-30
        check(out, want, torch.full_like(want, tol), what)

    n = 131071
    q = torch.zeros(1, 1, n + 1, D, device=dev, dtype=dtype)
    q[..., 0] = 8.0
    k = torch.zeros(1, 1, n + 1, D, device=dev, dtype=dtype)
    k[0, 0, 0, 0] = gap
    v = torch.ones(1, 1, n + 1, D, device=dev, dtype=dtype)
    v[0, 0, 0] = 0
    if dtype != torch.float32:
        out, _ = kb.attention_b200(q, k, v, causal=True)
        for r in (n, n // 2, 4000):
            close(out[0, 0, r], r, f"prompt row {r}")
    cache_k, cache_v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    for T, Hq in ((1, 4), (3, 8), (40, 8)):
        for off in (None, torch.zeros(1, 1, n + 1, device=dev)):
            out, _ = kb.attention_cached(q[:, :, :1].expand(1, Hq, T, D).contiguous(), cache_k, cache_v, None,
                                         torch.tensor([n + 1]), log_offsets=off)
            for t in range(T):
                close(out[0, :, t], n - (T - 1 - t), f"T={T}")


@pytest.mark.parametrize("wrong", [2 ** 32, -2 ** 32, 2 ** 40 + 3])
def test_ids_and_lengths_past_32_bits(cuda_device, wrong):
    """int64 lengths are clamped and int64 page ids are outside the cache, whatever their low 32 bits say."""
    c = Case([100, 40], 16, 4, 2, 64, 1, torch.bfloat16, cuda_device, seed=2)
    full = torch.tensor([c.L if wrong > 0 else 0, 40], device=cuda_device)
    for lens in (torch.tensor([wrong + 9, 40]), torch.tensor([wrong + 9, 40], device=cuda_device)):
        a = kb.attention_cached(c.q, c.k, c.v, c.table, full)
        b = kb.attention_cached(c.q, c.k, c.v, c.table, lens)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        w = torch.rand(2, 2, c.L, device=cuda_device)
        e, f = (kb.evict_cache(c.k, c.v, c.table, x, w, 40) for x in (full, lens))
        assert torch.equal(e.kept, f.kept) and torch.equal(e.seq_lens, f.seq_lens) and torch.equal(e.k, f.k)
    q, k, v = _inputs(2, 4, 2, 150, 64, torch.bfloat16, 43, cuda_device)
    a = kb.attention_b200(q, k, v, seq_lens=torch.tensor([150 if wrong > 0 else 0, 77]))
    b = kb.attention_b200(q, k, v, seq_lens=torch.tensor([wrong + 5, 77]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    qp, kp, vp = (t[0].transpose(0, 1).contiguous() for t in (q, k, v))
    cu = torch.tensor([0, 70, wrong + 100] if wrong > 0 else [wrong, 70, 150])
    a = kb.attention_varlen(qp, kp, vp, torch.tensor([0, 70, 150]), 150, causal=True)
    b = kb.attention_varlen(qp, kp, vp, cu, 150, causal=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for table in (c.table.long(),):
        kb.check_device_errors()
        table[0, 2] += wrong
        out, lse = kb.attention_cached(c.q, c.k, c.v, table, c.seq_lens)
        with pytest.raises(RuntimeError):
            kb.check_device_errors()
        kb.evict_cache(c.k, c.v, table, c.seq_lens, torch.rand(2, 2, c.L, device=cuda_device), 60)
        with pytest.raises(RuntimeError):
            kb.check_device_errors()
        kb.block_mass_paged(q[:, :, :100].expand(2, 4, 100, 64).contiguous(), c.k, table, seq_lens=c.seq_lens)
        with pytest.raises(RuntimeError):
            kb.check_device_errors()
        pg = int(c.table[0, 2])
        c.k[pg] = 0
        c.v[pg] = 0
        _check(c, out, lse)
    a = kb.block_mass_b200(q, k, causal=True, seq_lens=torch.tensor([150 if wrong > 0 else 0, 77]))
    b = kb.block_mass_b200(q, k, causal=True, seq_lens=torch.tensor([wrong + 5, 77]))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(1, 8), (3, 8), (40, 8)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_non_finite_values_of_small_weight(cuda_device, dtype, T, Hq, value):
    """A non-finite v of a kept key does not vanish where the part of a split cache that holds it weighs next to
    nothing: its column is not finite (a weight that rounds to 0 makes NaN of an infinity), every other one is."""
    n = 6001
    c = Case([n], 16, Hq, 2, 64, T, dtype, cuda_device, seed=T)
    off = torch.zeros(1, 1, c.L, device=cuda_device)
    off[..., :3000] = -1000.0
    for slot, col in ((0, 3), (777, 9), (2999, 20)):
        _put(c, c.v, 0, slot, col, value)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off)
    odd = torch.zeros(64, dtype=torch.bool, device=cuda_device)
    odd[[3, 9, 20]] = True
    assert torch.equal(~torch.isfinite(out), odd.expand(out.shape))
    assert bool(torch.isfinite(lse).all())


def test_device_errors_are_read_together(cuda_device):
    """Words of different kernels set at once: one check reports them (a wait that ran out first) and clears all."""
    lib = _lib.load()
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    c = Case([100, 40], 16, 4, 2, 64, 1, torch.bfloat16, cuda_device, seed=2)
    c.table[0, 2] = -1
    kb.check_device_errors()
    for attend, mass, wait in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 1, 1)):
        if attend:
            kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
        if mass:
            kb.block_mass_paged(c.q.expand(2, 4, 100, 64).contiguous(), c.k, c.table, seq_lens=c.seq_lens)
        if wait:
            waited = ctypes.c_int(-1)
            assert lib.kvbm_selftest_wait_timeout(stream, 20_000, ctypes.byref(waited)) == _lib.KVBM_OK
        want = _lib.KVBM_ERR_TIMEOUT if wait else _lib.KVBM_ERR_PAGE
        assert lib.kvbm_check_device_errors(stream) == want
        assert lib.kvbm_check_device_errors(stream) == _lib.KVBM_OK


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,D", [(1, 8, 64), (1, 32, 128), (4, 8, 128), (1, 4, 256)])
def test_weights_in_two_parts(cuda_device, dtype, T, Hq, D):
    """Up to 32 rows a kv head the weights enter the product with v in two 16-bit parts, u^2 off together: the
    result's own rounding (u) is the only one of its size."""
    c = Case([900, 2500, 77], 16, Hq, 2, D, T, dtype, cuda_device, seed=D + T)
    out, _ = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    u = half_step(dtype)
    for b, n in enumerate(c.lens):
        for h in range(Hq):
            k, v = c.rows(b, h // (Hq // 2))
            o, _, p, tol, _, _ = softmax_rows(c.q[b, h], k, v, cached_keep(n, T, None, cuda_device), 1 / math.sqrt(D),
                                              dtype=torch.float32)
            sub = n * 2.0 ** -32 * float(v.abs().max()) if dtype == torch.float16 else 0.0
            check(out[b, h], o, tol + u * o.abs() + u * u * (1 + 2 * u) * (p @ v.double().abs()) + sub, f"out[{b},{h}]")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [False, True])
def test_decoding_on_after_evictions(cuda_device, dtype, shared):
    """Evictions of uneven caches (empty, shorter than the budget, longer) with decoding in between: each sequence's
    new tokens go to its own next slots, its weights into an array of the compact cache's size."""
    dev, Hq, Hkv, D, budget, room = cuda_device, 8, 2, 64, 60, 12
    c = Case([40, 300, 0, 61, 150], 16, Hq, Hkv, D, 1, dtype, dev, seed=31)
    B, G = len(c.lens), Hq // Hkv
    g = torch.Generator().manual_seed(5)
    rows = torch.arange(B, device=dev)
    k, v, table, lens = c.k, c.v, c.table, c.seq_lens
    w = torch.rand(B, 1 if shared else Hkv, c.L, generator=g).to(dev)
    for turn in range(2):
        old = [[(c.rows(b, h) if turn == 0 else (k[b, :int(lens[b]), h], v[b, :int(lens[b]), h])) for h in range(Hkv)]
               for b in range(B)]
        e = kb.evict_cache(k, v, table, lens, w, budget, n_sinks=4, recency=16, capacity=budget + room)
        want = lens.clamp(max=budget)
        assert torch.equal(e.seq_lens, want)
        for b in range(B):
            for h in range(Hkv):
                kept = evict_rows(w[b, h % w.shape[1]].tolist(), int(lens[b]), budget, 4, 16)
                assert e.kept[b, h % w.shape[1], :len(kept)].tolist() == kept
                assert torch.equal(e.k[b, :len(kept), h], old[b][h][0][kept])
                assert torch.equal(e.v[b, :len(kept), h], old[b][h][1][kept])
        k, v, table, lens = e.k, e.v, None, e.seq_lens
        w = torch.zeros(B, Hkv, budget + room, device=dev)
        w[:, :, :budget] = e.weights
        for _ in range(3):  # one token at a time
            k[rows, lens], v[rows, lens] = (torch.randn(B, Hkv, D, generator=g).to(dtype).to(dev) for _ in range(2))
            lens = lens + 1
            q = torch.randn(B, Hq, 1, D, generator=g).to(dtype).to(dev)
            before = w.clone()
            out, lse, w = kb.attention_cached(q, k, v, table, lens, weights=w)
            for b in range(B):
                n = int(lens[b])
                for h in range(Hkv):
                    total, tol = before[b, h, :n].double(), 0.0
                    for i in range(h * G, (h + 1) * G):
                        o, l, p, ot, lt, pt = softmax_rows(q[b, i], k[b, :n, h], v[b, :n, h],
                                                           cached_keep(n, 1, None, dev), 1 / math.sqrt(D), dtype=dtype)
                        check(out[b, i], o, ot, f"out[{b},{i}]")
                        check(lse[b, i], l, lt, f"lse[{b},{i}]")
                        total, tol = total + p[0], tol + pt[0]
                    check(w[b, h, :n], total, tol + 2.0 ** -23 * total, f"weights[{b},{h}]")
                    assert bool((w[b, h, n:] == 0).all())
        # drafted tokens, dropped again afterwards
        T = 5
        tree = _tree(B, T, turn, dev)
        slots = lens[:, None] + torch.arange(T, device=dev)
        k[rows[:, None], slots], v[rows[:, None], slots] = (torch.randn(B, T, Hkv, D, generator=g).to(dtype).to(dev)
                                                            for _ in range(2))
        q = torch.randn(B, Hq, T, D, generator=g).to(dtype).to(dev)
        out, lse = kb.attention_cached(q, k, v, table, lens + T, tree_mask=tree)
        for b in range(B):
            n = int(lens[b]) + T
            for i in range(Hq):
                o, l, _, ot, lt, _ = softmax_rows(q[b, i], k[b, :n, i // G], v[b, :n, i // G],
                                                  cached_keep(n, T, tree[b], dev), 1 / math.sqrt(D), dtype=dtype)
                check(out[b, i], o, ot, f"tree out[{b},{i}]")
                check(lse[b, i], l, lt, f"tree lse[{b},{i}]")
        if shared:
            w = w.sum(1, keepdim=True)


def test_outputs_over_small_inputs(cuda_device):
    """Outputs over lengths, offsets, tables and masks are refused, as those over q, k and v are."""
    dev = cuda_device
    c = Case([40, 20], 16, 4, 2, 64, 1, torch.bfloat16, dev)
    room = torch.zeros(2, 8, 64, device=dev)  # 4 KB to be shared
    ints, bits = room.view(torch.int32).flatten(), room.view(torch.bool).flatten()
    out = room.view(torch.bfloat16).flatten()[:512].view(2, 4, 1, 64)
    lse = room.flatten()[:8].view(2, 4, 1)
    lens, table = ints[2:4].copy_(c.seq_lens), ints[4:4 + c.table.numel()].view(c.table.shape)
    off = room.flatten()[:2 * c.L].view(2, 1, c.L)
    w = room.flatten()[:4 * c.L].view(2, 2, c.L)
    keep = bits[:1].view(1, 1)
    q, k, v = _inputs(2, 4, 2, 1, 64, torch.bfloat16, 61, dev)
    qp, kp, vp = (t[:, :, 0] for t in (q, k, v))
    call = lambda ln=c.seq_lens, tb=c.table, **kw: kb.attention_cached(c.q, c.k, c.v, tb, ln, **kw)  # noqa: E731
    bad = [
        lambda: kb.attention_b200(q, k, v, seq_lens=lens, out=out),
        lambda: kb.attention_b200(q, k, v, seq_lens=lens, lse_out=lse),
        lambda: kb.attention_b200(q, k, v, attn_mask=bits[:2].view(2, 1, 1), out=out),
        lambda: kb.attention_varlen(qp, kp, vp, ints[:3], 1, out=out[:, :, 0]),
        lambda: kb.attention_varlen(qp, kp, vp, ints[:3], 1, lse_out=room.flatten()[:8].view(4, 2)),
        lambda: call(ln=lens, out=out),
        lambda: call(tb=table, lse_out=lse),
        lambda: call(tree_mask=keep, out=out),
        lambda: call(log_offsets=off, out=out),
        lambda: call(ln=lens, weights=w),
        lambda: call(tb=table, weights=torch.zeros_like(w), weights_out=w),
        lambda: kb.evict_cache(c.k, c.v, c.table, lens, torch.zeros(2, 2, c.L, device=dev), 2, n_sinks=1, recency=1,
                               out=(room.view(torch.bfloat16).flatten()[:512].view(2, 2, 2, 64), torch.empty_like(c.k)[:2, :2])),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {i} was accepted")
