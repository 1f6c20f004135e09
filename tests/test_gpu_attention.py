"""Prompt attention on the GPU (``kvbm_attention``) against a 64-bit restatement.

Bounds: ``_attention_ref``."""

import math

import pytest
import torch

import kvblockmass_b200 as kb
from _attention_ref import check, prompt_keep, softmax_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(B, Hq, Hkv, N, D, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Hq, N, D, generator=g).mul_(1.3).to(dtype).to(dev)
    k = torch.randn(B, Hkv, N, D, generator=g).to(dtype).to(dev)
    v = torch.randn(B, Hkv, N, D, generator=g).to(dtype).to(dev)
    return q, k, v


def _check_dense(q, k, v, out, lse, causal, lens=None, mask=None, scale=None, outside=True):
    B, Hq, N, D = q.shape
    G = Hq // k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        n = N if lens is None else lens[b]
        m = None if mask is None else (mask if mask.dim() == 1 else mask[b, 0])
        keep = prompt_keep(n, causal, m, q.device)
        for h in range(Hq):
            if n:
                o, l, _, ot, lt, _ = softmax_rows(q[b, h, :n], k[b, h // G, :n], v[b, h // G, :n], keep, scale,
                                                  dtype=q.dtype)
                check(out[b, h, :n], o, ot, f"out[{b},{h}]")
                check(lse[b, h, :n], l, lt, f"lse[{b},{h}]")
            if outside:
                assert bool((out[b, h, n:] == 0).all()) and bool((lse[b, h, n:] == -math.inf).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,D,Hq,Hkv", [(1, 64, 2, 1), (2, 128, 4, 2), (63, 64, 3, 3), (64, 128, 2, 1), (65, 64, 8, 2),
                                        (127, 96, 2, 2), (128, 128, 4, 1), (129, 64, 2, 1), (255, 8, 1, 1),
                                        (257, 128, 4, 1), (383, 72, 2, 1), (640, 128, 2, 1), (1025, 64, 2, 2),
                                        (513, 128, 2, 1), (1024, 96, 2, 1), (1537, 128, 3, 1)])
def test_dense(cuda_device, dtype, causal, N, D, Hq, Hkv):
    q, k, v = _inputs(2, Hq, Hkv, N, D, dtype, N * 7 + D, cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=causal)
    assert out.dtype == dtype and lse.dtype == torch.float32
    _check_dense(q, k, v, out, lse, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 7, 20, 130, 192, 256])
def test_head_dims(cuda_device, dtype, D):
    q, k, v = _inputs(1, 4, 2, 150, D, dtype, D, cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=True)
    _check_dense(q, k, v, out, lse, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,D,lens", [(390, 64, [390, 0, 1, 129, 256]), (1300, 128, [1300, 513, 700, 129, 512]),
                                      (1101, 104, [1, 1101, 640, 0, 1024])])
def test_lengths_and_masks(cuda_device, dtype, causal, N, D, lens):
    """Ragged lengths (0 and 1 among them), a key mask that drops the first keys (causal rows left empty), whole
    tiles and single keys; NaN and infinities wherever nothing may be read."""
    B = 5
    q, k, v = _inputs(B, 4, 2, N, D, dtype, 5, cuda_device)
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(B, 1, N, generator=g) > 0.2).to(cuda_device)
    mask[0, 0, :3] = False      # causal: rows 0..2 keep nothing
    mask[3, 0, :] = False       # a sequence that keeps nothing at all
    mask[4, 0, 128:256] = False  # a whole key tile
    for b in range(B):
        gone = torch.ones(N, dtype=torch.bool, device=cuda_device)
        gone[:lens[b]] = ~mask[b, 0, :lens[b]]
        k[b][:, gone] = math.nan
        v[b][:, gone] = math.inf
        v[b][:, gone, ::2] = math.nan
        q[b][:, lens[b]:] = math.nan
    out, lse = kb.attention_b200(q, k, v, attn_mask=mask, causal=causal, seq_lens=torch.tensor(lens))
    _check_dense(q, k, v, out, lse, causal, lens, mask)
    one = mask[0, 0]
    q2, k2, v2 = _inputs(2, 4, 2, N, D, dtype, 6, cuda_device)
    out, lse = kb.attention_b200(q2, k2, v2, attn_mask=one, causal=causal)
    _check_dense(q2, k2, v2, out, lse, causal, None, one)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,at", [(300, 64, 0), (300, 64, 5), (300, 64, 127), (300, 64, 128), (300, 64, 200),
                                    (300, 64, 299), (1100, 128, 0), (1100, 128, 200), (1100, 128, 511),
                                    (1100, 128, 512), (1100, 96, 700), (1100, 128, 1099)])
def test_nan_behind_the_diagonal(cuda_device, dtype, N, D, at):
    """A NaN or an infinity in v (or k) of position j reaches the rows from j on, and none before."""
    q, k, v = _inputs(1, 2, 1, N, D, dtype, 9, cuda_device)
    v[0, 0, at, 3] = math.nan
    v[0, 0, at, 9] = math.inf
    v[0, 0, at, 17] = -math.inf
    v[0, 0, at, D - 1] = math.nan
    out, lse = kb.attention_b200(q, k, v, causal=True)
    _check_dense(q, k, v, out, lse, True)
    assert bool(torch.isfinite(out[:, :, :at]).all())
    clean, _ = kb.attention_b200(q, k, torch.where(torch.isfinite(v), v, 0), causal=True)
    assert torch.equal(out[:, :, :at], clean[:, :, :at])
    k[0, 0, at, 0] = math.nan
    out2, _ = kb.attention_b200(q, k, torch.where(torch.isfinite(v), v, 0), causal=True)
    assert torch.equal(out2[:, :, :at], clean[:, :, :at])
    assert bool(torch.isnan(out2[:, :, at:]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,D", [([1], 64), ([5, 0, 130, 1, 64], 64), ([0, 0, 257], 64), ([300, 128, 2], 64),
                                    ([600, 0, 1, 1000, 513, 64], 128), ([1025], 120), ([3, 2049, 512], 128)])
def test_packed(cuda_device, dtype, causal, lens, D):
    Hq, Hkv, lead, tail = 4, 2, 3, 5
    T = lead + sum(lens) + tail
    q, k, v = (t[0].transpose(0, 1).contiguous() for t in _inputs(1, Hq, Hkv, T, D, dtype, 11, cuda_device))
    q, k, v = q[:, :Hq], k[:, :Hkv], v[:, :Hkv]
    cu = torch.tensor([lead + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=cuda_device)
    for t in (k, v):  # rows of no sequence
        t[:lead] = math.nan
        t[T - tail:] = math.inf
    out, lse = kb.attention_varlen(q, k, v, cu, causal=causal)
    for b, n in enumerate(lens):
        r0 = int(cu[b])
        if n:
            _check_dense(*(t[r0:r0 + n].transpose(0, 1)[None] for t in (q, k, v)),
                         out[r0:r0 + n].transpose(0, 1)[None], lse[:, r0:r0 + n][None], causal)
    gone = torch.ones(T, dtype=torch.bool, device=cuda_device)
    gone[lead:T - tail] = False
    assert bool((out[gone] == 0).all()) and bool((lse[:, gone] == -math.inf).all())
    # given memory: rows of no sequence stay as they were, the rest has the same bits
    o2, l2 = torch.full_like(out, 7), torch.full_like(lse, 7)
    kb.attention_varlen(q, k, v, cu, max(max(lens), 1), causal=causal, out=o2, lse_out=l2)
    assert bool((o2[gone] == 7).all()) and bool((l2[:, gone] == 7).all())
    assert torch.equal(o2[~gone], out[~gone]) and torch.equal(l2[:, ~gone], lse[:, ~gone])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,Hq", [(70, 64, 2), (33, 128, 3), (200, 64, 1)])
def test_many_sequences(cuda_device, dtype, B, D, Hq):
    """More sequences than a warp has lanes, packed and padded, most of one row tile or two."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 270, (B,), generator=g).tolist()
    lens[1], lens[31], lens[32], lens[-1] = 0, 1, 600, 300
    N = max(lens)
    q, k, v = _inputs(B, Hq, 1, N, D, dtype, 12, cuda_device)
    rows = torch.tensor(lens, device=cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=True, seq_lens=rows)
    _check_dense(q, k, v, out, lse, True, lens)
    inside = (torch.arange(N, device=cuda_device) < rows[:, None])
    pq, pk, pv = (t.transpose(1, 2)[inside].contiguous() for t in (q, k, v))
    cu = torch.tensor([sum(lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=cuda_device)
    pout, plse = kb.attention_varlen(pq, pk, pv, cu, N, causal=True)
    back = torch.zeros_like(out).transpose(1, 2).contiguous()
    back[inside] = pout
    lback = torch.full_like(lse, -math.inf).transpose(1, 2).contiguous()
    lback[inside] = plse.T
    _check_dense(q, k, v, back.transpose(1, 2), lback.transpose(1, 2), True, lens)


def test_packed_cut_and_wrong_offsets(cuda_device):
    """Sequences longer than max_seqlen are cut there; offsets outside the rows are clamped."""
    q, k, v = (t[0].transpose(0, 1).contiguous() for t in _inputs(1, 2, 1, 200, 64, torch.bfloat16, 12, cuda_device))
    cu = torch.tensor([0, 150, 200], dtype=torch.int32, device=cuda_device)
    out, lse = kb.attention_varlen(q, k, v, cu, 100, causal=True)
    want, wl = kb.attention_varlen(q[:100], k[:100], v[:100], cu[:2].clamp(max=100), 100, causal=True)
    assert torch.equal(out[:100], want) and torch.equal(lse[:, :100], wl)
    assert bool((out[100:150] == 0).all()) and bool((lse[:, 100:150] == -math.inf).all())
    for bad in ([-5, 150, 900], [0, 300, 200]):
        out, lse = kb.attention_varlen(q, k, v, torch.tensor(bad, device=cuda_device), 200, causal=True)
        assert bool(torch.isfinite(out[:150]).all())
    kb.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_out(cuda_device, dtype):
    """[B, N, H, D] memory, rows with a gap, an offset that breaks 16-byte alignment, expanded kv heads."""
    g = torch.Generator().manual_seed(2)
    B, N, Hq, Hkv, D = 2, 140, 4, 2, 64
    base = torch.randn(B, N, Hq + 2 * Hkv, D + 8, generator=g).to(dtype).to(cuda_device)
    qkv = base[..., :D].transpose(1, 2)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    lens = torch.tensor([140, 77], device=cuda_device)
    out, lse = torch.full((B, N, Hq, D), 5.0, dtype=dtype, device=cuda_device).transpose(1, 2), \
        torch.full((B, Hq, N), 5.0, device=cuda_device)
    kb.attention_b200(q, k, v, causal=True, seq_lens=lens, out=out, lse_out=lse)
    _check_dense(q, k, v, out, lse, True, lens.tolist(), outside=False)
    assert bool((out[1, :, 77:] == 5).all()) and bool((lse[1, :, 77:] == 5).all())
    odd = torch.randn(B * Hkv * N * D + 1, generator=g).to(dtype).to(cuda_device)[1:].view(B, Hkv, N, D)
    out, lse = kb.attention_b200(q, odd, v, causal=False, scale=0.3)
    _check_dense(q, odd, v, out, lse, False, scale=0.3)
    k1 = k[:, :1].expand(B, Hkv, N, D)
    out, lse = kb.attention_b200(q, k1, v, causal=True)
    _check_dense(q, k1, v, out, lse, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(cuda_device, dtype):
    """Heads, and positions, more than 2^32 elements apart in one buffer."""
    dev, N, D = cuda_device, 200, 64
    q, k, v = _inputs(1, 2, 2, N, D, dtype, 21, dev)
    room = torch.empty(2 ** 32 + 2 ** 20, dtype=dtype, device=dev)
    apart = 2 ** 32 + 64 * 1024
    for strides in ((0, apart, D, 1), (0, D, (2 ** 32 // (N - 1) + 999) // 8 * 8, 1)):
        big = room.as_strided((1, 2, N, D), strides)
        for a in range(3):
            args = [q, k, v]
            big.copy_(args[a])
            args[a] = big
            out, lse = kb.attention_b200(*args, causal=True)
            _check_dense(*args, out, lse, True)
        o = torch.as_strided(room, (1, 2, N, D), strides)
        kb.attention_b200(q, k, v, causal=True, out=o)
        assert torch.equal(o, kb.attention_b200(q, k, v, causal=True)[0])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 4.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(cuda_device, dtype, scale):
    q, k, v = _inputs(1, 2, 1, 200, 64, dtype, 21, cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=True, scale=scale)
    _check_dense(q, k, v, out, lse, True, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_rows_sampled(cuda_device, dtype):
    """A long prompt: sampled rows, large and small scores (a running maximum that keeps growing)."""
    N, D = 6000, 128
    q, k, v = _inputs(1, 4, 1, N, D, dtype, 31, cuda_device)
    k *= torch.linspace(0.1, 4.0, N, device=cuda_device)[:, None].to(dtype)
    out, lse = kb.attention_b200(q, k, v, causal=True)
    for r in (0, 1, 127, 128, 255, 256, 3000, 4095, 4096, 5887, 5999):
        for h in range(4):
            keep = torch.ones(1, r + 1, dtype=torch.bool, device=cuda_device)
            o, l, _, ot, lt, _ = softmax_rows(q[0, h, r:r + 1], k[0, 0, :r + 1], v[0, 0, :r + 1], keep,
                                              1 / math.sqrt(D), dtype=dtype)
            check(out[0, h, r:r + 1], o, ot, f"row {r}")
            check(lse[0, h, r:r + 1], l, lt, f"lse {r}")


@pytest.mark.parametrize("N,D,Hq", [(300, 64, 8), (700, 128, 8), (2300, 128, 40)])
def test_deterministic_streams_and_graph(cuda_device, N, D, Hq):
    q, k, v = _inputs(2, Hq, 2, N, D, torch.bfloat16, 41, cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = kb.attention_b200(q, k, v, causal=True)
    side.synchronize()
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    o3, l3 = torch.zeros_like(out), torch.zeros_like(lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kb.attention_b200(q, k, v, causal=True, out=o3, lse_out=l3)
    q.copy_(q.flip(0))
    k.copy_(k.flip(0))
    v.copy_(v.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.flip(0), o3) and torch.equal(lse.flip(0), l3)


@pytest.mark.parametrize("N,D,Hq", [(300, 64, 8), (1000, 128, 4), (1030, 64, 40), (200, 200, 4)])
def test_fp32_deterministic_streams_and_graph(cuda_device, N, D, Hq):
    q, k, v = _inputs(2, Hq, 2, N, D, torch.float32, 42, cuda_device)
    lens = torch.tensor([N, N // 3], dtype=torch.int32, device=cuda_device)
    out, lse = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    _check_dense(q, k, v, out, lse, True, lens.tolist())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    o1, l1 = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    side.synchronize()
    assert torch.equal(out, o2) and torch.equal(lse, l2) and torch.equal(out, o1) and torch.equal(lse, l1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o3, l3 = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    lens.copy_(torch.tensor([1, N]))
    g.replay()
    want = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    assert torch.equal(o3, want[0]) and torch.equal(l3, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_out_of_range(cuda_device, dtype):
    """Lengths past N count as N, negative ones as 0."""
    q, k, v = _inputs(3, 4, 2, 150, 64, dtype, 43, cuda_device)
    for causal in (False, True):
        a = kb.attention_b200(q, k, v, causal=causal, seq_lens=torch.tensor([150, 0, 77]))
        b = kb.attention_b200(q, k, v, causal=causal, seq_lens=torch.tensor([2 ** 31 - 1, -1, 77]))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_feeds_block_mass(cuda_device):
    """The run of a prompt: attention, its lse into the block mass, and the mass of a call without it."""
    q, k, v = _inputs(2, 8, 2, 1000, 128, torch.bfloat16, 51, cuda_device)
    lens = torch.tensor([1000, 611], device=cuda_device)
    _, lse = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    a = kb.block_mass_b200(q, k, causal=True, seq_lens=lens, per_sequence=True, lse=lse)
    b = kb.block_mass_b200(q, k, causal=True, seq_lens=lens, per_sequence=True)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    assert torch.allclose(a.sum(1).cpu(), torch.tensor([8000.0, 611 * 8.0]), rtol=1e-4)
    cu = torch.tensor([0, 389, 1000], dtype=torch.int32, device=cuda_device)
    qp, kp, vp = (t[0].transpose(0, 1).contiguous() for t in (q, k, v))
    _, lse = kb.attention_varlen(qp, kp, vp, cu, 611, causal=True)
    a = kb.block_mass_varlen(qp, kp, cu, 611, causal=True, lse=lse)
    b = kb.block_mass_varlen(qp, kp, cu, 611, causal=True)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


def test_refusals(cuda_device):
    q, k, v = _inputs(1, 4, 2, 20, 64, torch.bfloat16, 61, cuda_device)
    bad = [
        (ValueError, lambda: kb.attention_b200(q.cpu(), k.cpu(), v.cpu())),
        (ValueError, lambda: kb.attention_b200(q, k.float(), v)),
        (ValueError, lambda: kb.attention_b200(q.double(), k.double(), v.double())),
        (ValueError, lambda: kb.attention_b200(q[:, :3], k, v)),
        (ValueError, lambda: kb.attention_b200(q, k[:, :, :10], v)),
        (ValueError, lambda: kb.attention_b200(q[0], k[0], v[0])),
        (ValueError, lambda: kb.attention_b200(q, k, v, attn_mask=torch.ones(20, 20, dtype=torch.bool))),
        (ValueError, lambda: kb.attention_b200(q, k, v, seq_lens=torch.tensor([1, 2]))),
        (ValueError, lambda: kb.attention_b200(q, k, v, seq_lens=torch.tensor([1.0]))),
        (ValueError, lambda: kb.attention_b200(q, k, v, scale=math.nan)),
        (ValueError, lambda: kb.attention_b200(q, k, v, scale=math.inf)),
        (ValueError, lambda: kb.attention_b200(q, k, v, out=q)),
        (ValueError, lambda: kb.attention_b200(q, k, v, out=torch.empty(1, 4, 20, 32, device=cuda_device))),
        (ValueError, lambda: kb.attention_b200(q, k, v, out=torch.empty_like(q)[:, :1].expand(1, 4, 20, 64))),
        (ValueError, lambda: kb.attention_b200(q[:, :, :0], k[:, :, :0], v[:, :, :0])),
        (TypeError, lambda: kb.attention_b200(q, k, None)),
        (ValueError, lambda: kb.attention_varlen(q, k, v, torch.tensor([0, 20]))),
        (ValueError, lambda: kb.attention_varlen(q[0], k[0], v[0], torch.tensor([0]))),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()
    big = torch.zeros(1, 1, 4, 264, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError):
        kb.attention_b200(big, big.clone(), big.clone())


def test_empty_packed(cuda_device):
    z = torch.zeros(0, 4, 64, dtype=torch.float16, device=cuda_device)
    out, lse = kb.attention_varlen(z, z[:, :2], z[:, :2], torch.zeros(3, dtype=torch.int32, device=cuda_device))
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
