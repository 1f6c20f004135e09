"""Attention of one token or a drafted tree over a paged cache, and eviction
from it (``kvbm_cached_attention``, ``kvbm_evict_cache``), against 64-bit
restatements.  Bounds: ``_attention_ref``."""

import math

import pytest
import torch

import kvblockmass_b200 as kb
from _attention_ref import cached_keep, check, evict_rows, softmax_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


class Case:
    def __init__(self, lens, page, Hq, Hkv, D, T, dtype, dev, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.T = lens, page, T
        B, per = len(lens), max(1, -(-max(lens) // page))
        pages = B * per + spare
        perm = torch.randperm(pages, generator=g)
        self.table = perm[:B * per].view(B, per).to(torch.int32).to(dev)
        self.unused = perm[B * per:].to(dev)
        self.q = torch.randn(B, Hq, T, D, generator=g).mul_(1.3).to(dtype).to(dev)
        self.k = torch.randn(pages, page, Hkv, D, generator=g).to(dtype).to(dev)
        self.v = torch.randn(pages, page, Hkv, D, generator=g).to(dtype).to(dev)
        self.k[self.unused] = math.nan
        self.v[self.unused] = math.nan
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.L = per * page

    def rows(self, b, g):
        n = self.lens[b]
        pos = torch.arange(n, device=self.k.device)
        at = self.table[b].long()[pos // self.page], pos % self.page, g
        return self.k[at], self.v[at]

    def poison_tail(self):
        """NaN in every slot past a sequence's end, and in table entries past its pages."""
        for b, n in enumerate(self.lens):
            for c in range(n, self.L):
                pg = int(self.table[b, c // self.page])
                self.k[pg, c % self.page] = math.nan
                self.v[pg, c % self.page] = math.nan
            used = -(-n // self.page)
            self.table[b, used:] = -7
        return self


def _check(c, out, lse, tree=None, off=None, scale=None, weights=None, wout=None, wbefore=None):
    B, Hq, T, D = c.q.shape
    Hkv = c.k.shape[2]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        n = c.lens[b]
        if n == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        keep = cached_keep(n, T, None if tree is None else (tree if tree.dim() == 2 else tree[b % tree.shape[0]]),
                           c.q.device)
        for g in range(Hkv):
            k, v = c.rows(b, g)
            o_off = None
            kp = keep
            if off is not None:
                o_off = off[b % off.shape[0], g % off.shape[1], :n]
                kp = keep & (o_off != -math.inf)[None]
            psum = 0
            ptol = 0
            for h in range(g * G, (g + 1) * G):
                o, l, p, ot, lt, pt = softmax_rows(c.q[b, h], k, v, kp, scale, o_off, dtype=c.q.dtype)
                check(out[b, h], o, ot, f"out[{b},{h}]")
                check(lse[b, h], l, lt, f"lse[{b},{h}]")
                psum, ptol = psum + p[0], ptol + pt[0]
            if wout is not None:
                w = weights[b, g, :n].double()
                check(wout[b, g, :n], w + psum, ptol + 2.0 ** -23 * (w + psum).abs(), f"weights[{b},{g}]")
                if wbefore is not None:
                    assert torch.equal(wout[b, g, n:], wbefore[b, g, n:])


def _tree(B, T, seed, dev):
    g = torch.Generator().manual_seed(seed)
    m = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
    for b in range(B):
        for t in range(1, T):
            m[b, t] |= m[b, int(torch.randint(0, t, (1,), generator=g))]
    return m.to(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 5, 16, 64, 200])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 2, 128), (7, 1, 64), (6, 2, 40), (32, 2, 128), (2, 1, 256)])
def test_single_token(cuda_device, dtype, page, Hq, Hkv, D):
    c = Case([1, 63, 64, 65, 0, 333, 129], page, Hq, Hkv, D, 1, dtype, cuda_device, seed=page + D).poison_tail()
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    _check(c, out, lse)
    kb.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D", [(64, 1, 64), (136, 1, 128), (72, 2, 96), (400, 1, 64)])
@pytest.mark.parametrize("offsets", [False, True])
def test_single_token_of_large_groups(cuda_device, dtype, Hq, Hkv, D, offsets):
    """More rows per kv head than 32 with one token, and more than 256."""
    c = Case([700, 1, 0, 129, 64], 16, Hq, Hkv, D, 1, dtype, cuda_device, seed=Hq)
    off = None
    if offsets:
        off = torch.randn(len(c.lens), Hkv, c.L, generator=torch.Generator().manual_seed(3))
        off[:, :, ::7] = -math.inf
        off[3] = -math.inf  # keeps nothing
        off = off.to(cuda_device)
    c.poison_tail()
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off)
    _check(c, out, lse, off=off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2, 5, 16, 33, 64])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 2, 128), (7, 1, 64), (2, 1, 192)])
def test_tree(cuda_device, dtype, T, Hq, Hkv, D):
    c = Case([T, T + 1, 64 + T // 2, 300, 0, 128 + T], 16, Hq, Hkv, D, T, dtype, cuda_device, seed=T).poison_tail()
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    _check(c, out, lse)
    tree = _tree(6, T, T, cuda_device)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    _check(c, out, lse, tree)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree[0], scale=0.07)
    _check(c, out, lse, tree[0], scale=0.07)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [1, 5, 8, 24, 32, 64, 128, 256, 384])
@pytest.mark.parametrize("T,Hq,D", [(21, 4, 128), (40, 8, 64), (64, 8, 96)])
def test_tree_pages(cuda_device, dtype, page, T, Hq, D):
    """Page sizes that tile 128 keys and ones that do not, bad pages among them, with and without offsets."""
    c = Case([T, 128, 129, 640, 777, 0], page, Hq, 2, D, T, dtype, cuda_device, seed=page).poison_tail()
    tree = _tree(6, T, page, cuda_device)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    _check(c, out, lse, tree)
    g = torch.Generator().manual_seed(page)
    off = (3 * torch.rand(6, 1, c.L, generator=g)).to(cuda_device)
    off[torch.rand(off.shape, generator=g).to(cuda_device) < 0.3] = -math.inf
    for b in range(6):
        for s in (off[b, 0, :c.lens[b]] == -math.inf).nonzero()[:, 0].tolist()[:40]:
            pg = int(c.table[b, s // page])
            c.k[pg, s % page] = math.nan
            c.v[pg, s % page] = math.inf
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree, log_offsets=off)
    _check(c, out, lse, tree, off=off)
    kb.check_device_errors()
    c = Case([640, 777], page, Hq, 2, D, T, dtype, cuda_device, seed=page + 1).poison_tail()
    pg = int(c.table[1, 100 // page])
    c.table[1, 100 // page] = 1 << 30
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    with pytest.raises(RuntimeError):
        kb.check_device_errors()
    c.table[1, 100 // page] = pg
    c.k[pg] = 0
    c.v[pg] = 0
    _check(c, out, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(9, 4), (20, 8), (40, 8), (30, 4)])
def test_tree_rows_of_their_own(cuda_device, dtype, T, Hq):
    """A mask row that keeps no drafted token (and with lens = T nothing at all), a cache shorter than the tree, and
    NaN or infinities in the k and v of one branch, which reach the tokens that attend to it and no other."""
    c = Case([T, T - 5, 70, 131, 300], 8, Hq, 2, 64, T, dtype, cuda_device, seed=5)
    tree = _tree(5, T, 1, cuda_device)
    tree[:, 3] = False
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    _check(c, out, lse, tree)
    assert bool((out[0, :, 3] == 0).all()) and bool((lse[0, :, 3] == -math.inf).all())
    clean = out.clone()
    tree[:, :, 5] = False
    tree[:, 5, 5] = tree[:, 7, 5] = True
    clean, _ = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    for b, n in enumerate(c.lens):
        s = n - T + 5
        if s >= 0:
            pg = int(c.table[b, s // 8])
            c.v[pg, s % 8, :, 1] = math.nan
            c.v[pg, s % 8, :, 2] = math.inf
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree)
    _check(c, out, lse, tree)
    rest = [t for t in range(T) if t not in (5, 7)]
    assert torch.equal(out[:, :, rest], clean[:, :, rest])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 6, 16, 40])
@pytest.mark.parametrize("heads", [1, 2])
def test_log_offsets(cuda_device, dtype, T, heads):
    c = Case([T + 9, 200, 64, 131], 16, 8, 2, 64, T, dtype, cuda_device, seed=8)
    g = torch.Generator().manual_seed(1)
    off = (3 * torch.rand(4, heads, c.L, generator=g)).to(cuda_device)
    off[torch.rand(off.shape, generator=g).to(cuda_device) < 0.4] = -math.inf
    off[2, :, :] = -math.inf  # nothing kept
    for b in range(4):
        for h in range(2):
            gone = (off[b, h % heads, :c.lens[b]] == -math.inf).nonzero()[:, 0]
            for s in gone.tolist():
                pg = int(c.table[b, s // 16])
                c.k[pg, s % 16, h] = math.nan
                c.v[pg, s % 16, h] = math.inf
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off)
    _check(c, out, lse, off=off)
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    flat = off[:, 0].contiguous()
    if heads == 1:
        out2, lse2 = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=flat)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lowest_value_offsets(cuda_device, dtype):
    """Offsets of float32's lowest value are a mask only next to others: where all keys have them, all weigh alike."""
    c = Case([50, 130], 16, 4, 2, 64, 1, dtype, cuda_device, seed=9)
    low = torch.finfo(torch.float32).min
    off = torch.zeros(2, 1, c.L, device=cuda_device)
    off[0] = low
    off[1, :, :100] = low
    w = torch.zeros(2, 2, c.L, device=cuda_device)
    out, lse, wo = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off, weights=w)
    for h in range(4):
        want = c.rows(0, h // 2)[1].double().mean(0)
        mass = c.rows(0, h // 2)[1].double().abs().mean(0)
        u = torch.finfo(dtype).eps / 2
        # equal weights: exact but for the sums, the rounded weights and the rounded result
        check(out[0, h, 0], want, 2 * u * mass + u * want.abs() + 2.0 ** -18 * mass, "uniform")
    assert bool((lse[0] == low).all())
    assert torch.allclose(wo[0, :, :50], torch.full((2, 50), 2 / 50, device=cuda_device), rtol=2.0 ** -18)
    k1, v1 = (t[100:130] for t in c.rows(1, 0))
    o, l, *_t = softmax_rows(c.q[1, 0], k1, v1, torch.ones(1, 30, dtype=torch.bool, device=cuda_device), 0.125,
                             dtype=dtype)
    check(out[1, 0], o, _t[1], "kept part")
    assert bool((wo[1, :, :100] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(5, 4), (20, 8), (40, 8)])
def test_lowest_value_offsets_of_a_tree(cuda_device, dtype, T, Hq):
    c = Case([150, 130, T], 16, Hq, 2, 64, T, dtype, cuda_device, seed=19)
    low = torch.finfo(torch.float32).min
    off = torch.full((3, 1, c.L), low, device=cuda_device)
    off[1, :, 60:] = 0.0
    tree = _tree(3, T, 2, cuda_device)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, tree_mask=tree, log_offsets=off)
    u = torch.finfo(dtype).eps / 2
    for b in (0, 2):  # every key alike
        keep = cached_keep(c.lens[b], T, tree[b], cuda_device).double()
        for h in range(Hq):
            v = c.rows(b, h // (Hq // 2))[1].double()
            want, mass = keep @ v / keep.sum(1, keepdim=True), keep @ v.abs() / keep.sum(1, keepdim=True)
            check(out[b, h], want, 2 * u * mass + u * want.abs() + 2.0 ** -18 * mass, "uniform")
        assert bool((lse[b] == low).all())
    keep = cached_keep(130, T, tree[1], cuda_device)[:, 60:]
    for h in range(Hq):
        k, v = (t[60:] for t in c.rows(1, h // (Hq // 2)))
        o, l, _, ot, lt, _ = softmax_rows(c.q[1, h], k, v, keep, 0.125, dtype=dtype)
        check(out[1, h], o, ot, "kept part")
        check(lse[1, h], l, lt, "kept part")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 12, 40])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(cuda_device, dtype, T, scale):
    c = Case([200, T, 77], 16, 8, 2, 64, T, dtype, cuda_device, seed=29)
    off = torch.rand(3, 2, c.L, device=cuda_device)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, scale=scale)
    _check(c, out, lse, scale=scale)
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, scale=scale, log_offsets=off)
    _check(c, out, lse, scale=scale, off=off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 8, 64), (8, 2, 128), (14, 2, 64), (40, 2, 64)])
def test_weights(cuda_device, dtype, Hq, Hkv, D):
    c = Case([1, 64, 257, 0, 700], 16, Hq, Hkv, D, 1, dtype, cuda_device, seed=D).poison_tail()
    g = torch.Generator().manual_seed(4)
    w = torch.rand(5, Hkv, c.L, generator=g).to(cuda_device)
    wo = torch.full_like(w, 3.0)
    out, lse, got = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, weights=w, weights_out=wo)
    assert got is wo
    _check(c, out, lse, weights=w, wout=wo, wbefore=torch.full_like(w, 3.0))
    w2 = w.clone()
    o2, l2, got = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, weights=w2)
    assert got is w2 and torch.equal(o2, out) and torch.equal(l2, lse)
    for b, n in enumerate(c.lens):
        assert torch.equal(w2[b, :, :n], wo[b, :, :n]) and torch.equal(w2[b, :, n:], w[b, :, n:])
    plain, pl = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    assert torch.equal(plain, out) and torch.equal(pl, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(1, 4), (1, 32), (16, 8), (13, 16), (40, 16)])
def test_many_sequences(cuda_device, dtype, T, Hq):
    """More units than CTAs, and lengths far apart: every way a unit can fall on the split."""
    g = torch.Generator().manual_seed(7)
    lens = [int(x) for x in torch.randint(T, 900, (45,), generator=g)]
    lens[3], lens[17], lens[44] = 0, T, 0
    c = Case(lens, 16, Hq, 4, 64, T, dtype, cuda_device, seed=13).poison_tail()
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    _check(c, out, lse)


def test_long_cache(cuda_device):
    """One sequence over every SM, with offsets past 2^31 bytes into the cache."""
    n, D, Hkv = 100_003, 128, 2
    dev = cuda_device
    k = torch.zeros(5_000_000 // 64, 64, Hkv, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    per = -(-n // 64)
    table = (k.shape[0] - 1 - torch.arange(per, device=dev)).to(torch.int32)[None]
    g = torch.Generator(device="cuda").manual_seed(3)
    k[-per:] = torch.randn(per, 64, Hkv, D, generator=g, device=dev).bfloat16()
    v[-per:] = torch.randn(per, 64, Hkv, D, generator=g, device=dev).bfloat16()
    q = torch.randn(1, 8, 1, D, generator=g, device=dev).bfloat16()
    out, lse = kb.attention_cached(q, k, v, table, torch.tensor([n]))
    pos = torch.arange(n, device=dev)
    for h in range(8):
        at = table[0].long()[pos // 64], pos % 64, h // 4
        o, l, _, ot, lt, _ = softmax_rows(q[0, h], k[at], v[at], torch.ones(1, n, dtype=torch.bool, device=dev),
                                          1 / math.sqrt(D), dtype=torch.bfloat16)
        check(out[0, h], o, ot, "out")
        check(lse[0, h], l, lt, "lse")


@pytest.mark.parametrize("dtype,T,page", [(torch.bfloat16, 1, 64), (torch.float16, 40, 64), (torch.bfloat16, 40, 24),
                                          (torch.float32, 1, 64), (torch.float32, 40, 24)])
def test_offsets_past_32_bits(cuda_device, dtype, T, page):
    """The last pages of a cache of more than 2^32 elements; their eviction."""
    n, D, Hkv, dev = 1001, 128, 2, cuda_device
    pages = 2 ** 32 // (page * Hkv * D) + 60
    k = torch.empty(pages, page, Hkv, D, dtype=dtype, device=dev)
    per = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(5)
    k[-per:] = torch.randn(per, page, Hkv, D, generator=g, device=dev).to(dtype)
    table = (pages - 1 - torch.arange(per, device=dev)).to(torch.int32)[None]
    q = torch.randn(1, 4, T, D, generator=g, device=dev).to(dtype)
    out, lse = kb.attention_cached(q, k, k, table, torch.tensor([n]))
    pos = torch.arange(n, device=dev)
    rows = k[table[0].long()[pos // page], pos % page]
    for h in range(4):
        o, l, _, ot, lt, _ = softmax_rows(q[0, h], rows[:, h // 2], rows[:, h // 2], cached_keep(n, T, None, dev),
                                          1 / math.sqrt(D), dtype=dtype)
        check(out[0, h], o, ot, "out")
        check(lse[0, h], l, lt, "lse")
    w = torch.rand(1, 1, per * page, generator=g, device=dev)
    e = kb.evict_cache(k, k, table, torch.tensor([n]), w, 500)
    assert torch.equal(e.k[0], rows[e.kept[0, 0].long()]) and torch.equal(e.v, e.k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_no_table(cuda_device, dtype):
    """Head-major memory without a table, rows with a gap, q and out transposed, k off 16-byte alignment."""
    B, L, Hq, Hkv, D, T = 3, 150, 4, 2, 64, 3
    g = torch.Generator().manual_seed(6)
    mem = torch.randn(2, B, Hkv, L, D + 8, generator=g).to(dtype).to(cuda_device)
    k, v = mem[0, ..., :D].transpose(1, 2), mem[1, ..., :D].transpose(1, 2)
    q = torch.randn(B, T, Hq, D, generator=g).to(dtype).to(cuda_device).transpose(1, 2)
    lens = torch.tensor([150, 71, 3], device=cuda_device)
    out = torch.empty(B, T, Hq, D, dtype=dtype, device=cuda_device).transpose(1, 2)
    lse = torch.empty(B, T, Hq, device=cuda_device).transpose(1, 2)
    kb.attention_cached(q, k, v, None, lens, out=out, lse_out=lse)

    class C:
        pass

    c = C()
    c.q, c.k, c.lens = q, k, lens.tolist()
    c.rows = lambda b, g: (k[b, :c.lens[b], g], v[b, :c.lens[b], g])
    _check(c, out, lse)
    flat = torch.randn(B * L * Hkv * D + 1, generator=g).to(dtype).to(cuda_device)
    k = c.k = flat[1:].view(B, L, Hkv, D)
    out, lse = kb.attention_cached(q, k, v, None, lens)
    _check(c, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_pages(cuda_device, dtype):
    """A page id outside the cache counts as zero vectors and is reported."""
    c = Case([100, 40], 16, 4, 2, 64, 1, dtype, cuda_device, seed=2)
    pg = int(c.table[0, 2])
    c.table[0, 2] = c.k.shape[0] + 5
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
    with pytest.raises(RuntimeError):
        kb.check_device_errors()
    kb.check_device_errors()
    c.table[0, 2] = pg
    c.k[pg] = 0
    c.v[pg] = 0
    _check(c, out, lse)
    w = torch.rand(2, 2, c.L, device=cuda_device)
    c.table[0, 2] = -1
    e = kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 90, n_sinks=64, recency=26)
    with pytest.raises(RuntimeError):
        kb.check_device_errors()
    assert bool((e.k[0, 32:48] == 0).all()) and bool((e.k[0, :32] != 0).any())


@pytest.mark.parametrize("T", [1, 8, 20, 50])
def test_two_calls_and_graphs(cuda_device, T):
    """Calls on two streams at once, and a captured call replayed on new lengths."""
    c = Case([900, 333, 64, 700], 16, 8, 2, 128, T, torch.bfloat16, cuda_device, seed=3)
    d = Case([100, 950, 7 + T, 180], 16, 8, 2, 128, T, torch.bfloat16, cuda_device, seed=4)
    want = [kb.attention_cached(x.q, x.k, x.v, x.table, x.seq_lens) for x in (c, d)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, (c, d)):
            with torch.cuda.stream(s):
                got.append(kb.attention_cached(x.q, x.k, x.v, x.table, x.seq_lens))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    need = kb.cached_attention_workspace_bytes(c.q, c.k, c.v, c.table, c.seq_lens)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    out, lse = torch.zeros_like(c.q), torch.zeros(4, 8, T, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, out=out, lse_out=lse, workspace=ws)
    for lens in ([900, 333, 64, 700], [T, 0, 301, 64], [899, 900, 900, 900]):
        c.seq_lens.copy_(torch.tensor(lens))
        ws.fill_(0xFF)
        graph.replay()
        w = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens)
        assert torch.equal(out, w[0]) and torch.equal(lse, w[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_run(cuda_device, dtype):
    """A decode step that accumulates weights, an eviction and a tree over the compact cache, captured as one graph with
    its own memory, replayed on new inputs beside eager calls of the same kind."""
    T = 5
    c = Case([900, 333, 64, 700], 16, 8, 2, 64, 1, dtype, cuda_device, seed=3)
    w = torch.rand(4, 2, c.L, device=cuda_device)
    qt = torch.randn(4, 8, T, 64, device=cuda_device).to(dtype)
    room = tuple(torch.zeros(4, 208, 2, 64, dtype=dtype, device=cuda_device) for _ in range(2))

    def run(w, room):
        out, lse, w2 = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, weights=w, weights_out=torch.zeros_like(w))
        e = kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w2, 200, out=room)
        return (out, lse, w2, e.kept, e.weights, e.seq_lens, *kb.attention_cached(qt, e.k, e.v, None, e.seq_lens))

    run(w, room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(w, room)
    other = tuple(t.clone() for t in room)
    for lens in ([900, 333, 64, 700], [200, 0, 201, 64], [899, 900, 900, 900]):
        c.seq_lens.copy_(torch.tensor(lens))
        w.copy_(torch.rand(w.shape))
        graph.replay()
        want = run(w, other)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_lengths_out_of_range(cuda_device, dtype, T):
    """Lengths past the table's pages count as all of them, negative ones as 0."""
    c = Case([320, 320, 100], 16, 8, 2, 64, T, dtype, cuda_device, seed=4)
    right = torch.tensor([320, 0, 100], dtype=torch.int32, device=cuda_device)
    wrong = torch.tensor([2 ** 31 - 1, -5, 100], dtype=torch.int32, device=cuda_device)
    for a, b in zip(kb.attention_cached(c.q, c.k, c.v, c.table, right),
                    kb.attention_cached(c.q, c.k, c.v, c.table, wrong)):
        assert torch.equal(a, b)
    w = torch.rand(3, 2, c.L, device=cuda_device)
    e, f = (kb.evict_cache(c.k, c.v, c.table, n, w, 64) for n in (right, wrong))
    for name in ("k", "v", "seq_lens", "kept", "weights"):
        assert torch.equal(getattr(e, name), getattr(f, name))
    if T == 1:
        a = kb.attention_cached(c.q, c.k, c.v, c.table, right, weights=w.clone())
        b = kb.attention_cached(c.q, c.k, c.v, c.table, wrong, weights=w.clone())
        assert torch.equal(a[2], b[2]) and torch.equal(a[2][1], w[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("budget,n_sinks,recency", [(1, 0, 0), (1, 1, 0), (40, 4, 32), (36, 4, 32), (100, 0, 7),
                                                    (257, 10, 0), (5000, 4, 32)])
def test_evict(cuda_device, dtype, shared, budget, n_sinks, recency):
    Hkv = 2
    c = Case([0, 1, 36, 100, 101, 1024, 2500], 24, 4, Hkv, 40, 1, dtype, cuda_device, seed=budget)
    B = len(c.lens)
    g = torch.Generator().manual_seed(budget + 1)
    w = torch.rand(B, 1 if shared else Hkv, c.L, generator=g)
    w[:, :, ::3] = 0.5   # ties
    w[:, :, 1::7] = 0.0
    w[:, :, 2::31] = -0.0
    w[:, :, 3::37] = math.nan
    w[:, :, 4::41] = -math.inf
    w[:, :, 5::43] = math.inf
    w[:, :, 6::47] = -2.5
    w[6, :, :] = 1.0     # all alike
    e = kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w.to(cuda_device), budget, n_sinks=n_sinks, recency=recency)
    assert e.seq_lens.tolist() == [min(n, budget) for n in c.lens]
    for b, n in enumerate(c.lens):
        for h in range(w.shape[1]):
            rows = evict_rows(w[b, h].tolist(), n, budget, n_sinks, recency)
            m = len(rows)
            assert e.kept[b, h].tolist() == rows + [-1] * (budget - m)
            ww = w[b, h][rows] if m else w[b, h][:0]
            assert torch.equal(e.weights[b, h, :m].cpu().view(torch.int32), ww.view(torch.int32))
            assert bool((e.weights[b, h, m:] == 0).all())
            for kv in range(Hkv) if shared else [h]:
                k, v = c.rows(b, kv)
                idx = torch.tensor(rows, device=cuda_device, dtype=torch.long)
                assert torch.equal(e.k[b, :m, kv], k[idx]) and torch.equal(e.v[b, :m, kv], v[idx])
                assert bool((e.k[b, m:, kv] == 0).all()) and bool((e.v[b, m:, kv] == 0).all())


@pytest.mark.parametrize("n", [40_000, 200_001])
def test_evict_long(cuda_device, n):
    """One long row, many equal weights at the border."""
    dev = cuda_device
    g = torch.Generator().manual_seed(n)
    w = torch.rand(1, 1, n, generator=g)
    w[0, 0, torch.rand(n, generator=g) < 0.6] = 0.25
    k = torch.randn(1, n, 1, 8, generator=g).half().to(dev)
    budget = n // 2
    e = kb.evict_cache(k, k.clone(), None, torch.tensor([n]), w.to(dev), budget)
    order = torch.sort(w[0, 0, 4:n - 32], descending=True, stable=True).indices[:budget - 36] + 4
    want = torch.cat([torch.arange(4), order, torch.arange(n - 32, n)]).sort().values
    assert torch.equal(e.kept[0, 0].cpu().long(), want)
    assert torch.equal(e.k[0, :, 0], k[0, want.to(dev), 0])


@pytest.mark.parametrize("B,n", [(30, 9001), (60, 9001), (2, 30_000), (80, 50_001)])
def test_evict_rows_and_clusters(cuda_device, B, n):
    """Rows shared by 4, 2, 8 and 1 CTAs; the last ones longer than shared memory holds."""
    dev = cuda_device
    g = torch.Generator().manual_seed(n + B)
    w = torch.rand(B, 1, n, generator=g).to(dev)
    w[:, 0, ::5] = 0.25
    k = torch.randn(B, n, 1, 8, generator=g).half().to(dev)
    lens = torch.full((B,), n, dtype=torch.int32)
    lens[1], lens[B // 2] = 17, n - 4099
    budget = n // 3
    e = kb.evict_cache(k, k, None, lens, w, budget)
    for b in range(B):
        m = int(lens[b])
        if m <= budget:
            want = torch.arange(m, device=dev)
        else:
            mid = torch.sort(w[b, 0, 4:m - 32], descending=True, stable=True).indices[:budget - 36] + 4
            want = torch.cat([torch.arange(4, device=dev), mid, torch.arange(m - 32, m, device=dev)]).sort().values
        assert torch.equal(e.kept[b, 0, :len(want)].long(), want) and bool((e.kept[b, 0, len(want):] == -1).all())
        assert torch.equal(e.k[b, :len(want), 0], k[b, want, 0]) and torch.equal(e.v[b], e.k[b])


def test_evict_into_given_memory(cuda_device):
    c = Case([60, 200, 10], 16, 4, 2, 64, 1, torch.float16, cuda_device, seed=1)
    w = torch.rand(3, 2, c.L, device=cuda_device)
    out = tuple(torch.full((3, 130, 2, 64), 9.0, dtype=torch.float16, device=cuda_device) for _ in range(2))
    e = kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 100, out=out)
    f = kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 100, capacity=130)
    assert e.k is out[0] and e.v is out[1] and torch.equal(e.kept, f.kept)
    for b, m in enumerate(f.seq_lens.tolist()):
        assert torch.equal(e.k[b, :m], f.k[b, :m]) and torch.equal(e.v[b, :m], f.v[b, :m])
        assert bool((e.k[b, m:] == 9).all()) and bool((f.v[b, m:] == 0).all()) and bool((f.k[b, m:] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_run_together(cuda_device, dtype):
    """Prompt attention and block mass, decode steps that accumulate weights, eviction, and decoding (one token and a
    tree) over the compact cache: each step against 64 bits."""
    dev = cuda_device
    g = torch.Generator().manual_seed(17)
    B, Hq, Hkv, D, N, page = 2, 8, 2, 64, 300, 16
    lens = torch.tensor([300, 177], dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(B, h, N, D, generator=g).to(dtype).to(dev) for h in (Hq, Hkv, Hkv))
    out, lse = kb.attention_b200(q, k, v, causal=True, seq_lens=lens)
    mass = kb.block_mass_b200(q, k, causal=True, seq_lens=lens, lse=lse, block_size=1, per_sequence=True)
    assert torch.allclose(mass.sum(1), (lens * Hq).float(), rtol=1e-3)
    # the prompt's keys and values go into pages, with room for new tokens
    per = 20
    table = torch.randperm(B * per, generator=g).to(torch.int32).view(B, per).to(dev)
    kc = torch.zeros(B * per, page, Hkv, D, dtype=dtype, device=dev)
    vc = torch.zeros_like(kc)

    def put(cache, rows, b, at):
        pos = torch.arange(at, at + rows.shape[0], device=dev)
        cache[table[b].long()[pos // page], pos % page] = rows

    for b in range(B):
        put(kc, k[b, :, :lens[b]].transpose(0, 1), b, 0)
        put(vc, v[b, :, :lens[b]].transpose(0, 1), b, 0)
    w = torch.zeros(B, Hkv, per * page, device=dev)
    w[:, :, :N] = (mass / Hkv)[:, None]
    before = w.clone()
    total = torch.zeros_like(w, dtype=torch.float64)
    for step in range(3):
        nk, nv = (torch.randn(B, 1, Hkv, D, generator=g).to(dtype).to(dev) for _ in range(2))
        nq = torch.randn(B, Hq, 1, D, generator=g).to(dtype).to(dev)
        for b in range(B):
            put(kc, nk[b], b, int(lens[b]))
            put(vc, nv[b], b, int(lens[b]))
        lens += 1
        _, _, w = kb.attention_cached(nq, kc, vc, table, lens, weights=w)
        for b in range(B):
            n = int(lens[b])
            pos = torch.arange(n, device=dev)
            rows = kc[table[b].long()[pos // page], pos % page]
            for h in range(Hq):
                x = nq[b, h].double() @ rows[:, h // 4].double().T / math.sqrt(D)
                total[b, h // 4, :n] += torch.softmax(x, -1)[0]
    assert torch.allclose(w.double(), before.double() + total, rtol=2e-5, atol=2e-6)
    e = kb.evict_cache(kc, vc, table, lens, w, 96, capacity=112)
    for b in range(B):
        for h in range(Hkv):
            assert e.kept[b, h].tolist() == evict_rows(w[b, h].tolist(), int(lens[b]), 96, 4, 32)
    # decoding goes on in the compact cache
    T = 7
    tree = _tree(B, T, 3, dev)
    nk, nv = (torch.randn(B, T, Hkv, D, generator=g).to(dtype).to(dev) for _ in range(2))
    nq = torch.randn(B, Hq, T, D, generator=g).to(dtype).to(dev)
    e.k[:, 96:96 + T], e.v[:, 96:96 + T] = nk, nv
    out, lse = kb.attention_cached(nq, e.k, e.v, None, e.seq_lens + T, tree_mask=tree)
    for b in range(B):
        for h in range(Hq):
            o, l, _, ot, lt, _ = softmax_rows(nq[b, h], e.k[b, :96 + T, h // 4], e.v[b, :96 + T, h // 4],
                                              cached_keep(96 + T, T, tree[b], dev), 1 / math.sqrt(D), dtype=dtype)
            check(out[b, h], o, ot, "tree out")
            check(lse[b, h], l, lt, "tree lse")


def test_design_offsets(cuda_device):
    """design_from_mass's log offsets and keep mask as the offsets of a thinned cache."""
    dev = cuda_device
    c = Case([256], 16, 4, 2, 64, 1, torch.bfloat16, dev, seed=23)
    mass = torch.rand(16, device=dev)
    d = kb.design_from_mass(mass, 256, 16, 40, seed=5, with_log_offsets=True)
    off = torch.where(d.keep, d.log_offsets.float(), -math.inf)[None]
    out, lse = kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, log_offsets=off)
    _check(c, out, lse, off=off[:, None])


def test_refusals(cuda_device):
    c = Case([40, 20], 16, 4, 2, 64, 1, torch.bfloat16, cuda_device)
    w = torch.zeros(2, 2, c.L, device=cuda_device)
    both = torch.zeros(512, device=cuda_device)
    call = lambda **kw: kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens, **kw)  # noqa: E731
    bad = [
        lambda: kb.attention_cached(c.q.cpu(), c.k, c.v, c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q.float(), c.k, c.v, c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q.double(), c.k.double(), c.v.double(), c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q[:, :3], c.k, c.v, c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q, c.k, c.v[..., :32], c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q, c.k, c.v, c.table[:1], c.seq_lens),
        lambda: kb.attention_cached(c.q, c.k, c.v, c.table.float(), c.seq_lens),
        lambda: kb.attention_cached(c.q, c.k, c.v, c.table.cpu(), c.seq_lens),
        lambda: kb.attention_cached(c.q, c.k, c.v, None, c.seq_lens),  # 9 pages for 2 sequences
        lambda: kb.attention_cached(c.q, c.k, c.v, c.table, c.seq_lens[:1]),
        lambda: kb.attention_cached(c.q.expand(2, 4, 65, 64), c.k, c.v, c.table, c.seq_lens),
        lambda: kb.attention_cached(c.q.expand(2, 4, 2, 64), c.k, c.v, c.table, c.seq_lens, weights=w),
        lambda: call(weights=w[:, :1]),
        lambda: call(weights=w.double()),
        lambda: call(weights_out=w),
        lambda: call(weights=w, weights_out=w[:, :, :10]),
        lambda: call(weights=w[:, :1].expand(2, 2, c.L)),
        lambda: call(log_offsets=torch.zeros(2, c.L + 1, device=cuda_device)),
        lambda: call(log_offsets=torch.zeros(2, c.L)),
        lambda: call(tree_mask=torch.ones(2, 2)),
        lambda: call(scale=math.nan),
        lambda: call(out=c.q),
        lambda: call(out=both.view(torch.bfloat16)[:512].view(2, 4, 1, 64), lse_out=both[200:208].view(2, 4, 1)),
        lambda: call(weights=w, lse_out=w.view(-1)[8:16].view(2, 4, 1)),
        lambda: call(workspace=torch.empty(16, dtype=torch.uint8, device=cuda_device)),
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 0),
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 35),  # sinks + recency do not fit
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 40, capacity=39),
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w[:1], 40),
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w.cpu(), 40),
        lambda: kb.evict_cache(c.k, c.v.float(), c.table, c.seq_lens, w, 40),
        lambda: kb.evict_cache(c.k, c.v, c.table, c.seq_lens, w, 16, n_sinks=1, recency=1,
                               out=(c.k[:2], c.v[:2])),
        lambda: kb.evict_cache(c.k.cpu(), c.v.cpu(), c.table, c.seq_lens, w, 40),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {i} was accepted")
