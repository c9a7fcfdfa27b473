"""KV caches in 4 bits: rows stored and read back (K.cache4_store, cache4_load), attention of token trees over them
(K.tree_attn4), and their accepted rows and copies, against plain implementations in 64 bits.

The quantisation is a function of the elements alone, so that stored codes, scales and numbers are compared for equality.

Error bounds of the attention, elementwise, over the caches' own numbers, with A = sum_j p_j |v_j| of the reference and u = half a
step (2^-8 for bf16, 2^-24 for fp32):
* the output's own rounding: u |o|;
* bf16 queries: weights are rounded to bf16 before the product with V: u A; fp32 queries and weights are sums of three bf16 numbers,
  exact (8 of their 24 bits each);
* scores: the products of bf16 numbers are exact in fp32; C D of them (C = 1 for bf16, 3 for fp32 queries) are summed, each sum off by
  2^-24 of at most S = scale max sum |q_d k_d|, twice that for fp32 queries' three sums of partial magnitudes; scale and log2 e as fp32
  numbers, the product with them and the difference from the maximum add 7 S 2^-24, the hardware exp2 2^-23; a weight is off
  by e^delta - 1 and so is the sum: 2 delta A;
* sums over C N keys, in any order: 2 (C N + 8) 2^-24 A."""
import math

import pytest
import torch

from uno_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, F32, I64 = torch.bfloat16, torch.float32, torch.int64
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _quantised(x):
    """(codes, scale bytes) of x [..., D] (64 bits, on the CPU), from the definition: the least scale with max < 7 scale, the nearest
    of the grid by distance, ties to the even code."""
    g = x.double().cpu().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    odd = ~torch.isfinite(top)
    byte = torch.full(top.shape, 252, dtype=I64)
    for b in range(251, 1, -1):                         # the least byte that fits
        byte = torch.where(top < 7 * 2.0 ** (b - 127), b, byte)
    y = g.abs() / torch.exp2(byte - 127.0)
    far = (y[..., None] - GRID).abs()
    near = far == far.amin(-1, keepdim=True)
    even = torch.where(torch.arange(8) % 2 == 0, 0, 1)
    code = torch.where(near, even, 2).argmin(-1)       # of two, the even one
    code = code + 8 * torch.signbit(g)
    code = torch.where(odd, 0, code).flatten(-2)
    byte = torch.where(odd, 255, byte).squeeze(-1)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), byte.to(torch.uint8)


def _numbers(cache):
    """What a cache's bytes stand for, fp64 on its device."""
    codes, scales = cache
    grid = torch.cat([GRID, -GRID]).to(codes.device)
    c = codes.long()
    x = grid[torch.stack((c & 15, c >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32))
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127.0))
    return (x * s[..., None]).flatten(-2)


def _cache(dev, B, nk, max_len, D, g=None, fill=0):
    """A cache of numbers like quantised normal ones; without a generator, of ``fill`` bytes."""
    if g is None:
        return K.Rows4(torch.full((B, nk, max_len, D // 2), fill, device=dev, dtype=torch.uint8),
                       torch.full((B, nk, max_len, D // 32), fill, device=dev, dtype=torch.uint8))
    return K.Rows4(torch.randint(0, 256, (B, nk, max_len, D // 2), device=dev, generator=g).to(torch.uint8),
                   torch.randint(124, 127, (B, nk, max_len, D // 32), device=dev, generator=g).to(torch.uint8))


# ---- rows in and out -----------------------------------------------------------------------------
def _rows(dtype, M, width, seed):
    """Normal elements; some groups all zero, tiny, huge, with ties, infinities or NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, width // 32, 32, generator=g)
    kind = torch.randint(0, 12, (M, width // 32, 1), generator=g)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.9] * 2)
    x = torch.where(kind == 0, x * 0, x)
    x = torch.where(kind == 1, x * 2.0 ** -124, x)
    x = torch.where(kind == 2, x.sign() * 3.3e38 * torch.rand(x.shape, generator=g), x)
    x = torch.where(kind == 3, ties * 2.0 ** torch.randint(-9, 9, kind.shape, generator=g), x)
    x = torch.where(kind == 4, x * 2.0 ** torch.randint(-30, 30, kind.shape, generator=g), x)
    one = torch.randint(0, 32, kind.shape, generator=g) == torch.arange(32)
    x = torch.where((kind == 5) & one, math.nan, x)
    x = torch.where((kind == 6) & one, math.inf, x)
    x = torch.where((kind == 7) & one, 7.0, x)
    return x.view(M, width).to(dtype)


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,nk,D", [(1, 1, 1, 64), (1, 1, 8, 128), (3, 7, 2, 64), (2, 37, 3, 128), (5, 130, 1, 128)])
def test_store_and_load(dev, dtype, B, T, nk, D):
    """Rows at each sequence's start; rows before 0 and past the end do not exist; the cache's other rows stay as they were."""
    print(f"[cache4] {dtype} B={B} T={T} nk={nk} D={D}", flush=True)
    max_len = 2 * T + 3
    starts = torch.tensor([[3, 0, T + 3, max_len - T // 2, -(T // 2)][b] for b in range(B)])
    rows = [_rows(dtype, B * T, nk * D, 1).to(dev), _rows(dtype, B * T, (nk + 2) * D, 2).to(dev)[:, 2 * D:]]
    caches = [_cache(dev, B, nk, max_len, D, fill=0x5a + i) for i in range(2)]
    want = [[t.clone().cpu() for t in c] for c in caches]
    K.cache4_store(rows, caches, starts.to(dev))
    read = [torch.zeros(B * T, nk * D, dtype=torch.float64) for _ in rows]
    for x, w, r in zip(rows, want, read):
        codes, scales = _quantised(x.view(B, T, nk, D))
        for b in range(B):
            for t in range(T):
                at = int(starts[b]) + t
                if 0 <= at < max_len:
                    w[0][b, :, at], w[1][b, :, at] = codes[b, t], scales[b, t]
                    r[b * T + t] = _numbers((codes[b, t], scales[b, t])).reshape(-1)
    for c, w in zip(caches, want):
        assert torch.equal(c.scales.cpu(), w[1]) and torch.equal(c.codes.cpu(), w[0])
    for out in (BF, F32):
        for got, r in zip(K.cache4_load(caches, starts.to(dev), T, dtype=out), read):
            assert got.dtype == out and _same(got.double().cpu(), r)


def test_a_row_reads_back_near_itself(dev):
    """Finite rows in range: an element is off by at most half a step of its group, which is a seventh of the largest magnitude
    (between 3.5 and 7 scales, where numbers are at most two scales apart, the topmost one scale short)."""
    x = torch.randn(64, 256, device=dev)
    cache = _cache(dev, 1, 2, 64, 128)
    zero = torch.zeros(1, device=dev, dtype=I64)
    K.cache4_store([x], [cache], zero)
    y = K.cache4_load([cache], zero, 64, dtype=F32)[0]
    top = x.view(-1, 32).abs().amax(1, keepdim=True)
    assert bool(((x - y).view(-1, 32).abs() <= top / 3.5 * 1.0001).all())
    again = _cache(dev, 1, 2, 64, 128)
    K.cache4_store([y.bfloat16()], [again], zero)       # numbers of a cache are stored as they are
    assert torch.equal(K.cache4_load([again], zero, 64, dtype=F32)[0], y)


def test_many_tensors_and_nothing_to_do(dev):
    """More tensors than one launch takes; no rows; no sequences."""
    g = torch.Generator(device=dev).manual_seed(0)
    rows = [torch.randn(6, 64, device=dev, generator=g) for _ in range(70)]
    caches = [_cache(dev, 2, 1, 5, 64) for _ in rows]
    starts = torch.tensor([1, 2], device=dev)
    K.cache4_store(rows, caches, starts)
    for x, c, y in zip(rows, caches, K.cache4_load(caches, starts, 3, dtype=F32)):
        codes, scales = _quantised(x.view(2, 3, 64))
        assert torch.equal(c.codes[0, 0, 1:4].cpu(), codes[0]) and torch.equal(c.scales[1, 0, 2:5].cpu(), scales[1])
        assert torch.equal(y.double(), _numbers((codes, scales)).view(6, 64).to(dev))
    before = caches[0].codes.clone()
    K.cache4_store([torch.zeros(0, 64, device=dev)], caches[:1], starts)
    assert torch.equal(caches[0].codes, before) and K.cache4_load(caches[:1], starts, 0)[0].shape == (0, 64)
    empty = _cache(dev, 0, 1, 5, 64)
    K.cache4_store([torch.zeros(0, 64, device=dev)], [empty], starts[:0])
    assert K.cache4_load([empty], starts[:0], 3)[0].shape == (0, 64)


def test_rows_past_every_32_bit_offset(dev):
    """Codes of more than 2^32 bytes: a row in the last slot."""
    B, nk, max_len, D = 2, 9, 4_000_037, 128
    cache = _cache(dev, B, nk, max_len, D)
    assert cache.codes.numel() > 2 ** 32
    starts = torch.tensor([5, max_len - 2], device=dev)
    x = torch.randn(B * 2, nk * D, device=dev)
    K.cache4_store([x], [cache], starts)
    y = K.cache4_load([cache], starts, 2, dtype=F32)[0]
    codes, scales = _quantised(x.view(B * 2, nk, D))
    assert torch.equal(y.double(), _numbers((codes, scales)).view(B * 2, -1).to(dev))
    assert torch.equal(cache.codes[1, -1, -2:].cpu(), codes[2:, -1]) and int(cache.codes[0, :, 7:].count_nonzero()) == 0
    # and attention over it: two nodes at the end of the last slot
    q = torch.randn(B, nk * D, device=dev).bfloat16()
    lengths, parents = torch.tensor([1000, max_len - 1], device=dev), torch.tensor([[-1]] * B, device=dev, dtype=torch.int32)
    g = torch.Generator(device=dev).manual_seed(1)
    last = K.Rows4(cache.codes[:, -1:], cache.scales[:, -1:])
    last.codes.copy_(torch.randint(0, 256, last.codes.shape, device=dev, generator=g))
    last.scales.copy_(torch.randint(124, 127, last.scales.shape, device=dev, generator=g))
    out = K.tree_attn4(q, cache, cache, lengths, parents)
    part = K.Rows4(*(t.contiguous() for t in last))
    _check(out[:, -D:], _reference(q[:, -D:], part, part, lengths, parents.cpu(), D ** -0.5), BF)


# ---- attention -----------------------------------------------------------------------------------
def _parents(B, T, seed, pad=0):
    """Random trees with several roots; the last ``pad`` nodes of odd trees are padding."""
    g = torch.Generator().manual_seed(seed)
    p = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for t in range(1, T):
            p[b, t] = int(torch.randint(-1, t, (1,), generator=g))
        if pad and b % 2:
            p[b, T - pad:] = -2
    return p


def _visible(parents):
    """[B, T, T] bool by walking every chain."""
    B, T = parents.shape
    out = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            a = t
            while 0 <= a and parents[b, a] >= -1:
                out[b, t, a] = True
                p = int(parents[b, a])
                a = p if p < a else -1
    return out


def _reference(q, k4, v4, lengths, parents, scale):
    """(o, A, bound on everything but the roundings to bf16) in 64 bits."""
    B, nk, max_len = k4.codes.shape[:3]
    D = 2 * k4.codes.shape[3]
    T = parents.shape[1]
    rep = q.shape[1] // (nk * D)
    C = 3 if q.dtype == F32 else 1
    vis = _visible(parents).to(q.device)
    o = torch.zeros(B, T, nk, rep, D, device=q.device, dtype=torch.float64)
    A, err = torch.zeros_like(o), torch.zeros(B, T, nk, rep, 1, device=q.device, dtype=torch.float64)
    qs = q.view(B, T, nk, rep, D).double() if q.is_contiguous() else q.reshape(B, T, nk, rep, D).double()
    for b in range(B):
        n = min(max(int(lengths[b]), 0), max_len)
        end = min(n + T, max_len)
        seen = torch.ones(T, end, device=q.device, dtype=torch.bool)
        seen[:, n:] = vis[b, :, :end - n]
        seen &= (parents[b] >= -1).to(q.device)[:, None]
        for h in range(nk):
            kd, vd = (_numbers((c.codes[b, h, :end], c.scales[b, h, :end])) for c in (k4, v4))
            vd = torch.where(seen.any(0)[:, None], vd, 0.0)
            for r in range(rep):
                s = torch.where(seen, qs[b, :, h, r] @ kd.T * scale, -math.inf)
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                total = p.sum(1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                o[b, :, h, r], A[b, :, h, r] = p @ vd, p @ vd.abs()
                mag = ((qs[b, :, h, r].abs() @ kd.abs().T) * abs(scale)).where(seen, 0.0).amax(1)
                delta = 2.0 ** -24 * (((2 if C == 3 else 1) * C * D + 10) * mag + 2)
                err[b, :, h, r, 0] = 2 * delta + 2 * (C * end + 8) * 2.0 ** -24
    shape = (B * T, nk * rep * D)
    return o.view(shape), A.view(shape), err.expand_as(o).reshape(shape)


def _check(out, ref, dtype):
    o, A, err = ref
    u = HALF[dtype]
    bound = u * o.abs() + (u if dtype == BF else 0) * A * 1.01 + err * A + 1e-30
    bad = (out.double() - o).abs() - bound
    assert bool((bad <= 0).all()), (bad.max().item(), int((bad > 0).sum()))


def _case(dev, dtype, B, T, heads, lengths, room, pad=0, seed=0):
    nq, nk, D = heads
    g = torch.Generator(device=dev).manual_seed(seed + T)
    max_len = max(lengths) + T + room
    q = torch.randn(B * T, nq * D, device=dev, generator=g).to(dtype)
    return q, _cache(dev, B, nk, max_len, D, g), _cache(dev, B, nk, max_len, D, g), torch.tensor(lengths, device=dev), \
        _parents(B, T, seed, pad)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 2, 128), (3, 3, 128), (16, 1, 64)])
@pytest.mark.parametrize("T,lengths,pad", [(1, [0, 1, 700], 0), (2, [31, 32, 33], 1), (7, [1000, 3, 0], 2),
                                           (16, [127, 128, 2049], 5), (37, [255, 90, 513], 9)])
def test_attention(dev, dtype, heads, T, lengths, pad):
    print(f"[attn4] {dtype} heads={heads} T={T} lengths={lengths}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 3, T, heads, lengths, room=5, pad=pad)
    out = K.tree_attn4(q, k, v, n, parents.to(dev))
    _check(out, _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)
    assert torch.equal(out, K.tree_attn4(q, k, v, n, parents.to(dev)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(64, (8, 2, 128)), (100, (4, 4, 64)), (255, (2, 1, 128)), (256, (4, 2, 64)), (200, (4, 2, 128))])
def test_wide_trees(dev, dtype, T, heads):
    """Several row tiles, trees of up to 256 nodes, a chain as deep as the tree."""
    print(f"[attn4 wide] {dtype} T={T}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 2, T, heads, [300, 0], room=0, pad=3)
    parents[0] = torch.arange(T, dtype=torch.int32) - 1
    out = K.tree_attn4(q, k, v, n, parents.to(dev), scale=0.2)
    _check(out, _reference(q, k, v, n, parents, 0.2), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(1, (8, 2, 128)), (9, (4, 2, 64)), (30, (8, 2, 128)), (70, (8, 2, 128)), (70, (8, 2, 64))])
def test_long_caches(dev, dtype, T, heads):
    """Many key ranges, of sequences of very different lengths."""
    print(f"[attn4 long] {dtype} T={T} heads={heads}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 3, T, heads, [20011, 5003, 77], room=0, pad=min(2, T // 2))
    _check(K.tree_attn4(q, k, v, n, parents.to(dev)), _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)


@pytest.mark.parametrize("T,heads", [(1, (8, 4, 128)), (9, (16, 4, 64)), (30, (16, 4, 128)), (60, (8, 4, 128))])
def test_caches_larger_than_the_memory_side_cache(dev, T, heads):
    """0.5 GB of keys and values in two sequences, the last head's outputs compared."""
    nq, nk, D = heads
    rows = 2 ** 29 // (2 * 2 * nk * (D // 2 + D // 32))
    q, k, v, n, parents = _case(dev, BF, 2, T, heads, [rows - 1000, rows - 77], room=0)
    out = K.tree_attn4(q, k, v, n, parents.to(dev)).view(2 * T, nk, -1)
    last = q.view(2 * T, nk, -1)[:, -1].contiguous()
    part = [K.Rows4(*(t[:, -1:].contiguous() for t in c)) for c in (k, v)]
    _check(out[:, -1], _reference(last, *part, n, parents, D ** -0.5), BF)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_shared_tree_and_output(dev, dtype):
    """Padded query rows, one tree for all sequences, an output with a row stride whose other columns stay as they were."""
    B, T, nq, nk, D = 3, 12, 6, 2, 64
    g = torch.Generator(device=dev).manual_seed(3)
    qw = torch.randn(B * T, nq * D + 64, device=dev, generator=g).to(dtype)
    k, v = (_cache(dev, B, nk, 400, D, g) for _ in "kv")
    n = torch.tensor([300, 388, 17], device=dev)
    parents = _parents(1, T, 5)
    out = torch.full((B * T, nq * D + 32), 7.0, device=dev, dtype=dtype)
    K.tree_attn4(qw[:, :nq * D], k, v, n, parents[0].to(dev), out=out[:, :nq * D])
    _check(out[:, :nq * D], _reference(qw[:, :nq * D], k, v, n, parents.expand(B, T), D ** -0.5), dtype)
    assert bool((out[:, nq * D:] == 7).all())
    same = K.tree_attn4(qw[:, :nq * D].contiguous(), k, v, n, parents.expand(B, T).to(dev))
    assert torch.equal(same, out[:, :nq * D])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_past_the_cache_and_odd_parents(dev, dtype):
    """Nodes whose row would lie at or past max_len do not exist as keys; lengths outside the cache are clamped; parents
    that are no earlier node, or padding, end the chain."""
    B, T, nq, nk, D = 5, 9, 4, 2, 64
    g = torch.Generator(device=dev).manual_seed(4)
    q = torch.randn(B * T, nq * D, device=dev, generator=g).to(dtype)
    k, v = (_cache(dev, B, nk, 64, D, g) for _ in "kv")
    n = torch.tensor([60, 64, 99, -4, 10], device=dev)
    parents = _parents(B, T, 6)
    parents[4] = torch.tensor([0, 0, 7, 2, -2, 4, 1000, 3, 6], dtype=torch.int32)
    _check(K.tree_attn4(q, k, v, n, parents.to(dev)), _reference(q, k, v, n, parents, D ** -0.5), dtype)


@pytest.mark.parametrize("dtype,heads,T", [(BF, (8, 2, 64), 4), (BF, (8, 2, 64), 15), (BF, (8, 2, 128), 16), (BF, (8, 2, 64), 30),
                                           (BF, (8, 2, 128), 25), (BF, (8, 2, 64), 70), (BF, (8, 2, 128), 70), (BF, (2, 2, 128), 256),
                                           (F32, (4, 1, 128), 4), (F32, (4, 1, 64), 41), (F32, (2, 2, 128), 200)])
def test_masked_rows_in_every_kernel(dev, dtype, heads, T):
    """At every number of query rows, over several key ranges, one and none committed: what unseen rows hold (any bytes, NaN and
    scales too large for numbers among them) changes nothing; a node's NaN reaches those that see it and no other."""
    print(f"[attn4 masked] {dtype} heads={heads} T={T}", flush=True)
    nq, nk, D = heads
    B, lengths = 3, [1500, 33, 0]
    q, k, v, n, parents = _case(dev, dtype, B, T, heads, lengths, room=300, pad=1, seed=8)
    vis = _visible(parents)
    clean = K.tree_attn4(q, k, v, n, parents.to(dev)).view(B, T, nq, D)
    _check(clean.view(B * T, -1), _reference(q, k, v, n, parents, D ** -0.5), dtype)
    whole, part = T // 3, T // 2                # a node whose key has a NaN, one with NaN in a part of its value
    for b, m in enumerate(lengths):
        k.scales[b, :, m + T:], v.scales[b, :, m + T:] = 255, 254
        k.scales[b, :, m + T + 3], v.scales[b, :, m + T + 3] = 253, 0
        if parents[b, T - 1] < -1:
            k.scales[b, :, m + T - 1], v.scales[b, :, m + T - 1] = 254, 255
        k.scales[b, :, m + whole, -1] = 255
        v.scales[b, :, m + part, 0] = 255
    out = K.tree_attn4(q, k, v, n, parents.to(dev)).view(B, T, nq, D)
    for b in range(B):
        for t in range(T):
            if parents[b, t] < -1:
                assert not out[b, t].any()
            elif vis[b, t, whole]:
                assert bool(out[b, t].isnan().all()), (b, t)
            elif vis[b, t, part]:
                assert bool(out[b, t, :, :32].isnan().all()), (b, t)
                assert torch.equal(out[b, t, :, 32:], clean[b, t, :, 32:]), (b, t)
            else:
                assert torch.equal(out[b, t], clean[b, t]), (b, t)


@pytest.mark.parametrize("dtype,heads,T", [(BF, (8, 2, 64), 4), (BF, (8, 2, 128), 30), (BF, (8, 2, 128), 70), (F32, (4, 1, 128), 4),
                                           (F32, (4, 1, 64), 41)])
def test_nan_among_committed_rows(dev, dtype, heads, T):
    """A NaN in a committed value reaches its 32 columns of every row of that head; one in a key every column."""
    nq, nk, D = heads
    q, k, v, n, parents = _case(dev, dtype, 2, T, heads, [700, 40], room=3, seed=2)
    clean = K.tree_attn4(q, k, v, n, parents.to(dev)).view(2, T, nk, -1, D)
    v.scales[0, 0, 123, 1] = 255
    k.scales[1, nk - 1, 39, 0] = 255
    out = K.tree_attn4(q, k, v, n, parents.to(dev)).view(2, T, nk, -1, D)
    assert bool(out[0, :, 0, :, 32:64].isnan().all()) and bool(out[1, :, nk - 1].isnan().all())
    assert torch.equal(out[0, :, 0, :, :32], clean[0, :, 0, :, :32]) and torch.equal(out[0, :, 0, :, 64:], clean[0, :, 0, :, 64:])
    if nk > 1:
        assert torch.equal(out[0, :, 1:], clean[0, :, 1:]) and torch.equal(out[1, :, :nk - 1], clean[1, :, :nk - 1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(4, (4, 2, 64)), (20, (4, 2, 128)), (90, (4, 2, 128))])
@pytest.mark.parametrize("B", [70, 200])
def test_many_sequences(dev, dtype, B, T, heads):
    """More sequences than a wave has lanes, of very different lengths: one long, most short, some empty."""
    print(f"[attn4 many] {dtype} B={B} T={T} heads={heads}", flush=True)
    lengths = [(37 * b) % 90 for b in range(B)]
    lengths[B - 3], lengths[5], lengths[66] = 2900, 0, 1100
    q, k, v, n, parents = _case(dev, dtype, B, T, heads, lengths, room=1, pad=2)
    _check(K.tree_attn4(q, k, v, n, parents.to(dev)), _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(4, (8, 2, 64)), (30, (8, 2, 128)), (70, (4, 2, 64)), (256, (2, 1, 128))])
@pytest.mark.parametrize("scale", [-0.2, 0.0, -3.0])
def test_scales_that_are_not_positive(dev, dtype, T, heads, scale):
    print(f"[attn4 scale] {dtype} T={T} heads={heads} scale={scale}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 3, T, heads, [1500, 33, 0], room=300, pad=1, seed=13)
    out = K.tree_attn4(q, k, v, n, parents.to(dev), scale=scale)
    _check(out, _reference(q, k, v, n, parents, scale), dtype)


def test_numbers_far_apart(dev):
    """Keys and values over 60 binades, the largest last."""
    B, T, nk, D, n = 1, 4, 1, 64, 900
    g = torch.Generator(device=dev).manual_seed(9)
    k, v = (_cache(dev, B, nk, n + T, D, g) for _ in "kv")
    k.scales.copy_((95 + torch.arange(n + T, device=dev) * 32 // (n + T))[:, None].expand(n + T, 2))
    v.scales.copy_(torch.randint(97, 157, v.scales.shape, device=dev, generator=g))
    q = torch.randn(B * T, D, device=dev, generator=g) * 20
    parents, lengths = _parents(B, T, 1), torch.tensor([n], device=dev)
    for dtype in (F32, BF):
        out = K.tree_attn4(q.to(dtype), k, v, lengths, parents.to(dev))
        _check(out, _reference(q.to(dtype), k, v, lengths, parents, D ** -0.5), dtype)


@pytest.mark.parametrize("empty", ["B", "T"])
def test_nothing_to_do(dev, empty):
    B, T = (0, 4) if empty == "B" else (3, 0)
    k = _cache(dev, B, 2, 16, 64)
    out = K.tree_attn4(torch.zeros(B * T, 256, device=dev), k, k, torch.zeros(B, device=dev, dtype=I64),
                       torch.zeros(B, T, device=dev, dtype=torch.int32))
    assert out.shape == (0, 256)


# ---- a cache's life --------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [1, 5, 256])
def test_accepted_rows_and_copies(dev, D, P):
    """cache_keep and cache_copy move codes and scales (rows of 2 and 4 bytes) alike."""
    B, nk, max_len = 6, 3, 300
    g = torch.Generator(device=dev).manual_seed(P)
    cache = _cache(dev, B, nk, max_len, D, g)
    n = torch.tensor([0, 20, 44, 290, 300, 7])
    nodes = torch.randint(-2, 260, (B, P), generator=torch.Generator().manual_seed(P))
    counts = torch.tensor([P, P, P, P, P, max(0, P - 2)])
    want = [t.clone() for t in cache]
    for t, w in zip(cache, want):
        for b in range(B):
            for i in range(int(counts[b])):
                src, dst = int(n[b]) + int(nodes[b, i]), int(n[b]) + i
                if int(nodes[b, i]) >= 0 and src < max_len and dst < max_len:
                    w[b, :, dst] = t[b, :, src]
    for t in cache:
        K.cache_keep([t], n.to(dev), nodes.to(dev), counts.to(dev))
    assert all(torch.equal(t, w) for t, w in zip(cache, want))
    other, m = _cache(dev, 4, nk, 41, D, g), torch.arange(4, device=dev)
    want, length = [t.clone() for t in other], m.clone()
    for a, b in [(1, 0), (2, 3), (0, 1)]:
        rows = min(int(n[a]), 41)
        length[b] = rows
        for t, w in zip(cache, want):
            w[b, :, :rows] = t[a, :, :rows]
    for s, d in zip(cache, other):
        K.cache_copy([s], [d], n.to(dev), m, [(1, 0), (2, 3), (0, 1)])
    assert all(torch.equal(t, w) for t, w in zip(other, want)) and torch.equal(m, length)


def test_rows_of_eight_bytes_move_too(dev):
    c = torch.arange(2 * 3 * 9 * 8, device=dev).to(torch.uint8).view(2, 3, 9, 8)
    want = c.clone()
    want[:, :, 2], want[:, :, 3] = c[:, :, 3], c[:, :, 6]
    K.cache_keep([c], torch.tensor([2, 2], device=dev), torch.tensor([[1, 4]] * 2, device=dev), torch.tensor([2, 2], device=dev))
    assert torch.equal(c, want)
    d = torch.zeros_like(c)
    K.cache_copy([c], [d], torch.tensor([9, 5], device=dev), torch.zeros(2, device=dev, dtype=I64), [(1, 0)])
    assert torch.equal(d[0, :, :5], c[1, :, :5]) and not d[0, :, 5:].any() and not d[1].any()


def test_captured_and_replayed(dev):
    """Rows stored, attended over and read back in one graph, replayed over changing rows, lengths and trees with eager work
    between the replays, each against the eager calls on another stream."""
    B, T, nq, nk, D, max_len = 2, 10, 8, 2, 128, 1500
    q, k, v, n, parents = _case(dev, BF, B, T, (nq, nk, D), [1200, 700], room=290)
    parents = parents.to(dev)
    rows = [torch.randn(B * T, nk * D, device=dev).bfloat16() for _ in "kv"]

    def work():
        K.cache4_store(rows, [k, v], n)
        return [K.tree_attn4(q, k, v, n, parents), *K.cache4_load([k, v], n, T)]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    stream = torch.cuda.Stream()
    for i in range(4):
        n.sub_(i * 97)
        parents.copy_(_parents(B, T, 20 + i))
        for r in rows:
            r.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for c in (k, v):                                # what the graph stored is stored again
            for b in range(B):
                m = int(n[b])
                c.codes[b, :, m:m + T] = 0
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            eager = work()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        torch.randn(4096, device=dev).sum().item()


def test_two_streams_at_once(dev):
    """Calls of one cache on several streams, each with its own workspace."""
    g = torch.Generator(device=dev).manual_seed(23)
    B, T, nq, nk, D, n = 3, 20, 8, 2, 128, 2000
    k, v = ((torch.randn(B * n, nk * D, device=dev, generator=g)).to(BF) for _ in range(2))
    caches = [K.Rows4(torch.zeros(B, nk, n, D // 2, device=dev, dtype=torch.uint8), torch.zeros(B, nk, n, D // 32, device=dev, dtype=torch.uint8))
              for _ in range(2)]
    K.cache4_store((k, v), caches, torch.zeros(B, device=dev, dtype=torch.int64))
    lengths = torch.tensor([1900, 700, 0], device=dev)
    parents = torch.tensor([-1] + [i // 2 for i in range(T - 1)], device=dev, dtype=torch.int32)
    q = torch.randn(B * T, nq * D, device=dev, generator=g).to(BF)
    want, rows = K.tree_attn4(q, *caches, lengths, parents), K.cache4_load(caches, lengths, T)
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in [torch.cuda.Stream() for _ in range(3)]:
            with torch.cuda.stream(s):
                got.append((K.tree_attn4(q, *caches, lengths, parents), *K.cache4_load(caches, lengths, T)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, (want, *rows)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(12, (8, 2, 128)), (70, (4, 2, 64))])
def test_a_query_without_numbers_leaves_the_others(dev, dtype, T, heads):
    """A row of NaN or infinities among the queries: its own output is NaN, every other row keeps its bits."""
    nq, nk, D = heads
    g = torch.Generator(device=dev).manual_seed(29)
    B, n = 2, 300 + T
    rows = [torch.randn(B * n, nk * D, device=dev, generator=g).to(dtype) for _ in range(2)]
    caches = [K.Rows4(torch.zeros(B, nk, n, D // 2, device=dev, dtype=torch.uint8), torch.zeros(B, nk, n, D // 32, device=dev, dtype=torch.uint8))
              for _ in range(2)]
    K.cache4_store(rows, caches, torch.zeros(B, device=dev, dtype=torch.int64))
    lengths = torch.tensor([300, 17], device=dev)
    parents = torch.tensor([-1] + [i // 3 for i in range(T - 1)], device=dev, dtype=torch.int32)
    q = torch.randn(B * T, nq * D, device=dev, generator=g).to(dtype)
    want = K.tree_attn4(q, *caches, lengths, parents)
    for bad in (math.nan, math.inf):
        p = q.clone()
        p[3, :D], p[T + 5, D:2 * D] = bad, bad
        got = K.tree_attn4(p, *caches, lengths, parents)
        assert got[3, :D].isnan().all() and got[T + 5, D:2 * D].isnan().all()
        got[3, :D], got[T + 5, D:2 * D] = want[3, :D], want[T + 5, D:2 * D]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_caches_of_no_rows(dev, dtype):
    """A cache without rows takes none, and all of its rows read as zeros."""
    B, nk, D, T = 2, 3, 64, 5
    caches = [_cache(dev, B, nk, 0, D) for _ in "kv"]
    starts = torch.tensor([0, -2], device=dev)
    K.cache4_store([torch.ones(B * T, nk * D, device=dev, dtype=dtype)] * 2, caches, starts)
    for rows in K.cache4_load(caches, starts, T, dtype=dtype):
        assert rows.shape == (B * T, nk * D) and rows.dtype == dtype and not rows.any()
