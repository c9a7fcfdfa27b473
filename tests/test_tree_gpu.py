"""Trees of drafted tokens over a KV cache: attention (K.tree_attn), node depths, keeping the accepted path
(K.cache_keep) and copying sequences between slots (K.cache_copy), against plain implementations in 64 bits.

Error bounds of the attention, elementwise, with A = sum_j p_j |v_j| of the reference and u = half a step (2^-8 for
bf16, 2^-24 for fp32):
* the output's own rounding: u |o|;
* bf16 weights are rounded before the product with V: u A (fp32: none);
* scores: D fp32 products and sums off by at most (D + 3) 2^-24 S, S = scale max sum |q_d k_d| >= |s|; scale and log2 e as
  fp32 numbers, the product with them and the difference from the maximum add 7 S 2^-24, the hardware exp2 2^-23; a
  weight is off by e^delta - 1 and so is the sum: 2 delta A;
* sums over N keys, in any order: 2 (N + 8) 2^-24 A.
"""
import math

import pytest
import torch

from uno_amd import kernels as K

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


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


def _reference(q, k, v, lengths, parents, scale):
    """(o, A, bound on 2 delta) in 64 bits, per sequence and K/V head."""
    B, nk, max_len, D = k.shape
    T = parents.shape[1]
    rep = q.shape[1] // (nk * D)
    vis = _visible(parents).to(q.device)
    o = torch.zeros(B, T, nk, rep, D, device=q.device, dtype=torch.float64)
    A, err = torch.zeros_like(o), torch.zeros(B, T, nk, rep, 1, device=q.device, dtype=torch.float64)
    qs = q.view(B, T, nk, rep, D).double()
    for b in range(B):
        n = min(max(int(lengths[b]), 0), max_len)
        end = min(n + T, max_len)
        seen = torch.ones(T, end, device=q.device, dtype=torch.bool)
        seen[:, n:] = vis[b, :, :end - n]
        real = (parents[b] >= -1).to(q.device)
        for h in range(nk):
            kd, vd = k[b, h, :end].double(), v[b, h, :end].double()
            for r in range(rep):
                s = qs[b, :, h, r] @ kd.T * scale
                s = torch.where(seen, s, -math.inf)
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
                total = p.sum(1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                p[~real] = 0
                # a masked key adds nothing, whatever its row holds
                vm = torch.where(seen.any(0)[:, None], vd, torch.zeros_like(vd))
                o[b, :, h, r], A[b, :, h, r] = p @ vm, p @ vm.abs()
                mag = ((qs[b, :, h, r].abs() @ kd.abs().T) * scale).where(seen, torch.zeros_like(s)).amax(1)
                err[b, :, h, r, 0] = 2 * 2.0 ** -24 * ((D + 10) * mag + 2) + 2 * (end + 8) * 2.0 ** -24
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
    k, v = (torch.randn(B, nk, max_len, D, device=dev, generator=g).to(dtype) for _ in "kv")
    parents = _parents(B, T, seed, pad)
    return q, k, v, torch.tensor(lengths, device=dev), parents


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 2, 128), (3, 3, 128), (16, 1, 64)])
@pytest.mark.parametrize("T,lengths,pad", [(1, [0, 1, 700], 0), (2, [31, 32, 33], 1), (7, [1000, 3, 0], 2),
                                           (16, [127, 128, 2049], 5), (37, [255, 90, 513], 9)])
def test_tree_attention(dev, dtype, heads, T, lengths, pad):
    print(f"[tree] {dtype} heads={heads} T={T} lengths={lengths}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 3, T, heads, lengths, room=5, pad=pad)
    out = K.tree_attn(q, k, v, n, parents.to(dev))
    _check(out, _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)
    assert torch.equal(out, K.tree_attn(q, k, v, n, parents.to(dev)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(64, (8, 2, 128)), (100, (4, 4, 64)), (255, (2, 1, 128)), (256, (4, 2, 64))])
def test_wide_trees(dev, dtype, T, heads):
    """Several row tiles, trees of up to 256 nodes, a chain as deep as the tree."""
    print(f"[tree wide] {dtype} T={T}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 2, T, heads, [300, 0], room=0, pad=3)
    parents[0] = torch.arange(T, dtype=torch.int32) - 1
    out = K.tree_attn(q, k, v, n, parents.to(dev), scale=0.2)
    _check(out, _reference(q, k, v, n, parents, 0.2), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_shared_tree_and_output(dev, dtype):
    """Cache rows in another order ([B, max_len, nk, D] in memory), padded query rows, one tree for all sequences, an
    output with a row stride whose other columns stay as they were."""
    B, T, nq, nk, D, max_len = 3, 12, 6, 2, 64, 400
    g = torch.Generator(device=dev).manual_seed(3)
    qw = torch.randn(B * T, nq * D + 64, device=dev, generator=g).to(dtype)
    k, v = (torch.randn(B, max_len, nk, D, device=dev, generator=g).to(dtype).transpose(1, 2) for _ in "kv")
    n = torch.tensor([300, 388, 17], device=dev)
    parents = _parents(1, T, 5)
    out = torch.full((B * T, nq * D + 32), 7.0, device=dev, dtype=dtype)
    K.tree_attn(qw[:, :nq * D], k, v, n, parents[0].to(dev), out=out[:, :nq * D])
    _check(out[:, :nq * D], _reference(qw[:, :nq * D], k, v, n, parents.expand(B, T), D ** -0.5), dtype)
    assert bool((out[:, nq * D:] == 7).all())
    same = K.tree_attn(qw[:, :nq * D].contiguous(), k.contiguous(), v.contiguous(), n, parents.expand(B, T).to(dev))
    assert torch.equal(same, out[:, :nq * D])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_past_the_cache_and_odd_parents(dev, dtype):
    """Nodes whose row would lie at or past max_len do not exist as keys; lengths outside the cache are clamped; parents
    that are no earlier node, or padding, end the chain."""
    B, T, nq, nk, D, max_len = 5, 9, 4, 2, 64, 64
    g = torch.Generator(device=dev).manual_seed(4)
    q = torch.randn(B * T, nq * D, device=dev, generator=g).to(dtype)
    k, v = (torch.randn(B, nk, max_len, D, device=dev, generator=g).to(dtype) for _ in "kv")
    n = torch.tensor([60, 64, 99, -4, 10], device=dev)
    parents = _parents(B, T, 6)
    parents[4] = torch.tensor([0, 0, 7, 2, -2, 4, 1000, 3, 6], dtype=torch.int32)
    out = K.tree_attn(q, k, v, n, parents.to(dev))
    _check(out, _reference(q, k, v, n, parents, D ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_rows_may_hold_anything(dev, dtype, D):
    """NaN and infinities in rows behind the tree, in padding rows, and in branches that a node does not see change
    no output that does not see them; a node that sees one gets what the formula gives."""
    B, T, nq, nk, max_len = 2, 6, 4, 2, 200
    q, k, v, n, _ = _case(dev, dtype, B, T, (nq, nk, D), [150, 33], room=44)
    parents = torch.tensor([[-1, 0, 0, 1, 2, -2], [-1, -1, 1, 2, -2, -2]], dtype=torch.int32)
    clean = K.tree_attn(q, k, v, n, parents.to(dev)).view(B, T, -1)
    for b, length in enumerate([150, 33]):
        k[b, :, length + T:] = math.nan
        v[b, :, length + T:] = math.nan
        k[b, :, length + 5] = math.inf
        v[b, :, length + 5] = -math.inf
    assert torch.equal(K.tree_attn(q, k, v, n, parents.to(dev)).view(B, T, -1), clean)
    v[0, :, 150 + 2, 3] = math.nan              # node 2 of the first tree: seen by 2 and 4
    v[0, :, 150 + 2, 7] = math.inf
    k[1, :, 33 + 0] = math.nan                  # node 0 of the second: seen by itself only
    out = K.tree_attn(q, k, v, n, parents.to(dev)).view(B, T, nq, D)
    clean = clean.view(B, T, nq, D)
    for b, t in ((0, 0), (0, 1), (0, 3), (0, 5), (1, 1), (1, 2), (1, 3), (1, 4)):
        assert torch.equal(out[b, t], clean[b, t]), (b, t)
    for t in (2, 4):
        assert bool(out[0, t, :, 3].isnan().all()) and bool((out[0, t, :, 7] == math.inf).all())
        rest = [d for d in range(D) if d not in (3, 7)]
        assert torch.equal(out[0, t][:, rest], clean[0, t][:, rest])
    assert bool(out[1, 0].isnan().all())


@pytest.mark.parametrize("dtype,heads,T", [(BF, (8, 2, 64), 4), (BF, (8, 2, 64), 15), (BF, (8, 2, 128), 16), (BF, (8, 2, 64), 30),
                                           (BF, (8, 2, 128), 25), (BF, (8, 2, 64), 70), (BF, (8, 2, 128), 70), (BF, (2, 2, 128), 256),
                                           (F32, (4, 1, 128), 4), (F32, (4, 1, 64), 41), (F32, (2, 2, 128), 200)])
def test_masked_rows_in_every_kernel(dev, dtype, heads, T):
    """The same at every number of query rows (with nodes over several key tiles), over several key ranges, one and none
    committed: a node's NaN reaches those that see it and no other."""
    print(f"[tree masked] {dtype} heads={heads} T={T}", flush=True)
    nq, nk, D = heads
    B, lengths = 3, [1500, 33, 0]
    q, k, v, n, parents = _case(dev, dtype, B, T, heads, lengths, room=300, pad=1, seed=8)
    vis = _visible(parents)
    clean = K.tree_attn(q, k, v, n, parents.to(dev)).view(B, T, nq, D)
    _check(clean.view(B * T, -1), _reference(q, k, v, n, parents, D ** -0.5), dtype)
    whole, part = T // 3, T // 2                # a node whose key is NaN, one with odd elements in its value
    for b, m in enumerate(lengths):
        k[b, :, m + T:], v[b, :, m + T:] = math.nan, -math.inf
        if parents[b, T - 1] < -1:
            k[b, :, m + T - 1], v[b, :, m + T - 1] = math.inf, math.nan
        k[b, :, m + whole] = math.nan
        v[b, :, m + part, 5] = math.nan
        v[b, :, m + part, D - 1] = math.inf
    out = K.tree_attn(q, k, v, n, parents.to(dev)).view(B, T, nq, D)
    rest = [d for d in range(D) if d not in (5, D - 1)]
    for b in range(B):
        for t in range(T):
            if parents[b, t] < -1:
                assert not out[b, t].any()
            elif vis[b, t, whole]:
                assert bool(out[b, t].isnan().all()), (b, t)
            elif vis[b, t, part]:
                assert bool(out[b, t, :, 5].isnan().all()) and bool((out[b, t, :, D - 1] == math.inf).all()), (b, t)
                assert torch.equal(out[b, t][:, rest], clean[b, t][:, rest]), (b, t)
            else:
                assert torch.equal(out[b, t], clean[b, t]), (b, t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(4, (4, 2, 64)), (20, (4, 2, 128)), (40, (4, 2, 64)), (90, (4, 2, 128))])
@pytest.mark.parametrize("B", [70, 200])
def test_many_sequences(dev, dtype, B, T, heads):
    """More sequences than a wave has lanes, of very different lengths: one long, most short, some empty."""
    print(f"[tree many] {dtype} B={B} T={T} heads={heads}", flush=True)
    lengths = [(37 * b) % 90 for b in range(B)]
    lengths[B - 3], lengths[5], lengths[66] = 2900, 0, 1100
    q, k, v, n, parents = _case(dev, dtype, B, T, heads, lengths, room=1, pad=2)
    out = K.tree_attn(q, k, v, n, parents.to(dev))
    _check(out, _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sequences_that_share_their_rows(dev, dtype):
    """Caches with a batch or head stride of 0: one prefix read by every sequence (its nodes' rows are then the same)."""
    B, T, nq, nk, D = 4, 9, 8, 2, 64
    q, k, v, n, parents = _case(dev, dtype, 1, T, (nq, nk, D), [900], room=0)
    q = q.repeat(B, 1) * torch.arange(1, B + 1, device=dev).repeat_interleave(T)[:, None].to(dtype)
    n, parents = n.repeat(B), parents.repeat(B, 1)
    for kk, vv in ((k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1)),
                   (k[:, :1].expand(B, nk, -1, -1), v[:, :1].expand(B, nk, -1, -1))):
        out = K.tree_attn(q, kk, vv, n, parents.to(dev))
        _check(out, _reference(q, kk, vv, n, parents, D ** -0.5), dtype)


def test_an_output_over_its_queries_is_refused(dev):
    q, k, v, n, parents = _case(dev, BF, 2, 6, (4, 2, 64), [40, 3], room=0)
    with pytest.raises(ValueError, match="overlaps"):
        K.tree_attn(q, k, v, n, parents.to(dev), out=q)
    both = torch.zeros(12, 512, device=dev, dtype=BF)    # columns of one tensor do not
    both[:, :256] = q
    K.tree_attn(both[:, :256], k, v, n, parents.to(dev), out=both[:, 256:])
    assert torch.equal(both[:, 256:], K.tree_attn(q, k, v, n, parents.to(dev)))


def test_scores_far_apart(dev):
    """Scores spread over thousands, the largest last: weights of the far ones are 0, and the maximum moves in steps."""
    B, T, nk, D, n = 1, 4, 1, 64, 900
    g = torch.Generator(device=dev).manual_seed(9)
    k = torch.randn(B, nk, n + T, D, device=dev, generator=g) * torch.linspace(0.1, 40, n + T, device=dev)[:, None]
    v = torch.randn(B, nk, n + T, D, device=dev, generator=g)
    q = torch.randn(B * T, D, device=dev, generator=g) * 20
    parents = _parents(B, T, 1)
    lengths = torch.tensor([n], device=dev)
    out = K.tree_attn(q, k, v, lengths, parents.to(dev))
    _check(out, _reference(q, k, v, lengths, parents, D ** -0.5), F32)


def test_long_cache(dev):
    """A cache of more than 2^32 bytes per tensor: the rows of the last head lie past every 32-bit offset."""
    B, T, nk, D, max_len = 1, 3, 9, 128, 2_000_003
    k = torch.zeros(B, nk, max_len, D, device=dev, dtype=BF)
    v = torch.zeros(B, nk, max_len, D, device=dev, dtype=BF)
    assert k.numel() * 2 > 2 ** 32
    g = torch.Generator(device=dev).manual_seed(2)
    for h in range(nk):
        k[0, h].normal_(generator=g)
        v[0, h].normal_(generator=g)
    q = torch.randn(B * T, 2 * nk * D, device=dev, generator=g).bfloat16()
    lengths, parents = torch.tensor([max_len - T], device=dev), _parents(B, T, 2)
    out = K.tree_attn(q, k, v, lengths, parents.to(dev)).view(B, T, nk, 2, D)
    h = nk - 1
    ref = _reference(q.view(B * T, nk, 2 * D)[:, h].contiguous(), k[:, h:], v[:, h:], lengths, parents, D ** -0.5)
    _check(out[:, :, h].reshape(B * T, 2 * D), ref, BF)


@pytest.mark.parametrize("dtype,T,heads", [(BF, 1, (8, 4, 128)), (BF, 9, (16, 4, 64)), (BF, 30, (16, 4, 128)), (BF, 60, (8, 4, 128)),
                                           (F32, 3, (8, 4, 64)), (F32, 20, (8, 4, 128))])
def test_caches_larger_than_the_memory_side_cache(dev, dtype, T, heads):
    """1 GB of keys and values in two sequences, the last head's outputs compared."""
    nq, nk, D = heads
    rows = 2 ** 30 // (2 * 2 * nk * D * (2 if dtype == BF else 4))
    q, k, v, n, parents = _case(dev, dtype, 2, T, heads, [rows - 1000, rows // 2 + 77], room=0)
    out = K.tree_attn(q, k, v, n, parents.to(dev)).view(2 * T, nk, -1)
    last = q.view(2 * T, nk, -1)[:, -1].contiguous()
    _check(out[:, -1], _reference(last, k[:, -1:], v[:, -1:], n, parents, D ** -0.5), dtype)


def test_tree_depths(dev):
    parents = _parents(5, 256, 11, pad=40)
    parents[2] = torch.arange(256, dtype=torch.int32) - 1
    parents[4, :9] = torch.tensor([0, 0, 7, 2, -2, 4, 1000, 3, 6], dtype=torch.int32)
    ref = (_visible(parents).sum(2) - 1).clamp(min=0)
    assert torch.equal(K.tree_depths(parents.to(dev)).cpu().long(), ref)
    assert K.tree_depths(torch.full((3, 1), -1, device=dev, dtype=torch.int32)).tolist() == [[0]] * 3


@pytest.mark.parametrize("empty", ["B", "T"])
def test_nothing_to_do(dev, empty):
    B, T = (0, 4) if empty == "B" else (3, 0)
    k = torch.zeros(B, 2, 16, 64, device=dev)
    out = K.tree_attn(torch.zeros(B * T, 256, device=dev), k, k, torch.zeros(B, device=dev, dtype=torch.int64),
                      torch.zeros(B, T, device=dev, dtype=torch.int32))
    assert out.shape == (0, 256)


# ---- cache rows ----------------------------------------------------------------------------------
def _caches(dev, count, B, nk, max_len, D, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(B, nk, max_len, D, device=dev, generator=g).to(dtype) for _ in range(count)]


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("P,count", [(1, 2), (5, 3), (17, 4), (256, 2)])
def test_cache_keep(dev, dtype, D, P, count):
    """Increasing paths, arbitrary lists (descending, the same node twice), entries that do not exist, counts past the
    list and below zero, rows at the cache's end."""
    B, nk, max_len = 6, 2, 300
    caches = _caches(dev, count, B, nk, max_len, D, dtype, P)
    g = torch.Generator().manual_seed(P)
    n = torch.tensor([0, 20, 44, 290, 300, 7])
    nodes = torch.randint(0, 260, (B, P), generator=g)
    nodes[0] = torch.sort(torch.randperm(260, generator=g)[:P]).values
    nodes[1] = torch.arange(P).flip(0)
    nodes[2, ::3] = -1
    nodes[2, 1::5] = 2 ** 40
    nodes[3] = torch.randint(0, 14, (P,), generator=g)
    counts = torch.tensor([P, P, P, P, P, max(0, P - 2)])
    if P == 5:
        counts[0], counts[5] = 99, -3
    want = [c.clone() for c in caches]
    for c, w in zip(caches, want):
        for b in range(B):
            for i in range(min(max(int(counts[b]), 0), P)):
                src, dst = int(n[b]) + int(nodes[b, i]), int(n[b]) + i
                if int(nodes[b, i]) >= 0 and src < max_len and dst < max_len:
                    w[b, :, dst] = c[b, :, src]
    K.cache_keep(caches, n.to(dev), nodes.to(dev), counts.to(dev))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_cache_keep_many_tensors(dev):
    """More tensors than one launch takes."""
    caches = _caches(dev, 150, 1, 1, 8, 64, BF, 0)
    want = [c.clone() for c in caches]
    for w, c in zip(want, caches):
        w[0, :, 3], w[0, :, 4] = c[0, :, 4], c[0, :, 6]
    K.cache_keep(caches, torch.tensor([3], device=dev), torch.tensor([[1, 3]], device=dev), torch.tensor([2], device=dev))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 128)])
@pytest.mark.parametrize("src_max,dst_max", [(77, 100), (300, 300), (300, 120)])
def test_cache_copy(dev, dtype, D, src_max, dst_max):
    """Copies between caches of other batch sizes and capacities: committed rows move, the rest stays, lengths follow;
    a destination too short takes what it holds."""
    nk, count = 3, 4
    src, dst = _caches(dev, count, 3, nk, src_max, D, dtype, 1), _caches(dev, count, 7, nk, dst_max, D, dtype, 2)
    n, m = torch.tensor([0, src_max, 41], device=dev), torch.arange(7, device=dev)
    pairs = [(2, 5), (1, 0), (2, 1), (0, 6)]
    want, lengths = [d.clone() for d in dst], m.clone()
    for a, b in pairs:
        rows = min(int(n[a]), dst_max)
        lengths[b] = rows
        for s, w in zip(src, want):
            w[b, :, :rows] = s[a, :, :rows]
    before = [s.clone() for s in src]
    K.cache_copy(src, dst, n, m, pairs)
    assert all(torch.equal(d, w) for d, w in zip(dst, want)) and torch.equal(m, lengths)
    assert all(torch.equal(s, w) for s, w in zip(src, before))


def test_cache_copy_within_one_cache_and_many_slots(dev):
    """A fork inside one cache (sources are not destinations), and more destinations and tensors than one launch
    takes."""
    caches = _caches(dev, 100, 140, 1, 9, 64, BF, 3)
    n = torch.arange(140, device=dev) % 10
    want, lengths = [c.clone() for c in caches], n.clone()
    pairs = [(7, d) for d in range(20, 120)] + [(3, 0), (9, 1)]
    for a, b in pairs:
        rows = min(int(n[a]), 9)
        lengths[b] = rows
        for w, c in zip(want, caches):
            w[b, :, :rows] = c[a, :, :rows]
    K.cache_copy(caches, caches, n, n, pairs)
    assert all(torch.equal(c, w) for c, w in zip(caches, want)) and torch.equal(n, lengths)
    K.cache_copy(caches, caches, n, n, [])
    assert torch.equal(n, lengths)


def test_captured_and_replayed(dev):
    """Attention, the kept path and a copy in one graph, replayed over changing lengths, trees and nodes with eager work
    between the replays; every replay equals the eager calls. Another stream than the default runs the same."""
    B, T, nq, nk, D, max_len = 2, 10, 8, 2, 128, 1500
    q, k, v, n, parents = _case(dev, BF, B, T, (nq, nk, D), [1200, 700], room=290)
    parents = parents.to(dev)
    nodes, counts = torch.tensor([[0, 2, 5], [1, 3, 4]], device=dev), torch.tensor([3, 2], device=dev)
    other, other_n = [torch.zeros_like(k), torch.zeros_like(v)], torch.zeros_like(n)

    def work():
        out = K.tree_attn(q, k, v, n, parents)
        K.cache_keep([k, v], n, nodes, counts)
        K.cache_copy([k, v], other, n, other_n, [(0, 1), (1, 0)])
        return out

    state = [t.clone() for t in (k, v, n, parents)]
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    stream = torch.cuda.Stream()
    for i in range(4):
        for t, s in zip((k, v, n, parents), state):
            t.copy_(s)
        n.sub_(i * 97)
        parents.copy_(_parents(B, T, 20 + i))
        begin = [t.clone() for t in (k, v)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (captured, k, v, *other, other_n)]
        for t, s in zip((k, v), begin):
            t.copy_(s)
        for t in other:
            t.zero_()
        other_n.zero_()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            eager = work()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        # rows that a shorter sequence does not fill keep what an earlier copy left: compare what is committed
        assert torch.equal(got[0], eager) and torch.equal(got[1], k) and torch.equal(got[2], v)
        assert torch.equal(got[5], other_n)
        for b, m in enumerate(other_n.tolist()):
            assert torch.equal(got[3][b, :, :m], other[0][b, :, :m]) and torch.equal(got[4][b, :, :m], other[1][b, :, :m])
        torch.randn(4096, device=dev).sum().item()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,heads", [(4, (8, 2, 64)), (17, (2, 2, 128)), (30, (8, 2, 128)), (70, (4, 2, 64)), (70, (4, 2, 128)),
                                     (256, (2, 1, 128))])
@pytest.mark.parametrize("scale", [-0.2, 0.0, -3.0])
def test_scales_that_are_not_positive(dev, dtype, T, heads, scale):
    """At every number of query rows, over one key range and several: softmax(scale q.k) is softmax(|scale| (-q).k), and with
    scale 0 the mean over the visible rows."""
    print(f"[tree scale] {dtype} T={T} heads={heads} scale={scale}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, 3, T, heads, [1500, 33, 0], room=300, pad=1, seed=13)
    out = K.tree_attn(q, k, v, n, parents.to(dev), scale=scale)
    _check(out, _reference(-q if scale else q * 0, k, v, n, parents, abs(scale) or 1.0), dtype)


def test_copies_of_more_than_two_gigabytes(dev):
    """One sequence to eight slots, 2.1 GB: committed rows moved, others as they were."""
    nk, D, rows = 8, 128, 32768
    src = [torch.empty(1, nk, rows, D, device=dev, dtype=BF).normal_() for _ in range(4)]
    dst = [torch.full((9, nk, rows + 1, D), 7.0, device=dev, dtype=BF) for _ in range(4)]
    n, m = torch.tensor([rows], device=dev), torch.zeros(9, device=dev, dtype=torch.int64)
    K.cache_copy(src, dst, n, m, [(0, d) for d in range(1, 9)])
    assert m.tolist() == [0] + [rows] * 8
    for s, d in zip(src, dst):
        assert bool((d[1:, :, :rows] == s).all()) and bool((d[:, :, rows] == 7).all()) and bool((d[0] == 7).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,heads,length", [(1, 16, (32, 8, 128), 1000), (4, 16, (32, 8, 128), 500), (5, 16, (32, 8, 128), 890),
                                              (8, 16, (32, 8, 128), 500), (8, 16, (32, 8, 128), 1000), (16, 3, (4, 2, 64), 900),
                                              (33, 3, (4, 2, 64), 1000), (1, 2, (4, 2, 64), 255), (2, 3, (4, 2, 64), 260)])
def test_sequences_of_few_key_blocks(dev, dtype, B, T, heads, length):
    """Numbers and lengths of sequences on both sides of the lines where their keys are cut into single blocks."""
    print(f"[tree blocks] {dtype} B={B} T={T} length={length}", flush=True)
    q, k, v, n, parents = _case(dev, dtype, B, T, heads, [length - b for b in range(B)], room=0)
    out = K.tree_attn(q, k, v, n, parents.to(dev))
    _check(out, _reference(q, k, v, n, parents, heads[2] ** -0.5), dtype)
