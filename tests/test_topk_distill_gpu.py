"""Top logits of rows (K.row_top_k, objectives.teacher_top_k) and the distillation loss from a teacher's top logits,
forward and backward, against plain implementations in 64 bits.

Values and columns of the top are exact. Bounds, with u = 2^-24:
* log-sum-exp of V terms below the maximum m: the sum is off by at most (V + 40) u relative (hardware exp2 and the
  product before it are off by (2 |x| + 2) u, and terms beyond |x| = 20 weigh nothing at this scale), m + log by one rounding
  of its size: (V + 60) u + 2 u |lse|. (Sums are taken by 256 threads, so V / 256 + 20 terms in a row count.)
* loss: a row's term sums p_i (log p_i - log q_i), each log off by the above: E = (V / 256 + 100) u + 4 u max |z| / tau per unit
  of weight, plus the sum over rows.
* gradient g tau inv_n (q - p): q and p are off by (V / 256 + 100 + 4 max |z| / tau) u relative, the result is rounded to
  its type once (half a step).
"""
import math

import pytest
import torch

from uno_amd import kernels as K
from uno_amd import objectives
from uno_amd.objectives import teacher_top_k, top_k_distillation_loss
from uno_amd.training.losses import token_normalized_top_k_distillation

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def _reference_top(z, k):
    v, i = torch.sort(z.double() + 0.0, dim=1, descending=True, stable=True)
    return v[:, :k], i[:, :k]


def _check_top(z, k, got):
    values, cols, lse = got
    v, i = _reference_top(z, k)
    assert values.dtype == F32 and cols.dtype == torch.int64 and lse.dtype == F32
    assert torch.equal(cols, i)
    assert torch.equal(values.double().nan_to_num(1e300), v.nan_to_num(1e300))
    ref = torch.logsumexp(z.double(), 1)
    finite = ref.isfinite()
    tol = (z.shape[1] / 256 + 80) * U + 2 * U * ref.abs()
    assert bool(((lse.double() - ref).abs() <= tol)[finite].all())
    odd = ~finite
    assert torch.equal(lse[odd].double().nan_to_num(1e300), ref[odd].nan_to_num(1e300))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 7, 7), (2, 40, 1), (5, 257, 256), (64, 1000, 17), (7, 4096, 64), (600, 5003, 33),
                                   (1, 151936, 10), (3, 151936, 256), (17, 32000, 128), (1, 8191, 64), (2, 8200, 256)])
def test_row_top_k(dev, dtype, R, V, k):
    print(f"[topk] {dtype} R={R} V={V} k={k}", flush=True)
    g = torch.Generator(device=dev).manual_seed(R + V + k)
    z = (torch.randn(R, V, device=dev, generator=g) * 3).to(dtype)
    got = K.row_top_k(z, k)
    _check_top(z, k, got)
    assert all(torch.equal(a, b) for a, b in zip(got, K.row_top_k(z, k)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [300, 9000, 40001])
@pytest.mark.parametrize("k", [1, 20, 256])
def test_row_top_k_orders(dev, dtype, V, k):
    """Orders that are worst for a running threshold, ties, signed zeros, infinities, NaN."""
    rows = []
    g = torch.Generator(device=dev).manual_seed(V)
    ramp = torch.arange(V, device=dev, dtype=F32)
    rows.append(ramp)                                             # ascending: every element is a new maximum
    rows.append(-ramp)
    rows.append(torch.full((V,), 0.5, device=dev))                # all equal
    rows.append((ramp % 3 == 0).float())                          # many ties
    rows.append(torch.where(ramp % 2 == 0, -0.0, 0.0))            # signed zeros are equal
    rows.append(torch.full((V,), -math.inf, device=dev))
    rows.append(torch.where(ramp % 50 == 7, ramp, -math.inf))     # fewer finite values than k
    r = torch.randn(V, device=dev, generator=g)
    r[V // 2], r[5], r[V - 1] = math.nan, math.nan, math.inf
    rows.append(r)
    rows.append(torch.full((V,), math.nan, device=dev))
    r = torch.randn(V, device=dev, generator=g)
    r[V // 3:V // 3 + 4] = math.inf
    rows.append(r)
    rows.append(torch.where(ramp % 11 == 3, math.nan, -math.inf))
    rows.append(torch.randint(0, 4, (V,), device=dev, generator=g).float() - 2)
    rows.append(ramp * 1e34)
    z = torch.stack(rows).to(dtype)
    _check_top(z, k, K.row_top_k(z, k))
    many = z.repeat(60, 1)                                        # one part per row
    _check_top(many, k, K.row_top_k(many, k))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [5, 3001, 70001])
def test_row_top_k_far_from_zero(dev, dtype, V):
    """Values whose product with log2 e is coarse, or no float."""
    g = torch.Generator(device=dev).manual_seed(V)
    r = torch.randn(V, device=dev, generator=g)
    step = torch.randint(0, 4, (V,), device=dev, generator=g).float()
    rows = [1e5 + r, -1e5 + r, 1048576.0 + step, -1048570.0 - step, 1e7 + step, -1e7 - step, 3e38 + 0 * r, -3e38 + 0 * r,
            torch.where(step == 0, 2e38, -2e38), torch.where(step == 0, 1e7, r), torch.where(step == 0, -1e7, -3e38)]
    _check_top(torch.stack(rows).to(dtype), min(V, 9), K.row_top_k(torch.stack(rows).to(dtype), min(V, 9)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("offset,stride", [(0, 1009), (1, 1010), (3, 1024), (7, 1111)])
def test_row_top_k_strides(dev, dtype, offset, stride):
    """Rows at every alignment; what lies between the rows is not read as a value."""
    R, V, k = 9, 1001, 40
    buf = torch.full((R * stride + 16,), math.inf, device=dev, dtype=dtype)
    z = buf[offset:offset + R * stride].view(R, stride)[:, :V]
    z.copy_(torch.randn(R, V, device=dev))
    _check_top(z, k, K.row_top_k(z, k))


def test_row_top_k_empty(dev):
    v, i, l = K.row_top_k(torch.zeros(0, 50, device=dev), 5)
    assert v.shape == i.shape == (0, 5) and l.shape == (0,)


# ---- distillation --------------------------------------------------------------------------------
def _reference_loss(z, values, indices, n, tau):
    """(loss, gradient, weight of the loss's error bound) in 64 bits; entries of -inf or outside the columns do not count."""
    z, V = z.detach().double() / tau, z.shape[1]
    ok = (values > -math.inf) & (indices >= 0) & (indices < V)
    t = torch.where(ok, values.double() / tau, -math.inf)
    live = ok.any(1)
    logp = torch.where(live[:, None], torch.log_softmax(torch.where(live[:, None], t, 0.0), 1), -math.inf)
    p = torch.where(ok, logp.exp(), 0.0)
    logq = torch.log_softmax(z, 1)
    at = logq.gather(1, indices.clamp(0, V - 1))
    terms = torch.where(p > 0, p * (logp - at), 0.0)
    grad = torch.where(live[:, None], logq.exp(), 0.0)
    grad.scatter_add_(1, indices.clamp(0, V - 1), -p)
    pd = torch.zeros_like(grad).scatter_add_(1, indices.clamp(0, V - 1), p)
    return terms.sum() * tau * tau / n, grad * tau / n, p.sum() * tau * tau / n, pd * tau / n


def _check_loss(z, values, indices, n, tau, loss, grad):
    ref, gref, weight, pd = _reference_loss(z, values, indices, n, tau)
    V = z.shape[1]
    E = (V / 256 + 100) * U + 6 * U * z.double().abs().max() / tau
    assert abs(loss.double() - ref) <= E * weight * (1 + math.log(V)) + 2 * U * abs(ref) + 1e-30
    bound = HALF[z.dtype] * gref.abs() + 1.01 * E * (gref.abs() + 2 * pd) + 2.0 ** -126
    bad = (grad.double() - gref).abs() - bound
    assert bool((bad <= 0).all()), (bad.max().item(), int((bad > 0).sum()))


def _teacher(z, k, g):
    t = z.float() + torch.randn(z.shape, device=z.device, generator=g)
    return tuple(x.contiguous() for x in torch.topk(t, k, dim=1))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V,k,tau", [(1, 1, 1, 1.0), (3, 40, 40, 0.5), (33, 1001, 17, 2.0), (5, 151936, 256, 1.0), (1, 32000, 64, 1.0),
                                       (300, 4096, 65, 1.3), (2000, 513, 3, 1.0)])
def test_distillation(dev, dtype, R, V, k, tau):
    print(f"[distill] {dtype} R={R} V={V} k={k} tau={tau}", flush=True)
    g = torch.Generator(device=dev).manual_seed(R + V)
    z = (torch.randn(R, V, device=dev, generator=g) * 3).to(dtype).requires_grad_(True)
    values, indices = _teacher(z.detach(), k, g)
    loss = token_normalized_top_k_distillation(z, values, indices, R + 3, temperature=tau)
    (grad,) = torch.autograd.grad(loss, z)
    assert grad.dtype == dtype
    _check_loss(z.detach(), values, indices, R + 3, tau, loss.detach(), grad)
    again = token_normalized_top_k_distillation(z, values, indices, R + 3, temperature=tau)
    assert torch.equal(again, loss) and torch.equal(torch.autograd.grad(again * 2, z)[0], (grad.float() * 2).to(dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distillation_ragged_and_odd_entries(dev, dtype):
    """Rows with fewer entries, none at all, columns outside the vocabulary, the same column twice and k times, teachers of
    one entry, student logits of -inf."""
    R, V, k, n = 9, 777, 12, 5
    g = torch.Generator(device=dev).manual_seed(1)
    z = torch.randn(R, V, device=dev, generator=g).to(dtype)
    values, indices = _teacher(z, k, g)
    values[1, 5:] = -math.inf
    values[2] = -math.inf
    indices[3, ::2] = -100
    indices[4] = V + 3
    indices[4, 1] = 2 ** 40
    indices[5, 3] = indices[5, 0]
    indices[6] = 700
    values[7, 1:] = -math.inf
    z[8, ::2] = -math.inf
    indices[8] = indices[8] // 2 * 2 + 1
    indices[8].clamp_(max=V - 2)
    values[8, 4], indices[8, 4] = -math.inf, 0
    z.requires_grad_(True)
    loss = token_normalized_top_k_distillation(z, values, indices, n)
    (grad,) = torch.autograd.grad(loss, z)
    zd = z.detach()
    sub = [0, 1, 2, 3, 4, 5, 6, 7]
    _check_loss(zd[sub], values[sub], indices[sub], n, 1.0,
                token_normalized_top_k_distillation(zd[sub], values[sub], indices[sub], n), grad[sub])
    assert bool((grad[2] == 0).all()) and bool((grad[4] == 0).all())
    # the row with logits of -inf: they get no gradient, and the rest is the loss over the other columns
    keep = torch.arange(1, V, 2, device=dev)
    _check_loss(zd[8:, keep], values[8:], indices[8:] // 2, n, 1.0,
                token_normalized_top_k_distillation(zd[8:], values[8:], indices[8:], n), grad[8:][:, keep])
    assert bool((grad[8, ::2] == 0).all())
    # a student logit of -inf where the teacher has weight: an infinite loss, as the formula has it
    zd[0, indices[0, 0]] = -math.inf
    assert token_normalized_top_k_distillation(zd, values, indices, n).item() == math.inf


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distillation_strides(dev, dtype):
    """Student rows with a stride of their own, at odd alignments, and a transposed matrix."""
    R, V, k = 6, 1003, 20
    g = torch.Generator(device=dev).manual_seed(2)
    buf = torch.full((R, V + 6), math.nan, device=dev, dtype=dtype)
    z = buf[:, 3:3 + V]
    z.copy_(torch.randn(R, V, device=dev, generator=g))
    values, indices = _teacher(z, k, g)
    for view in (z, z.t().contiguous().t()):
        zr = view.detach().requires_grad_(True)
        loss = token_normalized_top_k_distillation(zr, values, indices, R)
        (grad,) = torch.autograd.grad(loss, zr)
        _check_loss(view, values, indices, R, 1.0, loss.detach(), grad)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distillation_broadcast_inputs(dev, dtype):
    """One row of logits for all teacher rows, one teacher row for all logits: the shared row's gradient is the sum."""
    R, V, k = 5, 640, 9
    g = torch.Generator(device=dev).manual_seed(12)
    z = torch.randn(1, V, device=dev, generator=g).to(dtype)
    values, indices = _teacher(torch.randn(R, V, device=dev, generator=g), k, g)
    leaf = z.clone().requires_grad_(True)
    wide = leaf.expand(R, V)
    loss = token_normalized_top_k_distillation(wide, values, indices, R)
    per_row, shared = torch.autograd.grad(loss, (wide, leaf))
    _check_loss(z.expand(R, V), values, indices, R, 1.0, loss.detach(), per_row)
    # autograd's sum of R rows in the leaf's type: each addition rounds by half a step of at most the sum of magnitudes
    assert bool(((shared.double() - per_row.double().sum(0)).abs() <= R * HALF[dtype] * per_row.double().abs().sum(0)).all())
    many = torch.randn(R, V, device=dev, generator=g).to(dtype).requires_grad_(True)
    one = (values[:1].expand(R, k), indices[:1].expand(R, k))
    loss = token_normalized_top_k_distillation(many, *one, R)
    (grad,) = torch.autograd.grad(loss, many)
    _check_loss(many.detach(), *one, R, 1.0, loss.detach(), grad)


def test_distillation_gradient_against_differences(dev):
    """Central differences of the loss in 64 bits around the kernel's inputs: step h, so off by h^2 / 6 of a third derivative
    that a softmax bounds by 1, and by the rounding of two losses of 64 bits."""
    R, V, k, n, tau, h = 2, 60, 5, 3, 1.5, 1e-4
    g = torch.Generator(device=dev).manual_seed(3)
    z = torch.randn(R, V, device=dev, generator=g)
    values, indices = _teacher(z, k, g)
    zr = z.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(token_normalized_top_k_distillation(zr, values, indices, n, temperature=tau), zr)
    for r, j in [(0, 0), (0, int(indices[0, 0])), (1, int(indices[1, 4])), (1, 59)]:
        d = torch.zeros_like(z, dtype=torch.float64)
        d[r, j] = h
        diff = (_reference_loss(z.double() + d, values, indices, n, tau)[0]
                - _reference_loss(z.double() - d, values, indices, n, tau)[0]) / (2 * h)
        assert abs(diff.item() - grad[r, j].item()) <= h * h + 1e-11 / h * 1e-4 + 300 * U


class _Head(torch.nn.Module):
    def __init__(self, w):
        super().__init__()
        self.weight, self.weight_t = w, w.t().contiguous()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_teacher_and_student_over_the_lm_head(dev, dtype):
    """The run of them together: the clean stream's top logits, then the student's loss and the gradient of its hidden
    rows, equal to the same operators over the logits (bit for bit) and its product with the LM head."""
    R, H, V, k = 200, 256, 5000, 32
    g = torch.Generator(device=dev).manual_seed(5)
    head = _Head((torch.randn(V, H, device=dev, generator=g) * 0.1).to(dtype))
    h_t, h_s = (torch.randn(R, H, device=dev, generator=g).to(dtype) for _ in "ts")
    values, indices, lse = teacher_top_k(head, h_t, k, rows=77)
    same = [K.row_top_k(K.gemm_nt(h_t[r:r + 77], head.weight), k) for r in range(0, R, 77)]
    assert all(torch.equal(torch.cat([s[i] for s in same]), (values, indices, lse)[i]) for i in range(3))
    inv_n = torch.full((), 1 / 150, device=dev)
    hs = h_s.clone().requires_grad_(True)
    loss = top_k_distillation_loss(head, hs, values, indices, inv_n, temperature=1.5)
    (dh,) = torch.autograd.grad(loss, hs)
    z = K.gemm_nt(h_s, head.weight).requires_grad_(True)
    ref = token_normalized_top_k_distillation(z, values, indices, 150, temperature=1.5)
    (dz,) = torch.autograd.grad(ref, z)
    assert torch.equal(loss, ref) and torch.equal(dh, K.gemm_nt(dz, head.weight_t))
    # a batch without rows stays differentiable
    e = h_s[:0].clone().requires_grad_(True)
    none = top_k_distillation_loss(head, e, values[:0], indices[:0], inv_n)
    none.backward()
    assert none.item() == 0 and e.grad.shape == (0, H)
    assert teacher_top_k(head, h_t[:0], k)[0].shape == (0, k)


def test_captured_and_replayed(dev):
    """Top logits, loss and gradient in one graph, replayed over changing logits with eager work between the replays."""
    R, V, k = 12, 9001, 21
    g = torch.Generator(device=dev).manual_seed(6)
    z = torch.randn(R, V, device=dev, generator=g).bfloat16()
    t = torch.randn(R, V, device=dev, generator=g).bfloat16()
    one = torch.ones((), device=dev)

    def work():
        values, indices, lse = K.row_top_k(t, k)
        leaf = z.detach().requires_grad_(True)
        loss = token_normalized_top_k_distillation(leaf, values, indices, R)
        (grad,) = torch.autograd.grad(loss, leaf, one)
        return values, indices, lse, loss.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for i in range(4):
        z.copy_(torch.randn(R, V, device=dev, generator=g))
        t.copy_(torch.randn(R, V, device=dev, generator=g) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        for a, b in zip(got, work()):
            assert torch.equal(a, b), i
        torch.randn(4096, device=dev).sum().item()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [40, 9001, 40009])
@pytest.mark.parametrize("low", ["lowest", -3e10])
@pytest.mark.parametrize("rows", [1, 700])
def test_row_top_k_masked_by_low_values(dev, dtype, V, low, rows):
    """Columns masked with the type's lowest value (or another whose product with log2 e is no small number): the first half,
    the first one, all but the last, the second half, all but one in the middle, every one."""
    low = torch.finfo(dtype).min if low == "lowest" else low
    g = torch.Generator(device=dev).manual_seed(V)
    z = (torch.randn(6, V, device=dev, generator=g) * 3).to(dtype)
    z[0, :V // 2] = low
    z[1, 0] = low
    z[2, :-1] = low
    z[3, V // 2:] = low
    z[4, :V // 2], z[4, V // 2 + 1:] = low, low
    z[5] = low
    z = z.repeat((rows + 5) // 6, 1)
    _check_top(z, min(V, 20), K.row_top_k(z, min(V, 20)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,R", [(777, 8), (40009, 8)])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_distillation_over_lowest_values(dev, dtype, V, R, tau):
    """Columns masked with the type's lowest value: most of a student's row, all of it, a teacher's entries but one, all of
    them (finite, so they count), and a whole row raised to where its values over tau are no numbers of fp32. With z and t the
    same numbers as in the kernel, q and p are softmaxes of differences, which the reference takes of values less their maximum."""
    k, n = 12, 5
    g = torch.Generator(device=dev).manual_seed(V)
    z = torch.randn(R, V, device=dev, generator=g).to(dtype)
    values, indices = _teacher(z, k, g)
    low = torch.finfo(dtype).min
    kept = torch.zeros(V, device=dev, dtype=torch.bool)
    kept[indices[0]] = True
    z[0] = torch.where(kept, z[0], low)
    z[1] = low
    values[2, 1:] = torch.finfo(F32).min
    values[3] = torch.finfo(F32).min
    z[4], values[5] = 3e38, 3e38
    leaf = z.clone().requires_grad_(True)
    loss = token_normalized_top_k_distillation(leaf, values, indices, n, temperature=tau)
    (grad,) = torch.autograd.grad(loss, leaf)
    zs = z.double() - z.double().amax(1, keepdim=True)
    vs = values.double() - values.double().amax(1, keepdim=True)
    ref, gref, weight, pd = _reference_loss(zs, vs, indices, n, tau)
    # a row's values less its maximum, where they weigh anything, are of the size of the unmasked ones: below 16
    E = (V / 256 + 100) * U + 6 * U * 16 / tau
    assert abs(loss.double() - ref) <= E * weight * (1 + math.log(V)) + 2 * U * abs(ref) + 1e-30
    bound = HALF[dtype] * gref.abs() + 1.01 * E * (gref.abs() + 2 * pd) + 2.0 ** -126
    bad = (grad.double() - gref).abs() - bound
    assert bool((bad <= 0).all()), (bad.max().item(), int((bad > 0).sum()))


@pytest.mark.parametrize("dtype,R", [(BF, 900), (F32, 450)])
@pytest.mark.parametrize("extra", [0, 5])
def test_logits_larger_than_the_memory_side_cache(dev, dtype, R, extra):
    """More than 256 MB, rows with and without elements between them: top logits, loss, gradient."""
    V, k, tau = 151936, 40, 1.5
    print(f"[large] {dtype} R={R} extra={extra}", flush=True)
    g = torch.Generator(device=dev).manual_seed(R)
    z = (torch.randn(R, V + extra, device=dev, generator=g) * 3).to(dtype)[:, :V]
    assert R * V * z.element_size() > 2 ** 28
    _check_top(z, k, K.row_top_k(z, k))
    values, indices = _teacher(z, k, g)
    leaf = z.detach().requires_grad_(True)
    loss = token_normalized_top_k_distillation(leaf, values, indices, R, temperature=tau)
    (grad,) = torch.autograd.grad(loss, leaf)
    _check_loss(z, values, indices, R, tau, loss.detach(), grad)


def test_more_than_two_to_the_31_logits(dev):
    """14,140 rows of 151936: the loss over all rows, the gradient of the first, the last and those around element 2^31."""
    R, V, k, n = 14140, 151936, 7, 14140
    assert R * V > 2 ** 31
    g = torch.Generator(device=dev).manual_seed(4)
    z = torch.empty(R, V, device=dev, dtype=BF)
    for r in range(0, R, 1000):
        z[r:r + 1000].normal_(generator=g)
    values = torch.randn(R, k, device=dev, generator=g)
    indices = torch.randint(0, V, (R, k), device=dev, generator=g)
    z.requires_grad_(True)
    loss = token_normalized_top_k_distillation(z, values, indices, n)
    (grad,) = torch.autograd.grad(loss, z)
    zd = z.detach()
    ref = weight = 0.0
    for r in range(0, R, 500):
        part = _reference_loss(zd[r:r + 500], values[r:r + 500], indices[r:r + 500], n, 1.0)
        ref, weight = ref + part[0], weight + part[2]
    E = (V / 256 + 100) * U + 6 * U * zd.abs().max().double()
    assert abs(loss.detach().double() - ref) <= E * weight * (1 + math.log(V)) + 2 * U * abs(ref)
    for r in (0, 2 ** 31 // V - 1, 2 ** 31 // V, 2 ** 31 // V + 1, R - 1):
        row = slice(r, r + 1)
        one = token_normalized_top_k_distillation(zd[row], values[row], indices[row], n)
        _check_loss(zd[row], values[row], indices[row], n, 1.0, one, grad[row])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [5000, 32000, 151936])
@pytest.mark.parametrize("R", [1, 16, 300])
@pytest.mark.parametrize("extra,offset", [(0, 0), (1, 0), (13, 3)])
def test_gradient_in_the_logits_place(dev, dtype, V, R, extra, offset):
    """As the loss over the LM head takes it, rows in one part and in several, at any alignment: bit for bit the gradient in a
    tensor of its own; what lies between the rows stays as it was."""
    k, tau = 30, 0.8
    g = torch.Generator(device=dev).manual_seed(V + R)
    buf = torch.full((R * (V + extra) + offset,), 7.0, device=dev, dtype=dtype)
    z = buf[offset:].view(R, V + extra)[:, :V]
    z.copy_(torch.randn(R, V, device=dev, generator=g) * 3)
    values, indices = _teacher(z, k, g)
    indices[0, 3] = indices[0, 0]
    inv_n, up = torch.full((), 1 / 9, device=dev), torch.full((), 1.5, device=dev)
    loss, stat = objectives._distill_fwd(z, values, indices, inv_n, 1.0, tau)
    apart = objectives._distill_bwd(z, values, indices, stat, up, inv_n, 1.0, tau, torch.empty(R, V, device=dev, dtype=dtype))
    ref, gref, _, _ = _reference_loss(z, values, indices, 9, tau)
    assert ((apart.double() - 1.5 * gref).norm() / (1.5 * gref).norm()).item() < HALF[dtype] + 1e-5
    objectives._distill_bwd(z, values, indices, stat, up, inv_n, 1.0, tau, z)
    assert torch.equal(z, apart)
    assert bool((buf[:offset] == 7).all()) and bool((buf[offset:].view(R, V + extra)[:, V:] == 7).all())


def test_a_second_derivative_is_refused(dev):
    """With create_graph the gradient is the same, and a derivative of it refused."""
    R, V, k = 4, 300, 7
    g = torch.Generator(device=dev).manual_seed(3)
    z = torch.randn(R, V, device=dev, generator=g).requires_grad_(True)
    values, indices = _teacher(z.detach(), k, g)
    (plain,) = torch.autograd.grad(token_normalized_top_k_distillation(z, values, indices, R), z)
    (grad,) = torch.autograd.grad(token_normalized_top_k_distillation(z, values, indices, R), z, create_graph=True)
    assert torch.equal(plain, grad) and not plain.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        (grad.sum() + (z ** 2).sum()).backward()
