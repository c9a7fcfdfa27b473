"""LM-head objectives of the Uno step on the HIP kernels.

* ``fused_weighted_ce``: CE with the diffusion 1/t weighting (training/trainer.py:267-283). In
  bf16 the LM-head GEMM's epilogue reduces each 128-column block of logits to per-row softmax
  statistics and picks the target logit; it also stores the rows' fp32 logits when they fit
  CE_STORED_LOGITS_MAX_BYTES, and the backward then forms dz = g w (softmax - onehot) from them one
  vocabulary chunk at a time. Above that size the forward stores no logits and the backward
  recomputes them chunk by chunk in a GEMM whose epilogue emits dz. Either way dz passes through
  one [rows x chunk] bf16 buffer into the data-gradient GEMM.
* ``teacher_argmax``: first-index argmax of the clean-stream logits, chunked the same way
  (training/losses.py:38-56, target source "clean_argmax").
* ``distribution_losses``: reverse KL and total variation (training/losses.py:59-183) over
  bf16 logits of the supervised rows, fp32 per-row statistics, with hand-written backward.
* ``top_k_distillation_loss``: forward KL from a teacher of which only the top logits are kept
  (``teacher_top_k``), over the student's logits.
"""
from __future__ import annotations

import torch

from . import _native as N
from . import kernels as K

# Vocabulary columns per chunk of the CE backward (and of the fp32 / argmax chunk buffers).
DEFAULT_CE_CHUNK = 32768
# The bf16 CE keeps the LM-head logits of its rows (fp32) from the forward for the backward when
# they take at most this many bytes; beyond it the backward recomputes them inside its GEMM.
CE_STORED_LOGITS_MAX_BYTES = 6 << 30
# Rows of teacher logits that teacher_top_k holds at a time (2.5 GB in bf16 at 151936 columns).
TOP_K_ROWS = 8192


def lm_head_logits(lm_head, x: torch.Tensor) -> torch.Tensor:
    """Plain logits (used by project_hidden_states); differentiable w.r.t. x."""
    shape = x.shape
    out = _Logits.apply(x.reshape(-1, shape[-1]), lm_head.weight, lm_head.weight_t)
    return out.view(*shape[:-1], lm_head.weight.shape[0])


class _Logits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_t):
        x = x.contiguous()
        ctx.w_t = w_t
        return K.gemm_nt(x, w)

    @staticmethod
    def backward(ctx, dz):
        return K.gemm_nt(dz.contiguous(), ctx.w_t), None, None


def _chunks(V: int, chunk: int):
    for c0 in range(0, V, chunk):
        yield c0, min(V, c0 + chunk)


def _fused_ce_ok(h: torch.Tensor, w_lm: torch.Tensor) -> bool:
    """The GEMM-epilogue path: bf16, K a multiple of 64, and a vocabulary whose chunk ends keep the
    data-gradient GEMM's 8-element K granularity."""
    return (h.dtype == torch.bfloat16 and w_lm.dtype == torch.bfloat16 and h.shape[1] % 64 == 0
            and w_lm.shape[0] % 8 == 0 and w_lm.stride(1) == 1)


class ChunkedWeightedCE(torch.autograd.Function):
    """loss = inv_n * sum_r w_r * CE(h_r W^T, y_r); inv_n is a device scalar.

    bf16 (the step): the forward is one LM-head GEMM whose epilogue keeps per-row softmax
    statistics per 128 vocabulary columns and the target logit. When the rows' fp32 logits fit
    CE_STORED_LOGITS_MAX_BYTES, the same epilogue also stores them and the backward forms dz
    (bf16, one [rows x chunk] buffer) from them with a row kernel, chunk by chunk; otherwise it
    recomputes the logits inside a GEMM whose epilogue writes dz. Both give the same dz bit for
    bit (the same logits, the same arithmetic), which feeds the data-gradient GEMM.
    fp32 (parity mode) and other shapes: the logits of one vocabulary chunk at a time go through a
    chunk buffer and the row kernels, recomputed in the backward."""

    @staticmethod
    def forward(ctx, h, w_lm, w_lm_t, targets, weights, inv_n, chunk):
        h = h.contiguous()
        R, V = h.shape[0], w_lm.shape[0]
        dev = h.device
        f32 = dict(device=dev, dtype=torch.float32)
        run_max, run_sum, zt = torch.empty(R, **f32), torch.empty(R, **f32), torch.zeros(R, **f32)
        lse = torch.empty(R, **f32)
        loss = torch.empty((), **f32)
        fused = _fused_ce_ok(h, w_lm)
        z_all = None
        if fused:
            nparts = (V + 127) // 128
            pmax, psum = torch.empty((R, nparts), **f32), torch.empty((R, nparts), **f32)
            if V % 4 == 0 and R * V * 4 <= CE_STORED_LOGITS_MAX_BYTES:
                z_all = torch.empty((R, V), **f32)
            N.call("unok_lmhead_ce_stats", R, V, h.shape[1], N.ptr(h), h.stride(0), N.ptr(w_lm), w_lm.stride(0),
                   N.ptr(targets), 0, N.ptr(pmax), N.ptr(psum), nparts, N.ptr(zt), N.ptr(z_all), V, N.stream())
            N.call("unok_ce_parts_reduce", R, nparts, N.ptr(pmax), N.ptr(psum), nparts, N.ptr(run_max),
                   N.ptr(run_sum), N.stream())
            del pmax, psum
        else:
            buf = torch.empty((R, min(chunk, V)), **f32)
            for i, (c0, c1) in enumerate(_chunks(V, chunk)):
                z = buf[:, :c1 - c0]
                K.gemm_nt(h, w_lm[c0:c1], out=z)
                N.call("unok_row_lse_update", N.F32, R, c1 - c0, N.ptr(z), buf.stride(0), c0, N.ptr(targets),
                       N.ptr(run_max), N.ptr(run_sum), N.ptr(zt), int(i == 0), N.stream())
            del buf
        N.call("unok_ce_finish", R, N.ptr(run_max), N.ptr(run_sum), N.ptr(zt), N.ptr(weights), N.ptr(inv_n),
               N.ptr(lse), N.ptr(loss), N.stream())
        ctx.save = (h, w_lm, w_lm_t, targets, weights, inv_n, lse, chunk, fused, z_all)
        return loss

    @staticmethod
    def backward(ctx, g):
        h, w_lm, w_lm_t, targets, weights, inv_n, lse, chunk, fused, z_all = ctx.save
        ctx.save = None
        R, V = h.shape[0], w_lm.shape[0]
        g = g.reshape(1).float().contiguous()
        f32 = dict(device=h.device, dtype=torch.float32)
        width = min(chunk, V)
        dz = torch.empty((R, (width + 7) // 8 * 8), device=h.device, dtype=h.dtype)
        dh = torch.zeros(h.shape, **f32)
        buf = None if fused else torch.empty((R, width), **f32)
        for c0, c1 in _chunks(V, chunk):
            d = dz[:, :c1 - c0]
            if z_all is not None:
                N.call("unok_ce_grad_chunk", N.dtype_code(h.dtype), R, c1 - c0, N.ptr(z_all[:, c0:]), z_all.stride(0),
                       c0, N.ptr(lse), N.ptr(targets), N.ptr(weights), N.ptr(g), N.ptr(inv_n), N.ptr(d), dz.stride(0),
                       N.stream())
            elif fused:
                N.call("unok_lmhead_ce_grad", R, c1 - c0, h.shape[1], N.ptr(h), h.stride(0), N.ptr(w_lm[c0:c1]),
                       w_lm.stride(0), N.ptr(targets), c0, N.ptr(lse), N.ptr(weights), N.ptr(g), N.ptr(inv_n),
                       N.ptr(dz), dz.stride(0), N.stream())
            else:
                z = buf[:, :c1 - c0]
                K.gemm_nt(h, w_lm[c0:c1], out=z)
                N.call("unok_ce_grad_chunk", N.dtype_code(h.dtype), R, c1 - c0, N.ptr(z), buf.stride(0), c0,
                       N.ptr(lse), N.ptr(targets), N.ptr(weights), N.ptr(g), N.ptr(inv_n), N.ptr(d), dz.stride(0),
                       N.stream())
            K.gemm_nt(d, w_lm_t[:, c0:c1], out=dh, residual=dh)
        return dh.to(h.dtype), None, None, None, None, None, None


def fused_weighted_ce(lm_head, h_rows: torch.Tensor, targets: torch.Tensor, weights: torch.Tensor,
                      inv_n: torch.Tensor, chunk: int = DEFAULT_CE_CHUNK) -> torch.Tensor:
    if h_rows.shape[0] == 0:
        return h_rows.sum() * 0.0
    return ChunkedWeightedCE.apply(h_rows, lm_head.weight, lm_head.weight_t, targets.contiguous(),
                                   weights.contiguous().float(), inv_n, chunk)


@torch.no_grad()
def teacher_argmax(lm_head, h_rows: torch.Tensor, chunk: int = DEFAULT_CE_CHUNK) -> torch.Tensor:
    R, V = h_rows.shape[0], lm_head.weight.shape[0]
    h_rows = h_rows.contiguous()
    best_val = torch.empty(R, device=h_rows.device, dtype=torch.float32)
    best_idx = torch.empty(R, device=h_rows.device, dtype=torch.int64)
    if R == 0:
        return best_idx
    buf = torch.empty((R, min(chunk, V)), device=h_rows.device, dtype=h_rows.dtype)
    for i, (c0, c1) in enumerate(_chunks(V, chunk)):
        z = buf[:, :c1 - c0]
        K.gemm_nt(h_rows, lm_head.weight[c0:c1], out=z)
        N.call("unok_row_argmax_update", N.dtype_code(z.dtype), R, c1 - c0, N.ptr(z), buf.stride(0), c0,
               N.ptr(best_val), N.ptr(best_idx), int(i == 0), N.stream())
    return best_idx


@torch.no_grad()
def logits_argmax(z: torch.Tensor) -> torch.Tensor:
    """First-index argmax of each row of given [R, V] logits (fp32 or bf16) on the argmax kernel."""
    if z.dim() != 2:
        raise RuntimeError(f"logits must be [rows, vocab], got {tuple(z.shape)}")
    if z.shape[1] > 1 and z.stride(1) != 1:
        z = z.contiguous()
    R, V = z.shape
    best_val = torch.empty(R, device=z.device, dtype=torch.float32)
    best_idx = torch.empty(R, device=z.device, dtype=torch.int64)
    if R:
        N.call("unok_row_argmax_update", N.dtype_code(z.dtype), R, V, N.ptr(z), z.stride(0) if R > 1 else V, 0,
               N.ptr(best_val), N.ptr(best_idx), 1, N.stream())
    return best_idx


@torch.no_grad()
def teacher_top_k(lm_head, h_rows: torch.Tensor, k: int, rows: int = TOP_K_ROWS):
    """The top k logits of a teacher's hidden rows: (values [R, k] fp32, vocabulary indices [R, k], log-sum-exp [R]),
    ``rows`` rows of logits at a time (K.row_top_k)."""
    h_rows = h_rows.contiguous()
    parts = [K.row_top_k(K.gemm_nt(h_rows[r:r + rows], lm_head.weight), k) for r in range(0, h_rows.shape[0], rows)]
    if not parts:
        f32 = dict(device=h_rows.device, dtype=torch.float32)
        return torch.empty((0, k), **f32), torch.empty((0, k), device=h_rows.device, dtype=torch.int64), torch.empty(0, **f32)
    return parts[0] if len(parts) == 1 else tuple(torch.cat(p) for p in zip(*parts))


def _distill_operands(z: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, temperature: float) -> None:
    if z.dim() != 2 or values.shape != indices.shape or values.dim() != 2 or values.shape[0] != z.shape[0]:
        raise RuntimeError(f"top-k distillation: teacher values and indices [rows, k] must match the student's rows, got "
                           f"{tuple(values.shape)} {tuple(indices.shape)} for {tuple(z.shape)}")
    if indices.dtype != torch.int64:
        raise RuntimeError("top-k distillation: teacher indices must be int64")
    if not values.is_floating_point():
        raise RuntimeError(f"top-k distillation: teacher values must be floating-point, got {values.dtype}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("top-k distillation: the temperature must be positive and finite")
    for t in (values, indices):
        if t.device != z.device:
            raise RuntimeError(f"top-k distillation: teacher on {t.device}, student on {z.device}")


def _distill_fwd(z, values, indices, inv_n, scale, temperature):
    """(loss, row statistics for _distill_bwd) over [R, V] logits with unit column stride; inv_n None: 1."""
    K._same_device("top-k distillation", z, values, indices, *(() if inv_n is None else (inv_n,)))
    R, V = z.shape
    K._sizes("top-k distillation", R, V, values.shape[1])
    f32 = dict(device=z.device, dtype=torch.float32)
    nbytes = N.lib().unok_distill_workspace(R, V)
    stat, loss, ws = torch.empty((R, 2), **f32), torch.empty((), **f32), torch.empty(nbytes // 4, **f32)
    N.call("unok_distill_fwd", N.dtype_code(z.dtype), R, V, values.shape[1], N.ptr(z), z.stride(0), N.ptr(values),
           N.ptr(indices), temperature, N.ptr(inv_n), scale * temperature * temperature, N.ptr(stat), N.ptr(loss), N.ptr(ws),
           nbytes, N.stream())
    return loss, stat


def _distill_bwd(z, values, indices, stat, g, inv_n, scale, temperature, grad):
    g = g.float()
    N.call("unok_distill_bwd", N.dtype_code(z.dtype), *z.shape, values.shape[1], N.ptr(z), z.stride(0), N.ptr(values),
           N.ptr(indices), temperature, N.ptr(stat), N.ptr(g), N.ptr(inv_n), scale * temperature, N.ptr(grad), grad.stride(0),
           N.stream())
    return grad


class _OnceDifferentiable(torch.autograd.Function):
    """A gradient that has no derivative of its own; one that passes here is refused."""

    @staticmethod
    def forward(ctx, grad, anchor):
        return grad

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("top-k distillation is differentiable once")


def _once(grad: torch.Tensor) -> torch.Tensor:
    """``grad``; under create_graph, a second derivative through it is refused instead of left out."""
    return _OnceDifferentiable.apply(grad, grad.new_empty(0).requires_grad_()) if torch.is_grad_enabled() else grad


class TopKDistillation(torch.autograd.Function):
    """Distillation from a teacher's top logits over the LM head: logits from h_s (differentiable), gradient formed in
    their place. See top_k_distillation_loss."""

    @staticmethod
    def forward(ctx, h_s, values, indices, w_lm, w_lm_t, inv_n, temperature):
        z = K.gemm_nt(h_s.contiguous(), w_lm)
        loss, stat = _distill_fwd(z, values, indices, inv_n, 1.0, temperature)
        ctx.save = (z, values, indices, stat, inv_n, w_lm_t, temperature)
        return loss

    @staticmethod
    def backward(ctx, g):
        if ctx.save is None:
            raise RuntimeError("top-k distillation: backward a second time, but the first one overwrote the logits")
        z, values, indices, stat, inv_n, w_lm_t, temperature = ctx.save
        ctx.save = None
        _distill_bwd(z, values, indices, stat, g, inv_n, 1.0, temperature, z)
        return _once(K.gemm_nt(z, w_lm_t)), None, None, None, None, None, None


def top_k_distillation_loss(lm_head, h_s: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, inv_n: torch.Tensor,
                            temperature: float = 1.0) -> torch.Tensor:
    """tau^2 inv_n sum over rows of KL(p || q): p = softmax(values / tau) over a row's teacher entries ([R, k] logits and
    their vocabulary indices, k <= 256, as teacher_top_k returns them), q = softmax of the student's logits / tau over the
    whole vocabulary. Entries of value -inf, or with an index outside the vocabulary, do not count; a row without
    entries contributes nothing, to the loss and to the gradient. The teacher is not differentiated. tau is positive, 1 / tau
    and tau^2 numbers of fp32."""
    _distill_operands(h_s, values, indices, temperature)
    if inv_n.dtype != torch.float32 or inv_n.numel() != 1:
        raise RuntimeError(f"top-k distillation: inv_n must be one fp32 number, got {inv_n.dtype} {tuple(inv_n.shape)}")
    if h_s.shape[0] == 0:
        return h_s.sum() * 0.0
    return TopKDistillation.apply(h_s, values.detach().float().contiguous(), indices.contiguous(), lm_head.weight,
                                  lm_head.weight_t, inv_n, float(temperature))


class LogitsTopKDistillation(torch.autograd.Function):
    """The same over given logits (the losses.py call surface), scaled by a number; gradient w.r.t. the student's."""

    @staticmethod
    def forward(ctx, z, values, indices, scale, temperature):
        if (z.stride(1) != 1 and z.shape[1] > 1) or z.stride(0) < z.shape[1]:   # (an expanded row: copied)
            z = z.contiguous()
        loss, stat = _distill_fwd(z, values, indices, None, scale, temperature)
        ctx.save_for_backward(z, values, indices, stat)
        ctx.scale, ctx.temperature = scale, temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        z, values, indices, stat = ctx.saved_tensors
        grad = torch.empty(z.shape, device=z.device, dtype=z.dtype)
        return _once(_distill_bwd(z, values, indices, stat, g, None, ctx.scale, ctx.temperature, grad)), None, None, None, None


class DistributionLoss(torch.autograd.Function):
    """kind 'tv': sum |p_s - p_t| * inv_n;  kind 'kl': sum p_s (log p_s - log p_t) * inv_n.
    Student logits are computed from h_s (differentiable), teacher logits from h_t (detached)."""

    @staticmethod
    def forward(ctx, h_s, h_t, w_lm, w_lm_t, inv_n, kind):
        h_s, h_t = h_s.contiguous(), h_t.contiguous()
        R, V = h_s.shape[0], w_lm.shape[0]
        zs = K.gemm_nt(h_s, w_lm)
        zt = K.gemm_nt(h_t, w_lm)
        f32 = dict(device=h_s.device, dtype=torch.float32)
        ms, ss, mt, st = (torch.empty(R, **f32) for _ in range(4))
        dt = N.dtype_code(zs.dtype)
        N.call("unok_softmax_stats", dt, R, V, N.ptr(zs), V, N.ptr(ms), N.ptr(ss), N.stream())
        N.call("unok_softmax_stats", dt, R, V, N.ptr(zt), V, N.ptr(mt), N.ptr(st), N.stream())
        rows = torch.empty(R, **f32)
        extra = torch.empty(R, **f32)
        if kind == "tv":
            N.call("unok_tv_fwd", dt, R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt), N.ptr(st),
                   N.ptr(rows), N.ptr(extra), N.stream())
        elif kind == "kl":
            N.call("unok_kl_fwd", dt, R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt), N.ptr(st),
                   N.ptr(rows), N.stream())
            extra = rows
        else:
            raise ValueError(kind)
        loss = torch.empty((), **f32)
        N.call("unok_sum_scaled", R, N.ptr(rows), N.ptr(inv_n), N.ptr(loss), N.stream())
        ctx.save = (zs, zt, ms, ss, mt, st, extra, inv_n, w_lm_t, kind)
        return loss

    @staticmethod
    def backward(ctx, g):
        zs, zt, ms, ss, mt, st, extra, inv_n, w_lm_t, kind = ctx.save
        ctx.save = None
        R, V = zs.shape
        g = g.reshape(1).float().contiguous()
        dt = N.dtype_code(zs.dtype)
        fn = "unok_tv_bwd" if kind == "tv" else "unok_kl_bwd"
        N.call(fn, dt, R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt), N.ptr(st), N.ptr(extra),
               N.ptr(g), N.ptr(inv_n), N.ptr(zs), V, N.stream())
        dh = K.gemm_nt(zs, w_lm_t)
        return dh, None, None, None, None, None


def distribution_loss(lm_head, h_s, h_t, inv_n, kind: str) -> torch.Tensor:
    if h_s.shape[0] == 0:
        return h_s.sum() * 0.0
    return DistributionLoss.apply(h_s, h_t.detach(), lm_head.weight, lm_head.weight_t, inv_n, kind)


class LogitsDistributionLoss(torch.autograd.Function):
    """TV / reverse KL over given logits (the losses.py call surface); gradient w.r.t. student."""

    @staticmethod
    def forward(ctx, zs, zt, inv_n, kind):
        zs, zt = zs.contiguous(), zt.contiguous()
        R, V = zs.shape
        f32 = dict(device=zs.device, dtype=torch.float32)
        ms, ss, mt, st = (torch.empty(R, **f32) for _ in range(4))
        dt = N.dtype_code(zs.dtype)
        if zt.dtype != zs.dtype:
            raise RuntimeError("student and teacher logits must share a dtype")
        N.call("unok_softmax_stats", dt, R, V, N.ptr(zs), V, N.ptr(ms), N.ptr(ss), N.stream())
        N.call("unok_softmax_stats", dt, R, V, N.ptr(zt), V, N.ptr(mt), N.ptr(st), N.stream())
        rows, extra = torch.empty(R, **f32), torch.empty(R, **f32)
        if kind == "tv":
            N.call("unok_tv_fwd", dt, R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt), N.ptr(st),
                   N.ptr(rows), N.ptr(extra), N.stream())
        else:
            N.call("unok_kl_fwd", dt, R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt), N.ptr(st),
                   N.ptr(rows), N.stream())
            extra = rows
        loss = torch.empty((), **f32)
        N.call("unok_sum_scaled", R, N.ptr(rows), N.ptr(inv_n), N.ptr(loss), N.stream())
        ctx.save = (zs, zt, ms, ss, mt, st, extra, inv_n, kind)
        return loss

    @staticmethod
    def backward(ctx, g):
        zs, zt, ms, ss, mt, st, extra, inv_n, kind = ctx.save
        ctx.save = None
        R, V = zs.shape
        g = g.reshape(1).float().contiguous()
        grad = torch.empty_like(zs)
        fn = "unok_tv_bwd" if kind == "tv" else "unok_kl_bwd"
        N.call(fn, N.dtype_code(zs.dtype), R, V, N.ptr(zs), V, N.ptr(zt), V, N.ptr(ms), N.ptr(ss), N.ptr(mt),
               N.ptr(st), N.ptr(extra), N.ptr(g), N.ptr(inv_n), N.ptr(grad), V, N.stream())
        return grad, None, None, None
