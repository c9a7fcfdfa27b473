"""Functional wrappers over the HIP kernel library (one per C-ABI entry point).

Every wrapper validates shapes and strides on the host, allocates outputs with torch (which
owns all device memory) and enqueues the kernel on torch's current stream. There is no
non-HIP code path.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Sequence

import torch

from . import _native as N


class LaunchRecorder:
    """Brackets selected GEMM launches with HIP events (torch's current stream, which is the
    stream the kernels run on) to measure their live duration inside a timed region."""

    def __init__(self, predicate):
        self.predicate = predicate
        self.records = []   # (start_event, end_event, flops, (M, N, K, K2))

    def elapsed(self):
        torch.cuda.synchronize()
        ms = [r[0].elapsed_time(r[1]) for r in self.records]
        fl = [r[2] for r in self.records]
        return ms, fl

    def shapes(self):
        return [r[3] for r in self.records]


_recorder: LaunchRecorder | None = None


def set_recorder(rec: LaunchRecorder | None) -> None:
    global _recorder
    _recorder = rec


@lru_cache(maxsize=4096)
def nt_plan(M: int, N_: int, K: int, K2: int = 0, seg_end: tuple = ()) -> tuple[int, int]:
    """(tile, K ranges) the library takes for a bf16 product with a workspace (unok_gemm_nt_plan);
    tile 0 is the register-staged kernel. A function of the sizes alone."""
    code = N.lib().unok_gemm_nt_plan(N.BF16, M, N_, K, K2, len(seg_end), N.int_array(seg_end))
    return code & 15, max(1, code >> 4)


def nt_uses_256_tiles(M: int, N: int, seg_end, K: int, K2: int = 0) -> bool:
    """Whether gemm_nt runs a bf16 product (with an extension of K2 columns) on the 256x256 MFMA kernel in
    one range of K."""
    return nt_plan(M, N, K, K2, tuple(seg_end) if K2 else ()) == (1, 1)


def _rowmajor(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{name} must have unit stride along its last dimension")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a device tensor")


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def gemm_nt(a: torch.Tensor, b: torch.Tensor, *, a2: torch.Tensor | None = None,
            b2: torch.Tensor | None = None, segments: Sequence[tuple[int, int]] | None = None,
            out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
            gate: torch.Tensor | None = None, alpha: float = 1.0,
            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """out = alpha * gate (.) (a @ b.T + a2[:, seg] @ b2.T) + residual.

    a [M,K], b [N,K]; a2 [M,*], b2 [N,K2] (the LoRA extension); ``segments`` is a list of
    (n_end, a2_col) pairs: output columns < n_end (and >= the previous end) use
    a2[:, a2_col:a2_col+K2]. ``gate`` is a [M] bool/uint8 row gate on the product.
    """
    _rowmajor(a, "a")
    _rowmajor(b, "b")
    M, K = a.shape
    Nn = b.shape[0]
    if b.shape[1] != K:
        raise RuntimeError(f"gemm_nt: inner dims differ: a {tuple(a.shape)} b {tuple(b.shape)}")
    if b.dtype != a.dtype:
        raise RuntimeError("gemm_nt: a and b dtypes differ")
    out_dtype = out_dtype or (out.dtype if out is not None else a.dtype)
    if out is None:
        out = torch.empty((M, Nn), device=a.device, dtype=out_dtype)
    _rowmajor(out, "out")
    if tuple(out.shape) != (M, Nn) or out.dtype != out_dtype:
        raise RuntimeError("gemm_nt: out has the wrong shape or dtype")
    K2 = 0
    seg_end, seg_col = [], []
    if a2 is not None:
        _rowmajor(a2, "a2")
        _rowmajor(b2, "b2")
        if a2.dtype != a.dtype or b2.dtype != a.dtype:
            raise RuntimeError("gemm_nt: extension dtypes must match a")
        if a2.shape[0] != M or b2.shape[0] != Nn:
            raise RuntimeError("gemm_nt: extension operand shapes do not match M/N")
        K2 = b2.shape[1]
        segs = list(segments) if segments else [(Nn, 0)]
        for n_end, col in segs:
            if col + K2 > a2.shape[1]:
                raise RuntimeError("gemm_nt: extension segment exceeds a2 columns")
        seg_end = [s[0] for s in segs]
        seg_col = [s[1] for s in segs]
    if residual is not None:
        _rowmajor(residual, "residual")
        if tuple(residual.shape) != (M, Nn) or residual.dtype != out_dtype:
            raise RuntimeError("gemm_nt: residual must match out")
    if gate is not None:
        if gate.dtype not in (torch.bool, torch.uint8) or gate.numel() != M or not gate.is_contiguous():
            raise RuntimeError("gemm_nt: gate must be a contiguous bool/uint8 vector of length M")
    rec = _recorder
    if rec is not None and rec.predicate(a.dtype, M, Nn, K, K2, seg_end):
        ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev0.record()
    else:
        rec = None
    ranges = nt_plan(M, Nn, K, K2, tuple(seg_end))[1] if a.dtype == torch.bfloat16 and M > 0 and Nn > 0 else 1
    ws = torch.empty(ranges * M * Nn, device=a.device, dtype=torch.float32) if ranges > 1 else None
    N.call("unok_gemm_nt_ws", N.dtype_code(a.dtype), N.dtype_code(out_dtype), M, Nn, K,
           N.ptr(a), _ld(a), N.ptr(b), _ld(b),
           N.ptr(a2), _ld(a2) if a2 is not None else 0, N.ptr(b2), _ld(b2) if b2 is not None else 0, K2,
           len(seg_end), N.int_array(seg_end), N.int_array(seg_col),
           N.ptr(out), _ld(out), N.ptr(residual), _ld(residual) if residual is not None else 0,
           N.ptr(gate), float(alpha), 0, N.ptr(ws), ranges * M * Nn * 4 if ws is not None else 0, N.stream())
    if rec is not None:
        ev1.record()
        rec.records.append((ev0, ev1, 2.0 * M * Nn * (K + K2), (M, Nn, K, K2)))
    return out


def gemm_nt_rows(a: torch.Tensor, b: torch.Tensor, *, lora_a: torch.Tensor | None = None,
                 lora_b: torch.Tensor | None = None, segments: Sequence[tuple[int, int]] | None = None,
                 residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                 swiglu: bool = False, splits: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Few-row gated LoRA linear (decode and draft blocks), bf16:
    y = a b^T + h[:, seg] lora_b^T + residual with h = bf16(gate (.) a lora_a^T).

    a [M,K], b [N,K]; lora_a [R,K] (all segments' A rows), lora_b [N,r] ((alpha/r) B);
    ``segments`` is a list of (n_end, h_col) pairs: output columns < n_end (and >= the previous
    end) use h[:, h_col:h_col+r]. With ``swiglu`` the result is silu(G) * U of y = [G | U],
    [M, N/2]. ``splits`` = 0 lets the library choose the K ranges."""
    _rowmajor(a, "a")
    _rowmajor(b, "b")
    M, K = a.shape
    Nn = b.shape[0]
    if b.shape[1] != K or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise RuntimeError(f"gemm_nt_rows: bf16 a [M,K] and b [N,K] required, got {tuple(a.shape)} {tuple(b.shape)}")
    R = r = 0
    seg_end, seg_col = [], []
    if lora_a is not None:
        _rowmajor(lora_a, "lora_a")
        _rowmajor(lora_b, "lora_b")
        if lora_a.dtype != a.dtype or lora_b.dtype != a.dtype or lora_a.shape[1] != K or lora_b.shape[0] != Nn:
            raise RuntimeError("gemm_nt_rows: LoRA operands must be bf16 lora_a [R,K] and lora_b [N,r]")
        R, r = lora_a.shape[0], lora_b.shape[1]
        segs = list(segments) if segments else [(Nn, 0)]
        seg_end = [s[0] for s in segs]
        seg_col = [s[1] for s in segs]
    ncol = Nn // 2 if swiglu else Nn
    if out is None:
        out = torch.empty((M, ncol), device=a.device, dtype=a.dtype)
    _rowmajor(out, "out")
    if tuple(out.shape) != (M, ncol) or out.dtype != a.dtype:
        raise RuntimeError("gemm_nt_rows: out has the wrong shape or dtype")
    if residual is not None:
        _rowmajor(residual, "residual")
        if swiglu or tuple(residual.shape) != (M, Nn) or residual.dtype != a.dtype:
            raise RuntimeError("gemm_nt_rows: residual must match out (and is not taken with swiglu)")
    if gate is not None:
        if gate.dtype not in (torch.bool, torch.uint8) or gate.numel() != M or not gate.is_contiguous():
            raise RuntimeError("gemm_nt_rows: gate must be a contiguous bool/uint8 vector of length M")
    epi = 1 if swiglu else 0
    nbytes = N.lib().unok_gemm_nt_rows_workspace(M, Nn, K, R, epi, int(splits))
    ws = torch.empty((nbytes + 3) // 4, device=a.device, dtype=torch.float32) if nbytes > 0 else None
    N.call("unok_gemm_nt_rows", M, Nn, K, N.ptr(a), _ld(a), N.ptr(b), _ld(b),
           N.ptr(lora_a), _ld(lora_a) if lora_a is not None else 0, R,
           N.ptr(lora_b), _ld(lora_b) if lora_b is not None else 0, r,
           len(seg_end), N.int_array(seg_end), N.int_array(seg_col),
           N.ptr(out), _ld(out), N.ptr(residual), _ld(residual) if residual is not None else 0,
           N.ptr(gate), epi, int(splits), N.ptr(ws), nbytes, N.stream())
    return out


def gemm_tn(a: torch.Tensor, b: torch.Tensor, *, out: torch.Tensor | None = None,
            alpha: float = 1.0, beta: float = 0.0) -> torch.Tensor:
    """out[P,Q] (fp32) = beta * out + alpha * a[Mrows,P].T @ b[Mrows,Q] (split-K over rows)."""
    _rowmajor(a, "a")
    _rowmajor(b, "b")
    if a.shape[0] != b.shape[0] or a.dtype != b.dtype:
        raise RuntimeError("gemm_tn: operands must share rows and dtype")
    Mr, P = a.shape
    Q = b.shape[1]
    if out is None:
        out = torch.empty((P, Q), device=a.device, dtype=torch.float32)
        beta = 0.0
    _rowmajor(out, "out")
    if out.dtype != torch.float32 or tuple(out.shape) != (P, Q):
        raise RuntimeError("gemm_tn: out must be fp32 [P,Q]")
    ws_bytes = int(N.lib().unok_gemm_tn_workspace(Mr, P, Q))
    ws = torch.empty(max(ws_bytes // 4, 1), device=a.device, dtype=torch.float32)
    N.call("unok_gemm_tn", N.dtype_code(a.dtype), Mr, P, Q, N.ptr(a), _ld(a), N.ptr(b), _ld(b),
           N.ptr(out), _ld(out), float(alpha), float(beta), N.ptr(ws), ws_bytes, N.stream())
    return out


def gemm_tn_noalloc(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor, *, alpha: float = 1.0,
                    beta: float = 0.0) -> torch.Tensor:
    """As ``gemm_tn`` into an existing fp32 ``out``, with the split-K partials in the library's own
    per-device scratch array: nothing is allocated, by torch or by the library."""
    _rowmajor(a, "a")
    _rowmajor(b, "b")
    _rowmajor(out, "out")
    if a.shape[0] != b.shape[0] or a.dtype != b.dtype:
        raise RuntimeError("gemm_tn_noalloc: operands must share rows and dtype")
    Mr, P = a.shape
    Q = b.shape[1]
    if out.dtype != torch.float32 or tuple(out.shape) != (P, Q):
        raise RuntimeError("gemm_tn_noalloc: out must be fp32 [P,Q]")
    N.call("unok_gemm_tn_noalloc", N.dtype_code(a.dtype), Mr, P, Q, N.ptr(a), _ld(a), N.ptr(b), _ld(b),
           N.ptr(out), _ld(out), float(alpha), float(beta), N.stream())
    return out


# ------------------------------------------------------------------------------------------
# Row-wise kernels
# ------------------------------------------------------------------------------------------
def _contig(t: torch.Tensor, name: str) -> None:
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def rmsnorm_fwd(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor | None = None):
    """y = round(x * rsqrt(mean(x^2) + eps) * w); returns (y, rstd[M] fp32)."""
    _rowmajor(x, "x")
    M, Hd = x.shape
    if w.numel() != Hd or w.dtype != x.dtype:
        raise RuntimeError("rmsnorm: weight must match the hidden size and dtype")
    y = out if out is not None else torch.empty((M, Hd), device=x.device, dtype=x.dtype)
    rstd = torch.empty(M, device=x.device, dtype=torch.float32)
    N.call("unok_rmsnorm_fwd", N.dtype_code(x.dtype), M, Hd, N.ptr(x), _ld(x), N.ptr(w), N.ptr(y), _ld(y),
           N.ptr(rstd), float(eps), N.stream())
    return y, rstd


def rmsnorm_bwd(dy, x, w, rstd, dres=None, out=None):
    """dx = rmsnorm backward (+ dres); ``out`` may alias ``dres``."""
    for t, n in ((dy, "dy"), (x, "x")):
        _contig(t, n)
    M, Hd = x.shape
    dx = out if out is not None else torch.empty_like(x)
    if dres is not None:
        _contig(dres, "dres")
    N.call("unok_rmsnorm_bwd", N.dtype_code(x.dtype), M, Hd, N.ptr(dy), N.ptr(x), N.ptr(w), N.ptr(rstd),
           N.ptr(dres), N.ptr(dx), N.stream())
    return dx


def qknorm_rope_fwd(qkv, nq, nk, d, wq, wk, pos, inv_freq, eps, *, out_dtype=None, with_v=False):
    """Per-head q/k RMSNorm (when wq/wk are given) then RoPE; returns (q, k, rstd), or (q, k, v, rstd)
    with ``with_v`` (v: the v heads of qkv as a contiguous [M, nk*d] copy). ``out_dtype`` (default:
    qkv's) may be bf16 for an fp32 qkv: the normalisation then sees the unrounded projection."""
    _rowmajor(qkv, "qkv")
    M = qkv.shape[0]
    out_dtype = out_dtype or qkv.dtype
    q = torch.empty((M, nq * d), device=qkv.device, dtype=out_dtype)
    k = torch.empty((M, nk * d), device=qkv.device, dtype=out_dtype)
    v = torch.empty((M, nk * d), device=qkv.device, dtype=out_dtype) if with_v else None
    rstd = torch.empty((M, nq + nk), device=qkv.device, dtype=torch.float32)
    if pos.dtype != torch.int64 or pos.numel() != M:
        raise RuntimeError("qknorm_rope: pos must be int64 [M]")
    N.call("unok_qknorm_rope_fwd", N.dtype_code(out_dtype), N.dtype_code(qkv.dtype), M, nq, nk, d, N.ptr(qkv),
           _ld(qkv), N.ptr(wq), N.ptr(wk), N.ptr(pos), N.ptr(inv_freq), float(eps), N.ptr(q), N.ptr(k), N.ptr(v),
           _ld(v) if v is not None else 0, N.ptr(rstd), N.stream())
    return (q, k, v, rstd) if with_v else (q, k, rstd)


def qknorm_rope_bwd(dq, dk, qkv, nq, nk, d, wq, wk, pos, inv_freq, rstd, dqkv):
    """Writes the q and k column blocks of ``dqkv`` ([M, (nq+2nk)*d]). dq and dk share a dtype,
    dqkv's or fp32; ``qkv`` holds the pre-norm q/k columns first (the projection output, or its q/k
    block alone) in that dtype, or in bf16 beside fp32 gradients."""
    _contig(dq, "dq")
    _contig(dk, "dk")
    if dq.dtype != dk.dtype:
        raise RuntimeError("qknorm_rope_bwd: dq and dk must share a dtype")
    M = qkv.shape[0]
    N.call("unok_qknorm_rope_bwd", N.dtype_code(dqkv.dtype), N.dtype_code(dq.dtype), N.dtype_code(qkv.dtype), M, nq,
           nk, d, N.ptr(dq), N.ptr(dk), N.ptr(qkv), _ld(qkv), N.ptr(wq), N.ptr(wk), N.ptr(pos), N.ptr(inv_freq),
           N.ptr(rstd), N.ptr(dqkv), _ld(dqkv), N.stream())
    return dqkv


def rope_table(P: int, inv_freq: torch.Tensor):
    """cos / sin [P, len(inv_freq)] of fl32(p * inv_freq[j]) for positions p < P."""
    half = inv_freq.numel()
    cos = torch.empty((P, half), device=inv_freq.device, dtype=torch.float32)
    sin = torch.empty((P, half), device=inv_freq.device, dtype=torch.float32)
    N.call("unok_rope_table", P, half, N.ptr(inv_freq), N.ptr(cos), N.ptr(sin), N.stream())
    return cos, sin


def qkv_rope_fused_ok(M: int, K: int, K2: int, nq: int, nk: int, d: int, dtype, any_rows: bool = False) -> bool:
    """Whether gemm_nt_qkv_rope takes this q|k|v projection; ``any_rows``: row counts that are no
    multiple of 256 too."""
    return (dtype == torch.bfloat16 and d == 128 and (any_rows or M % 256 == 0) and (128 * (nq + 2 * nk)) % 256 == 0
            and K % 64 == 0 and K2 % 32 == 0 and M * (nq + 2 * nk) >= 256 * 2
            and (not any_rows or K2 == 0 or (nq % 2 == 0 and nk % 2 == 0)))   # the extension's segments on tiles


def gemm_nt_qkv_rope(x, w_qkv, nq, nk, wq, wk, pos, cos_tab, sin_tab, eps, *, a2=None, b2=None, segments=None,
                     want_rstd=True, want_pre=False, any_rows=False, pre_dtype=torch.bfloat16):
    """q|k|v projection (+ LoRA extension) with q/k RMSNorm + RoPE in the GEMM epilogue (bf16, head dim
    128). Returns (q, k, v, rstd or None, pre or None); ``pre`` = the pre-norm q/k columns in ``pre_dtype``
    (bf16; with ``any_rows`` also fp32). ``any_rows`` takes any number of rows; otherwise M must be a multiple
    of 256."""
    _rowmajor(x, "x")
    _rowmajor(w_qkv, "w_qkv")
    M, Kd = x.shape
    if w_qkv.shape != (128 * (nq + 2 * nk), Kd) or w_qkv.dtype != x.dtype:
        raise RuntimeError("gemm_nt_qkv_rope: w_qkv must be [128 (nq + 2 nk), K] in the dtype of x")
    for w in (wq, wk):
        if w is not None and (w.numel() != 128 or w.dtype != x.dtype):
            raise RuntimeError("gemm_nt_qkv_rope: norm weights must be [128] in the dtype of x")
    K2 = 0
    seg_end, seg_col = [], []
    if a2 is not None:
        _rowmajor(a2, "a2")
        _rowmajor(b2, "b2")
        K2 = b2.shape[1]
        if a2.dtype != x.dtype or b2.dtype != x.dtype or a2.shape[0] != M or b2.shape[0] != w_qkv.shape[0]:
            raise RuntimeError("gemm_nt_qkv_rope: a2 [M,*] and b2 [N,K2] in the dtype of x required")
        segs = list(segments) if segments else [(w_qkv.shape[0], 0)]
        for _, col in segs:
            if col + K2 > a2.shape[1]:
                raise RuntimeError("gemm_nt_qkv_rope: extension segment exceeds a2 columns")
        seg_end = [s[0] for s in segs]
        seg_col = [s[1] for s in segs]
    if not qkv_rope_fused_ok(M, Kd, K2, nq, nk, 128, x.dtype, any_rows):
        raise RuntimeError("gemm_nt_qkv_rope: shape outside the fused kernel")
    if pos.dtype != torch.int64 or pos.numel() != M:
        raise RuntimeError("gemm_nt_qkv_rope: pos must be int64 [M]")
    if pre_dtype != torch.bfloat16 and not (any_rows and pre_dtype == torch.float32):
        raise RuntimeError("gemm_nt_qkv_rope: pre is bf16, or fp32 with any_rows")
    e = dict(device=x.device, dtype=x.dtype)
    q = torch.empty((M, 128 * nq), **e)
    k = torch.empty((M, 128 * nk), **e)
    v = torch.empty((M, 128 * nk), **e)
    rstd = torch.empty((M, nq + nk), device=x.device, dtype=torch.float32) if want_rstd else None
    pre = torch.empty((M, 128 * (nq + nk)), device=x.device, dtype=pre_dtype) if want_pre else None
    Nn = w_qkv.shape[0]
    rec = _recorder
    if rec is not None and rec.predicate(x.dtype, M, Nn, Kd, K2, seg_end or [Nn]):
        ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev0.record()
    else:
        rec = None
    N.call("unok_gemm_nt_qkv_rope_any" if any_rows else "unok_gemm_nt_qkv_rope", M, Kd, nq, nk, N.ptr(x), _ld(x),
           N.ptr(w_qkv), _ld(w_qkv), N.ptr(a2), _ld(a2) if a2 is not None else 0, N.ptr(b2),
           _ld(b2) if b2 is not None else 0, K2, len(seg_end), N.int_array(seg_end), N.int_array(seg_col),
           N.ptr(wq), N.ptr(wk), N.ptr(pos), N.ptr(cos_tab), N.ptr(sin_tab), cos_tab.shape[0], float(eps), N.ptr(q),
           N.ptr(k), N.ptr(v), N.ptr(rstd), N.ptr(pre), *((int(pre_dtype == torch.float32),) if any_rows else ()),
           N.stream())
    if rec is not None:
        ev1.record()
        rec.records.append((ev0, ev1, 2.0 * M * Nn * (Kd + K2), (M, Nn, Kd, K2)))
    return q, k, v, rstd, pre


def gemm_nt_swiglu(a: torch.Tensor, b_interleaved: torch.Tensor, *, a2: torch.Tensor | None = None,
                   b2_interleaved: torch.Tensor | None = None, gu: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, any_rows: bool = False, plain_rows: bool = False) -> torch.Tensor:
    """silu(gate) * up of a @ b.T (+ a2 @ b2.T) for gate/up weight rows interleaved in blocks of 64
    (``interleave_gate_up``; b2 likewise); bf16, M and the row count of b multiples of 256, K and
    K2 = b2.shape[1] of 32 (with ``any_rows`` any M). ``plain_rows`` (with ``any_rows``): b is [gate; up] as the
    fused projection stores it (b2 stays interleaved). With ``gu`` ([M, rows]), also stores the product as
    [gate | up]."""
    if plain_rows and not any_rows:
        raise RuntimeError("gemm_nt_swiglu: plain_rows goes with any_rows")
    _rowmajor(a, "a")
    _rowmajor(b_interleaved, "b")
    M, K = a.shape
    rows = b_interleaved.shape[0]
    if b_interleaved.shape[1] != K or a.dtype != torch.bfloat16 or b_interleaved.dtype != torch.bfloat16:
        raise RuntimeError("gemm_nt_swiglu: bf16 a [M,K] and b [N,K] required")
    K2 = 0
    if a2 is not None:
        _rowmajor(a2, "a2")
        _rowmajor(b2_interleaved, "b2")
        K2 = b2_interleaved.shape[1]
        if b2_interleaved.shape[0] != rows or a2.shape[0] != M or a2.shape[1] < K2 or a2.dtype != a.dtype \
                or b2_interleaved.dtype != a.dtype:
            raise RuntimeError("gemm_nt_swiglu: a2 [M,>=K2] and b2 [N,K2] in the dtype of a required")
    if gu is not None:
        _rowmajor(gu, "gu")
        if tuple(gu.shape) != (M, rows) or gu.dtype != a.dtype:
            raise RuntimeError("gemm_nt_swiglu: gu must be [M, N] in the dtype of a")
    out = out if out is not None else torch.empty((M, rows // 2), device=a.device, dtype=a.dtype)
    _rowmajor(out, "out")
    if tuple(out.shape) != (M, rows // 2) or out.dtype != a.dtype:
        raise RuntimeError("gemm_nt_swiglu: out must be [M, N/2] in the dtype of a")
    rec = _recorder
    if rec is not None and rec.predicate(a.dtype, M, rows, K, K2, [rows]):
        ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev0.record()
    else:
        rec = None
    N.call("unok_gemm_nt_swiglu_any" if any_rows else "unok_gemm_nt_swiglu", M, rows, K, N.ptr(a), _ld(a),
           N.ptr(b_interleaved), _ld(b_interleaved), N.ptr(a2), _ld(a2) if a2 is not None else 0,
           N.ptr(b2_interleaved), _ld(b2_interleaved) if b2_interleaved is not None else 0, K2, N.ptr(out), _ld(out),
           N.ptr(gu), _ld(gu) if gu is not None else 0, *((int(plain_rows),) if any_rows else ()), N.stream())
    if rec is not None:
        ev1.record()
        rec.records.append((ev0, ev1, 2.0 * M * rows * (K + K2), (M, rows, K, K2)))
    return out


def gemm_nt_swiglu_bwd(a: torch.Tensor, b: torch.Tensor, a2: torch.Tensor | None, b2: torch.Tensor | None,
                       gu: torch.Tensor, dgu: torch.Tensor | None = None, any_rows: bool = False) -> torch.Tensor:
    """dgu = SwiGLU backward of dS = a @ b.T (+ a2 @ b2.T) against gu = [gate | up]; dS is never
    stored. bf16; M (unless ``any_rows``) and F = b.shape[0] multiples of 256."""
    for t, n in ((a, "a"), (b, "b"), (gu, "gu")):
        _rowmajor(t, n)
    M, K = a.shape
    F = b.shape[0]
    if b.shape[1] != K or tuple(gu.shape) != (M, 2 * F) or any(t.dtype != torch.bfloat16 for t in (a, b, gu)):
        raise RuntimeError("gemm_nt_swiglu_bwd: bf16 a [M,K], b [F,K] and gu [M,2F] required")
    K2 = 0
    if a2 is not None:
        _rowmajor(a2, "a2")
        _rowmajor(b2, "b2")
        K2 = b2.shape[1]
        if b2.shape[0] != F or a2.shape[0] != M or a2.shape[1] < K2 or a2.dtype != a.dtype or b2.dtype != a.dtype:
            raise RuntimeError("gemm_nt_swiglu_bwd: bf16 a2 [M,>=K2] and b2 [F,K2] required")
    dgu = dgu if dgu is not None else torch.empty((M, 2 * F), device=a.device, dtype=a.dtype)
    _rowmajor(dgu, "dgu")
    if tuple(dgu.shape) != (M, 2 * F) or dgu.dtype != a.dtype:
        raise RuntimeError("gemm_nt_swiglu_bwd: dgu must be [M, 2F] in the dtype of a")
    rec = _recorder
    if rec is not None and rec.predicate(a.dtype, M, F, K, K2, [F]):
        ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev0.record()
    else:
        rec = None
    N.call("unok_gemm_nt_swiglu_bwd_any" if any_rows else "unok_gemm_nt_swiglu_bwd", M, F, K, N.ptr(a), _ld(a), N.ptr(b), _ld(b), N.ptr(a2),
           _ld(a2) if a2 is not None else 0, N.ptr(b2), _ld(b2) if b2 is not None else 0, K2, N.ptr(gu), _ld(gu),
           N.ptr(dgu), _ld(dgu), N.stream())
    if rec is not None:
        ev1.record()
        rec.records.append((ev0, ev1, 2.0 * M * F * (K + K2), (M, F, K, K2)))
    return dgu


def swiglu_fused_ok(M: int, F: int, K: int, any_rows: bool = False) -> bool:
    """Shapes the fused gate/up + SwiGLU product accepts (F K: a tile's gate and up rows lie within the
    32-bit byte offsets of one buffer)."""
    return ((any_rows or M % 256 == 0) and (2 * F) % 256 == 0 and K % 64 == 0 and K > 0
            and (F + 128) * K * 2 <= 0xFFFFFFFF)


def interleave_gate_up(w_gu: torch.Tensor, F: int) -> torch.Tensor:
    """[gate; up] rows [2F, H] -> rows interleaved in blocks of 64 (gate 64 b.., then up 64 b..)."""
    H = w_gu.shape[1]
    g, u = w_gu[:F].reshape(F // 64, 64, H), w_gu[F:].reshape(F // 64, 64, H)
    return torch.stack((g, u), dim=1).reshape(2 * F, H).contiguous()


def swiglu_fwd(gu, F, out=None):
    _rowmajor(gu, "gu")
    M = gu.shape[0]
    out = out if out is not None else torch.empty((M, F), device=gu.device, dtype=gu.dtype)
    N.call("unok_swiglu_fwd", N.dtype_code(gu.dtype), M, F, N.ptr(gu), _ld(gu), N.ptr(out), N.stream())
    return out


def swiglu_bwd(dout, gu, F, dgu=None):
    _contig(dout, "dout")
    M = gu.shape[0]
    dgu = dgu if dgu is not None else torch.empty((M, 2 * F), device=gu.device, dtype=gu.dtype)
    N.call("unok_swiglu_bwd", N.dtype_code(gu.dtype), M, F, N.ptr(dout), N.ptr(gu), _ld(gu), N.ptr(dgu),
           _ld(dgu), N.stream())
    return dgu


def embedding(ids: torch.Tensor, table: torch.Tensor, out=None):
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        raise RuntimeError("embedding: ids must be contiguous int64")
    _contig(table, "table")
    M = ids.numel()
    out = out if out is not None else torch.empty((M, table.shape[1]), device=table.device, dtype=table.dtype)
    N.call("unok_embedding", table.element_size(), M, table.shape[1], N.ptr(ids), N.ptr(table), table.shape[0],
           N.ptr(out), N.stream())
    return out


def rows_copy(src: torch.Tensor, dst: torch.Tensor, M: int, smap=None, dmap=None):
    """dst[dmap[r]] = src[smap[r]] for r < M (maps are int32; None = identity)."""
    _rowmajor(src, "src")
    _rowmajor(dst, "dst")
    if src.dtype != dst.dtype or src.shape[1] != dst.shape[1]:
        raise RuntimeError("rows_copy: src and dst rows differ")
    for m in (smap, dmap):
        if m is not None and (m.dtype != torch.int32 or m.numel() < M):
            raise RuntimeError("rows_copy: maps must be int32 with >= M entries")
    es = src.element_size()
    N.call("unok_rows_copy", src.shape[1] * es, M, N.ptr(src), _ld(src) * es, N.ptr(smap), N.ptr(dst),
           _ld(dst) * es, N.ptr(dmap), N.stream())
    return dst


# ------------------------------------------------------------------------------------------
# Block-diffusion attention
# ------------------------------------------------------------------------------------------
def attn_fwd(q, k1, v1, iv, Hq, Hkv, D, *, k2=None, v2=None, scale=None):
    """Returns (O [Mq, Hq*D], LSE2 [Mq, Hq] fp32 = log2-sum-exp2 of the scaled scores)."""
    _rowmajor(q, "q")
    Mq = q.shape[0]
    scale = D ** -0.5 if scale is None else scale
    if iv.dtype != torch.int32 or tuple(iv.shape) != (Mq, 8):
        raise RuntimeError("attn_fwd: interval table must be int32 [Mq, 8]")
    o = torch.empty((Mq, Hq * D), device=q.device, dtype=q.dtype)
    lse = torch.empty((Mq, Hq), device=q.device, dtype=torch.float32)
    N.call("unok_attn_fwd", N.dtype_code(q.dtype), Mq, Hq, Hkv, D, N.ptr(q), _ld(q), N.ptr(k1), _ld(k1),
           N.ptr(v1), _ld(v1), N.ptr(k2), _ld(k2) if k2 is not None else 0, N.ptr(v2),
           _ld(v2) if v2 is not None else 0, N.ptr(iv), N.ptr(o), _ld(o), N.ptr(lse), float(scale), N.stream())
    return o, lse


def attn_fwd_split(q, k, v, iv, QR: int, S: int, D: int, *, scale=None):
    """Split-key attention of decode blocks: S * QR rows, row i reading query q[i % QR] (one head)
    against k / v rows over its interval iv[i]; returns (O [S*QR, D], LSE2 [S*QR] fp32)."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _rowmajor(t, nm)
    scale = D ** -0.5 if scale is None else scale
    rows = QR * S
    if iv.dtype != torch.int32 or tuple(iv.shape) != (rows, 8) or q.shape[0] < QR:
        raise RuntimeError("attn_fwd_split: int32 iv [S*QR, 8] and q [>= QR, D] required")
    o = torch.empty((rows, D), device=q.device, dtype=q.dtype)
    lse = torch.empty(rows, device=q.device, dtype=torch.float32)
    N.call("unok_attn_fwd_split", QR, S, D, N.ptr(q), _ld(q), N.ptr(k), _ld(k), N.ptr(v), _ld(v), N.ptr(iv),
           N.ptr(o), _ld(o), N.ptr(lse), float(scale), N.stream())
    return o, lse


def attn_split_combine(o, lse, dst, QR: int, S: int, D: int, out):
    """out[dst[i]] = merge of the S partial rows s * QR + i (rows with dst[i] < 0 skipped)."""
    _rowmajor(o, "o")
    _rowmajor(out, "out")
    if dst.dtype != torch.int32 or dst.numel() < QR or lse.numel() < QR * S:
        raise RuntimeError("attn_split_combine: int32 dst [QR] and lse [S*QR] required")
    N.call("unok_attn_split_combine", QR, S, D, N.ptr(o), _ld(o), N.ptr(lse), N.ptr(dst), N.ptr(out), _ld(out),
           N.stream())
    return out


def decode_prep(qkv, wq, wk, lengths, inv_freq, eps: float, kc, vc, qd, B: int, L: int, nq: int, nk: int, D: int):
    """q/k norm + RoPE of a draft block's qkv rows [B*L, (nq+2nk)*D], its K/V rows into the caches
    kc / vc [B, nk, max_len, D] at the committed lengths, its queries into qd [B*nk*128, D]."""
    _rowmajor(qkv, "qkv")
    if qkv.dtype != torch.bfloat16 or lengths.dtype != torch.int64 or not kc.is_contiguous() or not vc.is_contiguous():
        raise RuntimeError("decode_prep: bf16 qkv, int64 lengths and contiguous caches required")
    N.call("unok_decode_prep", B, L, nq, nk, D, N.ptr(qkv), _ld(qkv), N.ptr(wq), N.ptr(wk), N.ptr(lengths),
           N.ptr(inv_freq), float(eps), N.ptr(kc), N.ptr(vc), kc.shape[2], N.ptr(qd), N.stream())
    return qd


def decode_maps(lengths, B: int, L: int, nq: int, nk: int, max_len: int, S: int):
    """Key intervals [S*QR, 8] and output rows [QR] (QR = 128 B nk) of a draft block's split-key attention
    at the committed lengths."""
    if lengths.dtype != torch.int64 or lengths.numel() != B or not lengths.is_contiguous():
        raise RuntimeError("decode_maps: contiguous int64 lengths [B] required")
    QR = B * nk * 128
    ivs = torch.empty((S * QR, 8), device=lengths.device, dtype=torch.int32)
    dst = torch.empty(QR, device=lengths.device, dtype=torch.int32)
    N.call("unok_decode_maps", B, L, nq, nk, max_len, S, N.ptr(lengths), N.ptr(ivs), N.ptr(dst), N.stream())
    return ivs, dst


# ------------------------------------------------------------------------------------------
# Trees of drafted tokens over the KV cache
# ------------------------------------------------------------------------------------------
def _same_device(what: str, *tensors: torch.Tensor) -> None:
    """The operands lie on the current device, whose current stream the kernels are enqueued on."""
    dev = torch._C._cuda_getDevice() if tensors and tensors[0].is_cuda else None
    for t in tensors:
        if t.get_device() != dev:                        # (-1 for a host tensor)
            raise RuntimeError(f"{what}: operands must be on the current device, got {t.device}")


def _sizes(what: str, *sizes: int) -> None:
    """Sizes that travel as 32-bit numbers."""
    if max(sizes) >= 1 << 31:
        raise ValueError(f"{what}: sizes {sizes} exceed 2^31 - 1")


def _int64_vector(what: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.int64 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be contiguous int64 [{n}], got {t.dtype} {tuple(t.shape)}")


def _check_caches(what: str, caches: Sequence[torch.Tensor]) -> torch.Tensor:
    """Cache tensors of one shape [B, nk, max_len, D], dtype and device, contiguous; returns the first."""
    if not caches:
        raise RuntimeError(f"{what}: no cache tensors")
    c = caches[0]
    shape, dtype, device = c.shape, c.dtype, c.device
    if c.dim() != 4:
        raise RuntimeError(f"{what}: caches must be [B, nk, max_len, D], got {tuple(shape)}")
    for t in caches:
        if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
            raise RuntimeError(f"{what}: caches must be contiguous {dtype} {tuple(shape)} on {device}, got {t.dtype} "
                               f"{tuple(t.shape)} on {t.device}")
    return c


def _parents(what: str, parents: torch.Tensor, B: int) -> int:
    """Checks parents int32 [B, T] or [T]; returns the stride between their rows (0: one tree for all)."""
    if parents.dtype != torch.int32 or parents.dim() not in (1, 2) or (parents.dim() == 2 and parents.shape[0] != B) \
            or (parents.shape[-1] > 1 and parents.stride(-1) != 1):
        raise RuntimeError(f"{what}: parents must be int32 [{B}, T] or [T], got {parents.dtype} {tuple(parents.shape)}")
    return parents.stride(0) if parents.dim() == 2 and B > 1 else 0


def _tree_operands(what: str, q: torch.Tensor, B: int, nk: int, D: int, lengths: torch.Tensor,
                   parents: torch.Tensor) -> tuple[int, int, int]:
    """Checks the queries, lengths and trees of an attention over caches [B, nk, max_len, D]; returns (nq, T, parents' row stride)."""
    _int64_vector(what, "lengths", lengths, B)
    ldp = _parents(what, parents, B)
    T = parents.shape[-1]
    nq = q.shape[1] // D if D else 0
    if q.shape[0] != B * T or nk == 0 or nq == 0 or nq % nk or nq * D != q.shape[1]:
        raise RuntimeError(f"{what}: q must be [{B} * {T}, nq * {D}] with nq a multiple of {nk}, got {tuple(q.shape)}")
    return nq, T, ldp


def _tree_out(what: str, q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return q.new_empty(q.shape)
    _rowmajor(out, "out")
    if out.shape != q.shape or out.dtype != q.dtype:
        raise RuntimeError(f"{what}: out must have the shape and dtype of q")
    return out


def tree_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor, *,
              scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens over a KV cache; returns [B*T, nq*D].

    q [B*T, nq*D]: row b*T + t is node t of sequence b. k, v [B, nk, max_len, D] (any strides but the last): rows
    [0, lengths[b]) are committed, row lengths[b] + t holds node t (rows at or past max_len do not exist).
    lengths int64 [B]. parents int32 [B, T], or [T] for one tree of all sequences: the index of an earlier node,
    -1 for a root, below -1 for padding, whose output rows are 0; a parent that is no earlier node, or is padding,
    ends the chain. A node sees the committed rows, its ancestors and itself; what else the cache holds does not
    matter. ``out`` shares no row with q. ``scale`` (default D^-0.5) may be any finite number. T <= 256, D 64 or
    128, fp32 or bf16."""
    _rowmajor(q, "q")
    if k.dim() != 4 or v.shape != k.shape or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError(f"tree_attn: k and v must be [B, nk, max_len, D] in the dtype of q, got {tuple(k.shape)} "
                           f"{tuple(v.shape)}")
    B, nk, max_len, D = k.shape
    if D > 1 and (k.stride(3) != 1 or v.stride(3) != 1):
        raise RuntimeError("tree_attn: k and v must have unit stride along their last dimension")
    nq, T, ldp = _tree_operands("tree_attn", q, B, nk, D, lengths, parents)
    out = _tree_out("tree_attn", q, out)
    _same_device("tree_attn", q, k, v, lengths, parents, out)
    ks, vs = ((*t.stride()[:2], t.stride(2) if max_len > 1 else D) for t in (k, v))
    nbytes = N.lib().unok_tree_attn_workspace(N.dtype_code(q.dtype), B, T, nq, nk, D, max_len)
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes > 0 else None
    N.call("unok_tree_attn", N.dtype_code(q.dtype), B, T, nq, nk, D, N.ptr(q), _ld(q), N.ptr(k), *ks, N.ptr(v), *vs, max_len,
           N.ptr(lengths), N.ptr(parents), ldp, float(D ** -0.5 if scale is None else scale), N.ptr(out), _ld(out), N.ptr(ws),
           max(nbytes, 0), N.stream())
    return out


def tree_depths(parents: torch.Tensor) -> torch.Tensor:
    """Depth [B, T] int32 of every node of the trees ``parents`` (int32 [B, T], as tree_attn reads them): roots and
    padding 0."""
    if parents.dtype != torch.int32 or parents.dim() != 2 or not parents.is_contiguous():
        raise RuntimeError("tree_depths: contiguous int32 parents [B, T] required")
    _same_device("tree_depths", parents)
    out = torch.empty_like(parents)
    N.call("unok_tree_depths", *parents.shape, N.ptr(parents), N.ptr(out), N.stream())
    return out


def tree_prep(qkv, wq, wk, lengths, depths, inv_freq, eps: float, kc, vc, B: int, T: int, nq: int, nk: int, D: int):
    """q/k norm + RoPE of a tree's qkv rows [B*T, (nq+2nk)*D] at positions lengths + depths, its K/V rows into the
    caches kc / vc [B, nk, max_len, D] at rows lengths + t; returns the queries [B*T, nq*D]."""
    _rowmajor(qkv, "qkv")
    if qkv.dtype != torch.bfloat16 or qkv.shape != (B * T, (nq + 2 * nk) * D):
        raise RuntimeError("tree_prep: bf16 qkv [B*T, (nq+2nk)*D] required")
    _int64_vector("tree_prep", "lengths", lengths, B)
    if depths.dtype != torch.int32 or depths.shape != (B, T) or not depths.is_contiguous():
        raise RuntimeError("tree_prep: contiguous int32 depths [B, T] required")
    if _check_caches("tree_prep", (kc, vc)).shape[:2] != (B, nk) or kc.shape[3] != D or kc.dtype != qkv.dtype:
        raise RuntimeError("tree_prep: bf16 caches [B, nk, max_len, D] required")
    for w in (wq, wk):
        if w is not None and (w.numel() != D or w.dtype != qkv.dtype or not w.is_contiguous()):
            raise RuntimeError("tree_prep: norm weights must be [D] in the dtype of qkv")
    if inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2 or not inv_freq.is_contiguous():
        raise RuntimeError("tree_prep: fp32 inv_freq [D/2] required")
    q = torch.empty((B * T, nq * D), device=qkv.device, dtype=qkv.dtype)
    _same_device("tree_prep", qkv, lengths, depths, inv_freq, kc, *(w for w in (wq, wk) if w is not None))
    N.call("unok_tree_prep", B, T, nq, nk, D, N.ptr(qkv), _ld(qkv), N.ptr(wq), N.ptr(wk), N.ptr(lengths), N.ptr(depths),
           N.ptr(inv_freq), float(eps), N.ptr(kc), N.ptr(vc), kc.shape[2], N.ptr(q), N.stream())
    return q


def cache_keep(caches: Sequence[torch.Tensor], lengths: torch.Tensor, nodes: torch.Tensor, counts: torch.Tensor) -> None:
    """Keeps the accepted nodes of drafted trees: in every cache tensor ([B, nk, max_len, D], contiguous, K and V of
    all layers) row lengths[b] + nodes[b, i] moves to row lengths[b] + i for i < counts[b]. Every row is read before
    any is written. nodes int64 [B, P], P <= 256; entries whose row does not exist are skipped. The lengths
    stay as they are."""
    c = _check_caches("cache_keep", caches)
    B, nk, max_len, D = c.shape
    _int64_vector("cache_keep", "lengths", lengths, B)
    _int64_vector("cache_keep", "counts", counts, B)
    if nodes.dtype != torch.int64 or nodes.dim() != 2 or nodes.shape[0] != B or not nodes.is_contiguous():
        raise RuntimeError(f"cache_keep: nodes must be contiguous int64 [{B}, P], got {nodes.dtype} {tuple(nodes.shape)}")
    if nodes.shape[1] > 256:
        raise RuntimeError(f"cache_keep: paths hold at most 256 nodes, got {nodes.shape[1]}")
    _same_device("cache_keep", c, lengths, nodes, counts)
    N.call("unok_cache_keep", len(caches), N.ptr_array(caches), D * c.element_size(), B, nk, max_len, nodes.shape[1],
           N.ptr(lengths), N.ptr(nodes), N.ptr(counts), N.stream())


def cache_copy(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor], src_lengths: torch.Tensor,
               dst_lengths: torch.Tensor, pairs: Sequence[tuple[int, int]]) -> None:
    """Copies sequences between cache slots: for every (source slot, destination slot) of ``pairs`` and every tensor
    ([batch, nk, max_len, D], contiguous; the batch and max_len of src and dst may differ) the source's committed
    rows, as many as both caches hold, and dst_lengths[destination] becomes their number. src and dst may be the same
    tensors: then no slot is both read and written. No slot is written twice."""
    s, d = _check_caches("cache_copy", src), _check_caches("cache_copy", dst)
    if len(src) != len(dst) or s.shape[1] != d.shape[1] or s.shape[3] != d.shape[3] or s.dtype != d.dtype:
        raise RuntimeError(f"cache_copy: {len(src)} caches {s.dtype} {tuple(s.shape)} do not match {len(dst)} {d.dtype} "
                           f"{tuple(d.shape)}")
    _int64_vector("cache_copy", "source lengths", src_lengths, s.shape[0])
    _int64_vector("cache_copy", "destination lengths", dst_lengths, d.shape[0])
    _same_device("cache_copy", s, d, src_lengths, dst_lengths)
    if any(len(pair) != 2 for pair in pairs):
        raise RuntimeError("cache_copy: pairs must be (source slot, destination slot)")
    flat = [int(i) for pair in pairs for i in pair]
    if flat and not (0 <= min(flat[::2]) and max(flat[::2]) < s.shape[0] and 0 <= min(flat[1::2]) and max(flat[1::2]) < d.shape[0]):
        raise ValueError(f"cache_copy: slots {list(pairs)} of batches {s.shape[0]} -> {d.shape[0]}")
    N.call("unok_cache_copy", len(src), N.ptr_array(src), N.ptr_array(dst), s.shape[3] * s.element_size(), s.shape[1],
           s.shape[0], s.shape[2], d.shape[0], d.shape[2], N.ptr(src_lengths), N.ptr(dst_lengths), len(pairs),
           N.int_array(flat), N.stream())


# ------------------------------------------------------------------------------------------
# KV caches in 4 bits
# ------------------------------------------------------------------------------------------
class Rows4(NamedTuple):
    """A cache tensor in 4 bits: codes uint8 [B, nk, max_len, D/2] and scales uint8 [B, nk, max_len, D/32], contiguous.

    32 consecutive elements share the scale 2^(byte - 127), the least power of two of which the largest magnitude is below
    seven; an element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 scales (codes 0 .. 7, ties to the even one, bit 3 the sign; the
    even element is its byte's low half). An infinity or NaN makes its 32 elements NaN (byte 255)."""
    codes: torch.Tensor
    scales: torch.Tensor


def _check_caches4(what: str, caches: Sequence[Rows4]) -> tuple[int, int, int, int]:
    """4-bit caches of one shape; returns (B, nk, max_len, D)."""
    if not caches:
        raise RuntimeError(f"{what}: no cache tensors")
    first, fscales = caches[0]
    shape, sshape = first.shape, fscales.shape
    if len(shape) != 4 or shape[3] not in (32, 64) or sshape != (*shape[:3], shape[3] // 16):
        raise RuntimeError(f"{what}: uint8 codes [B, nk, max_len, D/2] and scales [B, nk, max_len, D/32] of D 64 or 128 required, "
                           f"got {tuple(shape)} and {tuple(sshape)}")
    for c, s in caches:
        if c.dtype != torch.uint8 or s.dtype != torch.uint8 or not c.is_contiguous() or not s.is_contiguous() \
                or (c is not first and (c.shape != shape or s.shape != sshape)) or (s is not fscales and s.shape != sshape):
            raise RuntimeError(f"{what}: caches must be contiguous uint8 codes {tuple(shape)} and scales {tuple(sshape)}, got "
                               f"{c.dtype} {tuple(c.shape)} and {s.dtype} {tuple(s.shape)}")
    return shape[0], shape[1], shape[2], 2 * shape[3]


def cache4_store(rows: Sequence[torch.Tensor], caches: Sequence[Rows4], starts: torch.Tensor) -> None:
    """Puts rows into 4-bit caches (see Rows4): row b*T + t of each of ``rows`` ([B*T, nk*D], fp32 or bf16, rows on 16 bytes)
    becomes cache row starts[b] + t of its cache; rows that the cache does not have are skipped. starts int64 [B]."""
    if len(rows) != len(caches):
        raise RuntimeError(f"cache4_store: {len(rows)} tensors for {len(caches)} caches")
    B, nk, max_len, D = _check_caches4("cache4_store", caches)
    _int64_vector("cache4_store", "starts", starts, B)
    shape, dtype = rows[0].shape, rows[0].dtype
    for x in rows:
        _rowmajor(x, "cache4_store: rows")
        if x.shape != shape or x.dtype != dtype:
            raise RuntimeError(f"cache4_store: rows must be of one shape and type, got {dtype} {tuple(shape)} and {x.dtype} "
                               f"{tuple(x.shape)}")
    M, width = shape
    if width != nk * D or (M % B if B else M):
        raise RuntimeError(f"cache4_store: rows must be [{B} * T, {nk * D}], got {tuple(shape)}")
    codes, scales = [c.codes for c in caches], [c.scales for c in caches]
    _same_device("cache4_store", starts, *rows, *codes, *scales)
    T = M // B if B else 0
    _sizes("cache4_store", B, T, nk, max_len)
    N.call("unok_cache4_store", N.dtype_code(dtype), len(rows), N.ptr_array(rows), N.int64_array([_ld(x) for x in rows]),
           N.ptr_array(codes), N.ptr_array(scales), B, T, nk, D, max_len, N.ptr(starts), N.stream())


def cache4_load(caches: Sequence[Rows4], starts: torch.Tensor, T: int, dtype: torch.dtype = torch.bfloat16) -> list[torch.Tensor]:
    """The numbers that rows starts[b] .. starts[b] + T - 1 of 4-bit caches stand for, [B*T, nk*D] each (fp32 or bf16, both exact);
    rows that the cache does not have are zeros."""
    B, nk, max_len, D = _check_caches4("cache4_load", caches)
    _int64_vector("cache4_load", "starts", starts, B)
    code = N.dtype_code(dtype)
    if T < 0:
        raise ValueError(f"cache4_load: {T} rows")
    _sizes("cache4_load", B, T, nk, max_len)
    codes, scales = [c.codes for c in caches], [c.scales for c in caches]
    _same_device("cache4_load", starts, *codes, *scales)
    rows = [starts.new_empty((B * T, nk * D), dtype=dtype) for _ in caches]
    N.call("unok_cache4_load", code, len(rows), N.ptr_array(rows), N.int64_array([nk * D] * len(rows)), N.ptr_array(codes),
           N.ptr_array(scales), B, T, nk, D, max_len, N.ptr(starts), N.stream())
    return rows


def tree_attn4(q: torch.Tensor, k: Rows4, v: Rows4, lengths: torch.Tensor, parents: torch.Tensor, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``tree_attn`` over caches in 4 bits (Rows4): the same queries, trees, lengths and output; fp32 or bf16 queries over either."""
    _rowmajor(q, "q")
    B, nk, max_len, D = _check_caches4("tree_attn4", (k, v))
    nq, T, ldp = _tree_operands("tree_attn4", q, B, nk, D, lengths, parents)
    out = _tree_out("tree_attn4", q, out)
    _same_device("tree_attn4", q, *k, *v, lengths, parents, out)
    _sizes("tree_attn4", B, T, nq, max_len)
    code = N.dtype_code(q.dtype)
    nbytes = N.lib().unok_tree_attn4_workspace(code, B, T, nq, nk, D, max_len)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes > 0 else None
    N.call("unok_tree_attn4", code, B, T, nq, nk, D, N.ptr(q), _ld(q), N.ptr(k.codes), N.ptr(k.scales), N.ptr(v.codes),
           N.ptr(v.scales), max_len, N.ptr(lengths), N.ptr(parents), ldp, float(D ** -0.5 if scale is None else scale), N.ptr(out),
           _ld(out), N.ptr(ws), max(nbytes, 0), N.stream())
    return out


# ------------------------------------------------------------------------------------------
# Verification of drafted tokens
# ------------------------------------------------------------------------------------------
def _verify_operands(what: str, z: torch.Tensor, rows: int, u: torch.Tensor, shape: tuple[int, int],
                     temperature: float | torch.Tensor) -> tuple[float, torch.Tensor | None]:
    """Checks logits, random numbers and temperature; returns the temperature for the library."""
    _rowmajor(z, f"{what}: logits")
    if z.shape[0] != rows or z.shape[1] == 0:
        raise RuntimeError(f"{what}: logits must be [{rows}, V], got {tuple(z.shape)}")
    N.dtype_code(z.dtype)
    if u.dtype != torch.float32 or tuple(u.shape) != shape or not u.is_contiguous():
        raise RuntimeError(f"{what}: u must be contiguous fp32 {shape}, got {u.dtype} {tuple(u.shape)}")
    _sizes(what, *shape, z.shape[1])
    if not torch.is_tensor(temperature):
        if not 0 <= temperature < float("inf"):
            raise ValueError(f"{what}: temperature {temperature} must be finite and not negative")
        return float(temperature), None
    if temperature.dtype != torch.float32 or tuple(temperature.shape) != shape[:1] or not temperature.is_contiguous():
        raise RuntimeError(f"{what}: temperatures must be contiguous fp32 {shape[:1]}, got {temperature.dtype} "
                           f"{tuple(temperature.shape)}")
    return 0.0, temperature


def verify_draft(logits: torch.Tensor, draft_logits: torch.Tensor | None, tokens: torch.Tensor, u: torch.Tensor, *,
                 counts: torch.Tensor | None = None, temperature: float | torch.Tensor = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens against the target's logits: (accepted int64 [B], next token int64 [B]).

    logits [B*(L+1), V] (fp32 or bf16): row b*(L+1) + i is the target's at drafted token i of tokens int64 [B, L], the last
    one behind them all. draft_logits [B*L, V] of the same type: what each token was drawn from at the same temperature; None
    for tokens that were chosen, not drawn. counts int64 [B]: sequence b drafted its first counts[b] tokens only (its rows
    behind counts[b] are not read). u fp32 [B, L+1] in [0, 1).

    Token i is accepted while u[b, i] < p_i / q_i (of its target and draft probability; q_i = 1 without draft_logits). The next token
    is drawn at u[b, L]: at the refused token from max(p - q, 0), so that every token is distributed as the target says, or from p
    behind the last. Drawing takes the lowest token at which the distribution function exceeds u (below 0: as 0; 1 and above: the last
    token with a probability), all in fp64. temperature: a number or
    fp32 [B]; 0 accepts what the target's largest logit says, and takes that (draft_logits are not read). A row of logits with
    a NaN or +inf, or of -inf alone, ends its sequence there, and the next token is -1."""
    if tokens.dtype != torch.int64 or tokens.dim() != 2 or not tokens.is_contiguous():
        raise RuntimeError(f"verify_draft: tokens must be contiguous int64 [B, L], got {tokens.dtype} {tuple(tokens.shape)}")
    B, L = tokens.shape
    temp, temps = _verify_operands("verify_draft", logits, B * (L + 1), u, (B, L + 1), temperature)
    if draft_logits is not None:
        _rowmajor(draft_logits, "verify_draft: draft_logits")
        if tuple(draft_logits.shape) != (B * L, logits.shape[1]) or draft_logits.dtype != logits.dtype:
            raise RuntimeError(f"verify_draft: draft_logits must be {logits.dtype} {(B * L, logits.shape[1])}, got "
                               f"{draft_logits.dtype} {tuple(draft_logits.shape)}")
    if counts is not None:
        _int64_vector("verify_draft", "counts", counts, B)
    _same_device("verify_draft", logits, tokens, u, *(t for t in (draft_logits, counts, temps) if t is not None))
    V, code = logits.shape[1], N.dtype_code(logits.dtype)
    accepted, token = tokens.new_empty(B), tokens.new_empty(B)
    nbytes = N.lib().unok_verify_draft_workspace(code, B, L, V)
    ws = tokens.new_empty(max(nbytes, 0), dtype=torch.uint8)
    N.call("unok_verify_draft", code, B, L, V, N.ptr(logits), _ld(logits), N.ptr(draft_logits),
           _ld(draft_logits) if draft_logits is not None else 0, N.ptr(tokens), N.ptr(counts), N.ptr(u), temp, N.ptr(temps),
           N.ptr(accepted), N.ptr(token), N.ptr(ws), nbytes, N.stream())
    return accepted, token


def verify_tree(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, u: torch.Tensor, *,
                temperature: float | torch.Tensor = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Follows drafted trees along tokens drawn from the target's logits: (nodes int64 [B, T], counts int64 [B], next token int64
    [B]), the first two as ``cache_keep`` takes them.

    logits [B*T, V] (fp32 or bf16): row b*T + t is node t's. tokens int64 [B, T] and parents int32 [B, T] (or [T]) as tree_attn
    reads them; T <= 256. From node 0, the one root that counts, the token drawn at a node (at u fp32 [B, T], in [0, 1)) leads
    to its first child that holds it; the next token is what was drawn at the path's end, and nodes are -1 behind the path. Every
    token is distributed as the target says, whatever the tree holds. With T = 1 this samples one token for each row. Drawing,
    temperature and rows without a distribution (which end the path, next token -1) as in ``verify_draft``. A sequence whose node
    0 is padding has the count 0 and the next token -1."""
    if tokens.dtype != torch.int64 or tokens.dim() != 2 or not tokens.is_contiguous() or tokens.shape[1] == 0:
        raise RuntimeError(f"verify_tree: tokens must be contiguous int64 [B, T], got {tokens.dtype} {tuple(tokens.shape)}")
    B, T = tokens.shape
    ldp = _parents("verify_tree", parents, B)
    if parents.shape[-1] != T:
        raise RuntimeError(f"verify_tree: parents {tuple(parents.shape)} do not match the tokens {(B, T)}")
    temp, temps = _verify_operands("verify_tree", logits, B * T, u, (B, T), temperature)
    _same_device("verify_tree", logits, tokens, parents, u, *(() if temps is None else (temps,)))
    V, code = logits.shape[1], N.dtype_code(logits.dtype)
    nodes, counts, token = torch.empty_like(tokens), tokens.new_empty(B), tokens.new_empty(B)
    nbytes = N.lib().unok_verify_tree_workspace(code, B, T, V)
    ws = tokens.new_empty(max(nbytes, 0), dtype=torch.uint8)
    N.call("unok_verify_tree", code, B, T, V, N.ptr(logits), _ld(logits), N.ptr(tokens), N.ptr(parents), ldp, N.ptr(u), temp,
           N.ptr(temps), N.ptr(nodes), N.ptr(counts), N.ptr(token), N.ptr(ws), nbytes, N.stream())
    return nodes, counts, token


def row_top_k(z: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The k <= 256 largest values of each row of z [R, V] (fp32 or bf16) in descending order: (values [R, k] fp32,
    columns [R, k] int64, log-sum-exp [R] fp32 of the whole row). Equal values: the lower column first; NaN counts as
    larger than every number."""
    _rowmajor(z, "z")
    R, V = z.shape
    _same_device("row_top_k", z)
    _sizes("row_top_k", R, V)
    if not 1 <= k <= min(256, V):
        raise ValueError(f"row_top_k: k={k} must lie in [1, min(256, V={V})]")
    values = torch.empty((R, k), device=z.device, dtype=torch.float32)
    cols = torch.empty((R, k), device=z.device, dtype=torch.int64)
    lse = torch.empty(R, device=z.device, dtype=torch.float32)
    nbytes = N.lib().unok_row_topk_workspace(R, V, k)
    ws = torch.empty(nbytes, device=z.device, dtype=torch.uint8) if nbytes > 0 else None
    N.call("unok_row_topk", N.dtype_code(z.dtype), R, V, k, N.ptr(z), _ld(z), N.ptr(values), N.ptr(cols), N.ptr(lse),
           N.ptr(ws), nbytes, N.stream())
    return values, cols, lse


def attn_bwd_qknorm(q, k1, v1, iv, o, lse, do, Hq, Hkv, D, k2, v2, pre, rstd, wq, wk, pos, cos_tab, sin_tab, dqkv,
                    scale=None):
    """Noisy-stream backward with the q/k RMSNorm + RoPE backward in the dQ / dK epilogues (bf16): writes
    the gradient before the norm into the q and k column blocks of ``dqkv`` and dV into its v block."""
    Mq = q.shape[0]
    scale = D ** -0.5 if scale is None else scale
    _contig(do, "do")
    _rowmajor(pre, "pre")
    _rowmajor(dqkv, "dqkv")
    if q.dtype != torch.bfloat16 or pre.dtype not in (torch.bfloat16, torch.float32) or dqkv.dtype != torch.bfloat16:
        raise RuntimeError("attn_bwd_qknorm: bf16 only (pre: bf16 or fp32)")
    if pre.shape != (Mq, (Hq + Hkv) * D) or dqkv.shape != (Mq, (Hq + 2 * Hkv) * D) or k2.shape[0] != Mq:
        raise RuntimeError("attn_bwd_qknorm: pre [Mq, (Hq+Hkv) D], dqkv [Mq, (Hq+2Hkv) D] and Mq keys required")
    if pos.dtype != torch.int64 or pos.numel() != Mq:
        raise RuntimeError("attn_bwd_qknorm: pos must be int64 [Mq]")
    dsum = torch.empty((Mq, Hq), device=q.device, dtype=torch.float32)
    N.call("unok_attn_bwd_qknorm" if pre.dtype == torch.bfloat16 else "unok_attn_bwd_qknorm_f32", Mq, Hq, Hkv, D,
           N.ptr(q), _ld(q), N.ptr(k1), _ld(k1), N.ptr(v1), _ld(v1),
           N.ptr(k2), _ld(k2), N.ptr(v2), _ld(v2), N.ptr(iv), N.ptr(o), _ld(o), N.ptr(lse), N.ptr(do), _ld(do),
           N.ptr(dsum), N.ptr(pre), _ld(pre), N.ptr(rstd), N.ptr(wq), N.ptr(wk), N.ptr(pos), N.ptr(cos_tab),
           N.ptr(sin_tab), cos_tab.shape[0], N.ptr(dqkv), _ld(dqkv), float(scale), N.stream())
    return dqkv


def attn_bwd(q, k1, v1, iv, o, lse, do, Hq, Hkv, D, *, k2=None, v2=None, ivk=None, dk=None, dv=None,
             scale=None, grad_dtype=None):
    """Returns dQ; writes dK/dV of source-2 keys into ``dk``/``dv`` when given. ``grad_dtype`` (default
    q's) is the dtype of dQ and dK, fp32 allowed for bf16 inputs; dV has q's dtype."""
    Mq = q.shape[0]
    scale = D ** -0.5 if scale is None else scale
    grad_dtype = grad_dtype or q.dtype
    _contig(do, "do")
    if dk is not None and dk.dtype != grad_dtype:
        raise RuntimeError("attn_bwd: dk must have the gradient dtype")
    dq = torch.empty((Mq, Hq * D), device=q.device, dtype=grad_dtype)
    dsum = torch.empty((Mq, Hq), device=q.device, dtype=torch.float32)
    Mk2 = k2.shape[0] if k2 is not None else 0
    N.call("unok_attn_bwd", N.dtype_code(q.dtype), N.dtype_code(grad_dtype), Mq, Mk2, Hq, Hkv, D, N.ptr(q), _ld(q),
           N.ptr(k1), _ld(k1),
           N.ptr(v1), _ld(v1), N.ptr(k2), _ld(k2) if k2 is not None else 0, N.ptr(v2),
           _ld(v2) if v2 is not None else 0, N.ptr(iv), N.ptr(ivk), N.ptr(o), _ld(o), N.ptr(lse), N.ptr(do),
           _ld(do), N.ptr(dsum), N.ptr(dq), _ld(dq), N.ptr(dk), _ld(dk) if dk is not None else 0, N.ptr(dv),
           _ld(dv) if dv is not None else 0, float(scale), N.stream())
    return dq
