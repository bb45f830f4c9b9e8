"""Torch-facing W8A8 operators over the C ABI.

These are the host-side mirror of the op the reference runs at every
projection of a streamed decoder layer: ``nn.Linear`` inside HF
``LlamaDecoderLayer`` (created at adapters/_llama.py:80, called at
adapters/_llama.py:245-250), wrapped by ``LoRAWrapper.forward``
(_lora.py:23-26). The quantised operator is defined in include/lema_b200.h:

* ``quantize_rows``      per-row symmetric int8 (per token / per output channel)
* ``w8a8_gemm``          int8 x int8 -> s32 (tcgen05) + dequant/bias/bf16 epilogue
* ``w8a8_linear``        differentiable y = x W^T (+ b) with straight-through
                         backward dx = dy . (wq * sw) through ``w8a8_dgrad``
* ``grouped_w8a8_gemm``  the same per expert over pre-sorted token ranges

and of the losses over the head's logits (each with a ``*_grad`` form that returns the
logits' gradient in the same call):

* ``token_logprobs``     log-probability of each target token, differentiable
* ``preference_loss``    pairs of chosen / rejected sequences
* ``policy_loss``        clipped policy ratios with a KL term
* ``distill_loss``       a teacher's top logits

All tensors must live on a CUDA device; there is no CPU fallback. Calls run
on the current torch stream of the tensors' device.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import _native as N


class GemmTimer:
    """Optional timing of every int8 GEMM launch (for the bench's roofline): the
    library records a pre-created CUDA event pair around each launch on its
    stream (``lema_gemm_timer_start`` / ``lema_gemm_timer_stop``), so a timed
    step runs the same fused entry points as an untimed one."""

    enabled = False
    max_records = 1 << 16
    dropped = 0

    @classmethod
    def enable(cls, on: bool = True) -> None:
        if on:
            N.call("lema_gemm_timer_start", cls.max_records)
        elif cls.enabled:
            cls.summary()
        cls.enabled = on

    @classmethod
    def summary(cls) -> tuple[float, float, int]:
        """(total ops, total ms, launches) over the recorded GEMMs since
        ``enable()`` (synchronises; recording stops)."""
        ops_, ms = C.c_double(0.0), C.c_double(0.0)
        n, dropped = C.c_int64(0), C.c_int64(0)
        N.call("lema_gemm_timer_stop", C.byref(ops_), C.byref(ms), C.byref(n), C.byref(dropped))
        cls.enabled = False
        cls.dropped = dropped.value
        return ops_.value, ms.value, n.value


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _require_cuda(*ts: torch.Tensor | None) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "lema_b200 ops run only on CUDA tensors (no CPU fallback); got a tensor on "
                f"{t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} vs {t.device}")
    if dev is None:
        raise RuntimeError("no tensor given")
    return dev


def _rows_view(t: torch.Tensor) -> torch.Tensor:
    """2-D view with unit stride along the last dim (copies only if needed)."""
    if t.dim() != 2:
        raise ValueError(f"expected a 2-D tensor, got shape {tuple(t.shape)}")
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))


def pad_to(n: int, m: int) -> int:
    return (n + m - 1) // m * m


# ---------------------------------------------------------------------------
# K1: quantisation
# ---------------------------------------------------------------------------

def quantize_rows(x: torch.Tensor, out: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None, ldq: int | None = None
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row int8 quantisation of a bf16 or fp32 [R, C] tensor.

    Returns (q int8 [R, C] (a view of an [R, ldq] buffer), scale fp32 [R]).
    ``ldq`` defaults to C rounded up to 16 so the result can feed the GEMM.
    """
    dev = _require_cuda(x)
    x = _rows_view(x)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"quantize_rows takes bf16 or fp32, got {x.dtype}")
    rows, cols = x.shape
    if ldq is None:
        ldq = pad_to(max(cols, 1), 16)
    if out is None:
        buf = torch.empty(rows, ldq, dtype=torch.int8, device=dev)
        if ldq > cols:
            buf[:, cols:].zero_()
    else:
        buf = out
        if buf.dtype != torch.int8 or buf.shape[0] != rows or buf.stride(1) != 1:
            raise ValueError("out must be int8 [rows, >=cols] with unit column stride")
        ldq = buf.stride(0) if rows > 1 else ldq
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    fn = "lema_quantize_rows" if x.dtype == torch.bfloat16 else "lema_quantize_rows_f32"
    N.call(fn, _ptr(x), rows, cols, _ld(x), _ptr(buf), ldq, _ptr(scale), _stream(dev))
    return buf[:, :cols], scale


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-output-channel int8 quantisation of an nn.Linear weight [N, K].

    Returns (wq int8 [N, K] with row stride padded to 16, sw fp32 [N]).
    """
    if w.dtype not in (torch.bfloat16, torch.float32):
        w = w.to(torch.bfloat16)
    return quantize_rows(w)


# ---------------------------------------------------------------------------
# K2+K3: int8 GEMM with fused epilogue
# ---------------------------------------------------------------------------

def w8a8_gemm(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
              bias: torch.Tensor | None = None, want_y: bool = True, want_acc: bool = False,
              out: torch.Tensor | None = None):
    """y[M,N] = bf16((acc * sx[m]) * sw[n] + bias[n]), acc = xq . wq^T (exact s32).

    Returns y, or (y, acc) when ``want_acc`` (y is None if not ``want_y``).
    """
    dev = _require_cuda(xq, sx, wq, sw, bias)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise TypeError("xq and wq must be int8")
    M, K = xq.shape
    Nn, K2 = wq.shape
    if K2 != K:
        raise ValueError(f"K mismatch: {K} vs {K2}")
    if xq.stride(1) != 1 or wq.stride(1) != 1:
        raise ValueError("xq and wq need unit column stride")
    sx = sx.contiguous().float()
    sw = sw.contiguous().float()
    if bias is not None:
        bias = bias.contiguous().to(torch.bfloat16)
    y = None
    if want_y:
        y = out if out is not None else torch.empty(M, Nn, dtype=torch.bfloat16, device=dev)
    acc = torch.empty(M, Nn, dtype=torch.int32, device=dev) if want_acc else None
    N.call("lema_w8a8_gemm", _ptr(xq), _ld(xq), _ptr(sx), _ptr(wq), _ld(wq), _ptr(sw),
           _ptr(bias), _ptr(y), Nn if y is None else _ld(y), _ptr(acc), Nn, M, Nn, K,
           _stream(dev))
    if want_acc:
        return y, acc
    return y


def w8a8_linear_forward(x2d: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
                        bias: torch.Tensor | None = None) -> torch.Tensor:
    """K1 + K2/K3 on a bf16 [M, K] input: the forward of one W8A8 projection."""
    dev = _require_cuda(x2d, wq, sw, bias)
    x2d = _rows_view(x2d)
    if x2d.dtype != torch.bfloat16:
        raise TypeError("w8a8 forward takes bf16 activations")
    M, K = x2d.shape
    Nn = wq.shape[0]
    if wq.shape[1] != K:
        raise ValueError(f"weight in_features {wq.shape[1]} != input features {K}")
    ldq = pad_to(max(K, 1), 16)
    xq = torch.empty(M, ldq, dtype=torch.int8, device=dev)
    sx = torch.empty(M, dtype=torch.float32, device=dev)
    y = torch.empty(M, Nn, dtype=torch.bfloat16, device=dev)
    if bias is not None:
        bias = bias.contiguous().to(torch.bfloat16)
    N.call("lema_w8a8_linear_fwd", _ptr(x2d), _ld(x2d), _ptr(wq), _ld(wq), _ptr(sw),
           _ptr(bias), _ptr(y), Nn, _ptr(xq), ldq, _ptr(sx), M, Nn, K, _stream(dev))
    return y


# ---------------------------------------------------------------------------
# K4: backward of the frozen base
# ---------------------------------------------------------------------------

def dequant_transpose(wq: torch.Tensor, sw: torch.Tensor) -> torch.Tensor:
    """wdT[K, ldt] bf16 with wdT[k, n] = bf16(float(wq[n, k]) * sw[n]); returns [K, N] view."""
    dev = _require_cuda(wq, sw)
    Nn, K = wq.shape
    ldt = pad_to(max(Nn, 1), 8)
    wdT = torch.empty(K, ldt, dtype=torch.bfloat16, device=dev)
    N.call("lema_dequant_transpose", _ptr(wq), _ld(wq), _ptr(sw.contiguous().float()), Nn, K,
           _ptr(wdT), ldt, _stream(dev))
    return wdT[:, :Nn]


def quantize_rows_colscaled(x: torch.Tensor, cs: torch.Tensor
                            ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of fp32(x[r, c]) * cs[c] (bf16 x, fp32 cs) quantised per row:
    (q int8 [R, C] view of an [R, ldq] buffer, scale fp32 [R])."""
    dev = _require_cuda(x, cs)
    x = _rows_view(x).to(torch.bfloat16)
    rows, cols = x.shape
    ldq = pad_to(max(cols, 1), 16)
    buf = torch.empty(rows, ldq, dtype=torch.int8, device=dev)
    if ldq > cols:
        buf[:, cols:].zero_()
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    N.call("lema_quantize_rows_colscaled", _ptr(x), _ptr(cs.contiguous().float()), rows, cols,
           _ld(x), _ptr(buf), ldq, _ptr(scale), _stream(dev))
    return buf[:, :cols], scale


def transpose_i8(wq: torch.Tensor) -> torch.Tensor:
    """wqT[K, N] = wq[N, K] for int8 (a view of a [K, round_up(N, 16)] buffer)."""
    dev = _require_cuda(wq)
    wq = _rows_view(wq)
    if wq.dtype != torch.int8:
        raise TypeError("transpose_i8 takes int8")
    Nn, K = wq.shape
    ldt = pad_to(max(Nn, 1), 16)
    out = torch.zeros(K, ldt, dtype=torch.int8, device=dev)
    N.call("lema_transpose_i8", _ptr(wq), _ld(wq), Nn, K, _ptr(out), ldt, _stream(dev))
    return out[:, :Nn]


def bf16_gemm_tn(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """y = bf16(a . b^T) with fp32 accumulation (tcgen05 kind::f16)."""
    dev = _require_cuda(a, b)
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise TypeError("bf16 operands required")
    a = _rows_view(a)
    b = _rows_view(b)
    M, K = a.shape
    Nn = b.shape[0]
    y = torch.empty(M, Nn, dtype=torch.bfloat16, device=dev)
    N.call("lema_bf16_gemm_tn", _ptr(a), _ld(a), _ptr(b), _ld(b), _ptr(y), Nn, M, Nn, K,
           _stream(dev))
    return y


# Straight-through dgrad of the frozen W8A8 projections: "bf16" (the contract:
# dy . bf16(wq * sw) with fp32 accumulation) or the opt-in "int8" variant
# (dy * sw quantised per row, int8 GEMM with wq^T; looser tolerance).
_DGRAD_MODE = "bf16"


def set_dgrad_mode(mode: str) -> None:
    global _DGRAD_MODE
    if mode not in ("bf16", "int8"):
        raise ValueError(f"dgrad mode must be 'bf16' or 'int8', not {mode!r}")
    _DGRAD_MODE = mode


def dgrad_mode() -> str:
    return _DGRAD_MODE


def w8a8_dgrad_int8(dy: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor) -> torch.Tensor:
    """dx[M, K] ~ dy[M, N] . (wq * sw): dy * sw quantised per row to int8, int8
    GEMM with the transposed int8 weight, dx = bf16(sd[m] * acc)."""
    dev = _require_cuda(dy, wq, sw)
    dy = _rows_view(dy).to(torch.bfloat16)
    M, Nn = dy.shape
    K = wq.shape[1]
    ld = pad_to(max(Nn, 1), 16)
    wqT = torch.empty(K, ld, dtype=torch.int8, device=dev)
    dq = torch.empty(M, ld, dtype=torch.int8, device=dev)
    if ld > Nn:
        wqT[:, Nn:].zero_()
        dq[:, Nn:].zero_()
    sd = torch.empty(M, dtype=torch.float32, device=dev)
    dx = torch.empty(M, K, dtype=torch.bfloat16, device=dev)
    N.call("lema_w8a8_dgrad_int8", _ptr(dy), _ld(dy), _ptr(wq), _ld(wq),
           _ptr(sw.contiguous().float()), _ptr(dx), K, _ptr(wqT), ld, _ptr(dq), ld, _ptr(sd),
           M, Nn, K, _stream(dev))
    return dx


def w8a8_dgrad(dy: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor) -> torch.Tensor:
    """dx[M, K] = bf16(dy[M, N] . wdeq[N, K]), wdeq = bf16(wq * sw) (straight-through);
    the int8 variant when ``set_dgrad_mode("int8")`` is in effect."""
    if _DGRAD_MODE == "int8":
        return w8a8_dgrad_int8(dy, wq, sw)
    dev = _require_cuda(dy, wq, sw)
    dy = _rows_view(dy)
    if dy.dtype != torch.bfloat16:
        dy = dy.to(torch.bfloat16)
    if (dy.stride(0) * 2) % 16 != 0 or dy.data_ptr() % 16 != 0:
        # TMA needs 16-byte row pitch: re-lay dy out with a padded pitch.
        M0, N0 = dy.shape
        buf = torch.zeros(M0, pad_to(N0, 8), dtype=torch.bfloat16, device=dev)
        buf[:, :N0] = dy
        dy = buf[:, :N0]
    M, Nn = dy.shape
    K = wq.shape[1]
    ldt = pad_to(max(Nn, 1), 8)
    ws = torch.empty(K, ldt, dtype=torch.bfloat16, device=dev)
    dx = torch.empty(M, K, dtype=torch.bfloat16, device=dev)
    N.call("lema_w8a8_dgrad", _ptr(dy), _ld(dy), _ptr(wq), _ld(wq), _ptr(sw.contiguous().float()),
           _ptr(dx), K, _ptr(ws), ldt, M, Nn, K, _stream(dev))
    return dx


# ---------------------------------------------------------------------------
# K6: grouped W8A8 GEMM (MoE experts)
# ---------------------------------------------------------------------------

def grouped_w8a8_gemm(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
                      offsets: list[int], bias: torch.Tensor | None = None) -> torch.Tensor:
    """Per-expert W8A8 GEMM. xq [T, K] rows sorted by expert, wq [E, N, K], sw [E, N],
    offsets: E+1 host ints (rows of expert e are offsets[e]:offsets[e+1])."""
    dev = _require_cuda(xq, sx, wq, sw, bias)
    E, Nn, K = wq.shape
    if len(offsets) != E + 1:
        raise ValueError("offsets must have E+1 entries")
    if wq.stride(2) != 1 or wq.stride(0) != Nn * wq.stride(1):
        raise ValueError("expert weights must be stacked contiguously: [E, N, ldw]")
    T = xq.shape[0]
    y = torch.empty(T, Nn, dtype=torch.bfloat16, device=dev)
    offs = (C.c_int64 * (E + 1))(*[int(o) for o in offsets])
    if bias is not None:
        bias = bias.contiguous().to(torch.bfloat16)
    args = ("lema_grouped_w8a8_gemm", _ptr(xq), _ld(xq), _ptr(sx.contiguous().float()),
            _ptr(wq), wq.stride(1), _ptr(sw.contiguous().float()), _ptr(bias), _ptr(y), Nn,
            offs, E, Nn, K, _stream(dev))
    N.call(*args)
    return y


# ---------------------------------------------------------------------------
# Differentiable linear
# ---------------------------------------------------------------------------

class _W8A8LinearFn(torch.autograd.Function):
    """y = W8A8(x); dx = dy . (wq * sw) (STE through both quantisers); no dW (frozen base)."""

    @staticmethod
    def forward(ctx, x2d, wq, sw, bias):
        y = w8a8_linear_forward(x2d, wq, sw, bias)
        ctx.save_for_backward(wq, sw)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        wq, sw = ctx.saved_tensors
        dx = w8a8_dgrad(dy, wq, sw) if ctx.needs_input_grad[0] else None
        dbias = None
        if ctx.has_bias and ctx.needs_input_grad[3]:
            dbias = dy.float().sum(0).to(torch.bfloat16)
        return dx, None, None, dbias


class _W8A8TrainableFn(torch.autograd.Function):
    """W8A8 forward of a trainable projection (the int8 copy of its current true
    weight); backward: straight-through dx and the fp32 weight gradient
    dW = dy^T . x, added into ``sink.wgrad_acc``."""

    @staticmethod
    def forward(ctx, x2d, wq, sw, sink):
        y = w8a8_linear_forward(x2d, wq, sw, None)
        ctx.save_for_backward(x2d, wq, sw)
        ctx.sink = sink
        return y

    @staticmethod
    def backward(ctx, dy):
        x2d, wq, sw = ctx.saved_tensors
        dx = w8a8_dgrad(dy, wq, sw) if ctx.needs_input_grad[0] else None
        ctx.sink.wgrad_acc.add_(w8a8_wgrad(dy, x2d))
        return dx, None, None, None


def w8a8_linear_trainable(x: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, sink) -> torch.Tensor:
    K = x.shape[-1]
    lead = x.shape[:-1]
    x2d = x.reshape(-1, K)
    if x2d.dtype != torch.bfloat16:
        x2d = x2d.to(torch.bfloat16)
    return _W8A8TrainableFn.apply(x2d, wq, sw, sink).reshape(*lead, wq.shape[0])


def w8a8_linear(x: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """Functional W8A8 linear over [..., K] -> [..., N] (bf16 compute, input dtype out)."""
    K = x.shape[-1]
    lead = x.shape[:-1]
    in_dtype = x.dtype
    x2d = x.reshape(-1, K)
    if x2d.dtype != torch.bfloat16:
        x2d = x2d.to(torch.bfloat16)
    y = _W8A8LinearFn.apply(x2d, wq, sw, bias)
    y = y.reshape(*lead, wq.shape[0])
    if in_dtype != torch.bfloat16 and in_dtype.is_floating_point:
        y = y.to(in_dtype)
    return y


def _offsets_array(offsets) -> tuple[C.Array, int]:
    offs = [int(o) for o in offsets]
    return (C.c_int64 * len(offs))(*offs), len(offs) - 1


def grouped_w8a8_dgrad(dy: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
                       offsets: list[int]) -> torch.Tensor:
    """Per-expert straight-through dgrad: rows of expert e get dy . bf16(wq[e] * sw[e]).
    dy [T, N] bf16 sorted by expert, wq [E, N, K] int8, sw [E, N]. The int8-dy
    variant when ``set_dgrad_mode("int8")`` is in effect."""
    if _DGRAD_MODE == "int8":
        return grouped_w8a8_dgrad_int8(dy, wq, sw, offsets)
    dev = _require_cuda(dy, wq, sw)
    dy = _rows_view(dy.to(torch.bfloat16))
    E, Nn, K = wq.shape
    if wq.stride(2) != 1 or wq.stride(0) != Nn * wq.stride(1):
        raise ValueError("expert weights must be stacked contiguously: [E, N, ldw]")
    offs, E2 = _offsets_array(offsets)
    if E2 != E:
        raise ValueError("offsets must have E+1 entries")
    ldt = pad_to(max(Nn, 1), 8)
    ws = torch.empty(E, K, ldt, dtype=torch.bfloat16, device=dev)
    T = dy.shape[0]
    dx = torch.empty(T, K, dtype=torch.bfloat16, device=dev)
    N.call("lema_grouped_w8a8_dgrad", _ptr(dy), _ld(dy), _ptr(wq), wq.stride(1),
           _ptr(sw.contiguous().float()), _ptr(dx), K, _ptr(ws), ldt, offs, E, Nn, K,
           _stream(dev))
    return dx


def grouped_w8a8_dgrad_int8(dy: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
                            offsets: list[int]) -> torch.Tensor:
    """Per-expert int8-dy dgrad: the rows of expert e, dy * sw[e], quantised per
    row (column-scaled quantiser), wq[e] transposed in int8, then one grouped int8
    GEMM with unit column scales: dx ~ dy . (wq[e] * sw[e]). Experts without rows
    are skipped."""
    dev = _require_cuda(dy, wq, sw)
    dy = _rows_view(dy.to(torch.bfloat16))
    E, Nn, K = wq.shape
    if wq.stride(2) != 1 or wq.stride(0) != Nn * wq.stride(1):
        raise ValueError("expert weights must be stacked contiguously: [E, N, ldw]")
    offs, E2 = _offsets_array(offsets)
    if E2 != E:
        raise ValueError("offsets must have E+1 entries")
    bounds = [int(o) for o in offsets]
    T = dy.shape[0]
    ld = pad_to(max(Nn, 1), 16)
    dq = torch.empty(T, ld, dtype=torch.int8, device=dev)
    wqT = torch.empty(E, K, ld, dtype=torch.int8, device=dev)
    if ld > Nn:
        dq[:, Nn:].zero_()
        wqT[:, :, Nn:].zero_()
    sd = torch.empty(T, dtype=torch.float32, device=dev)
    swc = sw.contiguous().float()
    stream = _stream(dev)
    lddy = _ld(dy)
    for e in range(E):
        r0, r1 = bounds[e], bounds[e + 1]
        if r1 <= r0:
            continue
        N.call("lema_quantize_rows_colscaled", dy.data_ptr() + r0 * lddy * 2,
               swc[e].data_ptr(), r1 - r0, Nn, lddy, dq.data_ptr() + r0 * ld, ld,
               sd.data_ptr() + r0 * 4, stream)
        N.call("lema_transpose_i8", wq[e].data_ptr(), wq.stride(1), Nn, K, wqT[e].data_ptr(), ld,
               stream)
    dx = torch.empty(T, K, dtype=torch.bfloat16, device=dev)
    N.call("lema_grouped_w8a8_gemm", _ptr(dq), ld, _ptr(sd), _ptr(wqT), ld, None, None,
           _ptr(dx), K, offs, E, K, Nn, stream)
    return dx


def grouped_bf16_gemm_tn(a: torch.Tensor, b: torch.Tensor, offsets: list[int]) -> torch.Tensor:
    """Rows [offsets[e], offsets[e+1]) of a times b[e]^T; a [T, K], b [E, N, K] bf16."""
    dev = _require_cuda(a, b)
    a = _rows_view(a)
    E, Nn, K = b.shape
    offs, E2 = _offsets_array(offsets)
    if E2 != E:
        raise ValueError("offsets must have E+1 entries")
    y = torch.empty(a.shape[0], Nn, dtype=torch.bfloat16, device=dev)
    N.call("lema_grouped_bf16_gemm_tn", _ptr(a), _ld(a), _ptr(b), b.stride(1), _ptr(y), Nn,
           offs, E, Nn, K, _stream(dev))
    return y


def bf16_gemm_tn_f32(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """fp32 y = a . b^T (bf16 operands, fp32 accumulators returned as is)."""
    dev = _require_cuda(a, b)
    a = _rows_view(a.to(torch.bfloat16))
    b = _rows_view(b.to(torch.bfloat16))
    M, K = a.shape
    Nn = b.shape[0]
    y = torch.empty(M, Nn, dtype=torch.float32, device=dev)
    N.call("lema_bf16_gemm_tn_f32", _ptr(a), _ld(a), _ptr(b), _ld(b), _ptr(y), Nn, M, Nn, K,
           _stream(dev))
    return y


def w8a8_wgrad(dy: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """Straight-through weight gradient of a W8A8 projection: dW[N, K] = dy^T . x
    (bf16 inputs, fp32 accumulation) for dy [M, N], x [M, K]."""
    dyt = dy.to(torch.bfloat16).t().contiguous()
    xt = x.to(torch.bfloat16).t().contiguous()
    K = xt.shape[0]
    if (dyt.shape[1] * 2) % 16 != 0:  # TMA row pitch: pad the token dimension
        M8 = pad_to(dyt.shape[1], 8)
        dyt = torch.nn.functional.pad(dyt, (0, M8 - dyt.shape[1]))
        xt = torch.nn.functional.pad(xt, (0, M8 - xt.shape[1]))
    return bf16_gemm_tn_f32(dyt, xt) if K else torch.zeros(dyt.shape[0], 0, device=dy.device)


# ---------------------------------------------------------------------------
# Fused producers of the decoder block (RMSNorm -> quantise, RoPE, SwiGLU ->
# quantise) and the autograd functions of the fused block path
# ---------------------------------------------------------------------------

def rmsnorm_quant(x2d: torch.Tensor, g: torch.Tensor, eps: float, want_q: bool = True):
    """(hn bf16 [M, H], xq int8 [M, H] | None, sx fp32 [M] | None, rstd fp32 [M])."""
    dev = _require_cuda(x2d, g)
    x2d = _rows_view(x2d)
    M, H = x2d.shape
    hn = torch.empty(M, H, dtype=torch.bfloat16, device=dev)
    rstd = torch.empty(M, dtype=torch.float32, device=dev)
    xq = sx = None
    if want_q:
        xq = torch.empty(M, pad_to(H, 16), dtype=torch.int8, device=dev)[:, :H]
        sx = torch.empty(M, dtype=torch.float32, device=dev)
    N.call("lema_rmsnorm_quant", _ptr(x2d), _ld(x2d), _ptr(g.contiguous()), M, H, float(eps),
           _ptr(hn), H, _ptr(xq), (xq.stride(0) if xq is not None else 0), _ptr(sx), _ptr(rstd),
           _stream(dev))
    return hn, xq, sx, rstd


def rmsnorm_bwd(x2d, g, rstd, dhn):
    dev = _require_cuda(x2d, g, rstd, dhn)
    x2d, dhn = _rows_view(x2d), _rows_view(dhn.to(torch.bfloat16))
    M, H = x2d.shape
    dx = torch.empty(M, H, dtype=torch.bfloat16, device=dev)
    N.call("lema_rmsnorm_bwd", _ptr(x2d), _ld(x2d), _ptr(g.contiguous()), _ptr(rstd), _ptr(dhn),
           _ld(dhn), M, H, _ptr(dx), H, _stream(dev))
    return dx


def _rope_tables(cos: torch.Tensor, sin: torch.Tensor, seq: int, d: int) -> None:
    """The kernel reads rows 0 .. seq - 1 of both tables."""
    if min(cos.numel(), sin.numel()) < seq * d:
        raise ValueError(f"cos and sin must have [{seq}, {d}] elements at least, got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")


def rope(q2d, k2d, cos, sin, seq: int, hq: int, hk: int, d: int, mode: int = 0):
    """Rotary embedding of q [T, hq*d] and k [T, hk*d] rows (may be strided);
    cos/sin [seq, d] bf16. Returns contiguous (q_out, k_out)."""
    _rope_tables(cos, sin, seq, d)
    dev = _require_cuda(q2d, k2d, cos, sin)
    T = q2d.shape[0]
    qo = torch.empty(T, hq * d, dtype=torch.bfloat16, device=dev)
    ko = torch.empty(T, hk * d, dtype=torch.bfloat16, device=dev)
    N.call("lema_rope", _ptr(q2d), q2d.stride(0), _ptr(k2d), k2d.stride(0),
           _ptr(cos.contiguous()), _ptr(sin.contiguous()), T, seq, hq, hk, d, _ptr(qo), _ptr(ko),
           mode, _stream(dev))
    return qo, ko


def swiglu_quant(gu: torch.Tensor, want_m: bool = False):
    """Rows of [gate | up] -> (mq int8 [M, I], sm fp32 [M], m bf16 [M, I] | None)."""
    dev = _require_cuda(gu)
    M, I2 = gu.shape
    I = I2 // 2
    mq = torch.empty(M, pad_to(I, 16), dtype=torch.int8, device=dev)[:, :I]
    sm = torch.empty(M, dtype=torch.float32, device=dev)
    m = torch.empty(M, I, dtype=torch.bfloat16, device=dev) if want_m else None
    N.call("lema_swiglu_quant", _ptr(gu), gu.stride(0), M, I, _ptr(mq), mq.stride(0), _ptr(sm),
           _ptr(m), I, _stream(dev))
    return mq, sm, m


# ---------------------------------------------------------------------------
# Selective full fine-tuning: fused AdamW step + re-quantisation
# ---------------------------------------------------------------------------

def adamw_coefficients(step: int, lr: float, wd: float, beta1: float = 0.9,
                       beta2: float = 0.999, eps: float = 1e-8) -> tuple[float, ...]:
    """The fp32 scalars of one AdamW step as the reference forms them
    (src/lema/_full_ft.py:204-229; Python doubles rounded once to fp32):
    (decay, beta1, c1, beta2, c2, sqrt_bc2, step_size, eps)."""
    import numpy as np
    b1 = 1 - beta1 ** step
    b2 = 1 - beta2 ** step
    f = np.float32
    decay = f(1 - lr * wd) if wd else f(1.0)
    return tuple(float(x) for x in (decay, f(beta1), f(1 - beta1), f(beta2), f(1 - beta2),
                                    f(math.sqrt(b2)), f(-(lr / b1)), f(eps)))


def adamw_requant_rows(w: torch.Tensor, g: torch.Tensor, m: torch.Tensor, v: torch.Tensor,
                       step: int, lr: float, wd: float, zero_grad: bool = True
                       ) -> tuple[torch.Tensor, torch.Tensor]:
    """One AdamW step of a [N, K] weight in place (w bf16, g / m / v fp32 on the
    device; g cleared when ``zero_grad``) fused with the per-output-channel int8
    quantisation of the new weight: returns (wq [N, K] view of [N, round_up(K, 16)],
    sw [N])."""
    dev = _require_cuda(w, g, m, v)
    if w.dtype != torch.bfloat16 or g.dtype != torch.float32 or m.dtype != torch.float32 \
            or v.dtype != torch.float32:
        raise TypeError("adamw_requant_rows takes bf16 w and fp32 g, m, v")
    for t in (w, g, m, v):
        if t.dim() != 2 or t.stride(1) != 1:
            raise ValueError("2-D tensors with unit column stride required")
    if m.stride(0) != v.stride(0) or not (w.shape == g.shape == m.shape == v.shape):
        raise ValueError("w, g, m, v must have one shape (m and v one row stride)")
    rows, cols = w.shape
    ldq = pad_to(max(cols, 1), 16)
    q = torch.empty(rows, ldq, dtype=torch.int8, device=dev)
    if ldq > cols:
        q[:, cols:].zero_()
    sw = torch.empty(rows, dtype=torch.float32, device=dev)
    N.call("lema_adamw_requant_rows", _ptr(w), _ld(w), _ptr(g), _ld(g), _ptr(m), _ptr(v),
           _ld(m), rows, cols, *adamw_coefficients(step, lr, wd), int(zero_grad), _ptr(q), ldq,
           _ptr(sw), _stream(dev))
    return q[:, :cols], sw


def swiglu_bwd(gu: torch.Tensor, dm: torch.Tensor) -> torch.Tensor:
    dev = _require_cuda(gu, dm)
    dm = _rows_view(dm.to(torch.bfloat16))
    M, I2 = gu.shape
    dgu = torch.empty(M, I2, dtype=torch.bfloat16, device=dev)
    N.call("lema_swiglu_bwd", _ptr(gu), gu.stride(0), _ptr(dm), _ld(dm), M, I2 // 2, _ptr(dgu),
           I2, _stream(dev))
    return dgu


def gemm_from_quant(xq, sx, wq, sw) -> torch.Tensor:
    """bf16 y = W8A8 GEMM of already-quantised rows (xq, sx) with (wq, sw)."""
    dev = _require_cuda(xq, wq)
    M, K = xq.shape
    Nn = wq.shape[0]
    y = torch.empty(M, Nn, dtype=torch.bfloat16, device=dev)
    N.call("lema_w8a8_gemm", _ptr(xq), _ld(xq), _ptr(sx), _ptr(wq), _ld(wq), _ptr(sw), None,
           _ptr(y), Nn, None, Nn, M, Nn, K, _stream(dev))
    return y


class RMSNormQuantFn(torch.autograd.Function):
    """hn = RMSNorm(x) (bf16 rounding of HF LlamaRMSNorm) plus its int8 rows."""

    @staticmethod
    def forward(ctx, x2d, g, eps):
        hn, xq, sx, rstd = rmsnorm_quant(x2d, g, eps)
        ctx.save_for_backward(x2d, g, rstd)
        ctx.mark_non_differentiable(xq, sx)
        return hn, xq, sx

    @staticmethod
    def backward(ctx, dhn, _dxq, _dsx):
        x2d, g, rstd = ctx.saved_tensors
        return rmsnorm_bwd(x2d, g, rstd, dhn), None, None


class QKVFn(torch.autograd.Function):
    """Stacked q/k/v W8A8 projection of pre-quantised rows; returns (q, k, v) views.
    Backward: one straight-through dgrad over the concatenated gradients."""

    @staticmethod
    def forward(ctx, hn, xq, sx, wq, sw, nq, nk):
        y = gemm_from_quant(xq, sx, wq, sw)
        ctx.save_for_backward(wq, sw)
        ctx.split = (nq, nk)
        return y[:, :nq], y[:, nq:nq + nk], y[:, nq + nk:]

    @staticmethod
    def backward(ctx, dq, dk, dv):
        wq, sw = ctx.saved_tensors
        nq, nk = ctx.split
        rows = next(g for g in (dq, dk, dv) if g is not None).shape[0]
        parts = []
        for g, n in ((dq, nq), (dk, nk), (dv, wq.shape[0] - nq - nk)):
            parts.append(g if g is not None else
                         torch.zeros(rows, n, dtype=torch.bfloat16, device=wq.device))
        dy = torch.cat([p.to(torch.bfloat16) for p in parts], dim=1)
        return w8a8_dgrad(dy, wq, sw), None, None, None, None, None, None


class RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q2d, k2d, cos, sin, seq, hq, hk, d):
        ctx.save_for_backward(cos, sin)
        ctx.meta = (seq, hq, hk, d)
        return rope(q2d, k2d, cos, sin, seq, hq, hk, d, 0)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin = ctx.saved_tensors
        seq, hq, hk, d = ctx.meta
        dqi, dki = rope(dq.contiguous().to(torch.bfloat16), dk.contiguous().to(torch.bfloat16),
                        cos, sin, seq, hq, hk, d, 1)
        return dqi, dki, None, None, None, None, None, None


class MLPFn(torch.autograd.Function):
    """down(silu(gate) * up) with stacked [gate; up] W8A8 weights: gate_up GEMM on the
    pre-quantised RMSNorm rows, fused SwiGLU -> quantise, down GEMM. Backward:
    straight-through dgrads around the SwiGLU backward kernel."""

    @staticmethod
    def forward(ctx, hn, xq, sx, wq_gu, sw_gu, wq_dn, sw_dn):
        gu = gemm_from_quant(xq, sx, wq_gu, sw_gu)
        mq, sm, _ = swiglu_quant(gu)
        y = gemm_from_quant(mq, sm, wq_dn, sw_dn)
        ctx.save_for_backward(gu, wq_gu, sw_gu, wq_dn, sw_dn)
        return y

    @staticmethod
    def backward(ctx, dy):
        gu, wq_gu, sw_gu, wq_dn, sw_dn = ctx.saved_tensors
        dm = w8a8_dgrad(dy, wq_dn, sw_dn)
        dgu = swiglu_bwd(gu, dm)
        return w8a8_dgrad(dgu, wq_gu, sw_gu), None, None, None, None, None, None


def rope_qkv(q2d, k2d, v2d, q_add, k_add, v_add, cos, sin, seq, hq, hk, d):
    """Forward RoPE of q and k plus the contiguous copy of v, each after adding its
    optional LoRA output (bf16 rounding). Returns contiguous (q_out, k_out, v_out)."""
    _rope_tables(cos, sin, seq, d)
    dev = _require_cuda(q2d, k2d, v2d, cos, sin)
    T = q2d.shape[0]
    qo = torch.empty(T, hq * d, dtype=torch.bfloat16, device=dev)
    ko = torch.empty(T, hk * d, dtype=torch.bfloat16, device=dev)
    vo = torch.empty(T, hk * d, dtype=torch.bfloat16, device=dev)
    adds = [None if t is None else t.contiguous().to(torch.bfloat16) for t in (q_add, k_add, v_add)]
    N.call("lema_rope_qkv", _ptr(q2d), q2d.stride(0), _ptr(k2d), k2d.stride(0), _ptr(v2d),
           v2d.stride(0), _ptr(adds[0]), _ptr(adds[1]), _ptr(adds[2]), _ptr(cos.contiguous()),
           _ptr(sin.contiguous()), T, seq, hq, hk, d, _ptr(qo), _ptr(ko), _ptr(vo), 0,
           _stream(dev))
    return qo, ko, vo


class RopeQKVFn(torch.autograd.Function):
    """(q + lq, k + lk) rotated and v + lv made contiguous in one kernel."""

    @staticmethod
    def forward(ctx, q, k, v, lq, lk, lv, cos, sin, seq, hq, hk, d):
        ctx.save_for_backward(cos, sin)
        ctx.meta = (seq, hq, hk, d)
        ctx.has_add = (lq is not None, lk is not None, lv is not None)
        return rope_qkv(q, k, v, lq, lk, lv, cos, sin, seq, hq, hk, d)

    @staticmethod
    def backward(ctx, dq, dk, dv):
        cos, sin = ctx.saved_tensors
        seq, hq, hk, d = ctx.meta
        dqi, dki = rope(dq.contiguous().to(torch.bfloat16), dk.contiguous().to(torch.bfloat16),
                        cos, sin, seq, hq, hk, d, 1)
        dv = dv.contiguous()
        hq_, hk_, hv_ = ctx.has_add
        return (dqi, dki, dv, dqi if hq_ else None, dki if hk_ else None, dv if hv_ else None,
                None, None, None, None, None, None)


def attention_fwd(q2d: torch.Tensor, k2d: torch.Tensor, v2d: torch.Tensor, B: int, S: int,
                  H: int, Hkv: int, scale: float):
    """Causal attention on the tcgen05 kernel: q2d [B*S, H*128], k2d / v2d
    [B*S, Hkv*128] token-major bf16 -> (o [B*S, H*128] bf16, lse [B, H, S] fp32
    log2-domain log-sum-exp of the scaled scores)."""
    dev = _require_cuda(q2d, k2d, v2d)
    q2d, k2d, v2d = (_rows_view(t) for t in (q2d, k2d, v2d))
    o = torch.empty(B * S, H * 128, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=dev)
    N.call("lema_attn_fwd", _ptr(q2d), _ld(q2d), _ptr(k2d), _ld(k2d), _ptr(v2d), _ld(v2d),
           _ptr(o), H * 128, _ptr(lse), B, S, H, Hkv, 128, float(scale), _stream(dev))
    return o, lse


def attention_bwd(q2d, k2d, v2d, o2d, lse, dout2d, B: int, S: int, H: int, Hkv: int,
                  scale: float, split_heads: bool = True):
    """(dq [B*S, H*128], dk, dv [B*S, Hkv*128]) of attention_fwd. With GQA the
    library may split dK / dV per query head through a workspace (when the kv
    heads alone would leave SMs idle); ``split_heads=False`` withholds it."""
    dev = _require_cuda(q2d, k2d, v2d, o2d, lse, dout2d)
    q2d, k2d, v2d, o2d = (_rows_view(t) for t in (q2d, k2d, v2d, o2d))
    dout2d = _rows_view(dout2d.to(torch.bfloat16))
    dq = torch.empty(B * S, H * 128, dtype=torch.bfloat16, device=dev)
    dk = torch.empty(B * S, Hkv * 128, dtype=torch.bfloat16, device=dev)
    dv = torch.empty(B * S, Hkv * 128, dtype=torch.bfloat16, device=dev)
    delta = torch.empty(B, H, S, dtype=torch.float32, device=dev)
    ws = (torch.empty(2 * B * S * H * 128, dtype=torch.float32, device=dev)
          if H != Hkv and split_heads else None)
    N.call("lema_attn_bwd", _ptr(q2d), _ld(q2d), _ptr(k2d), _ld(k2d), _ptr(v2d), _ld(v2d),
           _ptr(o2d), _ld(o2d), _ptr(dout2d), _ld(dout2d), _ptr(lse.contiguous()), _ptr(delta),
           _ptr(ws), _ptr(dq), H * 128, _ptr(dk), Hkv * 128, _ptr(dv), Hkv * 128, B, S, H, Hkv,
           128, float(scale), _stream(dev))
    n_sm = torch.cuda.get_device_properties(dev).multi_processor_count
    if ws is not None and B * Hkv * -(-S // 128) < n_sm:
        N.kernel_launches += 1  # the library split dK/dV per query head: the reduce kernel
    return dq, dk, dv


class AttentionFn(torch.autograd.Function):
    """Causal attention (head_dim 128, GQA) on the tcgen05 kernels over the
    token-major q [B*S, H*128], k / v [B*S, Hkv*128]; returns o [B*S, H*128]."""

    @staticmethod
    def forward(ctx, q2d, k2d, v2d, B, S, H, Hkv, scale):
        o, lse = attention_fwd(q2d, k2d, v2d, B, S, H, Hkv, scale)
        ctx.save_for_backward(q2d, k2d, v2d, o, lse)
        ctx.meta = (B, S, H, Hkv, scale)
        return o

    @staticmethod
    def backward(ctx, do):
        q2d, k2d, v2d, o, lse = ctx.saved_tensors
        dq, dk, dv = attention_bwd(q2d, k2d, v2d, o, lse, do, *ctx.meta)
        return dq, dk, dv, None, None, None, None, None


# ---------------------------------------------------------------------------
# Losses over vocabulary logits: token log-probabilities, preference pairs,
# clipped policy, distillation from a teacher's top logits
# ---------------------------------------------------------------------------

class _Logits:
    """Logits [..., V] as the sequences of rows the kernels address, with the
    checks every loss makes. Copies only when the last stride is not 1 or the
    leading dimensions cannot be seen as [sequences, rows]."""

    __slots__ = ("t", "dev", "lead", "n0", "n1", "V", "args")

    def __init__(self, logits: torch.Tensor):
        if not logits.is_cuda:
            _require_cuda(logits)
        dtype = logits.dtype
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            raise TypeError(f"logits must be bf16 or fp32, got {dtype}")
        shape = logits.shape
        V = shape[-1] if len(shape) > 1 else 0
        if V < 1:
            raise ValueError(f"logits must be [..., V] with V >= 1, got shape {tuple(shape)}")
        self.lead = shape[:-1]
        self.V = V
        self.dev = logits.device
        t = logits
        if len(shape) == 2:
            t = t[None]
        elif len(shape) > 3:
            t = t.reshape(math.prod(shape[:-2]), shape[-2], V)
        st = t.stride()
        if st[2] != 1 and V > 1:
            t = t.contiguous()
            st = t.stride()
        self.t = t
        self.n0, self.n1 = t.shape[0], t.shape[1]
        self.args = (t.data_ptr(), 1 if dtype is torch.float32 else 0, self.n0, self.n1, st[0],
                     st[1], V)

    def per_row(self, t: torch.Tensor | None, name: str, dtype: torch.dtype):
        """A contiguous [rows] companion of the logits, on their device."""
        if t is None:
            return None
        if t.device != self.dev:
            raise RuntimeError(f"{name} on {t.device}, logits on {self.dev}")
        if t.dtype is not dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.shape != self.lead:
            raise ValueError(f"{name} must have shape {tuple(self.lead)}, got {tuple(t.shape)}")
        if t.requires_grad:
            raise ValueError(f"{name} is a constant of the loss: detach it")
        return t.contiguous()

    def grad_out(self, logits: torch.Tensor, out: torch.Tensor | None):
        """(gradient tensor, its pointer, its two row strides)."""
        if out is None:
            # the quickest of torch's allocations, here and below: a short call is their sum
            out = (torch.empty_like(logits) if logits.is_contiguous()
                   else torch.empty(logits.shape, dtype=logits.dtype, device=self.dev))
            return out, (out.data_ptr(), self.n1 * self.V, self.V)
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != self.dev:
            raise ValueError("out must have the logits' shape, type and device")
        if out.requires_grad:
            raise ValueError("out must not require grad: detach it")
        same = (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride())
        if out.untyped_storage().data_ptr() == logits.untyped_storage().data_ptr() \
                and out.numel() and not same:
            raise ValueError("out shares the logits' storage without being the logits")
        if not _rows_disjoint(out):
            raise ValueError("out needs a unit last stride and rows that do not overlap")
        if same and self.t.data_ptr() != logits.data_ptr():
            raise ValueError("out: these logits have to be copied, so out cannot be they")
        torch.autograd.graph.increment_version(out)
        view = out
        if out.dim() > 3:
            view = out.view(self.n0, self.n1, self.V)
        elif out.dim() == 2:
            view = out[None]
        return out, (view.data_ptr(), view.stride(0), view.stride(1))

    def workspace(self, more: int = 0):
        """(scratch, its bytes for the call); `more` bytes behind those, 8-byte aligned."""
        n = _loss_workspace_bytes(self.n0, self.n1)
        return torch.empty(n + more, dtype=torch.uint8, device=self.dev), n

    def scalar(self):
        return torch.empty_strided((), (), dtype=torch.float32, device=self.dev)

    def call(self, name: str, *args) -> None:
        """One entry point on the logits' device and its current stream."""
        index = self.dev.index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                N.call(name, *self.args, *args, _raw_stream(index))
        else:
            N.call(name, *self.args, *args, _raw_stream(index))


_NO_GRAD = (None, 0, 0)


@functools.lru_cache(maxsize=256)
def _loss_workspace_bytes(n0: int, n1: int) -> int:
    n = N.lib().lema_loss_workspace_bytes(n0, n1)
    if n < 0:
        raise ValueError("more than 2^31 - 1 rows of logits")
    return n


# The current stream's handle without a Stream object around it, where torch offers that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


def _rows_disjoint(t: torch.Tensor) -> bool:
    """Unit stride along the last dimension and no two elements at one address."""
    if t.numel() == 0:
        return True
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return False
    extent = t.shape[-1]
    for size, stride in sorted(((t.shape[d], t.stride(d)) for d in range(t.dim() - 1)
                                if t.shape[d] > 1), key=lambda p: p[1]):
        if stride < extent:
            return False
        extent = stride * (size - 1) + extent
    return True


def _targets(x: _Logits, targets: torch.Tensor) -> torch.Tensor:
    return x.per_row(targets, "targets", torch.int64)


def _logprobs_bwd(logits, targets, ignore_index, temperature, stats, dlogps, upstream=None):
    x = _Logits(logits)
    dx, where = x.grad_out(logits, None)
    x.call("lema_token_logprobs_bwd", targets.data_ptr(), ignore_index, temperature,
           stats.data_ptr(), dlogps.data_ptr(), _ptr(upstream), *where)
    return dx


def _first_order(backward):
    """An autograd backward that has no derivative of its own. Only a graph that is to be
    differentiated again pays for saying so."""
    once = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _logprobs_fwd(logits, targets, temperature, ignore_index, want_stats):
    x = _Logits(logits)
    targets = _targets(x, targets)
    logps = torch.empty_like(targets, dtype=torch.float32)
    stats = (torch.empty(x.n0, x.n1, 2, dtype=torch.float32, device=x.dev) if want_stats
             else None)
    x.call("lema_token_logprobs", targets.data_ptr(), ignore_index, temperature,
           logps.data_ptr(), _ptr(stats))
    return logps, targets, stats


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, ignore_index):
        logps, targets, stats = _logprobs_fwd(logits, targets, temperature, ignore_index, True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.meta = (temperature, ignore_index)
        return logps

    @staticmethod
    @_first_order
    def backward(ctx, dlogps):
        logits, targets, stats = ctx.saved_tensors
        temperature, ignore_index = ctx.meta
        return _logprobs_bwd(logits, targets, ignore_index, temperature, stats,
                             dlogps.contiguous()), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0,
                   ignore_index: int = -100) -> torch.Tensor:
    """log softmax(logits / temperature) at ``targets``: logits [..., V] bf16 or
    fp32, targets [...] int64 -> fp32 [...] (0 where the target is ``ignore_index``;
    those rows are not read). Differentiable in the logits. ``targets`` are aligned
    with the logits: position t holds the token the row predicts."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogprobsFn.apply(logits, targets, float(temperature), int(ignore_index))
    return _logprobs_fwd(logits, targets, float(temperature), int(ignore_index), False)[0]


def _preference(logits, targets, ref_logps, beta, label_smoothing, ignore_index, grad_scale, out,
                want_dx):
    x = _Logits(logits)
    if logits.dim() != 3 or x.n0 % 2 or x.n0 == 0:
        raise ValueError("preference_loss takes logits [2 P, S, V]: P chosen sequences, then "
                         "their P rejected ones")
    targets = _targets(x, targets)
    ref = x.per_row(ref_logps, "ref_logps", torch.float32)
    T = x.n0 * x.n1
    # statistics (pairs, 8-byte aligned), log-probabilities, coefficients: for a backward, or
    # for this call alone
    ws, n = x.workspace(16 * T if want_dx else 0)
    saved = None if want_dx else torch.empty(4 * T, dtype=torch.float32, device=x.dev)
    rewards = torch.empty(x.n0, dtype=torch.float32, device=x.dev)
    loss = x.scalar()
    dx, where = x.grad_out(logits, out) if want_dx else (None, _NO_GRAD)
    at = ws.data_ptr() + n if want_dx else saved.data_ptr()
    x.call("lema_preference_loss", targets.data_ptr(), int(ignore_index), _ptr(ref), float(beta),
           float(label_smoothing), float(grad_scale), ws.data_ptr(), n, at + 8 * T, at,
           at + 12 * T, loss.data_ptr(), rewards.data_ptr(), *where)
    if want_dx and T:
        N.kernel_launches += 1  # the gradient rows
    return targets, loss, rewards, saved, dx


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ref_logps, beta, label_smoothing, ignore_index):
        targets, loss, rewards, saved, _ = _preference(
            logits, targets, ref_logps, beta, label_smoothing, ignore_index, 1.0, None, False)
        ctx.save_for_backward(logits, targets, saved)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @_first_order
    def backward(ctx, dloss, _drewards):
        logits, targets, saved = ctx.saved_tensors
        return (_logprobs_bwd(logits, targets, ctx.ignore_index, 1.0, saved,
                              saved[3 * targets.numel():],
                              dloss.float()), None, None, None, None, None)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor,
                    ref_logps: torch.Tensor | None = None, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100):
    """Preference loss of paired sequences over their summed log ratios.

    logits [2 P, S, V] (bf16 or fp32): the P chosen sequences, then their rejected
    ones in the same order; targets [2 P, S] int64, ``ignore_index`` on prompts and
    padding; ref_logps [2 P, S] fp32, the frozen reference model's
    ``token_logprobs`` (None: 0). Returns (loss, rewards): the mean over pairs of
    (1 - e) softplus(-h) + e softplus(h), h the chosen reward less the rejected
    one, e = ``label_smoothing``, and rewards [2 P] = beta * sum of log ratios
    (no gradient). Differentiable in the logits."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _PreferenceFn.apply(logits, targets, ref_logps, beta, label_smoothing, ignore_index)
    return _preference(logits, targets, ref_logps, beta, label_smoothing, ignore_index, 1.0, None,
                       False)[1:3]


def preference_loss_grad(logits: torch.Tensor, targets: torch.Tensor,
                         ref_logps: torch.Tensor | None = None, *, beta: float = 0.1,
                         label_smoothing: float = 0.0, ignore_index: int = -100,
                         grad_scale: float = 1.0, out: torch.Tensor | None = None):
    """``preference_loss`` and its gradient in one call: (loss, rewards, dlogits).
    dlogits = grad_scale * dloss/dlogits, written into ``out`` when given (which
    may be ``logits`` itself)."""
    _, loss, rewards, _, dx = _preference(logits, targets, ref_logps, beta, label_smoothing,
                                          ignore_index, grad_scale, out, True)
    return loss, rewards, dx


def _policy(logits, targets, old_logps, advantages, ref_logps, clip, kl_coef, temperature,
            reduction, ignore_index, grad_scale, out, want_dx, want_saved):
    x = _Logits(logits)
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction must be 'token' or 'sequence', not {reduction!r}")
    clip_lo, clip_hi = clip
    targets = _targets(x, targets)
    old = x.per_row(old_logps, "old_logps", torch.float32)
    ref = x.per_row(ref_logps, "ref_logps", torch.float32)
    adv = advantages
    if adv.shape == x.lead:
        adv = x.per_row(adv, "advantages", torch.float32)
        s0, s1 = x.n1, 1
    elif logits.dim() == 3 and adv.shape == x.lead[:1]:
        if adv.device != x.dev or adv.dtype != torch.float32 or adv.requires_grad:
            raise ValueError("advantages must be fp32 constants on the logits' device")
        adv = adv.contiguous()
        s0, s1 = 1, 0
    else:
        raise ValueError(f"advantages must have shape {tuple(x.lead)}, or one per sequence")
    ws, n = x.workspace()
    logps = torch.empty_like(targets, dtype=torch.float32)
    loss, kl = x.scalar(), x.scalar()
    # statistics (pairs, 8-byte aligned), coefficients
    T = x.n0 * x.n1
    saved = torch.empty(3 * T, dtype=torch.float32, device=x.dev) if want_saved else None
    at = saved.data_ptr() if want_saved else None
    dx, where = x.grad_out(logits, out) if want_dx else (None, _NO_GRAD)
    x.call("lema_policy_loss", targets.data_ptr(), int(ignore_index), float(temperature),
           _ptr(old), adv.data_ptr(), s0, s1, _ptr(ref), float(clip_lo), float(clip_hi),
           float(kl_coef), int(reduction == "sequence"), float(grad_scale), ws.data_ptr(), n,
           logps.data_ptr(), at, at + 8 * T if want_saved else None, loss.data_ptr(),
           kl.data_ptr(), *where)
    return targets, loss, logps, kl, saved, dx


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, old_logps, advantages, ref_logps, clip, kl_coef, temperature,
                reduction, ignore_index):
        targets, loss, logps, kl, saved, _ = _policy(
            logits, targets, old_logps, advantages, ref_logps, clip, kl_coef, temperature,
            reduction, ignore_index, 1.0, None, False, True)
        ctx.save_for_backward(logits, targets, saved)
        ctx.meta = (ignore_index, float(temperature))
        ctx.mark_non_differentiable(logps, kl)
        return loss, logps, kl

    @staticmethod
    @_first_order
    def backward(ctx, dloss, _dlogps, _dkl):
        logits, targets, saved = ctx.saved_tensors
        ignore_index, temperature = ctx.meta
        dx = _logprobs_bwd(logits, targets, ignore_index, temperature, saved,
                           saved[2 * targets.numel():], dloss.float())
        return (dx,) + (None,) * 9


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logps: torch.Tensor | None,
                advantages: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                temperature: float = 1.0, reduction: str = "token", ignore_index: int = -100):
    """Clipped policy loss with a KL term.

    logits [B, S, V] or [T, V]; targets (the sampled tokens, aligned with the rows
    that predict them), old_logps (the sampling policy's, None: on-policy, ratio
    1) and ref_logps (the KL's reference, None: no KL) of shape [B, S] / [T];
    advantages of that shape, or [B]. With r = exp(lp - old), d = ref - lp:
    loss = sum w (-min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef
    (exp(d) - 1 - d)), w = 1 / counted tokens ("token") or the mean over sequences
    of their tokens' means ("sequence"). Returns (loss, logps, kl): logps fp32, kl
    the weighted sum of exp(d) - 1 - d (neither with a gradient). Differentiable in
    the logits; every other argument is a constant."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _PolicyFn.apply(logits, targets, old_logps, advantages, ref_logps, clip, kl_coef,
                               temperature, reduction, ignore_index)
    return _policy(logits, targets, old_logps, advantages, ref_logps, clip, kl_coef, temperature,
                   reduction, ignore_index, 1.0, None, False, False)[1:4]


def policy_loss_grad(logits: torch.Tensor, targets: torch.Tensor, old_logps: torch.Tensor | None,
                     advantages: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                     clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                     temperature: float = 1.0, reduction: str = "token",
                     ignore_index: int = -100, grad_scale: float = 1.0,
                     out: torch.Tensor | None = None):
    """``policy_loss`` and its gradient in one pass over the logits: (loss, logps,
    kl, dlogits). dlogits = grad_scale * dloss/dlogits, written into ``out`` when
    given (which may be ``logits`` itself)."""
    _, loss, logps, kl, _, dx = _policy(logits, targets, old_logps, advantages, ref_logps, clip,
                                        kl_coef, temperature, reduction, ignore_index,
                                        grad_scale, out, True, False)
    return loss, logps, kl, dx


def _teacher(x: _Logits, ids: torch.Tensor, logits: torch.Tensor, mask):
    if ids.device != x.dev or logits.device != x.dev:
        raise RuntimeError("teacher tensors must be on the logits' device")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"teacher_ids must be int32 or int64, got {ids.dtype}")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"teacher_logits must be bf16 or fp32, got {logits.dtype}")
    if ids.shape != logits.shape or ids.shape[:-1] != x.lead or ids.dim() != len(x.lead) + 1:
        raise ValueError(f"teacher_ids and teacher_logits must be {tuple(x.lead)} + (K,)")
    if logits.requires_grad:
        raise ValueError("teacher_logits are constants of the loss: detach them")
    mask = x.per_row(mask, "mask", torch.bool)
    return ids.contiguous(), logits.contiguous(), mask


def _distill(x, logits, ids, tl, mask, temperature, grad_scale, upstream, out, want_dx):
    """One call on checked teacher tensors: (loss, dlogits or None)."""
    ws, n = x.workspace()
    loss = x.scalar()
    dx, where = x.grad_out(logits, out) if want_dx else (None, _NO_GRAD)
    x.call("lema_distill_loss", ids.data_ptr(), int(ids.dtype is torch.int32), tl.data_ptr(),
           int(tl.dtype is torch.float32), ids.shape[-1], _ptr(mask), float(temperature),
           float(grad_scale), _ptr(upstream), ws.data_ptr(), n, loss.data_ptr(), *where)
    return loss, dx


class _DistillFn(torch.autograd.Function):
    """The backward runs the fused pass: rows are held on chip while their statistics are
    taken, so it moves no more bytes than one from saved statistics. Over 8 x 512 rows of
    32000 bf16 with 64 entries forward and backward take 180 us, the forward alone 78 and
    ``distill_loss_grad`` 111."""

    @staticmethod
    def forward(ctx, logits, ids, tl, mask, temperature):
        ctx.save_for_backward(logits, ids, tl, mask)
        ctx.temperature = temperature
        return _distill(_Logits(logits), logits, ids, tl, mask, temperature, 1.0, None, None,
                        False)[0]

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        logits, ids, tl, mask = ctx.saved_tensors
        dx = _distill(_Logits(logits), logits, ids, tl, mask, ctx.temperature, 1.0, dloss.float(),
                      None, True)[1]
        return dx, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                 mask: torch.Tensor | None = None, *, temperature: float = 1.0) -> torch.Tensor:
    """Distillation from the K (at most 1024) best logits a teacher gave for each row:
    temperature^2 * mean over counted rows of KL(p || q), p the softmax over
    the teacher's K entries and q the student's over the whole vocabulary, both at
    ``temperature``. logits [..., V] bf16 or fp32; teacher_ids [..., K] int32 or
    int64; teacher_logits [..., K] bf16 or fp32 (-inf: no entry, whatever its
    index; an index that repeats adds its weights); mask [...] bool, False rows
    are not read. Differentiable in the logits."""
    x = _Logits(logits)
    ids, tl, mask = _teacher(x, teacher_ids, teacher_logits, mask)
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillFn.apply(logits, ids, tl, mask, temperature)
    return _distill(x, logits, ids, tl, mask, temperature, 1.0, None, None, False)[0]


def distill_loss_grad(logits: torch.Tensor, teacher_ids: torch.Tensor,
                      teacher_logits: torch.Tensor, mask: torch.Tensor | None = None, *,
                      temperature: float = 1.0, grad_scale: float = 1.0,
                      out: torch.Tensor | None = None):
    """``distill_loss`` and its gradient in one pass over the logits: (loss, dlogits).
    dlogits = grad_scale * dloss/dlogits, written into ``out`` when given (which may
    be ``logits`` itself)."""
    x = _Logits(logits)
    ids, tl, mask = _teacher(x, teacher_ids, teacher_logits, mask)
    return _distill(x, logits, ids, tl, mask, temperature, grad_scale, None, out, True)
