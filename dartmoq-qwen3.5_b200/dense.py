"""Dense operators beside the packed experts: 8-bit products and the 16-bit gated feed-forward block.

  quantize_int8_tokens   rows of a 16-bit tensor -> 8-bit codes and one scale a row
  int8_matmul            codes x 8-bit weight, one scale a token and one a weight row (+ bias)
  int8_linear            both of the above in one call
  int8_gated_linear      silu(x Wg^T) * (x Wu^T) with 8-bit operands: the first half of a feed-forward block
  gated_feed_forward     (silu(x Wg^T) * (x Wu^T)) Wd^T in 16 bits, with its gradients

The modules over them are ``linear.W8A8Linear`` and ``ffn.GatedFeedForward`` / ``ffn.W8A8GatedFeedForward``; the latter two
serve as ``shared_expert`` of the MoE modules.

All work goes to the current stream of the tensors' device, whichever device is current; nothing synchronises and every
buffer comes from torch's allocator.  Errors follow ``kernels``: ``DmoqError`` for tensors that are not on a CUDA device,
``TypeError`` for a wrong dtype, ``ValueError`` for shapes.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_HALF = (torch.bfloat16, torch.float16)


def _call(name: str, device: torch.device, *args) -> None:
    """One entry point on the current stream of ``device``; that device is current during the call."""
    index = device.index
    fn = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor, cols: int) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of ``cols`` elements that the kernels can read where they lie (unit inner stride, 16-byte aligned rows),
    copied only if they cannot; and the pitch between rows in elements."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    n = t.shape[0]
    if n > 1 << 30:
        raise ValueError(f"at most 2^30 rows, got {n}")
    pitch = t.stride(0) if n > 1 else cols
    per16 = 16 // t.element_size()
    if t.stride(1) != 1 or pitch < cols or pitch % per16 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        pitch = cols
    return t, pitch


def _need(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _check_input(x: torch.Tensor, what: str = "x") -> None:
    if not x.is_cuda:
        raise _lib.DmoqError("libdmoq operators take CUDA tensors only (no CPU path)")
    if x.dtype not in _HALF:
        raise TypeError(f"{what} must be fp16 or bf16, got {x.dtype}")
    _need(x.dim() >= 1, f"{what} needs at least one dimension")


def _check_weight8(w: torch.Tensor, scale: torch.Tensor, k: int, device, what: str) -> torch.Tensor:
    if w.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"{what} must be int8 with an fp32 scale, got {w.dtype} and {scale.dtype}")
    _need(w.dim() == 2 and w.shape[1] == k and w.shape[0] >= 1, f"{what} must have shape (outputs, {k}), got {tuple(w.shape)}")
    _need(scale.numel() == w.shape[0], f"{what} needs one scale a row: {w.shape[0]} rows, {scale.numel()} scales")
    _need(w.device == device and scale.device == device, f"{what} and its scale must be on {device}")
    return w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)


def _check_k8(k: int) -> None:
    _need(k >= 16 and k % 16 == 0, f"8-bit products need an inner size that is a multiple of 16, got {k}")


def _check_bias(bias: Optional[torch.Tensor], n: int, dtype, device) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    if bias.dtype != dtype:
        raise TypeError(f"bias must have the output's type {dtype}, got {bias.dtype}")
    _need(tuple(bias.shape) == (n,) and bias.device == device, f"bias must have shape ({n},) on {device}")
    return bias.contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


@torch.no_grad()
def quantize_int8_tokens(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit codes of each row of ``x`` (..., K): scale = max|x| / 127 in fp32, code = rint(127 x / max|x|) with ties
    to even, correctly rounded.  A row of zeros has scale 0; a row with an infinity or a NaN has codes 0 and scale NaN, so
    that what is computed from it is NaN.  Returns (int8 (..., K), fp32 (...)).  K is a multiple of 16."""
    _check_input(x)
    k = x.shape[-1]
    _check_k8(k)
    rows, pitch = _rows(x, k)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call("dmoq_token_quant", x.device, rows.data_ptr(), x.dtype == torch.bfloat16, rows.shape[0], k, pitch, codes.data_ptr(),
          scale.data_ptr())
    return codes, scale


@torch.no_grad()
def int8_matmul(codes: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[t, n] = scale[t] * weight_scale[n] * sum_k codes[t, k] * weight[n, k] (+ bias[n]); exact int32 sums, scales and bias
    in fp32, one rounding to ``out_dtype``.  ``codes`` int8 (..., K), ``weight`` int8 (N, K); K a multiple of 16, at most
    131056; any N."""
    if not codes.is_cuda:
        raise _lib.DmoqError("libdmoq operators take CUDA tensors only (no CPU path)")
    if codes.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"codes must be int8 with an fp32 scale, got {codes.dtype} and {scale.dtype}")
    if out_dtype not in _HALF:
        raise TypeError(f"out_dtype must be fp16 or bf16, got {out_dtype}")
    _need(codes.dim() >= 1, "codes need at least one dimension")
    k, dev = codes.shape[-1], codes.device
    _check_k8(k)
    _need(scale.shape == codes.shape[:-1] and scale.device == dev, f"one scale a token on {dev}: got {tuple(scale.shape)}")
    w = _check_weight8(weight, weight_scale, k, dev, "weight")
    n = w.shape[0]
    bias = _check_bias(bias, n, out_dtype, dev)
    a, pitch = _rows(codes, k)
    if pitch != k:
        a = a.contiguous()
    scale, weight_scale = scale.contiguous(), weight_scale.contiguous()
    out = torch.empty(codes.shape[:-1] + (n,), dtype=out_dtype, device=dev)
    _call("dmoq_int8_gemm", dev, a.data_ptr(), scale.data_ptr(), w.data_ptr(), weight_scale.data_ptr(), _ptr(bias),
          out_dtype == torch.bfloat16, a.shape[0], n, k, out.data_ptr())
    return out


@torch.no_grad()
def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``int8_matmul(*quantize_int8_tokens(x), weight, weight_scale, bias, x.dtype)`` in one call: x (..., K) -> (..., N)."""
    _check_input(x)
    k, dev = x.shape[-1], x.device
    _check_k8(k)
    w = _check_weight8(weight, weight_scale, k, dev, "weight")
    n = w.shape[0]
    bias = _check_bias(bias, n, x.dtype, dev)
    rows, pitch = _rows(x, k)
    t = rows.shape[0]
    codes = torch.empty((t, k), dtype=torch.int8, device=dev)
    scale = torch.empty((t,), dtype=torch.float32, device=dev)
    weight_scale = weight_scale.contiguous()
    out = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    _call("dmoq_int8_linear", dev, rows.data_ptr(), x.dtype == torch.bfloat16, pitch, w.data_ptr(), weight_scale.data_ptr(),
          _ptr(bias), t, n, k, codes.data_ptr(), scale.data_ptr(), out.data_ptr())
    return out


@torch.no_grad()
def int8_gated_linear(x: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                      up_scale: torch.Tensor) -> torch.Tensor:
    """silu(g) * u with g, u the 8-bit products of x's codes with ``w_gate`` and ``w_up`` (each int8 (I, K), one scale a row):
    both products, the activation and the multiplication in one kernel, in fp32 up to one rounding.  x (..., K) -> (..., I)."""
    _check_input(x)
    k, dev = x.shape[-1], x.device
    _check_k8(k)
    wg = _check_weight8(w_gate, gate_scale, k, dev, "w_gate")
    wu = _check_weight8(w_up, up_scale, k, dev, "w_up")
    _need(wg.shape == wu.shape, f"w_gate and w_up must have one shape, got {tuple(wg.shape)} and {tuple(wu.shape)}")
    n = wg.shape[0]
    rows, pitch = _rows(x, k)
    t = rows.shape[0]
    codes = torch.empty((t, k), dtype=torch.int8, device=dev)
    scale = torch.empty((t,), dtype=torch.float32, device=dev)
    gate_scale, up_scale = gate_scale.contiguous(), up_scale.contiguous()
    out = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    _call("dmoq_int8_gated_linear", dev, rows.data_ptr(), x.dtype == torch.bfloat16, pitch, wg.data_ptr(), gate_scale.data_ptr(),
          wu.data_ptr(), up_scale.data_ptr(), t, n, k, codes.data_ptr(), scale.data_ptr(), out.data_ptr())
    return out


def _ffn_forward(x: torch.Tensor, pitch: int, wg: torch.Tensor, wu: torch.Tensor, wd: torch.Tensor, save: bool):
    """y, and the hidden values h; with ``save`` also what the gradients need of them."""
    (t, hidden), inter, dev = x.shape, wg.shape[0], x.device
    h = torch.empty((t, inter), dtype=x.dtype, device=dev)
    saved = torch.empty((3, t, inter), dtype=torch.int16, device=dev) if save else None
    y = torch.empty((t, hidden), dtype=x.dtype, device=dev)
    _call("dmoq_gated_ffn", dev, x.data_ptr(), x.dtype == torch.bfloat16, pitch, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), t,
          hidden, inter, h.data_ptr(), _ptr(saved), y.data_ptr())
    return y, h, saved


class _GatedFeedForward(torch.autograd.Function):
    """What the gradients need of the hidden values is kept as silu(g) and u silu'(g) to 24 bits each, not as g and u in 16: dg =
    dh * (u silu'(g)) and du = dh * silu(g) are then rounded to 16 bits (they are operands of the next products) from values
    that carry no other rounding of that type, and backward computes no exponentials.  With h that is 8 bytes a hidden
    value, as much as g, u, silu(g) and h in 16 bits."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down):
        rows, pitch = _rows(x, x.shape[-1])
        inner = any(ctx.needs_input_grad[:3])
        y, h, saved = _ffn_forward(rows, pitch, w_gate, w_up, w_down, inner)
        ctx.save_for_backward(rows, w_gate, w_up, w_down, h if ctx.needs_input_grad[3] else None, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, h, saved = ctx.saved_tensors
        need_x, need_g, need_u, need_d = ctx.needs_input_grad
        (t, hidden), inter, dev, dt = x.shape, wg.shape[0], x.device, x.dtype
        dy, dy_pitch = _rows(dy, hidden)
        x_pitch = x.stride(0) if t > 1 else hidden
        inner = need_x or need_g or need_u
        dgu = torch.empty((t, 2 * inter), dtype=dt, device=dev) if inner else None
        dx = torch.empty((t, hidden), dtype=dt, device=dev) if need_x else None
        # the two halves of one buffer: one product computes both
        dw = torch.empty((int(need_g) + int(need_u), inter, hidden), dtype=dt, device=dev) if need_g or need_u else None
        dwg = dw[0] if need_g else None
        dwu = dw[-1] if need_u else None
        dwd = torch.empty((hidden, inter), dtype=dt, device=dev) if need_d else None
        _call("dmoq_gated_ffn_backward", dev, dy.data_ptr(), dy_pitch, x.data_ptr(), dt == torch.bfloat16, x_pitch, wg.data_ptr(),
              wu.data_ptr(), wd.data_ptr(), t, hidden, inter, _ptr(h), _ptr(saved), _ptr(dgu), _ptr(dx), _ptr(dwg),
              _ptr(dwu), _ptr(dwd))
        return dx, dwg, dwu, dwd


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """(silu(x w_gate^T) * (x w_up^T)) w_down^T for x (..., H), w_gate and w_up (I, H), w_down (H, I), all bf16 or all fp16; H and I
    multiples of 8.  Sums in fp32; the hidden values are rounded to the 16-bit type between the two kernels (they are the second
    product's operand), so fp16 hidden values beyond 65504 become infinite.  Differentiable once in every argument; each gradient
    that is not needed is not computed."""
    _check_input(x)
    hidden, dev, dt = x.shape[-1], x.device, x.dtype
    for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if w.dtype != dt:
            raise TypeError(f"{name} must have x's type {dt}, got {w.dtype}")
        _need(w.dim() == 2 and w.device == dev, f"{name} must be a matrix on {dev}")
    inter = w_gate.shape[0]
    _need(tuple(w_gate.shape) == (inter, hidden) and tuple(w_up.shape) == (inter, hidden) and tuple(w_down.shape) == (hidden, inter),
          f"weights must be ({inter}, {hidden}) twice and ({hidden}, {inter}), got {tuple(w_gate.shape)}, {tuple(w_up.shape)}, "
          f"{tuple(w_down.shape)}")
    _need(hidden >= 8 and hidden % 8 == 0 and inter >= 8 and inter % 8 == 0,
          f"hidden and intermediate sizes must be multiples of 8, got {hidden} and {inter}")
    weights = [w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)
               for w in (w_gate, w_up, w_down)]
    rows = x if x.dim() == 2 else x.reshape(-1, hidden)
    if torch.is_grad_enabled() and (x.requires_grad or any(w.requires_grad for w in weights)):
        y = _GatedFeedForward.apply(rows, *weights)
    else:
        rows, pitch = _rows(rows, hidden)
        y = _ffn_forward(rows, pitch, *weights, save=False)[0]
    return y if x.dim() == 2 else y.reshape(x.shape)
