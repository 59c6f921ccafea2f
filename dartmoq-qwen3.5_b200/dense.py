"""Dense operators beside the packed experts: 8-bit products and the 16-bit gated feed-forward block.

  quantize_int8_tokens   rows of a 16-bit tensor -> 8-bit codes and one scale a row
  int8_matmul            codes x 8-bit weight, one scale a token and one a weight row (+ bias)
  int8_linear            both of the above in one call
  int8_gated_linear      silu(x Wg^T) * (x Wu^T) with 8-bit operands: the first half of a feed-forward block
  int8_gated_matmul      the same of codes that are there already
  gated_feed_forward     (silu(x Wg^T) * (x Wu^T)) Wd^T in 16 bits, with its gradients

The modules over them are ``linear.W8A8Linear`` and ``ffn.GatedFeedForward`` / ``ffn.W8A8GatedFeedForward``; the latter two
serve as ``shared_expert`` of the MoE modules.

All work goes to the current stream of the tensors' device, whichever device is current; nothing synchronises and every
buffer comes from torch's allocator.  The 8-bit operators have no gradients: their results never require one and carry no
tangent.  Errors follow ``kernels``: ``DmoqError`` for tensors that are not on a CUDA device, for calls inside a trace and for
inner sizes above 131056 of an 8-bit product, ``TypeError`` for a wrong dtype, ``ValueError`` for all other shapes.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_BF16, _FP16, _FP32, _INT8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
_MAX_ROWS = 1 << 30
_MAX_SIDE = 1 << 29          # of a feed-forward block
_MAX_GRAD_TOKENS = 1 << 26
_tracing, _modes, _mode, _PROXY = (torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode,
                                   torch._C._TorchDispatchModeKey.PROXY)
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


_entries: dict = {}


def _entry(name: str):
    fn = _entries[name] = getattr(_lib.load(), name)
    return fn


def _call(name: str, index: int, *args) -> None:
    """One entry point on the current stream of device ``index``, which is current during the call."""
    fn = _entries.get(name) or _entry(name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor, cols: int) -> Tuple[torch.Tensor, int, int]:
    """``t`` as rows of ``cols`` elements that the kernels can read where they lie (unit inner stride, 16-byte aligned rows),
    copied only if they cannot; their number, and the pitch between them in elements."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    n = t.shape[0]
    if n > _MAX_ROWS:
        raise ValueError(f"at most 2^30 rows, got {n}")
    if not t.is_contiguous() or t.data_ptr() & 15:
        pitch = t.stride(0) if n > 1 else cols
        if t.stride(1) == 1 and pitch >= cols and not (pitch * t.element_size() | t.data_ptr()) & 15:
            return t, n, pitch
        t = t.clone(memory_format=torch.contiguous_format)
    return t, n, cols


def _matrix(w: torch.Tensor, cols: int) -> Tuple[torch.Tensor, int]:
    """A matrix of ``cols`` columns as the kernels can read it, and its pitch."""
    if w.is_contiguous() and not w.data_ptr() & 15:
        return w, cols
    w, _, pitch = _rows(w, cols)
    return w, pitch


def _need(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _check_cuda(t: torch.Tensor) -> None:
    # a trace (torch.jit or torch.fx) would hold the outputs' allocation and not the call that fills them
    if _tracing() is not None or (_modes() and _mode(_PROXY) is not None):
        raise _lib.DmoqError("libdmoq operators cannot be traced")
    if not t.is_cuda:
        raise _lib.DmoqError("libdmoq operators take CUDA tensors only (no CPU path)")


def _check_input(x: torch.Tensor) -> None:
    _check_cuda(x)
    if x.dtype is not _BF16 and x.dtype is not _FP16:
        raise TypeError(f"x must be fp16 or bf16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x needs at least one dimension")


def _check_k8(k: int) -> None:
    if k < 16 or k & 15:
        raise ValueError(f"8-bit products need an inner size that is a multiple of 16, got {k}")
    if k > _MAX_ROWS:        # sizes travel as 32-bit numbers: a larger one would arrive as another
        raise ValueError(f"at most 2^30 columns, got {k}")


def _weight8(w: torch.Tensor, scale: torch.Tensor, k: int, index: int, what: str) -> Tuple[torch.Tensor, int, int, torch.Tensor]:
    """The weight as the kernels take it, its rows and pitch, and its scales."""
    if w.dtype is not _INT8 or scale.dtype is not _FP32:
        raise TypeError(f"{what} must be int8 with an fp32 scale, got {w.dtype} and {scale.dtype}")
    shape = w.shape
    if len(shape) != 2 or shape[1] != k or not 1 <= shape[0] <= _MAX_ROWS:
        raise ValueError(f"{what} must have shape (outputs, {k}) with at most 2^30 outputs, got {tuple(shape)}")
    if scale.shape != shape[:1]:
        raise ValueError(f"{what} needs one scale a row: {shape[0]} rows, scales of shape {tuple(scale.shape)}")
    if w.get_device() != index or scale.get_device() != index:      # -1 on the CPU
        raise ValueError(f"{what} and its scale must be on cuda:{index}")
    w, pitch = _matrix(w, k)
    return w, shape[0], pitch, scale if scale.is_contiguous() else scale.contiguous()


def _bias_ptr(bias: Optional[torch.Tensor], n: int, dtype: torch.dtype, index: int):
    """(the bias as the kernels take it, its address); the caller holds the former until its call has been made."""
    if bias is None:
        return None, None
    if bias.dtype is not dtype:
        raise TypeError(f"bias must have the output's type {dtype}, got {bias.dtype}")
    _need(tuple(bias.shape) == (n,) and bias.is_cuda and bias.get_device() == index, f"bias must have shape ({n},) on cuda:{index}")
    bias = bias.contiguous()
    return bias, bias.data_ptr()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def quantize_int8_tokens(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit codes of each row of ``x`` (..., K): scale = max|x| / 127 in fp32, code = rint(127 x / max|x|) with ties
    to even, correctly rounded.  A row of zeros has scale 0; a row with an infinity or a NaN has codes 0 and scale NaN, so
    that what is computed from it is NaN.  Returns (int8 (..., K), fp32 (...)).  K is a multiple of 16, at most 2^30."""
    _check_input(x)
    k = x.shape[-1]
    _check_k8(k)
    rows, t, pitch = _rows(x, k)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call("dmoq_token_quant", x.get_device(), rows.data_ptr(), x.dtype is _BF16, t, k, pitch, codes.data_ptr(), scale.data_ptr())
    return codes, scale


def int8_matmul(codes: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[t, n] = scale[t] * weight_scale[n] * sum_k codes[t, k] * weight[n, k] (+ bias[n]); exact int32 sums, scales and bias
    in fp32, one rounding to ``out_dtype``.  ``codes`` int8 (..., K), ``weight`` int8 (N, K); K a multiple of 16, at most
    131056; any N.  Codes whose rows do not follow one another are copied first."""
    codes, t, k, scale, index = _token_codes(codes, scale, out_dtype)
    w, n, w_pitch, ws = _weight8(weight, weight_scale, k, index, "weight")
    bias, bias_ptr = _bias_ptr(bias, n, out_dtype, index)
    out = torch.empty(scale.shape + (n,), dtype=out_dtype, device=codes.device)
    _call("dmoq_int8_gemm", index, codes.data_ptr(), scale.data_ptr(), w.data_ptr(), w_pitch, ws.data_ptr(), bias_ptr, out_dtype is _BF16,
          t, n, k, out.data_ptr())
    return out


def int8_gated_matmul(codes: torch.Tensor, scale: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                      up_scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """silu(g) * u of given codes, g and u as ``int8_matmul`` has them (see ``int8_gated_linear``): for tokens whose codes are
    there already, because another product of theirs needed them."""
    codes, t, k, scale, index = _token_codes(codes, scale, out_dtype)
    wg, n, gate_pitch, sg, wu, up_pitch, su = _gated_weights(w_gate, gate_scale, w_up, up_scale, k, index)
    out = torch.empty(scale.shape + (n,), dtype=out_dtype, device=codes.device)
    _call("dmoq_int8_gated_gemm", index, codes.data_ptr(), scale.data_ptr(), wg.data_ptr(), gate_pitch, sg.data_ptr(), wu.data_ptr(), up_pitch,
          su.data_ptr(), out_dtype is _BF16, t, n, k, out.data_ptr())
    return out


def _token_codes(codes: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype):
    """Codes (without a pitch: the entry points take none) and scales as the kernels take them, their sizes and device."""
    _check_cuda(codes)
    if codes.dtype is not _INT8 or scale.dtype is not _FP32:
        raise TypeError(f"codes must be int8 with an fp32 scale, got {codes.dtype} and {scale.dtype}")
    if out_dtype is not _BF16 and out_dtype is not _FP16:
        raise TypeError(f"out_dtype must be fp16 or bf16, got {out_dtype}")
    _need(codes.dim() >= 1, "codes need at least one dimension")
    k, index = codes.shape[-1], codes.get_device()
    _check_k8(k)
    _need(scale.shape == codes.shape[:-1] and scale.is_cuda and scale.get_device() == index,
          f"one scale a token on cuda:{index}: got {tuple(scale.shape)}")
    rows, t, pitch = _rows(codes, k)
    return rows if pitch == k else rows.contiguous(), t, k, scale.contiguous(), index


def _gated_weights(w_gate, gate_scale, w_up, up_scale, k: int, index: int):
    wg, n, gate_pitch, sg = _weight8(w_gate, gate_scale, k, index, "w_gate")
    wu, n_up, up_pitch, su = _weight8(w_up, up_scale, k, index, "w_up")
    if n_up != n:
        raise ValueError(f"w_gate and w_up must have one shape, got {tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    return wg, n, gate_pitch, sg, wu, up_pitch, su


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``int8_matmul(*quantize_int8_tokens(x), weight, weight_scale, bias, x.dtype)`` in one call: x (..., K) -> (..., N)."""
    _check_input(x)
    shape, index = x.shape, x.get_device()
    k = shape[-1]
    _check_k8(k)
    w, n, w_pitch, ws = _weight8(weight, weight_scale, k, index, "weight")
    bias, bias_ptr = _bias_ptr(bias, n, x.dtype, index)
    rows, t, pitch = _rows(x, k)
    scratch = _int8_scratch(x, t, n, k, False)
    out = x.new_empty((t, n) if len(shape) == 2 else shape[:-1] + (n,))
    _call("dmoq_int8_linear", index, rows.data_ptr(), x.dtype is _BF16, pitch, w.data_ptr(), w_pitch, ws.data_ptr(), bias_ptr, t, n, k,
          _ptr(scratch), out.data_ptr())
    return out


def _int8_scratch(x: torch.Tensor, t: int, n: int, k: int, gated: bool) -> Optional[torch.Tensor]:
    need = (_entries.get("dmoq_int8_scratch_bytes") or _entry("dmoq_int8_scratch_bytes"))(t, n, k, gated)
    return x.new_empty((need,), dtype=torch.uint8) if need else None


def int8_gated_linear(x: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                      up_scale: torch.Tensor) -> torch.Tensor:
    """silu(g) * u with g, u the 8-bit products of x's codes with ``w_gate`` and ``w_up`` (each int8 (I, K), one scale a row):
    both products, the activation and the multiplication in one kernel, in fp32 up to one rounding.  x (..., K) -> (..., I)."""
    _check_input(x)
    shape, index = x.shape, x.get_device()
    k = shape[-1]
    _check_k8(k)
    wg, n, gate_pitch, sg, wu, up_pitch, su = _gated_weights(w_gate, gate_scale, w_up, up_scale, k, index)
    rows, t, pitch = _rows(x, k)
    scratch = _int8_scratch(x, t, n, k, True)
    out = x.new_empty((t, n) if len(shape) == 2 else shape[:-1] + (n,))
    _call("dmoq_int8_gated_linear", index, rows.data_ptr(), x.dtype is _BF16, pitch, wg.data_ptr(), gate_pitch, sg.data_ptr(),
          wu.data_ptr(), up_pitch, su.data_ptr(), t, n, k, _ptr(scratch), out.data_ptr())
    return out


def _ffn_forward(x: torch.Tensor, t: int, pitch: int, wg: torch.Tensor, wu: torch.Tensor, wd: torch.Tensor, save: bool):
    """y, and the hidden values h; with ``save`` also what the gradients need of them."""
    hidden, inter = wd.shape
    wg, gate_pitch = _matrix(wg, hidden)
    wu, up_pitch = _matrix(wu, hidden)
    wd, down_pitch = _matrix(wd, inter)
    h = x.new_empty((t, (inter + 63) & -64))       # rows on whole 128-byte lines
    saved = x.new_empty((3, t, inter), dtype=torch.int16) if save else None
    y = x.new_empty((t, hidden))
    _call("dmoq_gated_ffn", x.get_device(), x.data_ptr(), x.dtype is _BF16, pitch, wg.data_ptr(), gate_pitch, wu.data_ptr(), up_pitch,
          wd.data_ptr(), down_pitch, t, hidden, inter, h.data_ptr(), h.shape[1], _ptr(saved), y.data_ptr())
    return y, h, saved


class _GatedFeedForward(torch.autograd.Function):
    """What the gradients need of the hidden values is kept as silu(g) and u silu'(g) in the upper 24 bits of their floats, not as
    g and u in 16: dg = dh * (u silu'(g)) and du = dh * silu(g) are then rounded to 16 bits (they are operands of the next
    products) from values that carry no other rounding of that type, and backward computes no exponentials.  With h that is
    8 bytes a hidden value, as much as g, u, silu(g) and h in 16 bits."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down):
        rows, t, pitch = _rows(x, x.shape[-1])
        need_x, need_g, need_u, need_d = ctx.needs_input_grad
        y, h, saved = _ffn_forward(rows, t, pitch, w_gate, w_up, w_down, need_x or need_g or need_u)
        ctx.save_for_backward(rows, w_gate, w_up, w_down, h if need_d else None, saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _ffn_backward(ctx, dy)
        # grad mode is on only where a graph of the backward pass is asked for, which this has none of.  The gradients depend on
        # x and the weights whether or not dy requires one, so they always require one that raises.
        with torch.no_grad():
            grads = _ffn_backward(ctx, dy)
        anchor = torch.empty(0, requires_grad=True)
        marked = iter(_DifferentiableOnce.apply(anchor, *(g for g in grads if g is not None)))
        return tuple(None if g is None else next(marked) for g in grads)


class _DifferentiableOnce(torch.autograd.Function):
    """Gradients as they are; asking for theirs raises."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(g.detach() for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("gated_feed_forward is differentiable once: it has no second derivatives")


def _ffn_backward(ctx, dy):
    x, wg, wu, wd, h, saved = ctx.saved_tensors
    need_x, need_g, need_u, need_d = ctx.needs_input_grad
    hidden, inter = wd.shape
    dy, t, dy_pitch = _rows(dy, hidden)
    # saved-tensor hooks may have laid them out anew
    x, _, x_pitch = _rows(x, hidden)
    wg, gate_pitch = _matrix(wg, hidden)
    wu, up_pitch = _matrix(wu, hidden)
    wd, down_pitch = _matrix(wd, inter)
    h_pitch = 0
    if h is not None:
        h, h_pitch = _matrix(h, h.shape[1])
    if saved is not None:
        saved = saved.contiguous()
    d_pitch = (2 * inter + 63) & -64
    dgu = x.new_empty((t, d_pitch)) if need_x or need_g or need_u else None
    dx = x.new_empty((t, hidden)) if need_x else None
    # the two halves of one buffer: one product computes both
    dw = x.new_empty((int(need_g) + int(need_u), inter, hidden)) if need_g or need_u else None
    dwg = dw[0] if need_g else None
    dwu = dw[-1] if need_u else None
    dwd = x.new_empty((hidden, inter)) if need_d else None
    _call("dmoq_gated_ffn_backward", x.get_device(), dy.data_ptr(), dy_pitch, x.data_ptr(), x.dtype is _BF16, x_pitch,
          wg.data_ptr(), gate_pitch, wu.data_ptr(), up_pitch, wd.data_ptr(), down_pitch, t, hidden, inter, _ptr(h), h_pitch,
          _ptr(saved), _ptr(dgu), d_pitch, _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dwd))
    return dx, dwg, dwu, dwd


def _has_tangent(*tensors: torch.Tensor) -> bool:
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """(silu(x w_gate^T) * (x w_up^T)) w_down^T for x (..., H), w_gate and w_up (I, H), w_down (H, I), all bf16 or all fp16; H and I
    multiples of 8, at most 2^29.  Sums in fp32; the hidden values are rounded to the 16-bit type between the two kernels (they are
    the second product's operand), and so are their gradients in the backward pass: beyond 65504 fp16 ones become infinite.
    Differentiable once in every argument (a second derivative raises, forward-mode ones are refused) for at most 2^26 tokens;
    each gradient that is not needed is not computed.  Those of w_gate and w_up are halves of one buffer: memory is given back
    when neither is held."""
    _check_input(x)
    dt, index = x.dtype, x.get_device()
    hidden = x.shape[-1]
    if w_gate.dtype is not dt or w_up.dtype is not dt or w_down.dtype is not dt:
        raise TypeError(f"the weights must have x's type {dt}, got {w_gate.dtype}, {w_up.dtype}, {w_down.dtype}")
    inter = w_gate.shape[0] if w_gate.dim() else 0
    if w_gate.shape != (inter, hidden) or w_up.shape != (inter, hidden) or w_down.shape != (hidden, inter):
        raise ValueError(f"for x of {hidden} columns the weights must be (I, {hidden}) twice and ({hidden}, I), got {tuple(w_gate.shape)}, "
                         f"{tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if hidden < 8 or inter < 8 or (hidden | inter) & 7 or hidden > _MAX_SIDE or inter > _MAX_SIDE:
        raise ValueError(f"hidden and intermediate sizes must be multiples of 8 up to 2^29, got {hidden} and {inter}")
    if w_gate.get_device() != index or w_up.get_device() != index or w_down.get_device() != index:
        raise ValueError(f"all weights must be on cuda:{index}")
    if _has_tangent(x, w_gate, w_up, w_down):
        raise NotImplementedError("gated_feed_forward has no forward-mode derivative")
    rows = x if x.dim() == 2 else x.reshape(-1, hidden)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        if rows.shape[0] > _MAX_GRAD_TOKENS:
            raise ValueError(f"at most 2^26 tokens where gradients are needed, got {rows.shape[0]}")
        y = _GatedFeedForward.apply(rows, w_gate, w_up, w_down)
    else:
        rows, t, pitch = _rows(rows, hidden)
        y = _ffn_forward(rows, t, pitch, w_gate, w_up, w_down, False)[0]
    return y if x.dim() == 2 else y.reshape(x.shape)
