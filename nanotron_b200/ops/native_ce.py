"""Bindings of the linear cross entropy (``csrc/linear_ce.cu``): scores of a linear head, their softmax statistics and the gradients
of both operands, with the scores kept on chip (forward) or in pieces of the vocabulary (backward).

Operands: hidden states [T, H] and head weight [V, H] in bf16, H a multiple of 64; targets int64 [T].  Every launch goes to the
current stream of the tensors' device; scratch comes from torch's allocator per call, so calls on several streams share nothing."""
from __future__ import annotations

from ctypes import c_int, c_int64, c_void_p
from typing import Optional, Tuple

import torch

PIECE_ELEMENTS = 1 << 27  # scores of one piece of the backward pass: 256 MiB of bf16
PIECE_MIN = 4096          # narrowest piece: below it the sums of dx over the pieces cost more than the pieces save


def declare(L):
    L.ntb_linear_ce_stats.restype = c_int
    L.ntb_linear_ce_stats.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p]
    L.ntb_linear_ce_join.restype = c_int
    L.ntb_linear_ce_join.argtypes = [c_void_p, c_void_p, c_void_p, c_int64, c_int, c_int] + [c_void_p] * 6
    L.ntb_linear_ce_row_coefficients.restype = c_int
    L.ntb_linear_ce_row_coefficients.argtypes = [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p]
    L.ntb_linear_ce_dlogits.restype = c_int
    L.ntb_linear_ce_dlogits.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_int64, c_void_p, c_int, c_void_p]
    L.ntb_linear_ce_dx_split.restype = c_int
    L.ntb_linear_ce_dx_split.argtypes = [c_int] * 4
    L.ntb_linear_ce_dx.restype = c_int
    L.ntb_linear_ce_dx.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int, c_int, c_int, c_int, c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p]
    L.ntb_linear_ce_scale_cast.restype = c_int
    L.ntb_linear_ce_scale_cast.argtypes = [c_void_p, c_void_p, c_void_p, c_int64, c_void_p]
    L.ntb_linear_ce_dw.restype = c_int
    L.ntb_linear_ce_dw.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p]


def check_operands(x2: torch.Tensor, weight: torch.Tensor, target: torch.Tensor) -> None:
    """Raises ValueError where the kernels have no form for the operands."""
    for name, t in (("hidden states", x2), ("weight", weight)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"linear cross entropy on CUDA takes bf16 {name}, got {t.dtype} (other types: apply the head, then sharded_cross_entropy)")
    if x2.shape[1] % 64 or x2.shape[1] == 0:
        raise ValueError(f"linear cross entropy on CUDA needs a hidden size that is a multiple of 64, got {x2.shape[1]}")
    if weight.device != x2.device or target.device != x2.device:
        raise ValueError(f"linear cross entropy: hidden states on {x2.device}, weight on {weight.device}, targets on {target.device}")
    if max(x2.shape[0], weight.shape[0]) >= 1 << 31:
        raise ValueError("linear cross entropy: more than 2^31 - 1 rows")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with rows that the kernels can read in place (contiguous, 16-byte aligned, pitch a multiple of 64), or a copy."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] and t.stride(0) % 64 == 0 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _status(device) -> torch.Tensor:
    from nanotron_b200.ops import native, native_gemm

    if str(device) not in native_gemm._STATUS and torch.cuda.is_current_stream_capturing():
        raise native.NativeKernelError("the first tensor-core call on a device cannot be captured into a CUDA graph: run it once before the capture")
    return native_gemm.status_word(device)


def forward(x2: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, vocab_start: int, finish: bool) -> Tuple[torch.Tensor, ...]:
    """``finish``: (logZ, loss) of a whole vocabulary; otherwise this shard's (max, sum of exp(score - max), target score or 0)."""
    from nanotron_b200.ops import native, native_gemm

    x2, weight = _rows(x2), _rows(weight)
    (T, H), V, dev = x2.shape, weight.shape[0], x2.device
    L, sms = native.lib(), native_gemm._sms(dev)
    with torch.cuda.device(dev):
        status, stream = _status(dev), torch.cuda.current_stream(dev).cuda_stream
        part = torch.empty(((V + 255) // 256 + 1, T, 2), dtype=torch.float32, device=dev)  # the last plane holds the targets' scores
        out = torch.empty((2 if finish else 3, T), dtype=torch.float32, device=dev)
        tgt = part[-1].view(-1)
        native._check(L.ntb_linear_ce_stats(x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0), target.data_ptr(), vocab_start, T, V, H,
                                            part.data_ptr(), tgt.data_ptr(), status.data_ptr(), sms, stream), "linear_ce_stats")
        ptrs = [o.data_ptr() for o in out]
        native._check(L.ntb_linear_ce_join(part.data_ptr(), tgt.data_ptr(), target.data_ptr(), vocab_start, T, V, *((None,) * 3 + tuple(ptrs) if finish else tuple(ptrs) + (None,) * 2), stream),
                      "linear_ce_join")
    return tuple(out.unbind(0))


def piece_width(T: int, V: int) -> int:
    """Vocabulary entries per piece of the backward pass: about PIECE_ELEMENTS scores, pieces of equal width in whole tiles."""
    most = max(PIECE_MIN, PIECE_ELEMENTS // T)
    pieces = (V + most - 1) // most
    return ((V + pieces - 1) // pieces + 255) // 256 * 256


def backward(x2, weight, target, logz, g, gz: Optional[torch.Tensor], vocab_start: int, need_dx: bool, need_dw: bool, main_grad: Optional[torch.Tensor] = None):
    """(dx, dw) in bf16; with ``main_grad`` (fp32 [V, H], contiguous) dw is added to it and None is returned in its place."""
    from nanotron_b200.ops import native, native_gemm

    x2, weight = _rows(x2), _rows(weight)
    (T, H), V, dev = x2.shape, weight.shape[0], x2.device
    L, sms = native.lib(), native_gemm._sms(dev)
    with torch.cuda.device(dev):
        status, stream = _status(dev).data_ptr(), torch.cuda.current_stream(dev).cuda_stream
        width = piece_width(T, V)
        pitch = (min(width, V) + 63) // 64 * 64
        d = torch.empty((T, pitch), dtype=torch.bfloat16, device=dev)
        rows = torch.empty(2 * T + 1, dtype=torch.float32, device=dev)
        coef, gn, unit = rows[:T].data_ptr(), rows[T : 2 * T].data_ptr(), rows[2 * T :].data_ptr()
        dx = torch.empty((T, H), dtype=torch.bfloat16, device=dev) if need_dx else None
        dw = torch.empty((V, H), dtype=torch.bfloat16, device=dev) if need_dw and main_grad is None else None
        acc = torch.empty((T, H), dtype=torch.float32, device=dev) if need_dx and width < V else None
        split = L.ntb_linear_ce_dx_split(T, min(width, V), H, sms) if need_dx else 1
        ws = torch.empty(split * ((T + 255) // 256) * ((H + 255) // 256) * 65536, dtype=torch.float32, device=dev) if split > 1 else None
        native._check(L.ntb_linear_ce_row_coefficients(g.data_ptr(), native._ptr(gz), T, coef, gn, unit, stream), "linear_ce_row_coefficients")
        for v0 in range(0, V, width):
            n = min(width, V - v0)
            w0 = weight.data_ptr() + v0 * weight.stride(0) * 2
            native._check(L.ntb_linear_ce_dlogits(x2.data_ptr(), x2.stride(0), w0, weight.stride(0), target.data_ptr(), vocab_start + v0, logz.data_ptr(), coef, gn,
                                                  T, n, H, d.data_ptr(), pitch, status, sms, stream), "linear_ce_dlogits")
            if need_dx:
                out, mode = (dx, 0) if acc is None else (acc, 1 if v0 == 0 else 2)
                native._check(L.ntb_linear_ce_dx(d.data_ptr(), pitch, w0, weight.stride(0), out.data_ptr(), H, T, n, H, mode, unit, split, native._ptr(ws), status, sms, stream), "linear_ce_dx")
            if need_dw:
                if main_grad is None:
                    out, ld, accumulate = dw.data_ptr() + v0 * H * 2, H, 0
                else:
                    out, ld, accumulate = main_grad.data_ptr() + v0 * main_grad.stride(0) * 4, main_grad.stride(0), 1
                native._check(L.ntb_linear_ce_dw(d.data_ptr(), pitch, x2.data_ptr(), x2.stride(0), out, ld, T, n, H, accumulate, unit, status, sms, stream), "linear_ce_dw")
        if acc is not None:
            native._check(L.ntb_linear_ce_scale_cast(acc.data_ptr(), unit, dx.data_ptr(), T * H, stream), "linear_ce_scale_cast")
    return dx, dw
