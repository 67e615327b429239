"""Bindings of the linear cross entropy (``csrc/linear_ce.cu``): scores of a linear head, their softmax statistics and the gradients
of both operands, with the scores kept on chip (forward) or in pieces of the vocabulary (backward).

Operands: hidden states [T, H] and head weight [V, H] in bf16, H a multiple of 64; targets int64 [T].  Every launch goes to the
current stream of the tensors' device; scratch comes from torch's allocator per call, so calls on several streams share nothing."""
from __future__ import annotations

from ctypes import c_float, c_int, c_int64, c_void_p
from functools import lru_cache
from itertools import accumulate
from typing import Optional

import torch

from nanotron_b200.ops import native, native_gemm

# Scores of one piece of the backward pass: 512 MiB of bf16.  Backward pass with 128 | 256 | 512 MiB, us: 4096 x 1024 x 151936 3604 | 3230 | 3051,
# 8192 x 2048 x 128256 11288 | 10143 | 10051, 8192 x 4096 x 128256 20585 | 20487 | 20015 (fewer sums of dx, fuller last rounds of tiles).
PIECE_ELEMENTS = 1 << 28
PIECE_MIN = 4096          # narrowest piece: below it the sums of dx over the pieces cost more than the pieces save


def declare(L):
    L.ntb_linear_ce_forward.restype = c_int
    L.ntb_linear_ce_forward.argtypes = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int, c_int, c_int] + [c_void_p] * 4 + [c_int, c_float, c_void_p, c_int, c_void_p]
    L.ntb_linear_ce_dx_split.restype = c_int
    L.ntb_linear_ce_dx_split.argtypes = [c_int] * 4
    L.ntb_linear_ce_backward.restype = c_int
    L.ntb_linear_ce_backward.argtypes = (
        [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_float, c_int, c_int, c_int, c_int]
        + [c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int64, c_int, c_void_p, c_int, c_void_p]
    )


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


_key = lru_cache(maxsize=None)(str)  # of a device: str(device) takes longer than a launch needs for anything else


def _status(device) -> torch.Tensor:
    word = native_gemm._STATUS.get(_key(device))
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise native.NativeKernelError("the first tensor-core call on a device cannot be captured into a CUDA graph: run it once before the capture")
        word = native_gemm.status_word(device)
    return word


def _sms(device) -> int:
    return native_gemm._SMS.get(_key(device)) or native_gemm._sms(device)


def forward(x2: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, vocab_start: int, finish: bool, z_coef: float = 0.0):
    """Three fp32 [T]; ``finish``: logZ and loss of a whole vocabulary, and z_coef logZ^2 (None when z_coef is 0); otherwise this shard's
    largest score, sum of exp(score - largest), and target score or 0."""
    x2, weight = _rows(x2), _rows(weight)
    (T, H), V, dev = x2.shape, weight.shape[0], x2.device
    with native.on_device(dev):
        status, sms = _status(dev), _sms(dev)
        part = torch.empty((max((V + 255) // 256 * 4, 2 * sms) + 1) * T, dtype=torch.float32, device=dev)  # per part two numbers, and the target's score
        a, b = torch.empty(T, dtype=torch.float32, device=dev), torch.empty(T, dtype=torch.float32, device=dev)
        c = torch.empty(T, dtype=torch.float32, device=dev) if z_coef > 0 or not finish else None
        native._check(native.lib().ntb_linear_ce_forward(x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0), target.data_ptr(), vocab_start, T, V, H, part.data_ptr(),
                                                         a.data_ptr(), b.data_ptr(), None if c is None else c.data_ptr(), finish, z_coef, status.data_ptr(), sms, native.raw_stream(x2)),
                      "linear_ce_forward", launches=2)
    return a, b, c


def piece_width(T: int, V: int) -> int:
    """Vocabulary entries per piece of the backward pass: about PIECE_ELEMENTS scores, pieces of equal width in whole tiles."""
    most = max(PIECE_MIN, PIECE_ELEMENTS // T)
    pieces = (V + most - 1) // most
    return ((V + pieces - 1) // pieces + 255) // 256 * 256


@lru_cache(maxsize=64)
def _backward_plan(T: int, V: int, H: int, sms: int, need_dx: bool, piece_elements: int, piece_min: int):
    """(piece width, pitch of d, chunks of the dx product, words of scratch, word offsets of its parts or None).  Parts, each on a
    1024-byte boundary: d (bf16 [T, pitch]), coefficients (2 T + 1), dx over several pieces (fp32 [T, H]), partial sums of a dx that is cut
    along the vocabulary."""
    width = piece_width(T, V)
    pitch = (min(width, V) + 63) // 64 * 64
    split = native.lib().ntb_linear_ce_dx_split(T, min(width, V), H, sms) if need_dx else 1
    parts = [T * pitch // 2, 2 * T + 1, T * H if need_dx and width < V else 0, split * ((T + 255) // 256) * ((H + 255) // 256) * 65536 if split > 1 else 0]
    ends = list(accumulate((n + 255) // 256 * 256 for n in parts))
    return width, pitch, split, ends[-1], [e - (n + 255) // 256 * 256 if n else None for n, e in zip(parts, ends)]


def backward(x2, weight, target, logz, g, gz: Optional[torch.Tensor], z_coef: float, vocab_start: int, need_dx: bool, need_dw: bool, main_grad: Optional[torch.Tensor] = None):
    """(dx, dw) in bf16 for the upstream gradients ``g`` of the losses and ``gz`` of the terms z_coef logZ^2 (fp32 [T]); with
    ``main_grad`` (fp32 [V, H]) dw is added to it and None is returned in its place."""
    x2, weight = _rows(x2), _rows(weight)
    (T, H), V, dev = x2.shape, weight.shape[0], x2.device
    sms = _sms(dev)
    width, pitch, split, words, offsets = _backward_plan(T, V, H, sms, need_dx, PIECE_ELEMENTS, PIECE_MIN)
    with native.on_device(dev):
        scratch = torch.empty(words, dtype=torch.float32, device=dev)
        base = scratch.data_ptr()
        d, rows, acc, ws = [None if at is None else base + 4 * at for at in offsets]
        dx = torch.empty((T, H), dtype=torch.bfloat16, device=dev) if need_dx else None
        dw = torch.empty((V, H), dtype=torch.bfloat16, device=dev) if need_dw and main_grad is None else None
        into = (dw if main_grad is None else main_grad) if need_dw else None
        rc = native.lib().ntb_linear_ce_backward(
            x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0), target.data_ptr(), vocab_start, logz.data_ptr(), g.data_ptr(), None if gz is None else gz.data_ptr(), z_coef,
            T, V, H, width, d, pitch, rows, None if dx is None else dx.data_ptr(), acc, split, ws, None if into is None else into.data_ptr(), H if into is None else into.stride(0),
            main_grad is not None, _status(dev).data_ptr(), sms, native.raw_stream(x2))
        pieces = (V + width - 1) // width
        native._check(rc, "linear_ce_backward", launches=1 + pieces * (1 + (1 + (split > 1)) * need_dx + need_dw) + (acc is not None))
    return dx, dw
