"""Training and serving low-rank adapters on a packed (cdclq-v1) model, on the GPU engine.

The operators that a quantized model needs once its weights are frozen:

  checkpoint_save / checkpoint_restore   a layer's input kept in 8 bits until the backward pass
  vocab_loss / vocab_loss_backward       softmax cross entropy over a large vocabulary and its
                                         gradient, without the logits in memory

Tensors are torch tensors on the context's GPU, bfloat16 or float16, with contiguous rows (any row
stride). Every call is enqueued on torch's current stream and returns without waiting; scratch
memory comes from torch's allocator, so that calls may be made on several streams and captured into
a graph. A refused argument raises CdclqError (or TypeError / ValueError for a tensor of the wrong
kind) before anything is enqueued.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import DTYPE_BF16, DTYPE_F16, CdclqError, Context, lib

BLOCK = 128  # features per scale of an 8-bit checkpoint
_CODES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}


def _code(x: torch.Tensor, name: str) -> int:
    if x.dtype not in _CODES:
        raise TypeError(f"{name} is {x.dtype}, need bfloat16 or float16")
    return _CODES[x.dtype]


def _matrix(ctx: Context, x: torch.Tensor, name: str, dtype=None, rows=None, cols=None) -> int:
    """Checks a 2-D tensor with contiguous rows on ctx's GPU; returns its row stride."""
    if not x.is_cuda or x.device.index != ctx.device:
        raise ValueError(f"{name} is on {x.device}, the context on cuda:{ctx.device}")
    if x.dim() != 2 or (rows is not None and x.shape[0] != rows) or (cols is not None and x.shape[1] != cols):
        want = f"{'rows' if rows is None else rows} x {'columns' if cols is None else cols}"
        raise ValueError(f"{name} has shape {tuple(x.shape)}, need {want}")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{name} is {x.dtype}, need {dtype}")
    r, c = x.stride()
    if (c != 1 and x.shape[1] > 1) or (r < x.shape[1] and x.shape[0] > 1):
        raise ValueError(f"{name} has strides {(r, c)}; its rows must be contiguous")
    return max(r, x.shape[1])


def _vector(ctx: Context, x: torch.Tensor, name: str, dtype, n: int):
    if not x.is_cuda or x.device.index != ctx.device:
        raise ValueError(f"{name} is on {x.device}, the context on cuda:{ctx.device}")
    if x.dtype != dtype:
        raise TypeError(f"{name} is {x.dtype}, need {dtype}")
    if tuple(x.shape) != (n,) or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} values, got shape {tuple(x.shape)}")


def _stream(ctx: Context) -> int:
    return torch.cuda.current_stream(ctx.device).cuda_stream


def _work(n: int, device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


# ---------------------------------------------------------------- 8-bit activation checkpoints
@dataclass
class Checkpoint:
    """An activation in 8 bits: codes (int8, T x n), one float32 scale per token and block of 128
    features, and the type it had."""

    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype


def checkpoint_save(ctx: Context, x: torch.Tensor) -> Checkpoint:
    """x (T x n) in 8 bits: scale = max |x| / 127 per block of 128 features, code = x / scale
    rounded to nearest, ties to even. A block with a NaN or an infinity is restored as NaN."""
    code, ld = _code(x, "x"), _matrix(ctx, x, "x")
    t, n = x.shape
    codes = torch.empty(t, n, dtype=torch.int8, device=x.device)
    scales = torch.empty(t, -(-n // BLOCK), dtype=torch.float32, device=x.device)
    ctx.check(lib().cdclq_checkpoint_save_device(ctx.ptr, x.data_ptr(), ld, t, n, code, codes.data_ptr(),
                                                 scales.data_ptr(), _stream(ctx)))
    return Checkpoint(codes, scales, x.dtype)


def _check_saved(ctx: Context, ck: Checkpoint, rows=None, cols=None):
    if _matrix(ctx, ck.codes, "codes", torch.int8, rows, cols) != ck.codes.shape[1]:
        raise ValueError("codes must be contiguous")
    t, n = ck.codes.shape
    if _matrix(ctx, ck.scales, "scales", torch.float32, t, -(-n // BLOCK)) != ck.scales.shape[1]:
        raise ValueError("scales must be contiguous")


def checkpoint_restore(ctx: Context, ck: Checkpoint) -> torch.Tensor:
    """The activation that a checkpoint holds, scale * code, in its own type."""
    _check_saved(ctx, ck)
    t, n = ck.codes.shape
    out = torch.empty(t, n, dtype=ck.dtype, device=ck.codes.device)
    ctx.check(lib().cdclq_checkpoint_restore_device(ctx.ptr, ck.codes.data_ptr(), ck.scales.data_ptr(), t, n,
                                                    _code(out, "out"), out.data_ptr(), n, _stream(ctx)))
    return out


# ---------------------------------------------------------------- cross entropy over a vocabulary
def _loss_args(ctx: Context, x, w, targets):
    code, ldx = _code(x, "x"), _matrix(ctx, x, "x")
    t, d = x.shape
    ldw = _matrix(ctx, w, "w", x.dtype, None, d)
    _vector(ctx, targets, "targets", torch.int64, t)
    return code, ldx, ldw, t, d, w.shape[0]


def vocab_loss(ctx: Context, x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100):
    """Softmax cross entropy of each token over the logits x w^T (x T x d hidden states, w V x d head
    weights, targets int64): (loss, lse), float32 vectors. A token whose target is ignore_index has
    loss = lse = 0 and does not take part; any other target outside 0..V gives a NaN loss."""
    code, ldx, ldw, t, d, v = _loss_args(ctx, x, w, targets)
    L = lib()
    out = torch.empty(2, t, dtype=torch.float32, device=x.device)
    loss, lse = out[0], out[1]
    work = _work(L.cdclq_vocab_work_bytes(t, d, v, w.data_ptr(), ldw, 0), x.device)
    ctx.check(L.cdclq_vocab_loss_device(ctx.ptr, x.data_ptr(), ldx, w.data_ptr(), ldw, t, d, v, code,
                                        targets.data_ptr(), ignore_index, loss.data_ptr(), lse.data_ptr(),
                                        work.data_ptr(), work.numel(), _stream(ctx)))
    return loss, lse


def vocab_loss_backward(ctx: Context, x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                        dloss: torch.Tensor, ignore_index: int = -100, need_dw: bool = True):
    """The gradient of vocab_loss for dloss (float32, one weight per token: 1 / N for a mean):
    (dx, dw), dw None unless need_dw. lse is vocab_loss's. dx is 0 at ignored tokens."""
    code, ldx, ldw, t, d, v = _loss_args(ctx, x, w, targets)
    _vector(ctx, lse, "lse", torch.float32, t)
    _vector(ctx, dloss, "dloss", torch.float32, t)
    L = lib()
    dx = torch.empty(t, d, dtype=x.dtype, device=x.device)
    dw = torch.empty(v, d, dtype=w.dtype, device=x.device) if need_dw else None
    work = _work(L.cdclq_vocab_work_bytes(t, d, v, w.data_ptr(), ldw, 1), x.device)
    ctx.check(L.cdclq_vocab_loss_backward_device(ctx.ptr, x.data_ptr(), ldx, w.data_ptr(), ldw, t, d, v, code,
                                                 targets.data_ptr(), ignore_index, lse.data_ptr(), dloss.data_ptr(),
                                                 dx.data_ptr(), d, dw.data_ptr() if need_dw else None, d,
                                                 work.data_ptr(), work.numel(), _stream(ctx)))
    return dx, dw
