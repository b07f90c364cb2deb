"""Training and serving low-rank adapters on a packed (cdclq-v1) model, on the GPU engine.

The operators that a quantized model needs once its weights are frozen:

  PackedLinear, Adapters                 a packed layer laid out for products; adapters A, B of one layer
  adapter_linear / _backward             the packed projection with each token's adapter beside it
  checkpoint_save / checkpoint_restore   a layer's input kept in 8 bits until the backward pass
  vocab_loss / vocab_loss_backward       softmax cross entropy over a large vocabulary and its
                                         gradient, without the logits in memory
  linear, cross_entropy                  the same as differentiable functions of torch's autograd

Tensors are torch tensors on the context's GPU, bfloat16 or float16, with contiguous rows (any row
stride). Every call is enqueued on torch's current stream and returns without waiting; scratch
memory comes from torch's allocator, so that calls may be made on several streams and captured into
a graph. A refused argument raises CdclqError (or TypeError / ValueError for a tensor of the wrong
kind) before anything is enqueued.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np
import torch

from . import DTYPE_BF16, DTYPE_F16, Context, check_row_width, lib as _L

BLOCK = 128  # features per scale of an 8-bit checkpoint
_CODES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}


_empty = torch.empty
_current_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: a Stream object costs a microsecond


def _code(x: torch.Tensor, name: str) -> int:
    c = _CODES.get(x.dtype)
    if c is None:
        raise TypeError(f"{name} is {x.dtype}, need bfloat16 or float16")
    return c


def _matrix(ctx: Context, x: torch.Tensor, name: str, dtype=None, rows=None, cols=None) -> int:
    """Checks a 2-D tensor with contiguous rows on ctx's GPU; returns its row stride."""
    if x.get_device() != ctx.device:
        raise ValueError(f"{name} is on {x.device}, the context on cuda:{ctx.device}")
    shape = x.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        want = f"{'rows' if rows is None else rows} x {'columns' if cols is None else cols}"
        raise ValueError(f"{name} has shape {tuple(shape)}, need {want}")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{name} is {x.dtype}, need {dtype}")
    r, c = x.stride()
    n = shape[1]
    if (c != 1 and n > 1) or (r < n and shape[0] > 1):
        raise ValueError(f"{name} has strides {(r, c)}; its rows must be contiguous")
    return r if r > n else n


def _vector(ctx: Context, x: torch.Tensor, name: str, dtype, n: int):
    if x.get_device() != ctx.device:
        raise ValueError(f"{name} is on {x.device}, the context on cuda:{ctx.device}")
    if x.dtype != dtype:
        raise TypeError(f"{name} is {x.dtype}, need {dtype}")
    if x.shape != (n,) or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} values, got shape {tuple(x.shape)}")


def _stream(ctx: Context) -> int:
    return _current_stream(ctx.device)


def _work(n: int, device) -> torch.Tensor:
    return _empty(n, dtype=torch.uint8, device=device)


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
    codes = _empty(t, n, dtype=torch.int8, device=x.device)
    scales = _empty(t, -(-n // BLOCK), dtype=torch.float32, device=x.device)
    ctx.check(_L().cdclq_checkpoint_save_device(ctx.ptr, x.data_ptr(), ld, t, n, code, codes.data_ptr(),
                                                 scales.data_ptr(), _stream(ctx)))
    return Checkpoint(codes, scales, x.dtype)


def _check_saved(ctx: Context, ck: Checkpoint, rows=None, cols=None):
    _matrix(ctx, ck.codes, "codes", torch.int8, rows, cols)
    t, n = ck.codes.shape
    _matrix(ctx, ck.scales, "scales", torch.float32, t, -(-n // BLOCK))
    if not (ck.codes.is_contiguous() and ck.scales.is_contiguous()):
        raise ValueError("codes and scales must be contiguous")


def checkpoint_restore(ctx: Context, ck: Checkpoint) -> torch.Tensor:
    """The activation that a checkpoint holds, scale * code, in its own type."""
    _check_saved(ctx, ck)
    t, n = ck.codes.shape
    out = _empty(t, n, dtype=ck.dtype, device=ck.codes.device)
    ctx.check(_L().cdclq_checkpoint_restore_device(ctx.ptr, ck.codes.data_ptr(), ck.scales.data_ptr(), t, n,
                                                    _code(out, "out"), out.data_ptr(), n, _stream(ctx)))
    return out


# ---------------------------------------------------------------- packed projection with adapters
class PackedLinear:
    """A packed (cdclq-v1) layer laid out once for products: qweight (uint8, d_out x row bytes), scales
    (float16, or their uint16 bit patterns), qzeros (uint8), perm (int32), as torch tensors on the
    context's GPU or as the host arrays of packed_tensors(); gbits (uint8 per group) and the group
    size. The tensors are not needed afterwards."""

    def __init__(self, ctx: Context, qweight, scales, qzeros, perm, gbits, group: int):
        self.ptr = None
        self.ctx = ctx
        dev = torch.device("cuda", ctx.device)

        def put(a, kinds, name):
            if isinstance(a, np.ndarray) and a.dtype == np.uint16:
                a = a.view(np.float16)
            t = torch.as_tensor(a)
            if t.dtype not in kinds:
                raise TypeError(f"{name} is {t.dtype}, need {kinds[0]}")
            return t.to(dev).contiguous()

        qw, s16 = put(qweight, (torch.uint8,), "qweight"), put(scales, (torch.float16,), "scales")
        qz, p32 = put(qzeros, (torch.uint8,), "qzeros"), put(perm, (torch.int32,), "perm")
        gb = np.ascontiguousarray(gbits.cpu().numpy() if isinstance(gbits, torch.Tensor) else gbits, np.uint8)
        if qw.dim() != 2 or p32.dim() != 1 or tuple(s16.shape) != (qw.shape[0], gb.size) or qz.shape != s16.shape:
            raise ValueError(f"qweight {tuple(qw.shape)}, scales {tuple(s16.shape)}, qzeros {tuple(qz.shape)} and "
                             f"{gb.size} groups do not belong together")
        self.d_out, self.d_in = qw.shape[0], p32.shape[0]
        check_row_width(qw.shape[1], self.d_in, int(group), gb)
        torch.cuda.current_stream(dev).synchronize()
        out = C.c_void_p()
        ctx.check(_L().cdclq_packed_open_device(ctx.ptr, self.d_out, self.d_in, int(group), gb.ctypes.data, gb.size,
                                                 qw.data_ptr(), qw.numel(), s16.data_ptr(), qz.data_ptr(),
                                                 p32.data_ptr(), C.byref(out)))
        self.ptr = out

    @classmethod
    def from_tensors(cls, ctx: Context, tensors: dict, layer: str) -> "PackedLinear":
        """From a dict in the packed_tensors() form, or of a packed shard's tensors."""
        def get(suffix):
            v = tensors[f"{layer}.{suffix}"]
            return v[1] if isinstance(v, tuple) else v
        return cls(ctx, get("qweight"), get("scales"), get("qzeros"), get("perm"), get("gbits"),
                   int(np.asarray(get("gsize")).ravel()[0]))

    def nbytes(self) -> int:
        """Device memory that the layer holds."""
        return _L().cdclq_packed_bytes(self.ptr)

    def close(self):
        if getattr(self, "ptr", None):
            _L().cdclq_packed_close(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Adapters:
    """The low-rank adapters of one layer: a (R x rank x d_in), b (R x d_out x rank), both contiguous
    and of one 16-bit type, scaling (float32, R). Adapters of smaller rank are padded with zeros."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor):
        _code(a, "a")
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} are not R x rank x d_in and R x d_out x rank")
        if b.dtype != a.dtype or scaling.dtype != torch.float32:
            raise TypeError(f"a is {a.dtype}, b {b.dtype}, scaling {scaling.dtype}; need one 16-bit type and float32")
        if tuple(scaling.shape) != (a.shape[0],) or not (a.is_contiguous() and b.is_contiguous() and
                                                         scaling.is_contiguous()):
            raise ValueError("a, b and scaling (one value per adapter) must be contiguous")
        if not (a.device == b.device == scaling.device):
            raise ValueError("a, b and scaling are on different devices")
        self.a, self.b, self.scaling = a, b, scaling
        self.count, self.rank, self.d_in = a.shape
        self.d_out = b.shape[1]


def _adapter_args(packed: PackedLinear, x, adapters, request, name: str):
    """(a, b, scaling, count, rank, request) addresses after checks against the layer."""
    if adapters is None:
        if request is not None:
            raise ValueError("request without adapters")
        return None, None, None, 0, 0, None
    a = adapters.a
    if a.get_device() != x.get_device() or a.dtype != x.dtype:
        raise TypeError(f"the adapters are {a.dtype} on {a.device}, {name} is {x.dtype} on {x.device}")
    if adapters.d_in != packed.d_in or adapters.d_out != packed.d_out:
        raise ValueError(f"adapters of a {adapters.d_out} x {adapters.d_in} layer, the packed layer is "
                         f"{packed.d_out} x {packed.d_in}")
    if request is None:
        raise ValueError("adapters need the request of each token")
    _vector(packed.ctx, request, "request", torch.int32, x.shape[0])
    return (a.data_ptr(), adapters.b.data_ptr(), adapters.scaling.data_ptr(), adapters.count, adapters.rank,
            request.data_ptr())


def adapter_linear(packed: PackedLinear, x: torch.Tensor, adapters: Adapters | None = None,
                   request: torch.Tensor | None = None, return_low: bool = False):
    """y (T x d_out) = x W^T with each token's adapter beside it: y_t = W x_t + scaling[q] B_q (A_q x_t),
    q = request[t] (int32, -1: none). With return_low also low = A_q x_t (T x rank, float32), which the
    backward pass takes. The requests may come in any order; calls of more than 192 tokens and the backward
    pass are faster when the tokens of an adapter stand together.

    Up to 192 tokens the weights are exact; in larger calls, and in every backward pass, each weight is rounded
    to x's type (so a token's bits differ between the two; split a call where that matters). The time and the
    workspace of such calls go by all adapters of the set, with or without tokens."""
    ctx = packed.ctx
    code, ld = _code(x, "x"), _matrix(ctx, x, "x", None, None, packed.d_in)
    t = x.shape[0]
    a, b, s, count, rank, req = _adapter_args(packed, x, adapters, request, "x")
    L = _L()
    y = _empty(t, packed.d_out, dtype=x.dtype, device=x.device)
    low = _empty(t, rank, dtype=torch.float32, device=x.device) if return_low else None
    xp = x.data_ptr()
    work = _work(L.cdclq_adapter_work_bytes(packed.ptr, xp, ld, t, a, b, count, rank, 0), x.device)
    ctx.check(L.cdclq_adapter_linear_device(ctx.ptr, packed.ptr, xp, ld, t, code, a, b, s, count, rank, req,
                                            y.data_ptr(), packed.d_out, low.data_ptr() if return_low else None,
                                            work.data_ptr(), work.numel(), _stream(ctx)))
    return (y, low) if return_low else y


def adapter_linear_backward(packed: PackedLinear, dy: torch.Tensor, saved: Checkpoint | None = None,
                            low: torch.Tensor | None = None, adapters: Adapters | None = None,
                            request: torch.Tensor | None = None):
    """The gradient of adapter_linear for dy (T x d_out): (dx, da, db). saved is checkpoint_save of its
    x, low what adapter_linear returned. W is frozen. Without adapters da and db are None."""
    ctx = packed.ctx
    code, ld = _code(dy, "dy"), _matrix(ctx, dy, "dy", None, None, packed.d_out)
    t = dy.shape[0]
    a, b, s, count, rank, req = _adapter_args(packed, dy, adapters, request, "dy")
    L = _L()
    dx = _empty(t, packed.d_in, dtype=dy.dtype, device=dy.device)
    da = db = codes = scales = lp = None
    if rank:
        if saved is None or low is None:
            raise ValueError("the adapters' gradient needs the saved input and low")
        _check_saved(ctx, saved, t, packed.d_in)
        _matrix(ctx, low, "low", torch.float32, t, rank)
        if not low.is_contiguous():
            raise ValueError("low must be contiguous")
        codes, scales, lp = saved.codes.data_ptr(), saved.scales.data_ptr(), low.data_ptr()
        da, db = torch.empty_like(adapters.a), torch.empty_like(adapters.b)
    dyp = dy.data_ptr()
    work = _work(L.cdclq_adapter_work_bytes(packed.ptr, dyp, ld, t, a, b, count, rank, 1), dy.device)
    ctx.check(L.cdclq_adapter_backward_device(ctx.ptr, packed.ptr, dyp, ld, t, code, codes, scales, lp, a, b, s, count,
                                              rank, req, dx.data_ptr(), packed.d_in, da.data_ptr() if rank else None,
                                              db.data_ptr() if rank else None, work.data_ptr(), work.numel(),
                                              _stream(ctx)))
    return dx, da, db


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
    L = _L()
    out = _empty(2, t, dtype=torch.float32, device=x.device)
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
    L = _L()
    dx = _empty(t, d, dtype=x.dtype, device=x.device)
    dw = _empty(v, d, dtype=w.dtype, device=x.device) if need_dw else None
    work = _work(L.cdclq_vocab_work_bytes(t, d, v, w.data_ptr(), ldw, 1), x.device)
    ctx.check(L.cdclq_vocab_loss_backward_device(ctx.ptr, x.data_ptr(), ldx, w.data_ptr(), ldw, t, d, v, code,
                                                 targets.data_ptr(), ignore_index, lse.data_ptr(), dloss.data_ptr(),
                                                 dx.data_ptr(), d, dw.data_ptr() if need_dw else None, d,
                                                 work.data_ptr(), work.numel(), _stream(ctx)))
    return dx, dw


# ---------------------------------------------------------------- as differentiable functions
def _first_order(backward):
    """A backward pass that has no gradient of its own and refuses to take part in a graph (create_graph). Its
    results would count there as constants and lose terms without a word; an error tied to them, as torch's
    once_differentiable makes, is reached only where the graph happens to lead through it."""
    def run(fn, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("cdclq.tune: linear and cross_entropy have gradients of first order only "
                               "(create_graph is not supported)")
        return backward(fn, *grads)
    return run


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(fn, x, a, b, scaling, packed, adapters, request):
        fn.packed, fn.has_adapters = packed, adapters is not None
        if adapters is None:
            fn.save_for_backward()
            return adapter_linear(packed, x, None, request)
        y, low = adapter_linear(packed, x, adapters, request, return_low=True)
        ck = checkpoint_save(packed.ctx, x)
        fn.dtype = x.dtype
        fn.save_for_backward(ck.codes, ck.scales, low, request, a, b, scaling)
        return y

    @staticmethod
    @_first_order
    def backward(fn, dy):
        dy = dy.contiguous()
        if not fn.has_adapters:
            return adapter_linear_backward(fn.packed, dy)[0], None, None, None, None, None, None
        # the operands of the forward call, whatever the Adapters hold by now; changed in place is an error here
        codes, scales, low, request, a, b, scaling = fn.saved_tensors
        dx, da, db = adapter_linear_backward(fn.packed, dy, Checkpoint(codes, scales, fn.dtype), low,
                                             Adapters(a, b, scaling), request)
        return dx, da, db, None, None, None, None


def linear(packed: PackedLinear, x: torch.Tensor, adapters: Adapters | None = None,
           request: torch.Tensor | None = None) -> torch.Tensor:
    """adapter_linear for autograd: gradients of x and of adapters.a and .b, of first order only; between the
    passes x is kept as an 8-bit checkpoint. scaling is a constant."""
    wanted = (x,) if adapters is None else (x, adapters.a, adapters.b, adapters.scaling)
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in wanted)):
        return adapter_linear(packed, x, adapters, request)  # no checkpoint, no low
    if adapters is None:
        return _Linear.apply(x, None, None, None, packed, None, request)
    if adapters.scaling.requires_grad:
        raise ValueError("scaling asks for a gradient; linear has none for it")
    return _Linear.apply(x, adapters.a, adapters.b, adapters.scaling, packed, adapters, request)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(fn, x, w, ctx, targets, ignore_index):
        loss, lse = vocab_loss(ctx, x, w, targets, ignore_index)
        weight = 1.0 / (targets != ignore_index).sum().clamp(min=1).float()
        fn.save_for_backward(x, w, targets, lse, weight)
        fn.ctx, fn.ignore_index = ctx, ignore_index
        return loss.sum() * weight

    @staticmethod
    @_first_order
    def backward(fn, grad):
        x, w, targets, lse, weight = fn.saved_tensors
        dloss = (grad * weight).float().expand(len(x)).contiguous()
        dx, dw = vocab_loss_backward(fn.ctx, x, w, targets, lse, dloss, fn.ignore_index, fn.needs_input_grad[1])
        return dx, dw, None, None, None


def cross_entropy(ctx: Context, x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor,
                  ignore_index: int = -100) -> torch.Tensor:
    """The mean of vocab_loss over the tokens that take part (0 if none does), for autograd: gradients (of
    first order only) of x and, where w asks for it, of w."""
    return _CrossEntropy.apply(x, w, ctx, targets, ignore_index)
