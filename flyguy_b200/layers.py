"""The layers around a memory over ticks (flyguy_b200.memory, flyguy_b200.delta):

  layer_norm   rows less their mean, over their deviation, with weight and bias; gradients of all three
  dropout      values dropped by a counter-based generator, added to a residual in the same pass; no mask is kept

They run in the library (fg_layer_norm, fg_dropout of include/flyguy_b200.h) on CUDA tensors, on torch's current stream, and have
gradients (of the first order). Values are float32, bfloat16 or float16; statistics, sums and products are float32, and results
are rounded to the type once."""
from __future__ import annotations

import struct
from functools import lru_cache

import torch

from .memory import TYPES, _call, _float32, _kept, _no_tangents, _once, _ptr, _room
from .native import FlyguyError, lib

# fg_norm_args: x, y, gy, gx, w, b, gw, gb, rows, dim, x_row, gy_row, type, eps, work, work_bytes
_NORM = struct.Struct("=13qd2q")
# fg_dropout_args: x, add, y, seed, seed_value, call, n, least, type
_DROPOUT = struct.Struct("=9q")


def _tensor(name: str, t, like=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise FlyguyError(f"{name} must be a CUDA tensor (flyguy_b200 has no CPU path)")
    if t.dtype not in TYPES:
        raise FlyguyError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if like is not None and (t.dtype is not like.dtype or t.shape != like.shape or t.get_device() != like.get_device()):
        raise FlyguyError(f"{name} must have the type, shape and device of x: {tuple(like.shape)}, not {tuple(t.shape)}")
    return t


# ---- layer norm ----------------------------------------------------------------------------------------------------

def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t as rows that lie at equal distances, and that distance in values; copied if they do not."""
    dim = t.shape[-1]
    if t.is_contiguous():
        return t, dim
    shape, stride = t.shape, t.stride()
    if (stride[-1] == 1 or dim == 1) and t.dim() > 1:
        step = stride[-2] if shape[-2] > 1 else None
        at, even = (step or 0) * shape[-2], True
        for n, s in zip(shape[-3::-1], stride[-3::-1]):      # each dimension goes on where the one inside it ends
            if n > 1:
                if step is None:
                    step = at = s
                elif s != at:
                    even = False
                at = s * n
        if even and step is not None and step >= 0:
            return t, step
    return t.contiguous(), dim


class _Norm:
    """What forward and backward of one call share."""

    def __init__(self, x, eps):
        self.dim, self.eps, self.type, self.device = x.shape[-1], eps, TYPES[x.dtype], x.get_device()
        self.rows = x.numel() // self.dim if self.dim else 0

    def forward(self, x, w, b):
        x, step = _rows(x)
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        _call(lib().fg_layer_norm, _NORM.pack(x.data_ptr(), y.data_ptr(), 0, 0, _ptr(w), _ptr(b), 0, 0, self.rows, self.dim, step, 0, self.type,
                                              self.eps, 0, 0), self.device)
        return y

    def backward(self, x, w, b, gy, want_w, want_b):
        (x, x_row), (gy, gy_row) = _rows(x), _rows(gy if gy.dtype is x.dtype else gy.to(x.dtype))
        gx = torch.empty_like(x, memory_format=torch.contiguous_format)
        gw = torch.empty_like(w) if want_w else None
        gb = torch.empty_like(b) if want_b else None
        room, work = None, (0, 0)
        if want_w or want_b:
            room, work = _room(_norm_room(self.rows, self.dim), x.device)
        _call(lib().fg_layer_norm_bwd, _NORM.pack(x.data_ptr(), 0, gy.data_ptr(), gx.data_ptr(), _ptr(w), 0, _ptr(gw), _ptr(gb), self.rows, self.dim,
                                                  x_row, gy_row, self.type, self.eps, *work), self.device)
        return gx, gw, gb


@lru_cache(maxsize=256)
def _norm_room(rows: int, dim: int) -> int:
    """Bytes of workspace for the sums of so many rows (fg_layer_norm_work; the same for all types)."""
    size = lib().fg_layer_norm_work(_NORM.pack(0, 0, 0, 0, 0, 0, 1, 1, rows, dim, dim, dim, 0, 1.0, 0, 0))
    if size < 0:                                          # (raised here: an error is not kept)
        raise FlyguyError(lib().fg_mem_last_error().decode())
    return size


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, job):
        y = job.forward(x, w, b)
        ctx.job = job
        ctx.save_for_backward(_kept(x), _kept(w), _kept(b))
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, w, b = ctx.saved_tensors
        return *ctx.job.backward(x, w, b, gy, *ctx.needs_input_grad[1:3]), None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias over the last dimension of x [.., dim], any strides (rows that
    do not lie at equal distances are copied first). weight and bias: float32 [dim] or None. Gradients of x, weight and bias;
    the sums over rows are the same bits on every run. A NaN or an infinity makes its whole row NaN."""
    x = _tensor("x", x)
    if x.dim() < 1 or not x.shape[-1]:
        raise FlyguyError("x must have a last dimension to norm over")
    if not eps > 0:
        raise FlyguyError(f"eps must be positive, not {eps}")
    if weight is not None:
        weight = _float32("weight", weight, x, x.shape[-1:])
    if bias is not None:
        bias = _float32("bias", bias, x, x.shape[-1:])
    _no_tangents(x, weight, bias)
    job = _Norm(x, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _NormFn.apply(x, weight, bias, job)
    return job.forward(x, weight, bias)


# ---- dropout -------------------------------------------------------------------------------------------------------

class _Drop:
    """The mask of one call: where the generator begins, and what it leaves."""

    def __init__(self, x, p, seed, call):
        self.least, self.call, self.device = round(p * 65536), call, x.get_device()
        self.seed, self.value = (seed, 0) if isinstance(seed, torch.Tensor) else (None, seed)

    def run(self, x, add=None):
        x = x.contiguous()
        add = None if add is None else add.contiguous()
        y = torch.empty_like(x)
        _call(lib().fg_dropout, _DROPOUT.pack(x.data_ptr(), _ptr(add), y.data_ptr(), _ptr(self.seed), self.value, self.call, x.numel(),
                                              self.least, TYPES[x.dtype]), self.device)
        return y

    def let_go(self):
        kept, self.seed = _kept(self.seed), None
        return kept

    def take_up(self, seed):
        again = object.__new__(_Drop)
        again.__dict__.update(self.__dict__, seed=seed)
        return again


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, add, job):
        y = job.run(x, add)
        ctx.job = job
        ctx.save_for_backward(job.let_go())
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        want_x, want_add = ctx.needs_input_grad[:2]
        return ctx.job.take_up(*ctx.saved_tensors).run(gy) if want_x else None, gy if want_add else None, None


def dropout(x, p: float, seed, call: int = 0, add=None) -> torch.Tensor:
    """x / (1 - p) where a random number leaves it, 0 elsewhere (also for a NaN), added to `add` (of x's shape and type) if given.

    The random numbers are a function of seed, call and a value's place in x: value i takes 16 bits of block i / 8 of
    Philox4x32-10 with the key `seed` and the counter (block, call). So the mask is never kept (the gradient makes it again), and a
    seed and call used twice give the same mask: count calls. seed: an int of 64 bits, or an int64 tensor of one element on
    x's device, read when the kernel runs (a captured graph may be replayed with another; it may not change between a call and
    its backward). p is taken to the nearest 1 / 65536, and at most 65535 / 65536."""
    x = _tensor("x", x)
    if add is not None:
        add = _tensor("add", add, x)
    if not 0 <= p < 1 or round(p * 65536) > 65535:
        raise FlyguyError(f"p must be 0 to 65535 / 65536, not {p}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.get_device() != x.get_device():
            raise FlyguyError(f"seed must be an int or an int64 tensor of one element on {x.device}")
    elif not isinstance(seed, int) or not -(1 << 63) <= seed < 1 << 63:
        raise FlyguyError("seed must be an int of 64 bits, or an int64 tensor of one element")
    if not isinstance(call, int) or not 0 <= call < 1 << 63:
        raise FlyguyError(f"call must be an int of 0 to 2^63 - 1, not {call!r}")
    _no_tangents(x, add)
    job = _Drop(x, p, seed, call)
    if torch.is_grad_enabled() and (x.requires_grad or (add is not None and add.requires_grad)):
        return _DropoutFn.apply(x, add, job)
    return job.run(x, add)
