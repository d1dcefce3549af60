"""A memory over ticks beside the fly actor. The reference's actor answers each tick from that tick's observation alone
(FlyActor.memory = 0, flyguy/fly.py:76); the operators here carry what earlier ticks showed, learned on whole recordings
at once and played a tick at a time with a state of fixed size:

  rotary_turns      the rotation's plan: a tick's angle of each pair of a head's values
  rotate            queries or keys turned by their position
  norm_rotate       the norms of queries and keys for each head and the rotation in one pass
  decay_attention   linear attention with a decay for each head over whole recordings (also packed end to end)
  decay_step        the same for one tick, the states updated in place
  sync              waits for their work and tells whether a kernel gave up

They run in the library (fg_norm_rotate, fg_decay_attn, fg_decay_step of include/flyguy_b200.h) on CUDA tensors, on
torch's current stream; rotate, norm_rotate and decay_attention have gradients (of the first order). TickMemory puts them
together.

Queries, keys and values are float32, bfloat16 or float16 of one type, [batch, ticks, heads, dim] or, for recordings packed
end to end, [ticks, heads, dim]; any strides with a head's values adjacent (others are copied first). Norms, sums,
states and decays are float32, and results are rounded to the type once. decay_attention of bfloat16 on the tensor cores (dims
of multiples of 16 up to 128, 16-byte strides) rounds two operands on the way, too, each once: the weights within a tile of 128
ticks and the copy of the state that a tile's queries meet. Each is of the size of the result's own rounding, so that results are
2.3e-3 of their norm off where that rounding alone is 1.7e-3. What is carried from tile to tile stays float32.
"""
from __future__ import annotations

import math
import struct
from decimal import Decimal, localcontext
from functools import lru_cache, wraps

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .native import FlyguyError, lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
LAYOUTS = {"half": 0, "interleaved": 1}
_PI = Decimal("3.14159265358979323846264338327950288419716939937510")


# ---- argument checks and the library's argument structures ----------------------------------------------------------

def _values(name: str, t, dims: tuple[int, ...], like=None) -> torch.Tensor:
    """t as the library takes it; its last dimension made adjacent if it is not."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise FlyguyError(f"{name} must be a CUDA tensor (flyguy_b200 has no CPU path)")
    if t.dtype not in TYPES:
        raise FlyguyError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.dim() not in dims:
        raise FlyguyError(f"{name} must have {' or '.join(map(str, dims))} dimensions, not {t.dim()}")
    if like is not None and (t.dtype is not like.dtype or t.dim() != like.dim() or t.get_device() != like.get_device()):
        raise FlyguyError(f"{name} must have the type, device and number of dimensions of the first tensor")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _float32(name: str, t, like: torch.Tensor, *shapes) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != like.get_device():
        raise FlyguyError(f"{name} must be a float32 tensor on {like.device}")
    if t.shape not in shapes:
        raise FlyguyError(f"{name} must be {' or '.join(map(str, map(tuple, shapes)))}, not {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _state(t: torch.Tensor | None) -> torch.Tensor | None:
    """A state, or its gradient, as the kernels read it fastest: contiguous, from a 16-byte boundary on."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ticks(t: torch.Tensor) -> tuple[int, int, int, int]:
    """fg_ticks of [batch, ticks, heads, dim] or [ticks, heads, dim]."""
    st = t.stride()
    return (t.data_ptr(), st[0], st[1], st[2]) if len(st) == 4 else (t.data_ptr(), 0, st[0], st[1])


def _no_tangents(*tensors) -> None:
    """Tangents would be dropped: they are refused."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise FlyguyError("the memory operators have no forward-mode derivatives")


_NONE = (0, 0, 0, 0)
_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice   # (torch.cuda's own, without its objects)


def _kept(t: torch.Tensor | None) -> torch.Tensor | None:
    """t for autograd to keep (it keeps none that was made in inference mode)."""
    return t.clone() if t is not None and t.is_inference() else t


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _call(fn, packed: bytes, device: int) -> None:
    """fn(arguments, the current stream) on the tensors' device."""
    if _device() != device:
        with torch.cuda.device(device):
            rc = fn(packed, _raw_stream(device))
    else:
        rc = fn(packed, _raw_stream(device))
    if rc:
        raise FlyguyError(lib().fg_mem_last_error().decode())


def _room(size: int, device) -> tuple[torch.Tensor | None, tuple[int, int]]:
    """A workspace of so many bytes, and its fields in an argument structure."""
    if size < 0:
        raise FlyguyError(lib().fg_mem_last_error().decode())
    if not size:
        return None, (0, 0)
    t = torch.empty(size, dtype=torch.uint8, device=device)
    return t, (t.data_ptr(), size)


def _offsets(t, like: torch.Tensor) -> torch.Tensor:
    """The first ticks of recordings packed end to end, as the library takes them."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int64 or t.get_device() != like.get_device() or t.dim() != 1 or not t.numel():
        raise FlyguyError(f"offsets must be an int64 vector [recordings + 1] on {like.device}")
    return t.contiguous()


def _grad(name: str, g, like: torch.Tensor, shape=None) -> torch.Tensor:
    """An incoming gradient as the library takes it (None: zeros)."""
    if g is None:
        return torch.zeros(like.shape if shape is None else shape, dtype=like.dtype, device=like.device)
    g = _values(name, g if g.dtype is like.dtype else g.to(like.dtype), (like.dim(),))
    return g if 0 not in g.stride() else g.contiguous()   # (an expanded sum)


class _AgainFn(torch.autograd.Function):
    """The first `n` tensors as they are, and an error for whoever differentiates them."""
    @staticmethod
    def forward(ctx, n, *tensors):
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise FlyguyError("gradients of the memory operators cannot be differentiated again")


def _once(backward):
    """A backward whose gradients, where a graph of them is asked for (create_graph), are not taken for constants."""
    @wraps(backward)
    def once(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            outs = backward(ctx, *grads)
        of = (t for t in (*ctx.saved_tensors, *grads) if t is not None)
        given = [t for t in outs if isinstance(t, torch.Tensor)]
        kept = iter(_AgainFn.apply(len(given), *given, *of))
        return tuple(next(kept) if isinstance(t, torch.Tensor) else None for t in outs)
    return once


# ---- rotation ------------------------------------------------------------------------------------------------------

def rotary_turns(turned: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                 original: int = 1024, device=None) -> torch.Tensor:
    """[turned / 2] int64: pair i's angle a tick, base^(-2i / turned) radians, as a fraction of a turn times 2^64.

    For recordings longer than those learned from (`original` ticks), by `factor`:
      "linear"  every angle divided by factor
      "base"    the base raised so that the slowest pair's angle is divided by factor, the fastest's kept
      "parts"   kept where a pair turns over 32 times in `original` ticks, divided by factor where it turns less than
                once, in proportion between (to be used with rotate's amplitude 0.1 ln(factor) + 1)"""
    if turned < 0 or turned % 2:
        raise FlyguyError(f"turned must be even and not negative, not {turned}")
    if not (base > 1 and math.isfinite(base) and factor >= 1 and original >= 1):
        raise FlyguyError("base must be over 1, factor and original at least 1")
    if scaling not in (None, "linear", "base", "parts"):
        raise FlyguyError(f"scaling must be None, 'linear', 'base' or 'parts', not {scaling!r}")
    n = turned // 2
    with localcontext() as c:                              # (doubles would be off by some units at 2^64)
        c.prec = 40
        pace, by, two_pi = Decimal(base), Decimal(factor), 2 * _PI
        if scaling == "base" and n > 1:
            pace *= by ** (Decimal(n) / (n - 1))
        f = [pace ** (Decimal(-i) / n) for i in range(n)]
        if scaling == "linear":
            f = [x / by for x in f]
        elif scaling == "parts":
            keep = [min(Decimal(1), max(Decimal(0), (original * x / two_pi - 1) / 31)) for x in f]
            f = [x * a + x / by * (1 - a) for x, a in zip(f, keep)]
        return torch.tensor([int((x / two_pi * 2 ** 64).to_integral_value()) for x in f], dtype=torch.int64, device=device)


# fg_rotate_args: x, y, gy, gx (two fg_ticks each), w, w_head, gw, heads (two each), batch, ticks, dim, turned, turns,
# positions, pos_batch, pos_tick, pos_bytes, type, interleaved, norm, eps, amplitude, work, work_bytes
_ROTATE = struct.Struct("=32q8q12q2d2q")


class _Rotation:
    """What forward and backward of one call share: the sizes and settings as the argument structure has them."""

    def __init__(self, q, k, turns, positions, layout, amplitude, eps):
        shape = q.shape
        dim = shape[-1]
        if k is not None and (k.shape[:-2] != shape[:-2] or k.shape[-1] != dim):
            raise FlyguyError(f"k must be {(*shape[:-2], 'key heads', dim)}, not {tuple(k.shape)}")
        batch, ticks = (shape[0], shape[1]) if len(shape) == 4 else (1, shape[0])
        if layout not in LAYOUTS:
            raise FlyguyError(f"layout must be one of {list(LAYOUTS)}, not {layout!r}")
        turned = 0
        if turns is not None:
            if not isinstance(turns, torch.Tensor) or turns.dtype is not torch.int64 or turns.get_device() != q.get_device() or turns.dim() != 1:
                raise FlyguyError(f"turns must be an int64 vector on {q.device} (rotary_turns)")
            turned = 2 * turns.shape[0]
            if turned > dim:
                raise FlyguyError(f"turns are of {turned} values, a head has {dim}")
            if not turns.is_contiguous():
                turns = turns.contiguous()
        if positions is not None:
            if not isinstance(positions, torch.Tensor) or positions.get_device() != q.get_device() or positions.dtype not in (torch.int64, torch.int32):
                raise FlyguyError(f"positions must be int64 or int32 on {q.device}")
            if positions.shape != (batch, ticks):
                try:
                    positions = positions.expand(batch, ticks)
                except RuntimeError:
                    raise FlyguyError(f"positions {tuple(positions.shape)} do not fit {batch} x {ticks} ticks") from None
        self.turns, self.positions = turns, positions
        self.dim, self.device = dim, q.get_device()
        self.sizes = (shape[-2], 0 if k is None else k.shape[-2], batch, ticks, dim, turned)
        self.settings = (TYPES[q.dtype], LAYOUTS[layout], int(eps is not None), float(eps or 1.0), float(amplitude))

    def let_go(self) -> tuple:
        """The plan and the positions, for autograd to keep (and to guard against changes in place) until the backward."""
        kept = _kept(self.turns), _kept(self.positions)
        self.turns = self.positions = None
        return kept

    def take_up(self, turns, positions):
        """This call with the tensors that autograd has kept."""
        again = object.__new__(_Rotation)
        again.__dict__.update(self.__dict__, turns=turns, positions=positions)
        return again

    def pack(self, x, z=_NONE, y=_NONE, yk=_NONE, gy=_NONE, gz=_NONE, gx=_NONE, gk=_NONE, wq=None, wk=None, gwq=None, gwk=None,
             work=(0, 0)) -> bytes:
        p = self.positions
        pos = (0, 0, 0, 8) if p is None else (p.data_ptr(), *p.stride(), p.element_size())
        return _ROTATE.pack(*x, *z, *y, *yk, *gy, *gz, *gx, *gk, _ptr(wq), _ptr(wk),
                            self.dim if wq is not None and wq.dim() == 2 else 0, self.dim if wk is not None and wk.dim() == 2 else 0,
                            _ptr(gwq), _ptr(gwk), *self.sizes, _ptr(self.turns), *pos, *self.settings, *work)

    def forward(self, q, k=None, wq=None, wk=None):
        y = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if k is None:
            _call(lib().fg_norm_rotate, self.pack(_ticks(q), y=_ticks(y)), self.device)
            return y
        z = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        _call(lib().fg_norm_rotate, self.pack(_ticks(q), _ticks(k), _ticks(y), _ticks(z), wq=wq, wk=wk), self.device)
        return y, z

    def backward(self, gy, gz=None, q=None, k=None, wq=None, wk=None, want_w=(False, False)):
        gx = torch.empty(gy.shape, dtype=gy.dtype, device=gy.device)
        if q is None:                                         # the rotation alone
            _call(lib().fg_norm_rotate_bwd, self.pack(_NONE, gy=_ticks(gy), gx=_ticks(gx)), self.device)
            return gx
        gk = torch.empty(gz.shape, dtype=gz.dtype, device=gz.device)
        gwq = torch.empty_like(wq) if wq is not None and want_w[0] else None
        gwk = torch.empty_like(wk) if wk is not None and want_w[1] else None
        a = (_ticks(q), _ticks(k), _NONE, _NONE, _ticks(gy), _ticks(gz), _ticks(gx), _ticks(gk), wq, wk, gwq, gwk)
        room, work = None, (0, 0)
        if gwq is not None or gwk is not None:
            room, work = _room(lib().fg_norm_rotate_work(self.pack(*a)), q.device)
        _call(lib().fg_norm_rotate_bwd, self.pack(*a, work), self.device)
        return gx, gk, gwq, gwk


class _RotateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rotation):
        y = rotation.forward(x)
        ctx.rotation = rotation
        ctx.save_for_backward(*rotation.let_go())
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        return ctx.rotation.take_up(*ctx.saved_tensors).backward(_grad("the gradient", gy, gy)), None


class _NormRotateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, rotation):
        ctx.set_materialize_grads(False)
        q, k = _values("q", q, (3, 4)), _values("k", k, (3, 4))
        out = rotation.forward(q, k, wq, wk)
        ctx.rotation = rotation
        ctx.save_for_backward(q, k, wq, wk, *rotation.let_go())
        return out

    @staticmethod
    @_once
    def backward(ctx, gy, gz):
        q, k, wq, wk, *plan = ctx.saved_tensors
        gy, gz = _grad("the gradient of the queries", gy, q), _grad("the gradient of the keys", gz, k)
        return *ctx.rotation.take_up(*plan).backward(gy, gz, q, k, wq, wk, ctx.needs_input_grad[2:4]), None


def rotate(x, turns, positions=None, layout: str = "half", amplitude: float = 1.0) -> torch.Tensor:
    """x [batch, ticks, heads, dim] or [ticks, heads, dim] with the first 2 * len(turns) values of each head turned pair by
    pair: (a, b) -> amplitude (a cos - b sin, b cos + a sin) at the angle position * turns (rotary_turns).

    positions: int64 / int32 that expand to [batch, ticks] (None: 0, 1, ..). layout "half": pairs (i, i + turned / 2);
    "interleaved": (2i, 2i + 1). The gradient is the rotation back."""
    x = _values("x", x, (3, 4))
    _no_tangents(x)
    r = _Rotation(x, None, turns, positions, layout, amplitude, None)
    if x.requires_grad and torch.is_grad_enabled():
        return _RotateFn.apply(x, r)
    return r.forward(x)


def norm_rotate(q, k, turns=None, q_weight=None, k_weight=None, positions=None, layout: str = "half",
                amplitude: float = 1.0, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """rotate(x / sqrt(mean(x^2) + eps) * weight) over each head of queries [.., heads, dim] and keys [.., key heads, dim],
    in one pass over both. Weights: float32 [dim] (one for all heads) or [heads, dim], or None; turns None: the
    norms alone. Gradients of q, k and the weights; the weights' are the same bits on every run."""
    q = _values("q", q, (3, 4))
    k = _values("k", k, (3, 4), q)
    if not eps > 0:
        raise FlyguyError(f"eps must be positive, not {eps}")
    if q_weight is not None:
        q_weight = _float32("q_weight", q_weight, q, q.shape[-1:], q.shape[-2:])
    if k_weight is not None:
        k_weight = _float32("k_weight", k_weight, k, k.shape[-1:], k.shape[-2:])
    _no_tangents(q, k, q_weight, k_weight)
    r = _Rotation(q, k, turns, positions, layout, amplitude, eps)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return _NormRotateFn.apply(q, k, q_weight, k_weight, r)
    return r.forward(q, k, q_weight, k_weight)


# ---- attention whose state decays -----------------------------------------------------------------------------------

# fg_decay_args: q, k, v, o, go, gq, gk, gv (fg_ticks), log_decay, state, state_out, gstate_out, gstate, offsets, batch, ticks,
# heads, key_heads, dim, value_dim, type, scale, work, work_bytes
_DECAY = struct.Struct("=32q6q7qd2q")
# fg_step_args: q, k, v, o (fg_ticks), log_decay, state, slots, n_slots, batch, heads, key_heads, dim, value_dim, type, scale
_STEP = struct.Struct("=16q10qd")


@lru_cache(maxsize=256)
def _decay_room(sizes: tuple, packed: bool, backward: bool) -> int:
    """Bytes of workspace that a call of these sizes needs (fg_decay_work)."""
    size = lib().fg_decay_work(_DECAY.pack(*(0,) * 37, int(packed), *sizes, 1.0, 0, 0), int(backward))
    if size < 0:                                          # (raised here: an error is not kept)
        raise FlyguyError(lib().fg_mem_last_error().decode())
    return size


class _Decay:
    """What forward and backward of one call share."""

    def __init__(self, q, k, v, log_decay, state, scale, offsets):
        lead, heads, dim = q.shape[:-2], q.shape[-2], q.shape[-1]
        key_heads, value_dim = v.shape[-2], v.shape[-1]
        if k.shape != (*lead, key_heads, dim) or v.shape[:-2] != lead:
            raise FlyguyError(f"k and v must be {(*lead, 'key heads', dim)} and {(*lead, 'key heads', 'value dim')}, not "
                              f"{tuple(k.shape)} and {tuple(v.shape)}")
        if not key_heads or heads % key_heads:
            raise FlyguyError(f"{heads} query heads cannot share {key_heads} key heads")
        if offsets is None:
            batch, ticks = lead if len(lead) == 2 else (1, lead[0])
        else:
            if len(lead) != 1:
                raise FlyguyError("offsets go with recordings packed end to end: q is [ticks, heads, dim]")
            offsets = _offsets(offsets, q)
            batch, ticks = offsets.shape[0] - 1, lead[0]
        self.log_decay = _float32("log_decay", log_decay, q, (heads,))
        if log_decay.requires_grad:
            raise FlyguyError("log_decay is a constant of each head: it has no gradient")
        self.states, self.device, self.offsets = (batch, heads, dim, value_dim), q.get_device(), offsets
        if state is not None:
            _float32("state", state, q, self.states)
        self.sizes = (batch, ticks, heads, key_heads, dim, value_dim, TYPES[q.dtype])
        self.scale = float(dim ** -0.5 if scale is None else scale)

    def let_go(self) -> tuple:
        """The decays and the offsets, for autograd to keep until the backward."""
        kept = _kept(self.log_decay), _kept(self.offsets)
        self.log_decay = self.offsets = None
        return kept

    def take_up(self, log_decay, offsets):
        again = object.__new__(_Decay)
        again.__dict__.update(self.__dict__, log_decay=log_decay, offsets=offsets)
        return again

    def run(self, fn, backward: bool, tensors, state=None, state_out=None, gstate_out=None, gstate=None) -> None:
        room, work = _room(_decay_room(self.sizes, self.offsets is not None, backward), tensors[0].device)
        packed = _DECAY.pack(*(f for t in tensors for f in (_NONE if t is None else _ticks(t))), self.log_decay.data_ptr(),
                             _ptr(state), _ptr(state_out), _ptr(gstate_out), _ptr(gstate), _ptr(self.offsets), *self.sizes,
                             self.scale, *work)
        _call(fn, packed, self.device)

    def forward(self, q, k, v, state):
        o = torch.empty((*q.shape[:-1], v.shape[-1]), dtype=q.dtype, device=q.device)
        end = torch.empty(self.states, dtype=torch.float32, device=q.device)
        self.run(lib().fg_decay_attn, False, (q, k, v, o, None, None, None, None), state, end)
        return o, end

    def backward(self, q, k, v, state, go, gend, want_state: bool):
        go = _grad("the gradient of o", go, q, (*q.shape[:-1], v.shape[-1]))
        if gend is not None:
            gend = _state(gend.float())
        gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        gstate = torch.empty(self.states, dtype=torch.float32, device=q.device) if want_state else None
        self.run(lib().fg_decay_attn_bwd, True, (q, k, v, None, go, gq, gk, gv), state, None, gend, gstate)
        return gq, gk, gv, gstate


class _DecayFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, job):
        ctx.set_materialize_grads(False)
        q, k, v = (_values("q", t, (3, 4)) for t in (q, k, v))
        state = _state(state)
        out = job.forward(q, k, v, state)
        ctx.job = job
        ctx.save_for_backward(q, k, v, state, *job.let_go())
        return out

    @staticmethod
    @_once
    def backward(ctx, go, gend):
        q, k, v, state, *kept = ctx.saved_tensors
        return *ctx.job.take_up(*kept).backward(q, k, v, state, go, gend, ctx.needs_input_grad[3]), None


def decay_attention(q, k, v, log_decay, state=None, scale: float | None = None,
                    offsets=None) -> tuple[torch.Tensor, torch.Tensor]:
    """S_t = exp(log_decay) S_{t-1} + k_t v_t^T, o_t = scale q_t S_t for every recording and head.

    q [batch, ticks, heads, dim], k [.., key heads, dim], v [.., key heads, value dim], each key head serving heads / key
    heads query heads; or [ticks, ..] with recordings packed end to end and offsets int64 [recordings + 1], not falling
    (recordings may be empty; ticks before the first and after the last get zeros, in o and in the gradients). log_decay
    float32 [heads], at most 0, a constant. state float32 [recordings, heads, dim, value dim] before the first ticks (None:
    zeros). scale: dim^-0.5 when None. dim and value dim at most 256.
    Returns o [.., heads, value dim] and the states after the last ticks; gradients of q, k, v and state.

    A recording's ticks are worked on in tiles of 64 or 128: a NaN or an infinity stays in its recording and head and out of
    the tiles before it, but reaches all ticks of its own, and infinities become NaN (decay_step goes tick by tick)."""
    q = _values("q", q, (3, 4))
    k, v = _values("k", k, (3, 4), q), _values("v", v, (3, 4), q)
    job = _Decay(q, k, v, log_decay, state, scale, offsets)
    _no_tangents(q, k, v, state, job.log_decay)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _DecayFn.apply(q, k, v, state, job)
    return job.forward(q, k, v, _state(state))


def decay_step(q, k, v, log_decay, state, scale: float | None = None, slots=None) -> torch.Tensor:
    """One tick of decay_attention for a batch: q [batch, heads, dim], k [batch, key heads, dim], v [batch, key heads, value
    dim]. state float32 [slots, heads, dim, value dim], contiguous, is updated in place at each row's slot (slots int64
    [batch], no two alike; None: row b's is b); a row whose slot is outside answers 0 and changes nothing. Returns o
    [batch, heads, value dim]. No gradient: for learning, decay_attention."""
    q, k, v = _values("q", q, (3,)), _values("k", k, (3,), q), _values("v", v, (3,), q)
    batch, heads, dim = q.shape
    key_heads, value_dim = v.shape[1:]
    if k.shape != (batch, key_heads, dim) or v.shape[0] != batch:
        raise FlyguyError(f"k and v must be {(batch, 'key heads', dim)} and {(batch, 'key heads', 'value dim')}, not "
                          f"{tuple(k.shape)} and {tuple(v.shape)}")
    if not key_heads or heads % key_heads:
        raise FlyguyError(f"{heads} query heads cannot share {key_heads} key heads")
    log_decay = _float32("log_decay", log_decay, q, (heads,))
    if (not isinstance(state, torch.Tensor) or state.dtype is not torch.float32 or state.get_device() != q.get_device()
            or state.dim() != 4 or state.shape[1:] != (heads, dim, value_dim) or not state.is_contiguous()):
        raise FlyguyError(f"state must be contiguous float32 {('slots', heads, dim, value_dim)} on {q.device}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise FlyguyError("decay_step has no gradient (decay_attention has): call it under torch.no_grad()")
    _no_tangents(q, k, v, state, log_decay)
    if slots is not None:
        if (not isinstance(slots, torch.Tensor) or slots.dtype is not torch.int64 or slots.get_device() != q.get_device()
                or slots.shape != (batch,)):
            raise FlyguyError(f"slots must be int64 [{batch}] on {q.device}")
        if not slots.is_contiguous():
            slots = slots.contiguous()
    elif state.shape[0] < batch:
        raise FlyguyError(f"{batch} rows need as many states, not {state.shape[0]}")
    o = torch.empty((batch, heads, value_dim), dtype=q.dtype, device=q.device)
    f = []
    for t in (q, k, v, o):
        st = t.stride()
        f += (t.data_ptr(), st[0], 0, st[1])
    packed = _STEP.pack(*f, log_decay.data_ptr(), state.data_ptr(), _ptr(slots), state.shape[0], batch, heads, key_heads, dim,
                        value_dim, TYPES[q.dtype], float(dim ** -0.5 if scale is None else scale))
    _call(lib().fg_decay_step, packed, q.get_device())
    increment_version(state)                              # (autograd sees that it has changed, should it have kept it)
    return o


def sync(device=None) -> None:
    """Waits for the current stream of `device` (None: the current one). An error if a wait inside a kernel of these operators has
    run out on it, now or earlier in this process; what that call left holds NaN (of delta.delta_step: outputs alone, the states of those
    rows are as they were)."""
    with torch.cuda.device(device):
        if lib().fg_mem_sync(_raw_stream(_device())):
            raise FlyguyError(lib().fg_mem_last_error().decode())


# ---- the operators together ---------------------------------------------------------------------------------------

class TickMemory(nn.Module):
    """What earlier ticks add to an actor's logits: logits = actor(obs) + memory(obs).

    Queries, keys and values are projections of the observations in `dtype`; norm_rotate turns queries and keys,
    decay_attention carries the states (the heads' memories spread from ticks[0] to ticks[1] ticks), a last projection
    gives the logits. That one starts at zero, so that a fresh memory changes nothing. Learning sees whole recordings
    (forward), playing one tick of every car at a time (step); both give the same answers, to the rounding of `dtype`."""

    def __init__(self, obs_dim: int, n_actions: int, heads: int = 8, key_heads: int = 2, dim: int = 64,
                 ticks: tuple[float, float] = (16.0, 4096.0), base: float = 10000.0, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if key_heads < 1 or heads % key_heads:
            raise FlyguyError(f"{heads} query heads cannot share {key_heads} key heads")
        if not 1 < ticks[0] <= ticks[1]:
            raise FlyguyError(f"memories of {ticks} ticks: over 1, the shorter first")
        self.heads, self.key_heads, self.dim, self.dtype = heads, key_heads, dim, dtype
        self.qkv = nn.Linear(obs_dim, (heads + 2 * key_heads) * dim, bias=False)
        self.out = nn.Linear(heads * dim, n_actions, bias=False)
        nn.init.zeros_(self.out.weight)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.ones(dim))
        span = torch.logspace(math.log10(ticks[0]), math.log10(ticks[1]), heads, dtype=torch.float64)
        self.register_buffer("log_decay", torch.log1p(-1 / span).float(), persistent=False)
        self.register_buffer("turns", rotary_turns(dim // 2 * 2, base), persistent=False)

    def states(self, cars: int) -> torch.Tensor:
        """The states of so many cars that remember nothing: float32 [cars, heads, dim, dim]."""
        return torch.zeros(cars, self.heads, self.dim, self.dim, device=self.log_decay.device)

    def _places(self, obs: torch.Tensor, state, positions, offsets):
        """Offsets and positions as forward's operators take them."""
        if state is not None and positions is None:
            raise FlyguyError("a recording carried on from a state needs its ticks' positions")
        if offsets is not None and positions is None and obs.dim() == 2:   # (the states that come out are step's to go on from)
            offsets, tick = _offsets(offsets, obs), torch.arange(len(obs), device=obs.device)
            positions = tick - offsets[(torch.searchsorted(offsets, tick, right=True) - 1).clamp(min=0)]
        return offsets, positions

    def _qkv(self, obs: torch.Tensor, positions):
        x = nn.functional.linear(obs.to(self.dtype), self.qkv.weight.to(self.dtype))
        x = x.unflatten(-1, (self.heads + 2 * self.key_heads, self.dim))
        q, k, v = x.split((self.heads, self.key_heads, self.key_heads), -2)
        return *norm_rotate(q, k, self.turns, self.q_weight, self.k_weight, positions), v

    def _logits(self, o: torch.Tensor) -> torch.Tensor:
        return nn.functional.linear(o.flatten(-2), self.out.weight.to(self.dtype)).float()

    def forward(self, obs: torch.Tensor, state=None, positions=None, offsets=None) -> tuple[torch.Tensor, torch.Tensor]:
        """obs [recordings, ticks, obs_dim], or [ticks, obs_dim] packed end to end with offsets: logits of every tick and
        the states after the last. Positions are the ticks of each recording unless given. A recording carried on needs its
        states and positions (a rotation depends on them)."""
        offsets, positions = self._places(obs, state, positions, offsets)
        q, k, v = self._qkv(obs, positions)
        o, end = decay_attention(q, k, v, self.log_decay, state, offsets=offsets)
        return self._logits(o), end

    @torch.no_grad()
    def step(self, obs: torch.Tensor, state: torch.Tensor, positions: torch.Tensor, slots=None) -> torch.Tensor:
        """One tick of every car: obs [cars, obs_dim], positions [cars] the tick of each car's recording; the states are updated
        in place (at `slots`, see decay_step)."""
        q, k, v = self._qkv(obs.unsqueeze(1), positions.unsqueeze(1))
        o = decay_step(q.squeeze(1), k.squeeze(1), v.squeeze(1), self.log_decay, state, slots=slots)
        return self._logits(o)
