"""A memory over ticks that overwrites (beside flyguy_b200.memory, whose states only fade): the gated delta rule.

  delta_attention   the rule over whole recordings (also packed end to end), with gradients of all its inputs
  delta_step        the same for one tick, the states updated in place

S_t = g_t S_{t-1} + k_t u_t^T with u_t = beta_t (v_t - g_t k_t S_{t-1}): what the state holds at a tick's key is moved towards the tick's
value by beta, everything else fades by g = exp(log_decay). Both gates are each tick's own. o_t = scale q_t S_t. Bounded where
beta |k|^2 is at most 2: keys of about unit length (memory.norm_rotate with k_weight dim^-0.5).

They run in the library (fg_delta_attn, fg_delta_step of include/flyguy_b200.h) on CUDA tensors, on torch's current stream.
Queries, keys and values are float32, bfloat16 or float16 of one type, any strides with a head's values adjacent (others are copied
first); gates and states are float32. Gradients are of the first order. DeltaMemory puts the operators together.

Products run on the tensor cores in bfloat16 terms: what is carried from chunk to chunk (states, corrections and their gradients)
and the gates' gradients have three, 2^-24 of each value; outputs and the gradients of q and k of 16-bit types two, where one would
be of the size of the result's own rounding. Sums are float32."""
from __future__ import annotations

import math
import struct
from functools import lru_cache

import torch
from torch import nn
from torch.autograd.graph import increment_version

from . import layers, memory
from .memory import TYPES, _call, _float32, _grad, _kept, _no_tangents, _offsets, _once, _ptr, _room, _state, _ticks, _values
from .native import FlyguyError, lib

# fg_delta_args: q, k, v, o, go, gq, gk, gv, log_decay, beta, glog_decay, gbeta (fg_ticks), state, state_out, gstate_out, gstate, offsets,
# batch, ticks, heads, query_heads, key_heads, value_heads, dim, value_dim, type, scale, work, work_bytes
_DELTA = struct.Struct("=48q5q9qd2q")
# fg_delta_step_args: q, k, v, o, log_decay, beta (fg_ticks), state, slots, n_slots, batch, heads, query_heads, key_heads, value_heads, dim,
# value_dim, type, scale
_STEP = struct.Struct("=24q11qd")
_STEP_HEAD, _DOUBLE, _FLOAT = struct.Struct("=26q"), struct.Struct("=d"), struct.Struct("=f")


def _gate(name: str, t, lead: tuple, like: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != like.get_device():
        raise FlyguyError(f"{name} must be a float32 tensor on {like.device}")
    if t.dim() != len(lead) + 1 or t.shape[:-1] != lead:
        raise FlyguyError(f"{name} must be {(*lead, 'heads')}, not {tuple(t.shape)}")
    return t


def _head_counts(q, k, v, log_decay, beta) -> tuple[int, int, int, int]:
    """heads, query heads, key heads, value heads."""
    heads = log_decay.shape[-1]
    if beta.shape != log_decay.shape:
        raise FlyguyError(f"beta must be {tuple(log_decay.shape)} as log_decay is, not {tuple(beta.shape)}")
    counts = q.shape[-2], k.shape[-2], v.shape[-2]
    for name, n in zip("qkv", counts):
        if not n or not heads or heads % n:
            raise FlyguyError(f"{heads} heads (of the gates) cannot share {n} heads of {name}")
    return heads, *counts


def _gate_ticks(t: torch.Tensor) -> tuple[int, int, int, int]:
    """fg_ticks of [batch, ticks, heads] or [ticks, heads]."""
    st = t.stride()
    return (t.data_ptr(), *st) if len(st) == 3 else (t.data_ptr(), 0, *st)


@lru_cache(maxsize=256)
def _delta_sizes(q, k, v, log_decay, beta, typ, recordings) -> tuple[tuple, tuple, bytes, tuple, int]:
    """Of a call of these shapes and this type: the states' and o's shape, its fields from batch to type, the bytes of workspace
    that it and its gradients need, by themselves and with what is held between them (fg_delta_work), and the bytes held
    (fg_delta_held). recordings: None, or how many the offsets name."""
    lead, dim, value_dim = q[:-2], q[-1], v[-1]
    if recordings is None:
        batch, ticks = lead if len(lead) == 2 else (1, lead[0])
    else:
        batch, ticks = recordings, lead[0]
    heads = log_decay[-1]
    sizes = (batch, ticks, heads, q[-2], k[-2], v[-2], dim, value_dim, TYPES[typ])
    packed = _DELTA.pack(*(0,) * 52, int(recordings is not None), *sizes, 1.0, 0, 0)
    rooms = *(lib().fg_delta_work(packed, which) for which in range(4)), lib().fg_delta_held(packed)
    if min(rooms) < 0:                                    # (raised here: an error is not kept)
        raise FlyguyError(lib().fg_mem_last_error().decode())
    return (batch, heads, dim, value_dim), (*lead, heads, value_dim), struct.pack("=9q", *sizes), rooms[:4], rooms[4]


# A forward with gradients holds what its backward needs (states of every 64 ticks, corrections and outputs in float32, X and P: at dim 128 of
# bfloat16 2.4 KB a tick and head, where q, k, v and o are 1 KB) if that is at most so many bytes; else the backward makes it again. 64
# recordings of 1,024 ticks, 8 heads of 128: 1.32 GB, 2,953 us for both ways; made again 3,518.
HELD_AT_MOST = 4 << 30
_NOTHING = bytes(32)                                      # an fg_ticks of NULL
_FORWARD, _NO_GRADIENTS = struct.Struct("=48q"), (0,) * 16
_TICKS, _POINTERS, _END = struct.Struct("=4q"), struct.Struct("=5q"), struct.Struct("=d2q")


class _Delta:
    """What forward and backward of one call share."""

    def __init__(self, device: int, sizes: tuple, scale: float, offsets=None):
        self.device, self.offsets, self.scale = device, offsets, scale
        self.states, self.o_shape, self.sizes, self.rooms, self.held = sizes

    def let_go(self) -> torch.Tensor | None:
        """The offsets, for autograd to keep until the backward."""
        kept, self.offsets = _kept(self.offsets), None
        return kept

    def take_up(self, offsets):
        return _Delta(self.device, (self.states, self.o_shape, self.sizes, self.rooms, self.held), self.scale, offsets)

    def run(self, backward: int, held, ticks: bytes, device, state=0, state_out=0, gstate_out=0, gstate=0) -> None:
        room, work = _room(self.rooms[backward if held is None else 2 + backward], device)
        if held is None:
            fn = lib().fg_delta_attn_bwd if backward else lib().fg_delta_attn
        else:
            holding, at = lib().fg_delta_attn_bwd_held if backward else lib().fg_delta_attn_hold, held.data_ptr()
            fn = lambda packed, stream: holding(packed, at, self.held, stream)   # noqa: E731
        _call(fn, ticks + _POINTERS.pack(state, state_out, gstate_out, gstate, _ptr(self.offsets)) + self.sizes + _END.pack(self.scale, *work),
              self.device)

    def forward(self, q, k, v, log_decay, beta, state, held=None):
        o = q.new_empty(self.o_shape)
        end = log_decay.new_empty(self.states)
        ticks = _FORWARD.pack(*_ticks(q), *_ticks(k), *_ticks(v), *_ticks(o), *_NO_GRADIENTS, *_gate_ticks(log_decay), *_gate_ticks(beta),
                              0, 0, 0, 0, 0, 0, 0, 0)
        self.run(0, held, ticks, q.device, _ptr(state), end.data_ptr())
        return o, end

    def backward(self, q, k, v, log_decay, beta, state, held, go, gend, want_state: bool):
        go = _grad("the gradient of o", go, q, self.o_shape)
        if gend is not None:
            gend = _state(gend.float())
        gq, gk, gv, gl, gb = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v, log_decay, beta))
        gstate = torch.empty(self.states, dtype=torch.float32, device=q.device) if want_state else None
        ticks = b"".join([_TICKS.pack(*_ticks(t)) for t in (q, k, v)] + [_NOTHING] + [_TICKS.pack(*_ticks(t)) for t in (go, gq, gk, gv)]
                         + [_TICKS.pack(*_gate_ticks(t)) for t in (log_decay, beta, gl, gb)])
        self.run(1, held, ticks, q.device, _ptr(state), 0, _ptr(gend), _ptr(gstate))
        return gq, gk, gv, gl, gb, gstate


class _DeltaFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, state, job):
        ctx.set_materialize_grads(False)
        q, k, v = (_values("q", t, (3, 4)) for t in (q, k, v))
        state = _state(state)
        held = _room(job.held, q.device)[0] if job.held <= HELD_AT_MOST else None
        out = job.forward(q, k, v, log_decay, beta, state, held)
        ctx.job = job
        ctx.save_for_backward(*map(_kept, (q, k, v, log_decay, beta, state)), held, job.let_go())
        return out

    @staticmethod
    @_once
    def backward(ctx, go, gend):
        *ins, offsets = ctx.saved_tensors
        return *ctx.job.take_up(offsets).backward(*ins, go, gend, ctx.needs_input_grad[5]), None


@lru_cache(maxsize=256)
def _delta_shapes(q, k, v, log_decay, beta, state, *types) -> tuple:
    """_delta_sizes of a call of these shapes and types without offsets; an error without words."""
    if not (len(q) == len(k) == len(v) in (3, 4) and q[:-2] == k[:-2] == v[:-2] == log_decay[:-1] and q[-1] == k[-1] and log_decay == beta
            and types[0] in TYPES and types[0] is types[1] is types[2] and types[3:5] == (torch.float32,) * 2):
        raise FlyguyError
    heads = log_decay[-1]
    if not heads or any(not t[-2] or heads % t[-2] for t in (q, k, v)):
        raise FlyguyError
    sizes = _delta_sizes(q, k, v, log_decay, beta, types[0], None)
    if state is not None and (state != sizes[0] or types[5] is not torch.float32):
        raise FlyguyError
    return sizes


def _delta_inputs(q, k, v, log_decay, beta, state, offsets) -> tuple:
    """The inputs as the library takes them and the call's sizes, or what is wrong with them."""
    q = _values("q", q, (3, 4))
    k, v = _values("k", k, (3, 4), q), _values("v", v, (3, 4), q)
    log_decay, beta = _gate("log_decay", log_decay, q.shape[:-2], q), _gate("beta", beta, q.shape[:-2], q)
    lead, dim = q.shape[:-2], q.shape[-1]
    if k.shape[:-2] != lead or k.shape[-1] != dim or v.shape[:-2] != lead:
        raise FlyguyError(f"k and v must be {(*lead, 'key heads', dim)} and {(*lead, 'value heads', 'value dim')}, not "
                          f"{tuple(k.shape)} and {tuple(v.shape)}")
    if offsets is not None:
        if len(lead) != 1:
            raise FlyguyError("offsets go with recordings packed end to end: q is [ticks, heads, dim]")
        offsets = _offsets(offsets, q)
    _head_counts(q, k, v, log_decay, beta)
    sizes = _delta_sizes(q.shape, k.shape, v.shape, log_decay.shape, beta.shape, q.dtype, None if offsets is None else offsets.shape[0] - 1)
    if state is not None:
        _float32("state", state, q, sizes[0])
    return q, k, v, log_decay, beta, offsets, sizes


def delta_attention(q, k, v, log_decay, beta, state=None, scale: float | None = None,
                    offsets=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule for every recording and head: S_t = exp(log_decay_t) S_{t-1} + k_t u_t^T, u_t = beta_t (v_t -
    exp(log_decay_t) k_t S_{t-1}), o_t = scale q_t S_t.

    log_decay and beta float32 [batch, ticks, heads]; q [batch, ticks, query heads, dim], k [.., key heads, dim] and v [.., value
    heads, value dim], each number of heads a divisor of `heads` (head h has query head h / (heads / query heads), and so on). Or
    [ticks, ..] with recordings packed end to end and offsets int64 [recordings + 1], not falling (recordings may be empty; ticks
    before the first and after the last get zeros, in o and in the gradients). state float32 [recordings, heads, dim, value
    dim] before the first ticks (None: zeros). scale: dim^-0.5 when None. dim at most 128, value dim at most 256.
    log_decay is at most 0, minus infinity forgets the state (anything below -256 does, in float32).
    Returns o [.., heads, value dim] and the states after the last ticks; gradients of q, k, v, log_decay, beta and state. A
    forward with gradients holds what its backward needs, up to HELD_AT_MOST bytes; o of one that does is made of more terms than o alone or
    above that (the states are the same bits).

    A recording's ticks are worked on in tiles of 64: a NaN or an infinity stays in its recording and head and out of the tiles
    before it, but reaches all ticks of its own and those after it, and infinities become NaN (delta_step goes tick by tick)."""
    try:                                                  # (what most calls are, by the sizes alone)
        if offsets is not None:
            raise FlyguyError
        sizes = _delta_shapes(q.shape, k.shape, v.shape, log_decay.shape, beta.shape, None if state is None else state.shape,
                              q.dtype, k.dtype, v.dtype, log_decay.dtype, beta.dtype, None if state is None else state.dtype)
        device = q.get_device()
        if not (q.stride(-1) == k.stride(-1) == v.stride(-1) == 1 and device >= 0 and (state is None or state.get_device() == device)
                and k.get_device() == v.get_device() == log_decay.get_device() == beta.get_device() == device):
            raise FlyguyError
    except (AttributeError, FlyguyError):
        q, k, v, log_decay, beta, offsets, sizes = _delta_inputs(q, k, v, log_decay, beta, state, offsets)
        device = q.get_device()
    job = _Delta(device, sizes, q.shape[-1] ** -0.5 if scale is None else float(scale), offsets)
    _no_tangents(q, k, v, log_decay, beta, state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or beta.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _DeltaFn.apply(q, k, v, log_decay, beta, state, job)
    return job.forward(q, k, v, log_decay, beta, _state(state))


@lru_cache(maxsize=256)
def _step_sizes(q, k, v, log_decay, beta, state, *types) -> tuple[tuple, bytes]:
    """(batch, heads, value dim) of a step of these shapes and types, and its fields from n_slots to type; an error without words."""
    *types, own_slots = types
    if not (len(q) == len(k) == len(v) == 3 and len(log_decay) == 2 and log_decay == beta and len(state) == 4 and types[0] in TYPES
            and types[0] is types[1] is types[2] and types[3:] == [torch.float32] * 3):
        raise FlyguyError
    (batch, heads), (slots, *of_state), dim, value_dim = log_decay, state, q[2], v[2]
    if not (q[0] == k[0] == v[0] == batch and k[2] == dim and of_state == [heads, dim, value_dim] and heads and q[1] and k[1] and v[1]
            and dim and value_dim and not heads % q[1] and not heads % k[1] and not heads % v[1] and (slots >= batch or not own_slots)):
        raise FlyguyError
    return (batch, heads, value_dim), struct.pack("=9q", slots, batch, heads, q[1], k[1], v[1], dim, value_dim, TYPES[types[0]])


def _step_inputs(q, k, v, log_decay, beta, state, slots) -> tuple:
    """The inputs as the library takes them, or what is wrong with them."""
    q, k, v = _values("q", q, (3,)), _values("k", k, (3,), q), _values("v", v, (3,), q)
    batch, _, dim = q.shape
    value_dim = v.shape[-1]
    if not dim or not value_dim:
        raise FlyguyError("dim and value dim must be at least 1")
    if k.shape[0] != batch or k.shape[-1] != dim or v.shape[0] != batch:
        raise FlyguyError(f"k and v must be {(batch, 'key heads', dim)} and {(batch, 'value heads', 'value dim')}, not "
                          f"{tuple(k.shape)} and {tuple(v.shape)}")
    log_decay, beta = _gate("log_decay", log_decay, (batch,), q), _gate("beta", beta, (batch,), q)
    heads = _head_counts(q, k, v, log_decay, beta)
    if (not isinstance(state, torch.Tensor) or state.dtype is not torch.float32 or state.get_device() != q.get_device()
            or state.dim() != 4 or state.shape[1:] != (heads[0], dim, value_dim) or not state.is_contiguous()):
        raise FlyguyError(f"state must be contiguous float32 {('slots', heads[0], dim, value_dim)} on {q.device}")
    if slots is None and state.shape[0] < batch:
        raise FlyguyError(f"{batch} rows need as many states, not {state.shape[0]}")
    return q, k, v, log_decay, beta


def delta_step(q, k, v, log_decay, beta, state, scale: float | None = None, slots=None) -> torch.Tensor:
    """One tick of delta_attention for a batch: q [batch, query heads, dim], k [batch, key heads, dim], v [batch, value heads, value
    dim], log_decay and beta float32 [batch, heads]. state float32 [slots, heads, dim, value dim], contiguous, is updated in place
    at each row's slot (slots int64 [batch], no two alike; None: row b's is b); a row whose slot is outside answers 0 and changes
    nothing. dim and value dim at most 256. Returns o [batch, heads, value dim]. No gradient: for learning, delta_attention."""
    try:                                                  # (what most calls are, by the sizes alone)
        sizes, tail = _step_sizes(q.shape, k.shape, v.shape, log_decay.shape, beta.shape, state.shape, q.dtype, k.dtype, v.dtype,
                                  log_decay.dtype, beta.dtype, state.dtype, slots is None)
        at, device = [x.stride() for x in (q, k, v)], q.get_device()
        if not (at[0][2] == at[1][2] == at[2][2] == 1 and state.is_contiguous() and device >= 0
                and k.get_device() == v.get_device() == log_decay.get_device() == beta.get_device() == state.get_device() == device):
            raise FlyguyError
    except (AttributeError, FlyguyError):
        q, k, v, log_decay, beta = _step_inputs(q, k, v, log_decay, beta, state, slots)
        sizes, tail = _step_sizes(q.shape, k.shape, v.shape, log_decay.shape, beta.shape, state.shape, q.dtype, k.dtype, v.dtype,
                                  log_decay.dtype, beta.dtype, state.dtype, slots is None)
        at, device = [x.stride() for x in (q, k, v)], q.get_device()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or beta.requires_grad
                                    or state.requires_grad):
        raise FlyguyError("delta_step has no gradient (delta_attention has): call it under torch.no_grad()")
    _no_tangents(q, k, v, log_decay, beta, state)
    if slots is not None:
        if not isinstance(slots, torch.Tensor) or slots.dtype is not torch.int64 or slots.get_device() != device or slots.shape != sizes[:1]:
            raise FlyguyError(f"slots must be int64 [{sizes[0]}] on {q.device}")
        if not slots.is_contiguous():
            slots = slots.contiguous()
    o = q.new_empty(sizes)
    (qb, qh, _), (kb, kh, _), (vb, vh, _), (lb, lh), (bb, bh) = *at, log_decay.stride(), beta.stride()
    packed = _STEP_HEAD.pack(q.data_ptr(), qb, 0, qh, k.data_ptr(), kb, 0, kh, v.data_ptr(), vb, 0, vh, o.data_ptr(), sizes[1] * sizes[2], 0,
                             sizes[2], log_decay.data_ptr(), lb, 0, lh, beta.data_ptr(), bb, 0, bh, state.data_ptr(),
                             0 if slots is None else slots.data_ptr())
    _call(lib().fg_delta_step, packed + tail + _DOUBLE.pack(q.shape[2] ** -0.5 if scale is None else scale), device)
    increment_version(state)                              # (autograd sees that it has changed, should it have kept it)
    return o


# ---- the operators together ---------------------------------------------------------------------------------------

class DeltaMemory(memory.TickMemory):
    """TickMemory with the gated delta rule: a memory that can replace what it holds, with gates that the observations set.

    The observations are normed (layer_norm) and projected in `dtype` to key_heads queries and keys (norm_rotate), heads values, and each
    head's gates: beta = sigmoid(b) and log_decay = -softplus(a) / span, the heads' spans spread from ticks[0] to ticks[1]. Keys are of
    unit length at first and no longer whatever k_weight learns (its largest value is brought down to dim^-0.5), so that no state grows
    by what it forgets. delta_attention carries the states, each head's output is normed, some of it dropped while learning (in training
    mode: dropout with `seed`, one call of the generator a forward; in a captured forward `seed` has to be an int64 tensor on the device,
    changed between replays), and a last projection, zero at first, gives the logits. state_dict has the count of calls, `seed` is the
    caller's to give again; memories, and ranks, of one seed drop alike."""

    def __init__(self, obs_dim: int, n_actions: int, heads: int = 8, key_heads: int = 2, dim: int = 64,
                 ticks: tuple[float, float] = (16.0, 4096.0), base: float = 10000.0, dropout: float = 0.0, seed: int = 0,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__(obs_dim, n_actions, heads, key_heads, dim, ticks, base, dtype)
        self.dropout, self.seed, self.calls = dropout, seed, 0
        self.qkv = nn.Linear(obs_dim, (2 * key_heads + heads) * dim, bias=False)
        self.gates = nn.Linear(obs_dim, 2 * heads)
        nn.init.zeros_(self.gates.weight)
        nn.init.zeros_(self.gates.bias)
        with torch.no_grad():
            self.k_weight.fill_(dim ** -0.5)               # keys of unit length
        self.obs_weight, self.obs_bias = nn.Parameter(torch.ones(obs_dim)), nn.Parameter(torch.zeros(obs_dim))
        self.o_weight, self.o_bias = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.zeros(dim))

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "calls"] = torch.tensor(self.calls, device="cpu")

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if prefix + "calls" in state_dict:                 # (dictionaries without it are loaded as before)
            self.calls = int(state_dict[prefix + "calls"])
            if prefix + "calls" in unexpected_keys:
                unexpected_keys.remove(prefix + "calls")

    def _key_weight(self) -> torch.Tensor:
        """k_weight, or where a value of it is over dim^-0.5 as much of it as leaves none: a normed key's square is dim at most.
        (Three small launches, some 20 us of a step's 220.)"""
        most, = _FLOAT.unpack(_FLOAT.pack(self.dim ** -0.5))   # (as a weight of float32 has it: its first values are not over it)
        return torch.renorm(self.k_weight.unsqueeze(0), math.inf, 0, most).squeeze(0)

    def _inputs(self, obs: torch.Tensor, positions):
        obs = layers.layer_norm(obs.float(), self.obs_weight, self.obs_bias)
        x = nn.functional.linear(obs.to(self.dtype), self.qkv.weight.to(self.dtype))
        x = x.unflatten(-1, (2 * self.key_heads + self.heads, self.dim))
        q, k, v = x.split((self.key_heads, self.key_heads, self.heads), -2)
        a, b = nn.functional.linear(obs, self.gates.weight, self.gates.bias).chunk(2, -1)
        q, k = memory.norm_rotate(q, k, self.turns, self.q_weight, self._key_weight(), positions)
        return q, k, v, nn.functional.softplus(a) * self.log_decay, torch.sigmoid(b)

    def _normed(self, o: torch.Tensor) -> torch.Tensor:
        return layers.layer_norm(o, self.o_weight, self.o_bias)

    def forward(self, obs: torch.Tensor, state=None, positions=None, offsets=None, call: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """As TickMemory.forward. call: the generator's, where values are dropped; None: `calls`, which counts such forwards. A forward that
        is run again for its backward (activation checkpointing) has to be given it, or it would drop other values: it is refused."""
        offsets, positions = self._places(obs, state, positions, offsets)
        o, end = delta_attention(*self._inputs(obs, positions), state, offsets=offsets)
        o = self._normed(o)
        if self.training and self.dropout:
            if not isinstance(self.seed, torch.Tensor) and torch.cuda.is_current_stream_capturing():
                raise FlyguyError("each replay of a captured forward would drop the same values: seed must be an int64 tensor")
            if call is None:
                if torch._C._current_graph_task_id() != -1:    # (inside a backward)
                    raise FlyguyError("a forward that is run again for its backward would drop other values: give it its call, as the first time")
                call, self.calls = self.calls, self.calls + 1
            o = layers.dropout(o, self.dropout, self.seed, call=call)
        return self._logits(o), end

    @torch.no_grad()
    def step(self, obs: torch.Tensor, state: torch.Tensor, positions: torch.Tensor, slots=None) -> torch.Tensor:
        """As TickMemory.step; nothing is dropped."""
        x = self._inputs(obs.unsqueeze(1), positions.unsqueeze(1))
        return self._logits(self._normed(delta_step(*(t.squeeze(1) for t in x), state, slots=slots)))
