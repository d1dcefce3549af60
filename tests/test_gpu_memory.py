"""The memory-over-ticks operators (flyguy_b200.memory) against their definitions in float64 numpy, written tick by tick
and pair by pair, at the sizes, layouts and masks where they can go wrong; gradients against the formulas and against
differences of the forward.

Tolerances, of ||got - want|| / ||want|| (TOL) and max|got - want| / max|want| (twice that):
  float32    5e-6: sums of up to some 1,000 products, each rounded at 2^-24 (about sqrt(1000) 2^-24 = 2e-6), and operands
             split into 16-bit terms keep 2^-17 of each value at worst (7e-6, 1e-6 in the mean)
  bfloat16   4e-3 = 2^-8: the result's rounding (2^-9 at worst) and as much again for states and weights rounded to the
             type inside a tile
  float16    5e-4 = 2^-11, the same at three more bits
"""
import math

import numpy as np
import pytest
import torch

from flyguy_b200 import memory
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 5e-6, torch.bfloat16: 4e-3, torch.float16: 5e-4}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda t: str(t).replace("torch.", "")   # noqa: E731


def _near(got, want, tol, what="", of=None):
    """of: what the rounding is relative to, where `want` is a difference of larger terms."""
    got = got.detach().double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.size:
        return
    assert np.isfinite(got).all() == np.isfinite(want).all(), what
    off = np.abs(got - want)
    of = want if of is None else of
    assert np.linalg.norm(off) <= tol * max(np.linalg.norm(of), 1e-30), (what, np.linalg.norm(off) / np.linalg.norm(of))
    assert off.max() <= 2 * tol * max(np.abs(of).max(), 1e-30), (what, off.max() / np.abs(of).max())


def _rand(g, *shape, typ=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(typ).cuda()


def _np(t):
    return t.detach().double().cpu().numpy()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- rotation ------------------------------------------------------------------------------------------------------

def _frequencies(turned):
    return np.array([10000.0 ** (-2 * i / turned) for i in range(turned // 2)])


def _turn(x, positions, turned, layout, amplitude, sign=1):
    """x [B, T, H, D] float64 with its pairs turned, as complex numbers."""
    n = turned // 2
    unit = amplitude * np.exp(1j * sign * positions[..., None].astype(np.float64) * _frequencies(turned))[:, :, None, :]
    p = np.arange(n) if layout == "half" else 2 * np.arange(n)
    q = p + n if layout == "half" else p + 1
    z = (x[..., p] + 1j * x[..., q]) * unit
    y = x.copy()
    y[..., p], y[..., q] = z.real, z.imag
    return y


def _norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def _norm_grads(x, w, g, eps):
    """gradients of sum(g * _norm(x, w)) in x and w (w [H, D])."""
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh, gw = x * r, g * w
    return r * (gw - xh * (gw * xh).mean(-1, keepdims=True)), (g * xh).sum((0, 1))


SHAPES = [(1, 1, 1, 64, 64), (3, 7, 5, 128, 64), (2, 33, 3, 80, 80), (1, 5, 2, 7, 6), (2, 4, 1, 1, 0), (1, 3, 8, 256, 256),
          (2, 3, 2, 300, 40), (5, 1, 4, 72, 72), (1, 130, 12, 96, 48)]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotate(shape, layout, typ, cuda):
    B, T, H, D, R = shape
    g = _gen(1)
    x, gy = _rand(g, B, T, H, D, typ=typ).requires_grad_(), _rand(g, B, T, H, D, typ=typ)
    positions = torch.randint(-1000, 2_000_000, (B, T), generator=g)
    y = memory.rotate(x, memory.rotary_turns(R, device="cuda"), positions.cuda(), layout, 1.25)
    y.backward(gy)
    p = positions.numpy()
    _near(y, _turn(_np(x), p, R, layout, 1.25), TOL[typ], "y")
    _near(x.grad, _turn(_np(gy), p, R, layout, 1.25, -1), TOL[typ], "gx")


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("each", [False, True], ids=["one", "each"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotate(shape, layout, each, typ, cuda):
    """Queries and keys as slices of one projection's result; weights for all heads or each head's own; one empty tick."""
    B, T, H, D, R = shape
    K = max(1, H // 2)
    g = _gen(2)
    packed = _rand(g, B, T, H + 2 * K, D, typ=typ, scale=2.0)
    packed[0, 0, 0] = 0                                                     # a head of zeros stays zeros
    packed.requires_grad_()
    q, k = packed[:, :, :H], packed[:, :, H:H + K]
    wq = (1 + 0.2 * _rand(g, *((H, D) if each else (D,)))).requires_grad_()
    wk = (1 + 0.2 * _rand(g, *((K, D) if each else (D,)))).requires_grad_()
    gy, gz = _rand(g, B, T, H, D, typ=typ), _rand(g, B, T, K, D, typ=typ)
    positions = torch.randint(0, 100_000, (T,), generator=g, dtype=torch.int32)
    y, z = memory.norm_rotate(q, k, memory.rotary_turns(R, device="cuda"), wq, wk, positions.cuda(), layout, eps=1e-3)
    torch.autograd.backward((y, z), (gy, gz))
    p = np.broadcast_to(positions.numpy(), (B, T))
    grads = _np(packed.grad)
    for x, w, out, gout, gx in ((q, wq, y, gy, grads[:, :, :H]), (k, wk, z, gz, grads[:, :, H:H + K])):
        w64 = np.broadcast_to(_np(w), (x.shape[2], D))
        _near(out, _turn(_norm(_np(x), w64, 1e-3), p, R, layout, 1.0), TOL[typ], "out")
        back = _turn(_np(gout), p, R, layout, 1.0, -1)
        want_x, want_w = _norm_grads(_np(x), w64, back, 1e-3)
        terms = back * w64 / np.sqrt((_np(x) ** 2).mean(-1, keepdims=True) + 1e-3)  # (a head of one value: they cancel)
        _near(gx, want_x, TOL[typ], "gx", terms if D == 1 else None)
        _near(w.grad, want_w if each else want_w.sum(0), TOL[torch.float32], "gw")
    assert not grads[:, :, H + K:].any()


# heads of whole 16-byte units: lanes without one, part of a head turned, groups of lanes without a tick, ticks that go round
# the blocks several times
UNITS = [(2, 3, 5, 96, 48), (1, 1, 3, 80, 40), (3, 33, 4, 160, 160), (2, 301, 3, 48, 16), (1, 5, 2, 512, 96), (1, 8000, 1, 512, 512),
         (7, 1, 2, 16, 16), (1, 129, 1, 224, 0)]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("each", [False, True], ids=["one", "each"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", UNITS)
def test_norm_rotate_in_units(shape, layout, each, typ, cuda):
    test_norm_rotate(shape, layout, each, typ, cuda)


def test_norm_rotate_plain_forms(cuda):
    """Without turns, weights or positions; packed ticks; a transposed input; the batch's positions from one row."""
    g = _gen(3)
    q, k = _rand(g, 9, 4, 64), _rand(g, 9, 2, 64)
    y, z = memory.norm_rotate(q, k)
    _near(y, _norm(_np(q), 1.0, 1e-6), 5e-6)
    _near(z, _norm(_np(k), 1.0, 1e-6), 5e-6)
    turns = memory.rotary_turns(64, device="cuda")
    want = _turn(_np(q)[None], np.arange(9)[None], 64, "half", 1.0)[0]
    _near(memory.rotate(q, turns), want, 5e-6)
    _near(memory.rotate(q.transpose(1, 2).contiguous().transpose(1, 2), turns), want, 5e-6)
    x = _rand(g, 3, 9, 4, 64)
    row = torch.arange(9, device="cuda").unsqueeze(0) + 5
    _near(memory.rotate(x, turns, row), _turn(_np(x), np.broadcast_to(np.arange(9) + 5, (3, 9)), 64, "half", 1.0), 5e-6)
    odd = torch.empty(9 * 4 * 64 + 1, device="cuda")[1:].view(9, 4, 64).copy_(q)           # not 16-byte aligned
    _near(memory.rotate(odd, turns), want, 5e-6)
    assert memory.rotate(x[:, :0], turns).shape == (3, 0, 4, 64)
    assert torch.equal(memory.rotate(q, memory.rotary_turns(0, device="cuda")), q)


def test_rotation_far_out_is_exact(cuda):
    """Positions past 2^31: the turns of 64-bit fixed point keep the angle (here against Python's own integers)."""
    pos = [2 ** 31 + 7, 2 ** 40 + 123456789, -5]
    x = torch.tensor([1.0, 0.0], device="cuda").expand(3, 1, 2)
    turns = memory.rotary_turns(2, base=10000.0, device="cuda")
    y = memory.rotate(x, turns, torch.tensor(pos, device="cuda")).cpu().numpy()[:, 0]
    for p, got in zip(pos, y):
        a = 2 * math.pi * ((p * int(turns[0])) % 2 ** 64) / 2 ** 64
        assert abs(got[0] - math.cos(a)) < 3e-7 and abs(got[1] - math.sin(a)) < 3e-7


def test_norm_rotate_gradient_against_differences(cuda):
    """Central differences of the forward along random directions, step 1e-2: third-order terms of about step^2 and the
    rounding of sums of 3,000 products over the step leave 1e-3."""
    g = _gen(4)
    ins = [_rand(g, 2, 11, 4, 64), _rand(g, 2, 11, 2, 64), 1 + 0.1 * _rand(g, 64), 1 + 0.1 * _rand(g, 2, 64)]
    turns = memory.rotary_turns(32, device="cuda")
    gy, gz = _rand(g, 2, 11, 4, 64), _rand(g, 2, 11, 2, 64)

    def loss(q, k, wq, wk):
        y, z = memory.norm_rotate(q, k, turns, wq, wk, layout="interleaved")
        return (y.double() * gy).sum() + (z.double() * gz).sum()

    leaves = [t.clone().requires_grad_() for t in ins]
    loss(*leaves).backward()
    for i, t in enumerate(leaves):
        d = t.grad / t.grad.norm()                                          # along the gradient itself
        step = 1e-2 * t.detach().norm()
        plus, minus = list(ins), list(ins)
        plus[i], minus[i] = ins[i] + step * d, ins[i] - step * d
        slope = (loss(*plus) - loss(*minus)).item() / (2 * step.item())
        assert abs(slope - t.grad.norm().item()) <= 1e-3 * t.grad.norm().item(), i


def test_infinities_stay_in_what_is_turned(cuda):
    """An infinite value turns its partner into infinity or not-a-number, and nothing else: not the values left alone."""
    for layout, partner in (("half", 24), ("interleaved", 9)):
        x = _rand(_gen(5), 1, 3, 2, 128, typ=torch.bfloat16)
        x[0, 1, 0, 8] = x[0, 1, 0, 100] = float("inf")
        y = memory.rotate(x, memory.rotary_turns(32, device="cuda"), layout=layout).float()
        bad = ~torch.isfinite(y)
        assert bad[0, 1, 0, 100] and bad[0, 1, 0, 8] and bad[0, 1, 0, partner]
        assert bad.sum().item() == 3, layout


# ---- attention whose state decays ----------------------------------------------------------------------------------

def _wide(x, heads):
    return np.repeat(x, heads // x.shape[-2], -2)


def _scan(q, k, v, log_decay, state, scale):
    """One recording tick by tick in float64: q [T, H, D], k [T, K, D], v [T, K, E], state [H, D, E]."""
    H = q.shape[1]
    k, v = _wide(k, H), _wide(v, H)
    with np.errstate(over="ignore"):
        gamma = np.exp(log_decay)[:, None, None]
    S, o, states = state.copy(), np.zeros((*q.shape[:2], v.shape[-1])), []
    for t in range(len(q)):
        S = gamma * S + k[t][:, :, None] * v[t][:, None, :]
        states.append(S)
        o[t] = np.einsum("hd,hde->he", q[t], S) * scale
    return o, S, states


def _scan_grads(q, k, v, log_decay, state, scale, go, gend):
    H, K = q.shape[1], k.shape[1]
    _, _, states = _scan(q, k, v, log_decay, state, scale)
    kw, vw = _wide(k, H), _wide(v, H)
    gamma = np.exp(log_decay)[:, None, None]
    gq, gk, gv = np.zeros_like(q), np.zeros_like(kw), np.zeros_like(vw)
    R = gend.copy()
    for t in reversed(range(len(q))):
        R = R + scale * q[t][:, :, None] * go[t][:, None, :]
        gq[t] = scale * np.einsum("hde,he->hd", states[t], go[t])
        gk[t] = np.einsum("hde,he->hd", R, vw[t])
        gv[t] = np.einsum("hde,hd->he", R, kw[t])
        R = gamma * R
    add = lambda x: x.reshape(len(x), K, H // K, x.shape[-1]).sum(2)   # noqa: E731
    return gq, add(gk), add(gv), R


def _decays(H, kind="spread"):
    if kind == "strong":                                                   # forgets within a tick or at once
        return torch.tensor([-100.0, -5.0, -float("inf"), -0.7, 0.0])[torch.arange(H) % 5]
    return torch.log1p(-torch.exp2(-4.0 - 6.0 * torch.arange(H) / max(1, H - 1)))


# batch, ticks, heads, key heads, dim, value dim
ATTENTION = [(2, 1, 2, 2, 64, 64), (1, 2, 4, 1, 64, 64), (3, 127, 2, 2, 64, 64), (2, 128, 1, 1, 128, 128),
             (1, 129, 6, 3, 128, 128), (2, 300, 2, 1, 64, 128), (1, 77, 3, 3, 40, 24), (1, 50, 1, 1, 1, 1),
             (2, 33, 2, 2, 100, 17), (1, 20, 2, 2, 256, 256), (1, 1100, 1, 1, 128, 128), (1, 900, 4, 2, 64, 64),
             (1, 700, 1, 1, 128, 64), (2, 640, 1, 1, 96, 80)]


def _attention_case(shape, typ, decays, with_state, seed=5):
    B, T, H, K, D, E = shape
    g = _gen(seed)
    q, k, v = _rand(g, B, T, H, D, typ=typ), _rand(g, B, T, K, D, typ=typ), _rand(g, B, T, K, E, typ=typ)
    state = _rand(g, B, H, D, E, scale=2.0) if with_state else None
    go, gend = _rand(g, B, T, H, E, typ=typ), _rand(g, B, H, D, E, scale=0.3)
    return q, k, v, _decays(H, decays).cuda(), state, go, gend


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("decays,with_state", [("spread", True), ("spread", False), ("strong", True)])
@pytest.mark.parametrize("shape", ATTENTION)
def test_decay_attention(shape, decays, with_state, typ, cuda):
    q, k, v, ld, state, go, gend = _attention_case(shape, typ, decays, with_state)
    leaves = [t.requires_grad_() for t in (q, k, v)] + ([state.requires_grad_()] if with_state else [])
    o, end = memory.decay_attention(q, k, v, ld, state)
    grads = torch.autograd.grad((o, end), leaves, (go, gend))
    scale = shape[4] ** -0.5
    zero = np.zeros(tuple(end.shape[1:]))
    want = [(*_scan(_np(q)[b], _np(k)[b], _np(v)[b], _np(ld), _np(state)[b] if with_state else zero, scale)[:2],
             *_scan_grads(_np(q)[b], _np(k)[b], _np(v)[b], _np(ld), _np(state)[b] if with_state else zero, scale,
                          _np(go)[b], _np(gend)[b])) for b in range(shape[0])]
    want = [np.stack(x) for x in zip(*want)]
    tols = [TOL[typ], TOL[torch.float32], TOL[typ], TOL[typ], TOL[typ], TOL[torch.float32]]
    for name, got, w, tol in zip(("o", "end", "gq", "gk", "gv", "gstate"), (o, end, *grads), want, tols):
        _near(got, w, tol, name)


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("dims", [(4, 2, 64, 64), (2, 2, 128, 128), (3, 1, 20, 36)])
@pytest.mark.parametrize("lengths", [[0], [5], [0, 130, 0, 0, 1, 257, 128, 0], [700, 3, 1500], [1] * 9])
def test_packed_recordings(lengths, dims, typ, cuda):
    """Recordings end to end, empty ones among them: each as if alone, an empty one's state and its gradient handed on."""
    H, K, D, E = dims
    g, n, N = _gen(6), sum(lengths), len(lengths)
    q, k, v = _rand(g, n, H, D, typ=typ), _rand(g, n, K, D, typ=typ), _rand(g, n, K, E, typ=typ)
    state, go, gend = _rand(g, N, H, D, E), _rand(g, n, H, E, typ=typ), _rand(g, N, H, D, E, scale=0.3)
    ld, scale = _decays(H).cuda(), 0.2
    leaves = [t.requires_grad_() for t in (q, k, v, state)]
    off = np.concatenate([[0], np.cumsum(lengths)])
    o, end = memory.decay_attention(q, k, v, ld, state, scale, torch.tensor(off, device="cuda"))
    gq, gk, gv, gs = torch.autograd.grad((o, end), leaves, (go, gend))
    per = []
    for i in range(N):
        a = slice(off[i], off[i + 1])
        one = [_np(x)[a] for x in (q, k, v)] + [_np(ld), _np(state)[i], scale]
        per.append((*_scan(*one)[:2], *_scan_grads(*one, _np(go)[a], _np(gend)[i])))
    cols = list(zip(*per))
    for name, got, col, stack, tol in (("o", o, 0, False, TOL[typ]), ("end", end, 1, True, 5e-6), ("gq", gq, 2, False, TOL[typ]),
                                       ("gk", gk, 3, False, TOL[typ]), ("gv", gv, 4, False, TOL[typ]), ("gs", gs, 5, True, 5e-6)):
        _near(got, np.stack(cols[col]) if stack else np.concatenate(cols[col]), tol, name)


@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_strided_inputs_and_pieces(typ, cuda):
    """q, k, v as slices of one projection, gradients of an expanded sum; a recording in pieces through its states equals
    the recording in one call."""
    g = _gen(7)
    B, T, H, D = 2, 260, 2, 64
    packed = _rand(g, B, T, 3 * H, D, typ=typ).requires_grad_()
    ld = _decays(H).cuda()
    o, end = memory.decay_attention(packed[:, :, :H], packed[:, :, H:2 * H], packed[:, :, 2 * H:], ld)
    o.sum().backward()                                                      # (an expanded gradient, all strides 0)
    x = _np(packed)
    for b in range(B):
        parts = [x[b][:, i * H:(i + 1) * H] for i in range(3)]
        zero, scale = np.zeros((H, D, D)), D ** -0.5
        w = _scan(*parts, _np(ld), zero, scale)
        _near(o[b], w[0], TOL[typ], "o")
        gr = _scan_grads(*parts, _np(ld), zero, scale, np.ones((T, H, D)), zero)
        _near(packed.grad[b], np.concatenate(gr[:3], 1), TOL[typ], "grad")
    with torch.no_grad():
        state, outs = None, []
        for a, z in ((0, 1), (1, 100), (100, 100), (100, 260)):
            y, state = memory.decay_attention(*(packed[:, a:z, i * H:(i + 1) * H] for i in range(3)), ld, state)
            outs.append(y)
    _near(torch.cat(outs, 1), _np(o), TOL[typ], "pieces")
    _near(state, _np(end), 5e-6, "state of the pieces")


def test_same_bits_on_every_run(cuda):
    q, k, v, ld, state, go, gend = _attention_case((1, 1500, 4, 2, 128, 128), torch.bfloat16, "spread", True)
    runs = []
    for _ in range(3):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, state)]
        o, end = memory.decay_attention(*leaves[:3], ld, leaves[3])
        runs.append([o, end, *torch.autograd.grad((o, end), leaves, (go, gend))])
    for r in runs[1:]:
        for a, b in zip(runs[0], r):
            assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 48])
@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_not_a_number_stays_in_its_recording_and_head(typ, D, cuda):
    """A recording with NaN and infinite values in its ticks, in the padding of a tile's other half or beyond its end, leaves
    the other recordings and heads alone, and the ticks before it in another tile of 128."""
    g = _gen(8)
    off = torch.tensor([0, 140, 330, 400], device="cuda")
    q, k, v = (_rand(g, 400, 2, D, typ=typ) for _ in range(3))
    clean, clean_end = memory.decay_attention(q, k, v, _decays(2).cuda(), offsets=off)
    k2, v2 = k.clone(), v.clone()
    k2[300, 0, 3], v2[301, 0, 5] = float("nan"), float("inf")               # recording 1, its second tile, head 0
    o, end = memory.decay_attention(q, k2, v2, _decays(2).cuda(), offsets=off)
    for a, b in ((slice(0, 140), 0), (slice(330, 400), 2)):
        assert torch.equal(o[a], clean[a]) and torch.equal(end[b], clean_end[b])
    assert torch.equal(o[:, 1], clean[:, 1]) and torch.equal(o[140:140 + 128, 0], clean[140:140 + 128, 0])
    assert not torch.isfinite(o[300:330, 0]).all()


def test_decay_attention_gradient_against_differences(cuda):
    """The forward is linear in each of q, k, v and the state: a difference over the whole step is the gradient, up to the
    rounding of its sums (1e-4 of it)."""
    q, k, v, ld, state, go, gend = _attention_case((2, 150, 4, 2, 64, 64), torch.float32, "spread", True)
    ins = [q, k, v, state]

    def loss(q, k, v, state):
        o, end = memory.decay_attention(q, k, v, ld, state)
        return (o.double() * go).sum() + (end.double() * gend).sum()

    leaves = [t.clone().requires_grad_() for t in ins]
    loss(*leaves).backward()
    for i, t in enumerate(leaves):
        d = t.grad / t.grad.norm() * t.detach().norm()
        plus = list(ins)
        plus[i] = ins[i] + d
        slope = (loss(*plus) - loss(*ins)).item()
        want = (t.grad.double() * d).sum().item()
        assert abs(slope - want) <= 1e-4 * want, i


# ---- one tick -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("dims", [(1, 1, 1, 64, 64), (8, 8, 2, 64, 64), (3, 4, 4, 128, 128), (5, 2, 1, 40, 24), (2, 1, 1, 1, 1),
                                  (2, 2, 2, 256, 256), (4, 3, 1, 17, 129), (2, 2, 1, 128, 64)])
def test_decay_step(dims, typ, cuda):
    B, H, K, D, E = dims
    g = _gen(9)
    q, k, v = _rand(g, B, H, D, typ=typ), _rand(g, B, K, D, typ=typ), _rand(g, B, K, E, typ=typ)
    pool = _rand(g, B + 3, H, D, E)
    slots = torch.randperm(B + 3, generator=g)[:B].cuda()
    ld, before = _decays(H).cuda(), _np(pool)
    o = memory.decay_step(q, k, v, ld, pool, slots=slots)
    want = before.copy()
    for b, s in enumerate(slots.tolist()):
        y, S, _ = _scan(_np(q)[b][None], _np(k)[b][None], _np(v)[b][None], _np(ld), before[s], D ** -0.5)
        want[s] = S
        _near(o[b], y[0], TOL[typ], "o")
    _near(pool, want, 1e-6, "states")                                       # (one product and one sum a value)


def test_decay_step_slots_out_of_range(cuda):
    """A slot below 0 or past the pool answers zeros and leaves every state as it was (rows that pad a batch)."""
    g = _gen(10)
    q, k, v, pool = _rand(g, 4, 2, 64), _rand(g, 4, 2, 64), _rand(g, 4, 2, 64), _rand(g, 3, 2, 64, 64)
    before = pool.clone()
    o = memory.decay_step(q, k, v, _decays(2).cuda(), pool, slots=torch.tensor([-1, 1, 3, 2 ** 40], device="cuda"))
    assert not o[[0, 2, 3]].any() and o[1].any()
    assert torch.equal(pool[[0, 2]], before[[0, 2]]) and not torch.equal(pool[1], before[1])


@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_steps_equal_the_whole_recording(typ, cuda):
    g = _gen(11)
    B, T, H, K, D = 3, 40, 4, 2, 64
    q, k, v = _rand(g, B, T, H, D, typ=typ), _rand(g, B, T, K, D, typ=typ), _rand(g, B, T, K, D, typ=typ)
    ld = _decays(H).cuda()
    o, end = memory.decay_attention(q, k, v, ld)
    state = torch.zeros_like(end)
    each = torch.stack([memory.decay_step(q[:, t], k[:, t], v[:, t], ld, state) for t in range(T)], 1)
    _near(each, _np(o), 2 * TOL[typ], "o")
    _near(state, _np(end), 5e-6, "state")


def test_on_another_stream(cuda):
    """The work runs on torch's current stream: behind a long kernel there, not beside it."""
    g = _gen(12)
    src = _rand(g, 2, 64, 2, 64)
    x = torch.zeros_like(src)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            big = big @ big * 1e-3
        x.copy_(src)
        o, _ = memory.decay_attention(x, x, x, _decays(2).cuda())
    s.synchronize()
    want, _ = memory.decay_attention(src, src, src, _decays(2).cuda())
    assert torch.equal(o, want)


# ---- refusals -------------------------------------------------------------------------------------------------------

def _refused(match, fn, *args, **kw):
    with pytest.raises(FlyguyError, match=match):
        fn(*args, **kw)


def test_rotation_refusals(cuda):
    x, turns = torch.zeros(2, 3, 4, 64, device="cuda"), memory.rotary_turns(64, device="cuda")
    w = torch.ones(64, device="cuda")
    _refused("CUDA", memory.rotate, x.cpu(), turns)
    _refused("float32, bfloat16 or float16", memory.rotate, x.double(), turns)
    _refused("dimensions", memory.rotate, x[0, 0], turns)
    _refused("int64", memory.rotate, x, turns.int())
    _refused("a head has 32", memory.rotate, x[..., :32], turns)
    _refused("layout", memory.rotate, x, turns, layout="whole")
    _refused("positions", memory.rotate, x, turns, torch.zeros(2, 4, dtype=torch.int64, device="cuda"))
    _refused("positions", memory.rotate, x, turns, torch.zeros(2, 3, device="cuda"))
    _refused("k must be", memory.norm_rotate, x, x[:, :2], turns)
    _refused("type", memory.norm_rotate, x, x.half(), turns)
    _refused("eps", memory.norm_rotate, x, x, turns, eps=0.0)
    _refused("q_weight", memory.norm_rotate, x, x, turns, w[:32], w)
    _refused("k_weight", memory.norm_rotate, x, x, turns, w, w.half())
    _refused("even", memory.rotary_turns, 3)
    _refused("scaling", memory.rotary_turns, 4, scaling="other")


def test_decay_refusals(cuda):
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)   # noqa: E731
    q, k, ld, state = z(2, 5, 4, 64), z(2, 5, 2, 64), z(4), z(2, 4, 64, 64)
    f = memory.decay_attention
    _refused("CUDA", f, q.cpu(), k, k, ld)
    _refused("k and v", f, q, z(2, 5, 2, 32), k, ld)
    _refused("k and v", f, q, k, k[:, :4], ld)
    _refused("share", f, q, z(2, 5, 3, 64), z(2, 5, 3, 64), ld)
    _refused("log_decay", f, q, k, k, z(3))
    _refused("log_decay", f, q, k, k, ld.double())
    _refused("constant", f, q, k, k, ld.clone().requires_grad_())
    _refused("state", f, q, k, k, ld, state[:1])
    _refused("state", f, q, k, k, ld, state.half())
    _refused("end to end", f, q, k, k, ld, offsets=z(3, dtype=torch.int64))
    _refused("offsets", f, q[0], k[0], k[0], ld, offsets=z(3, dtype=torch.int32))
    _refused("1 to 256", f, z(1, 2, 1, 257), z(1, 2, 1, 257), z(1, 2, 1, 8), z(1))
    s = memory.decay_step
    _refused("state", s, q[:, 0], k[:, 0], k[:, 0], ld, state.transpose(2, 3))
    _refused("as many states", s, q[:, 0], k[:, 0], k[:, 0], ld, state[:1])
    _refused("slots", s, q[:, 0], k[:, 0], k[:, 0], ld, state, slots=z(2, dtype=torch.int32))
    _refused("no gradient", s, q[:, 0].clone().requires_grad_(), k[:, 0], k[:, 0], ld, state)


def test_offsets_are_never_followed_out_of_the_buffers(cuda):
    """Offsets past the ticks or falling are clamped: what they name inside is worked on, nothing outside is read."""
    g = _gen(13)
    q, k, v = (_rand(g, 40, 1, 64) for _ in range(3))
    o, end = memory.decay_attention(q, k, v, _decays(1).cuda(), offsets=torch.tensor([0, 30, 10, 2 ** 50], device="cuda"))
    want, want_end = memory.decay_attention(q[:30], k[:30], v[:30], _decays(1).cuda(), offsets=torch.tensor([0, 30], device="cuda"))
    assert torch.equal(end[0], want_end[0]) and not end[1].any()
