"""The gated delta rule (flyguy_b200.delta) against its definition in float64, tick by tick (gradients: of that definition, and
differences of the forward), at the sizes, layouts and gates where it can go wrong.

Tolerances, of ||got - want|| / ||want|| (TOL) and max|got - want| / max|want| (twice that). A rounding to bf16 is 2^-9 of a value at
worst and 2^-9 / sqrt(3) in the mean, 1.1e-3.
  o, gq, gk, gv of bfloat16  2^-7: the result's rounding and those of three once rounded operands in each of up to four
             products, 1.1e-3 sqrt(4) sqrt(4) = 4.5e-3
  the same of float16        2^-10: operands have two terms, what is left is the result's rounding 2^-11 (2^-12.8 in the mean),
             and as much again for two gradients added before it
  states, gates' gradients of bfloat16 inputs  3e-5: two terms leave 2^-18 of a value, 2^-17 at worst, in up to five places; a gate's
             gradient is a sum of up to 64 differences of what these give
  float32, and states and gates of float16     1e-5: three terms leave 2^-26, sums of some 1,000 products round at 2^-24 each,
             sqrt(1000) 2^-24 = 2e-6, over the up to 5 products that follow one another"""
import itertools
import math

import numpy as np
import pytest
import torch

from flyguy_b200 import delta, memory
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
KEPT = {torch.float32: 1e-5, torch.bfloat16: 3e-5, torch.float16: 1e-5}
names = lambda t: str(t).replace("torch.", "")   # noqa: E731
NAMES = ("q", "k", "v", "log_decay", "beta", "state")


def _near(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.numel():
        return
    assert torch.isfinite(got).all(), what
    off = got - want
    assert off.norm() <= tol * want.norm().clamp(min=1e-30), (what, (off.norm() / want.norm()).item())
    assert off.abs().max() <= 2 * tol * want.abs().max().clamp(min=1e-30), (what, (off.abs().max() / want.abs().max()).item())


def _rule(q, k, v, log_decay, beta, state, scale):
    """[T, heads, .] of one recording, in float64: o [T, H, E] and the last state."""
    H = log_decay.shape[-1]
    wide = lambda x: x.repeat_interleave(H // x.shape[-2], -2)   # noqa: E731
    q, k, v, S, out = wide(q), wide(k), wide(v), state, []
    for t in range(len(q)):
        S = S * log_decay[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hd,hde->he", k[t], S))
        S = S + k[t].unsqueeze(-1) * u.unsqueeze(-2)
        out.append(scale * torch.einsum("hd,hde->he", q[t], S))
    return (torch.stack(out) if out else q.new_zeros(0, H, v.shape[-1])), S


def _inputs(seed, lead, recordings, H, heads, D, E, typ, state=True):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)               # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp(min=1e-6)   # noqa: E731
    x = {"q": unit(rand(*lead, heads[0], D) + 0.4).to(typ), "k": unit(rand(*lead, heads[1], D) + 0.4).to(typ),
         "v": (0.5 * rand(*lead, heads[2], E)).to(typ), "log_decay": -0.2 * torch.rand(*lead, H, generator=g) ** 3,
         "beta": torch.rand(*lead, H, generator=g)}
    if state:
        x["state"] = 0.3 * rand(recordings, H, D, E)
    go, gs = rand(*lead, H, E).to(typ), 0.1 * rand(recordings, H, D, E)
    return x, go, gs


def _want(x, spans, go, gs, scale):
    """o, states and gradients in float64; spans: (first, end) of each recording, or None: [batch, ticks, ..]."""
    leaves = {n: t.double().requires_grad_() for n, t in x.items()}
    H, D, E = x["log_decay"].shape[-1], x["q"].shape[-1], x["v"].shape[-1]
    rows = range(len(x["q"])) if spans is None else range(len(spans))
    cut = lambda t, b: t[b] if spans is None else t[spans[b][0]:spans[b][1]]   # noqa: E731
    outs, ends, total = [], [], 0.0
    for b in rows:
        first = leaves["state"][b] if "state" in x else torch.zeros(H, D, E, dtype=torch.float64)
        o, end = _rule(*(cut(leaves[n], b) for n in NAMES[:5]), first, scale)
        outs.append(o)
        ends.append(end)
        total = total + (o * cut(go.double(), b)).sum() + (end * gs[b].double()).sum()
    grads = torch.autograd.grad(total, list(leaves.values()), allow_unused=True) if isinstance(total, torch.Tensor) else [None] * len(leaves)
    grads = {n: torch.zeros_like(leaves[n]) if g is None else g for n, g in zip(leaves, grads)}
    return outs, ends, grads


def _run(x, go, gs, scale=None, offsets=None):
    leaves = {n: t.cuda().requires_grad_() for n, t in x.items()}
    o, end = delta.delta_attention(*leaves.values(), scale=scale, offsets=offsets)
    grads = torch.autograd.grad((o, end), list(leaves.values()), (go.cuda(), gs.cuda()))
    return o, end, dict(zip(leaves, grads))


def _compare(x, go, gs, typ, spans=None, offsets=None, scale=None):
    want_o, want_end, want = _want(x, spans, go, gs, x["q"].shape[-1] ** -0.5 if scale is None else scale)
    o, end, got = _run(x, go, gs, scale, offsets)
    _near(o, torch.cat(want_o) if spans is not None else torch.stack(want_o), TOL[typ], "o")
    _near(end, torch.stack(want_end), KEPT[typ], "state")
    for n in got:
        assert got[n].dtype is x[n].dtype
        _near(got[n], want[n], TOL[typ] if n in "qkv" else KEPT[typ], "gradient of " + n)
    with torch.no_grad():                                        # (forward alone: the same states, o of its own number of terms)
        again = delta.delta_attention(*(t.cuda() for t in x.values()), scale=scale, offsets=offsets)
    _near(again[0], torch.cat(want_o) if spans is not None else torch.stack(want_o), TOL[typ], "o alone")
    assert torch.equal(again[1], end)


# batch, ticks, heads, query / key / value heads, dim, value dim
SHAPES = [(1, 1, 1, (1, 1, 1), 1, 1), (2, 31, 2, (2, 2, 2), 64, 64), (1, 32, 4, (4, 2, 2), 40, 37), (3, 33, 2, (1, 1, 2), 7, 16),
          (1, 64, 2, (2, 1, 1), 128, 128), (2, 65, 3, (3, 3, 3), 72, 130), (1, 97, 2, (1, 2, 1), 16, 256), (1, 129, 1, (1, 1, 1), 127, 5),
          (2, 200, 4, (2, 1, 4), 96, 80), (5, 3, 6, (6, 3, 2), 65, 64), (1, 128, 2, (2, 2, 2), 100, 17)]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, (*s[:3], *s[3], *s[4:]))))
def test_delta_attention(shape, typ, cuda):
    B, T, H, heads, D, E = shape
    x, go, gs = _inputs(1, (B, T), B, H, heads, D, E, typ)
    _compare(x, go, gs, typ)


@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_packed_recordings(typ, cuda):
    """Empty ones first, last and between; one tick; whole chunks and slots; ends inside a chunk; four query heads a key head."""
    lengths = [0, 1, 64, 0, 0, 130, 32, 63, 96, 0]
    off = [0, *itertools.accumulate(lengths)]
    x, go, gs = _inputs(2, (off[-1],), len(lengths), 4, (4, 1, 1), 64, 48, typ)
    _compare(x, go, gs, typ, list(zip(off, off[1:])), torch.tensor(off, device=cuda))


def test_ticks_of_no_recording_are_zeros(cuda):
    x, go, gs = _inputs(3, (200,), 2, 2, (2, 1, 1), 64, 64, torch.bfloat16)
    off = torch.tensor([7, 40, 150], device=cuda)
    o, _, g = _run(x, go, gs, offsets=off)
    for t in (o, *(g[n] for n in NAMES[:5])):
        assert not t[:7].any() and not t[150:].any() and t[7:150].any()
    inside = {n: (t if n == "state" else t[7:150]) for n, t in x.items()}
    _compare(inside, go[7:150], gs, torch.bfloat16, [(0, 33), (33, 143)], off - 7)


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "packed"])
def test_long_recordings_in_parts(typ, ragged, cuda):
    """Few recordings of some 2,600 ticks run in parts (k_delta_join); one much shorter leaves parts without ticks; gates that remember
    the whole of it."""
    lengths = [2600, 64, 0, 2087] if ragged else [2100]
    off = [0, *itertools.accumulate(lengths)]
    lead = (off[-1],) if ragged else (1, 2100)
    x, go, gs = _inputs(4, lead, len(lengths), 1, (1, 1, 1), 40, 40, typ)
    x["log_decay"] *= 0.02
    x["beta"] *= 0.1
    if ragged:
        _compare(x, go, gs, typ, list(zip(off, off[1:])), torch.tensor(off, device=cuda))
    else:
        _compare(x, go, gs, typ)


def test_without_a_state_and_with_a_scale(cuda):
    x, go, gs = _inputs(5, (2, 70), 2, 2, (2, 2, 2), 48, 64, torch.float32, state=False)
    _compare(x, go, gs, torch.float32, scale=0.7)


@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_gates(typ, cuda):
    """Forgetting (minus infinity, the type's lowest, -300), no forgetting, beta 0, 1 and 2, and the same key each tick."""
    x, go, gs = _inputs(6, (2, 100), 2, 2, (2, 2, 2), 32, 32, typ)
    x["log_decay"][:, 10] = -math.inf
    x["log_decay"][:, 45, 0] = torch.finfo(torch.float32).min
    x["log_decay"][:, 50:53, 1] = -300.0
    x["log_decay"][:, 60:] = 0
    x["beta"][:, 20:40] = 0
    x["beta"][:, 64:70] = 1
    x["beta"][1, 70:80] = 2
    x["k"][1, 80:] = x["k"][1, 80:81]
    want_x = {n: t.clone() for n, t in x.items()}
    want_x["log_decay"].clamp_(min=-700)                        # (e^-700 squared is 0 in float64, too, and no inf - inf)
    want_o, want_end, want = _want(want_x, None, go, gs, 32 ** -0.5)
    o, end, got = _run(x, go, gs)
    _near(o, torch.stack(want_o), TOL[typ], "o")
    _near(end, torch.stack(want_end), KEPT[typ], "state")
    for n in got:
        _near(got[n], want[n], TOL[typ] if n in "qkv" else KEPT[typ], n)


def test_what_a_forgotten_state_held_is_gone(cuda):
    """Behind a tick with log_decay of minus infinity nothing of the ticks before is left, not even 1e30 of it."""
    x, _, _ = _inputs(7, (1, 96), 1, 1, (1, 1, 1), 64, 64, torch.float32)
    x["log_decay"][:, 40] = -math.inf
    cut = {n: (t if n == "state" else t[:, 40:]).cuda() for n, t in x.items()}
    cut["state"] = torch.zeros_like(cut["state"])
    x["state"] = x["state"] * 1e30
    x["v"][:, :40] *= 1e30
    _, end = delta.delta_attention(*(t.cuda() for t in x.values()))
    _, want = delta.delta_attention(*cut.values())
    _near(end, want, 1e-5, "state")


def test_a_nan_stays_in_its_recording_and_head(cuda):
    x, _, _ = _inputs(8, (2, 100), 2, 2, (2, 2, 2), 64, 64, torch.bfloat16)
    clean = delta.delta_attention(*(t.cuda() for t in x.values()))
    x["k"][1, 70, 1, 3] = math.nan
    o, end = delta.delta_attention(*(t.cuda() for t in x.values()))
    assert torch.equal(o[0], clean[0][0]) and torch.equal(o[1, :, 0], clean[0][1, :, 0]) and torch.equal(o[1, :64, 1], clean[0][1, :64, 1])
    assert o[1, 96:, 1].isnan().all() and end[1, 1].isnan().any() and torch.equal(end[1, 0], clean[1][1, 0])


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("layout", ["slices", "odd", "turned", "expanded"])
def test_strides(layout, typ, cuda):
    """Slices of one projection's result, heads at odd places, heads before ticks, expanded values: the bits of contiguous copies."""
    B, T, H, D = 2, 50, 2, 40
    g = torch.Generator().manual_seed(9)
    if layout == "slices":
        p = torch.randn(B, T, 3 * H, D, generator=g).to(typ).cuda()
        q, k, v = p.split(H, 2)
    elif layout == "odd":
        p = torch.randn(B, T, 3 * H * D + 3, generator=g).to(typ).cuda()
        q, k, v = (p[..., 1 + i * H * D:1 + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    elif layout == "turned":
        q, k, v = (torch.randn(B, H, T, D, generator=g).to(typ).cuda().transpose(1, 2) for _ in range(3))
    else:
        q, k = (torch.randn(B, T, H, D, generator=g).to(typ).cuda() for _ in range(2))
        v = torch.randn(B, 1, H, D, generator=g).to(typ).cuda().expand(B, T, H, D)
    k = k * (D ** -0.5) if layout == "expanded" else k
    gates = torch.rand(B, H, T, 2, generator=g).cuda()
    log_decay, beta = -0.1 * gates[..., 0].transpose(1, 2), 0.02 * gates[..., 1].transpose(1, 2)
    ins = [t.detach().requires_grad_() for t in (q, k, v, log_decay, beta)]
    o, end = delta.delta_attention(*ins)
    go = torch.randn(B, H, T, D, generator=g).to(typ).cuda().transpose(1, 2)
    grads = torch.autograd.grad((o, end), ins, (go, end.detach()))
    plain = [t.detach().contiguous().clone().requires_grad_() for t in ins]
    o2, end2 = delta.delta_attention(*plain)
    want = torch.autograd.grad((o2, end2), plain, (go.contiguous(), end.detach()))
    assert torch.equal(o, o2) and torch.equal(end, end2)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)


def test_gradients_against_differences(cuda):
    """(f(x + h d) - f(x - h d)) / 2 h along random directions; h = 2^-7: the differences' own error is h^2 of the third derivative,
    6e-5, and the forward's 1e-6 / h = 1e-4 of ||go|| ||o||."""
    x, go, gs = _inputs(10, (2, 75), 2, 2, (2, 1, 2), 24, 40, torch.float32)
    x["log_decay"] -= 0.05
    _, _, grads = _run(x, go, gs)
    x = {n: t.cuda() for n, t in x.items()}

    def f(y):
        o, end = delta.delta_attention(*y.values())
        return (o.double() * go.cuda().double()).sum().item() + (end.double() * gs.cuda().double()).sum().item()

    size = sum(t.double().norm().item() ** 2 for t in delta.delta_attention(*x.values())) ** 0.5
    scale = size * (go.norm() ** 2 + gs.norm() ** 2).sqrt().item()
    g = torch.Generator().manual_seed(11)
    for n in x:
        d = torch.randn(x[n].shape, generator=g).cuda()
        d *= x[n].norm() / d.norm()
        h = 2.0 ** -7
        slope = (f(x | {n: x[n] + h * d}) - f(x | {n: x[n] - h * d})) / (2 * h)
        want = (grads[n].double() * d.double()).sum().item()
        assert abs(slope - want) <= 1e-3 * scale, (n, slope, want, scale)


def test_same_bits_each_run(cuda):
    x, go, gs = _inputs(12, (3, 300), 3, 4, (4, 2, 2), 64, 64, torch.bfloat16)
    one, two = _run(x, go, gs), _run(x, go, gs)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    assert all(torch.equal(one[2][n], two[2][n]) for n in one[2])


@pytest.mark.parametrize("sizes", [(2, 100, 2, (1, 2, 1), 40, 72), (1, 2304, 2, (2, 1, 1), 72, 20)], ids=["chunks", "parts"])
def test_nothing_is_read_that_was_not_written(sizes, monkeypatch, cuda):
    """With every workspace full of NaN first."""
    B, T, H, heads, D, E = sizes
    x, go, gs = _inputs(13, (B, T), B, H, heads, D, E, torch.float16)
    want = _run(x, go, gs)

    def room(size, device):
        t = torch.full((-(-size // 4),), math.nan, device=device)
        return t, (t.data_ptr(), size)

    monkeypatch.setattr(delta, "_room", room)
    got = _run(x, go, gs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(got[2][n], want[2][n]) for n in got[2])


def test_captured_and_replayed(cuda):
    """A graph of forward and backward, replayed on other inputs while another captured call has its own workspace."""
    x, go, gs = _inputs(14, (2, 90), 2, 2, (2, 2, 2), 64, 64, torch.bfloat16)
    y, _, _ = _inputs(15, (2, 90), 2, 2, (2, 2, 2), 64, 64, torch.bfloat16)
    go, gs = go.cuda(), gs.cuda()
    leaves = [t.cuda().requires_grad_() for t in x.values()]

    def step():
        o, end = delta.delta_attention(*leaves)
        return o, end, *torch.autograd.grad((o, end), leaves, (go, gs))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        twin = step()
    for data in (y, x):
        with torch.no_grad():
            for leaf, t in zip(leaves, data.values()):
                leaf.copy_(t)
        want = [t.clone() for t in step()]
        graph.replay()
        other.replay()
        for a, b, c in zip(out, twin, want):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_on_two_streams_at_once(cuda):
    runs = [_inputs(16 + i, (2, 400), 2, 4, (4, 4, 4), 64, 64, torch.bfloat16) for i in range(2)]
    want = [_run(*r) for r in runs]
    runs = [({n: t.cuda() for n, t in x.items()}, go.cuda(), gs.cuda()) for x, go, gs in runs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _run(*runs[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in a[2])


def test_only_some_learn(cuda):
    x, go, gs = _inputs(18, (1, 40), 1, 2, (2, 2, 2), 32, 32, torch.float32)
    _, _, want = _run(x, go, gs)
    for n in x:
        leaves = {m: t.cuda().requires_grad_(m == n) for m, t in x.items()}
        o, end = delta.delta_attention(*leaves.values())
        torch.autograd.backward((o, end), (go.cuda(), gs.cuda()))
        assert torch.equal(leaves[n].grad, want[n]), n
        assert all(t.grad is None for m, t in leaves.items() if m != n)


def test_inputs_made_in_inference_mode_stay_constants(cuda):
    x, go, gs = _inputs(22, (1, 40), 1, 2, (2, 2, 2), 32, 32, torch.float32)
    _, _, want = _run(x, go, gs)
    with torch.inference_mode():
        fixed = {n: t.cuda() for n, t in x.items()}
    v = x["v"].cuda().requires_grad_()
    o, end = delta.delta_attention(*(fixed | {"v": v}).values())
    got, = torch.autograd.grad((o, end), v, (go.cuda(), gs.cuda()))
    assert torch.equal(got, want["v"])


def test_broadcast_gates_learn(cuda):
    """One gate for all ticks and heads, expanded: its gradient is the sum."""
    x, go, gs = _inputs(23, (2, 40), 2, 2, (2, 2, 2), 32, 32, torch.float32)
    x["log_decay"][:], x["beta"][:] = -0.1, 0.3
    _, _, want = _want(x, None, go, gs, 32 ** -0.5)
    gate = torch.tensor([-0.1, 0.3], device=cuda, requires_grad=True)
    c = {n: t.cuda() for n, t in x.items()}
    o, end = delta.delta_attention(c["q"], c["k"], c["v"], gate[0].expand(2, 40, 2), gate[1].expand(2, 40, 2), c["state"])
    got, = torch.autograd.grad((o, end), gate, (go.cuda(), gs.cuda()))
    for g, n in zip(got, ("log_decay", "beta")):
        assert abs(g.item() - want[n].sum().item()) <= 1e-5 * want[n].abs().sum().item()


def test_one_output_alone_learns(cuda):
    """The gradient of o alone, and of the states alone."""
    x, go, gs = _inputs(19, (2, 40), 2, 2, (2, 2, 2), 32, 32, torch.float32)
    for which in (0, 1):
        leaves = [t.cuda().requires_grad_() for t in x.values()]
        out = delta.delta_attention(*leaves)
        got = torch.autograd.grad(out[which], leaves, (go, gs)[which].cuda())
        zero = (go if which == 0 else torch.zeros_like(go), gs if which == 1 else torch.zeros_like(gs))
        _, _, want = _want(x, None, *zero, 32 ** -0.5)
        for n, g in zip(x, got):
            _near(g, want[n], 1e-5, n)


def test_second_derivatives_and_tangents_are_refused(cuda):
    x, go, gs = _inputs(20, (1, 8), 1, 1, (1, 1, 1), 16, 16, torch.float32)
    leaves = [t.cuda().requires_grad_() for t in x.values()]
    o, _ = delta.delta_attention(*leaves)
    g, = torch.autograd.grad(o.sum(), leaves[:1], create_graph=True)
    with pytest.raises(FlyguyError, match="again"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(leaves[4].detach(), torch.ones_like(leaves[4]))
        with pytest.raises(FlyguyError, match="forward-mode"):
            delta.delta_attention(*(t.detach() for t in leaves[:4]), dual, leaves[5].detach())


def test_empty_calls(cuda):
    for lead, n, off in (((0, 5), 0, None), ((2, 0), 2, None), ((0,), 3, [0, 0, 0, 0]), ((6,), 0, [0])):
        x, go, gs = _inputs(21, lead, n, 2, (2, 2, 2), 32, 16, torch.bfloat16)
        o, end, g = _run(x, go, gs, offsets=None if off is None else torch.tensor(off, device=cuda))
        assert o.shape == (*lead, 2, 16) and not o.any()
        assert torch.equal(end.cpu(), x["state"])
        assert torch.equal(g["state"].cpu(), gs)
        assert not any(g[m].any() for m in NAMES[:5])


# ---- a tick at a time ----------------------------------------------------------------------------------------------

# batch, heads, query / key / value heads, dim, value dim, slots
STEPS = [(1, 1, (1, 1, 1), 1, 1, 1), (3, 4, (2, 1, 4), 64, 64, 5), (2, 2, (2, 2, 2), 40, 37, 2), (5, 2, (1, 2, 1), 128, 130, 9),
         (2, 1, (1, 1, 1), 256, 256, 3), (4, 3, (3, 3, 3), 200, 72, 4), (301, 8, (8, 8, 8), 128, 128, 302), (700, 2, (2, 1, 1), 40, 72, 700),
         (600, 2, (2, 2, 2), 60, 256, 640), (1300, 1, (1, 1, 1), 7, 4, 1300)]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("shape", STEPS, ids=lambda s: "x".join(map(str, (*s[:2], *s[3:]))))
def test_delta_step(shape, typ, cuda):
    """Two ticks, the second of the same rows in another order; slots of no row stay as they were."""
    B, H, heads, D, E, slots = shape
    g = torch.Generator().manual_seed(30)
    state = torch.randn(slots, H, D, E, generator=g)
    want, own = state.double(), state.cuda()
    for tick in range(2):
        x, _, _ = _inputs(31 + tick, (B,), 1, H, heads, D, E, typ, state=False)
        at = torch.randperm(slots, generator=g)[:B]
        o = delta.delta_step(*(t.cuda() for t in x.values()), own, slots=at.cuda())
        q, k, v = (x[n].double().repeat_interleave(H // x[n].shape[1], 1) for n in "qkv")
        S = want[at] * x["log_decay"].double().exp()[..., None, None]
        u = x["beta"].double()[..., None] * (v - torch.einsum("bhd,bhde->bhe", k, S))
        want[at] = S + k.unsqueeze(-1) * u.unsqueeze(-2)
        _near(o, torch.einsum("bhd,bhde->bhe", q, want[at]) * D ** -0.5, max(TOL[typ], 1e-5), "o")
    _near(own, want, 1e-6, "state")
    rest = torch.ones(slots, dtype=torch.bool)
    rest[at] = False
    if tick == 0:
        assert torch.equal(own.cpu()[rest], state[rest])


@pytest.mark.parametrize("batch", [6, 1500], ids=["few", "many"])
def test_step_slots_outside_answer_zero(batch, cuda):
    x, _, _ = _inputs(33, (batch,), 1, 1, (1, 1, 1), 64, 64, torch.float32, state=False)
    state = torch.randn(batch, 1, 64, 64, generator=torch.Generator().manual_seed(34)).cuda()
    before, at = state.clone(), torch.arange(batch, device=cuda)
    at[1::3], at[2::3] = -1, batch + 7
    o = delta.delta_step(*(t.cuda() for t in x.values()), state, slots=at)
    assert not o[1::3].any() and not o[2::3].any() and o[0].any()
    assert torch.equal(state[1::3], before[1::3]) and torch.equal(state[2::3], before[2::3]) and not torch.equal(state[0], before[0])
    memory.sync()


def test_step_is_a_tick_of_attention(cuda):
    x, _, _ = _inputs(35, (4, 20), 4, 4, (2, 2, 4), 64, 64, torch.float32)
    c = {n: t.cuda() for n, t in x.items()}
    o, end = delta.delta_attention(*c.values())
    state, out = c["state"].clone(), []
    for t in range(20):
        out.append(delta.delta_step(*(c[n][:, t] for n in NAMES[:5]), state))
    _near(torch.stack(out, 1), o, 1e-5, "o")
    _near(state, end, 1e-5, "state")


def test_step_of_unaligned_states_and_captured(cuda):
    x, _, _ = _inputs(36, (3,), 1, 2, (2, 2, 2), 32, 32, torch.bfloat16, state=False)
    c = [t.cuda() for t in x.values()]
    room = torch.randn(3 * 2 * 32 * 32 + 1, generator=torch.Generator().manual_seed(37)).cuda()
    odd = room[1:].view(3, 2, 32, 32)
    even, first = odd.clone(), odd.clone()
    o = delta.delta_step(*c, odd)
    version = even._version
    assert torch.allclose(o.float(), delta.delta_step(*c, even).float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    assert even._version > version
    _near(odd, even, 1e-6, "state")
    even.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = delta.delta_step(*c, even)
    even.copy_(first)
    graph.replay()
    _near(even, odd, 1e-6, "state")
    assert torch.allclose(out.float(), o.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    with pytest.raises(FlyguyError, match="no gradient"):
        delta.delta_step(c[0].requires_grad_(), *c[1:], even)


# ---- refusals --------------------------------------------------------------------------------------------------------

def test_refusals(cuda):
    x, _, _ = _inputs(40, (2, 8), 2, 4, (4, 2, 2), 16, 24, torch.float32)
    ok = {n: t.cuda() for n, t in x.items()}
    bad = [("q", ok["q"].double(), "float32, bfloat16"), ("q", ok["q"][0, 0], "dimensions"), ("k", ok["k"].half(), "type, device"),
           ("k", ok["k"][..., :8], "must be"), ("v", ok["v"][:, :4], "must be"), ("q", ok["q"][:, :, :3], "cannot share"),
           ("log_decay", ok["log_decay"].double(), "float32 tensor"), ("beta", ok["beta"][:, :, :2], "beta must be"),
           ("beta", ok["beta"][:, :7], "beta must be"), ("state", ok["state"][:1], "state must be"), ("state", ok["state"].half(), "state must be"),
           ("log_decay", 0.1, "float32 tensor")]
    for n, t, words in bad:
        with pytest.raises(FlyguyError, match=words):
            delta.delta_attention(*(ok | {n: t}).values())
    with pytest.raises(FlyguyError, match="packed"):
        delta.delta_attention(*ok.values(), offsets=torch.tensor([0, 8], device=cuda))
    with pytest.raises(FlyguyError, match="int64 vector"):
        delta.delta_attention(*(ok[n][0] for n in NAMES[:5]), offsets=torch.tensor([0, 8], dtype=torch.int32, device=cuda))
    wide = torch.zeros(1, 2, 1, 129, device=cuda)
    gate = torch.zeros(1, 2, 1, device=cuda)
    with pytest.raises(FlyguyError, match="dim must be 1 to 128"):
        delta.delta_attention(wide, wide, wide, gate, gate)
    wide = torch.zeros(1, 2, 1, 257, device=cuda)
    with pytest.raises(FlyguyError, match="value_dim 1 to 256"):
        delta.delta_attention(wide[..., :64], wide[..., :64], wide, gate, gate)
    tick = {n: (t if n == "state" else t[:, 0]) for n, t in ok.items()}
    for n, t, words in (("state", tick["state"].transpose(2, 3), "contiguous float32"), ("k", tick["k"][:1], "must be"),
                        ("beta", tick["beta"][:1], "beta must be"), ("state", tick["state"][:1], "need as many")):
        with pytest.raises(FlyguyError, match=words):
            delta.delta_step(*(tick | {n: t}).values())
    with pytest.raises(FlyguyError, match="slots"):
        delta.delta_step(*tick.values(), slots=torch.zeros(3, dtype=torch.int64, device=cuda))
    assert np.isfinite(delta.delta_step(*tick.values()).cpu().numpy()).all()


def test_heads_of_no_values_are_refused(cuda):
    for dim, value_dim in ((0, 4), (4, 0)):
        q, v, gate = torch.zeros(2, 1, dim, device=cuda), torch.zeros(2, 1, value_dim, device=cuda), torch.zeros(2, 1, device=cuda)
        with pytest.raises(FlyguyError, match="dim"):
            delta.delta_step(q, q, v, gate, gate, torch.zeros(2, 1, dim, value_dim, device=cuda))
        with pytest.raises(FlyguyError, match="dim"):
            delta.delta_attention(q, q, v, gate, gate, offsets=torch.tensor([0, 2], device=cuda))


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("sizes", [(2, 100, 2, (1, 2, 1), 40, 72), (1, 2304, 2, (2, 1, 1), 72, 20), (2, 64, 1, (1, 1, 1), 128, 128)], ids=["chunks", "parts", "wide"])
def test_what_is_held_and_what_is_made_again_give_the_same_gradients(sizes, typ, monkeypatch, cuda):
    """The way back over what the forward held (twice), and over what it makes itself, its workspace full of NaN first."""
    B, T, H, heads, D, E = sizes
    x, go, gs = _inputs(50, (B, T), B, H, heads, D, E, typ)
    leaves = [t.cuda().requires_grad_() for t in x.values()]
    out = delta.delta_attention(*leaves)
    want = torch.autograd.grad(out, leaves, (go.cuda(), gs.cuda()), retain_graph=True)
    twice = torch.autograd.grad(out, leaves, (go.cuda(), gs.cuda()))
    monkeypatch.setattr(delta, "HELD_AT_MOST", 0)

    def room(size, device):
        t = torch.full((-(-size // 4),), math.nan, device=device)
        return t, (t.data_ptr(), size)

    monkeypatch.setattr(delta, "_room", room)
    again = torch.autograd.grad(delta.delta_attention(*leaves), leaves, (go.cuda(), gs.cuda()))
    for a, b, c in zip(want, twice, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_packed_recordings_made_again(monkeypatch, cuda):
    x, go, gs = _inputs(51, (300,), 4, 4, (4, 2, 2), 64, 64, torch.bfloat16)
    offsets = torch.tensor([3, 3, 100, 131, 290], device=cuda)
    want = _run(x, go, gs, None, offsets)
    monkeypatch.setattr(delta, "HELD_AT_MOST", 0)
    got = _run(x, go, gs, None, offsets)
    assert torch.equal(got[1], want[1]) and all(torch.equal(got[2][n], want[2][n]) for n in got[2])


def test_the_states_that_come_out_may_be_played_on_before_the_backward(cuda):
    """delta_step changes them in place; the backward has its own."""
    x, go, _ = _inputs(52, (2, 70), 2, 2, (2, 2, 2), 64, 64, torch.float32)
    leaves = [t.cuda().requires_grad_() for t in x.values()]
    want = torch.autograd.grad(delta.delta_attention(*leaves)[0], leaves, go.cuda())
    o, end = delta.delta_attention(*leaves)
    with torch.no_grad():
        delta.delta_step(*(t[:, -1] for t in leaves[:5]), end)
    for a, b in zip(torch.autograd.grad(o, leaves, go.cuda()), want):
        assert torch.equal(a, b)
