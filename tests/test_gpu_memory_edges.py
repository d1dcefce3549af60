"""The memory-over-ticks operators (flyguy_b200.memory) at their edges: what a caller may pass that the operators' own cases do
not reach. Tolerances as in test_gpu_memory.py: 2^-8 of the norm for bfloat16, 5e-6 for float32."""
import numpy as np
import pytest
import torch

from flyguy_b200 import memory
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 5e-6, torch.bfloat16: 4e-3, torch.float16: 5e-4}


def _rand(g, *shape, typ=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(typ).cuda()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _off(got, want):
    """||got - want|| / ||want||"""
    return ((got.double() - want).norm() / want.norm().clamp(min=1e-30)).item()


def _turn64(x, turns, positions, layout="half", sign=1):
    """x [B, T, H, D] in float64, its first pairs turned."""
    n = len(turns)
    part = (positions.unsqueeze(-1) * turns) >> 32
    unit = torch.polar(torch.ones_like(part, dtype=torch.float64), sign * part.double() * (2 * np.pi / 2.0 ** 32)).unsqueeze(2)
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    z = torch.complex(a, b) * unit
    y = x.clone()
    if layout == "half":
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = z.real, z.imag
    return y


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", [(1, 20011, 1, 128), (3, 7001, 2, 256), (1, 16384, 5, 64)])
def test_heads_of_ticks_that_a_block_takes_in_turn(shape, layout, typ, cuda):
    """Few heads and many ticks: a block goes from one set of ticks to the next with copies of the set before still asked for.
    Every head of every tick, the last ones of a set and the first of the next among them."""
    B, T, H, D = shape
    g = _gen(1)
    x, gy = _rand(g, B, T, H, D, typ=typ), _rand(g, B, T, H, D, typ=typ)
    w = (1 + 0.2 * _rand(g, H, D)).requires_grad_()
    turns = memory.rotary_turns(D, device="cuda")
    positions = torch.arange(T, device="cuda").expand(B, T)
    q = x.clone().requires_grad_()
    y, _ = memory.norm_rotate(q, x[:, :, :0], turns, w, None, positions, layout, eps=1e-3)
    y.backward(gy)
    x64 = x.double()
    r = (x64.square().mean(-1, keepdim=True) + 1e-3).rsqrt()
    back = _turn64(gy.double(), turns, positions, layout, -1)
    gw = back * w.detach().double()
    want = _turn64(x64 * r * w.detach().double(), turns, positions, layout)
    want_x = r * (gw - x64 * r * (gw * x64 * r).mean(-1, keepdim=True))
    for got, ref in ((y, want), (q.grad, want_x)):
        rows = (got.double() - ref).norm(dim=-1) / ref.norm(dim=-1)
        assert rows.max().item() <= 2 * TOL[typ]
    assert _off(w.grad, (back * x64 * r).sum((0, 1))) <= TOL[torch.float32]


@pytest.mark.parametrize("each_of", ["keys", "queries"])
@pytest.mark.parametrize("other", ["none", "frozen", "frozen each"])
@pytest.mark.parametrize("size", [(2, 8, 16, 4, 128), (3, 300, 2, 8, 64), (4, 200, 8, 2, 96)])
def test_weights_of_each_head_beside_weights_that_do_not_learn(size, other, each_of, cuda, monkeypatch):
    """One side learns a weight for each head, the other has none, or one that is held: the gradients, and not a byte behind
    the workspace."""
    B, T, H, K, D = size
    guard, rooms = 1 << 22, []

    def room(n, device):
        if not n:
            return None, (0, 0)
        t = torch.full((n + guard,), 0xa5, dtype=torch.uint8, device=device)
        rooms.append((t, n))
        return t, (t.data_ptr(), n)

    monkeypatch.setattr(memory, "_room", room)
    g = _gen(2)
    ins = [_rand(g, B, T, h, D, typ=torch.bfloat16).requires_grad_() for h in (H, K)]
    outs = [_rand(g, B, T, h, D, typ=torch.bfloat16) for h in (H, K)]
    learns = 1 if each_of == "keys" else 0
    w = [None, None]
    w[learns] = (1 + 0.2 * _rand(g, (H, K)[learns], D)).requires_grad_()
    if other != "none":
        w[1 - learns] = 1 + 0.2 * _rand(g, *(((H, K)[1 - learns], D) if other == "frozen each" else (D,)))
    turns = memory.rotary_turns(D, device="cuda")
    y = memory.norm_rotate(*ins, turns, *w, eps=1e-3)
    got = torch.autograd.grad(y, [*ins, w[learns]], outs)
    positions = torch.arange(T, device="cuda").expand(B, T)
    for i in range(2):
        x, w64 = ins[i].detach().double(), 1.0 if w[i] is None else w[i].detach().double()
        r = (x.square().mean(-1, keepdim=True) + 1e-3).rsqrt()
        back = _turn64(outs[i].double(), turns, positions, sign=-1)
        gw = back * w64
        assert _off(y[i].detach(), _turn64(x * r * w64, turns, positions)) <= TOL[torch.bfloat16]
        assert _off(got[i], r * (gw - x * r * (gw * x * r).mean(-1, keepdim=True))) <= TOL[torch.bfloat16]
        if i == learns:
            assert _off(got[2], (back * x * r).sum((0, 1))) <= TOL[torch.float32]
    assert len(rooms) == 1
    for t, n in rooms:
        assert (t[n:] == 0xa5).all()


def _at_float(t, offset):
    """t's values in a contiguous view that begins `offset` floats after a 16-byte boundary."""
    return torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)[offset:].view(t.shape).copy_(t)


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("dims", [(2, 1, 64, 64), (2, 2, 128, 128), (1, 1, 96, 80)])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_states_that_begin_at_any_float(offset, dims, typ, cuda):
    """States, and gradients of states, cut from a longer buffer: the bits of aligned ones. One recording is long enough to be
    split, so that its parts begin from such a state too."""
    H, K, D, E = dims
    for T in (70, 1500):
        g = _gen(3)
        ins = [_rand(g, 1, T, h, n, typ=typ).requires_grad_() for h, n in ((H, D), (K, D), (K, E))]
        state, go, gend = _rand(g, 1, H, D, E), _rand(g, 1, T, H, E, typ=typ), _rand(g, 1, H, D, E, scale=0.3)
        ld = torch.log1p(-torch.exp2(-4.0 - torch.arange(H, device="cuda")))
        runs = []
        for move in (lambda t: t, lambda t: _at_float(t, offset)):
            s = move(state).requires_grad_()
            assert s.data_ptr() % 16 == (0 if not runs else 4 * offset)
            o, end = memory.decay_attention(*ins, ld, s)
            runs.append((o, end, *torch.autograd.grad((o, end), (*ins, s), (go, move(gend)))))
        for a, b in zip(*runs):
            assert torch.equal(a, b)


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16, torch.float16], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dims", [(4, 2, 64, 64), (2, 2, 128, 128), (3, 1, 20, 7), (2, 1, 200, 130)])
@pytest.mark.parametrize("offsets", [[40, 170, 170, 300], [0, 130, 260], [7, 400], [400, 400], [0], [0, 0]])
def test_ticks_of_no_recording_are_zero(offsets, dims, typ, cuda):
    """A packed buffer of 400 ticks with room before and behind its recordings, NaN in what is there: zeros in the output and in
    the gradients, and the recordings' own as if packed without it. (What was in the outputs' memory before is made NaN, too.)"""
    H, K, D, E = dims
    n, N = 400, len(offsets) - 1
    g = _gen(4)
    ins = [_rand(g, n, h, d, typ=typ) for h, d in ((H, D), (K, D), (K, E))]
    state, go, gend = _rand(g, N, H, D, E), _rand(g, n, H, E, typ=typ), _rand(g, N, H, D, E, scale=0.3)
    a, z = offsets[0], offsets[-1]
    for t in (*ins, go):
        t[:a] = t[z:] = float("nan")
    ld = torch.log1p(-torch.exp2(-4.0 - torch.arange(H, device="cuda")))

    def run(parts, off):
        torch.full((1 << 24,), float("nan"), device="cuda")                 # (freed at once: what the outputs may be made from)
        leaves = [t.clone().requires_grad_() for t in (*parts[:3], state)]
        o, end = memory.decay_attention(*leaves[:3], ld, leaves[3], offsets=torch.tensor(off, device="cuda"))
        return (o, end), torch.autograd.grad((o, end), leaves, (parts[3], gend))

    (o, end), grads = run((*ins, go), offsets)
    (o1, end1), grads1 = run([t[a:z] for t in (*ins, go)], [x - a for x in offsets])
    for got, want in ((o, o1), *zip(grads[:3], grads1[:3])):
        assert torch.equal(got[a:z], want) and not got[:a].any() and not got[z:].any()
    assert torch.equal(end, end1) and torch.equal(grads[3], grads1[3])


@pytest.mark.parametrize("offsets", [[0, 70, 70, 100], [5, 30, 96]])
def test_states_of_packed_recordings_go_on_tick_by_tick(offsets, cuda):
    """What a packed forward hands on is what playing the same recordings one by one hands on, and a step from it answers alike: a
    tick's position is its place in its own recording. fp32: the same products in another order (1e-5 of the norm)."""
    torch.manual_seed(0)
    m = memory.TickMemory(24, 6, heads=4, key_heads=2, dim=64, dtype=torch.float32).cuda()
    torch.nn.init.normal_(m.out.weight, std=0.1)
    obs, then = torch.randn(offsets[-1] + 3, 24, device="cuda"), torch.randn(len(offsets) - 1, 24, device="cuda")
    with torch.no_grad():
        _, end = m(obs, offsets=torch.tensor(offsets, device="cuda"))
        states = m.states(len(offsets) - 1)
        for i, (a, z) in enumerate(zip(offsets, offsets[1:])):
            for t in range(z - a):
                m.step(obs[a + t].unsqueeze(0), states[i:i + 1], torch.full((1,), t, device="cuda"))
        assert _off(end, states.double()) <= 1e-5
        ticks = torch.tensor([z - a for a, z in zip(offsets, offsets[1:])], device="cuda")
        want = m.step(then, states, ticks)
        assert _off(m.step(then, end, ticks), want.double()) <= 1e-5


def test_offsets_of_a_memory_are_checked(cuda):
    m, obs = memory.TickMemory(8, 4, heads=2, key_heads=1, dim=16).cuda(), torch.zeros(6, 8, device=cuda)
    for offsets in ([0, 6], torch.tensor([0, 6]), torch.tensor([0.0, 6.0], device=cuda), torch.zeros(0, dtype=torch.int64, device=cuda)):
        with pytest.raises(FlyguyError, match="offsets"):
            m(obs, offsets=offsets)


def _operators(cuda, typ=torch.bfloat16):
    """name: (the tensors that a call reads beside its leaves, leaves, the call)"""
    g = _gen(5)
    x, k, wk = (_rand(g, 60, h, 64, typ=typ).requires_grad_() for h in (4, 2, 2))
    w = (1 + 0.2 * _rand(g, 64)).requires_grad_()
    turns, positions = memory.rotary_turns(64, device=cuda), torch.arange(60, device=cuda) + 7
    ld, offsets = torch.tensor([-0.3, -0.1, -0.02, -0.01], device=cuda), torch.tensor([0, 25, 60], device=cuda)
    state = _rand(g, 2, 4, 64, 64).requires_grad_()
    return {
        "rotate": ([turns, positions], [x], lambda: (memory.rotate(x, turns, positions),)),
        "norm_rotate": ([turns, positions], [x, k, w], lambda: memory.norm_rotate(x, k, turns, w, None, positions)),
        "decay_attention": ([ld, offsets], [x, k, wk, state], lambda: memory.decay_attention(x, k, wk, ld, state, offsets=offsets)),
    }


@pytest.mark.parametrize("name", ["rotate", "norm_rotate", "decay_attention"])
def test_what_a_backward_reads_is_guarded(name, cuda):
    """Plans, positions, decays and offsets changed in place between forward and backward: an error, as for any saved tensor,
    not gradients of another call; unchanged, or kept elsewhere meanwhile, the same gradients."""
    reads, leaves, call = _operators(cuda)[name]
    want = torch.autograd.grad([y.float().sum() for y in call()], leaves)
    with torch.autograd.graph.save_on_cpu():
        outs = call()
    for a, b in zip(torch.autograd.grad([y.float().sum() for y in outs], leaves), want):
        assert torch.equal(a, b)
    for t in reads:
        outs = call()
        t += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad([y.float().sum() for y in outs], leaves)
        t -= 1


def test_a_state_that_a_backward_needs_is_not_stepped_over_unseen(cuda):
    """decay_step changes its states in place: a backward that kept them says so."""
    g = _gen(6)
    q = _rand(g, 2, 9, 2, 64).requires_grad_()
    state, ld = _rand(g, 2, 2, 64, 64), torch.tensor([-0.1, -0.01], device=cuda)
    o, _ = memory.decay_attention(q, q, q, ld, state)
    x = q.detach()[:, 0]
    before = state._version
    memory.decay_step(x, x, x, ld, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


@pytest.mark.parametrize("name", ["rotate", "norm_rotate", "decay_attention"])
def test_gradients_are_not_taken_for_constants(name, cuda):
    """With create_graph the first gradients are the same; a penalty on them is refused, not lost."""
    _, leaves, call = _operators(cuda, torch.float32)[name]
    want = torch.autograd.grad([y.square().sum() for y in call()], leaves)
    got = torch.autograd.grad([y.square().sum() for y in call()], leaves, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.requires_grad
        with pytest.raises(FlyguyError, match="again"):
            torch.autograd.grad(a.square().sum(), leaves, allow_unused=True, retain_graph=True)
    flat = torch.autograd.grad([y.sum() for y in call()], leaves, create_graph=True)
    if name == "rotate":                                                    # linear: these are constants
        assert not flat[0].requires_grad
    else:
        with pytest.raises(FlyguyError, match="again"):
            flat[0].square().sum().backward()
    torch.autograd.backward([y.square().sum() for y in call()], create_graph=True)
    for t, b in zip(leaves, want):
        assert torch.equal(t.grad, b)
        t.grad = None


def test_tangents_are_not_dropped(cuda):
    """Forward-mode derivatives of any operand are refused, with gradients on or off; tensors without one go as ever."""
    from torch.autograd import forward_ad
    g = _gen(7)
    x, w, state = _rand(g, 2, 5, 2, 64), 1 + _rand(g, 64), _rand(g, 2, 2, 64, 64)
    turns, ld = memory.rotary_turns(64, device=cuda), torch.tensor([-0.1, -0.01], device=cuda)
    y, s = x[:, 0].contiguous(), state.clone()
    calls = [(lambda x: memory.rotate(x, turns), (x,)), (lambda q, k, w: memory.norm_rotate(q, k, turns, w, w), (x, x, w)),
             (lambda q, k, v, s: memory.decay_attention(q, k, v, ld, s), (x, x, x, state)),
             (lambda q, k, v, s: memory.decay_step(q, k, v, ld, s), (y, y, y, s))]
    for fn, args in calls:
        for i in range(len(args)):
            for on in (True, False):
                with forward_ad.dual_level(), torch.set_grad_enabled(on):
                    fn(*args)
                    dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                    with pytest.raises(FlyguyError, match="forward-mode"):
                        fn(*dual)


def test_decays_that_are_no_tensor_are_refused(cuda):
    x, state = torch.zeros(1, 2, 2, 64, device=cuda), torch.zeros(2, 2, 64, 64, device=cuda)
    for ld in ([-0.1, -0.1], -0.1, None):
        with pytest.raises(FlyguyError, match="log_decay"):
            memory.decay_attention(x, x, x, ld)
        with pytest.raises(FlyguyError, match="log_decay"):
            memory.decay_step(x[:, 0], x[:, 0], x[:, 0], ld, state)


def test_two_threads_with_tiles_of_different_sizes(cuda):
    """Backward calls from several threads at once (autograd itself makes them from one), one with much more shared memory than
    the other: neither's launch is refused, and the results are each thread's own."""
    import threading
    turns, wrong = memory.rotary_turns(128, device=cuda), []

    def work(heads, seed):
        g = _gen(seed)
        x, w = _rand(g, 4, 8, heads, 128, typ=torch.bfloat16), torch.ones(heads, 128, device=cuda)
        try:
            call = memory._Rotation(x, x[:, :, :0], turns, None, "half", 1.0, 1e-6)
            runs = [call.backward(x, x[:, :, :0], x, x[:, :, :0], w, None, (True, False)) for _ in range(1500)]
            assert all(torch.equal(runs[0][i], runs[-1][i]) for i in (0, 2))
        except Exception as e:                                              # noqa: BLE001  (told by the test's own thread)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in ((1, 8), (120, 9), (1, 10), (64, 11))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("shape", [(2, 5, 3, 0), (2, 5, 0, 3), (0, 5, 2, 2), (2, 0, 2, 2), (1, 1, 0, 0)])
def test_weights_that_nothing_used_have_zero_gradients(shape, cuda):
    """No heads on a side, no recordings or no ticks: a weight's gradient is zeros, not what its memory held."""
    B, T, H, K = shape
    g = _gen(10)
    q, k = _rand(g, B, T, H, 64), _rand(g, B, T, K, 64)
    wq, wk = (1 + 0.2 * _rand(g, 64) for _ in range(2))
    for t in (q, k, wq, wk):
        t.requires_grad_()
    y = memory.norm_rotate(q, k, memory.rotary_turns(64, device=cuda), wq, wk)
    for n in range(8):
        torch.full((64 << n,), float("nan"), device=cuda)                   # (freed at once: what the gradients may be made from)
    got = torch.autograd.grad(y, (q, k, wq, wk), [torch.ones_like(t) for t in y])
    for heads, t in ((H, got[2]), (K, got[3])):
        if not (B and T and heads):
            assert not t.any()
        else:
            assert t.isfinite().all() and t.any()


def test_sync_after_calls_that_went_well(cuda):
    x = _rand(_gen(11), 2, 300, 2, 64, typ=torch.bfloat16)
    o, _ = memory.decay_attention(x, x, x, torch.tensor([-0.1, -0.01], device=cuda))
    memory.sync()
    memory.sync(cuda)
    assert torch.cuda.current_stream().query() and o.isfinite().all()


@pytest.mark.parametrize("dims", [(2, 1, 64, 64), (2, 2, 128, 128)])
def test_the_library_takes_states_at_any_float(dims, cuda):
    """The same below memory's own copy: the kernel that reads such states value by value."""
    H, K, D, E = dims
    g = _gen(12)
    q, k, v = (_rand(g, 1, 300, h, n, typ=torch.bfloat16) for h, n in ((H, D), (K, D), (K, E)))
    state, go, gend = _rand(g, 1, H, D, E), _rand(g, 1, 300, H, E, typ=torch.bfloat16), _rand(g, 1, H, D, E, scale=0.3)
    job = memory._Decay(q, k, v, torch.tensor([-0.1, -0.01], device=cuda), state, None, None)
    runs = []
    for move in (lambda t: t, lambda t: _at_float(t, 1)):
        o, end = job.forward(q, k, v, move(state))
        job_end = move(gend)
        gq, gk, gv, gs = (torch.empty_like(t) for t in (q, k, v, state))
        job.run(memory.lib().fg_decay_attn_bwd, True, (q, k, v, None, go, gq, gk, gv), move(state), None, job_end, gs)
        runs.append((o, end, gq, gk, gv, gs))
    for a, b in zip(*runs):
        assert _off(b, a.double()) <= 2 * TOL[a.dtype]


@pytest.mark.parametrize("D", [64, 7])
def test_only_weights_of_no_heads_learn(D, cuda):
    """No key heads, and nothing but their weights asks for a gradient beside the queries."""
    q, k = _rand(_gen(13), 2, 5, 3, D).requires_grad_(), torch.zeros(2, 5, 0, D, device=cuda)
    wk = torch.ones(D, device=cuda).requires_grad_()
    y, z = memory.norm_rotate(q, k, None, None, wk)
    torch.autograd.backward((y, z), (torch.ones_like(y), torch.ones_like(z)))
    assert not wk.grad.any() and q.grad.isfinite().all()


@pytest.mark.parametrize("name", ["rotate", "norm_rotate", "decay_attention"])
def test_plans_made_in_inference_mode(name, cuda):
    """Positions, plans, decays and offsets from inference mode learn as others do."""
    reads, leaves, call = _operators(cuda)[name]
    want = torch.autograd.grad([y.float().sum() for y in call()], leaves)
    with torch.inference_mode():
        made = [t.clone() for t in reads]
    fns = {"rotate": lambda a, b: (memory.rotate(leaves[0], a, b),),
           "norm_rotate": lambda a, b: memory.norm_rotate(*leaves[:2], a, leaves[2], None, b),
           "decay_attention": lambda a, b: memory.decay_attention(*leaves[:3], a, leaves[3], offsets=b)}
    for a, b in zip(torch.autograd.grad([y.float().sum() for y in fns[name](*made)], leaves), want):
        assert torch.equal(a, b)
