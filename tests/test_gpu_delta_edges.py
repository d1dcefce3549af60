"""Calls of the delta rule that test_gpu_delta.py does not make: workspaces full of NaN beside rows of odd lengths, states that no
row has."""
import math

import pytest
import torch

from flyguy_b200 import delta, memory

pytestmark = pytest.mark.gpu


def _inputs(seed, lead, recordings, H, heads, D, E, typ):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)               # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp(min=1e-6)   # noqa: E731
    return [unit(rand(*lead, heads[0], D)).to(typ).cuda(), unit(rand(*lead, heads[1], D)).to(typ).cuda(), rand(*lead, heads[2], E).to(typ).cuda(),
            (-0.2 * rand(*lead, H).abs()).cuda(), torch.sigmoid(rand(*lead, H)).cuda(), rand(recordings, H, D, E).cuda()]


def _grads(ins):
    leaves = [t.detach().requires_grad_() for t in ins]
    out = delta.delta_attention(*leaves)
    return [*out, *torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])]


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16, torch.float16], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("sizes", [(2, 70, 2, (1, 1, 2), 40, 37), (1, 130, 2, (2, 2, 2), 72, 20), (1, 33, 1, (1, 1, 1), 16, 1), (2, 65, 2, (2, 2, 2), 64, 200)],
                         ids=lambda s: "x".join(map(str, (*s[:3], *s[4:]))))
def test_rows_of_odd_lengths_beside_workspaces_full_of_nan(sizes, typ, monkeypatch, cuda):
    B, T, H, heads, D, E = sizes
    ins = _inputs(2, (B, T), B, H, heads, D, E, typ)
    want = _grads(ins)

    def room(size, device):
        t = torch.full((-(-size // 4),), math.nan, device=device)
        return t, (t.data_ptr(), size)

    monkeypatch.setattr(delta, "_room", room)
    got = _grads(ins)
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("batch, slots, H, heads, D, E", [(3, 5, 4, (2, 1, 4), 64, 64), (5, 9, 2, (1, 2, 1), 128, 130), (301, 320, 8, (8, 8, 8), 128, 128),
                                                          (600, 640, 2, (2, 2, 2), 60, 256)], ids=["few", "columns", "many", "many wide"])
def test_states_that_no_row_has_stay_bit_by_bit(batch, slots, H, heads, D, E, cuda):
    """Over three ticks of other rows each, NaN among them; and those of the rows all change."""
    g = torch.Generator().manual_seed(3)
    q, k, v, log_decay, beta, _ = _inputs(4, (batch,), 1, H, heads, D, E, torch.bfloat16)
    state = torch.randn(slots, H, D, E, generator=g).cuda()
    for tick in range(3):
        at = torch.randperm(slots, generator=g)[:batch].cuda()
        rest = torch.ones(slots, dtype=torch.bool, device=cuda)
        rest[at] = False
        state[rest.nonzero()[0]] = math.nan
        before = state.clone()
        o = delta.delta_step(q, k, v, log_decay, beta, state, slots=at)
        assert torch.equal(state[rest].view(torch.int32), before[rest].view(torch.int32))
        mine = torch.isfinite(before[at]).flatten(1).all(1)
        assert torch.isfinite(o[mine]).all() and (state[at][mine] != before[at][mine]).flatten(1).any(1).all()
        state.nan_to_num_(0.5)
    memory.sync()
