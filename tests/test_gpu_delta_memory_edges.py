"""DeltaMemory in use that test_gpu_delta_memory.py does not make: weights far from their first values, forwards run again."""
import pytest
import torch

from torch.utils.checkpoint import checkpoint

from flyguy_b200 import delta, memory
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu


def test_states_stay_bounded_whatever_the_keys_weight_has_learned(cuda):
    """Keys 4 times as long as at first, the same observation 3,000 times over, all of it written (beta near 1): a factor of 1 - 16 a
    tick without a bound. With |k| <= 1 a tick adds no more than its value, |S| <= ticks |v|; and played on it is the same."""
    torch.manual_seed(1)
    m = delta.DeltaMemory(24, 6, heads=4, key_heads=2, dim=32, ticks=(64.0, 4096.0)).cuda()
    with torch.no_grad():
        m.k_weight.mul_(4)
        m.gates.bias[4:] = 6.0
        obs = torch.randn(1, 1, 24, device=cuda).expand(2, 3000, 24).contiguous()
        most = m._inputs(obs[:, :1], None)[2].float().norm(dim=-1).max()
        logits, end = m(obs)
        assert torch.isfinite(logits).all() and end.flatten(2).norm(dim=-1).max() <= 3000 * most
        state = end.clone()
        for t in range(3000, 3040):
            m.step(obs[:, 0], state, torch.full((2,), t, device=cuda))
        assert state.flatten(2).norm(dim=-1).max() <= 3040 * most
    memory.sync()


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_forward_run_again_drops_what_it_dropped(reentrant, cuda):
    """Activation checkpointing: with its call the gradients are those without it; without, the second run is refused. Two memories, so
    that a count of forwards is another by then."""
    torch.manual_seed(2)
    two = [delta.DeltaMemory(20, 20, heads=4, key_heads=2, dim=32, dropout=0.4, seed=s).cuda() for s in (3, 4)]
    for m in two:
        torch.nn.init.normal_(m.out.weight, std=0.1)
    obs, g = torch.randn(2, 37, 20, device=cuda, requires_grad=True), torch.randn(2, 37, 20, device=cuda)
    params = [p for m in two for p in m.parameters()]

    def grads(run):
        x = obs
        for m in two:
            x = x + run(m, x)
        return torch.autograd.grad(x, params, g) if not reentrant else (x.backward(g), [p.grad for p in params])[1]

    def again(*args):
        return lambda m, x: checkpoint(lambda y: m(y, None, None, None, *args)[0], x, use_reentrant=reentrant)

    if reentrant:                                                  # (the first run is one without gradients, whose o has its own bits)
        with torch.no_grad():
            between = obs + two[0](obs, call=7)[0]
        between.requires_grad_()
        behind, *of_second = torch.autograd.grad(between + two[1](between, call=7)[0], (between, *two[1].parameters()), g)
        want = [*torch.autograd.grad(obs + two[0](obs, call=7)[0], two[0].parameters(), behind), *of_second]
    else:
        want = grads(lambda m, x: m(x, call=7)[0])
    for a, b in zip(grads(again(7)), want):
        assert torch.equal(a, b)
    assert [m.calls for m in two] == [0, 0]
    with pytest.raises(FlyguyError, match="give it its call"):
        grads(again())
    with torch.no_grad():                                          # (counted as before, and not where the call is given)
        at = [m.calls for m in two]
        one = two[0](obs)[0]
        assert two[0].calls == at[0] + 1 and torch.equal(two[0](obs, call=at[0])[0], one) and two[0].calls == at[0] + 1
        two[0].eval()
        assert torch.equal(two[0](obs, call=1)[0], two[0](obs, call=2)[0])
    memory.sync()
