"""DeltaMemory in use that test_gpu_delta_memory.py does not make: weights far from their first values, forwards run again."""
import pytest
import torch

from flyguy_b200 import delta, memory

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
