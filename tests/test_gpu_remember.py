"""The memory operators together: TickMemory beside a fly network, learned on recordings, played tick by tick."""
import pytest
import torch

from flyguy_b200 import memory, remember
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def game(cuda):
    return remember.Game(seed=0, max_batch=4096)


def test_a_fresh_memory_changes_nothing(game, cuda):
    obs, _ = remember.recordings(2, 48, 5, game.obs_dim, game.n_act, torch.Generator().manual_seed(3), cuda)
    logits, _ = memory.TickMemory(game.obs_dim, game.all_actions).cuda()(obs)
    assert not logits.any()


def test_it_learns_what_only_a_memory_can_know(game, cuda):
    """The answer is what was shown 6 ticks before: chance is 1 in 16; the KL falls by more than half in 150 steps."""
    told = game.learn(150, 32, 96, 6, 3e-3)
    assert told[-1][0] < 0.5 * told[0][0], (told[0], told[-1])
    assert told[-1][1] > 0.5, told[-1]


def test_played_tick_by_tick_it_answers_as_on_the_whole_recording(game, cuda):
    """bf16 queries, keys, values and outputs: each rounded at 2^-9 on either way, the sequence form's weights and states
    too; 2^-6 of the logits' norm."""
    obs, _ = remember.recordings(8, 150, 6, game.obs_dim, game.n_act, torch.Generator().manual_seed(4), cuda)
    with torch.no_grad():
        torch.nn.init.normal_(game.memory.out.weight, std=0.05)
        whole = game.memory(obs)[0]
        state = game.memory.states(8)
        each = torch.stack([game.memory.step(obs[:, t], state, torch.full((8,), t, device=cuda)) for t in range(150)], 1)
    assert (each - whole).norm() <= 2 ** -6 * whole.norm()


def test_packed_recordings_equal_padded_ones(game, cuda):
    """Recordings of 70 and 30 ticks end to end; positions run on, the answers depend on their differences only (the turned
    queries and keys are rounded at other angles: 2^-6)."""
    obs, _ = remember.recordings(2, 70, 6, game.obs_dim, game.n_act, torch.Generator().manual_seed(5), cuda)
    packed = torch.cat((obs[0], obs[1, :30]))
    with torch.no_grad():
        both, end = game.memory(packed, offsets=torch.tensor([0, 70, 100], device=cuda))
        one, _ = game.memory(obs)
    want = torch.cat((one[0], one[1, :30]))
    assert (both - want).norm() <= 2 ** -6 * want.norm()
    assert end.shape == (2, 8, 64, 64)


def test_a_state_needs_positions(game, cuda):
    obs = torch.zeros(2, 4, game.obs_dim, device=cuda)
    with pytest.raises(FlyguyError, match="positions"):
        game.memory(obs, game.memory.states(2))
    with pytest.raises(FlyguyError, match="share"):
        memory.TickMemory(8, 4, heads=3, key_heads=2)
