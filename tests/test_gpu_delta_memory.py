"""The delta rule, layer norm and dropout together: DeltaMemory beside a fly network, in learning and in playing tick by tick."""
import sys

import pytest
import torch

from flyguy_b200 import delta, layers, memory, remember
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def game(cuda):
    return remember.Game(seed=0, max_batch=4096, rule="delta", dropout=0.25)


def _obs(game, n, ticks, seed, device):
    return remember.recordings(n, ticks, 5, game.obs_dim, game.n_act, torch.Generator().manual_seed(seed), device)[0]


def test_a_fresh_memory_changes_nothing(game, cuda):
    logits, end = delta.DeltaMemory(game.obs_dim, game.all_actions).cuda()(_obs(game, 2, 48, 1, cuda))
    assert not logits.any() and end.shape == (2, 8, 64, 64) and end.any()


def test_learning_steps_move_every_weight(game, cuda):
    before = {n: p.detach().clone() for n, p in game.memory.named_parameters()}
    told = game.learn(3, 8, 40, 5, 1e-2)
    assert len(told) == 3 and all(torch.isfinite(torch.tensor(t)).all() for t in told)
    for n, p in game.memory.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
    assert game.memory.calls == 3


def test_gradients_are_those_of_the_formulas(game, cuda):
    """A float32 memory against the same steps from elementary operations in float64; 3e-5: each operator's own tolerance is 1e-5."""
    torch.manual_seed(2)
    m = delta.DeltaMemory(20, 12, heads=4, key_heads=2, dim=32, dropout=0.3, seed=9, dtype=torch.float32).cuda()
    torch.nn.init.normal_(m.out.weight, std=0.1)
    torch.nn.init.normal_(m.gates.weight, std=0.3)
    obs, g = torch.randn(2, 37, 20, device=cuda), torch.randn(2, 37, 12, device=cuda)
    logits, _ = m(obs)
    names, params = zip(*m.named_parameters())
    got = torch.autograd.grad(logits, params, g)
    kept = layers.dropout(torch.ones(2, 37, 4, 32, device=cuda), 0.3, 9, call=0).double()

    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}

    def norm(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    x = norm(obs.double(), p["obs_weight"], p["obs_bias"])
    q, k, v = (x @ p["qkv.weight"].T).unflatten(-1, (8, 32)).split((2, 2, 4), -2)
    a, b = (x @ p["gates.weight"].T + p["gates.bias"]).chunk(2, -1)
    angle = torch.arange(37, device=cuda).double()[:, None] * m.turns.double() / 2.0 ** 64 * 2 * torch.pi

    def turn(x, w):
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        c, s, (e, f) = angle.cos()[:, None], angle.sin()[:, None], x.chunk(2, -1)
        return torch.cat((e * c - f * s, f * c + e * s), -1)

    wide = lambda t: t.repeat_interleave(2, 2)                   # noqa: E731
    q, k = wide(turn(q, p["q_weight"])), wide(turn(k, p["k_weight"]))
    fade, beta = (torch.nn.functional.softplus(a) * m.log_decay.double()).exp(), b.sigmoid()
    S, out = torch.zeros(2, 4, 32, 32, dtype=torch.float64, device=cuda), []
    for t in range(37):
        S = S * fade[:, t, :, None, None]
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhd,bhde->bhe", k[:, t], S))
        S = S + k[:, t].unsqueeze(-1) * u.unsqueeze(-2)
        out.append(torch.einsum("bhd,bhde->bhe", q[:, t], S) * 32 ** -0.5)
    o = norm(torch.stack(out, 1), p["o_weight"], p["o_bias"]) * kept
    want_logits = o.flatten(-2) @ p["out.weight"].T
    assert (logits.double() - want_logits).norm() <= 3e-5 * want_logits.norm()
    for n, x, y in zip(names, got, torch.autograd.grad(want_logits, [p[n] for n in names], g.double())):
        assert (x.double() - y).norm() <= 3e-5 * y.norm() + 1e-7, n


def test_played_tick_by_tick_it_answers_as_on_the_whole_recording(game, cuda):
    """bf16 queries, keys, values and outputs: each rounded at 2^-9 on either way, the sequence form's weights and states too, and
    what the norm of a head makes of them: 2^-5 of the logits' norm."""
    game.memory.eval()
    obs = _obs(game, 8, 150, 4, cuda)
    with torch.no_grad():
        torch.nn.init.normal_(game.memory.out.weight, std=0.05)
        whole, end = game.memory(obs)
        state = game.memory.states(8)
        each = torch.stack([game.memory.step(obs[:, t], state, torch.full((8,), t, device=cuda)) for t in range(150)], 1)
    assert (each - whole).norm() <= 2 ** -5 * whole.norm()
    assert (state - end).norm() <= 2 ** -6 * end.norm()
    assert game.play(obs).shape == (8, 150, game.all_actions)


def test_packed_recordings_equal_padded_ones_and_carry_on(game, cuda):
    """The same ticks at the same positions in other chunks: states as good as their terms, outputs at bf16 roundings, 2^-6."""
    game.memory.eval()
    obs = _obs(game, 2, 70, 5, cuda)
    with torch.no_grad():
        packed, end = game.memory(torch.cat((obs[0], obs[1, :30])), offsets=torch.tensor([0, 70, 100], device=cuda))
        one, _ = game.memory(obs)
        _, half = game.memory(obs[:, :41])
        rest, _ = game.memory(obs[:, 41:], half, torch.arange(41, 70, device=cuda))
    want = torch.cat((one[0], one[1, :30]))
    assert (packed - want).norm() <= 2 ** -6 * want.norm()
    assert (rest - one[:, 41:]).norm() <= 2 ** -6 * one.norm()
    with pytest.raises(FlyguyError, match="positions"):
        game.memory(obs, game.memory.states(2))


def test_dropout_is_for_learning_alone(game, cuda):
    m, obs = game.memory, _obs(game, 2, 32, 6, cuda)
    with torch.no_grad():
        m.eval()
        assert torch.equal(m(obs)[0], m(obs)[0])
        m.train()
        at = m.calls
        one, two = m(obs)[0], m(obs)[0]
        m.calls = at
        assert not torch.equal(one, two) and torch.equal(m(obs)[0], one)
    memory.sync()


def test_a_captured_forward_drops_by_a_seed_on_the_device(game, monkeypatch, cuda):
    m, obs = game.memory, _obs(game, 2, 32, 7, cuda)
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with torch.no_grad(), pytest.raises(FlyguyError, match="seed must be"):
            m(obs)
    monkeypatch.setattr(m, "seed", torch.tensor(3, device=cuda))
    graph, side, at = torch.cuda.CUDAGraph(), torch.cuda.Stream(), m.calls
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        m(obs)
        m.calls = at
        with torch.cuda.graph(graph, stream=side):
            got = m(obs)[0]
    torch.cuda.current_stream().wait_stream(side)
    for seed in (3, 4):
        m.seed.fill_(seed)
        graph.replay()
        m.calls = at
        with torch.no_grad():
            assert torch.equal(got, m(obs)[0])
    memory.sync()


def test_dropout_goes_with_the_delta_rule(monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", "remember --dropout 0.1".split())
    with pytest.raises(SystemExit):
        remember.main()
    assert "--rule delta" in capsys.readouterr().err


def test_the_command_runs_with_the_delta_rule(monkeypatch, capsys, cuda):
    monkeypatch.setattr(sys, "argv", "remember --rule delta --dropout 0.1 --steps 2 --recordings 4 --ticks 40 --cars 3".split())
    remember.main()
    said = capsys.readouterr().out
    assert "step 1: kl" in said and "played 3 cars tick by tick" in said
