"""A memory over ticks beside a fly network, learned on whole recordings and played a tick at a time.

  python -m flyguy_b200.remember [--steps 200] [--recordings 64] [--ticks 128] [--ago 12] [--lr 3e-3] [--cars 8]
                                 [--rule decay|delta] [--dropout 0]

A made-up game that no actor without a memory can play: each tick's observation shows an action, and the right answer is
the one shown `ago` ticks earlier. The fly network (a small synthetic one, its weights left alone) answers from the tick's
observation; flyguy_b200.memory.TickMemory (or flyguy_b200.delta.DeltaMemory: --rule delta) adds what it remembers. Learning
is distillation as elsewhere in this package: the library's KL loss of the sum against the teacher's logits gives the
gradient, here of a batch of whole recordings. Then `cars` cars play a recording tick by tick with the same weights."""
from __future__ import annotations

import argparse

import torch

from . import native, synth
from .delta import DeltaMemory
from .memory import TickMemory


def recordings(n: int, ticks: int, ago: int, obs_dim: int, n_act: int, generator, device):
    """Observations [n, ticks, obs_dim], the right answers [n, ticks] (of the first `ago` ticks: action 0)."""
    shown = torch.randint(0, n_act, (n, ticks), generator=generator).to(device)
    obs = 0.1 * torch.randn(n, ticks, obs_dim, generator=generator).to(device)
    obs.scatter_add_(2, shown.unsqueeze(-1), torch.ones(n, ticks, 1, device=device))
    right = torch.zeros_like(shown)
    right[:, ago:] = shown[:, :ticks - ago]
    return obs, right


class Game:
    """The fly network and the memory beside it."""

    def __init__(self, seed: int = 0, max_batch: int = 8192, n_act: int = 16, device: str = "cuda", rule: str = "decay",
                 dropout: float = 0.0):
        s, params = synth.make_synthetic(sizes=(300, 700, 500, 60), total_edges=30_000, seed=seed)
        self.device = torch.device(device)
        torch.manual_seed(seed)
        self.fly = native.Handle(s, max_batch, native.FG_INFER_ONLY)
        self.fly.set_params(params)
        self.obs_dim, self.all_actions, self.n_act = s["obs_dim"], s["n_act"], n_act
        if rule == "delta":
            self.memory = DeltaMemory(self.obs_dim, self.all_actions, ticks=(8.0, 256.0), dropout=dropout, seed=seed)
        else:
            self.memory = TickMemory(self.obs_dim, self.all_actions, ticks=(8.0, 256.0))
        self.memory.to(self.device)

    def fly_logits(self, obs: torch.Tensor) -> torch.Tensor:
        """The fly network's logits [.., n_act] of observations [.., obs_dim] (in batches of a multiple of 32)."""
        flat = obs.flatten(0, -2)
        pad = -len(flat) % 32
        return self.fly.forward(torch.nn.functional.pad(flat, (0, 0, 0, pad)))[:len(flat)].unflatten(0, obs.shape[:-1])

    def learn(self, steps: int, n: int, ticks: int, ago: int, lr: float, seed: int = 1, log=None) -> list[tuple[float, float]]:
        """`steps` steps of Adam on fresh recordings; (KL a tick, share of right answers) of each step."""
        g = torch.Generator().manual_seed(seed)
        opt = torch.optim.Adam(self.memory.parameters(), lr=lr)
        stats, told = torch.zeros(2, device=self.device), []
        for step in range(steps):
            obs, right = recordings(n, ticks, ago, self.obs_dim, self.n_act, g, self.device)
            teacher = 12.0 * torch.nn.functional.one_hot(right, self.all_actions).float().flatten(0, 1)
            logits = (self.fly_logits(obs) + self.memory(obs)[0]).flatten(0, 1)
            dlogits = torch.empty_like(logits)
            native.kl_loss_noalloc(logits.detach(), teacher, 1.0, dlogits, stats)
            opt.zero_grad()
            logits.backward(dlogits)
            opt.step()
            kl, agree = (stats / len(logits)).tolist()
            told.append((kl, agree))
            if log and (step % 20 == 0 or step + 1 == steps):
                log(f"step {step}: kl {kl:.4f} agree {agree:.3f}")
        return told

    @torch.no_grad()
    def play(self, obs: torch.Tensor) -> torch.Tensor:
        """Logits [cars, ticks, n_act] of recordings played a tick at a time."""
        state, out = self.memory.states(len(obs)), []
        for t in range(obs.shape[1]):
            at = torch.full((len(obs),), t, device=self.device)
            out.append(self.fly_logits(obs[:, t]) + self.memory.step(obs[:, t], state, at))
        return torch.stack(out, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--recordings", type=int, default=64)
    ap.add_argument("--ticks", type=int, default=128)
    ap.add_argument("--ago", type=int, default=12)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--cars", type=int, default=8)
    ap.add_argument("--rule", choices=("decay", "delta"), default="decay")
    ap.add_argument("--dropout", type=float, default=0.0, help="of the delta rule's outputs, while learning")
    a = ap.parse_args()
    if a.dropout and a.rule != "delta":
        ap.error("--dropout goes with --rule delta")
    game = Game(max_batch=-(-max(a.recordings * a.ticks, a.cars) // 32) * 32, rule=a.rule, dropout=a.dropout)
    game.learn(a.steps, a.recordings, a.ticks, a.ago, a.lr, log=print)
    obs, right = recordings(a.cars, a.ticks, a.ago, game.obs_dim, game.n_act, torch.Generator().manual_seed(99), game.device)
    game.memory.eval()
    played = game.play(obs)
    with torch.no_grad():
        whole = game.fly_logits(obs) + game.memory(obs)[0]
    agree = (played.argmax(-1) == right)[:, a.ago:].float().mean().item()
    print(f"played {a.cars} cars tick by tick: {agree:.3f} right; logits within "
          f"{((played - whole).norm() / whole.norm()).item():.1e} of the whole recordings'")


if __name__ == "__main__":
    main()
