"""How many terms the delta rule's products have: results and gradients against the definition in float64, close enough that a term less
in any of them shows (test_gpu_delta.py holds shapes, layouts and masks to wider limits).

  o, gq, gk, gv of 16 bits   against the definition's values rounded once. Two terms leave at most 2^-17 of a product; four such in a row,
             independent, 2^-16 of the value. A value that is off by d falls on the other side of a rounding to steps of s in d / s
             of all cases and is then off by s, d s in the mean square: with s at most finfo.eps of the value sqrt(2^-16 eps) of
             the norm, 3.5e-4 for bfloat16 and 1.2e-4 for float16. (A term less leaves 2^-9: 1.5e-3 to 2.5e-3, and 3e-4.)
  states, gates' gradients, and all of float32   three terms leave 2^-25 in the mean, sums of up to 128 products in float32 0.3 sqrt(128)
             2^-24 = 2e-7, twice that where the tensor cores cut off instead of rounding; five such in a row 1e-6, of which 1.5e-6 is
             the limit. (Two terms leave 4e-6 to 1e-5.)"""
import pytest
import torch

from flyguy_b200 import delta

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda t: str(t).replace("torch.", "")   # noqa: E731


def _inputs(typ, B, T, H, heads, D, E):
    g = torch.Generator().manual_seed(T)
    rand = lambda *s: torch.randn(*s, generator=g)               # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)            # noqa: E731
    return [unit(rand(B, T, heads[0], D) + 0.4).to(typ), unit(rand(B, T, heads[1], D) + 0.4).to(typ), (0.5 * rand(B, T, heads[2], E)).to(typ),
            -0.05 * torch.rand(B, T, H, generator=g) ** 2, torch.sigmoid(rand(B, T, H)), 0.3 * rand(B, H, D, E)], \
        (rand(B, T, H, E).to(typ), 0.05 * rand(B, H, D, E))


def _definition(q, k, v, log_decay, beta, S):
    H = log_decay.shape[-1]
    q, k, v = (t.repeat_interleave(H // t.shape[2], 2) for t in (q, k, v))
    out = []
    for t in range(q.shape[1]):
        S = S * log_decay[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhd,bhde->bhe", k[:, t], S))
        S = S + k[:, t].unsqueeze(-1) * u.unsqueeze(-2)
        out.append(torch.einsum("bhd,bhde->bhe", q[:, t], S) * q.shape[-1] ** -0.5)
    return torch.stack(out, 1), S


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("sizes", [(3, 300, 2, (2, 2, 2), 128, 128), (2, 257, 4, (4, 1, 1), 64, 64), (3, 200, 4, (2, 2, 4), 64, 37), (2, 130, 3, (1, 3, 3), 96, 200)],
                         ids=["128", "shared", "as in a memory", "wide values"])
def test_every_product_has_its_terms(sizes, typ, cuda):
    ins, grads = _inputs(typ, *sizes)
    leaves = [t.double().to(cuda).requires_grad_() for t in ins]
    outs = _definition(*leaves)
    want = *outs, *torch.autograd.grad(outs, leaves, [g.double().to(cuda) for g in grads])
    leaves = [t.to(cuda).requires_grad_() for t in ins]
    outs = delta.delta_attention(*leaves)
    got = *outs, *torch.autograd.grad(outs, leaves, [g.to(cuda) for g in grads])
    with torch.no_grad():
        alone = delta.delta_attention(*leaves)
    assert torch.equal(alone[1], outs[1])
    off = {}
    for n, x, y in zip(("o", "end", "q", "k", "v", "log_decay", "beta", "state", "o alone"), (*got, alone[0]), (*want, want[0])):
        limit = 1.5e-6 if x.dtype is torch.float32 else (2.0 ** -16 * torch.finfo(typ).eps) ** 0.5
        off[n] = ((x.double() - y.to(x.dtype).double()).norm() / y.norm()).item() / limit
    assert all(x <= 1 for x in off.values()), off
