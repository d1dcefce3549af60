"""Layer norm where a block shares a row, again and again, and other calls that the shapes of test_gpu_layers.py do not make."""
import pytest
import torch

from flyguy_b200 import layers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ, rows, dim", [(torch.bfloat16, 600, 4096), (torch.float16, 600, 8192), (torch.float32, 600, 2048), (torch.float32, 400, 8192),
                                            (torch.bfloat16, 600, 2047), (torch.float32, 600, 5001), (torch.bfloat16, 1200, 9000)],
                         ids=lambda v: str(v).replace("torch.", ""))
def test_rows_of_many_warps_are_the_same_bits_each_time(typ, rows, dim, cuda):
    """Blocks of 9 to 16 warps: all of a row's warps take the same mean, or its values were off by the difference of two."""
    g = torch.Generator().manual_seed(dim)
    x = (torch.randn(rows, dim, generator=g) + 3).to(typ).cuda().requires_grad_()
    w, b = (1 + 0.2 * torch.randn(dim, generator=g)).cuda().requires_grad_(), torch.randn(dim, generator=g).cuda().requires_grad_()
    gy = torch.randn(rows, dim, generator=g).to(typ).cuda()
    first = None
    for _ in range(30):
        y = layers.layer_norm(x, w, b)
        out = y, *torch.autograd.grad(y, (x, w, b), gy)
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(out, first))
    d = x.detach().double()
    h = (d - d.mean(1, keepdim=True)) / (d.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    want = h * w.double() + b.double()
    # (half a step of the type, and 1e-6 of the largest for sums of up to 9,000 values)
    assert ((first[0].double() - want).abs() <= torch.finfo(typ).eps / 2 * want.abs() * 1.001 + 1e-6 * want.abs().max()).all()


def test_one_row_of_a_million_values_learns(cuda):
    """Its sums' workspace is of the row's size, not of as many rows as there are blocks."""
    n = 1 << 20
    x = torch.randn(1, n, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_()
    w, b = torch.ones(n, device=cuda, requires_grad=True), torch.zeros(n, device=cuda, requires_grad=True)
    gy = torch.randn(1, n, generator=torch.Generator().manual_seed(4)).cuda()
    y = layers.layer_norm(x, w, b)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    gw, gb = torch.autograd.grad(y, (w, b), gy)
    assert torch.cuda.max_memory_allocated() - before <= 8 * 4 * n
    assert torch.equal(gb, gy[0])
    d = x.detach().double()
    want = gy.double() * (d - d.mean()) / (d.var(correction=0) + 1e-5).sqrt()
    assert (gw.double() - want[0]).abs().max() <= 5e-6 * want.abs().max()
