"""Layer norm and dropout (flyguy_b200.layers) against their definitions in float64 numpy.

Tolerances: a result's rounding, at most half a step of its type (2^-24, 2^-8 / 2, 2^-11 of the value; `eps` / 2 of torch.finfo), and for
layer norm what sums in fp32 leave: the mean of n values is off by sqrt(n) 2^-24 of their size at most in the mean, the rest of the
chain (5 roundings) 5 2^-24; 1e-6 covers rows of up to 20,000 values that are no more than 10 deviations from zero. Sums over rows
(gw, gb): 2^-24 sqrt(rows) of their terms' size, 5e-6."""
import math

import numpy as np
import pytest
import torch

from flyguy_b200 import layers
from flyguy_b200.native import FlyguyError

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda t: str(t).replace("torch.", "")   # noqa: E731


def _np(t):
    return t.detach().double().cpu().numpy()


def _near(got, want, typ, sums=1e-6, what="", of=None):
    """Each value within its own rounding and `sums` of the largest (of `of`, where `want` is a difference of larger terms)."""
    got = _np(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.size:
        limit = torch.finfo(typ).eps / 2 * np.abs(want) * (1 + 1e-3) + sums * np.abs(want if of is None else of).max() + 1e-30
        if typ is torch.float16:
            limit = limit + 2.0 ** -25                           # (subnormal results)
        assert (np.abs(got - want) <= limit).all(), (what, (np.abs(got - want) / limit).max())


def _norm(x, w, b, eps):
    d = x - x.mean(-1, keepdims=True)
    return d / np.sqrt((d * d).mean(-1, keepdims=True) + eps) * w + b


def _norm_grads(x, w, gy, eps):
    d = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    h, g = d * r, gy * w
    return r * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True)), (gy * h).reshape(-1, x.shape[-1]).sum(0), \
        gy.reshape(-1, x.shape[-1]).sum(0), r * g


# one value, parts of a unit, a unit, groups of 8 lanes, whole warps, odd lengths that begin anywhere, blocks, rows that no block holds;
# few rows and more than there are blocks
SHAPES = [(3, 1), (5, 3), (1, 8), (7, 16), (9, 63), (300, 64), (33, 127), (2500, 130), (8, 517), (2405, 517), (2400, 1024), (3001, 1021),
          (4, 1025), (40, 2048), (6, 4095), (3, 8192), (2, 8193), (2, 20000), (5000, 24), (2377, 257)]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(shape, typ, cuda):
    rows, dim = shape
    g = torch.Generator().manual_seed(rows * 31 + dim)
    x = (torch.randn(rows, dim, generator=g) + 2 * torch.randn(rows, 1, generator=g)).to(typ).cuda().requires_grad_()
    w, b = (1 + 0.2 * torch.randn(dim, generator=g)).cuda().requires_grad_(), torch.randn(dim, generator=g).cuda().requires_grad_()
    gy = torch.randn(rows, dim, generator=g).to(typ).cuda()
    y = layers.layer_norm(x, w, b, eps=1e-3)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    _near(y, _norm(_np(x), _np(w), _np(b), 1e-3), typ, what="y")
    want_x, want_w, want_b, terms = _norm_grads(_np(x), _np(w), _np(gy), 1e-3)
    _near(gx, want_x, typ, 3e-6, "gx", terms)
    _near(gw, want_w, torch.float32, 5e-6, "gw")
    _near(gb, want_b, torch.float32, 5e-6, "gb")
    again = torch.autograd.grad(layers.layer_norm(x, w, b, eps=1e-3), (x, w, b), gy)
    assert all(torch.equal(p, q) for p, q in zip(again, (gx, gw, gb)))
    with torch.no_grad():
        assert torch.equal(layers.layer_norm(x, w, b, eps=1e-3), y)
        _near(layers.layer_norm(x, w, eps=1e-3), _norm(_np(x), _np(w), 0.0, 1e-3), typ, what="no bias")
        _near(layers.layer_norm(x, None, b, eps=1e-3), _norm(_np(x), 1.0, _np(b), 1e-3), typ, what="no weight")
    plain, = torch.autograd.grad(layers.layer_norm(x, eps=1e-3), x, gy)
    _near(plain, _norm_grads(_np(x), 1.0, _np(gy), 1e-3)[0], typ, 3e-6, "gx alone", _norm_grads(_np(x), 1.0, _np(gy), 1e-3)[3])


def test_a_mean_far_from_zero_costs_no_digits(cuda):
    """Values 1 apart at 2^14: the mean is off by at most 2^-10 (fp32 at 2^14), the deviations by as much, 1e-3 of them."""
    x = (2.0 ** 14 + torch.randn(64, 1000, generator=torch.Generator().manual_seed(1))).cuda()
    want = _norm(_np(x), 1.0, 0.0, 1e-5)
    assert np.abs(_np(layers.layer_norm(x)) - want).max() <= 2.0 ** -10 * 1.01


@pytest.mark.parametrize("typ", TYPES, ids=names)
def test_layer_norm_rows_apart_and_other_strides(typ, cuda):
    """Rows of a wider tensor, rows that begin at odd places, heads before ticks, expanded rows; and the gradient's."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(2500, 600, generator=g).to(typ).cuda()
    views = [wide[:, :517], wide[:, 3:520], wide[:, 8:136], wide.view(50, 50, 600)[:, :, :64], wide[:2400].view(40, 60, 600).transpose(0, 1)[..., :130],
             wide[:1].expand(30, 600), wide[:, ::2], wide[::3, 1:2], wide[:2400, :517].as_strided((2400, 517), (600, 1), 1)]
    for i, v in enumerate(views):
        x = v.detach().requires_grad_()
        y = layers.layer_norm(x)
        gy = torch.randn(y.shape, generator=g).to(typ).cuda()
        gx, = torch.autograd.grad(y, x, gy)
        want, _, _, terms = _norm_grads(_np(v), 1.0, _np(gy), 1e-5)
        _near(y, _norm(_np(v), 1.0, 0.0, 1e-5), typ, 1e-6, i)
        _near(gx, want, typ, 3e-6, i, terms)
        c = v.detach().contiguous().clone().requires_grad_()
        gc, = torch.autograd.grad(layers.layer_norm(c), c, gy)
        assert y.is_contiguous() and y.shape == v.shape
        back, = torch.autograd.grad(layers.layer_norm(c), c, gy.transpose(0, -1).contiguous().transpose(0, -1))
        assert torch.equal(back, gc)


def test_layer_norm_of_nothing_and_of_bad_values(cuda):
    w = torch.ones(8, device=cuda, requires_grad=True)
    y = layers.layer_norm(torch.zeros(0, 8, device=cuda, requires_grad=True), w)
    y.sum().backward()
    assert y.shape == (0, 8) and not w.grad.any()
    x = torch.randn(2400, 64, device=cuda)
    clean = layers.layer_norm(x)
    x[7, 3], x[9, 5] = math.nan, math.inf
    y = layers.layer_norm(x)
    assert y[7].isnan().all() and y[9].isnan().all()
    rest = [i for i in range(2400) if i not in (7, 9)]
    assert torch.equal(y[rest], clean[rest])
    assert not layers.layer_norm(torch.full((3, 40), 5.0, device=cuda)).any()     # rows without deviations
    assert layers.layer_norm(torch.randn(70, device=cuda)).shape == (70,)


def test_layer_norm_captured_on_another_stream(cuda):
    x, w = torch.randn(3000, 517, device=cuda, requires_grad=True), torch.ones(517, device=cuda, requires_grad=True)
    gy = torch.randn(3000, 517, device=cuda)

    def step():
        y = layers.layer_norm(x, w)
        return y, *torch.autograd.grad(y, (x, w), gy)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn(3000, 517, device=cuda))
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_layer_norm_of_inputs_made_in_inference_mode(cuda):
    with torch.inference_mode():
        x = torch.randn(5, 40, device=cuda)
    w = torch.ones(40, device=cuda, requires_grad=True)
    gw, = torch.autograd.grad(layers.layer_norm(x, w).sum(), w)
    _near(gw, _norm(_np(x), 1.0, 0.0, 1e-5).sum(0), torch.float32, 5e-6)


def test_layer_norm_refusals(cuda):
    x = torch.zeros(4, 8, device=cuda)
    for args, words in (((torch.zeros(4, 8),), "CUDA"), ((x.double(),), "float32, bfloat16"), ((x, torch.zeros(7, device=cuda)), "weight must be"),
                        ((x, None, torch.zeros(8, device=cuda).half()), "bias must be"), ((torch.zeros(4, 0, device=cuda),), "last dimension"),
                        ((x, None, None, 0.0), "eps"), ((x, None, None, math.nan), "eps"), ((torch.zeros((), device=cuda),), "last dimension")):
        with pytest.raises(FlyguyError, match=words):
            layers.layer_norm(*args)
    g, = torch.autograd.grad(layers.layer_norm(x.requires_grad_()).sum(), x, create_graph=True)
    with pytest.raises(FlyguyError, match="again"):
        g.sum().backward()


# ---- dropout -------------------------------------------------------------------------------------------------------

def _bits(n, seed, call):
    """The 16 bits of values 0 .. n - 1."""
    from test_layers_host import philox
    block = np.arange(-(-n // 8), dtype=np.uint64)
    words = philox([block & 0xffffffff, block >> np.uint64(32), np.full_like(block, call & 0xffffffff), np.full_like(block, call >> 32)],
                   [seed & 0xffffffff, (seed >> 32) & 0xffffffff])
    return np.stack([h for w in words for h in (w & np.uint64(0xffff), w >> np.uint64(16))], -1).reshape(-1)[:n]


@pytest.mark.parametrize("typ", TYPES, ids=names)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 4099, 2048 * 148 * 64 + 13])
def test_dropout(n, typ, cuda):
    g = torch.Generator().manual_seed(n)
    seed, call = -12345678901234567, (3 << 32) + 5
    x, add, gy = (torch.randn(n, generator=g).to(typ).cuda() for _ in range(3))
    for p, with_add in ((0.1, True), (0.5, False)):
        least = round(65536 * p)
        kept = _bits(n, seed, call) >= least
        by = 65536 / (65536 - least)
        leaf, res = x.detach().requires_grad_(), add.detach().requires_grad_()
        y = layers.dropout(leaf, p, seed, call, res if with_add else None)
        want = np.where(kept, _np(x) * by, 0.0)
        _near(y, want + (_np(add) if with_add else 0.0), typ, 2.0 ** -23, "y")
        gx = torch.autograd.grad(y, (leaf, res) if with_add else (leaf,), gy)
        _near(gx[0], np.where(kept, _np(gy) * by, 0.0), typ, 2.0 ** -23, "gx")
        assert not with_add or torch.equal(gx[1], gy)
        if n > 1000:
            assert abs(kept.mean() - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n)


def test_dropout_keeps_all_and_drops_bad_values(cuda):
    x = torch.randn(100, 33, device=cuda)
    assert torch.equal(layers.dropout(x, 0.0, 1), x)
    y = layers.dropout(torch.full((4096,), math.inf, device=cuda), 0.5, 2, add=torch.ones(4096, device=cuda))
    assert not y.isnan().any() and set(y.tolist()) == {math.inf, 1.0}
    assert not layers.dropout(torch.full((4096,), math.nan, device=cuda), 65535 / 65536, 3)[:64].isfinite().logical_not().all()


def test_dropout_of_views_and_unaligned(cuda):
    """The mask goes by a value's place in the tensor, wherever it lies in memory."""
    g = torch.Generator().manual_seed(4)
    base = torch.randn(64, 101, generator=g).half().cuda()
    x = base[:, 1:]
    assert torch.equal(layers.dropout(x, 0.3, 9), layers.dropout(x.contiguous(), 0.3, 9))
    odd = base.view(-1)[1:6401].view(64, 100)
    assert torch.equal(layers.dropout(odd, 0.3, 9), layers.dropout(odd.clone(), 0.3, 9))
    assert torch.equal(layers.dropout(x.t(), 0.3, 9, add=odd.t()), layers.dropout(x.t().contiguous(), 0.3, 9, add=odd.t().contiguous()))
    assert layers.dropout(torch.zeros(0, 5, device=cuda), 0.3, 9).shape == (0, 5)


def test_dropout_seed_on_the_device_in_a_graph(cuda):
    """A captured call reads the seed when it is replayed; its backward, too, with the same mask."""
    x, gy = torch.randn(1000, device=cuda, requires_grad=True), torch.randn(1000, device=cuda)
    seed = torch.tensor([77], device=cuda)

    def step():
        y = layers.dropout(x, 0.4, seed, call=2)
        return y, *torch.autograd.grad(y, x, gy)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step()
    for s in (77, 78, (1 << 62) + 3):
        seed.fill_(s)
        graph.replay()
        want = layers.dropout(x.detach(), 0.4, s, call=2)
        assert torch.equal(y, want) and torch.equal(gx == 0, want == 0)
    assert not torch.equal(layers.dropout(x.detach(), 0.4, 77, 2), layers.dropout(x.detach(), 0.4, 77, 3))


def test_dropout_a_seed_that_changed_before_the_backward_is_told(cuda):
    x, seed = torch.randn(100, device=cuda, requires_grad=True), torch.tensor([5], device=cuda)
    y = layers.dropout(x, 0.4, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_refusals(cuda):
    x = torch.zeros(4, 8, device=cuda)
    for args, words in (((torch.zeros(4), 0.1, 1), "CUDA"), ((x.double(), 0.1, 1), "float32, bfloat16"), ((x, 1.0, 1), "p must be"),
                        ((x, -0.1, 1), "p must be"), ((x, 0.99999999, 1), "p must be"), ((x, 0.1, 1 << 63), "64 bits"), ((x, 0.1, 1.5), "64 bits"),
                        ((x, 0.1, torch.zeros(2, dtype=torch.int64, device=cuda)), "one element"), ((x, 0.1, torch.zeros(1, dtype=torch.int64)), "one element"),
                        ((x, 0.1, 1, -1), "call must be"), ((x, 0.1, 1, 0, x[:2]), "add must have"), ((x, math.nan, 1), "p must be")):
        with pytest.raises(FlyguyError, match=words):
            layers.dropout(*args)
