"""The ranges that the GPU tests of products and distances allow (tests/rows8_exact.py): what the tensor core's steps give lies
inside, sums and norms with fewer bits do not."""
import numpy as np
import pytest
import torch

from tests import rows8_exact as ex, rows8_oracle as ref


def stored(n, dim, seed):
    g = np.random.default_rng(seed)
    return torch.from_numpy(ref.quantise(g.standard_normal((n, dim)) * np.exp2(g.integers(-6, 6, (n, 1))))[2])


def cut(x, grid):
    return torch.trunc(x / grid) * grid


def cut_bits(x, bits):
    power = torch.frexp(x)[1].double()
    return torch.where(x == 0, x, cut(x, torch.exp2(power - bits)))


def steps(a, b, start=None, bits=24, kept=25):
    """The sum over steps of 32 elements as rows8_exact.sum_error describes a step."""
    acc = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64) if start is None else start.expand(a.shape[0], -1).clone()
    for d in range(0, a.shape[1], 32):
        t = torch.cat([a[:, None, d : d + 32] * b[None, :, d : d + 32], acc[:, :, None]], 2)
        top = torch.frexp(t.abs().amax(2))[1].double() - 1
        acc = cut_bits(cut(t, torch.exp2(top - kept)[:, :, None]).sum(2), bits)
    return acc


@pytest.mark.parametrize("dim", [31, 128, 256, 1024, 2050])
def test_product_range(dim):
    a, b = stored(40, dim, dim), stored(30, dim, dim + 1)
    want, off = ex.product_range(a, b, torch.float32)
    assert ((steps(a, b) - want).abs() <= off).all()
    assert ((steps(a.abs(), b.abs()) - ex.products(a.abs(), b.abs())).abs() <= off).all()
    for bits in (18, 16, 14):                                      # an accumulator of fewer bits
        assert ((steps(a, b, bits=bits) - want).abs() > off).any(), bits
    assert ((steps(a, b, kept=14) - want).abs() > off).any()      # terms of fewer bits
    lost = a.clone()
    lost[:, dim // 2] = 0                                            # an element left out
    assert ((ex.products(lost, b) - want).abs() > off).float().mean() > 0.9


@pytest.mark.parametrize("dim", [50, 128, 256, 600, 1100])
def test_distance_range(dim):
    c = stored(70, dim, dim)
    g = np.random.default_rng(dim)
    a = c[torch.from_numpy(g.integers(0, 70, 200))].clone()
    one = torch.from_numpy(g.integers(0, dim, (200, max(1, dim // 64))))
    a.scatter_(1, one, a.gather(1, one) * 1.125)
    a = torch.cat([torch.from_numpy(ref.quantise(a.numpy())[2]), stored(60, dim, dim + 5)])
    low, high = ex.distance_range(a, c)

    def inside(norms, bits=24):
        best = steps(a, c, start=-norms / 2, bits=bits).amax(1)
        d = ((a * a).sum(1) - 2 * best).clamp_min(0)
        return (d >= low) & (d <= high)
    norms = (c * c).sum(1)
    assert inside(norms.float().double()).all()
    for bits in (16, 12, 8):                                       # two, three and four of the six digits of a norm lost
        assert not inside(cut_bits(norms, bits)).all(), bits
    assert not inside(norms, bits=18).all()
    near = (a.square().sum(1)[:, None] + norms - 2 * a @ c.T).argmin(1)
    for i in near.unique()[::7]:                                   # a centre left out is seen by rows it is nearest to
        others = torch.arange(70) != i
        d = ((a * a).sum(1)[:, None] + norms[others] - 2 * a @ c[others].T).amin(1)
        assert (d > high)[near == i].any()
