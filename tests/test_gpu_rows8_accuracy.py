"""Rows in 8 bits: products and distances of rows that float32 does not hold exactly, within what the tensor core's steps may be
off (tests/rows8_exact.py says how that is derived)."""
import pytest
import torch

from coresets_b200 import coverage, quantise_rows, read_rows, row_products
from tests import rows8_exact as ex

pytestmark = pytest.mark.gpu


def stored(n, dim, seed, kind="normal"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, dim, generator=g, device="cuda")
    if kind == "one sign":
        x = x.abs()
    else:
        x *= torch.exp2(torch.randint(-6, 6, (n, 1), generator=g, device="cuda").float())
    store = quantise_rows(x)
    return store, read_rows(store)


@pytest.mark.parametrize("kind", ["normal", "one sign"])
@pytest.mark.parametrize("n,k,dim", [
    (300, 200, 31), (60, 200, 50), (300, 40, 64), (200, 130, 100), (128, 100, 256), (257, 300, 1024), (40, 9, 1024), (64, 70, 2050), (60, 50, 4096),
    (100, 90, 4096), (70, 90, 20011), (9, 30, 65536), (70, 80, 65536),
])
def test_products_within_the_steps_error(n, k, dim, kind):
    (a, x), (b, y) = stored(n, dim, dim, kind), stored(k, dim, dim + 1, kind)
    for dtype in (torch.float32, torch.bfloat16):
        want, off = ex.product_range(x, y, dtype)
        got = row_products(a, b, dtype=dtype).double()
        assert ((got - want).abs() <= off).all(), float(((got - want).abs() / off).max())


@pytest.mark.parametrize("n,k,dim", [
    (33, 2000, 128), (1000, 33, 100), (1000, 64, 256), (700, 300, 16), (500, 200, 48), (500, 65, 129), (300, 400, 513),
    (257, 300, 1024), (60, 50, 1100), (60, 70, 1100), (3000, 512, 64), (20, 70, 20011), (70, 80, 4096),
])
def test_coverage_within_the_steps_error(n, k, dim):
    (a, x), (c, y) = stored(n, dim, dim), stored(k, dim, dim + 1)
    low, high = ex.distance_range(x, y)
    got = coverage(a, c).double()
    assert ((got >= low) & (got <= high)).all()


@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("dim", [40, 128, 256, 600, 1100])
def test_coverage_of_rows_close_to_a_centre(k, dim):
    """Distances of about 2^-10 of the norms: the norm's lower digits and the product's lower bits decide."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    c, y = stored(k, dim, dim + 2)
    near = torch.randint(0, k, (900,), generator=g, device="cuda")
    x = y[near]
    one = torch.randint(0, dim, (900, max(1, dim // 64)), generator=g, device="cuda")      # these elements move by a code or two
    x.scatter_(1, one, x.gather(1, one) * 1.125)
    a = quantise_rows(x)
    x = read_rows(a)
    low, high = ex.distance_range(x, y)
    got = coverage(a, c).double()
    assert ((got >= low) & (got <= high)).all()


@pytest.mark.parametrize("k", [40, 300])
@pytest.mark.parametrize("n,dim", [(300, 70), (20000, 700)])
def test_coverage_of_single_elements_is_exact(n, dim, k):
    """One element a row, each at its own place: distances are sums of three exact numbers."""
    g = torch.Generator(device="cuda").manual_seed(dim + k)

    def rows(m):
        x = torch.zeros(m, dim, device="cuda")

        def whole(low, high):
            return torch.randint(low, high, (m, 1), generator=g, device="cuda")
        v = (1 + whole(0, 8) / 8) * torch.exp2(whole(-3, 4).float())
        return x.scatter_(1, whole(0, dim), v * (1 - 2 * whole(0, 2)))
    x, y = rows(n), rows(k)
    assert torch.equal(coverage(quantise_rows(x), quantise_rows(y)).double(), ex.distances(x, y))
