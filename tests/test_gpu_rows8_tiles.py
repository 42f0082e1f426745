"""Rows in 8 bits where every block or pair of SMs takes many tiles: stages, accumulators, scale slots and kept rows are
used again and again.  The rows are whole numbers (tests/rows8_exact.py), so results are compared for equality."""
import pytest
import torch

from coresets_b200 import RowStore, coverage, quantise_rows, read_rows, row_products
from tests import rows8_exact as ex

pytestmark = pytest.mark.gpu


def stored(n, dim, seed, powers=False):
    x = ex.whole_rows(n, dim, seed, powers)
    store = quantise_rows(x)
    assert torch.equal(read_rows(store), x)
    return store, x


# ---- coverage by more than 64 centres: pairs of SMs ------------------------------------------------------------------

@pytest.mark.parametrize("n,k,dim", [
    # about 12 tiles a pair, runs cut inside the rows of a segment: two issuing warps (dim <= 256), one, rows not kept (dim > 1024)
    (20000, 2000, 16), (20000, 2000, 30), (20000, 2000, 50), (20000, 2000, 128), (20000, 1999, 256), (20000, 2000, 384),
    (20000, 2000, 513), (20000, 2000, 1100),
    # several segments a pair: the kept rows are filled again in both slots (dim <= 512) and in the only one
    (60001, 300, 16), (60001, 300, 40), (60001, 300, 128), (60001, 300, 200), (60001, 300, 512), (60001, 300, 700), (60001, 300, 1024),
    (60001, 90, 256),
])
def test_coverage_of_many_tiles_is_exact(n, k, dim):
    (a, x), (c, y) = stored(n, dim, n + dim), stored(k, dim, k)
    want = ex.distances(x, y)
    assert torch.equal(coverage(a, c).double(), want)
    h = torch.where(torch.arange(n, device="cuda") % 3 == 0, want / 2, float("inf")).float()
    h[5::7] = -1.0
    prior = h.double()
    coverage(a, c, h=h)
    assert torch.equal(h.double(), torch.minimum(prior, want))
    a.check_status()


@pytest.mark.parametrize("dim", [16, 48, 128, 300, 1100])
def test_every_digit_of_a_centres_norm(dim):
    """Rows of zeros are as far from a centre as its norm says, in all 24 bits.  Each column of two tiles in turn has the only
    centre that is not NaN."""
    k = 384
    zeros = quantise_rows(torch.zeros(3, dim, device="cuda"))
    c, _ = stored(k, dim, 1)
    g = torch.Generator(device="cuda").manual_seed(dim)
    part = torch.randint(0, 1 << 23, (k,), generator=g, device="cuda", dtype=torch.int32)
    norms = (part | torch.randint(127 - 60, 127 + 61, (k,), generator=g, device="cuda", dtype=torch.int32) << 23).view(torch.float32)
    for i in range(6):                                                    # one digit alone, and all but one
        norms[2 * i] = float(0x800000 | 15 << 4 * i)
        norms[2 * i + 1] = float((0xFFFFFF & ~(15 << 4 * i)) | 0x800000)
    c = RowStore.from_tensors(c.codes, c.scales, norms, dim)
    got = []
    for p in range(k):
        pick = torch.full((k - p % 5,) if p < k - 5 else (k,), -1, device="cuda")
        pick[p] = p
        got.append(coverage(zeros, c.take(pick)))
    got = torch.stack(got)
    assert torch.equal(got, norms[:, None].expand(k, 3))


# ---- products of many rows with many: pairs of SMs --------------------------------------------------------------

@pytest.mark.parametrize("n,k", [(4096, 8192), (4001, 8191)])          # bulk stores, and the readers' own
@pytest.mark.parametrize("dim", [16, 40, 128, 256, 384, 1024, 2050])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_products_of_many_tiles_are_exact(n, k, dim, dtype):
    (a, x), (b, y) = stored(n, dim, n + dim, powers=True), stored(k, dim, k, powers=True)
    assert torch.equal(row_products(a, b, dtype=dtype), ex.products(x, y).float().to(dtype))
    a.check_status()


# ---- at most 64 columns: single SMs ------------------------------------------------------------------------

@pytest.mark.parametrize("k", [1, 9, 16, 20, 32, 33, 64])
@pytest.mark.parametrize("n,dim", [(200_000, 16), (200_003, 30), (200_000, 50), (200_003, 128), (200_000, 300), (50_001, 1100)])
def test_few_columns_of_many_tiles_are_exact(n, k, dim):
    (a, x), (b, y) = stored(n, dim, n + dim), stored(k, dim, k)
    want = ex.distances(x, y)
    assert torch.equal(coverage(a, b).double(), want)
    h = torch.where(torch.arange(n, device="cuda") % 3 == 0, want / 2, float("inf")).float()
    h[5::7] = -1.0
    prior = h.double()
    coverage(a, b, h=h)
    assert torch.equal(h.double(), torch.minimum(prior, want))
    want = ex.products(x, y).float()
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(row_products(a, b, dtype=dtype), want.to(dtype))       # rows of the result follow the columns
        assert torch.equal(row_products(b, a, dtype=dtype), want.T.to(dtype))     # and the lanes
    a.check_status()
    b.check_status()
