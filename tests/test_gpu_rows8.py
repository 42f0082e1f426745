"""Rows in 8 bits on the GPU against their definitions in 64 bits (tests/rows8_oracle.py)."""
import numpy as np
import pytest
import torch

import coresets_b200 as coresets
import oracle
from coresets_b200 import RowStore, _native, coverage, quantise_rows, read_rows, row_products
from coresets_b200.rows8 import store_matrix
from tests import rows8_oracle as ref
from tests.data import gaussian_mixture

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24        # half a step of float32


def rows(n, dim, seed=0, scale=1.0):
    g = np.random.default_rng(seed)
    return torch.from_numpy((g.standard_normal((n, dim)) * scale * np.exp2(g.integers(-6, 6, (n, 1)))).astype(np.float32))


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def check_rows(store, first, x):
    """The store's rows first .. are the definition's for x (codes, exponents: equal; norms: a bound)."""
    n, dim = x.shape
    codes, exps, _, norms = ref.quantise(f64(x))
    got = f64(store.codes[first : first + n, :dim].float())
    np.testing.assert_array_equal(got, codes)
    assert not store.codes.view(torch.uint8)[first : first + n, dim:].any()
    np.testing.assert_array_equal(store.exponents[first : first + n].cpu().numpy(), exps)
    norms = np.where(norms > torch.finfo(torch.float32).max, np.inf, norms)
    # positive terms: a sum in float32 is off by the depth of its tree times half a step; 8 in a lane, one a
    # block, 4 between lanes, and the two products with the scale
    np.testing.assert_allclose(f64(store.norms[first : first + n]), norms, rtol=(8 + exps.shape[1] + 4 + 2) * U, atol=2.0 ** -126)


# ---- write ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 16, 24, 33, 50, 64, 100, 128, 129, 256, 500, 513, 1024, 1100])
def test_write_is_the_definition(dim, dtype):
    x = rows(67, dim, dim).to(dtype)
    store = quantise_rows(x.cuda())
    assert len(store) == store.capacity == 67 and store.dim == dim
    check_rows(store, 0, x)


@pytest.mark.parametrize("n", [1, 2, 31, 127, 128, 129, 1000])
def test_append_leaves_the_other_rows(n):
    dim = 200
    store = RowStore(1300, dim)
    store.codes.view(torch.uint8).fill_(0xA5)
    store.scales.fill_(0x5A)
    store.norms.fill_(-7.0)
    a, b = rows(130, dim, 1), rows(n, dim, 2)
    quantise_rows(a.cuda(), store=store)
    quantise_rows(b.cuda(), store=store)
    assert len(store) == 130 + n
    check_rows(store, 0, a)
    check_rows(store, 130, b)
    assert (store.codes.view(torch.uint8)[130 + n :] == 0xA5).all() and (store.norms[130 + n :] == -7.0).all()
    t = store.scales.permute(0, 3, 2, 1, 4).reshape(-1, 4)          # one word of exponents a row
    assert (t[130 + n :] == 0x5A).all()
    c = rows(5, dim, 3)
    quantise_rows(c.cuda(), store=store, start=128)                 # over rows that are there
    assert len(store) == max(130 + n, 133)
    check_rows(store, 128, c)
    check_rows(store, 0, a[:128])


def test_write_special_values():
    f = torch.finfo(torch.float32)
    x = torch.zeros(12, 160)
    x[1, 3] = float("nan")
    x[1, 5] = 2.0
    x[2, :4] = torch.tensor([float("inf"), float("-inf"), 1.0, -3.5])
    x[3] = f.max
    x[4] = -f.tiny
    x[5] = 2.0 ** -140                                            # subnormal float32
    x[6] = torch.linspace(-448, 448, 160)
    x[7, :128] = 17.0 / 16 * 2.0 ** 5                             # halfway between two codes: ties to even
    x[7, 0] = 448.0
    x[7, 1:5] = torch.tensor([27.0, 29.0, -27.0, -29.0])          # halfway at a step of 2
    x[8, 0], x[8, 1] = 448.0, 448.0001
    x[9, 0], x[9, 1:6] = 448.0, torch.tensor([1.0, 3.0, 5.0, 0.5, 1.5]) * 2.0 ** -10   # around the smallest codes
    x[10] = float("nan")
    x[11, 0], x[11, 1], x[11, 130] = f.max, f.tiny, 2.0 ** -127
    check_rows(quantise_rows(x.cuda()), 0, x)
    y = torch.tensor([[65504.0, 2.0 ** -24, -(2.0 ** -14), float("inf"), 1.0]], dtype=torch.float16)
    check_rows(quantise_rows(y.cuda()), 0, y)
    z = torch.tensor([[float(torch.finfo(torch.bfloat16).max), 1e-38, 2.0 ** -130, float("nan")]], dtype=torch.bfloat16)
    check_rows(quantise_rows(z.cuda()), 0, z)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_strided_inputs(dtype):
    base = rows(90, 300, 5).to(dtype).cuda()
    for x in (base[:, 16:272], base[:, 3:131], base[::3, :64], base[1:, :299], base.t(), base[:1].expand(40, 300), base[:, ::2],
              base[7:8, 5:6], base.view(-1)[1 : 1 + 50 * 50].view(50, 50)):
        check_rows(quantise_rows(x), 0, x.cpu())


def test_write_empty_and_full():
    store = quantise_rows(torch.empty(0, 40, device="cuda"))
    assert len(store) == 0 and read_rows(store).shape == (0, 40)
    store = RowStore(3, 40)
    quantise_rows(torch.empty(0, 40, device="cuda"), store=store)
    assert len(store) == 0
    x = rows(3, 40)
    quantise_rows(x.cuda(), store=store)
    with pytest.raises(ValueError, match="do not fit"):
        quantise_rows(x.cuda(), store=store)
    with pytest.raises(ValueError, match="start=4"):
        quantise_rows(x.cuda(), store=store, start=4)
    quantise_rows(x.cuda() * 2, store=store, start=0)
    check_rows(store, 0, x * 2)


# ---- read, take -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 4, 7, 8, 50, 64, 128, 200, 520, 1024, 1100])
def test_read_is_what_is_stored(dim, dtype):
    x = rows(300, dim, dim + 1)
    store = quantise_rows(x.cuda())
    want = torch.from_numpy(ref.quantise(f64(x))[2]).to(torch.float32)        # 4 significant bits: exact in float32
    torch.testing.assert_close(read_rows(store, dtype=dtype).cpu(), want.to(dtype), rtol=0, atol=0)
    pick = torch.tensor([299, 0, 5, 5, 128, 127, 299], device="cuda")
    torch.testing.assert_close(read_rows(store, pick, dtype=dtype).cpu(), want[pick.cpu()].to(dtype), rtol=0, atol=0)
    wide = torch.full((7, dim + 9), -1.0, dtype=dtype, device="cuda")
    got = read_rows(store, pick.to(torch.int32), dtype=dtype, out=wide[:, 5 : 5 + dim])
    assert got.data_ptr() == wide[:, 5:].data_ptr()
    torch.testing.assert_close(wide[:, 5 : 5 + dim].cpu(), want[pick.cpu()].to(dtype), rtol=0, atol=0)
    assert (wide[:, :5] == -1).all() and (wide[:, 5 + dim :] == -1).all()


def test_read_rows_out_of_range():
    store = quantise_rows(rows(10, 20).cuda(), store=RowStore(16, 20))
    got = read_rows(store, torch.tensor([0, -1, 10, 15, 1 << 40, 9], device="cuda"))
    assert torch.isnan(got).all(1).tolist() == [False, True, True, True, True, False]
    for bad in ([10], [-1], torch.tensor([0, 16])):
        with pytest.raises(IndexError):
            read_rows(store, bad)
    for bad in (torch.zeros(2, 2, dtype=torch.int64), torch.ones(10, dtype=torch.bool, device="cuda"), torch.tensor([0.5])):
        with pytest.raises(ValueError):
            read_rows(store, bad)
    with pytest.raises(ValueError):
        read_rows(store, dtype=torch.float64)
    with pytest.raises(ValueError):
        read_rows(store, out=torch.empty(10, 21, device="cuda"))
    with pytest.raises(ValueError):
        read_rows(store, out=torch.empty(20, 10, device="cuda").t())


def test_read_extreme_exponents():
    x = torch.tensor([[3.0e38, 1.0, -2.0 ** 119], [2.0 ** -126, 2.0 ** -120, 0.0]])
    store = quantise_rows(x.cuda())
    want = torch.from_numpy(ref.quantise(f64(x))[2])
    torch.testing.assert_close(read_rows(store).cpu().double(), want, rtol=0, atol=0)
    torch.testing.assert_close(read_rows(store, dtype=torch.bfloat16).cpu().double(), want, rtol=0, atol=0)
    torch.testing.assert_close(read_rows(store, dtype=torch.float16).cpu(), want.to(torch.float16), rtol=0, atol=0)
    # arrays from elsewhere may hold any exponent byte: 0 is 2^-127, 255 NaN
    store.scales.zero_()
    assert read_rows(store)[1, 0].item() == store.codes.float()[1, 0].item() * 2.0 ** -127
    store.scales.fill_(255)
    assert torch.isnan(read_rows(store)).all()


@pytest.mark.parametrize("dim", [5, 64, 130, 1030])
def test_take_copies_rows_as_they_are(dim):
    store = quantise_rows(rows(400, dim, 9).cuda())
    pick = [399, 3, 3, 128, 0]
    part = store.take(pick)
    assert len(part) == 5
    assert torch.equal(part.codes.view(torch.uint8), store.codes.view(torch.uint8)[pick])
    assert torch.equal(part.exponents, store.exponents[pick]) and torch.equal(part.norms, store.norms[pick])
    odd = store.take(torch.tensor([1, -5, 400], device="cuda"))
    assert torch.isnan(read_rows(odd)).all(1).tolist() == [False, True, True] and torch.isnan(odd.norms[1:]).all()
    assert len(store.take(torch.empty(0, dtype=torch.int64))) == 0


# ---- products -------------------------------------------------------------------------------------------

def stored(n, dim, seed, scale=1.0):
    x = rows(n, dim, seed, scale)
    return quantise_rows(x.cuda()), ref.quantise(f64(x))[2]


def product_bound(a, b, dtype):
    """(the products, how far one may be off).  Terms are exact; D additions to a float32 accumulator, each off
    by a whole step 2^-23 at most (truncation) of what the terms' magnitudes sum to; one rounding, of half a step
    relative to the value, or half of the type's smallest step (float16: 2^-24, its subnormals' spacing) below
    its normal range."""
    want, mags = ref.products(a, b)
    f = torch.finfo(dtype)
    return want, mags * a.shape[1] * 2.0 ** -23 + np.maximum(np.abs(want) * f.eps / 2, f.smallest_normal * f.eps / 2)


@pytest.mark.parametrize("n,k,dim", [
    (1, 1, 1), (1, 1, 128), (1, 300, 64), (300, 1, 64), (5, 16, 50), (16, 5, 50), (17, 33, 128), (33, 17, 129), (64, 200, 256), (200, 64, 256),
    (65, 66, 100), (300, 300, 16), (400, 70, 13), (70, 400, 48), (500, 20, 16), (20, 500, 9), (300, 200, 24), (130, 129, 64), (128, 128, 512), (129, 127, 513), (130, 1000, 1024), (1000, 130, 31), (777, 409, 1100), (3, 2000, 2050), (500, 140, 32), (260, 257, 96),
])
def test_products(n, k, dim):
    a, av = stored(n, dim, 3)
    b, bv = stored(k, dim, 4)
    for dtype in DTYPES:
        want, off = product_bound(av, bv, dtype)
        got = row_products(a, b, dtype=dtype)
        assert got.shape == (n, k) and got.dtype == dtype
        ok = np.abs(f64(got) - want) <= off
        if dtype == torch.float16:
            ok |= np.abs(want) > 65000
        assert ok.all(), float((np.abs(f64(got) - want) - off).max())
    a.check_status()


def test_products_every_scale_and_place():
    """One non-zero element a row, each at its own place and with its own exponent: a scale or a code taken
    from another row or block gives another product."""
    n, dim = 256, 700
    place = (torch.arange(n) * 37) % dim
    x = torch.zeros(n, dim)
    x[torch.arange(n), place] = (1 + torch.arange(n) % 8 / 8) * torch.exp2((torch.arange(n) % 40 - 20).float())
    a = quantise_rows(x.cuda())
    y = torch.exp2(((torch.arange(dim)[None] // 128) * 5 + torch.arange(133)[:, None] % 9 - 15).float()) * torch.ones(133, dim)
    b = quantise_rows(y.cuda())
    want = f64(x) @ f64(y).T                                      # single terms with 4 + 1 significant bits: exact
    np.testing.assert_array_equal(f64(row_products(a, b)), want)
    np.testing.assert_array_equal(f64(row_products(b, a)), want.T)


def test_products_out_and_nan():
    a, av = stored(40, 60, 5)
    b, bv = stored(21, 60, 6)
    wide = torch.full((40, 30), -1.0, device="cuda")
    got = row_products(a, b, out=wide[:, 3:24])
    want, off = product_bound(av, bv, torch.float32)
    assert (np.abs(f64(got) - want) <= off).all() and (wide[:, :3] == -1).all() and (wide[:, 24:] == -1).all()
    c = b.take(torch.tensor([0, -1, 2], device="cuda"))           # a row of NaN spoils its own column only
    got = row_products(a, c)
    assert torch.isnan(got[:, 1]).all() and not torch.isnan(got[:, [0, 2]]).any()
    assert row_products(a, b.take([])).shape == (40, 0) and row_products(a.take([]), b).shape == (0, 21)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(5, 200), (60, 1000), (200, 5), (1000, 64), (1000, 33), (333, 200), (400, 1001), (129, 96)])
def test_products_into_part_of_a_matrix(n, k, dtype):
    """Rows of 16-byte multiples (bulk stores) and odd ones, at aligned and odd places: nothing beside the result is written."""
    dim = 72
    a, av = stored(n, dim, 30)
    b, bv = stored(k, dim, 31)
    want, off = product_bound(av, bv, dtype)
    for pitch, first in ((-(-k // 8) * 8 + 16, 8), (k + 3, 1), (k, 0)):
        wide = torch.full((n + 2, pitch), -1.0, dtype=dtype, device="cuda")
        got = row_products(a, b, dtype=dtype, out=wide[1 : n + 1, first : first + k])
        assert (np.abs(f64(got) - want) <= off).all()
        wide[1 : n + 1, first : first + k] = -1.0
        assert (wide == -1.0).all()


def test_wide_rows():
    dim = 20011
    a, av = stored(70, dim, 32, 0.1)
    b, bv = stored(90, dim, 33, 0.1)
    want, off = product_bound(av, bv, torch.float32)
    assert (np.abs(f64(row_products(a, b)) - want) <= off).all()
    off = coverage_bound(av, bv, dim)
    assert (np.abs(f64(coverage(a, b)) - ref.coverage(av, bv)) <= off).all()
    assert torch.equal(read_rows(a).cpu(), torch.from_numpy(av).float())


def test_offsets_past_32_bits():
    """Codes past 4 GiB, and a result of more than 2^31 elements (bulk stores and the readers' own)."""
    n, dim = 4_300_000, 1024
    store = RowStore.from_tensors(torch.zeros(n, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                                  torch.zeros(-(-n // 128), 2, 32, 4, 4, dtype=torch.uint8, device="cuda"), torch.zeros(n, device="cuda"), dim)
    x = rows(300, dim, 40)
    first = n - 301
    quantise_rows(x.cuda(), store=store, start=first)
    check_rows(store, first, x)
    _, _, xv, _ = ref.quantise(f64(x))
    assert not read_rows(store, torch.tensor([first - 1, n - 1], device="cuda")).any()
    np.testing.assert_array_equal(f64(read_rows(store, torch.arange(first, n - 1, device="cuda"))), xv)
    few, fv = stored(3, dim, 41)
    want, off = product_bound(fv, xv, torch.float32)
    got = row_products(few, store)
    assert (np.abs(f64(got[:, first : n - 1]) - want) <= off).all() and not got[:, :first].any()
    got = row_products(store, few)
    assert (np.abs(f64(got[first : n - 1]) - want.T) <= off.T).all() and not got[:first].any()
    part = store.take(torch.arange(first, first + 100, device="cuda"))
    h = f64(coverage(store, part))
    assert (np.abs(h[first : n - 1] - ref.coverage(xv, xv[:100])) <= coverage_bound(xv, xv[:100], dim)).all()
    assert (np.abs(h[:first] - (xv[:100] ** 2).sum(1).min()) <= (xv[:100] ** 2).sum(1).min() * 1e-5).all()
    del got, store, h
    for k in (1_000_000, 1_000_001):
        a, av = stored(2200, 16, 42)
        x = rows(1000, 16, 43)
        b = quantise_rows(x.cuda().repeat(-(-k // 1000), 1)[:k])
        got = row_products(a, b, dtype=torch.bfloat16)
        _, _, xv, _ = ref.quantise(f64(x))
        want, off = product_bound(av, xv, torch.bfloat16)
        for c in (0, k // 2000 * 1000, k // 1000 * 1000 - 1000):
            assert (np.abs(f64(got[:, c : c + 1000]) - want) <= off).all()
        del got


# ---- coverage -------------------------------------------------------------------------------------------

def coverage_bound(a, c, dim):
    """How far a squared distance may be off: both norms (16 + blocks halves of a step), twice the product (see
    product_bound) and the rounding of the two sums."""
    na, nc = (a * a).sum(1)[:, None], (c * c).sum(1)[None]
    mags = np.abs(a) @ np.abs(c).T
    off = (na + nc) * (16 + -(-dim // 128)) * U + 2 * mags * dim * 2.0 ** -23 + (na + nc + 2 * mags) * 3 * U
    return off.max(1)


@pytest.mark.parametrize("n,k,dim", [
    (1, 1, 1), (1, 700, 128), (33, 2000, 128), (130, 16, 50), (128, 17, 64), (1000, 33, 100), (1000, 64, 256), (700, 300, 16), (700, 300, 3), (500, 20, 16), (500, 90, 30), (500, 200, 48), (500, 65, 129), (300, 400, 513),
    (2000, 129, 31), (257, 300, 1024), (60, 50, 1100), (20000, 512, 64),
])
def test_coverage(n, k, dim):
    a, av = stored(n, dim, 7)
    c, cv = stored(k, dim, 8)
    want = ref.coverage(av, cv)
    got = f64(coverage(a, c))
    off = coverage_bound(av, cv, dim)
    assert got.shape == (n,) and (got >= 0).all() and (np.abs(got - want) <= off).all(), float((np.abs(got - want) - off).max())
    g = np.random.default_rng(1)
    prior = np.where(g.random(n) < 0.3, -1.0, want * g.uniform(0.5, 1.5, n)).astype(np.float32)
    prior[::5] = np.inf
    h = torch.from_numpy(prior).cuda()
    assert coverage(a, c, h=h) is h
    assert (np.abs(f64(h) - np.fmin(prior, want)) <= off).all()
    assert (f64(h)[prior == -1] == -1).all()
    a.check_status()


@pytest.mark.parametrize("k", [20, 200])
@pytest.mark.parametrize("scale", [2.0 ** -50, 2.0 ** -20, 2.0 ** 40, 2.0 ** 55])
def test_coverage_of_small_and_large_numbers(k, scale):
    dim = 100
    a, av = stored(200, dim, 13, scale)
    c, cv = stored(k, dim, 14, scale)
    assert (np.abs(f64(coverage(a, c)) - ref.coverage(av, cv)) <= coverage_bound(av, cv, dim)).all()


def test_coverage_of_the_same_rows_and_of_zeros():
    x = rows(300, 90, 15)
    x[7] = 0
    a = quantise_rows(x.cuda())
    _, _, av, _ = ref.quantise(f64(x))
    h = f64(coverage(a, a))
    assert (h <= coverage_bound(av, av, 90)).all() and h[7] == 0
    zeros = quantise_rows(torch.zeros(100, 90, device="cuda"))
    np.testing.assert_allclose(f64(coverage(a, zeros)), f64(a.norms), rtol=4 * U)


def test_coverage_of_chosen_rows_and_parts():
    a, av = stored(900, 70, 11)
    pick = torch.tensor([5, 800, 77, 301], device="cuda")
    h = coverage(a, pick)
    off = coverage_bound(av, av[pick.cpu().numpy()], 70)
    assert (f64(h)[pick.cpu().numpy()] <= off[pick.cpu().numpy()]).all()
    parts = coverage(a, pick[:1])
    coverage(a, pick[1:3], h=parts)
    coverage(a, pick[3:], h=parts)
    assert torch.equal(parts, h)                                  # a minimum has no order


def test_coverage_nothing_to_cover_with_and_nan():
    a, av = stored(50, 70, 12)
    empty = a.take([])
    assert torch.isinf(coverage(a, empty)).all()
    h = torch.arange(50, device="cuda").float()
    assert torch.equal(coverage(a, empty, h=h), torch.arange(50, device="cuda").float())
    assert coverage(empty, a).shape == (0,)
    some = a.take(torch.tensor([3, -1, 4], device="cuda"))        # the middle one is NaN and never the nearest
    assert torch.equal(coverage(a, some), coverage(a, a.take([3, 4])))
    assert torch.isinf(coverage(a, a.take(torch.tensor([-1], device="cuda")))).all()
    x = rows(50, 70, 12)
    x[9, 3] = float("inf")
    h = coverage(quantise_rows(x.cuda()), a.take([3, 4]))
    assert torch.isinf(h[9]) and torch.isfinite(h).sum() == 49


# ---- how they are called -------------------------------------------------------------------------------

def test_refusals():
    a, b = RowStore(4, 32), RowStore(4, 48)
    x = torch.zeros(2, 32, device="cuda")
    with pytest.raises(ValueError, match="columns"):
        quantise_rows(x, store=b)
    with pytest.raises(ValueError, match="gradient"):
        quantise_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="start needs a store"):
        quantise_rows(x, start=1)
    with pytest.raises(ValueError, match="elements"):
        row_products(a, b)
    with pytest.raises(ValueError, match="elements"):
        coverage(a, b)
    with pytest.raises(TypeError):
        row_products(a, x)
    with pytest.raises(TypeError):
        read_rows(x)
    with pytest.raises(TypeError):
        coverage(x, a)
    with pytest.raises(ValueError):
        row_products(a, a, dtype=torch.float64)
    quantise_rows(x, store=a)
    for h in (torch.zeros(3, device="cuda"), torch.zeros(2), torch.zeros(2, device="cuda", dtype=torch.float64), torch.zeros(4, device="cuda")[::2]):
        with pytest.raises(ValueError):
            coverage(a, a, h=h)
    with pytest.raises(ValueError):
        row_products(a, a, out=torch.zeros(2, 2, device="cuda").t()[:, :1].expand(2, 2))
    with pytest.raises(ValueError):
        RowStore.from_tensors(a.codes, b.scales[:0], a.norms, 32)
    with pytest.raises(ValueError):
        RowStore.from_tensors(a.codes.view(torch.uint8), a.scales, a.norms, 32)
    with pytest.raises(ValueError):
        RowStore.from_tensors(a.codes, a.scales, a.norms, 32, count=5)
    with pytest.raises(ValueError, match="n_to_select"):
        coresets.fps_cuda(a, 3)


@pytest.mark.parametrize("n,k", [(300, 5), (300, 200), (2000, 1000)])
def test_a_wait_that_runs_out_sets_the_status(n, k):
    """With the test hook the kernels' producer starts no copy: every wait ends by its bound, the block leaves, the status says
    so, and the next calls work."""
    a, c = quantise_rows(rows(n, 300, 1).cuda()), quantise_rows(rows(k, 300, 2).cuda())
    want = row_products(a, c), coverage(a, c)
    a._c.flags = c._c.flags = _native.ROWS8_TEST_STALL
    for call in (row_products, coverage):
        call(a, c)
        with pytest.raises(RuntimeError, match="ran out"):
            a.check_status()
        a._status.zero_()
    a._c.flags = c._c.flags = 0
    assert torch.equal(row_products(a, c), want[0]) and torch.equal(coverage(a, c), want[1])
    a.check_status()
    with pytest.raises(AttributeError):
        a.codes = c.codes


def test_calls_on_several_streams_at_once():
    a, b, c = (quantise_rows(rows(n, 256, n).cuda()) for n in (20000, 3000, 600))
    few = c.take(torch.arange(9))
    calls = [lambda: coverage(a, c), lambda: row_products(b, c, dtype=torch.bfloat16), lambda: row_products(few, a), lambda: coverage(a, few),
             lambda: read_rows(a), lambda: row_products(c, b)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(10):
        for f, s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(f())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_from_tensors_shares_memory():
    a, av = stored(10, 40, 1)
    b = RowStore.from_tensors(a.codes, a.scales, a.norms, 40, count=7)
    assert len(b) == 7 and torch.equal(read_rows(b), read_rows(a)[:7])
    quantise_rows(torch.ones(1, 40, device="cuda"), store=b, start=0)
    assert (read_rows(a)[0] == 1).all()


def test_other_stream_and_captured_calls():
    x, y = rows(500, 96, 20).cuda(), rows(500, 96, 21).cuda()
    store, c = quantise_rows(x), quantise_rows(rows(90, 96, 22).cuda())
    want = [t.clone() for t in (row_products(store, c), coverage(store, c), read_rows(store))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s2 = quantise_rows(x)
        got = [row_products(s2, c), coverage(s2, c), read_rows(s2)]
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    # two graphs over the same inputs, replayed on new contents, one after the other and at once
    X = x.clone()
    into = quantise_rows(X)
    pick = torch.arange(0, 500, 7, device="cuda")
    graphs, outs, h = [], [], [torch.empty(500, device="cuda") for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if i == 0:
                quantise_rows(X, store=into, start=0)
            outs.append([row_products(into, c), coverage(into, c), read_rows(into, pick), coverage(into, pick)])
        graphs.append(g)
    X.copy_(y)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    s3 = quantise_rows(y)
    want = [row_products(s3, c), coverage(s3, c), read_rows(s3, pick), coverage(s3, pick)]
    for out in outs:
        assert all(torch.equal(g, w) for g, w in zip(out, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip((graphs[1], graphs[1]), streams[:1]):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[1]):
            r = row_products(into, c)
    torch.cuda.synchronize()
    assert torch.equal(r, want[0]) and all(torch.equal(g, w) for g, w in zip(outs[1], want))


@pytest.mark.parametrize("scale,half", [(1.0, True), (2.0 ** 30, False)])
def test_selection_from_a_store(scale, half):
    """Write, select, take the picks, measure how they cover: the whole use in one run."""
    N, D, k = 3000, 72, 64
    X = torch.from_numpy(gaussian_mixture(N, D, 6, 3)).cuda() * scale
    store = RowStore(N, D)
    for a in range(0, N, 700):
        quantise_rows(X[a : a + 700], store=store)
    matrix = store_matrix(store)
    assert matrix.dtype == (torch.float16 if half else torch.float32)
    assert torch.equal(matrix.double(), read_rows(store).double())
    sel, eps = coresets.fps_cuda(store, k, return_epsilons=True)
    norms = store.norms.cpu().numpy()
    with oracle.element_order(half):
        o_sel, o_eps, o_h, _ = oracle.fps_cuda(read_rows(store).cpu().numpy(), norms, k)
    np.testing.assert_array_equal(sel.cpu().numpy(), o_sel)
    np.testing.assert_array_equal(eps.cpu().numpy().view(np.int32), o_eps.view(np.int32))
    seeded = coresets.fps_cuda(store, k, seed=sel[:5])
    assert torch.equal(seeded, sel)
    h = coverage(store, sel)
    values = f64(read_rows(store))
    off = coverage_bound(values, values[o_sel], D)
    want = ref.coverage(values, values[o_sel])
    assert (np.abs(f64(h) - want) <= off).all()
    assert torch.equal(coverage(store, store.take(sel)), h)
    # the selection's own h (float32, -1 on the picks) says the same of the other rows
    rest = np.setdiff1d(np.arange(N), o_sel)
    assert (np.abs(o_h[rest].astype(np.float64) - f64(h)[rest]) <= 2 * off[rest] + 2 * D * U * 4 * (norms[rest] + norms.max())).all()
    store.check_status()
