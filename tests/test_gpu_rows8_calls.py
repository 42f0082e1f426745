"""Rows in 8 bits: what a call does to what surrounds it (autograd, other streams, captured graphs, the status word)."""
import pytest
import torch
from torch.autograd import forward_ad

from coresets_b200 import RowStore, _native, coverage, quantise_rows, read_rows, row_products
from tests import rows8_exact as ex

pytestmark = pytest.mark.gpu


def stored(n, dim, seed=0):
    x = ex.whole_rows(n, dim, seed)
    return quantise_rows(x), x


@pytest.mark.parametrize("k", [0, 5, 33, 64, 65, 700])
def test_a_nan_in_h_stays(k):
    """A NaN of either sign, as torch.minimum leaves it; whatever the number of centres."""
    (a, x), (c, y) = stored(1000, 70, 1), stored(700, 70, 2)
    c = c.take(torch.arange(k))
    h = torch.full((1000,), float("inf"), device="cuda")
    h[::9] = float("nan")
    h.view(torch.int32)[3::9] = -1                        # a NaN with its sign bit set
    h[5::9] = -1.0
    want = torch.minimum(h.double(), ex.distances(x, y[:k]) if k else torch.full((1000,), float("inf"), device="cuda", dtype=torch.float64))
    nan = h.isnan()
    assert int(nan.sum()) > 200
    coverage(a, c, h=h)
    assert torch.equal(h.isnan(), nan) and torch.equal(h[~nan].double(), want[~nan])
    # nor does a row without any distance (NaN itself) lose it
    z = a.take(torch.full((1000,), -1, device="cuda"))
    coverage(z, c, h=h)
    assert torch.equal(h.isnan(), nan) and torch.equal(h[~nan].double(), want[~nan])


def test_writes_move_the_version_counter():
    """A graph that saved a tensor which a call then wrote to must not be differentiated with the new values."""
    (a, x), (c, _) = stored(300, 40, 1), stored(20, 40, 2)

    def saved(t):
        w = torch.ones_like(t, requires_grad=True)
        return (w * t).sum()
    h, wide = torch.zeros(300, device="cuda"), torch.zeros(300, 60, device="cuda")
    for t, call in ((h, lambda: coverage(a, c, h=h)), (wide, lambda: read_rows(a, out=wide[:, 3:43])),
                    (wide, lambda: row_products(a, c, out=wide[:, :20])), (a.norms, lambda: quantise_rows(x, store=a, start=0))):
        y, before = saved(t), t._version
        call()
        assert t._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    codes, scales = a.codes._version, a.scales._version
    quantise_rows(x[:1], store=a, start=0)
    assert a.codes._version > codes and a.scales._version > scales
    with torch.inference_mode():                          # (such tensors have no counter)
        t = torch.zeros(300, device="cuda")
    assert torch.equal(coverage(a, c, h=t), torch.zeros(300, device="cuda"))


def test_tangents_are_refused():
    (a, x), (c, _) = stored(30, 40, 1), stored(5, 40, 2)
    h, out = torch.zeros(30, device="cuda"), torch.zeros(30, 40, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="gradient"):
            quantise_rows(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="gradient"):
            coverage(a, c, h=forward_ad.make_dual(h, torch.ones_like(h)))
        with pytest.raises(ValueError, match="gradient"):
            read_rows(a, out=forward_ad.make_dual(out, torch.ones_like(out)))
        with pytest.raises(ValueError, match="gradient"):
            RowStore.from_tensors(a.codes, a.scales, forward_ad.make_dual(a.norms, torch.ones_like(a.norms)), 40)
        assert torch.equal(read_rows(quantise_rows(x)), x)
    with pytest.raises(ValueError, match="gradient"):
        RowStore.from_tensors(a.codes, a.scales, a.norms.clone().requires_grad_(), 40)


def test_negated_views():
    """A view that stands for the negative of its memory is read as that, and not written to."""
    z = torch.complex(torch.arange(40.0), torch.arange(1.0, 41.0)).cuda()[:, None]
    x = z.conj().imag
    assert x.is_neg()
    assert torch.equal(read_rows(quantise_rows(x)), read_rows(quantise_rows(x.clone())))
    z2 = torch.complex(torch.ones(20, 6), torch.arange(120.0).view(20, 6)).cuda()
    for wide in (z2.conj().imag, z2[:1].conj().imag, z2[:, :1].expand(20, 6).conj().imag):
        assert wide.is_neg() and torch.equal(read_rows(quantise_rows(wide)), read_rows(quantise_rows(wide.clone())))
    with pytest.raises(ValueError, match="negated"):
        read_rows(quantise_rows(x.clone()), out=z.conj().imag)
    with pytest.raises(ValueError, match="negated"):
        coverage(quantise_rows(x[:1].clone()), [0], h=torch._neg_view(torch.zeros(1, device="cuda")))


@pytest.mark.parametrize("n,k", [(300, 5), (300, 200)])
def test_the_status_is_reported_once(n, k):
    """Also of a call on another stream than the one that asks."""
    (a, x), (c, y) = stored(n, 300, 1), stored(k, 300, 2)
    side = torch.cuda.Stream()
    for call in (row_products, coverage):
        torch.cuda.synchronize()
        a._c.flags = c._c.flags = _native.ROWS8_TEST_STALL
        with torch.cuda.stream(side):
            call(a, c)
        a._c.flags = c._c.flags = 0
        with pytest.raises(RuntimeError, match="ran out"):
            a.check_status()
        a.check_status()
        assert torch.equal(coverage(a, c).double(), ex.distances(x, y))
        a.check_status()


def test_row_numbers_of_the_host_are_refused_while_capturing():
    (a, x), (c, _) = stored(300, 40, 1), stored(70, 40, 2)
    pick = torch.tensor([5, 299, 0], device="cuda")
    coverage(a, pick)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for call in (lambda: read_rows(a, [5, 299, 0]), lambda: a.take(torch.tensor([5])), lambda: coverage(a, [5])):
            with pytest.raises(ValueError, match="captur"):
                call()
        got = read_rows(a, pick)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, x[pick])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.uint16, torch.uint32, torch.uint64])
def test_row_numbers_of_every_type(dtype):
    a, x = stored(250, 40, 1)
    pick = torch.tensor([5, 249, 0])
    assert torch.equal(read_rows(a, pick.to(dtype)), x[pick.cuda()])
    assert torch.equal(read_rows(a, pick.to(dtype).cuda()), x[pick.cuda()])
    with pytest.raises(IndexError):
        read_rows(a, torch.tensor([5, 250]).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_numbers_are_stored_as_two_to_the_128(dtype):
    """248 * 2^120 and more round to 256 * 2^120, which float32 and bfloat16 do not have."""
    top = 2.0 ** 120
    x = torch.zeros(4, 200, dtype=torch.float64)
    x[0, 0], x[1, 0], x[2, 150], x[3, 7] = 247 * top, -248 * top, torch.finfo(dtype).max, 240 * top
    x = x.to(dtype)
    a = quantise_rows(x.cuda())
    assert torch.isfinite(x).all() and not a.codes.float().isnan().any()
    for out in (torch.float32, torch.bfloat16):
        got = read_rows(a, dtype=out).double().cpu()
        assert got[3, 7] == 240 * top and got[2, 150] == float("inf") and not got.isnan().any()
        assert got[0, 0] == (240 * top if x[0, 0].double() < 248 * top else float("inf")) and got[1, 0] == float("-inf")


def test_graphs_and_calls_at_once():
    """Two graphs, each with a coverage of its own (scratch of other norms), replayed on two streams at the same time, beside eager calls."""
    (a, x), (c, y), (e, z) = stored(20000, 200, 1), stored(600, 200, 2), stored(900, 200, 3)
    e2 = RowStore.from_tensors(e.codes, e.scales, e.norms, 200, count=431)
    pick = torch.arange(0, 20000, 97, device="cuda")
    want = [ex.distances(x, y), ex.distances(x, z), ex.distances(x, x[pick]), ex.distances(x, z[:431])]
    calls = [lambda: coverage(a, c), lambda: coverage(a, e), lambda: coverage(a, pick), lambda: coverage(a, e2)]
    for call in calls:
        call()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([calls[i](), calls[i + 2]()])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(8):
        for out in outs:
            for t in out:
                t.fill_(-5.0)
        torch.cuda.synchronize()
        eager = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
            with torch.cuda.stream(streams[2 + i]):
                eager.append((calls[i](), calls[i + 2]()))
        torch.cuda.synchronize()
        for i in range(2):
            for got in (outs[i], eager[i]):
                assert torch.equal(got[0].double(), want[i]) and torch.equal(got[1].double(), want[i + 2])
    a.check_status()
