"""Rows in 8 bits, what needs no GPU: the oracle's own pins, refusals of the Python layer and of the C ABI."""
import ctypes

import numpy as np
import pytest
import torch

import coresets_b200 as coresets
from coresets_b200 import _native, build
from coresets_b200.rows8 import _row_numbers
from tests import rows8_oracle as ref


def test_oracle_code_values_are_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    np.testing.assert_array_equal(codes, ref.code_values())


def test_oracle_rounds_like_the_type():
    x = np.random.default_rng(0).standard_normal((9, 300)).astype(np.float32)
    codes, exps, rows, norms = ref.quantise(x.astype(np.float64))
    scale = np.exp2(np.repeat(exps, 128, axis=1)[:, :300] - 127.0).astype(np.float32)
    want = torch.from_numpy(x / scale).to(torch.float8_e4m3fn).to(torch.float64).numpy()
    np.testing.assert_array_equal(codes, want)
    top = np.abs(np.pad(x, ((0, 0), (0, 84)))).reshape(9, 3, 128).max(2)
    e = exps - 127.0
    assert (top <= 448 * np.exp2(e)).all() and (top > 448 * np.exp2(e - 1)).all()
    # half a step of e4m3 relative, or half its smallest number times the scale
    assert (np.abs(rows - x) <= np.maximum(np.abs(x) * 2.0 ** -4, scale * 2.0 ** -10)).all()


def test_host_refusals():
    with pytest.raises(ValueError, match="CUDA device"):
        coresets.quantise_rows(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="2-D"):
        coresets.quantise_rows(torch.zeros(3))
    with pytest.raises(ValueError, match="CUDA device"):
        coresets.RowStore(4, 4, device="cpu")
    for capacity, dim in ((-1, 4), (4, 0), (2 ** 31, 4), (4, 65537)):
        with pytest.raises(ValueError):
            coresets.RowStore(capacity, dim)
    with pytest.raises(ValueError):
        coresets.RowStore.from_tensors(torch.zeros(4, 16, dtype=torch.uint8).view(torch.float8_e4m3fn),
                                       torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), torch.zeros(4), 16)
    for call in (coresets.read_rows, lambda x: coresets.row_products(x, x), lambda x: coresets.coverage(x, [0])):
        with pytest.raises(TypeError, match="RowStore"):
            call(torch.zeros(3, 4))


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _native.Native().lib


def _store(**kw):
    v = dict(codes=4096, scales=8192, norms=12288, status=None, capacity=100, count=50, dim=64, flags=0)
    v.update(kw)
    return _native.CsRows8(*v.values())


def test_c_abi_struct():
    assert ctypes.sizeof(_native.CsRows8) == 56 and _native.CsRows8.dim.offset == 48


def test_c_abi_refusals(lib):
    """Bad arguments are turned down before anything touches a device."""
    ARG, ALIGN, RANGE = -1, -2, -3
    r, p = ctypes.byref, 16384
    good = _store()
    for bad, code in ((_store(dim=0), ARG), (_store(codes=None), ARG), (_store(count=101), ARG), (_store(capacity=-1, count=-1), ARG), (_store(flags=1), ARG),
                      (_store(norms=12290), ALIGN), (_store(scales=8200), ALIGN), (_store(capacity=2 ** 31), RANGE), (_store(dim=65537), RANGE)):
        assert lib.cs_rows8_write(r(bad), p, 0, 1, 64, 0, None) == code
        assert lib.cs_rows8_read(r(bad), p, 1, p, 0, 64, None) == code
        assert lib.cs_rows8_take(r(bad), p, 1, r(good), 0, None) == code
        assert lib.cs_rows8_products(r(good), r(bad), p, 0, 64, None) == code
        assert lib.cs_rows8_coverage(r(bad), r(good), p, 0, p, None) == code
    assert lib.cs_rows8_write(None, p, 0, 1, 64, 0, None) == ARG
    for args in ((p, 3, 1, 64, 0), (p, 0, -1, 64, 0), (None, 0, 1, 64, 0), (p, 0, 2, 63, 0), (p, 0, 1, 64, 100), (p, 0, 51, 64, 50), (p, 0, 1, 64, -1),
                 (p, 0, 2 ** 62, 64, 2)):
        assert lib.cs_rows8_write(r(good), *args, None) == ARG, args
    for args in ((None, 51, p, 0, 64), (p, 2, p, 0, 60), (p, 1, None, 0, 64), (p, -1, p, 0, 64), (p, 1, p, 9, 64)):
        assert lib.cs_rows8_read(r(good), *args, None) == ARG, args
    other = _store(codes=40960, scales=81920, dim=65)
    assert lib.cs_rows8_take(r(good), p, 1, r(other), 0, None) == ARG
    assert lib.cs_rows8_take(r(good), p, 1, r(good), 60, None) == ARG          # onto itself
    assert lib.cs_rows8_products(r(good), r(other), p, 0, 64, None) == ARG
    assert lib.cs_rows8_products(r(good), r(good), p, 0, 49, None) == ARG
    assert lib.cs_rows8_products(r(good), r(good), p + 2, 0, 50, None) == ALIGN
    assert lib.cs_rows8_coverage(r(good), r(good), None, 0, None, None) == ARG
    assert lib.cs_rows8_coverage(r(good), r(good), p + 2, 0, None, None) == ALIGN
    many = _store(codes=40960, scales=81920, count=100)
    assert lib.cs_rows8_coverage_bytes(64) == 0 and lib.cs_rows8_coverage_bytes(100) >= 20 * 100 and lib.cs_rows8_coverage_bytes(-1) == ARG
    assert lib.cs_rows8_coverage(r(good), r(_store(capacity=2 ** 30, count=2 ** 30)), p, 0, p, None) == RANGE
    # nothing to do
    none = _store(count=0)
    assert lib.cs_rows8_write(r(good), None, 0, 0, 64, 100, None) == 0
    assert lib.cs_rows8_read(r(none), None, 0, None, 0, 64, None) == 0
    assert lib.cs_rows8_products(r(none), r(good), None, 0, 50, None) == 0
    assert lib.cs_rows8_coverage(r(none), r(good), None, 0, None, None) == 0


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32, torch.uint64])
def test_row_numbers_out_of_range_of_every_type(dtype):
    store = type("Store", (), {"device": torch.device("cuda", 0), "count": 50})()
    for bad in ([3, 50], [100]):
        with pytest.raises(IndexError, match=r"\[0, 50\)"):
            _row_numbers(store, torch.tensor(bad).to(dtype))
        with pytest.raises(IndexError, match=r"\[0, 50\)"):
            _row_numbers(store, np.array(bad).astype(str(dtype).split(".")[1]))


def test_row_numbers_of_a_list_are_the_hosts_under_another_default_device():
    store = type("Store", (), {"device": torch.device("cuda", 0), "count": 50})()
    with torch.device("meta"), pytest.raises(IndexError, match="50 .. 50"):
        _row_numbers(store, [50])
