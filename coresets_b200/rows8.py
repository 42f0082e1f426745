"""Rows in 8 bits: a store of e4m3 rows with one power-of-two scale per 128 elements, and what works on it.

    store = quantise_rows(X)                    # write (a whole matrix, or rows behind those it holds)
    X = read_rows(store, rows, dtype=...)       # read rows back
    P = row_products(a, b)                      # dot products of the rows of two stores
    h = coverage(store, centres)                # squared distance of every row to its nearest centre
    selected = fps_cuda(store, k)               # farthest points of the rows as stored

No counterpart in the reference, whose rows have 16 bits at the least (src/coresets/cuda/kernels/warp.cu:167).
An element takes one byte, and a row ``dim + 4 * ceil(dim / 512) + 4`` of them (``dim`` rounded up to 16): a quarter of
float32.  The rounding to e4m3 is off by at most 2^-4 of an element, or 2^-10 of its block's scale; everything behind it works on
the rows as stored, with float32 sums, those of products in the tensor cores' accumulators (see ``row_products``).

Every call is enqueued on the current stream of the store's device, allocates nothing but its result (and a
contiguous copy of an input whose columns are strided, and 20 bytes of scratch per centre of more than 64), synchronises
with nothing and can be captured into a CUDA graph.  Beyond that:

* row numbers that the host holds are checked and copied to the device, for which the host waits: they are refused while the
  stream is capturing;
* ``coverage`` by row numbers first takes these rows into a store of their own;
* ``fps_cuda`` reads the rows back into a matrix (``store_matrix``) and returns when it has selected; ``check_status`` waits.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native
from ._native import CsRows8

BLOCK = 128
MAX_DIM = 65536
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _dtype_code(dtype, what: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return code


def _has_tangent(t: Tensor) -> bool:
    # (no level is open: 0.05 us instead of unpack_dual's 0.7)
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _check_written(t: Tensor, name: str) -> None:
    """A tensor that a call writes to through its address."""
    if t.requires_grad or _has_tangent(t):
        raise ValueError(f"{name} must not require a gradient or carry a tangent (forward mode)")
    if t.is_neg():
        raise ValueError(f"{name} must not be a negated view (Tensor.is_neg)")


# the current stream's handle without building a Stream object (1.3 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """Enqueue the entry point ``name`` on the current stream of ``device``."""
    native, index = _native.get_native(), device.index
    fn = getattr(native.lib, name)
    here = torch.cuda.current_device()
    if here == index:
        rc = fn(*args, _raw_stream(index))
    else:
        torch.cuda.set_device(index)
        try:
            rc = fn(*args, _raw_stream(index))
        finally:
            torch.cuda.set_device(here)
    if rc:
        native._check(rc, name)


class RowStore:
    """Rows of ``dim`` elements in 8 bits, room for ``capacity`` of them, ``count`` (= ``len``) in use.

    ``codes``  float8_e4m3fn [capacity, dim rounded up to 16];
    ``scales`` uint8 [tiles of 128 rows, words, 32, 4, 4]: the exponent byte of block ``4 w + i`` of row
    ``128 t + 32 j + r`` is ``scales[t, w, r, j, i]`` and its value 2^(byte - 127) -- the order in which the tensor
    cores take scales (``exponents`` gives them row by row);
    ``norms``  float32 [capacity], squared norms of the rows as stored."""

    def __init__(self, capacity: int, dim: int, *, device=None):
        capacity, dim = int(capacity), int(dim)
        if capacity < 0 or capacity >= 2 ** 31:
            raise ValueError(f"capacity={capacity} must be in [0, 2^31)")
        if not 1 <= dim <= MAX_DIM:
            raise ValueError(f"dim={dim} must be in [1, {MAX_DIM}]")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"a RowStore lives on a CUDA device, got {device}")
        codes = torch.empty((capacity, (dim + 15) // 16 * 16), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        scales = torch.zeros((-(-capacity // 128), -(-dim // 512), 32, 4, 4), dtype=torch.uint8, device=device)
        norms = torch.empty(capacity, dtype=torch.float32, device=device)
        self._adopt(codes, scales, norms, dim, 0)

    @classmethod
    def from_tensors(cls, codes: Tensor, scales: Tensor, norms: Tensor, dim: int, *, count: Optional[int] = None) -> "RowStore":
        """A store on arrays that are there already (loaded, or another store's); nothing is copied.  All
        contiguous, shaped as the attributes of this class; ``count`` defaults to the capacity.  The codes
        behind ``dim`` have to be 0."""
        dim = int(dim)
        if not 1 <= dim <= MAX_DIM:
            raise ValueError(f"dim={dim} must be in [1, {MAX_DIM}]")
        if codes.dim() != 2 or norms.dim() != 1:
            raise ValueError(f"codes must be 2-D and norms 1-D, got shapes {tuple(codes.shape)} and {tuple(norms.shape)}")
        capacity = codes.shape[0]
        if capacity >= 2 ** 31:
            raise ValueError(f"capacity={capacity} must be in [0, 2^31)")
        want = {"codes": (codes, torch.float8_e4m3fn, (capacity, (dim + 15) // 16 * 16)),
                "scales": (scales, torch.uint8, (-(-capacity // 128), -(-dim // 512), 32, 4, 4)),
                "norms": (norms, torch.float32, (capacity,))}
        for name, (t, dtype, shape) in want.items():
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} of shape {shape}, got {t.dtype} of shape {tuple(t.shape)}")
            if not t.is_cuda or t.device != codes.device:
                raise ValueError(f"{name} must be on one CUDA device with the others, got {t.device}")
            if t.data_ptr() % 16:
                raise ValueError(f"{name} must be 16-byte aligned")
            _check_written(t, name)
        count = capacity if count is None else int(count)
        if not 0 <= count <= capacity:
            raise ValueError(f"count={count} must be in [0, capacity={capacity}]")
        self = cls.__new__(cls)
        self._adopt(codes, scales, norms, dim, count)
        return self

    def _adopt(self, codes, scales, norms, dim, count):
        self._codes, self._scales, self._norms = codes, scales, norms      # (read-only: the library holds their addresses)
        self._written = (codes, scales, norms)
        self.dim, self.capacity, self.device = dim, int(codes.shape[0]), codes.device
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = CsRows8(codes.data_ptr(), scales.data_ptr(), norms.data_ptr(), self._status.data_ptr(),
                          self.capacity, count, dim, 0)
        self._ref = ctypes.byref(self._c)

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    norms = property(lambda self: self._norms)

    @property
    def count(self) -> int:
        return self._c.count

    def __len__(self) -> int:
        return self._c.count

    def __repr__(self) -> str:
        return f"RowStore({self.count} of {self.capacity} rows x {self.dim}, {self.device})"

    @property
    def exponents(self) -> Tensor:
        """uint8 [count, ceil(dim / 128)]: the exponent bytes row by row (a copy)."""
        t, w = self.scales.shape[:2]
        return self.scales.permute(0, 3, 2, 1, 4).reshape(t * 128, w * 4)[: self.count, : -(-self.dim // BLOCK)].contiguous()

    def take(self, rows) -> "RowStore":
        """A new store of the given rows, as they are (an index out of range: see ``read_rows``)."""
        rows = _row_numbers(self, rows)
        out = RowStore(rows.shape[0], self.dim, device=self.device)
        _call(self.device, "cs_rows8_take", self._ref, rows.data_ptr(), rows.shape[0], out._ref, 0)
        out._c.count = rows.shape[0]
        return out

    def check_status(self) -> None:
        """Wait for everything on the device (the calls may have been made on any stream) and raise if a bounded wait
        inside a ``row_products`` or ``coverage`` with this store as its first argument has run out since the last time this
        was asked.  Those calls cannot tell by themselves: they do not wait for what they enqueue."""
        torch.cuda.synchronize(self.device)
        status = int(self._status.item())
        if status:
            self._status.zero_()
            torch.cuda.synchronize(self.device)         # (cleared before another stream may set it)
            raise RuntimeError(f"a bounded wait of a product over {self!r} ran out (status {status}); its result is not valid")


def _row_numbers(store: RowStore, rows) -> Tensor:
    if not isinstance(rows, Tensor):
        rows = torch.as_tensor(rows, device="cpu")       # (whatever the default device: these are checked)
        rows = rows.to(torch.int64) if rows.numel() == 0 else rows
    if rows.dtype == torch.int64 and rows.dim() == 1 and rows.device == store.device and rows.is_contiguous():
        return rows
    if rows.dim() != 1 or rows.dtype.is_floating_point or rows.dtype.is_complex or rows.dtype == torch.bool:
        raise ValueError(f"rows must be a 1-D tensor of whole numbers, got {rows.dtype} of shape {tuple(rows.shape)}")
    if not rows.is_cuda:
        rows = rows.to(torch.int64)                     # (wide unsigned types have no minimum)
        if rows.numel() and not (0 <= int(rows.min()) and int(rows.max()) < store.count):
            raise IndexError(f"rows must be in [0, {store.count}), got {int(rows.min())} .. {int(rows.max())}")
        if rows.numel():
            with torch.cuda.device(store.device):
                if torch.cuda.is_current_stream_capturing():
                    raise ValueError("row numbers on the host cannot be captured into a graph: pass them on the device")
    elif rows.device != store.device:
        raise ValueError(f"rows are on {rows.device}, the store on {store.device}")
    return rows.to(device=store.device, dtype=torch.int64).contiguous()


def _check_store(store, name: str) -> RowStore:
    if not isinstance(store, RowStore):
        raise TypeError(f"{name} must be a RowStore (see quantise_rows), got {type(store).__name__}")
    return store


def quantise_rows(X: Tensor, *, store: Optional[RowStore] = None, start: Optional[int] = None) -> RowStore:
    """Write the rows of ``X`` (float32, float16 or bfloat16, 2-D, on the device) into a store and return it.

    Without ``store`` a new one of exactly these rows.  With it they go to rows ``start .. start + n``
    (default: behind the rows it holds), over what stands there; the store has to have room for them and no
    row before ``start`` may be unwritten.  Per block of 128 elements the scale is 2^e with the least e >= -117
    for which every finite element fits e4m3 (448 at most); elements are rounded to nearest, ties to even.
    NaN and infinities are stored as NaN.  Magnitudes from 248 * 2^120 (3.3e38) to the largest float32 round to 2^128, which
    the store holds but float32 and bfloat16 do not: they are read as infinity.  No gradient flows through."""
    if X.dim() != 2:
        raise ValueError(f"X must be 2-D (N, D), got shape {tuple(X.shape)}")
    if not X.is_cuda:
        raise ValueError(f"X must be on a CUDA device, got {X.device}")
    code = _dtype_code(X.dtype, "X.dtype")
    if X.requires_grad and torch.is_grad_enabled():
        raise ValueError("quantise_rows has no gradient: pass X.detach()")
    if _has_tangent(X):
        raise ValueError("quantise_rows has no forward-mode gradient: pass forward_ad.unpack_dual(X).primal")
    n, dim = X.shape
    if store is None:
        if start:
            raise ValueError("start needs a store")
        store = RowStore(n, dim, device=X.device)
    _check_store(store, "store")
    if dim != store.dim:
        raise ValueError(f"X has {dim} columns, the store {store.dim}")
    if X.device != store.device:
        raise ValueError(f"X is on {X.device}, the store on {store.device}")
    start = store.count if start is None else int(start)
    if not 0 <= start <= store.count:
        raise ValueError(f"start={start} must be in [0, count={store.count}]: a store has no unwritten rows between others")
    if start + n > store.capacity:
        raise ValueError(f"rows {start} .. {start + n} do not fit the store's capacity {store.capacity}")
    if n == 0:
        return store
    if dim == 1:
        X = X.resolve_neg()                 # (z.conj().imag stands for the negative of its memory; wider ones are strided)
    ld, step = X.stride()
    if (dim > 1 and step != 1) or (n > 1 and ld < dim):
        X, ld = X.contiguous(), dim
    _call(store.device, "cs_rows8_write", store._ref, X.data_ptr(), code, n, ld if n > 1 else dim, start)
    increment_version(store._written)       # (autograd cannot know of writes through addresses)
    if start + n > store._c.count:
        store._c.count = start + n
    return store


def _result(out: Optional[Tensor], shape, dtype, like: Tensor) -> Tensor:
    device = like.device
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be {dtype} of shape {tuple(shape)} on {device}, got {out.dtype} of shape {tuple(out.shape)} on {out.device}")
    _check_written(out, "out")
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError(f"out must have rows of consecutive elements that do not overlap, got strides {out.stride()}")
    return out


def read_rows(store: RowStore, rows=None, *, dtype: torch.dtype = torch.float32, out: Optional[Tensor] = None) -> Tensor:
    """Rows of the store as ``dtype`` (exact in float32 and bfloat16 but for 2^128, which is infinity there; rounded once in
    float16).

    ``rows``: whole numbers in any order, repeats allowed; default all rows.  Numbers that the host holds are
    checked (``IndexError``); numbers on the device are not, and one outside ``[0, count)`` gives a row of NaN."""
    _check_store(store, "store")
    code = _dtype_code(dtype, "dtype")
    if rows is not None:
        rows = _row_numbers(store, rows)
    m = store.count if rows is None else rows.shape[0]
    given = out is not None
    out = _result(out, (m, store.dim), dtype, store._norms)
    if m:
        _call(store.device, "cs_rows8_read", store._ref, None if rows is None else rows.data_ptr(), m, out.data_ptr(), code,
              out.stride(0) if m > 1 else store.dim)
        if given:
            increment_version(out)
    return out


def _check_pair(a: RowStore, b: RowStore, names) -> None:
    _check_store(a, names[0])
    _check_store(b, names[1])
    if a.dim != b.dim:
        raise ValueError(f"{names[0]} has rows of {a.dim} elements, {names[1]} of {b.dim}")
    if a.device != b.device:
        raise ValueError(f"{names[0]} is on {a.device}, {names[1]} on {b.device}")


def row_products(a: RowStore, b: RowStore, *, dtype: torch.dtype = torch.float32, out: Optional[Tensor] = None) -> Tensor:
    """``[len(a), len(b)]``: the dot product of every row of ``a`` with every row of ``b``, summed in the tensor cores'
    float32 accumulators and rounded once to ``dtype``.  (Its waits inside the kernel are bounded: ``a.check_status()``.)

    The accumulators cut off (toward zero) instead of rounding, once per 32 elements: each time by less than 2^-23 of the
    sum so far, and terms under 2^-17 of it by less than 2^-25 of it.  So the error of a sum whose terms have one sign has one
    sign too and grows with the width: -1.8e-7 of it at 1024 elements, -1.5e-6 at 4096, -1e-5 at 16384, -6e-5 at 65536 (a float32
    product: 1e-7 at each, of either sign).  With random signs it is 3e-9 of the terms' magnitudes at 1024 (2e-9) and
    5e-8 at 65536 (1e-9)."""
    _check_pair(a, b, ("a", "b"))
    code = _dtype_code(dtype, "dtype")
    n, k = a.count, b.count
    given = out is not None
    out = _result(out, (n, k), dtype, a._norms)
    if n and k:
        _call(a.device, "cs_rows8_products", a._ref, b._ref, out.data_ptr(), code, out.stride(0) if n > 1 else k)
        if given:
            increment_version(out)
    return out


def coverage(store: RowStore, centres, *, h: Optional[Tensor] = None) -> Tensor:
    """float32 ``[len(store)]``: the squared distance of every row to the nearest of ``centres`` (a store, or
    numbers of rows of this one); its maximum is the squared Hausdorff radius of the selection.

    The products behind it are summed as ``row_products`` says, the norms in float32: a distance is off by a share of the
    norms, not of itself.  (Bounded waits: ``store.check_status()``.)

    With ``h`` the minimum is taken with what ``h`` holds, in place: a selection can be passed part by part,
    and rows that carry -1 (selected) keep it; rows that carry a NaN stay NaN.  A distance is never negative, one that is NaN
    never lowers ``h``, and without centres a new ``h`` is +inf."""
    _check_store(store, "store")
    if not isinstance(centres, RowStore):
        centres = store.take(centres)
    _check_pair(store, centres, ("store", "centres"))
    n = store.count
    keep = h is not None
    if keep:
        if h.dtype != torch.float32 or tuple(h.shape) != (n,) or h.device != store.device or not h.is_contiguous():
            raise ValueError(f"h must be contiguous float32 of shape ({n},) on {store.device}, got {h.dtype} of shape {tuple(h.shape)} on {h.device}")
        _check_written(h, "h")
    else:
        h = store._norms.new_empty(n)
    if n:
        size = _native.get_native().lib.cs_rows8_coverage_bytes(centres.count)
        work = store._norms.new_empty(size >> 2) if size else None
        _call(store.device, "cs_rows8_coverage", store._ref, centres._ref, h.data_ptr(), int(keep), work.data_ptr() if size else None)
        if keep:
            increment_version(h)
    return h


def store_matrix(store: RowStore) -> Tensor:
    """The store's rows as a matrix that the selection kernels read, holding exactly the stored values: float16 where
    every exponent lets it (2 bytes an element), float32 otherwise, also where a block of zeros, which carries the least
    exponent, is all that does not.  Reads two numbers back to the host."""
    e = store.exponents
    if e.numel():
        low, high = (int(v) - 127 for v in torch.stack(torch.aminmax(e)).tolist())
        # code * 2^e is a multiple of 2^(e - 9) and at most 448 * 2^e; float16 has multiples of 2^-24 up to 65504
        if low >= -15 and high <= 7:
            return read_rows(store, dtype=torch.float16)
    return read_rows(store, dtype=torch.float32)
