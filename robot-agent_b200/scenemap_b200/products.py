"""Embedding heads: ragged products by map, the residual norm, microscaled rows and their products
(ctypes binding of smg_group_product*, smg_norm_add*, smg_mx_* of include/smg.h).

All tensors are torch tensors on one CUDA device; the calls run on torch's current stream of that
device and return new tensors.  `off` (int32, groups + 1 entries, on the device) holds the first row
of every map among the packed rows.  Inputs may have any strides: one whose rows the kernels cannot
read (a last stride other than 1, or for the products rows off 16-byte boundaries) is laid out anew
within the call.  error(device) reads the word in which the kernels report bad offsets.
"""
from __future__ import annotations

import ctypes as C

import torch

from .smg import SmgError, _check, lib

_ready = None          # the library, once its argument types are set
_words: dict = {}      # error word of each device, and its address
_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HALF = (torch.bfloat16, torch.float16)
TIMEOUT, BAD_OFFSETS = 1, 2
MAX_GROUPS = 1024


def _lib():
    global _ready
    if _ready is None:
        L = lib()
        vp, i, q = C.c_void_p, C.c_int, C.c_int64
        L.smg_group_product.argtypes = [vp, q, vp, q, q, vp, i, i, i, i, i, vp, q, i, vp, vp]
        L.smg_group_product_dx.argtypes = [vp, q, vp, q, q, vp, i, i, i, i, i, vp, q, i, vp, vp]
        L.smg_group_product_dw.argtypes = [vp, q, vp, q, vp, i, i, i, i, i, vp, q, q, i, vp, vp]
        L.smg_mx_quantise.argtypes = [vp, q, i, i, i, i, vp, vp, vp, vp]
        L.smg_mx_values.argtypes = [vp, vp, i, i, i, vp, q, i, vp]
        L.smg_mx_product.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, i, vp, q, i, vp, vp]
        L.smg_norm_add.argtypes = [vp, q, vp, q, vp, i, i, i, C.c_float, vp, q, vp, i, vp, vp, vp, vp]
        L.smg_norm_add_bwd_work.argtypes = [i]
        L.smg_norm_add_bwd_work.restype = q
        L.smg_norm_add_bwd.argtypes = [vp, q, vp, q, vp, q, vp, vp, vp, q, i, i, i, vp, q, vp, vp, vp]
        _ready = L
    return _ready


def _index(device) -> int:
    device = torch.device(device)
    return torch.cuda.current_device() if device.index is None else device.index


def _word(index: int) -> int:
    """Address of the device's error word."""
    w = _words.get(index)
    if w is None:
        t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.synchronize(index)      # zero before any stream's kernel can set it
        w = _words[index] = (t, t.data_ptr())
    return w[1]


def error(device="cuda") -> int:
    """The device's error word: 0, or TIMEOUT (a wait inside a kernel ran out) and BAD_OFFSETS or'ed.
    Waits for the work on the current stream."""
    index = _index(device)
    _word(index)
    return int(_words[index][0].item())


def clear_error(device="cuda") -> None:
    index = _index(device)
    _word(index)
    _words[index][0].zero_()


def _refuse(text: str):
    raise SmgError(text)


# torch.cuda.current_stream() builds a Stream object (3 us); its handle alone is all that is needed here
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on_device(call):
    """Runs the call with its first tensor's device current."""

    def run(first, *args, **kw):
        index = first.get_device()
        if index < 0 or index == torch.cuda.current_device():
            return call(first, *args, **kw)
        with torch.cuda.device(index):
            return call(first, *args, **kw)

    run.__name__, run.__doc__, run.__wrapped__ = call.__name__, call.__doc__, call
    return run


def _same_device(name, index, *tensors) -> None:
    if index < 0:
        _refuse(f"{name}: tensors must be on a CUDA device")
    for t in tensors:
        if t is not None and t.get_device() != index:
            _refuse(f"{name}: all tensors must be on one CUDA device")


def _aligned(t: torch.Tensor):
    """(tensor, leading dimension): rows of a 16-bit matrix on 16-byte boundaries, copied if they are not."""
    rows, k = t.shape
    ld, step = t.stride()
    if rows <= 1:
        ld = (k + 7) & ~7
    if (step == 1 or k == 1) and ld >= k and not ld & 7 and not t.data_ptr() & 15:
        return t, ld
    ld = (k + 7) & ~7
    new = torch.empty((rows, ld), dtype=t.dtype, device=t.device)[:, :k]
    new.copy_(t)
    return new, ld


def _aligned3(w: torch.Tensor):
    """The same for groups of rows: (tensor, leading dimension, group stride)."""
    g, n, k = w.shape
    gs, ld, step = w.stride()
    if n <= 1:
        ld = (k + 7) & ~7
    if g <= 1:
        gs = n * ld
    if (step == 1 or k == 1) and ld >= k and gs >= (n - 1) * ld + k and not (ld | gs) & 7 and not w.data_ptr() & 15:
        return w, ld, gs
    ld = (k + 7) & ~7
    new = torch.empty((g, n, ld), dtype=w.dtype, device=w.device)[..., :k]
    new.copy_(w)
    return new, ld, n * ld


def _plain_rows(t: torch.Tensor):
    """(tensor, leading dimension) with the values of a row next to one another."""
    ld, step = t.stride()
    if step != 1 and t.shape[1] > 1:
        t = t.contiguous()
        ld = t.stride(0)
    return t, ld


def _offsets(name, off, groups, index) -> int:
    """Address of the offsets, 0 for one group of all rows."""
    if off is None:
        if groups != 1:
            _refuse(f"{name}: several groups need offsets")
        return 0
    if off.dtype != torch.int32 or off.shape != (groups + 1,) or not off.is_contiguous():
        _refuse(f"{name}: off must be {groups + 1} int32 values")
    if off.get_device() != index:
        _refuse(f"{name}: off must be on the device of the rows")
    return off.data_ptr()


def _out(name, out_dtype, default):
    t = out_dtype or default
    code = _CODE.get(t)
    if code is None:
        _refuse(f"{name}: bad out_dtype")
    return t, code


@_on_device
def grouped(x: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[r] = w[g] x[r] for the rows r of group g: x rows x k, w groups x n x k, y rows x n."""
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        _refuse("grouped: x must be rows x k and w groups x n x k")
    if x.dtype not in _HALF or w.dtype != x.dtype:
        _refuse("grouped: inputs must both be bf16 or both f16")
    index = x.get_device()
    _same_device("grouped", index, w)
    (rows, k), (groups, n, _) = x.shape, w.shape
    at = _offsets("grouped", off, groups, index)
    t, code = _out("grouped", out_dtype, x.dtype)
    x, ldx = _aligned(x)
    w, ldw, ws = _aligned3(w)
    y = x.new_empty((rows, n), dtype=t)
    _check(_lib().smg_group_product(x.data_ptr(), ldx, w.data_ptr(), ldw, ws, at, groups, rows, n, k, _CODE[x.dtype], y.data_ptr(), n, code,
                                    _word(index), _stream(index)), "smg_group_product")
    return y


@_on_device
def grouped_dx(dy: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for x: dx[r] = w[g]^T dy[r]."""
    if dy.dim() != 2 or w.dim() != 3 or dy.shape[1] != w.shape[1]:
        _refuse("grouped_dx: dy must be rows x n and w groups x n x k")
    if dy.dtype not in _HALF or w.dtype != dy.dtype:
        _refuse("grouped_dx: inputs must both be bf16 or both f16")
    index = dy.get_device()
    _same_device("grouped_dx", index, w)
    (rows, n), (groups, _, k) = dy.shape, w.shape
    at = _offsets("grouped_dx", off, groups, index)
    t, code = _out("grouped_dx", out_dtype, dy.dtype)
    dy, ld = _aligned(dy)
    w, ldw, ws = _aligned3(w)
    dx = dy.new_empty((rows, k), dtype=t)
    _check(_lib().smg_group_product_dx(dy.data_ptr(), ld, w.data_ptr(), ldw, ws, at, groups, rows, n, k, _CODE[dy.dtype], dx.data_ptr(), k,
                                       code, _word(index), _stream(index)), "smg_group_product_dx")
    return dx


@_on_device
def grouped_dw(dy: torch.Tensor, x: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for w: dw[g] = sum over the rows of group g of dy[r] x[r]^T (groups x n x k, zeros for
    an empty group)."""
    if dy.dim() != 2 or x.dim() != 2 or dy.shape[0] != x.shape[0]:
        _refuse("grouped_dw: dy and x must have the same rows")
    if x.dtype not in _HALF or dy.dtype != x.dtype:
        _refuse("grouped_dw: inputs must both be bf16 or both f16")
    index = dy.get_device()
    _same_device("grouped_dw", index, x)
    (rows, n), k = dy.shape, x.shape[1]
    groups = 1 if off is None else off.shape[0] - 1
    at = _offsets("grouped_dw", off, groups, index)
    t, code = _out("grouped_dw", out_dtype, x.dtype)
    dy, lddy = _aligned(dy)
    x, ldx = _aligned(x)
    dw = x.new_empty((groups, n, k), dtype=t)
    _check(_lib().smg_group_product_dw(dy.data_ptr(), lddy, x.data_ptr(), ldx, at, groups, rows, n, k, _CODE[x.dtype], dw.data_ptr(), k, n * k,
                                       code, _word(index), _stream(index)), "smg_group_product_dw")
    return dw


class MxRows:
    """Microscaled rows: codes (..., ceil(k/32)*32*bits/8 bytes) and scales (..., ceil(k/128)*4 bytes), both uint8;
    `values`, where asked for, is what the codes stand for (bf16).  Rows that the library makes lie in
    one buffer, out of which the two tensors are cut when first asked for."""

    __slots__ = ("_codes", "_scales", "_buf", "_shape", "bits", "k", "values")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bits: int, k: int, values: torch.Tensor | None = None):
        self._codes, self._scales, self.bits, self.k, self.values, self._buf = codes, scales, bits, k, values, None
        kb = (k + 31) // 32
        if bits not in (4, 8):
            _refuse("MxRows: bits must be 4 or 8")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_contiguous() or not scales.is_contiguous():
            _refuse("MxRows: codes and scales must be contiguous uint8")
        self._shape = tuple(codes.shape[:-1])
        if k < 1 or codes.shape[-1] != kb * 4 * bits or scales.shape != (*self._shape, (kb + 3) // 4 * 4):
            _refuse(f"MxRows: codes or scales of another shape than {k} values a row need")
        if codes.get_device() != scales.get_device():
            _refuse("MxRows: codes and scales must be on one device")

    @classmethod
    def _new(cls, like: torch.Tensor, bits: int, values: bool, more: int = 0) -> "MxRows":
        """Rows of `like`'s shape; `more` further bytes a row lie behind them in the buffer."""
        q = cls.__new__(cls)
        rows, k = like.shape
        kb = (k + 31) // 32
        q._codes = q._scales = None
        q._shape, q.bits, q.k = (rows,), bits, k
        q._buf = like.new_empty(rows * (kb * 4 * bits + (kb + 3) // 4 * 4 + more), dtype=torch.uint8)
        q.values = like.new_empty((rows, k), dtype=torch.bfloat16) if values else None
        return q

    def _code_bytes(self) -> int:
        return self._shape[0] * ((self.k + 31) // 32 * 4 * self.bits)

    def _bytes(self) -> int:
        return self._code_bytes() + self._shape[0] * ((self.k + 127) // 128 * 4)

    def _address(self):
        """(codes, scales)"""
        if self._buf is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        p = self._buf.data_ptr()
        return p, p + self._code_bytes()

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buf[:self._code_bytes()].view(self._shape[0], (self.k + 31) // 32 * 4 * self.bits)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buf[self._code_bytes():self._bytes()].view(self._shape[0], (self.k + 127) // 128 * 4)
        return self._scales

    @property
    def _any(self) -> torch.Tensor:
        return self._codes if self._buf is None else self._buf

    def dequantise(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for."""
        return _dequantise(self._any, self, dtype)


@_on_device
def _dequantise(t: torch.Tensor, q: MxRows, dtype: torch.dtype) -> torch.Tensor:
    _, code = _out("dequantise", dtype, None)
    _same_device("dequantise", t.get_device())
    out = t.new_empty((*q._shape, q.k), dtype=dtype)
    codes, scales = q._address()
    _check(_lib().smg_mx_values(codes, scales, out.numel() // q.k, q.k, q.bits, out.data_ptr(), q.k, code, _stream(t.get_device())),
           "smg_mx_values")
    return out


@_on_device
def mx_quantise(x: torch.Tensor, bits: int, values: bool = False) -> MxRows:
    """Rows in 4 bits (e2m1) or 8 bits (e4m3), a power of two for every 32 values."""
    if x.dim() != 2 or x.dtype not in _CODE or x.shape[1] < 1:
        _refuse("mx_quantise: x must be rows x k of f32, bf16 or f16")
    if bits not in (4, 8):
        _refuse("mx_quantise: bits must be 4 or 8")
    index = x.get_device()
    _same_device("mx_quantise", index)
    rows, k = x.shape
    x, ld = _plain_rows(x)
    q = MxRows._new(x, bits, values)
    codes, scales = q._address()
    _check(_lib().smg_mx_quantise(x.data_ptr(), ld, rows, k, _CODE[x.dtype], bits, codes, scales, q.values.data_ptr() if values else 0,
                                  _stream(index)), "smg_mx_quantise")
    return q


def mx_product(a: MxRows, b: MxRows, off: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y[r] = b[g] a[r] of microscaled rows: a rows x k, b (groups x) n x k, y rows x n."""
    return _mx_product(a._any, a, b, off, out_dtype)


@_on_device
def _mx_product(t, a, b, off, out_dtype):
    if len(a._shape) != 1 or len(b._shape) not in (1, 2):
        _refuse("mx_product: a must be rows, b rows or groups of rows")
    if a.bits != b.bits or a.k != b.k:
        _refuse("mx_product: a and b must have the same bits and length")
    index = t.get_device()
    _same_device("mx_product", index, b._any)
    rows, n = a._shape[0], b._shape[-1]
    groups = b._shape[0] if len(b._shape) == 2 else 1
    at = _offsets("mx_product", off, groups, index)
    _, code = _out("mx_product", out_dtype, None)
    y = t.new_empty((rows, n), dtype=out_dtype)
    (ac, asc), (bc, bsc) = a._address(), b._address()
    _check(_lib().smg_mx_product(ac, asc, bc, bsc, at, groups, rows, n, a.k, a.bits, y.data_ptr(), n, code, _word(index), _stream(index)),
           "smg_mx_product")
    return y


class NormRows:
    """What norm_add() returns: the sum h, 1 / rms of every row (rstd), the normalised rows in codes (rows, and their
    values), and the inputs that its gradient reads again."""

    __slots__ = ("h", "rows", "x", "residual", "_rstd")

    def __init__(self, h, rows, x, residual):
        self.h, self.rows, self.x, self.residual, self._rstd = h, rows, x, residual, None

    @property
    def rstd(self) -> torch.Tensor:
        if self._rstd is None:
            self._rstd = self.rows._buf[self.rows._bytes():].view(torch.float32)
        return self._rstd

    @property
    def values(self) -> torch.Tensor | None:
        return self.rows.values


def _gain(name, gain, x):
    if gain.dtype != torch.float32 or gain.shape != x.shape[1:] or not gain.is_contiguous():
        _refuse(f"{name}: gain must be dim float32 values")


@_on_device
def norm_add(x: torch.Tensor, residual: torch.Tensor | None, gain: torch.Tensor, eps: float = 1e-6, bits: int = 8,
             values: bool = False) -> NormRows:
    """h = x + residual and h / rms(h) * gain in microscaled rows of `bits`."""
    if x.dim() != 2 or x.dtype not in _CODE or x.shape[1] < 1:
        _refuse("norm_add: x must be rows x dim of f32, bf16 or f16")
    if bits not in (4, 8):
        _refuse("norm_add: bits must be 4 or 8")
    _gain("norm_add", gain, x)
    index = x.get_device()
    _same_device("norm_add", index, gain, residual)
    rows, dim = x.shape
    x, ldx = _plain_rows(x)
    ptr, ldr = 0, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            _refuse("norm_add: the residual must be like x")
        residual, ldr = _plain_rows(residual)
        ptr = residual.data_ptr()
    h = x.new_empty((rows, dim))
    q = MxRows._new(x, bits, values, 4)      # and 1 / rms, 4 bytes a row
    codes, scales = q._address()
    _check(_lib().smg_norm_add(x.data_ptr(), ldx, ptr, ldr, gain.data_ptr(), rows, dim, _CODE[x.dtype], eps, h.data_ptr(), dim,
                               codes + q._bytes(), bits, codes, scales, q.values.data_ptr() if values else 0, _stream(index)), "smg_norm_add")
    return NormRows(h, q, x, residual)


@_on_device
def norm_add_backward(dy: torch.Tensor, f: NormRows, gain: torch.Tensor, dh: torch.Tensor | None = None):
    """(dx, dgain) of norm_add(): dx is the gradient for x and for the residual alike; dh is the gradient that reaches
    h past the norm.  The rounding to codes counts as the identity."""
    x, r = f.x, f.residual
    if dy.shape != x.shape or dy.dtype != x.dtype:
        _refuse("norm_add_backward: dy must be like x")
    if dh is not None and (dh.shape != x.shape or dh.dtype != x.dtype):
        _refuse("norm_add_backward: dh must be like x")
    _gain("norm_add_backward", gain, x)
    index = dy.get_device()
    _same_device("norm_add_backward", index, x, gain, dh)
    rows, dim = x.shape
    dy, lddy = _plain_rows(dy)
    pr, ldr, pd, ldd = 0, 0, 0, 0
    if r is not None:
        pr, ldr = r.data_ptr(), r.stride(0)
    if dh is not None:
        dh, ldd = _plain_rows(dh)
        pd = dh.data_ptr()
    dx = x.new_empty((rows, dim))
    dgain = x.new_empty(dim, dtype=torch.float32)
    L = _lib()
    work = x.new_empty(L.smg_norm_add_bwd_work(dim), dtype=torch.uint8)
    _check(L.smg_norm_add_bwd(dy.data_ptr(), lddy, x.data_ptr(), x.stride(0), pr, ldr, f.rows._address()[0] + f.rows._bytes(), gain.data_ptr(), pd, ldd, rows,
                              dim, _CODE[x.dtype], dx.data_ptr(), dim, dgain.data_ptr(), work.data_ptr(), _stream(index)), "smg_norm_add_bwd")
    return dx, dgain
