"""Embedding heads: ragged products by map, the residual norm, microscaled rows and their products
(smg_group_product*, smg_norm_add*, smg_mx_* of include/smg.h).

All tensors are torch tensors on one CUDA device; the calls run on torch's current stream of that
device and return new tensors.  `off` (int32, groups + 1 entries, on the device) holds the first row
of every map among the packed rows.  Inputs may have any strides: one whose rows the kernels cannot
read (a last stride other than 1, or for the products rows off 16-byte boundaries) is laid out anew
within the call.  error(device) reads the word in which the kernels report bad offsets.  Nothing is
recorded for autograd: inputs that require gradients are refused while torch records them, and the
gradients are calls of their own.

The steps of a call (checks, outputs, the library's call) are C++: csrc/heads_py.cpp, built in-tree
as scenemap_b200/_heads.so over the same libsmg.so that smg.py loads.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import os

import torch

from .smg import LIB_PATH, SmgError, lib

TIMEOUT, BAD_OFFSETS = 1, 2
MAX_GROUPS = 1024
_heads = None


def _lib():
    """The C ABI with its argument types."""
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
    return L


def _load():
    global _heads
    lib()                                            # raises where the library is not built
    C.CDLL(LIB_PATH, mode=C.RTLD_GLOBAL)             # the extension's calls resolve to this library
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_heads.so")
    if not os.path.exists(path):
        raise RuntimeError(f"extension not built: {path} (run __graft_entry__.build())")
    spec = importlib.util.spec_from_file_location("_heads", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.set_error(SmgError)
    _heads = m


def _index(device) -> int:
    device = torch.device(device)
    return torch.cuda.current_device() if device.index is None else device.index


def error(device="cuda") -> int:
    """The device's error word: 0, or TIMEOUT (a wait inside a kernel ran out) and BAD_OFFSETS or'ed.
    Waits for the work on the current stream."""
    return int(_heads.error_word(_index(device)).item())


def failed(device="cuda") -> torch.Tensor:
    """Whether the word is set by what the current stream has queued so far: a bool of one entry on the device, without
    waiting."""
    return _heads.error_word(_index(device)) != 0


def clear_error(device="cuda") -> None:
    _heads.error_word(_index(device)).zero_()


def grouped(x: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[r] = w[g] x[r] for the rows r of group g: x rows x k, w groups x n x k, y rows x n."""
    return _heads.grouped(x, w, off, out_dtype)


def grouped_dx(dy: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for x: dx[r] = w[g]^T dy[r]."""
    return _heads.grouped_dx(dy, w, off, out_dtype)


def grouped_dw(dy: torch.Tensor, x: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for w: dw[g] = sum over the rows of group g of dy[r] x[r]^T (groups x n x k, zeros for
    an empty group)."""
    return _heads.grouped_dw(dy, x, off, out_dtype)


class MxRows:
    """Microscaled rows: codes (..., ceil(k/32)*32*bits/8 bytes) and scales (..., ceil(k/128)*4 bytes), both uint8;
    `values`, where asked for, is what the codes stand for (bf16).  Rows that the library makes lie in
    one buffer, out of which the two tensors are cut when first asked for; a run of them, codes[i:j] and scales[i:j], is a
    bank of its own.  Codes and scales made elsewhere must hold zeros past k and past the last block: a product
    reads them (zero times a scale of 255, NaN, is NaN)."""

    __slots__ = ("_codes", "_scales", "_buf", "_shape", "bits", "k", "values")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bits: int, k: int, values: torch.Tensor | None = None):
        self._codes, self._scales, self.bits, self.k, self.values, self._buf = codes, scales, bits, k, values, None
        if bits not in (4, 8):
            raise SmgError("MxRows: bits must be 4 or 8")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_contiguous() or not scales.is_contiguous():
            raise SmgError("MxRows: codes and scales must be contiguous uint8")
        self._shape = tuple(codes.shape[:-1])
        if k < 1 or codes.shape[-1] != (k + 31) // 32 * 4 * bits or scales.shape != (*self._shape, (k + 127) // 128 * 4):
            raise SmgError(f"MxRows: codes or scales of another shape than {k} values a row need")
        if codes.device != scales.device:
            raise SmgError("MxRows: codes and scales must be on one device")

    @classmethod
    def _of(cls, buf, rows, k, bits, values):
        q = cls.__new__(cls)
        q._codes = q._scales = None
        q._buf, q._shape, q.bits, q.k, q.values = buf, (rows,), bits, k, values
        return q

    def _bytes(self):
        """Bytes of the codes, and of codes and scales."""
        rows = self._shape[0]
        c = rows * ((self.k + 31) // 32 * 4 * self.bits)
        return c, c + rows * ((self.k + 127) // 128 * 4)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buf[:self._bytes()[0]].view(self._shape[0], (self.k + 31) // 32 * 4 * self.bits)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            c, s = self._bytes()
            self._scales = self._buf[c:s].view(self._shape[0], (self.k + 127) // 128 * 4)
        return self._scales

    def _parts(self):
        return (self._codes, self._scales) if self._buf is None else (self._buf, None)

    def dequantise(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for."""
        c, s = self._parts()
        rows = 1
        for d in self._shape:
            rows *= d
        return _heads.mx_values(c, s, rows, self.k, self.bits, dtype).view(*self._shape, self.k)


def mx_quantise(x: torch.Tensor, bits: int, values: bool = False) -> MxRows:
    """Rows in 4 bits (e2m1) or 8 bits (e4m3), a power of two for every 32 values."""
    buf, v = _heads.mx_quantise(x, bits, values)
    rows, k = x.shape
    return MxRows._of(buf, rows, k, bits, v)


def mx_product(a: MxRows, b: MxRows, off: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y[r] = b[g] a[r] of microscaled rows: a rows x k, b (groups x) n x k, y rows x n."""
    if len(a._shape) != 1 or len(b._shape) not in (1, 2):
        raise SmgError("mx_product: a must be rows, b rows or groups of rows")
    if a.bits != b.bits or a.k != b.k:
        raise SmgError("mx_product: a and b must have the same bits and length")
    groups = b._shape[0] if len(b._shape) == 2 else 1
    return _heads.mx_product(*a._parts(), a._shape[0], *b._parts(), groups, b._shape[-1], a.k, a.bits, off, out_dtype)


class NormRows:
    """What norm_add() returns: the sum h, 1 / rms of every row (rstd), the normalised rows in codes (rows, and their
    values), and the inputs that its gradient reads again (they are the caller's own tensors where their rows could be
    read in place: norm_add_backward refuses them once they were changed in place)."""

    __slots__ = ("h", "rows", "x", "residual", "_rstd", "_versions")

    def __init__(self, h, rows, x, residual, versions=-1):
        self.h, self.rows, self.x, self.residual, self._rstd, self._versions = h, rows, x, residual, None, versions

    @property
    def rstd(self) -> torch.Tensor:      # behind codes and scales in their buffer
        if self._rstd is None:
            self._rstd = self.rows._buf[self.rows._bytes()[1]:].view(torch.float32)
        return self._rstd

    @property
    def values(self) -> torch.Tensor | None:
        return self.rows.values


def norm_add(x: torch.Tensor, residual: torch.Tensor | None, gain: torch.Tensor, eps: float = 1e-6, bits: int = 8,
             values: bool = False) -> NormRows:
    """h = x + residual and h / rms(h) * gain in microscaled rows of `bits`."""
    h, buf, v, x, residual, versions = _heads.norm_add(x, residual, gain, eps, bits, values)
    rows, dim = x.shape
    return NormRows(h, MxRows._of(buf, rows, dim, bits, v), x, residual, versions)


def norm_add_backward(dy: torch.Tensor, f: NormRows, gain: torch.Tensor, dh: torch.Tensor | None = None):
    """(dx, dgain) of norm_add(): dx is the gradient for x and for the residual alike; dh is the gradient that reaches
    h past the norm.  The rounding to codes counts as the identity."""
    return _heads.norm_add_backward(dy, f.x, f.residual, f.rows._buf, f.rows._bytes()[1], gain, dh, f._versions)


_load()
