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
from dataclasses import dataclass

import torch

from .smg import SmgError, _check, lib

_ready = False
_words: dict = {}      # error word of each device
_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
TIMEOUT, BAD_OFFSETS = 1, 2
MAX_GROUPS = 1024


def _lib():
    global _ready
    L = lib()
    if not _ready:
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
        _ready = True
    return L


def _call(fn, *args):
    _check(fn(*args), fn.__name__)


def _word(device) -> torch.Tensor:
    w = _words.get(device.index)
    if w is None:
        w = _words[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
    return w


def error(device="cuda") -> int:
    """The device's error word: 0, or TIMEOUT (a wait inside a kernel ran out) and BAD_OFFSETS or'ed.
    Waits for the work on the current stream."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return int(_word(device).item())


def clear_error(device="cuda") -> None:
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    _word(device).zero_()


class _on:
    """Makes the tensor's device current where it is not."""

    def __init__(self, t):
        self.index, self.back = t.device.index, None

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.index:
            self.back = now
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *_):
        if self.back is not None:
            torch.cuda.set_device(self.back)


def _want(ok: bool, text: str) -> None:
    if not ok:
        raise SmgError(text)


def _cuda(name: str, *tensors) -> None:
    first = tensors[0]
    for t in tensors:
        _want(t.is_cuda and t.device == first.device, f"{name}: all tensors must be on one CUDA device")


def _aligned(t: torch.Tensor):
    """(tensor, leading dimension): rows of a 16-bit matrix on 16-byte boundaries, copied if they are not."""
    rows, k = t.shape
    ld = t.stride(0) if rows > 1 else (k + 7) & ~7
    if (t.stride(1) == 1 or k == 1) and ld >= k and not ld & 7 and not t.data_ptr() & 15:
        return t, ld
    ld = (k + 7) & ~7
    new = torch.empty((rows, ld), dtype=t.dtype, device=t.device)[:, :k]
    new.copy_(t)
    return new, ld


def _aligned3(w: torch.Tensor):
    """The same for groups of rows: (tensor, leading dimension, group stride)."""
    g, n, k = w.shape
    ld = w.stride(1) if n > 1 else (k + 7) & ~7
    gs = w.stride(0) if g > 1 else n * ld
    if (w.stride(2) == 1 or k == 1) and ld >= k and gs >= (n - 1) * ld + k and not (ld | gs) & 7 and not w.data_ptr() & 15:
        return w, ld, gs
    ld = (k + 7) & ~7
    new = torch.empty((g, n, ld), dtype=w.dtype, device=w.device)[..., :k]
    new.copy_(w)
    return new, ld, n * ld


def _plain_rows(t: torch.Tensor):
    """(tensor, leading dimension) with the values of a row next to one another."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _offsets(name, off, groups, x):
    if off is None:
        _want(groups == 1, f"{name}: several groups need offsets")
        return 0
    _want(off.dtype == torch.int32 and off.dim() == 1 and off.shape[0] == groups + 1 and off.is_contiguous(),
          f"{name}: off must be {groups + 1} int32 values")
    _want(off.device == x.device, f"{name}: off must be on the device of the rows")
    return off.data_ptr()


def _two(name, a, b):
    _want(a.dtype == b.dtype and a.dtype in (torch.bfloat16, torch.float16), f"{name}: inputs must both be bf16 or both f16")


def grouped(x: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[r] = w[g] x[r] for the rows r of group g: x rows x k, w groups x n x k, y rows x n."""
    _want(x.dim() == 2 and w.dim() == 3 and x.shape[1] == w.shape[2], "grouped: x must be rows x k and w groups x n x k")
    _two("grouped", x, w)
    _cuda("grouped", x, w)
    (rows, k), (groups, n, _) = x.shape, w.shape
    at = _offsets("grouped", off, groups, x)
    out = out_dtype or x.dtype
    _want(out in _CODE, "grouped: bad out_dtype")
    with _on(x) as stream:
        x, ldx = _aligned(x)
        w, ldw, ws = _aligned3(w)
        y = torch.empty((rows, n), dtype=out, device=x.device)
        _call(_lib().smg_group_product, x.data_ptr(), ldx, w.data_ptr(), ldw, ws, at, groups, rows, n, k, _CODE[x.dtype],
              y.data_ptr(), n, _CODE[out], _word(x.device).data_ptr(), stream)
    return y


def grouped_dx(dy: torch.Tensor, w: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for x: dx[r] = w[g]^T dy[r]."""
    _want(dy.dim() == 2 and w.dim() == 3 and dy.shape[1] == w.shape[1], "grouped_dx: dy must be rows x n and w groups x n x k")
    _two("grouped_dx", dy, w)
    _cuda("grouped_dx", dy, w)
    (rows, n), (groups, _, k) = dy.shape, w.shape
    at = _offsets("grouped_dx", off, groups, dy)
    out = out_dtype or dy.dtype
    _want(out in _CODE, "grouped_dx: bad out_dtype")
    with _on(dy) as stream:
        dy, ld = _aligned(dy)
        w, ldw, ws = _aligned3(w)
        dx = torch.empty((rows, k), dtype=out, device=dy.device)
        _call(_lib().smg_group_product_dx, dy.data_ptr(), ld, w.data_ptr(), ldw, ws, at, groups, rows, n, k, _CODE[dy.dtype],
              dx.data_ptr(), k, _CODE[out], _word(dy.device).data_ptr(), stream)
    return dx


def grouped_dw(dy: torch.Tensor, x: torch.Tensor, off: torch.Tensor | None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of grouped() for w: dw[g] = sum over the rows of group g of dy[r] x[r]^T (groups x n x k, zeros for
    an empty group)."""
    _want(dy.dim() == 2 and x.dim() == 2 and dy.shape[0] == x.shape[0], "grouped_dw: dy and x must have the same rows")
    _two("grouped_dw", dy, x)
    _cuda("grouped_dw", dy, x)
    (rows, n), k = dy.shape, x.shape[1]
    groups = 1 if off is None else off.shape[0] - 1
    at = _offsets("grouped_dw", off, groups, x)
    out = out_dtype or x.dtype
    _want(out in _CODE, "grouped_dw: bad out_dtype")
    with _on(x) as stream:
        dy, lddy = _aligned(dy)
        x, ldx = _aligned(x)
        dw = torch.empty((groups, n, k), dtype=out, device=x.device)
        _call(_lib().smg_group_product_dw, dy.data_ptr(), lddy, x.data_ptr(), ldx, at, groups, rows, n, k, _CODE[x.dtype],
              dw.data_ptr(), k, n * k, _CODE[out], _word(x.device).data_ptr(), stream)
    return dw


@dataclass
class MxRows:
    """Microscaled rows: codes (..., ceil(k/32)*32*bits/8 bytes) and scales (..., ceil(k/128)*4 bytes), both uint8;
    `values`, where asked for, is what the codes stand for (bf16)."""
    codes: torch.Tensor
    scales: torch.Tensor
    bits: int
    k: int
    values: torch.Tensor | None = None

    def check(self, name):
        kb = (self.k + 31) // 32
        _want(self.bits in (4, 8), f"{name}: bits must be 4 or 8")
        _want(self.codes.dtype == torch.uint8 and self.scales.dtype == torch.uint8 and self.codes.is_contiguous()
              and self.scales.is_contiguous(), f"{name}: codes and scales must be contiguous uint8")
        _want(self.codes.shape[-1] == kb * 4 * self.bits and self.scales.shape[-1] == (kb + 3) // 4 * 4
              and self.codes.shape[:-1] == self.scales.shape[:-1], f"{name}: codes or scales of another shape than {self.k} values a row need")

    def dequantise(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for."""
        self.check("dequantise")
        _cuda("dequantise", self.codes, self.scales)
        _want(dtype in _CODE, "dequantise: bad dtype")
        rows = self.codes.numel() // self.codes.shape[-1]
        with _on(self.codes) as stream:
            out = torch.empty((*self.codes.shape[:-1], self.k), dtype=dtype, device=self.codes.device)
            _call(_lib().smg_mx_values, self.codes.data_ptr(), self.scales.data_ptr(), rows, self.k, self.bits, out.data_ptr(), self.k,
                  _CODE[dtype], stream)
        return out


def _mx_empty(rows, k, bits, values, device):
    kb = (k + 31) // 32
    return MxRows(torch.empty((rows, kb * 4 * bits), dtype=torch.uint8, device=device),
                  torch.empty((rows, (kb + 3) // 4 * 4), dtype=torch.uint8, device=device), bits, k,
                  torch.empty((rows, k), dtype=torch.bfloat16, device=device) if values else None)


def mx_quantise(x: torch.Tensor, bits: int, values: bool = False) -> MxRows:
    """Rows in 4 bits (e2m1) or 8 bits (e4m3), a power of two for every 32 values."""
    _want(x.dim() == 2 and x.dtype in _CODE and x.shape[1] > 0, "mx_quantise: x must be rows x k of f32, bf16 or f16")
    _want(bits in (4, 8), "mx_quantise: bits must be 4 or 8")
    _cuda("mx_quantise", x)
    rows, k = x.shape
    with _on(x) as stream:
        x, ld = _plain_rows(x)
        q = _mx_empty(rows, k, bits, values, x.device)
        _call(_lib().smg_mx_quantise, x.data_ptr(), ld, rows, k, _CODE[x.dtype], bits, q.codes.data_ptr(), q.scales.data_ptr(),
              q.values.data_ptr() if values else 0, stream)
    return q


def mx_product(a: MxRows, b: MxRows, off: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y[r] = b[g] a[r] of microscaled rows: a rows x k, b (groups x) n x k, y rows x n."""
    a.check("mx_product")
    b.check("mx_product")
    _want(a.codes.dim() == 2 and b.codes.dim() in (2, 3), "mx_product: a must be rows, b rows or groups of rows")
    _want(a.bits == b.bits and a.k == b.k, "mx_product: a and b must have the same bits and length")
    _cuda("mx_product", a.codes, a.scales, b.codes, b.scales)
    _want(out_dtype in _CODE, "mx_product: bad out_dtype")
    rows, n = a.codes.shape[0], b.codes.shape[-2]
    groups = b.codes.shape[0] if b.codes.dim() == 3 else 1
    at = _offsets("mx_product", off, groups, a.codes)
    with _on(a.codes) as stream:
        y = torch.empty((rows, n), dtype=out_dtype, device=a.codes.device)
        _call(_lib().smg_mx_product, a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(), at, groups, rows, n,
              a.k, a.bits, y.data_ptr(), n, _CODE[out_dtype], _word(y.device).data_ptr(), stream)
    return y


@dataclass
class NormRows:
    """What norm_add() returns: the sum h, 1 / rms of every row, the normalised rows in codes (and their values),
    and the inputs that its gradient reads again."""
    h: torch.Tensor
    rstd: torch.Tensor
    rows: MxRows
    x: torch.Tensor
    residual: torch.Tensor | None

    @property
    def values(self) -> torch.Tensor | None:
        return self.rows.values


def norm_add(x: torch.Tensor, residual: torch.Tensor | None, gain: torch.Tensor, eps: float = 1e-6, bits: int = 8,
             values: bool = False) -> NormRows:
    """h = x + residual and h / rms(h) * gain in microscaled rows of `bits`."""
    _want(x.dim() == 2 and x.dtype in _CODE and x.shape[1] > 0, "norm_add: x must be rows x dim of f32, bf16 or f16")
    _want(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "norm_add: the residual must be like x")
    _want(gain.dtype == torch.float32 and gain.shape == x.shape[1:] and gain.is_contiguous(), "norm_add: gain must be dim float32 values")
    _want(bits in (4, 8), "norm_add: bits must be 4 or 8")
    _cuda("norm_add", x, gain, *(() if residual is None else (residual,)))
    rows, dim = x.shape
    with _on(x) as stream:
        x, ldx = _plain_rows(x)
        ptr, ldr = 0, 0
        if residual is not None:
            residual, ldr = _plain_rows(residual)
            ptr = residual.data_ptr()
        h = torch.empty((rows, dim), dtype=x.dtype, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        q = _mx_empty(rows, dim, bits, values, x.device)
        _call(_lib().smg_norm_add, x.data_ptr(), ldx, ptr, ldr, gain.data_ptr(), rows, dim, _CODE[x.dtype], eps, h.data_ptr(), dim,
              rstd.data_ptr(), bits, q.codes.data_ptr(), q.scales.data_ptr(), q.values.data_ptr() if values else 0, stream)
    return NormRows(h, rstd, q, x, residual)


def norm_add_backward(dy: torch.Tensor, f: NormRows, gain: torch.Tensor, dh: torch.Tensor | None = None):
    """(dx, dgain) of norm_add(): dx is the gradient for x and for the residual alike; dh is the gradient that reaches
    h past the norm.  The rounding to codes counts as the identity."""
    x, r = f.x, f.residual
    _want(dy.shape == x.shape and dy.dtype == x.dtype, "norm_add_backward: dy must be like x")
    _want(dh is None or (dh.shape == x.shape and dh.dtype == x.dtype), "norm_add_backward: dh must be like x")
    _want(gain.dtype == torch.float32 and gain.shape == x.shape[1:] and gain.is_contiguous(), "norm_add_backward: gain must be dim float32 values")
    _cuda("norm_add_backward", x, dy, gain, *(() if dh is None else (dh,)))
    rows, dim = x.shape
    with _on(x) as stream:
        dy, lddy = _plain_rows(dy)
        pr, ldr, pd, ldd = 0, 0, 0, 0
        if r is not None:
            pr, ldr = r.data_ptr(), r.stride(0)
        if dh is not None:
            dh, ldd = _plain_rows(dh)
            pd = dh.data_ptr()
        dx = torch.empty((rows, dim), dtype=x.dtype, device=x.device)
        dgain = torch.empty(dim, dtype=torch.float32, device=x.device)
        L = _lib()
        work = torch.empty(L.smg_norm_add_bwd_work(dim), dtype=torch.uint8, device=x.device)
        _call(L.smg_norm_add_bwd, dy.data_ptr(), lddy, x.data_ptr(), x.stride(0), pr, ldr, f.rstd.data_ptr(), gain.data_ptr(), pd, ldd, rows,
              dim, _CODE[x.dtype], dx.data_ptr(), dim, dgain.data_ptr(), work.data_ptr(), stream)
    return dx, dgain
