"""Embedding heads per map: what products.py's operators are for, run together.

A map sees its own rooms, lights and camera.  Its head is a linear map on top of the image embeddings,
kept close to them by the residual:  y = norm(z + W_g z) * gain.  The heads of all maps of a batch are
trained in one step on the maps' own pairs of detections and object vectors, and the normalised rows go into the
memory bank and the scores in 8 or 4 bits.
"""
from __future__ import annotations

import math

import torch

from . import products as P
from .smg import SmgError


class MapHeads:
    """Heads of n_maps maps for embeddings of `dim` values, on one device."""

    def __init__(self, n_maps: int, dim: int, device="cuda", dtype: torch.dtype = torch.bfloat16, eps: float = 1e-6):
        if n_maps < 1 or dim < 1 or n_maps > P.MAX_GROUPS:
            raise SmgError(f"MapHeads: 1 to {P.MAX_GROUPS} maps and a positive dim")
        self.n_maps, self.dim, self.eps = n_maps, dim, eps
        self.master = torch.zeros((n_maps, dim, dim), dtype=torch.float32, device=device)   # trained in 32 bits
        self.w = self.master.to(dtype)                                                       # what the products read
        self.gain = torch.ones(dim, dtype=torch.float32, device=device)

    def forward(self, z: torch.Tensor, off: torch.Tensor, bits: int = 8, values: bool = False) -> P.NormRows:
        """Rows z (all maps' packed, off[g] the first of map g) through their maps' heads; .rows holds the codes."""
        return P.norm_add(P.grouped(z, self.w, off), z, self.gain, self.eps, bits, values)

    def backward(self, dy: torch.Tensor, f: P.NormRows, z: torch.Tensor, off: torch.Tensor):
        """(dz, dw, dgain) for dy, the gradient for the values of forward()'s rows (the rounding to codes counts as the
        identity)."""
        dh, dgain = P.norm_add_backward(dy, f, self.gain)
        dw = P.grouped_dw(dh, z, off, torch.float32)
        dz = P.grouped_dx(dh, self.w, off) + dh        # through W, and past it
        return dz, dw, dgain

    @torch.no_grad()
    def train_step(self, z: torch.Tensor, target: torch.Tensor, off: torch.Tensor, lr: float) -> torch.Tensor:
        """One step of gradient descent on the mean over the rows of |y / sqrt(dim) - target|^2 / 2, target the unit vector of
        the object that row r shows.  Returns the loss (a tensor: nothing waits for it).  A step that finds the device's
        error word set (products.error: bad offsets, a wait that ran out) changes nothing and returns NaN."""
        f = self.forward(z, off, 8, True)
        scale = self.dim ** -0.5                       # |y| is sqrt(dim)
        e = f.values.float() * scale - target.float()
        rows = max(1, z.shape[0])
        loss = 0.5 * e.square().sum() / rows
        # The gradient for the values is e * scale / rows.  Its factor stays out of the 16-bit steps: a mean over many
        # rows would put f16's values below its smallest ones (65536 rows x 1152: 9 of 10 were lost).  In f16 a power of
        # two goes in where eps is so small that dh, up to |e| / sqrt(eps) in a row of zeros, would not fit.
        down = 1.0
        if z.dtype == torch.float16 and self.eps > 0:
            down = 2.0 ** min(0, 14 + math.floor(math.log2(self.eps) / 2))
        _, dw, dgain = self.backward((e * down if down != 1 else e).to(z.dtype), f, z, off)
        step = lr * scale / rows / down
        bad = P.failed(z.device)
        dw.masked_fill_(bad, 0)
        dgain.masked_fill_(bad, 0)
        self.master.sub_(dw, alpha=step)
        self.gain.sub_(dgain, alpha=step)
        self.w.copy_(self.master)
        return loss.masked_fill_(bad[0], float("nan"))

    def bank(self, vectors: torch.Tensor, bits: int = 4) -> P.MxRows:
        """Memory bank of the maps' object vectors (n_maps x n x dim) in microscaled rows."""
        if vectors.dim() != 3 or vectors.shape[0] != self.n_maps or vectors.shape[2] != self.dim:
            raise SmgError("MapHeads.bank: vectors must be maps x n x dim")
        q = P.mx_quantise(vectors.reshape(-1, self.dim), bits)
        shape = vectors.shape[:2]
        return P.MxRows(q.codes.view(*shape, -1), q.scales.view(*shape, -1), bits, self.dim)

    def scores(self, z: torch.Tensor, off: torch.Tensor, bank: P.MxRows, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """Each row's score against every object of its own map (rows x n): the cosine, up to the codes' rounding, for
        unit bank vectors."""
        f = self.forward(z, off, bank.bits)
        return P.mx_product(f.rows, bank, off, torch.float32).mul_(self.dim ** -0.5).to(out_dtype)
