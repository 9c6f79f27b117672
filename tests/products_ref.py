"""The embedding heads' definitions in 64 bits, map by map, and the bounds their tests use."""
import torch

# unit roundoff of the output types, and their smallest spacing
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def spans(off, groups, rows):
    o = [0, rows] if off is None else off.tolist()
    return [(g, slice(o[g], o[g + 1])) for g in range(groups)]


def y64(x, w, off):
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    for g, r in spans(off, w.shape[0], x.shape[0]):
        out[r] = x[r].double() @ w[g].double().T
    return out


def dx64(dy, w, off):
    out = torch.zeros(dy.shape[0], w.shape[2], dtype=torch.float64, device=dy.device)
    for g, r in spans(off, w.shape[0], dy.shape[0]):
        out[r] = dy[r].double() @ w[g].double()
    return out


def dw64(dy, x, off, groups):
    out = torch.zeros(groups, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    for g, r in spans(off, groups, x.shape[0]):
        out[g] = dy[r].double().T @ x[r].double()
    return out


def near(got, want, mags, terms, what):
    """A sum of `terms` products in 32-bit floats, rounded or truncated after every addition, is within
    terms * 2^-23 of the sum of magnitudes; then one rounding to the output's type."""
    tol = terms * 2.0 ** -23 * mags + U[got.dtype] * want.abs() * (1 + 2.0 ** -10) + TINY[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} of the bound"


def grid(bits, device):
    if bits == 4:
        pos = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    else:
        pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    return torch.tensor(pos, dtype=torch.float64, device=device)


def two(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64, device="cpu"), e.cpu().int()).to(e.device)


def exponents(x, bits):
    """e of every block of 32, by the definition."""
    v = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)
    most = v.abs().amax(2)
    e = torch.where(most > 0, torch.frexp(most).exponent - 1 - (2 if bits == 4 else 8), torch.full_like(most, -127).int())
    return e.clamp(-127, 127), v, most


def mx64(x, bits):
    """(values, e): every block of 32 over 2^e to the nearest value of the format, ties to the even one."""
    e, v, _ = exponents(x, bits)
    pos = grid(bits, x.device)
    s = two(e)[..., None]
    a = (v / s).abs().contiguous()
    hi = torch.searchsorted(pos, a).clamp(1, len(pos) - 1)
    down, up = a - pos[hi - 1], pos[hi] - a
    i = torch.where((down > up) | ((down == up) & (hi % 2 == 0)), hi, hi - 1)
    return (torch.sign(v) * pos[i] * s).reshape(x.shape[0], -1)[:, :x.shape[1]], e


def decode64(codes, scales, bits, k):
    pos = grid(bits, codes.device)
    if bits == 4:
        at = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
        at, neg = at % 8, at >= 8
    else:
        at, neg = codes.long() % 128, codes >= 128
    q = torch.where(neg, -pos[at], pos[at])
    q = q.reshape(*q.shape[:-1], -1, 32)
    return (q * two(scales[..., :q.shape[-2]].int() - 127)[..., None]).flatten(-2)[..., :k]


def offsets(counts, device):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device=device)
