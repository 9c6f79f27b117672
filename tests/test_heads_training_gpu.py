"""MapHeads.train_step on the B200 against 64 bits: what a step changes, for many rows (where a mean's 1 / rows is small)."""
import math

import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not has_gpu():
        pytest.skip("no GPU")


def unit(v):
    return v / v.norm(dim=-1, keepdim=True)


def check_step(t, counts, dim, eps=1e-6, zeros=0):
    """The changes of the weights and of the gain, which start at 0 and 1, with `zeros` rows of zeros.  With e the error of a
    value, the gradient for it is e / (sqrt(dim) rows).  Bounds, term by term: e is a difference of 32-bit values; the
    gradient and dh are each rounded once to the 16-bit type (relative u; below its normal range by half the least
    spacing, of what f16 is scaled by so that 1 / sqrt(eps) fits); the sums run in 32 bits."""
    import torch
    import products_ref as R
    from scenemap_b200 import products as P
    from scenemap_b200.heads import MapHeads
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[t]
    torch.manual_seed(7)
    P.clear_error()
    rows, off, lr = sum(counts), R.offsets(counts, "cuda"), 1000.0
    z = unit(torch.randn(rows, dim, device="cuda")).to(t)
    z[:zeros] = 0
    target = unit(torch.randn(rows, dim, device="cuda"))
    H = MapHeads(len(counts), dim, dtype=t, eps=eps)
    v = H.forward(z, off, 8, True).values.double()
    loss = H.train_step(z, target, off, lr)

    down = 2.0 ** min(0, 14 + math.floor(math.log2(eps) / 2)) if t == torch.float16 else 1.0
    scale, u, tiny = dim ** -0.5, R.U[t], R.TINY[t] / 2 / down
    e = v * scale - target.double()
    h = z.double()                                       # W = 0
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + H.eps)
    n = h * rstd
    dh = rstd * (e - n * (e * n).mean(1, keepdim=True))
    e_off = u * e.abs() + tiny + 2.0 ** -22 * (v.abs() * scale + target.double().abs())
    dh_mag = rstd * (e.abs() + n.abs() * (e * n).abs().mean(1, keepdim=True))
    dh_off = rstd * (e_off + n.abs() * (e_off * n.abs()).mean(1, keepdim=True)) + (u + (dim + 16) * 2.0 ** -23) * dh_mag + tiny
    dgain, dgain_off = (e * n).sum(0), (e_off * n.abs()).sum(0) + (rows + dim / 2 + 16) * 2.0 ** -23 * (e * n).abs().sum(0)
    f = scale / rows
    tol = 2 * f * dgain_off + 2.0 ** -22 / lr * (1 + lr * f * dgain.abs())     # (2: u is taken of the 64-bit values)
    assert (((1 - H.gain.double()) / lr - f * dgain).abs() <= tol).all()
    for g, r in R.spans(off, len(counts), rows):
        dw = dh[r].T @ h[r]
        off_w = dh_off[r].T @ h[r].abs() + max(1, r.stop - r.start) * 2.0 ** -23 * (dh[r].abs().T @ h[r].abs())
        got = -H.master[g].double() / lr
        assert ((got - f * dw).abs() <= 2 * f * off_w + 2.0 ** -22 * f * dw.abs()).all()
        assert torch.equal(H.w[g], H.master[g].to(t))
    want = 0.5 * (e * e).sum() / rows
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    assert P.error() == 0


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("counts,dim", [([30000, 0, 35536], 1152), ([4000, 99], 1152), ([5], 64)])
def test_step_matches_64_bits(t, counts, dim):
    check_step(t, counts, dim)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("eps", [1e-6, 1e-9, 1e-12, 1e-14])
def test_step_with_rows_of_zeros(t, eps):
    """An empty crop's embedding: 1 / rms is 1 / sqrt(eps), and the gradient for its sum that many times its error."""
    check_step(t, [150, 151], 64, eps, 3)


def test_step_with_bad_offsets_changes_nothing():
    """Offsets that break the rules leave unspecified results: none of them reaches the weights or the gain, and the loss says so."""
    import torch
    from scenemap_b200 import products as P
    from scenemap_b200.heads import MapHeads
    torch.manual_seed(2)
    P.clear_error()
    dim, rows = 96, 300
    H = MapHeads(2, dim)
    z, target = unit(torch.randn(rows, dim, device="cuda")).bfloat16(), unit(torch.randn(rows, dim, device="cuda"))
    good = torch.tensor([0, 100, rows], dtype=torch.int32, device="cuda")
    assert torch.isfinite(H.train_step(z, target, good, 10.0))
    before = H.master.clone(), H.gain.clone(), H.w.clone()
    filler = torch.full((64, rows, dim), float("nan"), device="cuda")        # what unwritten outputs may hold
    del filler
    for off in ([0, 400, rows], [5, 100, rows], [0, 100, 200]):
        loss = H.train_step(z, target, torch.tensor(off, dtype=torch.int32, device="cuda"), 10.0)
        assert torch.isnan(loss) and P.error() == P.BAD_OFFSETS
        assert all(torch.equal(a, b) for a, b in zip((H.master, H.gain, H.w), before))
        P.clear_error()
    assert torch.isfinite(H.train_step(z, target, good, 10.0)) and not torch.equal(H.master, before[0])
