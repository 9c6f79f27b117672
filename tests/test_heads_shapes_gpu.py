"""Shapes of the embedding heads' kernels that small calls do not reach: the norm's kernels for many rows (from 1185 on a row
has fewer warps; from 296 blocks on the gradient's go round), skewed maps, and as many maps as a call takes."""
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if has_gpu():
    import torch
    import products_ref as R
    from test_products_gpu import BF, FP, HF, check_codes, check_products, rnd
    from scenemap_b200 import products as P

TYPES = ["bf16", "f16", "f32"]


@pytest.fixture(autouse=True)
def _word():
    if not has_gpu():
        pytest.skip("no GPU")
    torch.manual_seed(6)
    P.clear_error()
    yield
    assert P.error() == 0


def check_norm(rows, dim, t, bits, eps=1e-5):
    """Forward and gradients against 64 bits, bounds as for few rows: sums of dim 32-bit squares (2^-24 each, halved by the
    root), of dim products, and of `rows` terms a column."""
    t = {"bf16": BF, "f16": HF, "f32": FP}[t]
    x, r, dy, dh = (rnd(rows, dim, t=t) for _ in range(4))
    gain = 1 + 0.2 * torch.randn(dim, device="cuda")
    h = x.double() + r.double()
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    n = h * rstd
    f = P.norm_add(x, r, gain, eps=eps, bits=bits, values=True)
    assert ((f.h.double() - h).abs() <= (R.U[t] + 2.0 ** -24) * h.abs() * (1 + 2.0 ** -10) + R.TINY[t]).all()
    assert ((f.rstd.double()[:, None] / rstd - 1).abs() <= (dim / 2 + 8) * 2.0 ** -24).all()
    check_codes(f.rows, n * gain.double(), (dim / 2 + 12) * 2.0 ** -24, bits)
    assert torch.equal(f.values, f.rows.dequantise(BF))
    dx, dgain = P.norm_add_backward(dy, f, gain, dh=dh)
    u = dy.double() * gain.double()
    want = rstd * (u - n * (u * n).mean(1, keepdim=True)) + dh.double()
    mags = rstd * (u.abs() + n.abs() * (u * n).abs().mean(1, keepdim=True)) + dh.double().abs()
    tol = (dim + 16) * 2.0 ** -23 * mags + R.U[t] * want.abs() * (1 + 2.0 ** -10) + R.TINY[t]
    assert ((dx.double() - want).abs() <= tol).all()
    g = dy.double() * n
    assert ((dgain.double() - g.sum(0)).abs() <= (rows + dim / 2 + 16) * 2.0 ** -23 * g.abs().sum(0) + 1e-30).all()
    again = P.norm_add_backward(dy, f, gain, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dgain, again[1])


@pytest.mark.parametrize("rows", [2500, 5001])
@pytest.mark.parametrize("dim", [64, 250, 257, 512, 520, 768, 1000, 1152, 1153, 1536, 1600, 2048, 3000])
@pytest.mark.parametrize("t", TYPES)
def test_norm_of_many_rows(rows, dim, t):
    check_norm(rows, dim, t, 8 if (rows + dim) % 2 else 4)


@pytest.mark.parametrize("rows", [1183, 1184, 1185])
@pytest.mark.parametrize("dim", [300, 1152, 2047])
@pytest.mark.parametrize("t", TYPES)
def test_norm_where_the_rows_get_fewer_warps(rows, dim, t):
    check_norm(rows, dim, t, 4 if rows % 2 else 8)


@pytest.mark.parametrize("rows,dim", [(700, 3073), (700, 4096), (311, 5121), (311, 6145), (311, 8192), (311, 10240), (311, 10241), (311, 16383)])
@pytest.mark.parametrize("t", TYPES)
def test_norm_of_long_rows(rows, dim, t):
    check_norm(rows, dim, t, 8 if dim % 2 else 4)


# one map with nearly all rows among silent ones, where the mean alone picks the few-row kernel; the same past it
@pytest.mark.parametrize("groups,rows,at", [(64, 512, 0), (64, 512, 63), (64, 505, 17), (64, 520, 17), (200, 1600, 101), (1024, 8192, 700)])
def test_one_map_has_all_the_rows(groups, rows, at):
    c = [0] * groups
    c[at] = rows
    check_products(c, 64, 96, BF, FP)
    c[at], c[(at + 1) % groups] = rows - 5, 5
    check_products(c, 40, 200, HF)


@pytest.mark.parametrize("groups", [255, 256, 257, 600, 1024])
@pytest.mark.parametrize("per", [1, 20])
def test_many_maps(groups, per):
    """dw's order of maps (by length up to 256 of them) and the largest count a call takes."""
    check_products([(11 * i) % (2 * per + 1) for i in range(groups)], 72, 104, BF, FP if per > 1 else None)


@pytest.mark.parametrize("groups", [256, 1024])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_of_many_maps(groups, bits):
    from test_products_gpu import check_scores
    check_scores([(5 * i) % 9 for i in range(groups)], 40, 160, bits)
    c = [0] * groups
    c[groups // 3] = 3 * groups
    check_scores(c, 24, 96, bits, HF)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", [(9000, 1152), (70000, 40), (3001, 2303)])
def test_dequantise_many_rows(bits, t, rows, k):
    """The values of many rows, as each type, equal those that the codes stand for."""
    t = {"bf16": BF, "f16": HF, "f32": FP}[t]
    q = P.mx_quantise(rnd(rows, k), bits)
    assert torch.equal(q.dequantise(t).double(), R.decode64(q.codes, q.scales, bits, k).to(t).double())
