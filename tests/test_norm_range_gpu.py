"""The residual norm at the ends of its inputs' range: rows whose squares leave the 32-bit range, with large and small
eps, and rows with an infinity."""
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if has_gpu():
    import torch
    import products_ref as R
    from test_products_gpu import BF, FP, HF, check_codes, rnd
    from scenemap_b200 import products as P


@pytest.fixture(autouse=True)
def _gpu():
    if not has_gpu():
        pytest.skip("no GPU")
    torch.manual_seed(11)


# factor of the rows, eps: squares above 2^128, below 2^-126 and below the least of all, each against an eps that counts, one that does
# not, and none
RANGE = [(1e18, 1e-6), (1e19, 0.0), (3e36, 1e-6), (1e-21, 1e-42), (1e-24, 0.0), (1e-30, 1e-40), (1e-30, 1e-6), (2e17, 1e36)]


@pytest.mark.parametrize("size,eps", RANGE)
@pytest.mark.parametrize("rows,dim", [(3, 64), (2, 1152), (1300, 520), (1300, 1152), (3, 5001), (2, 16384)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_rows_of_any_size(size, eps, rows, dim, t):
    t = {"bf16": BF, "f32": FP}[t]
    x, r = rnd(rows, dim, t=FP).mul_(size).to(t), rnd(rows, dim, t=FP).mul_(size).to(t)
    gain = 1 + 0.2 * torch.randn(dim, device="cuda")
    e32 = float(torch.tensor(eps, dtype=FP))           # as the call takes it
    h = x.double() + r.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + e32)
    rel = (dim / 2 + 12) * 2.0 ** -24                  # as in test_norm_add
    f = P.norm_add(x, r, gain, eps=eps, bits=8, values=True)
    assert ((f.rstd.double() - rstd).abs() <= rel * rstd + 2.0 ** -149).all()
    # (1 / rms of the largest rows is subnormal: half of its spacing more)
    sub = float((2.0 ** -149 / rstd).max())
    check_codes(f.rows, h * rstd[:, None] * gain.double(), rel + sub, 8)
    if size < 1:
        return                                          # dx, of the size of 1 / rms, may leave the type's range
    dy = rnd(rows, dim, t=t)
    dx, dgain = P.norm_add_backward(dy, f, gain)
    n, u = h * rstd[:, None], dy.double() * gain.double()
    mean = (u * n).mean(1, keepdim=True)
    want = rstd[:, None] * (u - n * mean)
    mags = rstd[:, None] * (u.abs() + n.abs() * (u * n).abs().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= ((dim + 16) * 2.0 ** -23 + 2 * sub) * mags + R.U[t] * want.abs() * (1 + 2.0 ** -10) + R.TINY[t]).all()
    g, gm = (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0)
    assert ((dgain.double() - g).abs() <= ((rows + dim / 2 + 16) * 2.0 ** -23 + sub) * gm + 1e-30).all()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,dim", [(3, 200), (1300, 1152), (3, 5001)])
def test_row_with_an_infinity(t, rows, dim):
    """1 / rms is 0: the infinity's block is NaN, the row's other values are 0, other rows are as before."""
    t = {"bf16": BF, "f16": HF, "f32": FP}[t]
    x, gain = rnd(rows, dim, t=t), torch.ones(dim, device="cuda")
    want = P.norm_add(x, None, gain)
    bad = x.clone()
    bad[1, 33] = float("-inf")
    f = P.norm_add(bad, None, gain, values=True)
    keep = [i for i in range(rows) if i != 1]
    assert torch.equal(f.rows.codes[keep], want.rows.codes[keep]) and torch.equal(f.rows.scales[keep], want.rows.scales[keep])
    assert f.rstd[1] == 0 and f.rows.scales[1, 1] == 255 and f.values[1, 32:64].isnan().all()
    assert not f.values[1, :32].any() and not f.values[1, 64:].any()


def test_as_many_rows_as_a_call_counts():
    """2^31 - 1 rows of one value: the last ones are those of a small call, and the gradient's sum counts them all."""
    rows, gain = 0x7fffffff, torch.full((1,), 1.5, device="cuda")
    L = P._lib()
    x = torch.zeros(rows, 1, dtype=BF, device="cuda")
    x[-100:] = rnd(100, 1)
    v, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    word = torch.cuda.current_stream().cuda_stream
    assert L.smg_norm_add(x.data_ptr(), 1, None, 0, gain.data_ptr(), rows, 1, 1, 1e-6, None, 1, rstd.data_ptr(), 8, None, None,
                          v.data_ptr(), word) == 0, L.smg_last_error()
    f = P.norm_add(x[-100:], None, gain, values=True)
    assert torch.equal(v[-100:], f.values) and torch.equal(rstd[-100:], f.rstd) and not v[:1000].any()
    dx, dgain = v, torch.empty(1, device="cuda")           # dx over the values
    work = torch.empty(L.smg_norm_add_bwd_work(1), dtype=torch.uint8, device="cuda")
    assert L.smg_norm_add_bwd(x.data_ptr(), 1, x.data_ptr(), 1, None, 0, rstd.data_ptr(), gain.data_ptr(), None, 0, rows, 1, 1,
                              dx.data_ptr(), 1, dgain.data_ptr(), work.data_ptr(), word) == 0, L.smg_last_error()
    want = P.norm_add_backward(x[-100:], f, gain)
    assert torch.equal(dx[-100:], want[0])
    # zeros elsewhere: the 100 terms' sum in another order
    assert abs(float(dgain - want[1])) <= 100 * 2.0 ** -23 * float((x[-100:].float().abs()).sum())
