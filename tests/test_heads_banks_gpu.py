"""Banks cut by rows: codes and scales of any run of rows are rows of their own."""
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if has_gpu():
    import torch
    import products_ref as R
    from test_products_gpu import FP, rnd
    from scenemap_b200 import products as P


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,n,k", [(3, 70, 1152), (256, 500, 1152), (40, 300, 96), (3000, 900, 640)])
def test_scores_of_sliced_banks(bits, rows, n, k):
    if not has_gpu():
        pytest.skip("no GPU")
    torch.manual_seed(4)
    q, b = P.mx_quantise(rnd(rows + 5, k), bits), P.mx_quantise(rnd(n + 9, k), bits)
    x, w = R.decode64(q.codes, q.scales, bits, k), R.decode64(b.codes, b.scales, bits, k)
    for a0, b0 in ((0, 1), (1, 0), (2, 3), (5, 9), (4, 7)):
        part = P.MxRows(q.codes[a0:a0 + rows], q.scales[a0:a0 + rows], bits, k)
        bank = P.MxRows(b.codes[b0:b0 + n], b.scales[b0:b0 + n], bits, k)
        y = P.mx_product(part, bank)
        want, mags = x[a0:a0 + rows] @ w[b0:b0 + n].T, x[a0:a0 + rows].abs() @ w[b0:b0 + n].abs().T
        R.near(y, want, mags, k, "scores")
        assert torch.equal(bank.dequantise(FP).double(), w[b0:b0 + n])
    assert P.error() == 0
