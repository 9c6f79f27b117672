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


def test_offsets_without_a_group():
    """No group at all is a refusal of the call's own, whichever tensor says so."""
    from scenemap_b200.smg import SmgError
    if not has_gpu():
        pytest.skip("no GPU")
    x, none = rnd(8, 64), torch.empty(0, dtype=torch.int32, device="cuda")
    for call in (lambda: P.grouped_dw(x, x, none), lambda: P.grouped_dw(x, x, none[:0].new_zeros(1)),
                 lambda: P.grouped(x, rnd(0, 16, 64), none.new_zeros(1)), lambda: P.grouped_dx(x, rnd(0, 64, 16), none.new_zeros(1))):
        with pytest.raises(SmgError, match="group"):
            call()


def test_flags_without_a_truth_value():
    """A flag that has no truth value is refused, not left as an exception behind a result."""
    from scenemap_b200.smg import SmgError
    if not has_gpu():
        pytest.skip("no GPU")
    x, gain, flag = rnd(8, 64), torch.ones(64, device="cuda"), torch.ones(2)
    for call in (lambda: P.mx_quantise(x, 4, values=flag), lambda: P.norm_add(x, None, gain, values=flag)):
        with pytest.raises(SmgError, match="values"):
            call()
