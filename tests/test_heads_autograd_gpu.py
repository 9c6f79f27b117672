"""Autograd and the embedding heads' calls, which record nothing for it: inputs that ask for gradients are refused while they
are recorded, and inputs changed between a norm and its gradient are noticed."""
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if has_gpu():
    import torch
    import products_ref as R
    from test_products_gpu import rnd
    from scenemap_b200 import products as P
    from scenemap_b200.smg import SmgError


@pytest.fixture(autouse=True)
def _gpu():
    if not has_gpu():
        pytest.skip("no GPU")
    torch.manual_seed(3)


def _calls(x, w, dy, gain, res, off):
    f = P.norm_add(x.detach(), res.detach(), gain.detach())
    return {"x": (lambda a: P.grouped(a, w, off), x), "w": (lambda a: P.grouped(x, a, off), w),
            "dx dy": (lambda a: P.grouped_dx(a, w, off), dy), "dx w": (lambda a: P.grouped_dx(dy, a, off), w),
            "dw dy": (lambda a: P.grouped_dw(a, x, off), dy), "dw x": (lambda a: P.grouped_dw(dy, a, off), x),
            "quantise": (lambda a: P.mx_quantise(a, 4), x), "norm x": (lambda a: P.norm_add(a, res, gain), x),
            "norm residual": (lambda a: P.norm_add(x, a, gain), res), "norm gain": (lambda a: P.norm_add(x, res, a), gain),
            "norm dy": (lambda a: P.norm_add_backward(a, f, gain), res), "norm gain back": (lambda a: P.norm_add_backward(res, f, a), gain),
            "norm dh": (lambda a: P.norm_add_backward(res, f, gain, dh=a), res)}


def test_inputs_that_require_gradients():
    """Refused where autograd would lose them; taken, with the same bits, under no_grad, inference_mode and detached."""
    off = R.offsets([30, 12], "cuda")
    x, w, dy, res, gain = rnd(42, 64), rnd(2, 40, 64), rnd(42, 40), rnd(42, 64), torch.ones(64, device="cuda")
    for name, (call, at) in _calls(x, w, dy, gain, res, off).items():
        with pytest.raises(SmgError, match="gradient"):
            call(at.clone().requires_grad_())
        call(at)
        with torch.no_grad():
            call(at.clone().requires_grad_())
        with torch.inference_mode():
            call(at.clone().requires_grad_())
        call(at.clone().requires_grad_().detach())
    p = w.clone().requires_grad_()
    with torch.no_grad():
        assert torch.equal(P.grouped(x, p, off), P.grouped(x, w, off))


@pytest.mark.parametrize("which", ["x", "residual"])
def test_inputs_changed_before_the_gradient(which):
    """The gradient reads the norm's inputs again: one changed in place since is refused, wherever it was changed from."""
    x, res, gain, dy = rnd(9, 120), rnd(9, 120), torch.ones(120, device="cuda"), rnd(9, 120)
    f = P.norm_add(x, res, gain)
    want = P.norm_add_backward(dy, f, gain)
    again = P.norm_add_backward(dy, f, gain)
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    at = {"x": x, "residual": res}[which]
    at[3:5].mul_(2)                                      # through a view
    with pytest.raises(SmgError, match="changed"):
        P.norm_add_backward(dy, f, gain)
    f = P.norm_add(x, None, gain)
    P.norm_add_backward(dy, f, gain)
    with torch.inference_mode():                         # inference tensors count no changes
        g = P.norm_add(x.clone(), None, gain)
        P.norm_add_backward(dy, g, gain)


def test_training_step_on_tensors_that_require_gradients():
    """A training step takes its own gradients: tensors of a caller's graph go in as they are, and none of it is recorded."""
    from scenemap_b200.heads import MapHeads
    off = R.offsets([20, 12], "cuda")
    z, target = rnd(32, 64), torch.nn.functional.normalize(torch.randn(32, 64, device="cuda"), dim=1)
    a, b = MapHeads(2, 64), MapHeads(2, 64)
    plain = a.train_step(z, target, off, 5.0)
    loss = b.train_step(z.clone().requires_grad_(), target.clone().requires_grad_(), off, 5.0)
    assert torch.equal(loss, plain) and not loss.requires_grad and torch.equal(a.master, b.master) and torch.equal(a.gain, b.gain)
