"""The embedding heads as they are used together: gradients of the whole head against 64-bit autograd, training,
and scores against banks in 4 and 8 bits (GPU)."""
import os
import sys

import pytest

from conftest import ROOT, has_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not has_gpu():
        pytest.skip("no GPU")


def test_head_gradients_match_autograd():
    """dz, dw and dgain of y = norm(z + W_g z) * gain.  The 16-bit steps in between (the head's product, dh, dz) are each
    rounded to 2^-8 relative; the sums' own errors are far below, so 2^-5 of the largest gradient bounds
    three of them with room for the products' growth."""
    import torch
    import products_ref as R
    from scenemap_b200.heads import MapHeads
    torch.manual_seed(3)
    maps, dim, counts = 3, 96, [40, 0, 75]
    off = R.offsets(counts, "cuda")
    H = MapHeads(maps, dim)
    H.w.copy_(0.3 * torch.randn(maps, dim, dim, device="cuda") / dim ** 0.5)
    H.gain += 0.1 * torch.randn(dim, device="cuda")
    z, dy = torch.randn(115, dim, device="cuda").bfloat16(), torch.randn(115, dim, device="cuda").bfloat16()
    f = H.forward(z, off, 8, True)
    dz, dw, dgain = H.backward(dy, f, z, off)
    z64, w64, g64 = z.double().requires_grad_(), H.w.double().requires_grad_(), H.gain.double().requires_grad_()
    h = z64 + torch.cat([z64[r] @ w64[g].T for g, r in R.spans(off, maps, 115)])
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + H.eps) * g64
    (y * dy.double()).sum().backward()
    for got, want in ((dz, z64.grad), (dw, w64.grad), (dgain, g64.grad)):
        assert float((got.double() - want).abs().max()) <= 2.0 ** -5 * float(want.abs().max())
    assert not dw[1].any()
    # the codes' values: within half a step of e4m3 (2^-4), or saturated (1/8), of the 64-bit rows
    assert float(((f.values.double() - y.detach()).abs() / y.detach().abs().amax(1, keepdim=True)).max()) <= 0.13


def test_example_learns_its_maps():
    """examples/map_heads.py: heads trained on ragged batches name the right object where untrained ones do not, with
    either bank."""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import map_heads
    out = map_heads.run(maps=4, objects=256, dim=128, steps=150, say=lambda *_: None)
    assert out["loss"][1] < 0.5 * out["loss"][0]
    for bits in (4, 8):
        assert out["after"][bits] > out["before"][bits] + 0.1 and out["after"][bits] > 0.9


def test_heads_refuse_bad_sizes():
    import torch
    from scenemap_b200.heads import MapHeads
    from scenemap_b200.smg import SmgError
    for n, d in ((0, 8), (2, 0), (2000, 8)):
        with pytest.raises(SmgError):
            MapHeads(n, d)
    H = MapHeads(2, 64)
    with pytest.raises(SmgError):
        H.bank(torch.zeros(3, 5, 64, device="cuda"))
