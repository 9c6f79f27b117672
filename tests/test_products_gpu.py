"""Embedding heads on the B200 against their definitions in 64 bits: ragged products by map and their gradients,
microscaled rows and their products, the residual norm and its gradients.  Tolerances are bounds
derived from the formats (products_ref.near), not fitted."""
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if has_gpu():
    import torch
    import products_ref as R
    from scenemap_b200 import products as P
    from scenemap_b200.smg import SmgError

    BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
    TYPE = {"bf16": BF, "f16": HF, "f32": FP}


@pytest.fixture(autouse=True)
def _word():
    if not has_gpu():
        pytest.skip("no GPU")
    torch.manual_seed(5)
    P.clear_error()
    yield
    assert P.error() == 0


def rnd(*shape, t=None):
    return torch.randn(*shape, device="cuda").to(t or BF)


def check_products(counts, n, k, t, out=None, x=None, w=None, dy=None):
    rows, groups = sum(counts), len(counts)
    off = R.offsets(counts, "cuda")
    x = rnd(rows, k, t=t) if x is None else x
    w = rnd(groups, n, k, t=t) if w is None else w
    dy = rnd(rows, n, t=t) if dy is None else dy
    y, dx, dw = P.grouped(x, w, off, out), P.grouped_dx(dy, w, off, out), P.grouped_dw(dy, x, off, out)
    assert y.shape == (rows, n) and dx.shape == (rows, k) and dw.shape == (groups, n, k)
    assert y.dtype == dx.dtype == dw.dtype == (out or t)
    R.near(y, R.y64(x, w, off), R.y64(x.abs(), w.abs(), off), k, "y")
    R.near(dx, R.dx64(dy, w, off), R.dx64(dy.abs(), w.abs(), off), n, "dx")
    R.near(dw, R.dw64(dy, x, off, groups), R.dw64(dy.abs(), x.abs(), off, groups), max(counts), "dw")


COUNTS = {"one": [1], "empty ends": [0, 5, 0, 0, 17, 0], "odd": [1, 127, 0, 129, 33, 64, 2], "tiles": [128, 256, 64],
          "long": [700, 3], "many": [(7 * i) % 5 for i in range(200)]}


@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("n,k", [(64, 64), (1, 1), (24, 200), (257, 129), (300, 72), (520, 1000)])
def test_grouped_products(counts, n, k):
    for t in (["bf16"] if n > 300 else ["bf16", "f16"]):
        check_products(COUNTS[counts], n, k, TYPE[t], FP if (n + k) % 3 else None)


@pytest.mark.parametrize("t,out", [("bf16", "f16"), ("f16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_grouped_output_types(t, out):
    check_products([40, 0, 300, 9], 96, 160, TYPE[t], TYPE[out])


@pytest.mark.parametrize("rows", [3, 40, 100, 260, 1300])
@pytest.mark.parametrize("groups", [1, 9])
def test_grouped_sizes_of_every_variant(rows, groups):
    """Few rows a group to many: every rule that picks a kernel by the sizes."""
    c = [rows // groups] * groups
    c[0] += rows - sum(c)
    check_products(c, 384, 192, BF)


@pytest.mark.parametrize("counts", [[700, 0, 1500, 513], [1, 3000], [2049], [0, 256, 1800, 255, 257]])
@pytest.mark.parametrize("n,k", [(520, 264), (256, 1000), (72, 2048)])
def test_grouped_many_rows(counts, n, k):
    """Groups of more rows than a tile of two CTAs has, sizes that no tile divides."""
    check_products(counts, n, k, HF if n == 256 else BF, FP if n == 72 else None)


def test_many_rows_do_not_leak():
    """NaN in one large group's rows stays there: tiles of two CTAs that reach into the next group."""
    c = [900, 700, 0, 800]
    off = R.offsets(c, "cuda")
    x, w, dy = rnd(2400, 264), rnd(4, 392, 264), rnd(2400, 392)
    want = P.grouped(x, w, off), P.grouped_dx(dy, w, off), P.grouped_dw(dy, x, off)
    x[900:1600], dy[900:1600], w[1], w[2] = (float("nan"),) * 4
    y, dx, dw = P.grouped(x, w, off), P.grouped_dx(dy, w, off), P.grouped_dw(dy, x, off)
    for got, ref in ((y, want[0]), (dx, want[1])):
        assert torch.equal(got[:900], ref[:900]) and torch.equal(got[1600:], ref[1600:]) and got[900:1600].isnan().all()
    assert torch.equal(dw[0], want[2][0]) and torch.equal(dw[3], want[2][3]) and not dw[2].any() and dw[1].isnan().all()


def test_one_group_without_offsets():
    x, w = rnd(50, 96), rnd(1, 40, 96)
    R.near(P.grouped(x, w, None, FP), R.y64(x, w, None), R.y64(x.abs(), w.abs(), None), 96, "y")


def test_grouped_strides_and_broadcasts():
    """Column slices, steps between rows, transposed and broadcast inputs, off 16-byte starts."""
    big, bw = rnd(90, 400), rnd(3, 70, 300)
    c = [30, 2, 13]
    check_products(c, 64, 120, BF, FP, x=big[::2, 8:128], w=bw[:, 3:67, 8:128])
    check_products(c, 64, 120, BF, FP, x=big[::2, 3:123], w=bw[:, 3:67, 5:125])
    check_products(c, 64, 120, BF, FP, x=rnd(120, 45).T, w=rnd(3, 120, 64).transpose(1, 2), dy=rnd(64, 45).T)
    check_products(c, 64, 120, BF, FP, x=rnd(1, 120).expand(45, 120), w=rnd(1, 64, 120).expand(3, 64, 120), dy=rnd(1, 64).expand(45, 64))


def test_other_groups_do_not_leak():
    """NaN and infinities in one group's rows and weights stay in that group, in tails of tiles too."""
    c = [37, 50, 0, 70]
    off = R.offsets(c, "cuda")
    for n, k in ((72, 104), (300, 136)):
        x, w, dy = rnd(157, k), rnd(4, n, k), rnd(157, n)
        want = P.grouped(x, w, off), P.grouped_dx(dy, w, off), P.grouped_dw(dy, x, off)
        for v in (float("nan"), float("inf")):
            xb, wb, db = x.clone(), w.clone(), dy.clone()
            xb[37:87], db[37:87], wb[1], wb[2] = v, v, v, v
            y, dx, dw = P.grouped(xb, wb, off), P.grouped_dx(db, wb, off), P.grouped_dw(db, xb, off)
            for got, ref in ((y, want[0]), (dx, want[1])):
                assert torch.equal(got[:37], ref[:37]) and torch.equal(got[87:], ref[87:])
                assert not torch.isfinite(got[37:87]).any()
            assert torch.equal(dw[0], want[2][0]) and torch.equal(dw[3], want[2][3]) and not dw[2].any()
            assert not torch.isfinite(dw[1]).any()


def test_grouped_no_rows():
    off = R.offsets([0, 0, 0], "cuda")
    x, w, dy = rnd(0, 32), rnd(3, 16, 32), rnd(0, 16)
    assert P.grouped(x, w, off).shape == (0, 16) and P.grouped_dx(dy, w, off).shape == (0, 32)
    dw = P.grouped_dw(dy, x, off)
    assert dw.shape == (3, 16, 32) and not dw.any()


def test_grouped_same_bits_again():
    c = [300, 1, 77]
    off = R.offsets(c, "cuda")
    x, w, dy = rnd(378, 256), rnd(3, 128, 256), rnd(378, 128)
    first = P.grouped(x, w, off), P.grouped_dx(dy, w, off), P.grouped_dw(dy, x, off)
    for _ in range(3):
        again = P.grouped(x, w, off), P.grouped_dx(dy, w, off), P.grouped_dw(dy, x, off)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_grouped_bad_offsets_set_the_word():
    x, w, dy = rnd(64, 32), rnd(2, 16, 32), rnd(64, 16)
    for o in ([0, 80, 64], [0, -3, 64], [0, 40, 30], [5, 40, 64]):
        off = torch.tensor(o, dtype=torch.int32, device="cuda")
        for call in (lambda: P.grouped(x, w, off), lambda: P.grouped_dx(dy, w, off), lambda: P.grouped_dw(dy, x, off)):
            P.clear_error()
            call()
            assert P.error() == P.BAD_OFFSETS
    P.clear_error()


def test_grouped_gradients_against_differences():
    """L = sum(y * dy) of the 64-bit definition, differenced along random directions."""
    c = [20, 0, 45]
    off = R.offsets(c, "cuda")
    x, w, dy = rnd(65, 48), rnd(3, 40, 48), rnd(65, 40)
    dx, dw = P.grouped_dx(dy, w, off, FP), P.grouped_dw(dy, x, off, FP)
    vx, vw = torch.randn(65, 48, device="cuda", dtype=torch.float64), torch.randn(3, 40, 48, device="cuda", dtype=torch.float64)

    def loss(a, b):
        return (R.y64(a, b, off) * dy.double()).sum()

    for got, v, plus, minus in ((dx, vx, loss(x.double() + vx, w), loss(x.double() - vx, w)),
                                (dw, vw, loss(x, w.double() + vw), loss(x, w.double() - vw))):
        d = (plus - minus) / 2                       # the loss is linear in each
        assert abs(float((got.double() * v).sum() - d)) <= 65 * 2.0 ** -23 * float((got.double() * v).abs().sum())


def test_another_stream():
    """Work queued on a side stream, with the inputs made on it."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x, w = rnd(2000, 512), rnd(2, 256, 512)
        off = R.offsets([700, 1300], "cuda")
        for _ in range(3):
            x = x * 0.5
        y = P.grouped(x, w, off, FP)
        q = P.mx_quantise(x, 4, values=True)
    s.synchronize()
    R.near(y, R.y64(x, w, off), R.y64(x.abs(), w.abs(), off), 512, "y")
    assert torch.equal(q.values.double(), R.mx64(x, 4)[0])


def test_in_a_graph():
    """Captured once and replayed on new inputs: nothing is allocated or kept by the library."""
    x, w, off = rnd(70, 128), rnd(2, 64, 128), R.offsets([33, 37], "cuda")
    gain = torch.ones(64, device="cuda")
    P.grouped(x, w, off)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = P.grouped(x, w, off)
        f = P.norm_add(y, None, gain)
        s = P.mx_product(f.rows, f.rows)
    for _ in range(2):
        x.copy_(rnd(70, 128))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, P.grouped(x, w, off))
        assert torch.equal(s, P.mx_product(P.norm_add(y, None, gain).rows, f.rows))


def test_rows_past_32_bit_offsets():
    """The last rows of an input of more than 2^31 values."""
    rows, k = 2_200_000, 1024
    x = torch.zeros(rows, k, dtype=BF, device="cuda")
    x[-300:] = rnd(300, k)
    w, off = rnd(2, 8, k), R.offsets([rows - 200, 200], "cuda")
    y = P.grouped(x, w, off, FP)
    tail = R.offsets([100, 200], "cuda")
    R.near(y[-300:], R.y64(x[-300:], w, tail), R.y64(x[-300:].abs(), w.abs(), tail), k, "y")
    assert not y[:-300].any()
    q = P.mx_quantise(x, 4)
    assert torch.equal(R.decode64(q.codes[-300:], q.scales[-300:], 4, k), R.mx64(x[-300:], 4)[0])
    del x
    s = P.mx_product(q, P.mx_quantise(w[0], 4))
    xq, wq = R.decode64(q.codes[-300:], q.scales[-300:], 4, k), R.mx64(w[0], 4)[0]
    R.near(s[-300:], xq @ wq.T, xq.abs() @ wq.abs().T, k, "scores")


# ------------------------------------------------------------------ microscaled rows

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 1000), (130, 1152), (4, 4099)])
def test_quantise(bits, t, rows, k):
    x = rnd(rows, k, t=TYPE[t])
    x[0] *= 0
    if rows > 2:
        x[1] = x[1] * 2.0 ** (-12 if t == "f16" else -100)
        x[2] = torch.sign(x[2].float()) * 2.5         # ties of both formats' grids
    q = P.mx_quantise(x, bits, values=True)
    want, e = R.mx64(x, bits)
    kb = (k + 31) // 32
    assert torch.equal(q.scales[:, :kb].int() - 127, e) and not q.scales[:, kb:].any()
    assert torch.equal(R.decode64(q.codes, q.scales, bits, k), want)
    assert not R.decode64(q.codes, q.scales, bits, kb * 32)[:, k:].any()
    assert torch.equal(q.values.double(), want)
    for out in (FP, BF):
        assert torch.equal(q.dequantise(out).double(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_every_value(bits):
    """Every bf16 value (as the largest of its block or below one) and the steps between the grid's values."""
    v = torch.arange(0, 0x7f80, dtype=torch.int32, device="cuda").to(torch.int16).view(BF)
    v = torch.cat((v, -v)).reshape(-1, 32)
    assert torch.equal(P.mx_quantise(v, bits).dequantise(FP).double(), R.mx64(v, bits)[0])
    top = 6.0 if bits == 4 else 448.0
    f = torch.linspace(-top * 1.3, top * 1.3, 65536, device="cuda").reshape(-1, 32).contiguous()
    f[:, 0] = top
    assert torch.equal(P.mx_quantise(f, bits).dequantise(FP).double(), R.mx64(f, bits)[0])


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_infinities_and_nan(bits):
    """A block with an infinity or NaN gets the scale NaN; its neighbours and its row's other blocks are as before."""
    x = rnd(4, 160)
    want = P.mx_quantise(x, bits)
    bad = x.clone()
    bad[0, 33], bad[1, 100], bad[3, 159] = float("nan"), float("-inf"), float("inf")
    q = P.mx_quantise(bad, bits, values=True)
    hit = torch.zeros(4, 5, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[1, 3] = hit[3, 4] = True
    assert torch.equal(q.scales[:, :5] == 255, hit)
    v, ref = q.values.reshape(4, 5, 32), want.dequantise(BF).reshape(4, 5, 32)
    assert torch.isnan(v[hit]).all() and torch.equal(v[~hit], ref[~hit])
    s = P.mx_product(q, want)
    assert torch.isnan(s[[0, 1, 3]]).all() and torch.equal(s[2], P.mx_product(want, want)[2])


def test_quantise_strides():
    x = rnd(60, 300)
    for v in (x[::3, 5:205], x.T[:40], x[:1].expand(9, 300), x[:, 8:108]):
        assert torch.equal(P.mx_quantise(v, 4, values=True).values.double(), R.mx64(v, 4)[0])


def check_scores(counts, n, k, bits, out=None, rows_type=None):
    rows, groups = sum(counts), len(counts)
    off = R.offsets(counts, "cuda")
    a = P.mx_quantise(rnd(rows, k, t=rows_type), bits)
    b = P.mx_quantise(rnd(groups * n, k), bits)
    b = P.MxRows(b.codes.reshape(groups, n, -1), b.scales.reshape(groups, n, -1), bits, k)
    y = P.mx_product(a, b, off, out or FP)
    x, w = R.decode64(a.codes, a.scales, bits, k), R.decode64(b.codes, b.scales, bits, k)
    R.near(y, R.y64(x, w, off), R.y64(x.abs(), w.abs(), off), k, "scores")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("n,k", [(64, 128), (1, 1), (24, 200), (200, 96), (257, 160), (130, 1152)])
def test_scores(bits, counts, n, k):
    check_scores(COUNTS[counts], n, k, bits, HF if (n + k) % 2 else None)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,n,k", [(1, 4096, 1152), (256, 2048, 1152), (100, 700, 640), (1000, 1000, 512), (3000, 260, 2304)])
def test_scores_of_one_bank(bits, rows, n, k):
    check_scores([rows], n, k, bits)


@pytest.mark.parametrize("bits,k", [(4, 1152), (4, 130), (8, 600), (8, 96)])
def test_scores_many_tiles_of_short_rows(bits, k):
    """Runs of tiles over the same rows: several row tiles, an empty group and ragged ends in one CTA's run."""
    check_scores([300, 0, 500, 201], 15001, k, bits, HF)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("counts,n,k", [([3000, 0, 2500, 700], 700, 640), ([6000], 1152, 1152), ([2049, 4000], 481, 2080)])
def test_scores_of_many_rows(bits, counts, n, k):
    """Tiles of two CTAs: ragged groups, a last tile of few columns, several chunks of scales."""
    check_scores(counts, n, k, bits, BF if n == 700 else None)


def test_scores_spread_of_magnitudes():
    """Blocks of very different sizes in one row: the scales' exponents add up right."""
    for bits in (4, 8):
        x, w = rnd(40, 512, t=FP), rnd(50, 512, t=FP)
        x *= 2.0 ** torch.randint(-30, 30, (40, 16), device="cuda").repeat_interleave(32, 1).float()
        w *= 2.0 ** torch.randint(-30, 30, (50, 16), device="cuda").repeat_interleave(32, 1).float()
        a, b = P.mx_quantise(x, bits), P.mx_quantise(w, bits)
        p, q = R.mx64(x, bits)[0], R.mx64(w, bits)[0]
        R.near(P.mx_product(a, b), p @ q.T, p.abs() @ q.abs().T, 512, "scores")


def test_scores_no_rows_and_bad_offsets():
    a, b = P.mx_quantise(rnd(0, 64), 4), P.mx_quantise(rnd(9, 64), 4)
    assert P.mx_product(a, b).shape == (0, 9)
    a = P.mx_quantise(rnd(20, 64), 4)
    P.mx_product(a, b, torch.tensor([0, 21], dtype=torch.int32, device="cuda"))
    assert P.error() == P.BAD_OFFSETS
    P.clear_error()


# ------------------------------------------------------------------ residual norm

DIMS = [1, 31, 64, 257, 520, 768, 1000, 1152, 1536, 2048, 2056, 5000, 16384]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_norm_add(dim, t):
    t = TYPE[t]
    rows = 9 if dim < 3000 else 3
    x, r = rnd(rows, dim, t=t), rnd(rows, dim, t=t)
    x[1], r[1] = 0, 0
    gain = 1 + 0.2 * torch.randn(dim, device="cuda")
    h = x.double() + r.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + 1e-5)
    y = h * rstd[:, None] * gain.double()
    for bits in (8, 4):
        f = P.norm_add(x, r, gain, eps=1e-5, bits=bits, values=True)
        assert ((f.h.double() - h).abs() <= (U(t) + 2.0 ** -24) * h.abs() * (1 + 2.0 ** -10) + R.TINY[t]).all()
        # the 32-bit sum of dim squares: dim * 2^-24 of it, halved by the root; a few more roundings
        assert ((f.rstd.double() / rstd - 1).abs() <= (dim / 2 + 8) * 2.0 ** -24).all()
        check_codes(f.rows, y, (dim / 2 + 12) * 2.0 ** -24, bits)
        assert torch.equal(f.values, f.rows.dequantise(BF))
    alone = P.norm_add(x, None, gain, eps=1e-5)
    assert torch.equal(alone.h, x)
    h = x.double()
    check_codes(alone.rows, h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * gain.double(), (dim / 2 + 12) * 2.0 ** -24, 8)


def U(t):
    return R.U[t]


def check_codes(q, y, rel, bits):
    """Codes of values within `rel` of y: the block's exponent is y's own (or a neighbour, where its largest
    magnitude is that near to a power of two), and every value is the format's nearest or saturated."""
    e64, v, most = R.exponents(y, bits)
    e = q.scales[:, :e64.shape[1]].int() - 127
    edge = torch.frexp(most * (1 + rel)).exponent != torch.frexp(most * (1 - rel)).exponent
    assert ((e == e64) | (edge & ((e - e64).abs() <= 1))).all()
    got = R.decode64(q.codes, q.scales, bits, e64.shape[1] * 32).reshape(v.shape)
    s = R.two(e)[..., None]
    top, half, least = (6.0, 0.25, 0.25) if bits == 4 else (448.0, 2.0 ** -4, 2.0 ** -10)
    tol = torch.maximum(half * v.abs(), (v.abs() - top * s)).clamp(min=0) + least * s + rel * v.abs()
    assert ((got - v).abs() <= tol * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_norm_add_backward(dim, t):
    t = TYPE[t]
    rows = 700 if dim < 1200 else 21
    x, r, dy, dh = (rnd(rows, dim, t=t) for _ in range(4))
    gain = 1 + 0.2 * torch.randn(dim, device="cuda")
    for res, past in ((r, dh), (None, None)):
        f = P.norm_add(x, res, gain, eps=1e-5)
        dx, dgain = P.norm_add_backward(dy, f, gain, dh=past)
        h = x.double() + (0 if res is None else res.double())
        rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
        n, u = h * rstd, dy.double() * gain.double()
        mean = (u * n).mean(1, keepdim=True)
        want = rstd * (u - n * mean) + (0 if past is None else past.double())
        # 32-bit steps on terms of these magnitudes (the mean is a sum of dim products), then the type
        mags = rstd * (u.abs() + n.abs() * (u * n).abs().mean(1, keepdim=True)) + (0 if past is None else past.double().abs())
        tol = (dim + 16) * 2.0 ** -23 * mags + U(t) * want.abs() * (1 + 2.0 ** -10) + R.TINY[t]
        assert ((dx.double() - want).abs() <= tol).all()
        g, gm = (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0)
        assert ((dgain.double() - g).abs() <= (rows + dim / 2 + 16) * 2.0 ** -23 * gm + 1e-30).all()


def test_norm_backward_against_differences():
    rows, dim = 6, 40
    x, r, dy, dh = (rnd(rows, dim, t=FP) for _ in range(4))
    gain = 1 + 0.2 * torch.randn(dim, device="cuda")
    dx, dgain = P.norm_add_backward(dy, P.norm_add(x, r, gain, eps=1e-3), gain, dh=dh)

    def loss(a, g):
        h = a + r.double()
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-3) * g
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    for got, at, other in ((dx, x.double(), gain.double()), (dgain, gain.double(), x.double())):
        v, step = torch.randn_like(at), 1e-4
        f = (lambda a: loss(a, other)) if got is dx else (lambda g: loss(other, g))
        d = (f(at + step * v) - f(at - step * v)) / (2 * step)
        # differences of step^2 (third derivatives of order 1) and 32-bit sums
        assert abs(float((got.double() * v).sum() - d)) <= 1e-5 * float((got.double() * v).abs().sum())


def test_norm_strides_rows_and_columns():
    """Steps between rows, column slices off 16 bytes, transposed and broadcast inputs: the bits of contiguous ones."""
    base, gain = rnd(40, 400), 1 + 0.1 * torch.randn(120, device="cuda")
    for x, r in ((base[::2, 3:123], base[1::2, 8:128]), (base.T[:20, :].T[:20, :].repeat(1, 6), base[:1, :120].expand(20, 120)),
                 (rnd(120, 20).T, base[:20, 1:121])):
        f, c = P.norm_add(x, r, gain, values=True), P.norm_add(x.contiguous(), r.contiguous(), gain, values=True)
        assert torch.equal(f.h, c.h) and torch.equal(f.rows.codes, c.rows.codes) and torch.equal(f.values, c.values)
        dy = rnd(120, 20).T
        a, b = P.norm_add_backward(dy, f, gain), P.norm_add_backward(dy.contiguous(), c, gain)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_norm_nan_stays_in_its_row():
    x, gain = rnd(5, 200), torch.ones(200, device="cuda")
    want = P.norm_add(x, None, gain)
    bad = x.clone()
    bad[2, 7] = float("nan")
    f = P.norm_add(bad, None, gain)
    keep = [0, 1, 3, 4]
    assert torch.equal(f.rows.codes[keep], want.rows.codes[keep]) and torch.equal(f.rows.scales[keep], want.rows.scales[keep])
    assert (f.rows.scales[2, :7] == 255).all()


def test_norm_no_rows():
    gain = torch.ones(32, device="cuda")
    f = P.norm_add(rnd(0, 32), None, gain)
    dx, dgain = P.norm_add_backward(rnd(0, 32), f, gain)
    assert f.h.shape == (0, 32) and dx.shape == (0, 32) and not dgain.any()


# ------------------------------------------------------------------ refusals

def test_refusals():
    x, w, off = rnd(8, 64), rnd(2, 16, 64), R.offsets([3, 5], "cuda")
    q4, q8 = P.mx_quantise(x, 4), P.mx_quantise(x, 8)
    gain = torch.ones(64, device="cuda")
    for call in (lambda: P.grouped(x, w, None), lambda: P.grouped(x, w.half(), off), lambda: P.grouped(x.float(), w.float(), off),
                 lambda: P.grouped(x, w[..., :63], off), lambda: P.grouped(x, w, off.long()), lambda: P.grouped(x, w, off[:2]),
                 lambda: P.grouped(x.cpu(), w.cpu(), off.cpu()), lambda: P.grouped(x, w, off, torch.int32),
                 lambda: P.grouped(x, w, off.cpu()), lambda: P.grouped_dx(x, w, off), lambda: P.grouped_dw(x[:4], x, off),
                 lambda: P.grouped(x, rnd(1100, 16, 64), R.offsets([0] * 1099 + [8], "cuda")),
                 lambda: P.mx_quantise(x, 6), lambda: P.mx_quantise(x.int(), 4), lambda: P.mx_product(q4, q8),
                 lambda: P.mx_product(q4, P.mx_quantise(x[:, :32], 4)),
                 lambda: P.mx_product(P.MxRows(q4.codes[:, :16], q4.scales, 4, 64), q4), lambda: P.norm_add(x, x[:4], gain),
                 lambda: P.norm_add(x, None, gain.half()), lambda: P.norm_add(rnd(2, 16400), None, torch.ones(16400, device="cuda")),
                 lambda: P.norm_add_backward(x.half(), P.norm_add(x, None, gain), gain)):
        with pytest.raises(SmgError):
            call()
