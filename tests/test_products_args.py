"""Refusals of the embedding heads' C entry points, which need no GPU: bad sizes, types, alignment and null
pointers come back as error codes with a text, before anything is launched."""
import ctypes as C
import os

import pytest

from conftest import ROOT

F32, BF16 = 0, 1
ARGS, CAPACITY = -1, -3


@pytest.fixture(scope="module", autouse=True)
def _built():
    pkg = os.path.join(ROOT, "robot-agent_b200")
    for f in ("libsmg.so", os.path.join("scenemap_b200", "_heads.so")):
        if not os.path.exists(os.path.join(pkg, f)):
            pytest.skip(f"{f} not built (python __graft_entry__.py build)")


@pytest.fixture(scope="module")
def L():
    from scenemap_b200 import products
    return products._lib()


def _text(L):
    return L.smg_last_error().decode()


def test_group_product_refusals(L):
    ok = dict(x=16, ldx=64, w=16, ldw=64, ws=64 * 8, off=16, groups=2, rows=4, n=8, k=64, type=BF16, y=16, ldy=8, yt=F32)

    def call(**kw):
        a = {**ok, **kw}
        return L.smg_group_product(a["x"], a["ldx"], a["w"], a["ldw"], a["ws"], a["off"], a["groups"], a["rows"], a["n"], a["k"], a["type"],
                                   a["y"], a["ldy"], a["yt"], None, None)

    for kw, text in (({"groups": 0}, "sizes"), ({"rows": -1}, "sizes"), ({"n": 0}, "sizes"), ({"k": 0}, "sizes"),
                     ({"off": None}, "no offsets"), ({"type": F32}, "bf16 or f16"), ({"yt": 7}, "output type"), ({"x": None}, "x is null"),
                     ({"w": None}, "w is null"), ({"y": None}, "output is null"), ({"x": 24}, "16 bytes"), ({"ldx": 65}, "16 bytes"),
                     ({"ldw": 68}, "16 bytes"), ({"ws": 516}, "16 bytes"), ({"ldx": 56}, "overlap"), ({"ws": 256}, "overlap"), ({"ldy": 7}, "overlap")):
        assert call(**kw) == ARGS, kw
        assert text in _text(L), (kw, _text(L))
    assert call(groups=1025) == CAPACITY and "1024" in _text(L)
    assert call(rows=0x7fffffff) == CAPACITY and "rows" in _text(L)
    assert call(rows=0, x=None, y=None) == 0          # nothing to do


def test_gradient_refusals(L):
    assert L.smg_group_product_dx(16, 8, 16, 64, 512, 16, 2, 4, 8, 64, BF16, 16, 63, F32, None, None) == ARGS and "overlap" in _text(L)
    assert L.smg_group_product_dx(16, 12, 16, 64, 512, 16, 2, 4, 12, 64, BF16, 16, 64, F32, None, None) == ARGS and "dy" in _text(L)
    assert L.smg_group_product_dw(16, 8, 16, 64, 16, 2, 4, 8, 64, BF16, 16, 64, 500, F32, None, None) == ARGS and "overlap" in _text(L)
    assert L.smg_group_product_dw(16, 8, 16, 64, 16, 2, 4, 8, 64, BF16, None, 64, 512, F32, None, None) == ARGS and "null" in _text(L)


def test_mx_refusals(L):
    assert L.smg_mx_quantise(16, 64, 4, 64, BF16, 5, 16, 16, None, None) == ARGS and "bits" in _text(L)
    assert L.smg_mx_quantise(16, 64, 4, 64, BF16, 4, 16, None, None, None) == ARGS and "together" in _text(L)
    assert L.smg_mx_quantise(16, 64, 4, 64, BF16, 4, None, None, None, None) == ARGS
    assert L.smg_mx_quantise(16, 64, 4, 64, 9, 4, 16, 16, None, None) == ARGS and "type" in _text(L)
    assert L.smg_mx_quantise(16, 64, 4, 64, BF16, 4, 20, 16, None, None) == ARGS and "16 bytes" in _text(L)
    assert L.smg_mx_quantise(16, 64, -1, 64, BF16, 4, 16, 16, None, None) == ARGS
    assert L.smg_mx_values(None, None, 4, 64, 4, 16, 64, F32, None) == ARGS
    assert L.smg_mx_values(16, 16, 4, 64, 4, 16, 60, F32, None) == ARGS and "overlap" in _text(L)
    assert L.smg_mx_product(16, 16, 16, None, None, 1, 4, 8, 64, 4, 16, 8, F32, None, None) == ARGS and "together" in _text(L)
    assert L.smg_mx_product(16, 16, 16, 16, None, 1, 4, 8, 64, 7, 16, 8, F32, None, None) == ARGS and "bits" in _text(L)
    assert L.smg_mx_product(16, 16, 16, 16, None, 2, 4, 8, 64, 4, 16, 8, F32, None, None) == ARGS


def test_norm_refusals(L):
    f = C.c_float(1e-6)
    assert L.smg_norm_add(None, 64, None, 0, 16, 4, 64, BF16, f, 16, 64, None, 8, 16, 16, None, None) == ARGS and "null" in _text(L)
    assert L.smg_norm_add(16, 64, None, 0, None, 4, 64, BF16, f, 16, 64, None, 8, 16, 16, None, None) == ARGS and "null" in _text(L)
    assert L.smg_norm_add(16, 64, None, 0, 16, 4, 64, BF16, f, 16, 60, None, 8, 16, 16, None, None) == ARGS and "overlap" in _text(L)
    assert L.smg_norm_add(16, 64, None, 0, 16, 4, 64, BF16, f, 16, 64, None, 3, 16, 16, None, None) == ARGS and "bits" in _text(L)
    assert L.smg_norm_add(16, 20000, None, 0, 16, 4, 20000, BF16, f, 16, 20000, None, 8, 16, 16, None, None) == CAPACITY
    assert L.smg_norm_add_bwd_work(0) == 0 and L.smg_norm_add_bwd_work(100) % 400 == 0
    assert L.smg_norm_add_bwd(16, 64, 16, 64, None, 0, 16, 16, None, 0, 4, 64, BF16, 16, 64, None, 16, None) == ARGS and "null" in _text(L)
    assert L.smg_norm_add_bwd(16, 64, 16, 64, None, 0, 16, 16, None, 0, 4, 64, BF16, 16, 64, 16, 20, None) == ARGS and "16 bytes" in _text(L)
    assert L.smg_norm_add_bwd(16, 64, 16, 64, None, 0, 16, 16, None, 0, 4, 64, BF16, 16, 32, 16, 16, None) == ARGS and "overlap" in _text(L)


def test_python_refusals_without_a_gpu():
    import torch
    from scenemap_b200 import products as P
    from scenemap_b200.smg import SmgError
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(1, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(SmgError, match="CUDA"):
        P.grouped(x, w, None)
    with pytest.raises(SmgError, match="both"):
        P.grouped(x, w.half(), None)
    with pytest.raises(SmgError, match="rows x k"):
        P.grouped(x[0], w, None)
