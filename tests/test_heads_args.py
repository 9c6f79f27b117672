"""Further refusals of the embedding heads' C entry points, which need no GPU."""
from test_products_args import ARGS, F32, L, _built, _text  # noqa: F401  (L, _built: fixtures)


def test_scales_need_only_their_words_aligned(L):
    """A bank sliced by rows: its codes start on 16 bytes, its scales on 4 (36 bytes a row of 1152 values)."""
    def call(sa, sb, codes=16):
        return L.smg_mx_product(codes, sa, 16, sb, None, 1, 0, 8, 1152, 8, 16, 8, F32, None, None)

    assert call(16, 52) == 0 and call(36, 16) == 0           # no rows: the checks alone
    assert call(18, 16) == ARGS and "4" in _text(L)
    assert call(16, 16, codes=20) == ARGS and "16 bytes" in _text(L)
