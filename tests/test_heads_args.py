"""Further refusals of the embedding heads' C entry points, which need no GPU."""
from test_products_args import ARGS, BF16, CAPACITY, F32, L, _built, _text  # noqa: F401  (L, _built: fixtures)


def test_scales_need_only_their_words_aligned(L):
    """A bank sliced by rows: its codes start on 16 bytes, its scales on 4 (36 bytes a row of 1152 values)."""
    def call(sa, sb, codes=16):
        return L.smg_mx_product(codes, sa, 16, sb, None, 1, 0, 8, 1152, 8, 16, 8, F32, None, None)

    assert call(16, 52) == 0 and call(36, 16) == 0           # no rows: the checks alone
    assert call(18, 16) == ARGS and "4" in _text(L)
    assert call(16, 16, codes=20) == ARGS and "16 bytes" in _text(L)


def test_sizes_that_tiles_cannot_count(L):
    """Widths whose last tile would end past 2^31 are refused, as such rows are."""
    big = 0x7fffffff
    ld = 1 << 31
    assert L.smg_group_product(16, 64, 16, 64, 0, None, 1, 4, big, 64, BF16, 16, big, F32, None, None) == CAPACITY
    assert L.smg_group_product(16, ld, 16, ld, 0, None, 1, 4, 8, big, BF16, 16, 8, F32, None, None) == CAPACITY
    assert L.smg_group_product_dx(16, ld, 16, 64, 0, None, 1, 4, big, 64, BF16, 16, 64, F32, None, None) == CAPACITY
    assert L.smg_group_product_dw(16, 8, 16, ld, None, 1, 4, 8, big, BF16, 16, ld, 0, F32, None, None) == CAPACITY
    assert L.smg_mx_product(16, 16, 16, 16, None, 1, 4, big, 64, 4, 16, big, F32, None, None) == CAPACITY
    assert "too" in _text(L)
