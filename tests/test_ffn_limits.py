"""Grids of the row-wise feed-forward kernels up to the widest rows that the entry points take."""
import ffn_probe


def test_strips_of_the_widest_rows():
    lib = ffn_probe.load()
    most = lib.probe_max_side()
    for cols in (1, 511, 512, 513, 14336, 0x7ffffdff, 0x7ffffe00, 0x7ffffe01, most - 1, most):
        strips = lib.probe_column_strips(cols)
        assert strips == -(-cols // 512)
        assert strips * 256 < 1 << 32                     # threads of a grid along x
        assert strips * 512 - 8 < 1 << 31                 # the last thread's first column, a 32-bit number
        assert (cols + 31) < 1 << 31 and cols + 255 < 1 << 31   # the blocks of a checkpoint, tiles of the products
