"""CPU-only checks of how the few-token experts divide their work: no kernel is launched."""
import ctypes

from moe_overlap_b200 import _lib


def test_no_part_of_ffn_is_empty():
    """The parts cover ffn in whole stages, none of them behind its end (the consumers that
    skip an item count its stages from its columns), and the workspace holds their sums."""
    lib, cols = _lib.load(), ctypes.c_int32()
    sizes = [(1, 1), (1, 2), (14, 2), (128, 2), (7, 5), (128, 7), (31, 16), (64, 16), (128, 8), (3, 1)]
    ffns = [*range(8, 3 * 2048, 8), *range(6144, 80000, 104), *range(65536, 140000, 1864), 73736, 2 ** 20, 2 ** 20 + 8]
    for T, k in sizes:
        for F in ffns:
            sums = 0
            for narrow, stage, slices in ((0, 64, 1), (1, 256, 4)):
                n = lib.moe_few_tokens_parts(T, F, 16, k, narrow, ctypes.byref(cols))
                c = cols.value
                assert n >= 1 and c % stage == 0 and (n - 1) * c < F <= n * c, (T, k, F, narrow, n, c)
                sums = max(sums, n * slices)
            need = T * k * (F * 4 + 64 * 4 * sums)
            assert lib.moe_few_tokens_workspace(T, 64, F, 16, k) >= need
    assert lib.moe_few_tokens_parts(14, 73736, 2, 2, 0, ctypes.byref(cols)) == 35
    for bad in ((129, 64, 4, 2, 0), (4, 60, 4, 2, 0), (4, 64, 4, 5, 0)):
        assert lib.moe_few_tokens_parts(*bad, ctypes.byref(cols)) == -1
    assert lib.moe_few_tokens_parts(4, 64, 4, 2, 0, None) == -1


def test_widths_past_what_an_int_holds_are_refused():
    """A column, and the stage behind the last one, have to fit in 32 bits."""
    lib, cols, wide = _lib.load(), ctypes.c_int32(), 2 ** 30 + 8
    assert lib.moe_few_tokens_parts(1, 2 ** 30, 4, 1, 0, ctypes.byref(cols)) > 0
    assert lib.moe_few_tokens_workspace(1, 2 ** 30, 64, 4, 1) > 0
    assert lib.moe_few_tokens_parts(1, wide, 4, 1, 0, ctypes.byref(cols)) == -1
    assert lib.moe_few_tokens_workspace(1, wide, 64, 4, 1) == -1
    assert lib.moe_few_tokens_workspace(1, 64, wide, 4, 1) == -1
    for H, F in ((wide, 64), (64, wide)):
        assert lib.moe_few_tokens(16, H, 16, H, None, 16, F * H, H, 16, F * H, F, 0, 1, H, F, 4, 1, 0, 16, 16, 16, H,
                                  16, 1 << 62, None, None) == _lib.MOE_ERR_INVALID_ARG
