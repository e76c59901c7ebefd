"""Scratch of the group norm, on the CPU: it follows the size of the GPU and of its cache, not the number of samples."""

import pytest

from pararnn_b200 import _lib

F32, BF16 = _lib.PRB_F32, _lib.PRB_BF16
PIECE = 72 << 20  # bytes of samples that one pair of launches covers

# samples, positions, channels, groups: rows wider than the one-pass kernels take, and many samples of few positions
SHAPES = [(32768, 1, 2048, 1), (8192, 1, 4096, 1), (32768, 1, 1056, 32), (65536, 4, 64, 8), (4_000_000, 2, 2, 1),
          (1_000_000, 2, 1024, 8), (500_000, 2, 512, 512), (200, 2, 65536, 32768), (100_000, 3, 999, 27),
          (3, 50, 4400, 2), (16, 4096, 256, 32)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_scratch_does_not_grow_with_the_samples(shape, dtype):
    n, pos, c, g = shape
    size = lambda k, back: _lib.lib().prb_group_norm_workspace_bytes(k, pos, c, g, dtype, back)  # noqa: E731
    # rows of partial sums, two floats a channel: a wave of CTAs and a rounding, or a sixteenth of a piece
    wide = max(2 * 296 * 2 * 4 * c, PIECE // 16)
    for back in (0, 1):
        assert size(n, back) <= PIECE + back * wide
        # ten times the samples need no more than the samples that fill a piece do
        full = max(1, PIECE // (pos * c * 2)) + 1
        assert size(10 * max(n, full), back) <= size(max(n, full), back)
    # and no more than the data itself once that is worth mentioning
    data = n * pos * c * (4 if dtype == F32 else 2)
    if data >= 16 << 20:
        assert size(n, 1) <= 2 * data


def test_rows_too_wide_for_the_grid_take_the_other_kernels():
    """Five channels a group in slots of eight lanes: 75000 CTAs side by side, where a grid's second axis ends at
    65535.  The one-pass kernels need no scratch forwards, the others do."""
    size = lambda c, g: _lib.lib().prb_group_norm_workspace_bytes(1, 1, c, g, F32, 0)  # noqa: E731
    assert size(12_000_000, 2_400_000) > 0
    assert size(1_200_000, 240_000) == 0


def c_pointer():
    import ctypes

    buf = ctypes.create_string_buffer(1024)
    return buf, (ctypes.addressof(buf) + 255) & ~255


def test_norm_refuses_positions_whose_steps_pass_32_bits():
    """PRB_ERR_UNSUPPORTED before any launch; the largest size that stays allowed ends at the missing workspace."""
    keep, p = c_pointer()
    call = lambda n: _lib.lib().prb_group_norm(p, None, None, p, None, 1, n, 1, 1, 1e-5, 0, 1, 0, None, 0, None)  # noqa: E731
    assert call(2 ** 31 - 1) == -3 and call(2 ** 31 - 4096) == -3 and call(2 ** 31 - 1 - 4096) == -2
    back = lambda n: _lib.lib().prb_bwd_group_norm(p, p, None, None, p, p, None, None, 1, n, 1, 1, 0, 1, 0, None, 0,  # noqa: E731
                                                   None)
    assert back(2 ** 31 - 1) == -3 and back(2 ** 31 - 1 - 4096) == -2


def test_attention_refuses_rows_whose_segments_pass_32_bits():
    import ctypes

    keep, p = c_pointer()
    h = ctypes.byref(_lib.Heads(p, 1, 1, 1))

    def call(n, cu):
        return _lib.lib().prb_linear_attention(h, h, h, p, None, p if cu else None, p, None, 1, n, 1, n, 1, 1, 1, 1, 1, 1.0,
                                               None, 0, None)

    for cu in (False, True):
        assert call(2 ** 31 - 1, cu) == -3 and call(2 ** 30 + 1, cu) == -3 and call(2 ** 30, cu) == -2


def test_embedding_gradient_refuses_counts_whose_sums_pass_32_bits():
    keep, p = c_pointer()
    most = 2 ** 31 - 2 ** 16
    size = _lib.lib().prb_bwd_embedding_workspace_bytes
    call = lambda n, v: _lib.lib().prb_bwd_embedding(p, 0, p, p, n, v, 1, 1, 1.0, None, 0, None)  # noqa: E731
    assert call(most + 1, 5) == -3 and call(5, most + 1) == -3 and call(most, most) == -2
    assert size(most + 1, 5, 1) == 0 and size(5, most + 1, 1) == 0 and size(most, most, 1) > 0


def test_step_refuses_tables_that_it_would_search_for_minutes():
    """Refusals only: a call that is allowed would go to the device."""
    keep, p = c_pointer()

    def call(rows, table):
        return _lib.lib().prb_linear_attention_step(p, p, p, p, p, p if table else None, 0, p, rows, rows, 1, 1, 1, 1, 0,
                                                    1.0, None)

    assert call(2 ** 20 + 1, True) == -3 and call(2 ** 31 - 1, True) == -3 and call(2 ** 30 + 1, False) == -3
