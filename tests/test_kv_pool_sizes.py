"""fi_kv_pool_bytes at sizes that pass 32 and 64 bits."""
import pytest

TOP = 2 ** 31 - 1


def test_sizes_past_32_bits():
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4, kv_pool_bytes

    for dtype, row in ((DTYPE_F32, 128 * 4), (DTYPE_BF16, 128 * 2), (DTYPE_MXFP4, 68)):
        assert kv_pool_bytes(dtype, TOP, 16, 8, 128) == TOP * 16 * 8 * row
        assert kv_pool_bytes(dtype, 16, TOP, 8, 128) == TOP * 16 * 8 * row


@pytest.mark.parametrize("sizes", [(TOP, TOP, TOP, 128), (TOP, TOP, 8, 128), (2 ** 30, 2 ** 30, 4, 32), (2 ** 24, 2 ** 24, 2 ** 10, 32)])
def test_sizes_past_63_bits_are_refused(sizes):
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4, FerrisError, kv_pool_bytes

    blocks, block_size, heads, d = sizes
    for dtype, row in ((DTYPE_F32, 4 * d), (DTYPE_BF16, 2 * d), (DTYPE_MXFP4, 17 * d // 32)):
        size = blocks * block_size * heads * row
        if size < 2 ** 63:  # (2^24, 2^24, 2^10, 32) in 4 bits: 17 * 2^58
            assert kv_pool_bytes(dtype, *sizes) == size
            continue
        with pytest.raises(FerrisError) as e:
            kv_pool_bytes(dtype, *sizes)
        assert e.value.kind == "InvalidShape"
