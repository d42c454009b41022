"""The KV pool's name in Runtime: an unknown one is refused, not served from another pool."""
import pytest


@pytest.mark.parametrize("name", ["fp4", "MXFP4", "mxfp8", "bfloat16", "F32", "", None, 3])
def test_unknown_kv_pools_are_refused(name):
    from ferrisinfer_amd import FerrisError
    from ferrisinfer_amd.runtime import Runtime

    with pytest.raises(FerrisError) as e:
        Runtime(hidden=256, intermediate=688, layers=1, heads=8, kv_heads=2, vocab=64, kv_dtype=name)
    assert e.value.kind == "InvalidType" and "mxfp4" in e.value.message


def test_names_and_dtypes():
    from ferrisinfer_amd import DTYPE_BF16, DTYPE_F32, DTYPE_MXFP4
    from ferrisinfer_amd.runtime import KV_DTYPES

    assert KV_DTYPES == {"f32": DTYPE_F32, "bf16": DTYPE_BF16, "mxfp4": DTYPE_MXFP4}
