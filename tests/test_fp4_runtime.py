"""What a serving runtime refuses of a 4-bit KV pool, before it looks for a device."""
import pytest


@pytest.mark.parametrize("change", [dict(hidden=384), dict(hidden=2048), dict(rotary_dims=28), dict(rotary_dims=4)])
def test_runtime_refuses_shapes_a_four_bit_pool_does_not_serve(change):
    from ferrisinfer_amd import FerrisError
    from ferrisinfer_amd.runtime import Runtime

    args = dict(dict(hidden=256, intermediate=688, layers=1, heads=8, kv_heads=2, vocab=64, kv_dtype="mxfp4"), **change)
    with pytest.raises(FerrisError) as e:
        Runtime(**args)
    assert e.value.kind == "Unsupported" and "4-bit KV pool" in e.value.message


def test_decoder_refuses_other_pools():
    from ferrisinfer_amd import DTYPE_F32, FerrisError
    from ferrisinfer_amd.bf16_decoder import LLAMA3_8B_C5, Bf16Decoder

    with pytest.raises(FerrisError) as e:
        Bf16Decoder(None, LLAMA3_8B_C5, 4, 16, 4, 1, kv_dtype=DTYPE_F32)
    assert e.value.kind == "InvalidType"
