"""Calls of more threads than one launch has are refused before any device work: a grid of 2^32 threads or more is cut without
an error, and what lay beyond was left unwritten (CPU)."""
import pytest

from nori_amd import _native as nat

F16, F32 = nat.NORI_F16, nat.NORI_F32
AT = 1 << 20  # an aligned address; nothing reads it


def _calls():
    lib = nat.lib()
    return {
        # 2^26 rows of a wavefront, 2^29 rows of 8 lanes
        "rms_norm odd": lambda: lib.nori_rms_norm(AT, F16, 2**26, 3, 3, None, F32, 1e-5, AT, 3, None),
        "rms_norm": lambda: lib.nori_rms_norm(AT, F16, 2**29, 64, 64, None, F32, 1e-5, AT, 64, None),
        "residual_add_rms_norm": lambda: lib.nori_residual_add_rms_norm(AT, AT, F16, None, 1.0, 2**28, 64, 1e-5, AT, AT, F16, 1, 64, 64,
                                                                         None),
        "rms_norm_rows": lambda: lib.nori_rms_norm_rows(AT, 2**28, 64, 1, 1, 64, 64, 64, 1e-5, AT, F16, None),
        "layer_norm": lambda: lib.nori_layer_norm(AT, F16, 2**27, 128, 128, None, None, 1e-5, 0, AT, F16, 128, None),
        "layer_norm rows": lambda: lib.nori_layer_norm(AT, F16, 2**26, 96, 96, None, None, 1e-5, 0, AT, F16, 96, None),
        "residual_add": lambda: lib.nori_residual_add(AT, AT, F16, 1.0, 2**34, AT, None),
        "silu_mul": lambda: lib.nori_silu_mul(AT, F16, 2**24, 3, 6, AT, 3, None),
        "quantize": lambda: lib.nori_kv_quantize_int8(AT, F16, 1, 2**32, 7, 0, 8, AT, 0, 7, AT, 0, 1, nat.SCALE_DIV_TRUE, None),
        "dequantize": lambda: lib.nori_kv_dequantize_int8(AT, AT, 1, 2**32, 64, 0, 64, 0, 1, AT, F16, 0, 64, None),
        "dequantize rows": lambda: lib.nori_kv_dequantize_int8(AT, AT, 1, 2**32, 7, 0, 8, 0, 1, AT, F16, 0, 7, None),
    }


@pytest.mark.parametrize("name", sorted(["rms_norm odd", "rms_norm", "residual_add_rms_norm", "rms_norm_rows", "layer_norm",
                                         "layer_norm rows", "residual_add", "silu_mul", "quantize", "dequantize", "dequantize rows"]))
def test_what_one_launch_does_not_hold_is_refused(name):
    assert _calls()[name]() == nat.NORI_ERR_UNSUPPORTED, nat.lib().nori_last_error()
    assert b"launch" in nat.lib().nori_last_error() or b"too many rows" in nat.lib().nori_last_error()
