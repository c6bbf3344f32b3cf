"""Capture numbers without a device."""
from speech_serving import _native as N


def test_no_capture_has_number_zero():
    lib = N.load()
    assert lib.spd_stream_capture_id(None) == 0


def test_a_misaligned_workspace_is_refused_on_the_host():
    """Partial results are stored 16 bytes at a time; addresses here are numbers that nothing reads."""
    lib = N.load()
    a, ws, size = 1 << 20, (1 << 20) + 8, 1 << 30
    assert lib.spd_paged_decode_attn_int4(a, a, a, a, a, 1, 4, 2, 64, 16, 4, 4, 1.0, N.SPD_F16, ws, size, None) == N.SPD_ERR_INVALID_ARG
    assert "16-byte aligned" in N.last_error()
    assert lib.spd_paged_decode_attn(a, a, a, a, a, a, 1, 2, 64, 16, 4, 4, 1.0, N.SPD_F16, None, None, ws, size,
                                     None) == N.SPD_ERR_INVALID_ARG
    assert "16-byte aligned" in N.last_error()
    assert lib.spd_cross_attn(a, a, a, a, a, 1, 2, 64, 100, 100 * 128, 100 * 64, 1.0, N.SPD_F16, ws, size, None) == N.SPD_ERR_INVALID_ARG
    assert "16-byte aligned" in N.last_error()
