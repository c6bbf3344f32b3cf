"""Capture numbers without a device."""
from speech_serving import _native as N


def test_no_capture_has_number_zero():
    lib = N.load()
    assert lib.spd_stream_capture_id(None) == 0
