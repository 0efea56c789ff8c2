"""What the host layer asks about streams (runs without a GPU)."""

from __future__ import annotations

from mmfp4 import _lib


def test_the_default_stream_is_in_no_capture():
    assert _lib.load().mm_capture_id(None) == 0
