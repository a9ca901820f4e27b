"""The block-scaled entry points' host side, further: what each call refuses or asks for."""

from __future__ import annotations

import ctypes

import pytest

from marathon_amd import _lib
from tests.test_scaled_plain import attend_desc


@pytest.mark.parametrize("token,head", [(128, 128), (256, 128), (128, 256), (0, 128), (512, 0),
                                        (512, 64), (64, 512)])
def test_attend_refuses_outputs_that_overlap(token, head):
    """Three tokens of four heads of 128."""
    desc = attend_desc(out_token_stride=token, out_head_stride=head)
    assert _lib.lib().mkv_attend_scaled(ctypes.byref(desc), None) == _lib.MKV_ERR_ARG
    assert b"overlap" in _lib.lib().mkv_last_error()
