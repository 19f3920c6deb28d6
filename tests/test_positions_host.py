"""Rotary positions as callers without a component see them (no GPU)."""
import ctypes as C

import hostapi as H

pkg = H.pkg


def test_a_null_component_is_refused():
    words = (C.c_uint32 * 1)(0)
    assert pkg.library().psi_gqa_set_positions(None, words, C.c_uint32(1)) == 1
