"""Preference and policy tuning: refusals and host logic beside those of the operators' own tests."""
from __future__ import annotations

from molt_b200 import _native

A, B, C, D, E = (0x10000 * i for i in range(1, 6))   # addresses that are only checked


def test_counted_adamw_needs_a_count(native_library):
    for skipped in (None, E + 4):
        rc = native_library.molt_adamw_step_counted(A, B, C, D, 4, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, skipped, 0)
        assert rc == _native.E_VALUE and b"skipped is NULL or not 8-byte aligned" in native_library.molt_last_error()
    for change, word in (((A, B, C, D, 3), b"multiple of 4"), ((None, B, C, D, 4), b"NULL"), ((A + 4, B, C, D, 4), b"16-byte aligned")):
        rc = native_library.molt_adamw_step_counted(*change, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, E, 0)
        assert rc == _native.E_VALUE and word in native_library.molt_last_error()
