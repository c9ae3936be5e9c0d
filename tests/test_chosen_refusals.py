"""Calls of the operators whose rows choose their weights that the library refuses, beside those of test_chosen_linears.py."""
import pytest


def test_adapters_without_a_slice(hip):
    p = hip.adapters_params(hip.HALF, 4, 16, 5, 64, [])
    for call in (lambda: hip.adapters_workspace(p), lambda: hip.adapters(p, *([64] * 10))):
        with pytest.raises(hip.ItexHipError, match="slices"):
            call()
