"""Coefficients that the orthogonalisation refuses, without a GPU."""
import ctypes

import pytest

ERR_ARG = -1


@pytest.mark.parametrize("steps, coeffs, word", [
    (5, (float("nan"), 0.0, 0.0), "finite"), (5, (1.0, float("inf"), 0.0), "finite"), (1, (1.0, 0.0, -float("inf")), "finite"),
    # any finite ones go on to the next check, of the device
    (5, (3.4445, -4.7750, 2.0315), None), (64, (1.5, -0.5, 0.0), None), (64, (100.0, 0.0, 0.0), None), (64, (0.01, 0.0, 0.0), None), (1, (0.0, 0.0, 1.0), None),
    (64, (3.0, 3.0, 3.0), None), (5, (8.0, -23.0, 17.0), None), (4, (1e30, -3e38, 1e38), None), (3, (0.0, 0.0, 0.0), None), (64, (0.0, 1.0, 0.0), None),
    (64, (0.5, 1.0, 0.0), None)], ids=str)
def test_coefficients(cake, steps, coeffs, word):
    L, p = cake.lib(), ctypes.c_void_p(0x100000)
    ws = L.cakeb200_orthogonalize_workspace(8, 12, 1, 0)
    for rc in (L.cakeb200_orthogonalize(p, 12, 96, p, 12, 96, 8, 12, 1, 0, steps, *coeffs, 0.0, ctypes.c_void_p(0x200000), ws, None),
               L.cakeb200_muon_step(p, 12, 0, p, 12, 0, ctypes.c_void_p(0x300000), 12, 8, 12, 0.1, 0.9, 1, 0.0, 1.0, steps, *coeffs, 0.0, ctypes.c_void_p(0x200000), ws, None)):
        text = L.cakeb200_last_error().decode()
        if word:
            assert rc == ERR_ARG and word in text, text
        else:
            assert "finite" not in text, text
