"""Orthogonalised updates far from the usual range: gradients far below eps, coefficients that let singular values grow or
shrink, and sums of a single product."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
EPS = 1e-7


def _plain(g, dtype, steps=5, coeffs=(A, B, C), eps=EPS):
    """The formula; the norm in float64 as in the operator."""
    norm = np.sqrt((g.astype(np.float64) ** 2).sum((-2, -1), keepdims=True))
    x = (g / (norm + np.float64(np.float32(eps)))).astype(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = np.swapaxes(x, -1, -2) if tall else x
    a, b, c = (dtype(np.float32(v)) for v in coeffs)
    for _ in range(steps):
        p = x @ np.swapaxes(x, -1, -2)
        x = a * x + (b * p + c * (p @ p)) @ x
    return np.swapaxes(x, -1, -2) if tall else x


def _hold(got, g, dtype, size, steps=5, coeffs=(A, B, C), eps=EPS):
    """An FP32 result is held to three times the error of the formula evaluated in FP32 and, beside it, 22-bit operands' rounding of
    X_0 grown 480-fold (`size` is X_0's norm); a BF16 one to its own rounding and the noise of operands of 16 bits."""
    import torch
    want, yard = _plain(g, np.float64, steps, coeffs, eps), _plain(g, np.float32, steps, coeffs, eps).astype(np.float64)
    err = np.linalg.norm(got - want)
    if dtype == "bfloat16":
        tol = torch.finfo(torch.bfloat16).eps / 2 * np.linalg.norm(want) + 480 * 5 ** 0.5 * 2.0 ** -18 * size
    else:
        tol = 3 * np.linalg.norm(yard - want) + 480 * 2.0 ** -24 * size
    assert np.all(np.isfinite(got)) and err <= tol, (err / np.linalg.norm(want), tol / np.linalg.norm(want))


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (5, 5), (16, 16), (12, 40), (150, 150)], ids=str)
def test_matrices_with_one_entry_a_row(cake, shape):
    """Every sum is one product, so nothing is truncated and nothing may be put back: what is left are the roundings of
    the formula itself in FP32, some six of 2^-24 a step, grown by its slope (at most 3.5, and 1.1 near its cycle)."""
    import torch
    n = min(shape)
    g = np.zeros(shape, np.float32)
    g[np.arange(n), np.arange(n)] = 1.0
    want = _plain(g, np.float64, eps=0.0)
    got = cake.cake_orthogonalize(torch.from_numpy(g).cuda(), eps=0.0).double().cpu().numpy()
    assert np.all(got[g == 0] == 0)
    assert float(np.abs(got - want).max()) <= 5 * 6 * 2.0 ** -24 * 3.5 * float(np.abs(want).max())


@pytest.mark.parametrize("pair", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 4, 16, 64, 256])
def test_powers_of_two_stay_exact(cake, n, pair):
    """X_0 of the identity is 2^-k of it, every product after it is exact, and so is the result.  What truncation takes from sums
    that grow is put back by their number of additions: none where up to 16 values are summed, and never in Q X."""
    import torch
    G = torch.eye(n, device="cuda")
    x = n ** -0.5
    cake.set_option("pair", pair)
    try:
        for coeffs, want in (((1.0, 0.0, 0.0), x), ((0.0, 1.0, 0.0), x ** 3), ((0.0, 0.0, 1.0), x ** 5)):
            if n <= 16 or coeffs[0]:
                assert torch.equal(cake.cake_orthogonalize(G, steps=1, coeffs=coeffs, eps=0.0), want * G)
    finally:
        cake.set_option("pair", 0)
