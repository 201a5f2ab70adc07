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
    """An FP32 result is held to three times the error of the formula evaluated in FP32, the rounding of X_0 (`size` is its norm) grown
    480-fold, and what a step adds to X: the tensor core truncates a sum at most eight times between folds, seven times after its
    largest term came in, below 2^-23 of it each; X and Q are rounded to 22 bits and a sign, and the fold to 24: three times
    2^-23.  A BF16 result to its own rounding and the noise of operands of 16 bits."""
    import torch
    want, yard = _plain(g, np.float64, steps, coeffs, eps), _plain(g, np.float32, steps, coeffs, eps).astype(np.float64)
    err = np.linalg.norm(got - want)
    if dtype == "bfloat16":
        tol = torch.finfo(torch.bfloat16).eps / 2 * np.linalg.norm(want) + 480 * 5 ** 0.5 * 2.0 ** -18 * size
    else:
        tol = 3 * np.linalg.norm(yard - want) + 480 * 2.0 ** -24 * size + steps * 10 * 2.0 ** -23 * np.linalg.norm(want)
    assert np.all(np.isfinite(got)) and err <= tol, (err / np.linalg.norm(want), tol / np.linalg.norm(want))


@pytest.mark.parametrize("pair", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(64, 90), (200, 70), (96, 960), (150, 210), (300, 256)], ids=str)
def test_gradients_far_below_eps(cake, shape, dtype, pair):
    """X_0 = G / (|G| + eps) is then small as a whole, and no less accurate for it."""
    import torch
    rng = np.random.default_rng(shape[0])
    unit = rng.standard_normal(shape)
    unit /= np.linalg.norm(unit)
    cake.set_option("pair", pair)
    try:
        for norm in (1.0, 1e-6, 3e-7, 1e-7, 2e-8, 1e-9, 1e-11, 1e-13, 1e-16, 1e-25):
            G = torch.from_numpy((unit * norm).astype(np.float32)).to(getattr(torch, dtype))
            got = cake.cake_orthogonalize(G.cuda()).double().cpu().numpy()
            _hold(got, G.double().numpy(), dtype, norm / (norm + EPS))
    finally:
        cake.set_option("pair", 0)


@pytest.mark.parametrize("shape", [(64, 90), (150, 210)], ids=str)
def test_a_batch_of_unlike_sizes(cake, shape):
    """Matrices of one batch, each with a norm of its own, give what they give alone."""
    import torch
    torch.manual_seed(0)
    G = torch.randn((6,) + shape, device="cuda") * torch.tensor([1e-15, 1.0, 1e-9, 0.0, 1e-7, 1e3], device="cuda")[:, None, None]
    O = cake.cake_orthogonalize(G)
    for i in range(6):
        assert torch.equal(O[i], cake.cake_orthogonalize(G[i]))
    assert bool((O[3] == 0).all())


@pytest.mark.parametrize("shape", [(40, 100), (211, 197)], ids=str)
def test_a_step_along_a_tiny_gradient(cake, shape):
    import torch
    rng = np.random.default_rng(shape[0])
    G = torch.from_numpy((rng.standard_normal(shape) * 1e-14).astype(np.float32))
    W, M = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    cake.cake_muon_step(W, G.cuda(), M, 1.0, momentum=0.0, nesterov=False, scale=1.0)
    g = G.double().numpy()
    norm = np.linalg.norm(g)
    _hold(-W.double().cpu().numpy(), g, "float32", norm / (norm + EPS))


@pytest.mark.parametrize("shape", [(100, 140), (150, 210)], ids=str)
def test_coefficients_that_shrink_or_grow(cake, shape):
    """Singular values that leave (0, 1.2], also far, and coefficients that let those near one run away, where there are none."""
    import torch
    rng = np.random.default_rng(shape[0])
    g = rng.standard_normal(shape).astype(np.float32)
    d = torch.from_numpy(g).cuda()
    for steps, coeffs in ((20, (0.5, 0.0, 0.0)), (3, (0.1, 0.3, -0.2)), (3, (4.0, 0.0, 0.0)), (2, (6.0, -3.0, 1.0)), (1, (100.0, 0.0, 0.0)), (64, (1.0, 0.0, 0.0)),
                          (64, (1.5, -0.5, 0.0)), (4, (-2.0, 1.5, -0.5)), (5, (100.0, 0.0, 0.0)), (30, (2.0, 0.0, 0.0)), (1, (1e6, 0.0, 0.0)), (2, (3.0, 3.0, 3.0)),
                          (3, (3.0, 3.0, 3.0)), (1, (0.0, 1.0, 0.0)), (64, (0.3, 0.0, 0.0))):
        want, yard = _plain(g, np.float64, steps, coeffs), _plain(g, np.float32, steps, coeffs).astype(np.float64)
        got = cake.cake_orthogonalize(d, steps=steps, coeffs=coeffs).double().cpu().numpy()
        # operands of 22 bits: three roundings a step of 2^-23 each, a power of x up to the fifth
        err, size = np.linalg.norm(got - want), np.linalg.norm(want)
        assert err <= 3 * np.linalg.norm(yard - want) + 8 * steps * 2.0 ** -22 * size, (steps, coeffs, err / size)
    for steps, coeffs in ((2, (float("inf"), 0.0, 0.0)), (2, (1.0, float("nan"), 0.0))):
        with pytest.raises(cake.CakeError):
            cake.cake_orthogonalize(d, steps=steps, coeffs=coeffs)
        with pytest.raises(cake.CakeError):
            cake.cake_muon_step(d.clone(), d, torch.zeros_like(d), 0.1, steps=steps, coeffs=coeffs)


@pytest.mark.parametrize("shape", [(20, 30), (150, 210)], ids=str)
def test_a_large_result_that_fp32_holds(cake, shape):
    """X grows to 1e35, and its square, which nothing needs, is beyond FP32: coefficients of zero stay zero."""
    import torch
    rng = np.random.default_rng(shape[0])
    g = rng.standard_normal(shape).astype(np.float32)
    got = cake.cake_orthogonalize(torch.from_numpy(g).cuda(), steps=18, coeffs=(100.0, 0.0, 0.0)).double().cpu().numpy()
    want = g.astype(np.float64) / (np.linalg.norm(g.astype(np.float64)) + np.float64(np.float32(EPS))) * 1e36
    # 18 roundings of X to 22 bits and a sign, and of 100, which 22 bits hold
    assert np.all(np.abs(got - want) <= 18 * 2.0 ** -22 * np.abs(want))


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
