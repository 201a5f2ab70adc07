"""What rounding leaves in products with 4-bit weights: 16-bit results are rounded once, features whose weight is zero leave
nothing behind, and sums of one product are exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(params=[False, True], ids=["", "expanded"])
def expanded(cake, request):
    """Second time round: products with more than 64 rows expand the weights whatever their sizes."""
    cake.set_option("pair", 2 if request.param else 0)
    yield request.param
    cake.set_option("pair", 0)


def _make(cake, rng, N, K, group, zeros, scale_dtype, q=None, scale=None):
    """(Q4Weights, the matrix in float64, zero points or None)."""
    import torch
    G = -(-K // group)
    q = rng.integers(0, 16, (N, K + (K & 1)), dtype=np.uint8) if q is None else q
    scales = torch.from_numpy(rng.uniform(0.01, 0.03, (N, G)).astype(np.float32) if scale is None else np.full((N, G), scale, np.float32)).to(scale_dtype)
    z = rng.integers(0, 16, (N, G), dtype=np.uint8) if zeros is None else zeros
    at = np.arange(K) // group
    w = scales.double().numpy()[:, at] * (q[:, :K].astype(np.float64) - (8.0 if z is False else z.astype(np.float64)[:, at]))
    codes = torch.from_numpy((q[:, 0::2] | (q[:, 1::2] << 4)).astype(np.uint8)).cuda()
    W4 = cake.Q4Weights(codes, scales.cuda(), None if z is False else torch.from_numpy(z).cuda(), group=group, in_features=K)
    return W4, w


def _one_rounding(want, dtype):
    """2-norm of the errors of one rounding each: an error is spread evenly over a unit in the last place, so its
    square is ulp^2 / 12 in the mean.  Over some thousand results the mean is off by less than a tenth (five deviations and more)."""
    import torch
    _, e = np.frexp(want)
    ulp = np.ldexp(torch.finfo(getattr(torch, dtype)).eps, e - 1)
    return 1.1 * np.sqrt((ulp ** 2).sum() / 12)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [20, 130, 400])
@pytest.mark.parametrize("group", [32, 128])
def test_16_bit_results_are_rounded_once(cake, rows, group, dtype, expanded):
    """The error of a 16-bit result is that of its own rounding: sums in FP32 (a random walk of K / 16 + 40 additions, 2^-22 each)
    and, between them, at most the second terms' product of FP16 planes (cut below 2^-7, rounded to 2^-8) or the cut of dy s
    below 2^-14, are smaller by far."""
    import torch
    rng = np.random.default_rng(rows + group)
    N, K = 210, 700
    W4, w = _make(cake, rng, N, K, group, None, torch.float16)
    t = getattr(torch, dtype)
    x, dy = (torch.from_numpy(rng.standard_normal((rows, n)).astype(np.float32)).to(t) for n in (K, N))
    for got, a, b, depth in ((cake.cake_q4_linear(x.cuda(), W4), x.double().numpy(), w.T, K), (cake.cake_q4_linear_dx(dy.cuda(), W4), dy.double().numpy(), w, N)):
        want, walk = a @ b, np.sqrt(a ** 2 @ b ** 2)
        err = np.linalg.norm(got.double().cpu().numpy() - want)
        tol = _one_rounding(want, dtype) + (np.sqrt(depth / 16 + 40) * 2.0 ** -22 + 2.0 ** -14) * np.linalg.norm(walk)
        assert err <= tol, (err / np.linalg.norm(want), tol / np.linalg.norm(want))
