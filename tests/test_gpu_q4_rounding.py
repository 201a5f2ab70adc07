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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 7, 12, 40, 90])
def test_large_features_of_zero_weights_leave_nothing(cake, rows, dtype, expanded):
    """Codes equal to their zero point are weights of zero, exactly, however large the feature is: errors go with sum |x| |w|."""
    import torch
    rng = np.random.default_rng(rows)
    N, K, group = 40, 384, 128
    for zeros in (False, None):
        z = rng.integers(0, 16, (N, K // group), dtype=np.uint8) if zeros is None else False
        q = rng.integers(0, 16, (N, K), dtype=np.uint8)
        for k in (5, 130, 131, 300):
            q[:, k] = 8 if z is False else z[:, k // group]
        W4, w = _make(cake, rng, N, K, group, z, torch.float16, q)
        t = getattr(torch, dtype)
        x = torch.from_numpy(0.1 * rng.standard_normal((rows, K)).astype(np.float32))
        x[:, 5], x[:, 130], x[:, 131], x[:, 300] = 60000.0, -31000.0, 47001.0, 12345.0
        x = x.to(t)
        got = cake.cake_q4_linear(x.cuda(), W4).double().cpu().numpy()
        a = x.double().numpy()
        want, S = a @ w.T, np.abs(a) @ np.abs(w).T
        operand = 0.0 if rows <= 64 or not expanded else {"float32": 2.0 ** -22, "float16": 2.0 ** -14, "bfloat16": 0.0}[dtype]
        tol = torch.finfo(t).eps / 2 * np.abs(want) * (1 + 2 ** -20) + ((K / 16 + 40) * 2.0 ** -22 + operand) * S
        assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_sums_of_one_product_are_exact(cake, rows, dtype, expanded):
    """One feature per row, the rest zero: x = 1 gives the weight itself, rounded once."""
    import torch
    rng = np.random.default_rng(rows)
    N, K, group = 100, 330, 64
    W4, w = _make(cake, rng, N, K, group, None, torch.float16)
    t = getattr(torch, dtype)
    for dx in (False, True):
        n = N if dx else K
        at = rng.integers(0, n, rows)
        x = torch.zeros((rows, n), dtype=t)
        x[torch.arange(rows), torch.from_numpy(at)] = 1.0
        y = (cake.cake_q4_linear_dx if dx else cake.cake_q4_linear)(x.cuda(), W4)
        want = torch.from_numpy(w[at] if dx else w[:, at].T.copy()).to(t)
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("rows", [3, 65, 200])
def test_ends_of_the_range_of_fp32(cake, rows, expanded):
    """The terms of an FP32 x neither overflow nor lose the smallest normal values, with few rows and with many."""
    import torch
    rng = np.random.default_rng(rows)
    W4, _ = _make(cake, rng, 16, 200, 64, False, torch.float16, np.full((16, 200), 9, np.uint8), 1.0)  # w = 1
    x = torch.zeros((rows, 200), device="cuda")
    x[0, 3], x[1, 5], x[2, 0] = torch.finfo(torch.float32).max, 1.1754944e-38 * 65536, 1 + 2.0 ** -23
    y = cake.cake_q4_linear(x, W4)
    assert torch.equal(y, x.sum(1, keepdim=True).expand(rows, 16))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 8, 30])
def test_gradients_of_few_rows_are_cut_on_either_side(cake, rows, dtype):
    """dy s goes into the product as two terms within 2^-17 of it.  With 16 output features a sum is one multiplication of 16 pairs, twice: four
    roundings of 2^-23 at most.  So a result is the correctly rounded one unless a border between two of them lies as near as that."""
    import torch
    rng = np.random.default_rng(rows)
    N, K = 16, 4000
    z = np.zeros((N, K // 32), dtype=np.uint8)
    W4, w = _make(cake, rng, N, K, 32, z, torch.float16)
    t = getattr(torch, dtype)
    dy = torch.from_numpy(np.abs(rng.standard_normal((rows, N))).astype(np.float32)).to(t)
    want = dy.double().numpy() @ w  # of positive terms
    got = cake.cake_q4_linear_dx(dy.cuda(), W4).double().cpu().numpy()
    _, e = np.frexp(want)
    ulp = np.ldexp(torch.finfo(t).eps, e - 1)
    assert np.all(np.abs(got - want) <= ulp / 2 + want * (2.0 ** -17 + 4 * 2.0 ** -23))
