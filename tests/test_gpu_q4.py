"""Products with weights held in 4 bits (Q4Weights, cake_q4_linear, cake_q4_linear_dx) against float64 on the host.

Tolerance of a product, element by element, with S = sum_k |x| |w| in float64:
    half a step of the result's type on |y|                                  finfo(t).eps / 2 * |y|
    FP32 summation: a row's K products enter at most K / 16 + 40 additions one after the other (16 products per
    tensor-core addition, which may drop bits below 2^-23 of the larger term; at most 8 warps x 8 CTAs and the scale's
    product on top), each off by at most 2^-22 S                             (K / 16 + 40) 2^-22 S
    operands: 16-bit x is exact, FP32 x is exact as three terms; the gradient's dy s is formed in FP32 (2^-24) and cut
    to two bf16 terms for 16-bit types (2^-15 of S at most), three for FP32 (2^-23).  From 65 rows on the weights are
    expanded, in bf16 planes.  A bf16 has 8 significant bits, so rounding to it is off by at most 2^-8 of the value and
    cutting by less than 2^-7.  BF16: one rounding, 2^-8.  FP16: w in two planes, 2^-8 2^-8; x exact in two cut ones;
    left out is the product of the second planes, 2^-7 2^-8: together below 2^-14.  FP32: w exact in two planes (11 bits of
    scale times 5 of a code), x exact in three cut ones, left out is the last of x (2^-14) by the second of w (2^-8): 2^-22
Errors of the additions have no common sign, so over a whole result they add up like a random walk: the 2-norm of the error
of an FP32 result is held to sqrt(K / 16 + 40) 2^-22 times the 2-norm of sqrt(sum x^2 w^2), the walk's own size.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _codes(rng, N, K, group, with_zeros, scale_dtype):
    import torch
    G = -(-K // group)
    q = rng.integers(0, 16, (N, K + (K & 1)), dtype=np.uint8)
    q[0, :] = 15
    q[-1, :] = 0
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).astype(np.uint8)
    scales = torch.from_numpy(rng.uniform(0.002, 0.05, (N, G)).astype(np.float32)).to(scale_dtype)
    zeros = rng.integers(0, 16, (N, G), dtype=np.uint8) if with_zeros else None
    z = np.full((N, G), 8.0) if zeros is None else zeros.astype(np.float64)
    at = np.arange(K) // group
    w = scales.double().numpy()[:, at] * (q[:, :K].astype(np.float64) - z[:, at])
    return codes, scales, zeros, w


def _weights(cake, codes, scales, zeros, group, K):
    import torch
    return cake.Q4Weights(torch.from_numpy(codes).cuda(), scales.cuda(), None if zeros is None else torch.from_numpy(zeros).cuda(), group=group,
                          in_features=K)


def _random(rng, shape, dtype):
    import torch
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(getattr(torch, dtype))


def _hold(got, want, S, walk, K, dtype, operand):
    import torch
    eps = torch.finfo(getattr(torch, dtype)).eps
    tol = eps / 2 * np.abs(want) * (1 + 2 ** -20) + ((K / 16 + 40) * 2.0 ** -22 + operand) * S
    err = np.abs(got - want)
    assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())
    if dtype == "float32":
        assert np.linalg.norm(err) <= (np.sqrt(K / 16 + 40) * 2.0 ** -22 + 2.0 ** -24) * np.linalg.norm(walk) + eps / 2 * np.linalg.norm(want)


MANY = {"float32": 2.0 ** -22, "float16": 2.0 ** -14, "bfloat16": 2.0 ** -8}
SHAPES = [  # rows, N, K, group
    (1, 1, 1, 32), (1, 16, 64, 64), (1, 100, 1000, 128), (2, 17, 33, 32), (3, 15, 65, 64), (5, 129, 127, 32), (7, 33, 129, 128),
    (8, 64, 200, 64), (9, 31, 96, 32), (16, 48, 2111, 128), (17, 20, 320, 64), (25, 40, 63, 32), (33, 50, 130, 128), (70, 19, 257, 64),
    (1, 2500, 511, 32), (4, 300, 4200, 128), (150, 130, 190, 64), (300, 520, 700, 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_and_gradient(cake, shape, dtype):
    import torch
    rows, N, K, group = shape
    rng = np.random.default_rng(rows * 7919 + N * 31 + K)
    with_zeros = (N + K) % 2 == 1
    scale_dtype = torch.float16 if K % 3 else torch.bfloat16
    codes, scales, zeros, w = _codes(rng, N, K, group, with_zeros, scale_dtype)
    W4 = _weights(cake, codes, scales, zeros, group, K)
    assert np.array_equal(W4.dequantize().double().cpu().numpy(), w.astype(np.float32).astype(np.float64))
    x, dy, b = _random(rng, (rows, K), dtype), _random(rng, (rows, N), dtype), _random(rng, (N,), dtype)
    x64, dy64, b64 = x.double().numpy(), dy.double().numpy(), b.double().numpy()
    for bias in (None, b):
        y = cake.cake_q4_linear(x.cuda(), W4, None if bias is None else bias.cuda())
        assert y.dtype == x.dtype and tuple(y.shape) == (rows, N)
        add = 0 if bias is None else b64[None]
        _hold(y.double().cpu().numpy(), x64 @ w.T + add, np.abs(x64) @ np.abs(w).T + np.abs(add), np.sqrt(x64 ** 2 @ (w ** 2).T + np.square(add)), K, dtype,
              MANY[dtype] if rows >= 65 else 0.0)
    dx = cake.cake_q4_linear_dx(dy.cuda(), W4)
    _hold(dx.double().cpu().numpy(), dy64 @ w, np.abs(dy64) @ np.abs(w), np.sqrt(dy64 ** 2 @ w ** 2), N, dtype,
          MANY[dtype] if rows >= 65 else 2.0 ** -22 if dtype == "float32" else 2.0 ** -14)
    # the same call gives the same bits
    assert torch.equal(cake.cake_q4_linear_dx(dy.cuda(), W4), dx)


@pytest.fixture(params=[False, True], ids=["", "expanded"])
def expanded(cake, request):
    """Second time round: products with more than 64 rows expand the weights whatever their sizes."""
    cake.set_option("pair", 2 if request.param else 0)
    yield request.param
    cake.set_option("pair", 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] > 64] + [(65, 33, 129, 32), (257, 300, 512, 128), (1024, 70, 96, 32), (1025, 70, 96, 32)], ids=str)
def test_more_than_64_rows_of_small_weights(cake, shape, dtype, expanded):
    """Both ways, and where one ends.  Without the expansion the tolerance is that of few rows."""
    import torch
    rows, N, K, group = shape
    rng = np.random.default_rng(rows + N)
    codes, scales, zeros, w = _codes(rng, N, K, group, rows % 2 == 0, torch.bfloat16)
    W4 = _weights(cake, codes, scales, zeros, group, K)
    x, dy, b = _random(rng, (rows, K), dtype), _random(rng, (rows, N), dtype), _random(rng, (N,), dtype)
    x64, dy64, b64 = x.double().numpy(), dy.double().numpy(), b.double().numpy()
    many = expanded or rows > 1024
    y = cake.cake_q4_linear(x.cuda(), W4, b.cuda())
    _hold(y.double().cpu().numpy(), x64 @ w.T + b64, np.abs(x64) @ np.abs(w).T + np.abs(b64), np.sqrt(x64 ** 2 @ (w ** 2).T + b64 ** 2), K, dtype,
          MANY[dtype] if many else 0.0)
    dx = cake.cake_q4_linear_dx(dy.cuda(), W4)
    _hold(dx.double().cpu().numpy(), dy64 @ w, np.abs(dy64) @ np.abs(w), np.sqrt(dy64 ** 2 @ w ** 2), N, dtype,
          MANY[dtype] if many else 2.0 ** -22 if dtype == "float32" else 2.0 ** -14)


@pytest.mark.parametrize("form", [(0, 0), (1, 1), (1, 3), (2, 1), (2, 4)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_in_every_form(cake, dtype, form):
    """Pairs and single SMs, tiles whole and cut along K, and more weights than one slab holds."""
    rng = np.random.default_rng(21)
    cake.set_option("pair", form[0])
    cake.set_option("k_pieces", form[1])
    try:
        for (rows, N, K, group) in [(65, 1000, 900, 128), (333, 260, 1500, 32)] + ([(129, 40, 70000, 64), (70, 33100, 1100, 64)] if form == (0, 0) else []):
            import torch
            codes, scales, zeros, w = _codes(rng, N, K, group, rows % 2 == 0, torch.float16)
            W4 = _weights(cake, codes, scales, zeros, group, K)
            x, dy, b = _random(rng, (rows, K), dtype), _random(rng, (rows, N), dtype), _random(rng, (N,), dtype)
            x64, dy64, b64 = x.double().numpy(), dy.double().numpy(), b.double().numpy()
            y = cake.cake_q4_linear(x.cuda(), W4, b.cuda()).double().cpu().numpy()
            _hold(y, x64 @ w.T + b64, np.abs(x64) @ np.abs(w).T + np.abs(b64), np.sqrt(x64 ** 2 @ (w ** 2).T + b64 ** 2), K, dtype, MANY[dtype])
            dx = cake.cake_q4_linear_dx(dy.cuda(), W4).double().cpu().numpy()
            _hold(dx, dy64 @ w, np.abs(dy64) @ np.abs(w), np.sqrt(dy64 ** 2 @ w ** 2), N, dtype, MANY[dtype])
    finally:
        cake.set_option("pair", 0)
        cake.set_option("k_pieces", 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_strides_alignment_and_what_lies_around_the_result(cake, rows, dtype, expanded):
    """Rows inside wider allocations, at an address that is only aligned to the element, and a result inside one."""
    import torch
    rng = np.random.default_rng(rows)
    N, K, group = 75, 168, 32
    codes, scales, zeros, w = _codes(rng, N, K, group, True, torch.float16)
    W4 = _weights(cake, codes, scales, zeros, group, K)
    t = getattr(torch, dtype)
    for off, extra in ((1, 2), (8, 16), (3, 0)):
        big = torch.full((rows, off + K + extra), float("nan"), dtype=t, device="cuda")
        x = _random(rng, (rows, K), dtype).cuda()
        big[:, off:off + K] = x
        frame = torch.full((rows, N + 9), 7.0, dtype=t, device="cuda")
        y = cake.cake_q4_linear(big[:, off:off + K], W4, out=frame[:, 4:4 + N])
        assert torch.equal(y, cake.cake_q4_linear(x, W4))
        assert bool((frame[:, :4] == 7).all()) and bool((frame[:, 4 + N:] == 7).all())
        dy = _random(rng, (rows, N), dtype).cuda()
        wide = torch.full((rows, N + 5), float("nan"), dtype=t, device="cuda")
        wide[:, 5:] = dy
        frame = torch.full((rows, K + 9), 7.0, dtype=t, device="cuda")
        dx = cake.cake_q4_linear_dx(wide[:, 5:], W4, out=frame[:, 1:1 + K])
        assert torch.equal(dx, cake.cake_q4_linear_dx(dy, W4))
        assert bool((frame[:, :1] == 7).all()) and bool((frame[:, 1 + K:] == 7).all())


def test_leading_dimensions_vectors_and_no_rows(cake):
    import torch
    rng = np.random.default_rng(5)
    codes, scales, zeros, w = _codes(rng, 40, 64, 64, False, torch.bfloat16)
    W4 = _weights(cake, codes, scales, zeros, 64, 64)
    x = _random(rng, (2, 3, 64), "float32").cuda()
    y = cake.cake_q4_linear(x, W4)
    assert tuple(y.shape) == (2, 3, 40)
    assert torch.equal(y[1, 2], cake.cake_q4_linear(x[1, 2], W4))  # a row's result does not depend on its neighbours
    assert tuple(cake.cake_q4_linear(x[:0], W4).shape) == (0, 3, 40)
    assert tuple(cake.cake_q4_linear_dx(torch.empty((0, 40), device="cuda"), W4).shape) == (0, 64)
    with pytest.raises(TypeError):
        cake.cake_q4_linear(x.transpose(0, 1), W4)  # rows that are not evenly spaced
    with pytest.raises(TypeError):
        cake.cake_q4_linear(x[0].t().contiguous().t(), W4)
    with pytest.raises(TypeError):
        cake.cake_q4_linear(x[0, :1].expand(4, 64), W4, out=torch.empty((1, 40), device="cuda").expand(4, 40))
    with pytest.raises(ValueError):
        cake.cake_q4_linear(x[..., :32], W4)
    with pytest.raises(TypeError):
        cake.cake_q4_linear(x.double(), W4)
    with pytest.raises(TypeError):
        cake.cake_q4_linear(x, W4, torch.zeros(40, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        cake.cake_q4_linear(x, W4, torch.zeros(41, device="cuda"))
    with pytest.raises(ValueError):
        cake.Q4Weights(torch.from_numpy(codes).cuda(), scales.cuda(), torch.full((40, 1), 16, dtype=torch.uint8, device="cuda"), group=64)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_row(cake, dtype, expanded):
    import torch
    rng = np.random.default_rng(11)
    N, K = 35, 150
    codes, scales, zeros, w = _codes(rng, N, K, 64, False, torch.float16)
    codes[:, :] = 0x9C  # codes 12 and 9: no weight is zero, so infinity times it is infinite
    W4 = _weights(cake, codes, scales, zeros, 64, K)
    for rows in (4, 12, 80):
        x = _random(rng, (rows, K), dtype).cuda()
        clean = cake.cake_q4_linear(x, W4)
        x[1, 7], x[2, 149] = float("inf"), float("nan")
        y = cake.cake_q4_linear(x, W4)
        # (an infinity meets itself where offsets or second planes are taken out again, so what comes of it may be a NaN)
        assert bool((~torch.isfinite(y[1])).all()) and bool(torch.isnan(y[2]).all())
        keep = [r for r in range(rows) if r not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])


def test_largest_and_smallest_values_of_fp32(cake):
    """The three terms of an FP32 x neither overflow nor lose the smallest normal values."""
    import torch
    W4 = _weights(cake, np.full((16, 32), 0x99, np.uint8), torch.ones((16, 1), dtype=torch.float16), None, 64, 64)  # w = 1
    x = torch.zeros((3, 64), device="cuda")
    x[0, 3], x[1, 5], x[2, 0] = torch.finfo(torch.float32).max, 1.1754944e-38 * 65536, 1 + 2.0 ** -23
    y = cake.cake_q4_linear(x, W4)
    assert torch.equal(y, x.sum(1, keepdim=True).expand(3, 16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("scale_name", ["float16", "bfloat16"])
def test_quantize(cake, dtype, symmetric, scale_name):
    """The stored numbers follow the documented formulas, and a code is the nearest one to its weight."""
    import torch
    rng = np.random.default_rng(3)
    for (N, K, group) in [(5, 1, 32), (9, 67, 32), (33, 300, 64), (4, 129, 128)]:
        W = _random(rng, (N, K + 3), dtype) * 0.1
        W[0] = 0
        if not symmetric and N > 5:
            W[1] = W[1].abs()  # a range that does not straddle zero
        W = W[:, 1:1 + K]
        codes, scales, zeros = cake.Q4Weights.quantize_codes(W.cuda(), group, symmetric, getattr(torch, scale_name))
        G = -(-K // group)
        assert tuple(codes.shape) == (N, (K + 1) // 2) and tuple(scales.shape) == (N, G) and (zeros is None) == symmetric
        w = np.zeros((N, G * group), np.float32)
        w[:, :K] = W.float().numpy()
        w = w.reshape(N, G, group)
        if symmetric:
            s = np.abs(w).max(2) / np.float32(7)
        else:
            s = np.maximum(w.max(2), 0) / np.float32(15) - np.minimum(w.min(2), 0) / np.float32(15)
        s = torch.from_numpy(s).to(getattr(torch, scale_name))
        assert torch.equal(scales.cpu(), s)
        q = codes.cpu().numpy()
        q = np.stack((q & 15, q >> 4), 2).reshape(N, -1)[:, :K].astype(np.float64)
        at = np.arange(K) // group
        s64 = s.double().numpy()[:, at]
        z = 8.0 if symmetric else zeros.cpu().numpy().astype(np.float64)[:, at]
        back = s64 * (q - z)
        # at most half a step away, plus what the clipped ends lose: the scale's own rounding times 8 (15) steps and, with
        # zero points, the rounding of the zero point
        step = torch.finfo(getattr(torch, scale_name)).eps / 2
        assert np.all(np.abs(back - W.double().numpy()) <= s64 * ((0.5 if symmetric else 1.0) + 15 * step + 1e-6))
        W4 = cake.Q4Weights.quantize(W.cuda(), group, symmetric, getattr(torch, scale_name))
        assert np.array_equal(W4.dequantize(torch.float32).double().cpu().numpy(), back.astype(np.float32).astype(np.float64))


def test_quantize_extremes(cake):
    import torch
    W = torch.zeros((4, 64), device="cuda")
    W[0, 3] = float("inf")
    W[1, 40] = 1e30   # clipped to what a float16 scale reaches
    W[2, 5] = 1e-12   # a scale below the smallest float16 becomes that one
    codes, scales, _ = cake.Q4Weights.quantize_codes(W, 32)
    assert bool(torch.isnan(scales[0, 0])) and float(scales[0, 1]) == 0
    assert float(scales[1, 1]) == 65504 and float(scales[2, 0]) == 2.0 ** -24
    back = cake.Q4Weights.quantize(W, 32).dequantize()
    assert float(back[1, 40]) == 7 * 65504 and bool((back[3] == 0).all()) and float(back[2, 5]) == 0
    assert bool((back[1, :32] == 0).all())


def test_streams_and_graphs(cake):
    """A product recorded into a graph and replayed with new inputs, while another one runs on a second stream."""
    import torch
    torch.manual_seed(0)
    W4 = cake.Q4Weights.quantize(torch.randn(700, 520, device="cuda"), 64)
    V4 = cake.Q4Weights.quantize(torch.randn(520, 700, device="cuda"), 128, symmetric=False)
    x, z = torch.randn(5, 520, device="cuda"), torch.randn(9, 700, device="cuda")
    cake.cake_q4_linear(x, W4), cake.cake_q4_linear_dx(z, W4)
    torch.cuda.synchronize()
    y, d = torch.empty(5, 700, device="cuda"), torch.empty(9, 520, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cake.cake_q4_linear(x, W4, out=y)
        cake.cake_q4_linear_dx(z, W4, out=d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for seed in range(3):
        x.normal_(), z.normal_()
        graph.replay()
        with torch.cuda.stream(side):
            other = [cake.cake_q4_linear(z, V4) for _ in range(4)]
        also = cake.cake_q4_linear(z, V4, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(y, cake.cake_q4_linear(x, W4)) and torch.equal(d, cake.cake_q4_linear_dx(z, W4))
        want = cake.cake_q4_linear(z, V4)
        assert all(torch.equal(o, want) for o in other + [also])
        side.wait_stream(torch.cuda.current_stream())
