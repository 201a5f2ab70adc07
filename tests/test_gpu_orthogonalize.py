"""Orthogonalised updates (cake_orthogonalize, cake_muon_step, cake_muon) against float64 on the host.

Error model.  The norm of X is 1 at the start and a rounding of relative size u puts noise of norm u into it.  A step multiplies
a small singular direction by a = 3.44, so noise beside it grows 480-fold in five steps; products of unit roundoff u put in as
much again at every step.  Hence
    BF16 results (operands of 16 bits, u = 2^-17):  |error|_F <= finfo.eps / 2 * |O|_F (the result's rounding)  +  480 sqrt(5) 2^-18
    FP32 results (24 bits):  the formula evaluated in FP32 on the host has the same kind of error; its size on the same
    input is the yardstick: |error|_F <= 3 |error of that|_F + 480 2^-24.
A single wrong element of ordinary size is far above either for the sizes here; single elements are held to 32 times
their share of the bound.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


def _plain(G, dtype, steps=5, coeffs=(A, B, C), eps=1e-7):
    x = G.astype(np.float64)
    x = (x / (np.sqrt((x * x).sum((-2, -1), keepdims=True)) + eps)).astype(dtype)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = np.swapaxes(x, -1, -2)
    a, b, c = (dtype(v) for v in coeffs)
    for _ in range(steps):
        p = x @ np.swapaxes(x, -1, -2)
        x = a * x + (b * p + c * (p @ p)) @ x
    return np.swapaxes(x, -1, -2) if tall else x


def _gradient(rng, rows, cols, kind):
    if kind == "noise":
        return rng.standard_normal((rows, cols)) * 1e-3
    # few tokens of unlike size, as backward leaves them: most singular values are tiny
    t = max(1, min(rows, cols) // 3)
    y = rng.standard_normal((t, rows)) * np.exp(0.5 * rng.standard_normal((1, rows)))
    x = rng.standard_normal((t, cols)) * np.exp(0.5 * rng.standard_normal((1, cols)))
    return y.T @ x / t + 0.02 * rng.standard_normal((rows, cols))


def _hold(got, want, yard, dtype):
    import torch
    err = np.abs(got - want)
    assert np.all(np.isfinite(got))
    if dtype == "bfloat16":
        tol = torch.finfo(torch.bfloat16).eps / 2 * np.linalg.norm(want) + 480 * 5 ** 0.5 * 2.0 ** -18
    else:
        tol = 3 * np.linalg.norm(yard - want) + 480 * 2.0 ** -24
    assert np.linalg.norm(err) <= tol, (np.linalg.norm(err), tol)
    assert err.max() <= 32 * tol / np.sqrt(err.size) or err.size < 64


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (8, 8), (31, 33), (33, 31), (64, 64), (64, 200), (96, 960), (127, 129), (130, 70), (128, 384),
          (257, 300), (520, 261), (513, 1030)]


@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_one_matrix(cake, shape, dtype, pair):
    import torch
    rng = np.random.default_rng(shape[0] * 1009 + shape[1])
    cake.set_option("pair", pair)
    try:
        for kind in ("noise", "tokens"):
            G = torch.from_numpy(_gradient(rng, *shape, kind).astype(np.float32)).to(getattr(torch, dtype))
            keep = G.clone()
            d = G.cuda()
            O = cake.cake_orthogonalize(d)
            assert O.dtype == G.dtype and O.shape == G.shape and torch.equal(d.cpu(), keep)
            g = G.double().numpy()
            _hold(O.double().cpu().numpy(), _plain(g, np.float64), _plain(g, np.float32).astype(np.float64), dtype)
            assert torch.equal(cake.cake_orthogonalize(d), O)  # the same bits every time
            assert cake.cake_orthogonalize(d, out=d) is d and torch.equal(d, O)  # in place
    finally:
        cake.set_option("pair", 0)


@pytest.mark.parametrize("form", [(1, 0), (1, 1), (1, 2), (1, 4), (2, 0), (2, 1), (2, 2), (2, 5), (2, 8)], ids=str)
@pytest.mark.parametrize("shape", [(31, 33), (130, 700), (520, 261)], ids=str)
def test_forms_of_the_product(cake, shape, form):
    """Every form the products can take (pairs or single SMs, units sharing a tile), several matrices at once."""
    import torch
    rng = np.random.default_rng(shape[1])
    G = np.stack([_gradient(rng, *shape, kind) for kind in ("noise", "tokens")]).astype(np.float32)
    cake.set_option("pair", form[0])
    cake.set_option("k_pieces", form[1])
    try:
        O = cake.cake_orthogonalize(torch.from_numpy(G).cuda()).double().cpu().numpy()
    finally:
        cake.set_option("pair", 0)
        cake.set_option("k_pieces", 0)
    for o, g in zip(O, G.astype(np.float64)):
        _hold(o, _plain(g, np.float64), _plain(g, np.float32).astype(np.float64), "float32")


# (batch, rows, cols): one CTA per matrix, with one and two squares of 128 columns; clusters of 2, 4 and 8; ends inside an
# eight, a block of 32 and a square; the last sizes that fit, and the first ones that do not
SMALL = [(1, 128, 128), (150, 65, 130), (150, 128, 256), (80, 33, 257), (40, 97, 1000), (1, 128, 2048), (1, 2, 2047), (3, 100, 1025), (20, 127, 1111),
         (1, 129, 128), (1, 128, 2056), (60, 30, 1300)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tall", [False, True], ids=["wide", "tall"])
@pytest.mark.parametrize("size", SMALL, ids=str)
def test_small_matrices(cake, size, tall, dtype):
    """Matrices that stay in the shared memory of a cluster from the first step to the last, inside wider rows: nothing around
    the result changes, and the same bits come every time."""
    import torch
    rng = np.random.default_rng(size[0] + size[2])
    b, m, n = size
    r, c = (n, m) if tall else (m, n)
    G = torch.from_numpy(np.stack([_gradient(rng, r, c, ("noise", "tokens")[i % 2]) for i in range(b)]).astype(np.float32)).to(getattr(torch, dtype))
    frame = torch.full((b, r + 1, c + 13), 7.0, dtype=G.dtype, device="cuda")
    O = frame[:, :r, 5:5 + c]
    cake.cake_orthogonalize(G.cuda(), out=O)
    for i in sorted({0, b // 2, b - 1}):
        g = G[i].double().numpy()
        _hold(O[i].double().cpu().numpy(), _plain(g, np.float64), _plain(g, np.float32).astype(np.float64), dtype)
    assert torch.equal(cake.cake_orthogonalize(G.cuda()), O)
    O.fill_(7.0)
    assert bool((frame == 7).all())


@pytest.mark.parametrize("pair", [1, 2])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_tiles(cake, dtype, pair):
    """More tiles than there are SMs (or pairs of them): every CTA walks several."""
    import torch
    rng = np.random.default_rng(4)
    G = torch.from_numpy(_gradient(rng, 2300, 2900, "noise").astype(np.float32)).to(getattr(torch, dtype))
    cake.set_option("pair", pair)
    try:
        O = cake.cake_orthogonalize(G.cuda(), steps=2).double().cpu().numpy()
    finally:
        cake.set_option("pair", 0)
    g = G.double().numpy()
    _hold(O, _plain(g, np.float64, 2), _plain(g, np.float32, 2).astype(np.float64), dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(3, 40, 100), (5, 150, 130), (2, 1, 5), (170, 20, 24)], ids=str)
def test_batches_and_strides(cake, shape, dtype):
    """Matrices inside wider rows, rows apart, batches apart, at addresses that are only aligned to the element; nothing
    around the result changes, and every matrix of a batch is what it is alone."""
    import torch
    rng = np.random.default_rng(shape[0])
    t = getattr(torch, dtype)
    b, r, c = shape
    G = torch.from_numpy(np.stack([_gradient(rng, r, c, "noise") for _ in range(b)]).astype(np.float32)).to(t).cuda()
    O = cake.cake_orthogonalize(G)
    for i in range(0, b, max(1, b // 3)):
        assert torch.equal(cake.cake_orthogonalize(G[i]), O[i])
        g = G[i].double().cpu().numpy()
        _hold(O[i].double().cpu().numpy(), _plain(g, np.float64), _plain(g, np.float32).astype(np.float64), dtype)
    for off in (1, 8):
        big = torch.full((b, r + 2, c + 2 * off), float("nan"), dtype=t, device="cuda")
        big[:, 1:1 + r, off:off + c] = G
        frame = torch.full((b, r + 3, c + 9), 7.0, dtype=t, device="cuda")
        cake.cake_orthogonalize(big[:, 1:1 + r, off:off + c], out=frame[:, :r, 1:1 + c])
        assert torch.equal(frame[:, :r, 1:1 + c], O)
        frame[:, :r, 1:1 + c] = 7.0
        assert bool((frame == 7).all())
    # one matrix for the whole batch (stride 0)
    same = cake.cake_orthogonalize(G[:1].expand(b, r, c))
    assert all(torch.equal(same[i], O[0]) for i in range(b))
    assert tuple(cake.cake_orthogonalize(G[:0]).shape) == (0, r, c)


def test_zero_tiny_huge_and_non_finite(cake):
    import torch
    rng = np.random.default_rng(2)
    G = torch.from_numpy(_gradient(rng, 60, 90, "noise").astype(np.float32)).cuda()
    want = cake.cake_orthogonalize(G, eps=0.0)
    # powers of two change neither the norm's quotient nor anything after it
    for e in (-80, -20, 60, 100):
        assert torch.equal(cake.cake_orthogonalize(G * 2.0 ** e, eps=0.0), want)
    assert bool((cake.cake_orthogonalize(torch.zeros_like(G)) == 0).all())
    batch = torch.stack([G, G, G, G])
    batch[1, 3, 4], batch[2, 59, 89] = float("nan"), float("inf")
    batch[3] = 0
    O = cake.cake_orthogonalize(batch, eps=0.0)
    assert torch.equal(O[0], want) and bool(torch.isnan(O[1]).all())
    assert bool(torch.isnan(O[2, 59, 89])) and bool(torch.isnan(O[3]).all())  # 0 / 0 without eps, as in the formula


def test_other_coefficients_and_steps(cake):
    import torch
    rng = np.random.default_rng(8)
    g = _gradient(rng, 100, 140, "noise").astype(np.float32)
    for steps, coeffs in ((1, (A, B, C)), (2, (A, B, C)), (12, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0))):
        O = cake.cake_orthogonalize(torch.from_numpy(g).cuda(), steps=steps, coeffs=coeffs).double().cpu().numpy()
        _hold(O, _plain(g, np.float64, steps, coeffs), _plain(g, np.float32, steps, coeffs).astype(np.float64), "float32")
    # the coefficients that converge do: X X^T is the identity
    O = cake.cake_orthogonalize(torch.from_numpy(g).cuda(), steps=16, coeffs=(1.875, -1.25, 0.375)).double()
    # 16 steps of FP32 roundings (2^-24 per product of 140 terms, undamped: the map's slope at 1 is zero, so only the last counts)
    assert float((O @ O.T - torch.eye(100, device="cuda")).abs().max()) <= 140 * 2.0 ** -22


@pytest.mark.parametrize("tw", ["float32", "bfloat16"])
@pytest.mark.parametrize("tg", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(40, 100), (211, 97), (1, 6), (300, 300)], ids=str)
def test_muon_step(cake, shape, tw, tg):
    import torch
    rng = np.random.default_rng(shape[0])
    W = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * 0.05).to(getattr(torch, tw))
    G = torch.from_numpy(_gradient(rng, *shape, "noise").astype(np.float32)).to(getattr(torch, tg))
    M = torch.from_numpy(_gradient(rng, *shape, "tokens").astype(np.float32) * 1e-3)
    for nesterov, lr, mu, wd, scale in ((True, 0.02, 0.95, 0.01, None), (False, 0.1, 0.5, 0.0, 0.2)):
        w, g, m = W.cuda(), G.cuda(), M.clone().cuda()
        assert cake.cake_muon_step(w, g, m, lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale) is w
        assert torch.equal(g.cpu(), G)
        m64 = mu * M.double().numpy() + (1 - mu) * G.double().numpy()
        # two products and a sum in FP32, and 1 - mu itself
        assert np.all(np.abs(m.double().cpu().numpy() - m64) <= 2.0 ** -22 * (mu * np.abs(M.double().numpy()) + (1 - mu) * np.abs(G.double().numpy())))
        u = mu * m64 + (1 - mu) * G.double().numpy() if nesterov else m64
        f = max(1.0, shape[0] / shape[1]) ** 0.5 if scale is None else scale
        o64, o32 = _plain(u, np.float64), _plain(u.astype(np.float32), np.float32).astype(np.float64)
        want = (1 - lr * wd) * W.double().numpy() - lr * f * o64
        err = np.linalg.norm(w.double().cpu().numpy() - want)
        if tw == "float32":  # the update's error and two FP32 roundings of W
            tol = lr * f * (3 * np.linalg.norm(o32 - o64) + 480 * 2.0 ** -23) + 2.0 ** -23 * np.linalg.norm(want)
        else:
            tol = lr * f * 480 * 5 ** 0.5 * 2.0 ** -18 + torch.finfo(torch.bfloat16).eps / 2 * np.linalg.norm(want)
        assert err <= tol, (err, tol)


@pytest.mark.parametrize("shape", [(128, 1500), (900, 70), (20, 2048), (5, 5)], ids=str)
def test_muon_step_of_small_matrices_is_the_steps_of_its_parts(cake, shape):
    """The step's result through the optimiser's entry is W - lr f O of the same update, to the roundings of that line."""
    import torch
    torch.manual_seed(shape[0])
    W, G, M = (torch.randn(shape, device="cuda") for _ in range(3))
    w, m = W.clone(), M.clone()
    cake.cake_muon_step(w, G, m, 0.1, momentum=0.5, nesterov=False, scale=1.0)
    assert torch.equal(m, 0.5 * M + 0.5 * G)  # exact but for one rounding, the same in both
    want = W.double() - 0.1 * cake.cake_orthogonalize(m).double()
    assert bool(((w.double() - want).abs() <= 2.0 ** -23 * (want.abs() + 0.2)).all())


def test_muon_step_inside_larger_tensors(cake):
    import torch
    rng = np.random.default_rng(6)
    W, G, M = (torch.from_numpy(rng.standard_normal((50, 70)).astype(np.float32)).cuda() for _ in range(3))
    w, m = W.clone(), M.clone()
    cake.cake_muon_step(w, G, m, 0.1)
    frames = [torch.full((52, 77), 3.0, device="cuda") for _ in range(3)]
    views = [f[1:51, 3:73] for f in frames]
    for v, x in zip(views, (W, G, M)):
        v.copy_(x)
    cake.cake_muon_step(*views, 0.1)
    assert torch.equal(views[0], w) and torch.equal(views[1], G) and torch.equal(views[2], m)
    for f, v in zip(frames, views):
        v.fill_(3.0)
        assert bool((f == 3).all())


@pytest.mark.parametrize("shape", [(5, 40, 100), (3, 96, 1500), (2, 150, 200)], ids=str)
def test_results_across_the_operands(cake, shape):
    """A result that lies over other matrices of the batch, and one beside its operand in the same rows."""
    import torch
    torch.manual_seed(shape[1])
    b, r, c = shape
    buf = torch.randn(b + 1, r, c, device="cuda")

    def hold(got):
        for i in (0, b - 1):
            g = buf[i].double().cpu().numpy()
            _hold(got[i].double().cpu().numpy(), _plain(g, np.float64), _plain(g, np.float32).astype(np.float64), "float32")

    for src, dst in ((0, 1), (1, 0)):
        two = torch.empty_like(buf)
        two[src:src + b] = buf[:b]
        hold(cake.cake_orthogonalize(two[src:src + b], out=two[dst:dst + b]))
    rows = torch.empty(b, r, 2 * c, device="cuda")
    rows[:, :, :c] = buf[:b]
    hold(cake.cake_orthogonalize(rows[:, :, :c], out=rows[:, :, c:]))
    assert torch.equal(rows[:, :, :c], buf[:b])
    # momentum, gradient and weight side by side in the rows of one matrix
    wide = torch.randn(r, 3 * c, device="cuda")
    W, G, M = (wide[:, i * c:(i + 1) * c].clone() for i in range(3))
    cake.cake_muon_step(W, G, M, 0.1)
    cake.cake_muon_step(wide[:, :c], wide[:, c:2 * c], wide[:, 2 * c:], 0.1)
    assert torch.equal(wide, torch.cat((W, G, M), 1))
    with pytest.raises(cake.CakeError):
        cake.cake_muon_step(W, M, M, 0.1)


def test_refusals(cake):
    import torch
    G = torch.randn(8, 12, device="cuda")
    with pytest.raises(TypeError):
        cake.cake_orthogonalize(G.half())
    with pytest.raises(TypeError):
        cake.cake_orthogonalize(G.t())
    with pytest.raises(ValueError):
        cake.cake_orthogonalize(G[0])
    with pytest.raises(ValueError):
        cake.cake_orthogonalize(G[:, :0])
    with pytest.raises(ValueError):
        cake.cake_orthogonalize(G, out=torch.empty(8, 11, device="cuda"))
    with pytest.raises(TypeError):
        cake.cake_orthogonalize(G, out=torch.empty(8, 12, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(cake.CakeError):
        cake.cake_orthogonalize(G, steps=0)
    with pytest.raises(cake.CakeError):
        cake.cake_orthogonalize(G, eps=-1.0)
    with pytest.raises(cake.CakeError):
        cake.cake_orthogonalize(torch.randn(2, 8, 12, device="cuda"), out=torch.empty(1, 8, 12, device="cuda").expand(2, 8, 12))
    with pytest.raises(TypeError):
        cake.cake_muon_step(G, G, G.bfloat16(), 0.1)
    with pytest.raises(ValueError):
        cake.cake_muon_step(G, G[:4], G, 0.1)


def test_graphs_and_streams(cake):
    """Two steps recorded into two graphs and replayed together on two streams: each has its own workspace."""
    import torch
    torch.manual_seed(1)
    shapes = [(300, 200), (150, 420)]
    sets = [[torch.randn(s, device="cuda") for _ in range(3)] for s in shapes]
    starts = [[t.clone() for t in s] for s in sets]
    cake.cake_orthogonalize(sets[0][1])
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cake.cake_muon_step(*s, 0.05)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, (w, gr, m) in zip(sets, starts):
        for _ in range(4):
            cake.cake_muon_step(w, gr, m, 0.05)
        assert torch.equal(s[0], w) and torch.equal(s[2], m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    O = cake.cake_orthogonalize(sets[0][1], stream=side)
    side.synchronize()
    assert torch.equal(O, cake.cake_orthogonalize(sets[0][1]))
