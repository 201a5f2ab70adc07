"""4-bit products with few rows of weights so large that a cluster takes several items one after the other: cursors that cross
items, two sets of sums, the join of an item behind the next one."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# rows, N, K, group.  A cluster has at most 148 * 5 CTAs to share out among them, and an item is 32 output features x 8, 16 or 32 rows.
# K of 130 and 300 have fewer steps (2 and 3) than a cluster has warps (4 and more), 100 has a single one; item counts that no
# number of clusters divides; rows in several chunks over the same weights
CASES = [(1, 33001, 1100, 128), (1, 70003, 130, 32), (3, 40000, 300, 64), (8, 50017, 100, 32), (9, 33001, 520, 64), (16, 45000, 130, 128), (17, 34567, 264, 32),
         (33, 33333, 300, 128), (64, 26001, 1100, 64)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_several_items_per_cluster(cake, case, dtype):
    import torch
    rows, N, K, group = case
    g = torch.Generator().manual_seed(N + K)
    G = -(-K // group)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, generator=g).cuda()
    scales = (torch.rand((N, G), generator=g) * 0.05 + 0.002).to(torch.bfloat16 if N % 2 else torch.float16).cuda()
    zeros = torch.randint(0, 16, (N, G), dtype=torch.uint8, generator=g).cuda() if K % 3 else None
    W4 = cake.Q4Weights(codes, scales, zeros, group=group, in_features=K)
    t = getattr(torch, dtype)
    x, bias = torch.randn((rows, K), generator=g).to(t).cuda(), torch.randn((N,), generator=g).to(t).cuda()
    at = torch.arange(K, device="cuda") // group
    q = torch.stack((codes & 15, codes >> 4), 2).view(N, -1)[:, :K].double()
    w = scales.double()[:, at] * (q - (zeros.double()[:, at] if zeros is not None else 8.0))
    y = cake.cake_q4_linear(x, W4, bias).double()
    want = x.double() @ w.t() + bias.double()
    S = x.double().abs() @ w.abs().t() + bias.double().abs()
    # half a step of the result and K / 16 + 40 additions in FP32, 2^-22 of their terms each
    tol = torch.finfo(t).eps / 2 * want.abs() * (1 + 2.0 ** -20) + (K / 16 + 40) * 2.0 ** -22 * S
    worst = float(((y - want).abs() / tol).max())
    assert worst <= 1, worst
    again = cake.cake_q4_linear(x, W4, bias)
    assert torch.equal(again.double(), y)
    # rows of a batch are what they are alone
    assert torch.equal(cake.cake_q4_linear(x[:1], W4, bias), cake.cake_q4_linear(x[:1].clone(), W4, bias))
    dy = torch.randn((rows, N), generator=g).to(t).cuda()
    dx = cake.cake_q4_linear_dx(dy, W4).double()
    want, S = dy.double() @ w, dy.double().abs() @ w.abs()
    tol = torch.finfo(t).eps / 2 * want.abs() * (1 + 2.0 ** -20) + ((N / 16 + 40) * 2.0 ** -22 + (2.0 ** -22 if dtype == "float32" else 2.0 ** -14)) * S
    assert bool(((dx - want).abs() <= tol).all())
