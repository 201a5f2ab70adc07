"""The operators on a linear layer's weight, as cases that can be run and timed.

Two things happen to the weight of ``cake_linear`` around the products this package had first: training moves it,
by an orthogonalised update, and serving keeps it in four bits.

``q4_linear``        y = x W^T + b with W held in 4 bits: codes q in 0..15, one scale s (and, where given, one zero
                     point z, else 8) for every ``group`` consecutive input features of an output feature,
                     w = s (q - z).  One row of x is a token being generated, hundreds are a prompt.
``q4_linear_dx``     its gradient for the input, dx = dy W: what training anything in front of a frozen 4-bit layer needs.
``orthogonalize``    X <- a X + b (X X^T) X + c (X X^T)^2 X, ``steps`` times from X = G / (|G|_F + eps), taken on
                     the transpose where the matrix is taller than wide.
``muon_step``        M <- mu M + (1 - mu) G;  U = mu M + (1 - mu) G (or M);  W <- (1 - lr wd) W - lr scale O(U) with O the
                     orthogonalisation and scale = sqrt(max(1, rows / cols)).

Types: q4_linear* in float32, bfloat16 and float16; orthogonalize in float32 and bfloat16; muon_step with weights and
gradients in either of these and the momentum in float32.
"""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------------------------------------ the cases

def _q4(name, op, rows, n, k, group, dtype, zeros, bias=False):
    return {"name": name, "op": op, "rows": rows, "n": n, "k": k, "group": group, "dtype": dtype, "zeros": zeros, "bias": bias}


def _orth(name, op, batch, rows, cols, dtype, **more):
    return dict({"name": name, "op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype, "steps": 5}, **more)


def listed():
    return [
        # one token through a small square layer: nothing but latency
        _q4("token-2048-bf16", "q4_linear", 1, 2048, 2048, 128, "bfloat16", False),
        # one token through the largest layer, 16384 square as in the matrix-vector benchmark: nothing but bytes
        _q4("token-16384-fp32", "q4_linear", 1, 16384, 16384, 64, "float32", True, True),
        # five sequences answering at once; sizes that divide nothing (2111 is one of the tests' awkward sizes)
        _q4("five-odd-fp16", "q4_linear", 5, 4097, 2111, 32, "float16", True),
        # a full batch of sequences answering at once through a wide layer
        _q4("batch32-8192-bf16", "q4_linear", 32, 16384, 8192, 128, "bfloat16", False, True),
        # a prompt of five hundred tokens
        _q4("prompt500-4096-bf16", "q4_linear", 500, 4096, 4096, 128, "bfloat16", True),
        # gradient for a handful of rows in front of a frozen layer, in the framework's own type
        _q4("dx-four-fp32", "q4_linear_dx", 4, 4096, 4096, 64, "float32", False),
        # gradient of a training batch of tokens
        _q4("dx-batch-bf16", "q4_linear_dx", 1000, 8192, 2048, 128, "bfloat16", True),
        # the projections of 12 heads, orthogonalised together
        _orth("heads-fp32", "orthogonalize", 12, 96, 960, "float32"),
        # a layer four times as wide as it is high, gradients in 16 bits
        _orth("wide-bf16", "orthogonalize", 1, 1024, 4096, "bfloat16"),
        # the largest: a square layer in the framework's own type
        _orth("square-4096-fp32", "orthogonalize", 1, 4096, 4096, "float32"),
        # an optimiser's step for a layer whose sizes divide nothing, taller than wide
        _orth("step-tall-fp32", "muon_step", 1, 2111, 961, "float32", nesterov=True),
        # an optimiser's step in 16 bits
        _orth("step-2048-bf16", "muon_step", 1, 2048, 2048, "bfloat16", nesterov=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm; half of them are multiples of 8."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        v = (v + 7) // 8 * 8
    return min(max(v, low), high)


def draw(rng):
    op = rng.choice(["q4_linear", "q4_linear", "q4_linear_dx", "orthogonalize", "orthogonalize", "muon_step"])
    if op.startswith("q4"):
        rows = _spread(rng, 1, 1000)
        n, k = _spread(rng, 256, 16384), _spread(rng, 256, 16384)
        while rows * n * k > 1000 * 8192 * 2048:
            n, k = max(256, n * 3 // 4), max(256, k * 3 // 4)
        return {"op": op, "rows": rows, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "dtype": rng.choice(sorted(DTYPES)),
                "zeros": rng.random() < 0.5, "bias": op == "q4_linear" and rng.random() < 0.5}
    small, large = _spread(rng, 32, 2048), _spread(rng, 64, 6000)
    small, large = min(small, large), max(small, large)
    batch = rng.choice([1, 1, 2, 3, 8]) if large < 1024 and op == "orthogonalize" else 1
    rows, cols = (small, large) if rng.random() < 0.6 else (large, small)
    case = {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": rng.choice(["float32", "bfloat16"]), "steps": 5}
    if op == "muon_step":
        case["nesterov"] = rng.random() < 0.5
    return case


def _orth_flops(case):
    """Operations of one orthogonalisation.  X X^T and its square are symmetric, so half of their entries follow from
    the other half.  A matrix much wider than high needs its long side in the first and the last product only: the steps
    between them are polynomials of the small square matrix X X^T."""
    m, n, s = min(case["rows"], case["cols"]), max(case["rows"], case["cols"]), case["steps"]
    return case["batch"] * min(s * (3.0 * m * m * n + 1.0 * m ** 3), 3.0 * m * m * n + (4.0 * s - 3.0) * m ** 3)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"].startswith("q4"):
        r, n, k = case["rows"], case["n"], case["k"]
        groups = -(-k // case["group"])
        weight = n * k / 2 + n * groups * (2 + (1 if case["zeros"] else 0)) + (n * size if case["bias"] else 0)
        return {"bytes": weight + r * (n + k) * size, "flops": 2.0 * r * n * k}
    count = case["batch"] * case["rows"] * case["cols"]
    if case["op"] == "orthogonalize":
        return {"bytes": 2.0 * count * size, "flops": _orth_flops(case)}
    return {"bytes": count * (3.0 * size + 8.0), "flops": _orth_flops(case)}  # W in and out, G in, M in and out


# ------------------------------------------------------------------------------------------------ the inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _quantise(w, group, zeros):
    """4-bit codes of w (n x k), two to a byte (even feature in the low half), with their scales and zero points."""
    n, k = w.shape
    groups = -(-k // group)
    padded = torch.zeros((n, groups * group), device=w.device)
    padded[:, :k] = w
    padded = padded.view(n, groups, group)
    if zeros:
        low, high = padded.amin(2).clamp(max=0), padded.amax(2).clamp(min=0)
        scale = ((high - low) / 15).clamp(min=1e-6).half()
        zero = torch.round(-low / scale.float()).clamp(0, 15)
    else:
        scale = (padded.abs().amax(2) / 7).clamp(min=1e-6).half()
        zero = torch.full((n, groups), 8.0, device=w.device)
    q = (torch.round(padded / scale.float()[:, :, None]) + zero[:, :, None]).clamp(0, 15).to(torch.uint8).view(n, -1)
    q = q[:, : k + (k & 1)]
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
    return codes, scale, zero.to(torch.uint8) if zeros else None


def _gradient(g, batch, rows, cols):
    """A weight gradient as backward leaves it: the sum over a batch of tokens of an outer product each, features of
    unlike size, and some noise from the accumulation of earlier batches."""
    tokens = 512
    dy = torch.randn((batch, tokens, rows), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((batch, 1, rows), generator=g, device="cuda"))
    x = torch.randn((batch, tokens, cols), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((batch, 1, cols), generator=g, device="cuda"))
    noise = torch.randn((batch, rows, cols), generator=g, device="cuda")
    return (dy.transpose(1, 2) @ x / tokens + 0.02 * noise) * 1e-3


def prepare(case, seed):
    g = _generator(seed)
    t = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"].startswith("q4"):
        r, n, k = case["rows"], case["n"], case["k"]
        w = torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)
        codes, scales, zeros = _quantise(w, case["group"], case["zeros"])
        if case["op"] == "q4_linear":
            state["x"] = torch.randn((r, k), generator=g, device="cuda").to(t)
            state["b"] = torch.randn((n,), generator=g, device="cuda").to(t) if case["bias"] else None
        else:
            state["x"] = (torch.randn((r, n), generator=g, device="cuda") * 1e-2).to(t)
        if own:
            import cake_on_cpu_b200 as cake
            state["w"] = cake.Q4Weights(codes, scales, zeros, group=case["group"], in_features=k)
        else:
            state["w"] = (codes, scales, zeros)
        return state
    grad = _gradient(g, case["batch"], case["rows"], case["cols"]).to(t)
    if case["op"] == "orthogonalize":
        state["g"] = grad if case["batch"] > 1 else grad[0]
        return state
    state["g"] = grad[0]
    state["w"] = (torch.randn((case["rows"], case["cols"]), generator=g, device="cuda") / math.sqrt(case["cols"])).to(t)
    state["m"] = _gradient(g, 1, case["rows"], case["cols"])[0]
    state.update(lr=0.02, mu=0.95, wd=0.01)
    return state


# ------------------------------------------------------------------------------------------------ one pass

def _weights(state):
    """W in 32 bits from its codes."""
    codes, scales, zeros = state["w"]
    n, k, group = state["n"], state["k"], state["group"]
    q = torch.stack((codes & 15, codes >> 4), 2).view(n, -1)[:, :k].float()
    at = torch.arange(k, device=codes.device) // group
    z = zeros.float()[:, at] if zeros is not None else 8.0
    return scales.float()[:, at] * (q - z)


def _orthogonal(g, steps, rounded=True):
    a, b, c = COEFFS
    tall = g.shape[-2] > g.shape[-1]
    x = g.float()
    x = x.mT if tall else x
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + EPS).float()
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    x = x.mT if tall else x
    return x.to(g.dtype) if rounded else x


def run(state):
    op = state["op"]
    if own:
        import cake_on_cpu_b200 as cake
        if op == "q4_linear":
            return cake.cake_q4_linear(state["x"], state["w"], state["b"])
        if op == "q4_linear_dx":
            return cake.cake_q4_linear_dx(state["x"], state["w"])
        if op == "orthogonalize":
            return cake.cake_orthogonalize(state["g"], steps=state["steps"], coeffs=COEFFS, eps=EPS)
        cake.cake_muon_step(state["w"], state["g"], state["m"], lr=state["lr"], momentum=state["mu"], nesterov=state["nesterov"],
                            weight_decay=state["wd"], steps=state["steps"], coeffs=COEFFS, eps=EPS)
        return state["w"], state["m"]
    if op == "q4_linear":
        y = state["x"].float() @ _weights(state).t()
        if state["b"] is not None:
            y = y + state["b"].float()
        return y.to(state["x"].dtype)
    if op == "q4_linear_dx":
        return (state["x"].float() @ _weights(state)).to(state["x"].dtype)
    if op == "orthogonalize":
        return _orthogonal(state["g"], state["steps"])
    w, g, m, lr, mu = state["w"], state["g"].float(), state["m"], state["lr"], state["mu"]
    m.copy_(mu * m + (1 - mu) * g)
    u = mu * m + (1 - mu) * g if state["nesterov"] else m
    o = _orthogonal(u, state["steps"], rounded=False)
    scale = math.sqrt(max(1.0, state["rows"] / state["cols"]))
    w.copy_((1 - lr * state["wd"]) * w.float() - lr * scale * o)
    return w, m


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("q4"):
        codes, scales, zeros = s["w"]
        n, k, group = case["n"], case["k"], case["group"]
        w = torch.empty((n, 2 * codes.shape[1]), dtype=torch.float64, device=codes.device)
        w[:, 0::2] = (codes % 16).double()
        w[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
        w = w[:, :k].contiguous()
        for j in range(scales.shape[1]):
            part = w[:, j * group:(j + 1) * group]
            part -= zeros[:, j:j + 1].double() if zeros is not None else 8.0
            part *= scales[:, j:j + 1].double()
        if case["op"] == "q4_linear_dx":
            return torch.mm(s["x"].double(), w)
        y = torch.mm(s["x"].double(), w.t())
        return y if s["b"] is None else y + s["b"].double()

    def orthogonalised(g):
        g = g.double()
        norm = torch.sqrt((g * g).sum(dim=(-1, -2), keepdim=True))
        x = g / (norm + EPS)
        for _ in range(case["steps"]):
            if x.shape[-2] <= x.shape[-1]:
                p = torch.matmul(x, x.transpose(-1, -2))
                y = torch.matmul(p, x)
                x = COEFFS[0] * x + COEFFS[1] * y + COEFFS[2] * torch.matmul(p, y)
            else:
                p = torch.matmul(x.transpose(-1, -2), x)
                y = torch.matmul(x, p)
                x = COEFFS[0] * x + COEFFS[1] * y + COEFFS[2] * torch.matmul(y, p)
        return x

    if case["op"] == "orthogonalize":
        return orthogonalised(s["g"])
    g, m, w = s["g"].double(), s["m"].double(), s["w"].double()
    m = s["mu"] * m + (1 - s["mu"]) * g
    u = s["mu"] * m + (1 - s["mu"]) * g if s["nesterov"] else m
    factor = max(1.0, case["rows"] / case["cols"]) ** 0.5
    return w - s["lr"] * s["wd"] * w - s["lr"] * factor * orthogonalised(u), m
