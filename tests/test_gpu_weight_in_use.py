"""The operators on a linear layer's weight as a program uses them: two layers trained with cake_muon, then held in 4 bits and
asked token by token."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _orthogonal(u):
    x = u / (np.linalg.norm(u) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(5):
        p = x @ x.T
        x = 3.4445 * x + (-4.7750 * p + 2.0315 * (p @ p)) @ x
    return x.T if tall else x


def test_train_then_serve(cake):
    """Three steps of two layers against the same steps in float64, then the same layers in 4 bits: rows of a batch one by one
    give what the batch gives, and both what the dequantised weights give."""
    import torch
    from cake_on_cpu_b200.cake import cake_linear, cake_linear_q4, cake_muon
    torch.manual_seed(3)
    first, second = cake_linear(96, 200).cuda(), cake_linear(200, 64).cuda()
    opt = cake_muon([first.weight, second.weight], lr=0.05, weight_decay=0.01)
    x, t = torch.randn(150, 96, device="cuda"), torch.randn(150, 64, device="cuda")
    w = [first.weight.detach().double().cpu().numpy(), second.weight.detach().double().cpu().numpy()]
    b = [first.bias.detach().double().cpu().numpy(), second.bias.detach().double().cpu().numpy()]
    m = [np.zeros_like(v) for v in w]
    x64, t64 = x.double().cpu().numpy(), t.double().cpu().numpy()
    for _ in range(3):
        opt.zero_grad()
        ((second(torch.tanh(first(x))) - t) ** 2).mean().backward()
        opt.step()
        h = np.tanh(x64 @ w[0].T + b[0])
        d = 2 * (h @ w[1].T + b[1] - t64) / t64.size
        grads = [((d @ w[1]) * (1 - h * h)).T @ x64, d.T @ h]
        for i in range(2):
            m[i] = 0.95 * m[i] + 0.05 * grads[i]
            w[i] = (1 - 0.05 * 0.01) * w[i] - 0.05 * max(1, w[i].shape[0] / w[i].shape[1]) ** 0.5 * _orthogonal(0.95 * m[i] + 0.05 * grads[i])
    for layer, want in zip((first, second), w):
        # a gradient in FP32 is off by some 2^-20; small singular directions of it come out 480 times as large, in every step
        assert np.linalg.norm(layer.weight.detach().double().cpu().numpy() - want) <= 3 * 0.05 * 480 * 2.0 ** -20 * want.shape[0] ** 0.5

    served = [cake_linear_q4.from_linear(layer, group=32, symmetric=False) for layer in (first, second)]
    with torch.no_grad():
        y = served[1](torch.tanh(served[0](x)))
        d = [s.weights.dequantize().double() for s in served]
        want = torch.tanh(x.double() @ d[0].T + first.bias.double()) @ d[1].T + second.bias.double()
        # two products of FP32 sums with 96 and 200 terms, tanh's slope is at most one
        assert float((y.double() - want).abs().max()) <= 2.0 ** -18 * float((d[1].abs().sum(1)).max())
        for i in (0, 77, 149):
            one = served[1](torch.tanh(served[0](x[i])))
            assert float((one.double() - want[i]).abs().max()) <= 2.0 ** -18 * float((d[1].abs().sum(1)).max())
        # half a step of the codes, one with the rounding of the zero point
        for s, layer in zip(served, (first, second)):
            worst = (layer.weight.detach().amax(1) - layer.weight.detach().amin(1)) / 15
            assert float(((s.weights.dequantize() - layer.weight.detach()).abs() / worst[:, None]).max()) <= 1.02


@pytest.mark.parametrize("rows", [3, 100])
def test_gradients_through_a_frozen_layer(cake, rows):
    """d(loss)/dx and d(loss)/db against the formula and against differences of the layer's own output."""
    import torch
    from cake_on_cpu_b200.cake import cake_linear, cake_linear_q4
    torch.manual_seed(rows)
    layer = cake_linear_q4.from_linear(cake_linear(130, 70).cuda(), group=64)
    x = torch.randn(2, rows, 130, device="cuda", requires_grad=True)
    c = torch.randn(2, rows, 70, device="cuda")
    (layer(x) * c).sum().backward()
    w = layer.weights.dequantize().double()
    S = c.double().abs() @ w.abs()
    assert bool(((x.grad.double() - c.double() @ w).abs() <= 2.0 ** -18 * S).all())  # 70 products in FP32
    want = c.double().sum((0, 1))
    assert bool(((layer.bias.grad.double() - want).abs() <= 2.0 ** -18 * c.double().abs().sum((0, 1))).all())
    # the layer is linear in x, so a central difference has no error but that of the outputs, 2^-18 of their terms, over the step
    step, where = 0.5, (1, rows // 2, 77)
    e = torch.zeros_like(x)
    e[where] = step
    with torch.no_grad():
        diff = float(((layer(x + e).double() - layer(x - e).double()) * c.double()).sum()) / (2 * step)
        terms = (x.detach().double().abs() + step) @ w.abs().T + layer.bias.detach().double().abs()
    assert abs(diff - float(x.grad[where])) <= 2 * 2.0 ** -18 * float((terms * c.double().abs())[where[0], where[1]].sum()) / (2 * step) + 1e-4 * abs(diff)
    # no gradient wanted: none computed
    y = layer(torch.randn(4, 130, device="cuda"))
    y.sum().backward()


def test_module_moves_and_reloads(cake):
    import torch
    from cake_on_cpu_b200.cake import cake_linear, cake_linear_q4
    a, b = (cake_linear_q4.from_linear(cake_linear(64, 48).cuda(), group=32) for _ in range(2))
    x = torch.randn(5, 64, device="cuda")
    assert not torch.equal(a(x), b(x))
    b.load_state_dict(a.state_dict())
    assert torch.equal(a(x), b(x))
    c = b.cpu().cuda()
    assert torch.equal(c(x), a(x))


def test_muon_refuses_what_is_not_a_matrix(cake):
    import torch
    from cake_on_cpu_b200.cake import cake_muon
    with pytest.raises(ValueError):
        cake_muon([torch.nn.Parameter(torch.zeros(4, device="cuda"))])
    with pytest.raises(ValueError):
        cake_muon([torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))], momentum=1.5)
    p = torch.nn.Parameter(torch.randn(6, 9, device="cuda"))
    q = torch.nn.Parameter(torch.randn(6, 9, device="cuda"))
    opt = cake_muon([p, q], lr=0.1)
    keep = q.detach().clone()
    (p * 2).sum().backward()
    opt.step()  # q has no gradient and stays
    assert torch.equal(q.detach(), keep) and opt.state[p]["momentum"].dtype == torch.float32
    # a gradient that is stored by columns
    p.grad = torch.randn(9, 6, device="cuda").t()
    opt.step()
    assert bool(torch.isfinite(p).all())


def test_step_is_seen_by_autograd(cake):
    """A graph that saved the weight before a step refuses to go backward after it; gradients of gradients are refused too."""
    import torch
    from cake_on_cpu_b200.cake import cake_linear_q4, cake_muon
    torch.manual_seed(5)
    w = torch.nn.Parameter(torch.randn(40, 70, device="cuda"))
    opt = cake_muon([w], lr=0.1)
    x = torch.randn(6, 70, device="cuda", requires_grad=True)
    old = (x @ w.t()).sum()
    (x.detach() @ w.t()).square().sum().backward()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        old.backward()
    layer = cake_linear_q4(cake.Q4Weights.quantize(w.detach()))
    y = layer(x.detach().requires_grad_())
    x2 = x.detach().requires_grad_()
    (g,) = torch.autograd.grad(layer(x2).square().sum(), x2, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert y.shape == (6, 40)


def test_resumed_training_goes_on_with_the_same_bits(cake):
    import io
    import torch
    from cake_on_cpu_b200.cake import cake_muon
    torch.manual_seed(6)
    start = torch.randn(130, 60, device="cuda", dtype=torch.bfloat16)
    grads = [torch.randn_like(start) for _ in range(4)]

    def run(p, opt, some):
        for g in some:
            p.grad = g.clone()
            opt.step()

    p = torch.nn.Parameter(start.clone())
    opt = cake_muon([p], lr=0.05)
    run(p, opt, grads[:2])
    f = io.BytesIO()
    torch.save((p.detach(), opt.state_dict()), f)
    run(p, opt, grads[2:])
    f.seek(0)
    kept, state = torch.load(f, map_location="cuda")
    q = torch.nn.Parameter(kept.clone())
    other = cake_muon([q], lr=0.9)
    other.load_state_dict(state)
    run(q, other, grads[2:])
    assert torch.equal(p, q)


@pytest.mark.parametrize("call", ["cake.cake_orthogonalize(g)", "cake.cake_orthogonalize(g[:, :30])", "cake.cake_muon_step(g.clone(), g, m, 0.1)",
                                  "cake.cake_q4_linear(g, cake.Q4Weights(codes, scales))"])
def test_first_call_of_a_process_is_captured(call):
    """Nothing of the library has run on the device when the capture begins."""
    import os
    import subprocess
    import sys
    code = """
import torch
import cake_on_cpu_b200 as cake
g, m = torch.randn(300, 256, device="cuda"), torch.zeros(300, 256, device="cuda")
codes, scales = torch.randint(0, 256, (64, 128), dtype=torch.uint8, device="cuda"), torch.ones((64, 2), dtype=torch.float16, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = CALL
graph.replay()
torch.cuda.synchronize()
first = out.clone()
m.zero_()
assert torch.equal(first, CALL) and bool(torch.isfinite(first).all())
""".replace("CALL", call)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]


def test_threads_with_streams_of_their_own(cake):
    """Eight host threads at once, each with its stream: nobody's result changes."""
    import threading
    import torch
    torch.manual_seed(0)
    W4 = cake.Q4Weights.quantize(torch.randn(900, 700, device="cuda"))
    gs = [torch.randn(96, 960, device="cuda") for _ in range(4)] + [torch.randn(300, 400, device="cuda") for _ in range(4)]
    xs = [torch.randn(r, 700, device="cuda") for r in (1, 7, 33, 70, 300, 1100, 2, 16)]
    want = [(cake.cake_orthogonalize(g), cake.cake_q4_linear(x, W4)) for g, x in zip(gs, xs)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = cake.cake_orthogonalize(gs[i]), cake.cake_q4_linear(xs[i], W4)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
