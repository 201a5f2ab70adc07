"""4-bit weights made on a stream of their own, copied, pickled and reloaded."""
import copy
import io

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _busy(stream):
    """A few milliseconds of work on a stream."""
    import torch
    with torch.cuda.stream(stream):
        a = torch.randn(6000, 6000, device="cuda")
        for _ in range(6):
            a = a @ a * 1e-2
    return a


def test_quantising_on_another_stream(cake):
    """Zero points are checked where they are written, not on the current stream: memory that held other bytes
    before is handed out again while the stream is still busy."""
    import torch
    torch.manual_seed(0)
    W = torch.randn(512, 640, device="cuda")
    want = cake.Q4Weights.quantize(W, 64, symmetric=False)
    codes, scales, zeros = cake.Q4Weights.quantize_codes(W, 64, symmetric=False)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            old = [torch.full(s, 255, dtype=torch.uint8, device="cuda") for s in ((512, 320), (512, 20), (512, 10)) for _ in range(4)]
        torch.cuda.synchronize()
        del old
        keep = _busy(side)
        got = cake.Q4Weights.quantize(W, 64, symmetric=False, stream=side)
        side.synchronize()
        assert torch.equal(got.packed, want.packed)
        # the constructor on that stream, with arrays written on it just before
        keep = _busy(side)
        with torch.cuda.stream(side):
            late = torch.full(zeros.shape, 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        keep = _busy(side)
        with torch.cuda.stream(side):
            late.copy_(zeros)
        got = cake.Q4Weights(codes, scales, late, group=64, stream=side)
        side.synchronize()
        assert torch.equal(got.packed, want.packed)
        with torch.cuda.stream(side):
            keep = _busy(side)
            late.fill_(16)
        with pytest.raises(ValueError):
            cake.Q4Weights(codes, scales, late, group=64, stream=side)
        del keep


def test_weights_are_made_while_their_stream_is_captured(cake):
    """The zero points cannot be looked at in the middle of a capture, whichever stream is the current one."""
    import torch
    torch.manual_seed(1)
    W = torch.randn(64, 256, device="cuda")
    codes, scales, zeros = cake.Q4Weights.quantize_codes(W, 64, symmetric=False)
    want = cake.Q4Weights(codes, scales, zeros, group=64)
    capture, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capture):
        with torch.cuda.stream(other):
            got = cake.Q4Weights(codes, scales, zeros, group=64, stream=capture)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.packed, want.packed)


def test_copies_and_pickles_have_memory_of_their_own(cake):
    import torch
    from cake_on_cpu_b200.cake import cake_linear, cake_linear_q4
    torch.manual_seed(2)
    x = torch.randn(7, 200, device="cuda")
    model = torch.nn.Sequential(cake_linear_q4.from_linear(cake_linear(200, 90).cuda(), group=64, symmetric=False), torch.nn.Tanh())
    want = model(x).detach()
    f = io.BytesIO()
    torch.save(model, f)
    twin = copy.deepcopy(model)
    weights = copy.deepcopy(model[0].weights)
    address = model[0].packed.data_ptr()
    assert twin[0].packed.data_ptr() != address and weights.packed.data_ptr() != address
    model[0].packed.fill_(255)  # whoever still looked at the original would notice
    del model
    f.seek(0)
    loaded = torch.load(f, weights_only=False)
    for m in (twin, loaded, copy.deepcopy(twin).cpu().cuda()):
        assert m[0].weights.packed is m[0].packed
        assert torch.equal(m(x), want)
    assert torch.equal(torch.tanh(cake.cake_q4_linear(x, weights, twin[0].bias)), want)


def test_reloading_another_geometry_is_refused(cake):
    """Packed sizes are padded and do not tell the scales' type: the state does."""
    import torch
    from cake_on_cpu_b200.cake import cake_linear_q4
    torch.manual_seed(3)

    def layer(n, k, group=128, scale=torch.float16, symmetric=True):
        return cake_linear_q4(cake.Q4Weights.quantize(torch.randn(n, k, device="cuda"), group, symmetric, scale))

    a, x = layer(100, 128), torch.randn(3, 128, device="cuda")
    before = a(x)
    for other in (layer(100, 128, scale=torch.bfloat16), layer(100, 100), layer(97, 128), layer(128, 128), layer(100, 128, 64), layer(100, 128, symmetric=False)):
        for strict in (True, False):
            with pytest.raises(RuntimeError):
                a.load_state_dict(other.state_dict(), strict=strict)
            assert torch.equal(a(x), before)  # nothing of it was taken
    same = layer(100, 128)
    a.load_state_dict(same.state_dict())
    assert torch.equal(a(x), same(x)) and not torch.equal(a(x), before)
    f = io.BytesIO()
    torch.save(torch.nn.Sequential(a).state_dict(), f)
    f.seek(0)
    b = torch.nn.Sequential(layer(100, 128))
    b.load_state_dict(torch.load(f))
    assert torch.equal(b(x), a(x))
    b.load_state_dict(torch.nn.Sequential(layer(100, 128)).state_dict(), assign=True)
    assert b[0].weights.packed is b[0].packed and not torch.equal(b(x), a(x))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_layer_takes_what_the_fp32_layer_takes(cake, dtype):
    """Activations whose rows are not contiguous or not evenly spaced are copied, as cake_linear does, and their gradients
    come out all the same."""
    import torch
    from cake_on_cpu_b200.cake import cake_linear, cake_linear_q4
    torch.manual_seed(4)
    plain = cake_linear(64, 40).cuda()
    layer = cake_linear_q4.from_linear(plain, group=32).to(getattr(torch, dtype))
    t = getattr(torch, dtype)
    heads = torch.randn(3, 5, 4, 64, device="cuda").to(t)
    for x in (heads.transpose(1, 2), heads[0, 0].t().contiguous().t(), heads[:, :, 1], heads[0, 0, 0].expand(6, 64), heads[:, :1].expand(3, 5, 4, 64),
              torch.randn(64, 9, device="cuda").to(t).t(), heads[:0].transpose(1, 2)):
        if dtype == "float32" and x.numel():
            plain(x)
        a, b = x.detach().requires_grad_(), x.detach().contiguous().requires_grad_()
        y, want = layer(a), layer(b)
        assert y.shape == x.shape[:-1] + (40,) and torch.equal(y, want)
        c = torch.randn_like(y)
        y.backward(c)
        want.backward(c)
        assert torch.equal(a.grad, b.grad)
