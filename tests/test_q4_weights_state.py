"""4-bit weights as Python objects, without a GPU: copies, pickles and the state of the layer."""
import copy
import ctypes
import io
import pickle

import pytest
import torch


def _weights(cake, n=40, k=100, group=64, scale_type=1, has_zeros=False, seed=0):
    """Weights whose packed form lies in host memory: nothing multiplies them here."""
    W = object.__new__(cake.Q4Weights)
    W.out_features, W.in_features, W.group, W.scale_type, W.has_zeros = n, k, group, scale_type, has_zeros
    size = cake.lib().cakeb200_q4_packed_bytes(n, k, group, int(has_zeros))
    W.packed = torch.randint(0, 256, (size,), dtype=torch.uint8, generator=torch.Generator().manual_seed(seed))
    W.device = W.packed.device
    W._bind()
    return W


def _points_at_its_own(W):
    c = ctypes.cast(W._ref, ctypes.POINTER(type(W._c))).contents
    return c.packed == W.packed.data_ptr() and (c.out_features, c.in_features, c.group, c.scale_type, c.has_zeros) == \
        (W.out_features, W.in_features, W.group, W.scale_type, int(W.has_zeros))


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "save"])
def test_copies_of_weights(cake, how):
    W = _weights(cake, has_zeros=True)
    if how == "deepcopy":
        V = copy.deepcopy(W)
    elif how == "pickle":
        V = pickle.loads(pickle.dumps(W))
    else:
        f = io.BytesIO()
        torch.save(W, f)
        f.seek(0)
        V = torch.load(f, weights_only=False)
    assert torch.equal(V.packed, W.packed) and V.packed.data_ptr() != W.packed.data_ptr() and V.device == W.device
    assert _points_at_its_own(V) and _points_at_its_own(W)
    assert _points_at_its_own(copy.copy(W))


def test_copies_of_the_layer(cake):
    from cake_on_cpu_b200.cake import cake_linear_q4
    model = torch.nn.Sequential(cake_linear_q4(_weights(cake), torch.ones(40)))
    f = io.BytesIO()
    torch.save(model, f)
    f.seek(0)
    for twin in (copy.deepcopy(model), torch.load(f, weights_only=False)):
        layer = twin[0]
        assert layer._weights.packed is layer.packed and layer.packed.data_ptr() != model[0].packed.data_ptr()
        assert _points_at_its_own(layer._weights) and torch.equal(layer.packed, model[0].packed)
