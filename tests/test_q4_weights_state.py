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


# two geometries that pad to the same number of bytes, and ones that do not
@pytest.mark.parametrize("change", [dict(scale_type=2), dict(k=128), dict(k=99), dict(n=64), dict(n=33), dict(group=32), dict(has_zeros=True), dict(n=100)], ids=str)
def test_state_of_another_geometry_is_refused(cake, change):
    from cake_on_cpu_b200.cake import cake_linear_q4
    mine = cake_linear_q4(_weights(cake))
    keep, address = mine.packed.clone(), mine.packed.data_ptr()
    other = cake_linear_q4(_weights(cake, seed=1, **change))
    for strict in (True, False):
        for assign in (True, False):
            with pytest.raises(RuntimeError):
                mine.load_state_dict(other.state_dict(), strict=strict, assign=assign)
            assert torch.equal(mine.packed, keep) and mine.packed.data_ptr() == address


def test_state_of_the_same_geometry(cake):
    from cake_on_cpu_b200.cake import cake_linear_q4
    model, other = (torch.nn.ModuleDict({"a": cake_linear_q4(_weights(cake, seed=s), torch.full((40,), float(s)))}) for s in (1, 2))
    f = io.BytesIO()
    torch.save(other.state_dict(), f)
    f.seek(0)
    model.load_state_dict(torch.load(f))  # tensors only
    assert torch.equal(model["a"].packed, other["a"].packed) and torch.equal(model["a"].bias, other["a"].bias)
    # a state that does not say what it holds is refused, unless the caller vouches for it
    state = {k: v for k, v in other.state_dict().items() if k in ("a.packed", "a.bias")}
    with pytest.raises(RuntimeError):
        model.load_state_dict(state)
    model.load_state_dict(state, strict=False)


def test_which_products_need_a_workspace(cake):
    """Up to 64 rows none; up to 128 none for y in 16 bits; beyond, by the sizes."""
    L = cake.lib()
    W = _weights(cake, 40, 100)
    W._c.out_features, W._c.in_features = 16384, 8192  # only looked at
    for t, rows, dx, none in ((2, 64, 0, True), (2, 65, 0, True), (1, 128, 0, True), (2, 129, 0, False), (0, 64, 0, True), (0, 65, 0, False), (2, 64, 1, True),
                              (2, 65, 1, False)):
        assert (L.cakeb200_q4_workspace(W._ref, rows, t, dx) == 0) == none, (t, rows, dx)
