"""Arguments the operators on a linear layer's weight refuse, without a GPU: the C ABI checks sizes, types and pointers
before it looks for a device, the Python layer checks kinds of arrays before it calls."""
import ctypes

import pytest

ERR_ARG, ERR_TOO_LARGE, ERR_NO_DEVICE = -1, -5, -3


def _last(cake):
    return cake.lib().cakeb200_last_error().decode()


def _q4(packed=0x10000, n=32, k=64, group=64, scale=1, zeros=0):
    from cake_on_cpu_b200.api import _Q4
    return _Q4(packed, n, k, group, scale, zeros)


def test_q4_sizes(cake):
    L = cake.lib()
    # pairs of 16 x 128 blocks of 1024 bytes, 16 scales (2 bytes) and zero points (1 byte) per block row and group
    assert L.cakeb200_q4_packed_bytes(16, 64, 64, 0) == 2 * (1024 + 2 * 32)
    assert L.cakeb200_q4_packed_bytes(33, 129, 32, 1) == 4 * 2 * 1024 + 4 * 8 * 16 * 3
    assert L.cakeb200_q4_packed_bytes(16384, 16384, 128, 0) == 16384 * 16384 // 2 + 16384 * 128 * 2
    for bad in ((0, 64, 64, 0), (16, 0, 64, 0), (16, 64, 48, 0), (16, -1, 64, 0), (2 ** 30 + 1, 64, 64, 0)):
        assert L.cakeb200_q4_packed_bytes(*bad) == 0


@pytest.mark.parametrize("change, word", [(dict(group=16), "group"), (dict(scale=0), "scales"), (dict(n=0), "positive"), (dict(packed=0), "null weights"),
                                          (dict(packed=0x10008), "16-byte")])
def test_q4_products_refuse_bad_weights(cake, change, word):
    w = _q4(**change)
    p = ctypes.c_void_p(0x20000)
    for rc in (cake.lib().cakeb200_q4_linear(ctypes.byref(w), p, 64, None, p, 64, 1, 0, None, 0, None),
               cake.lib().cakeb200_q4_linear_dx(ctypes.byref(w), p, 64, p, 64, 1, 0, None, 0, None),
               cake.lib().cakeb200_q4_dequantize(ctypes.byref(w), p, 64, 0, None)):
        assert rc == ERR_ARG and word in _last(cake)


def test_q4_products_refuse_bad_operands(cake):
    L, w, p = cake.lib(), _q4(), ctypes.c_void_p(0x20000)
    ref = ctypes.byref(w)
    for args, word in [((ref, p, 64, None, p, 32, 1, 7, None), "type"), ((ref, p, 64, None, p, 32, -1, 0, None), "negative"),
                       ((ref, None, 64, None, p, 32, 1, 0, None), "null"), ((ref, p, 64, None, None, 32, 1, 0, None), "null"),
                       ((ref, p, 63, None, p, 32, 2, 0, None), "leading dimension"), ((ref, p, 64, None, p, 31, 2, 0, None), "leading dimension"),
                       ((None, p, 64, None, p, 32, 1, 0, None), "null weights")]:
        assert L.cakeb200_q4_linear(*args[:-1], None, 0, None) == ERR_ARG and word in _last(cake), (args, _last(cake))
    assert L.cakeb200_q4_linear_dx(ref, p, 31, p, 64, 2, 0, None, 0, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_linear(ref, None, 0, None, None, 0, 0, 0, None, 0, None) == 0  # no rows: nothing to do
    assert L.cakeb200_q4_pack(p, 31, p, None, 32, 64, 64, 1, p, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_pack(p, 32, p, None, 32, 64, 64, 1, ctypes.c_void_p(0x20001), None) == ERR_ARG and "16-byte" in _last(cake)
    assert L.cakeb200_q4_quantize(p, 63, 0, 32, 64, 64, 1, p, 32, p, None, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_quantize(p, 64, 0, 32, 64, 64, 0, p, 32, p, None, None) == ERR_ARG and "scales" in _last(cake)


def test_q4_workspace(cake):
    L = cake.lib()
    w = _q4(n=300, k=500, group=128)
    ref = ctypes.byref(w)
    assert all(L.cakeb200_q4_workspace(ref, rows, t, dx) == 0 for rows in (0, 1, 64) for t in (0, 1, 2) for dx in (0, 1))
    assert L.cakeb200_q4_workspace(ref, 65, 7, 0) == 0
    # small products need none beyond that either: 2^29 multiply-adds of _linear, 2^28 of _linear_dx, 1024 rows
    for n, k, rows, dx, none in ((300, 500, 65, 0, True), (300, 500, 1024, 0, True), (300, 500, 1025, 0, False), (1024, 1024, 512, 0, True),
                                 (1024, 1024, 513, 0, False), (1024, 1024, 256, 1, True), (1024, 1024, 257, 1, False), (65536, 65536, 65, 1, False)):
        assert (L.cakeb200_q4_workspace(ctypes.byref(_q4(n=n, k=k, group=128)), rows, 0, dx) == 0) == none, (n, k, rows, dx)
    up = lambda n: -(-n // 1024) * 1024
    # planes of x (65 x 500, rows of 504) and of W (300 x 500), and 6 tiles of 8 K blocks of 128 x 128 or 2 of 256 x 256
    parts = max(min(160, 3 * 8) * 65536, min(80, 2 * 8) * 262144)
    cake.set_option("k_pieces", 1)
    try:
        for t, tx, tw in ((0, 3, 2), (1, 2, 2), (2, 1, 1)):
            assert L.cakeb200_q4_workspace(ref, 65, t, 0) == up(tx * 65 * 504 * 2) + up(tw * 300 * 504 * 2) + parts
    finally:
        cake.set_option("k_pieces", 0)


def test_q4_python_layer_takes_cuda_tensors_only(cake):
    import numpy as np
    import torch
    codes, scales = torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 1), dtype=torch.float16)
    for a, b in ((codes, scales), (codes.numpy(), scales), (np.zeros((4, 32), np.uint8), np.ones((4, 1), np.float16))):
        with pytest.raises(TypeError):
            cake.Q4Weights(a, b, group=64)
    with pytest.raises(TypeError):
        cake.Q4Weights.quantize(torch.zeros((4, 64)))
    with pytest.raises(TypeError):
        cake.cake_q4_linear(torch.zeros((1, 64)), None)


def test_q4_without_a_device(cake):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    w, p = _q4(), ctypes.c_void_p(0x20000)
    assert cake.lib().cakeb200_q4_linear(ctypes.byref(w), p, 64, None, p, 32, 1, 0, None, 0, None) == ERR_NO_DEVICE


def test_orthogonalize_refusals(cake):
    L, p = cake.lib(), ctypes.c_void_p(0x100000)
    ws = L.cakeb200_orthogonalize_workspace(8, 12, 2, 0)
    # X twice (8 x 12, rows padded to 16), P and Q (8 x 8): two planes of two matrices each; 512 partial norms each;
    # a counter; and the parts of cut tiles: two products of one 256 x 256 tile and one K block each
    up = lambda n: -(-n // 1024) * 1024
    assert ws == 2 * up(2 * 2 * 8 * 16 * 2) + 2 * up(2 * 2 * 8 * 8 * 2) + up(2 * 512 * 8) + 1024 + 2 * 256 * 256 * 4
    assert L.cakeb200_orthogonalize_workspace(0, 4, 1, 0) == 0 and L.cakeb200_orthogonalize_workspace(4, 4, 1, 1) == 0
    assert L.cakeb200_orthogonalize_workspace(2 ** 20 + 1, 4, 1, 0) == 0

    def call(**k):
        d = dict(G=p, ldg=12, sg=96, out=p, ldo=12, so=96, rows=8, cols=12, batch=2, type=0, steps=5, a=1.0, b=0.0, c=0.0, eps=0.0, w=p, n=ws)
        d.update(k)
        return L.cakeb200_orthogonalize(*d.values(), None)

    for change, word in [(dict(G=None), "null"), (dict(w=None), "null"), (dict(ldg=11), "leading dimension"), (dict(ldo=11), "leading dimension"),
                         (dict(so=95), "overlap"), (dict(rows=0), "positive"), (dict(batch=-1), "positive"), (dict(type=1), "type"),
                         (dict(steps=0), "steps"), (dict(steps=65), "steps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                         (dict(w=ctypes.c_void_p(0x100200)), "1024-byte"), (dict(n=ws - 1), "too small"), (dict(G=ctypes.c_void_p(0x100002)), "aligned")]:
        assert call(**change) == ERR_ARG and word in _last(cake), (change, _last(cake))
    assert call(rows=2 ** 20 + 1) == ERR_TOO_LARGE
    assert call(batch=0) == 0


def test_muon_refusals(cake):
    L, p = cake.lib(), ctypes.c_void_p(0x100000)
    ws = L.cakeb200_orthogonalize_workspace(8, 12, 1, 2)

    def call(**k):
        d = dict(W=p, ldw=12, tw=2, G=p, ldg=12, tg=0, M=p, ldm=12, rows=8, cols=12, lr=0.1, mu=0.9, nesterov=1, wd=0.0, scale=1.0, steps=5, a=1.0,
                 b=0.0, c=0.0, eps=0.0, w=p, n=ws)
        d.update(k)
        return L.cakeb200_muon_step(*d.values(), None)

    for change, word in [(dict(W=None), "null"), (dict(M=None), "null"), (dict(tw=1), "types"), (dict(tg=3), "types"), (dict(ldm=11), "leading dimension"),
                         (dict(n=ws - 1), "too small"), (dict(steps=0), "steps"), (dict(M=ctypes.c_void_p(0x100002)), "aligned"), (dict(cols=0), "positive")]:
        assert call(**change) == ERR_ARG and word in _last(cake), (change, _last(cake))


@pytest.mark.parametrize("where", ["W", "G"])
@pytest.mark.parametrize("off, ldm, refused", [(0, 12, True), (4 * 90, 12, True), (4 * 8 * 12, 12, False), (-4 * 8 * 12, 12, False), (4 * 11, 40, True),
                                               (4 * 12, 40, False), (4 * 28, 40, False), (4 * 29, 40, True), (-4 * 12, 40, False), (-4, 40, True)])
def test_muon_momentum_has_its_own_memory(cake, where, off, ldm, refused):
    """8 x 12 matrices at made-up addresses: overlapping ones are refused, ones that follow one another or lie side by side
    in the rows of a wider matrix go on to the next check, of the device."""
    L = cake.lib()
    base = 1 << 20
    at = {"W": 1 << 24, "G": 1 << 26, "M": base + off}
    at[where] = base
    ld = ldm if ldm == 40 else 12
    ws = L.cakeb200_orthogonalize_workspace(8, 12, 1, 0)
    rc = L.cakeb200_muon_step(at["W"], ld, 0, at["G"], ld, 0, at["M"], ldm, 8, 12, 0.1, 0.9, 1, 0.0, 1.0, 5, 1.0, 0.0, 0.0, 0.0, 1 << 28, ws, None)
    assert rc != 0 and ("overlaps" in _last(cake)) == refused, _last(cake)


def test_orthogonalize_python_layer_takes_cuda_tensors_only(cake):
    import numpy as np
    import torch
    for g in (torch.zeros((4, 4)), np.zeros((4, 4), np.float32), None):
        with pytest.raises(TypeError):
            cake.cake_orthogonalize(g)
        with pytest.raises(TypeError):
            cake.cake_muon_step(g, g, g, 0.1)


def test_muon_momentum_stays_in_float32_across_a_reload():
    import torch
    from cake_on_cpu_b200.cake import cake_muon
    w = [torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(2, 5))]
    m = [torch.full((3, 4), 1 + 2.0 ** -20), torch.full((2, 5), 3.0)]
    first = cake_muon(w, lr=0.3)
    first.state[w[0]]["momentum"], first.state[w[1]]["momentum"] = m
    again = [torch.nn.Parameter(p.detach().clone()) for p in w]
    second = cake_muon(again, lr=0.1)
    second.load_state_dict(first.state_dict())
    assert second.param_groups[0]["lr"] == 0.3
    for p, want in zip(again, m):
        got = second.state[p]["momentum"]
        assert got.dtype == torch.float32 and torch.equal(got, want) and got.data_ptr() != want.data_ptr()
