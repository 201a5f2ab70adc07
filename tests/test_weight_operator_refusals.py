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
    # 16 x 64 blocks of 512 bytes, 16 scales (2 bytes) and zero points (1 byte) per block row and group
    assert L.cakeb200_q4_packed_bytes(16, 64, 64, 0) == 512 + 32
    assert L.cakeb200_q4_packed_bytes(17, 65, 32, 1) == 2 * 2 * 512 + 2 * 4 * 16 * 3
    assert L.cakeb200_q4_packed_bytes(16384, 16384, 128, 0) == 16384 * 16384 // 2 + 16384 * 128 * 2
    for bad in ((0, 64, 64, 0), (16, 0, 64, 0), (16, 64, 48, 0), (16, -1, 64, 0), (2 ** 30 + 1, 64, 64, 0)):
        assert L.cakeb200_q4_packed_bytes(*bad) == 0


@pytest.mark.parametrize("change, word", [(dict(group=16), "group"), (dict(scale=0), "scales"), (dict(n=0), "positive"), (dict(packed=0), "null weights"),
                                          (dict(packed=0x10008), "16-byte")])
def test_q4_products_refuse_bad_weights(cake, change, word):
    w = _q4(**change)
    p = ctypes.c_void_p(0x20000)
    for rc in (cake.lib().cakeb200_q4_linear(ctypes.byref(w), p, 64, None, p, 64, 1, 0, None),
               cake.lib().cakeb200_q4_linear_dx(ctypes.byref(w), p, 64, p, 64, 1, 0, None),
               cake.lib().cakeb200_q4_dequantize(ctypes.byref(w), p, 64, 0, None)):
        assert rc == ERR_ARG and word in _last(cake)


def test_q4_products_refuse_bad_operands(cake):
    L, w, p = cake.lib(), _q4(), ctypes.c_void_p(0x20000)
    ref = ctypes.byref(w)
    for args, word in [((ref, p, 64, None, p, 32, 1, 7, None), "type"), ((ref, p, 64, None, p, 32, -1, 0, None), "negative"),
                       ((ref, None, 64, None, p, 32, 1, 0, None), "null"), ((ref, p, 64, None, None, 32, 1, 0, None), "null"),
                       ((ref, p, 63, None, p, 32, 2, 0, None), "leading dimension"), ((ref, p, 64, None, p, 31, 2, 0, None), "leading dimension"),
                       ((None, p, 64, None, p, 32, 1, 0, None), "null weights")]:
        assert L.cakeb200_q4_linear(*args) == ERR_ARG and word in _last(cake), (args, _last(cake))
    assert L.cakeb200_q4_linear_dx(ref, p, 31, p, 64, 2, 0, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_linear(ref, None, 0, None, None, 0, 0, 0, None) == 0  # no rows: nothing to do
    assert L.cakeb200_q4_pack(p, 31, p, None, 32, 64, 64, 1, p, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_pack(p, 32, p, None, 32, 64, 64, 1, ctypes.c_void_p(0x20001), None) == ERR_ARG and "16-byte" in _last(cake)
    assert L.cakeb200_q4_quantize(p, 63, 0, 32, 64, 64, 1, p, 32, p, None, None) == ERR_ARG and "leading dimension" in _last(cake)
    assert L.cakeb200_q4_quantize(p, 64, 0, 32, 64, 64, 0, p, 32, p, None, None) == ERR_ARG and "scales" in _last(cake)


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
    assert cake.lib().cakeb200_q4_linear(ctypes.byref(w), p, 64, None, p, 32, 1, 0, None) == ERR_NO_DEVICE
