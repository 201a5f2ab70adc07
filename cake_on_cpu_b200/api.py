"""ctypes binding of include/cake_b200.h and the reference-shaped operators."""
import ctypes
import os

import numpy as np

KMN, MKN, NKM, NA = 0, 1, 2, 3
KERNEL_AUTO, KERNEL_TF32X3, KERNEL_FFMA = 0, 1, 2

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libcake_b200.so")
_lib = None

_fp = ctypes.POINTER(ctypes.c_float)
_i, _vp, _sz = ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t


class CakeError(RuntimeError):
    """A C-ABI call returned a negative status."""

    def __init__(self, code, text):
        super().__init__("cake_b200 status %d: %s" % (code, text))
        self.code = code


class Stats(ctypes.Structure):
    """cakeb200_stats: timings (ms, CUDA events) and choices of the last call."""
    _fields_ = [("ms_h2d", ctypes.c_float), ("ms_prepass", ctypes.c_float), ("ms_gemm", ctypes.c_float),
                ("ms_d2h", ctypes.c_float), ("kernel", _i), ("sched", _i), ("tile_m", _i), ("tile_n", _i),
                ("tile_k", _i), ("launches", _i)]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_}


class ConvPlan(ctypes.Structure):
    """cakeb200_conv_plan: how a convolution is laid out on the tensor-core path."""
    _fields_ = [(n, _i) for n in ("route", "tiles", "channel_tile", "positions_tile", "k_slices", "stages", "ring", "smem_bytes")]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_}


class Cntx(ctypes.Structure):
    """cakeb200_cntx: the fields of cake_cntx_t the block-sizing formulas read
    (reference include/common.h:138-151)."""
    _fields_ = [("alpha_n", ctypes.c_double), ("mr", _i), ("nr", _i), ("L1", _i), ("L2", _i), ("L3", _i),
                ("ncores", _i)]

    @classmethod
    def make(cls, L1, L2, L3, ncores, mr=6, nr=16):
        c = cls()
        c.alpha_n, c.mr, c.nr, c.L1, c.L2, c.L3, c.ncores = 1.0, mr, nr, L1, L2, L3, ncores
        return c


class BlkDims(ctypes.Structure):
    """cakeb200_blk_dims == blk_dims_t (reference include/common.h:108-135)."""
    _names = ["m_c", "k_c", "n_c", "m_c1", "k_c1", "n_c1", "m_c1_last_core", "n_c1_last_core", "k_c1_last_core",
              "mr_rem", "nr_rem", "k_rem", "p_l", "pm_l", "pn_l", "pm", "pn", "m_pad", "k_pad", "n_pad", "Mb", "Kb",
              "Nb", "M_padded", "N_padded", "sch"]
    _fields_ = [(n, _i) for n in _names]

    def as_dict(self):
        return {n: getattr(self, n) for n in self._names}


_SIGNATURES = {
    "cakeb200_last_error": (ctypes.c_char_p, []),
    "cakeb200_get_stats": (None, [ctypes.POINTER(Stats)]),
    "cakeb200_device_count": (_i, []),
    "cakeb200_query_cntx": (_i, [ctypes.POINTER(Cntx)]),
    "cakeb200_sgemm": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "cakeb200_sgemm_after": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp, _vp]),
    "cakeb200_sgemm_async": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "cakeb200_sgemm_batched": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "cakeb200_sp_sgemm": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "cakeb200_conv2d": (_i, [_vp, _vp, _vp] + [_i] * 10 + [_vp]),
    "cakeb200_im2col": (_i, [_vp, _vp] + [_i] * 8 + [_vp]),
    "cakeb200_init_block_dims": (_i, [_i, _i, _i, _i, ctypes.POINTER(BlkDims), ctypes.POINTER(Cntx), _i, _i, _i, _i]),
    "cakeb200_derive_schedule": (_i, [_i, _i, _i, _i, _i, ctypes.POINTER(Cntx)]),
    "cakeb200_set_schedule": (_i, [_i, _i, _i, _i]),
    "cakeb200_packed_A_size": (_sz, [_i, _i, _i, ctypes.POINTER(BlkDims), ctypes.POINTER(Cntx), _i]),
    "cakeb200_packed_B_size": (_sz, [_i, _i, _i, ctypes.POINTER(BlkDims), ctypes.POINTER(Cntx)]),
    "cakeb200_packed_C_size": (_sz, [_i, _i, _i, ctypes.POINTER(BlkDims), ctypes.POINTER(Cntx), _i]),
}
for _n in ("pack_A", "unpack_A", "pack_B", "unpack_B", "pack_C", "unpack_C"):
    _SIGNATURES["cakeb200_" + _n] = (_i, [_vp, _vp, _i, _i, _i, ctypes.POINTER(BlkDims), ctypes.POINTER(Cntx), _vp])

_SIGNATURES["cakeb200_profile_begin"] = (_i, [])
_SIGNATURES["cakeb200_profile_end"] = (_i, [ctypes.POINTER(ctypes.c_float), ctypes.POINTER(ctypes.c_float), ctypes.POINTER(_i)])
_SIGNATURES["cakeb200_sgemm_ex"] = (_i, [_vp, _i, _i, _vp, _i, _i, _vp, _i, _i, _i, _i, _vp, _i, _i, _i, _vp])
_SIGNATURES["cakeb200_conv_plan_query"] = (_i, [_i] * 10 + [ctypes.POINTER(ConvPlan)])
_SIGNATURES["cakeb200_selftest_bounded_wait"] = (_i, [_i, _vp])
_SIGNATURES["cakeb200_selftest_bounded_wait_pair"] = (_i, [_i, _vp])
_pi = ctypes.POINTER(_i)
_SIGNATURES["cakeb200_kshard_rows"] = (_i, [_i, _i, _i, _pi, _pi])
_SIGNATURES["cakeb200_kshard_supported"] = (_i, [_i, _i, _i, _i])
_SIGNATURES["cakeb200_kshard_create"] = (_i, [_i, _i, _i, _i, ctypes.POINTER(_vp), _vp])
_SIGNATURES["cakeb200_kshard_connect_ipc"] = (_i, [_vp, _vp])
_SIGNATURES["cakeb200_kshard_connect_local"] = (_i, [_vp, ctypes.POINTER(_vp)])
_SIGNATURES["cakeb200_kshard_partial"] = (_i, [_vp, _vp, _i, _vp, _i, _i, _vp])
_SIGNATURES["cakeb200_kshard_finish"] = (_i, [_vp, _vp, _i, _vp])
_SIGNATURES["cakeb200_kshard_destroy"] = (_i, [_vp])
_SIGNATURES["cakeb200_sgemv"] = (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp])
_pf = ctypes.POINTER(ctypes.c_float)
_SIGNATURES["cakeb200_tf32_peak"] = (_i, [ctypes.c_float, _pf, _pf, _vp])
_SIGNATURES["cakeb200_planes_create"] = (_i, [_vp, _i, _i, _i, ctypes.POINTER(_vp), _vp])
_SIGNATURES["cakeb200_planes_destroy"] = (_i, [_vp])
_SIGNATURES["cakeb200_sgemm_planes"] = (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp])
TUNE_COST = ctypes.CFUNCTYPE(ctypes.c_double, _i, _i, _i, _vp)
TUNE_COST_SHAPE = ctypes.CFUNCTYPE(ctypes.c_double, _i, _i, _i, _i, _vp)
_SIGNATURES["cakeb200_tune"] = (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _i, _vp])
_SIGNATURES["cakeb200_tune_search"] = (_i, [_i, _i, _i, _i, _i, ctypes.c_ulonglong, TUNE_COST, _vp, _pi, _pi, _pi, _pf, _pi])
_SIGNATURES["cakeb200_tune_put"] = (_i, [_i, _i, _i, _i, _i, _i, _i, ctypes.c_float])
_SIGNATURES["cakeb200_tune_get"] = (_i, [_i, _i, _i, _i, _pi, _pi, _pi, _pf])
_SIGNATURES["cakeb200_tune_search_shape"] = (_i, [_i, _i, _i, _i, _i, ctypes.c_ulonglong, TUNE_COST_SHAPE, _vp, _pi, _pi, _pi, _pi, _pf, _pi])
_SIGNATURES["cakeb200_tune_put_shape"] = (_i, [_i, _i, _i, _i, _i, _i, _i, _i, ctypes.c_float])
_SIGNATURES["cakeb200_tune_get_shape"] = (_i, [_i, _i, _i, _i, _pi, _pi, _pi, _pi, _pf])
_SIGNATURES["cakeb200_tune_clear"] = (_i, [])
_SIGNATURES["cakeb200_tune_save"] = (_i, [ctypes.c_char_p])
_SIGNATURES["cakeb200_tune_load"] = (_i, [ctypes.c_char_p])
_SIGNATURES["cakeb200_set_option"] = (_i, [ctypes.c_char_p, _i])
_SIGNATURES["cakeb200_get_option"] = (_i, [ctypes.c_char_p])
_SIGNATURES["cakeb200_select_devices"] = (_i, [_pi, _i, _i, _i, _i, _i, _pi])
_SIGNATURES["cakeb200_sgemm_noalloc"] = (_i, [_vp, _vp, _vp, _i, _i, _i, _vp])

F32, F16, BF16 = 0, 1, 2
_ll = ctypes.c_longlong


class _Q4(ctypes.Structure):
    """cakeb200_q4."""
    _fields_ = [("packed", _vp), ("out_features", _i), ("in_features", _i), ("group", _i), ("scale_type", _i), ("has_zeros", _i)]


_pq4 = ctypes.POINTER(_Q4)
_SIGNATURES["cakeb200_q4_packed_bytes"] = (_sz, [_i, _i, _i, _i])
_SIGNATURES["cakeb200_q4_quantize"] = (_i, [_vp, _ll, _i, _i, _i, _i, _i, _vp, _ll, _vp, _vp, _vp])
_SIGNATURES["cakeb200_q4_pack"] = (_i, [_vp, _ll, _vp, _vp, _i, _i, _i, _i, _vp, _vp])
_SIGNATURES["cakeb200_q4_dequantize"] = (_i, [_pq4, _vp, _ll, _i, _vp])
_SIGNATURES["cakeb200_q4_workspace"] = (_sz, [_pq4, _i, _i, _i])
_SIGNATURES["cakeb200_q4_linear"] = (_i, [_pq4, _vp, _ll, _vp, _vp, _ll, _i, _i, _vp, _sz, _vp])
_SIGNATURES["cakeb200_q4_linear_dx"] = (_i, [_pq4, _vp, _ll, _vp, _ll, _i, _i, _vp, _sz, _vp])
_f, _d = ctypes.c_float, ctypes.c_double
_SIGNATURES["cakeb200_selftest_orthogonalize_wait"] = (_i, [_vp, _vp, _vp, _i, _i, _vp, _sz, _vp])
_SIGNATURES["cakeb200_orthogonalize_workspace"] = (_sz, [_i, _i, _i, _i])
_SIGNATURES["cakeb200_orthogonalize"] = (_i, [_vp, _ll, _ll, _vp, _ll, _ll] + [_i] * 5 + [_f] * 4 + [_vp, _sz, _vp])
_SIGNATURES["cakeb200_muon_step"] = (_i, [_vp, _ll, _i, _vp, _ll, _i, _vp, _ll, _i, _i, _d, _d, _i, _d, _d, _i, _f, _f, _f, _f, _vp, _sz, _vp])

EXPORTED_SYMBOLS = sorted(_SIGNATURES)


def library_path():
    return _LIB_PATH


def lib():
    """The loaded shared library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError("libcake_b200.so is missing: run `python -m cake_on_cpu_b200.build` "
                               "(there is no CPU fallback)")
        L = ctypes.CDLL(_LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


def _check(rc):
    if rc != 0:
        raise CakeError(rc, lib().cakeb200_last_error().decode(errors="replace"))


def last_stats():
    s = Stats()
    lib().cakeb200_get_stats(ctypes.byref(s))
    return s.as_dict()


def device_count():
    return lib().cakeb200_device_count()


def select_devices(cc_major, current, p, cap=0, M=1 << 30):
    """Device ordinals a host-pointer product with p > 1 is spread over by the C++ API
    (cakeb200_select_devices; host logic, no device needed)."""
    n = len(cc_major)
    majors = (_i * n)(*cc_major)
    out = (_i * max(n, 1))()
    got = lib().cakeb200_select_devices(majors, n, current, p, cap, M, out)
    return [out[k] for k in range(got)]


def _is_torch(x):
    return type(x).__module__.startswith("torch")


def _ptr(x):
    """Raw address of a contiguous float32 numpy array or torch tensor."""
    if _is_torch(x):
        import torch
        if x.dtype != torch.float32 or not x.is_contiguous():
            raise TypeError("expected a contiguous float32 tensor")
        return ctypes.c_void_p(x.data_ptr())
    if not isinstance(x, np.ndarray) or x.dtype != np.float32 or not x.flags["C_CONTIGUOUS"]:
        raise TypeError("expected a C-contiguous float32 array")
    return ctypes.c_void_p(x.ctypes.data)


def _empty_like_kind(ref, shape):
    if _is_torch(ref):
        import torch
        return torch.empty(shape, dtype=torch.float32, device=ref.device)
    return np.empty(shape, np.float32)


def _need_shape(x, shape, what):
    """Raise before any launch when a caller-supplied array does not have the shape the
    kernels will read or write through its raw pointer."""
    if tuple(x.shape) != tuple(shape):
        raise ValueError("%s has shape %s, expected %s" % (what, tuple(x.shape), tuple(shape)))


def _stream_of(x, stream):
    if stream is not None:
        return ctypes.c_void_p(int(stream))
    if _is_torch(x) and x.is_cuda:
        import torch
        return ctypes.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)
    return None


# ------------------------------------------------------------------ the product

def cake_sgemm(A, B, C=None, p=1, cake_cntx=None, packedA=False, packedB=False, alpha=1.0, beta=0.0, sch=NA,
               kernel=KERNEL_AUTO, stream=None, b_ready=None):
    """C = A @ B through the reference's operator interface
    (cake_sgemm, reference include/cake.h:12-14, src/cake_sgemm.cpp:9-175).

    ``alpha`` is accepted and ignored and ``beta`` is a flag, exactly as in the
    reference: K-first overwrites C, M-first / N-first add A@B to C when
    ``beta != 0``.  ``sch`` picks the tile order (NA = derive from the shape).
    ``p`` and ``cake_cntx`` are accepted for signature parity; one process
    drives one GPU here.  ``b_ready`` (a ``torch.cuda.Event`` already recorded, or a
    raw cudaEvent_t) makes the kernels wait until B is complete, see
    cakeb200_sgemm_after.  Returns C.
    """
    if packedA or packedB:
        raise NotImplementedError("pre-packed operands go through the C++ API (include/cake.h)")
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        C = _empty_like_kind(A, (M, N))
        beta = 0.0
    _need_shape(C, (M, N), "C")
    accumulate = 1 if (beta != 0 and sch in (MKN, NKM)) else 0
    if beta != 0 and sch == NA:
        # the schedule decides whether beta is honoured; resolve it the way the library will
        accumulate = 1 if last_schedule_for(M, N, K) != KMN else 0
    if stream is None and not (_is_torch(C) and C.is_cuda) and _is_torch(B) and B.is_cuda:
        stream = _stream_of(B, None).value  # host result, device B: run on the stream that produces B
    if b_ready is not None:
        ev = ctypes.c_void_p(b_ready.cuda_event if hasattr(b_ready, "cuda_event") else int(b_ready))
        _check(lib().cakeb200_sgemm_after(_ptr(A), _ptr(B), _ptr(C), M, N, K, accumulate, sch, kernel,
                                          _stream_of(C, stream), ev))
    else:
        _check(lib().cakeb200_sgemm(_ptr(A), _ptr(B), _ptr(C), M, N, K, accumulate, sch, kernel, _stream_of(C, stream)))
    return C


def cake_sgemm_ex(A, B, C=None, trans_a=False, trans_b=False, bias=None, accumulate=False, sch=NA,
                  kernel=KERNEL_AUTO, stream=None):
    """C (+)= op(A) @ op(B) (+ bias) on CUDA tensors, enqueued on the current stream.

    ``A`` and ``B`` are 2-D float32 tensors whose rows are contiguous (a row
    stride is allowed, so column slices work); ``trans_a`` / ``trans_b`` multiply
    the transpose of the tensor as stored.  ``bias`` has one entry per column of
    C and is added in the kernel's epilogue.  This is the product behind the
    linear layer (reference src/linear.cpp:12-102) without its transposed copies.
    """
    import torch
    for t in (A, B) + ((C,) if C is not None else ()) + ((bias,) if bias is not None else ()):
        if not (_is_torch(t) and t.is_cuda and t.dtype == torch.float32):
            raise TypeError("cake_sgemm_ex needs float32 CUDA tensors")
    for t in (A, B) + ((C,) if C is not None else ()):
        if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise TypeError("operands must be 2-D with contiguous rows")
    M, K = (A.shape[1], A.shape[0]) if trans_a else A.shape
    K2, N = (B.shape[1], B.shape[0]) if trans_b else B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        C = torch.empty((M, N), dtype=torch.float32, device=A.device)
        accumulate = False
    if tuple(C.shape) != (M, N):
        raise ValueError("C has the wrong shape")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != N or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous vector with one entry per column of C")
    ld = lambda t: t.stride(0) if t.shape[0] > 1 else t.shape[1]
    _check(lib().cakeb200_sgemm_ex(ctypes.c_void_p(A.data_ptr()), ld(A), int(trans_a), ctypes.c_void_p(B.data_ptr()), ld(B),
                                   int(trans_b), ctypes.c_void_p(C.data_ptr()), ld(C), M, N, K,
                                   ctypes.c_void_p(bias.data_ptr()) if bias is not None else None,
                                   int(bool(accumulate)), sch, kernel, _stream_of(C, stream)))
    return C


def last_schedule_for(M, N, K):
    """Schedule the library derives for a shape on the current device."""
    c = cake_query_cntx()
    c.ncores = 1
    return init_block_dims(M, N, K, 1, c, NA).sch


def cake_sgemm_async(dA, dB, dC, M, N, K, accumulate=0, sch=NA, kernel=KERNEL_AUTO, stream=0):
    """Enqueue C = A @ B on ``stream`` for raw device addresses; no synchronisation."""
    _check(lib().cakeb200_sgemm_async(ctypes.c_void_p(dA), ctypes.c_void_p(dB), ctypes.c_void_p(dC), M, N, K,
                                      accumulate, sch, kernel, ctypes.c_void_p(stream)))


def cake_sgemm_batched(A, B, C=None, kernel=KERNEL_AUTO, stream=None):
    """Batch of independent products, A[b] @ B[b] (the reference's small-matrix
    path, reference include/cake.h:52-72, is one cake_sgemm per item)."""
    batch, M, K = A.shape
    _, _, N = B.shape
    _need_shape(B, (batch, K, N), "B")
    if C is None:
        C = _empty_like_kind(A, (batch, M, N))
    _need_shape(C, (batch, M, N), "C")
    _check(lib().cakeb200_sgemm_batched(_ptr(A), _ptr(B), _ptr(C), M, N, K, batch, kernel, _stream_of(C, stream)))
    return C


def cake_sgemv(A, x, y=None, col_major=False, accumulate=False, stream=None):
    """y (+)= A x (cake_sgemv of reference examples/cake_gemv.cpp:716-765).  ``col_major``: A is given as
    the (K, M) array whose element [k, m] is A[m, k], the reference driver's layout; otherwise A is (M, K)."""
    if col_major:
        K, M = A.shape
    else:
        M, K = A.shape
    if (x.numel() if _is_torch(x) else x.size) != K:
        raise ValueError("vector length differs from the matrix")
    if y is None:
        y = _empty_like_kind(A, (M,))
        accumulate = False
    if (y.numel() if _is_torch(y) else y.size) != M:
        raise ValueError("y has %d elements, expected %d" % ((y.numel() if _is_torch(y) else y.size), M))
    _check(lib().cakeb200_sgemv(_ptr(A), _ptr(x), _ptr(y), M, K, int(bool(col_major)), int(bool(accumulate)),
                                _stream_of(y, stream)))
    return y


def cake_sp_sgemm(A, B, C=None, kernel=KERNEL_FFMA, stream=None):
    """C = A @ B for a mostly-zero A (row-skipping product of the reference's
    sparse microkernel, reference src/kernels/haswell/sparse.cpp:7-131)."""
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        C = _empty_like_kind(A, (M, N))
    _need_shape(C, (M, N), "C")
    _check(lib().cakeb200_sp_sgemm(_ptr(A), _ptr(B), _ptr(C), M, N, K, kernel, _stream_of(C, stream)))
    return C


def cake_conv2d(x, w, stride=1, pad=0, out=None, kernel=KERNEL_AUTO, stream=None):
    """NCHW convolution via im2col + SGEMM (reference examples/cake_conv.cpp:1007-1066)."""
    b, cin, H, W = x.shape
    cout, cin2, hf, wf = w.shape
    if cin != cin2:
        raise ValueError("channel mismatch")
    Ho, Wo = (H + 2 * pad - hf) // stride + 1, (W + 2 * pad - wf) // stride + 1
    if out is None:
        out = _empty_like_kind(x, (b, cout, Ho, Wo))
    _need_shape(out, (b, cout, Ho, Wo), "out")
    _check(lib().cakeb200_conv2d(_ptr(x), _ptr(w), _ptr(out), b, cin, H, W, cout, hf, wf, stride, pad, kernel,
                                 _stream_of(out, stream)))
    return out


def conv_plan(batch, cin, H, W, cout, hf, wf, stride=1, pad=0, sm_count=148):
    """Route and tiling cake_conv2d takes on the tensor-core path (host logic, no device needed)."""
    out = ConvPlan()
    _check(lib().cakeb200_conv_plan_query(batch, cin, H, W, cout, hf, wf, stride, pad, sm_count, ctypes.byref(out)))
    return out.as_dict()


def im2col(x, hf, wf, stride=1, pad=0, stream=None):
    """im_2_col (reference examples/cake_conv.cpp:1178-1213) with batch and padding."""
    b, cin, H, W = x.shape
    Ho, Wo = (H + 2 * pad - hf) // stride + 1, (W + 2 * pad - wf) // stride + 1
    col = _empty_like_kind(x, (cin * hf * wf, b * Ho * Wo))
    _check(lib().cakeb200_im2col(_ptr(x), _ptr(col), b, cin, H, W, hf, wf, stride, pad, _stream_of(col, stream)))
    return col


# ------------------------------------------------------- context and tiling

def cake_query_cntx():
    c = Cntx()
    _check(lib().cakeb200_query_cntx(ctypes.byref(c)))
    return c


def init_block_dims(M, N, K, p, cake_cntx, sch=NA, mcu=0, kcu=0, ncu=0):
    x = BlkDims()
    _check(lib().cakeb200_init_block_dims(M, N, K, p, ctypes.byref(x), ctypes.byref(cake_cntx), sch, mcu, kcu, ncu))
    return x


def derive_schedule(M, N, K, p, mc_ret, cake_cntx):
    return lib().cakeb200_derive_schedule(M, N, K, p, mc_ret, ctypes.byref(cake_cntx))


def set_schedule(sch, M, N, K):
    return lib().cakeb200_set_schedule(sch, M, N, K)


def cake_sgemm_packed_A_size(M, K, p, x, cake_cntx, sch):
    return lib().cakeb200_packed_A_size(M, K, p, ctypes.byref(x), ctypes.byref(cake_cntx), sch)


def cake_sgemm_packed_B_size(K, N, p, x, cake_cntx):
    return lib().cakeb200_packed_B_size(K, N, p, ctypes.byref(x), ctypes.byref(cake_cntx))


def cake_sgemm_packed_C_size(M, N, p, x, cake_cntx, sch):
    return lib().cakeb200_packed_C_size(M, N, p, ctypes.byref(x), ctypes.byref(cake_cntx), sch)


# ------------------------------------------------------------------ packing

def _pack(name, mat, packed, d0, d1, p, x, cake_cntx, stream):
    fn = getattr(lib(), "cakeb200_" + name)
    _need_shape(mat, (d0, d1), "matrix")
    kind = name[-1]
    want = (cake_sgemm_packed_A_size(d0, d1, p, x, cake_cntx, x.sch) if kind == "A" else
            cake_sgemm_packed_B_size(d0, d1, p, x, cake_cntx) if kind == "B" else
            cake_sgemm_packed_C_size(d0, d1, p, x, cake_cntx, x.sch)) // 4
    have = packed.numel() if _is_torch(packed) else packed.size
    if have < want:
        raise ValueError("packed buffer holds %d floats, the layout needs %d" % (have, want))
    _check(fn(_ptr(mat), _ptr(packed), d0, d1, p, ctypes.byref(x), ctypes.byref(cake_cntx), _stream_of(packed, stream)))


def pack_A(A, M, K, p, x, cake_cntx, A_p=None, stream=None):
    if A_p is None:
        A_p = _empty_like_kind(A, (cake_sgemm_packed_A_size(M, K, p, x, cake_cntx, x.sch) // 4,))
    _pack("pack_A", A, A_p, M, K, p, x, cake_cntx, stream)
    return A_p


def pack_B(B, K, N, p, x, cake_cntx, B_p=None, stream=None):
    if B_p is None:
        B_p = _empty_like_kind(B, (cake_sgemm_packed_B_size(K, N, p, x, cake_cntx) // 4,))
    _pack("pack_B", B, B_p, K, N, p, x, cake_cntx, stream)
    return B_p


def pack_C(C, M, N, p, x, cake_cntx, C_p=None, stream=None):
    if C_p is None:
        C_p = _empty_like_kind(C, (cake_sgemm_packed_C_size(M, N, p, x, cake_cntx, x.sch) // 4,))
    _pack("pack_C", C, C_p, M, N, p, x, cake_cntx, stream)
    return C_p


def unpack_C(C_p, M, N, p, x, cake_cntx, C=None, stream=None):
    if C is None:
        C = _empty_like_kind(C_p, (M, N))
    _pack("unpack_C", C, C_p, M, N, p, x, cake_cntx, stream)
    return C


def unpack_A(A_p, M, K, p, x, cake_cntx, A=None, stream=None):
    if A is None:
        A = _empty_like_kind(A_p, (M, K))
    _pack("unpack_A", A, A_p, M, K, p, x, cake_cntx, stream)
    return A


def unpack_B(B_p, K, N, p, x, cake_cntx, B=None, stream=None):
    if B is None:
        B = _empty_like_kind(B_p, (K, N))
    _pack("unpack_B", B, B_p, K, N, p, x, cake_cntx, stream)
    return B


NOALLOC_SCRATCH_BYTES = 17 << 20


def cake_sgemm_noalloc(A, B, C=None, stream=None):
    """C = A @ B for callers that must not allocate device memory (embedded in
    another framework's memory pool, fixed memory budget, plug-ins that are only
    handed buffers).  CUDA tensors only; the scratch is a fixed 17 MiB array in
    the library, so shapes are limited (1024 x 1024 x 1024 fits) and calls that
    overlap on the GPU race on it.  The first call on a device should happen
    outside any stream capture.  Pass ``C`` to keep the call itself free of
    allocations on the Python side as well."""
    if not (_is_torch(A) and A.is_cuda and _is_torch(B) and B.is_cuda):
        raise TypeError("cake_sgemm_noalloc takes CUDA tensors")
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        C = _empty_like_kind(A, (M, N))
    if not (_is_torch(C) and C.is_cuda):
        raise TypeError("cake_sgemm_noalloc takes CUDA tensors")
    _need_shape(C, (M, N), "C")
    _check(lib().cakeb200_sgemm_noalloc(_ptr(A), _ptr(B), _ptr(C), M, N, K, _stream_of(C, stream)))
    return C


IPC_HANDLE_BYTES = 64


def kshard_rows(M, world, rank):
    """[lo, hi) of the rows of C that `rank` owns in a K-sharded product (whole 128-row tiles)."""
    lo, hi = _i(), _i()
    _check(lib().cakeb200_kshard_rows(M, world, rank, ctypes.byref(lo), ctypes.byref(hi)))
    return lo.value, hi.value


def kshard_supported(M, N, K_local, sm_count=0):
    """Whether the K-sharded exchange takes a product of this shape per rank (few tiles, deep K).
    sm_count > 0 answers without a device."""
    return bool(lib().cakeb200_kshard_supported(M, N, K_local, sm_count))


class KShard:
    """One rank's end of a product whose K is sharded over the GPUs of a box: this rank's
    partial rows go straight into the owners' memory while its tiles are summed, and the
    owner adds the slots of all ranks in rank order.  `handle` is what the other ranks
    need (64 bytes) for `connect`; `KShard.connect_local` wires objects of one process."""

    def __init__(self, world, rank, M, N):
        self.world, self.rank, self.M, self.N = world, rank, M, N
        self._h = _vp()
        buf = (ctypes.c_ubyte * IPC_HANDLE_BYTES)()
        _check(lib().cakeb200_kshard_create(world, rank, M, N, ctypes.byref(self._h), buf))
        self.handle = bytes(buf)
        self.rows = kshard_rows(M, world, rank)

    def connect(self, handles):
        """handles: the `handle` of every rank, in rank order (one bytes object of world x 64, or a list)."""
        blob = handles if isinstance(handles, (bytes, bytearray)) else b"".join(handles)
        if len(blob) != self.world * IPC_HANDLE_BYTES:
            raise ValueError("expected one 64-byte handle per rank")
        arr = (ctypes.c_ubyte * len(blob)).from_buffer_copy(blob)
        _check(lib().cakeb200_kshard_connect_ipc(self._h, arr))

    @staticmethod
    def connect_local(objects):
        arr = (_vp * len(objects))(*[o._h.value for o in objects])
        for o in objects:
            _check(lib().cakeb200_kshard_connect_local(o._h, arr))

    def partial(self, A_k, B_k, stream=None):
        """A_k: this rank's columns of A (M x Kr, rows may be strided), B_k: the same rows of B (Kr x N)."""
        if A_k.stride(1) != 1 or B_k.stride(1) != 1:
            raise TypeError("operands need unit stride along their rows")
        M, Kr = A_k.shape
        if (M, B_k.shape[0], B_k.shape[1]) != (self.M, Kr, self.N):
            raise ValueError("operand shapes do not match this product")
        _check(lib().cakeb200_kshard_partial(self._h, _vp(A_k.data_ptr()), A_k.stride(0), _vp(B_k.data_ptr()), B_k.stride(0),
                                             Kr, _stream_of(A_k, stream)))

    def finish(self, out=None, wait_limit_us=0, stream=None):
        """This rank's rows of C (rows[0]:rows[1]); blocks until they are complete."""
        import torch
        lo, hi = self.rows
        if out is None:
            out = torch.empty((hi - lo, self.N), dtype=torch.float32, device="cuda")
        if out.numel() != (hi - lo) * self.N:
            raise ValueError("out has %d elements, expected %d" % (out.numel(), (hi - lo) * self.N))
        _check(lib().cakeb200_kshard_finish(self._h, _ptr(out), wait_limit_us, _stream_of(out, stream)))
        return out

    def close(self):
        if self._h:
            lib().cakeb200_kshard_destroy(self._h)
            self._h = _vp()


def tf32_peak(ms_target=0.0, stream=None):
    """(TFLOP/s, ms): measured dense TF32 issue rate of the current device (cakeb200_tf32_peak)."""
    t, ms = ctypes.c_float(), ctypes.c_float()
    _check(lib().cakeb200_tf32_peak(ms_target, ctypes.byref(t), ctypes.byref(ms), ctypes.c_void_p(int(stream)) if stream else None))
    return t.value, ms.value


class Planes:
    """An operand split once into its TF32 hi / lo planes and kept on the device (cakeb200_planes_create):
    the counterpart of an operand packed once with pack_A / pack_B and passed with packedA / packedB = 1.
    ``Planes(A)`` for the left operand (M x K), ``Planes(B, is_b=True)`` for the right one (K x N)."""

    def __init__(self, mat, is_b=False, stream=None):
        r, c = mat.shape
        self.rows, self.K, self.is_b = (c, r, True) if is_b else (r, c, False)
        self._h = _vp()
        _check(lib().cakeb200_planes_create(_ptr(mat), self.rows, self.K, int(is_b), ctypes.byref(self._h), _stream_of(mat, stream)))

    def close(self):
        if self._h:
            lib().cakeb200_planes_destroy(self._h)
            self._h = _vp()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def cake_sgemm_planes(A, B, C=None, sch=NA, accumulate=False, stream=None):
    """C (+)= A @ B where A and / or B is a ``Planes`` object (the other a matrix): cakeb200_sgemm_planes."""
    pa, pb = isinstance(A, Planes), isinstance(B, Planes)
    if not (pa or pb):
        raise TypeError("at least one operand must be a Planes object")
    M, K = (A.rows, A.K) if pa else A.shape
    K2, N = (B.K, B.rows) if pb else B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        if pa and pb:
            raise ValueError("give C when both operands are planes")
        C = _empty_like_kind(B if pa else A, (M, N))
        accumulate = False
    _need_shape(C, (M, N), "C")
    _check(lib().cakeb200_sgemm_planes(A._h if pa else None, None if pa else _ptr(A), B._h if pb else None, None if pb else _ptr(B),
                                       _ptr(C), M, N, K, int(bool(accumulate)), sch, _stream_of(C, stream)))
    return C


# ------------------------------------------------------- weights held in 4 bits

def _type_code(dtype, what, allowed=(F32, F16, BF16)):
    """The C ABI's number of a torch element type; raises for one the operator does not take."""
    import torch
    code = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}.get(dtype)
    if code not in allowed:
        raise TypeError("%s cannot be %s" % (what, dtype))
    return code


def _rows_of(t, cols, what, device, dtype=None):
    """Checks a CUDA matrix of `cols` columns given with any leading dimensions, and returns (address, rows, leading
    dimension) of it as one matrix; raises when its rows are not contiguous or not evenly spaced."""
    if not (_is_torch(t) and t.is_cuda):
        raise TypeError("%s must be a CUDA tensor" % what)
    if t.device != device:
        raise ValueError("%s is on %s, the weights are on %s" % (what, t.device, device))
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s is %s, expected %s" % (what, t.dtype, dtype))
    shape = t.shape
    if len(shape) == 0 or shape[-1] != cols:
        raise ValueError("%s has shape %s, expected (..., %d)" % (what, tuple(shape), cols))
    if len(shape) != 2:
        try:
            t = t.view(-1, cols)
        except RuntimeError:
            raise TypeError("%s: its leading dimensions cannot be taken as one row dimension; call .contiguous()" % what) from None
    rows = t.shape[0]
    ld, step = t.stride()
    if rows and step != 1 and cols > 1:
        raise TypeError("%s must have contiguous rows" % what)
    if rows <= 1:
        ld = cols
    if ld < cols:
        raise TypeError("%s: its rows overlap" % what)
    return t.data_ptr(), rows, ld


def _workspace(need, device):
    """(tensor to keep until the call is enqueued, its first 1024-byte aligned address) of `need` bytes of scratch.  It comes
    from torch's allocator: every call and every captured graph has its own."""
    import torch
    buf = torch.empty(need + 1024, dtype=torch.uint8, device=device)
    return buf, (buf.data_ptr() + 1023) & ~1023


def _current_stream(device):
    """The raw current stream of a CUDA device (torch's own short cut where it has one: a fourth of a small call's time)."""
    import torch
    short = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return short(device.index) if short is not None else torch.cuda.current_stream(device).cuda_stream


class _on_device:
    """Around a call on a tensor's device: makes the device current, and with an explicit ``stream`` (a raw
    cudaStream_t or a torch stream) that stream too, so that what the call allocates belongs to the stream it is
    used on.  Gives the raw stream."""

    def __init__(self, device, stream):
        import torch
        self.around = []
        raw = _current_stream(device)
        if stream is not None:
            wanted = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
            if wanted != raw:
                s = torch.cuda.ExternalStream(wanted, device=device) if wanted else torch.cuda.default_stream(device)
                self.around = [torch.cuda.stream(s)]
                raw = wanted
        if torch.cuda.current_device() != device.index:
            self.around.insert(0, torch.cuda.device(device))
        self.raw = raw

    def __enter__(self):
        for a in self.around:
            a.__enter__()
        return self.raw

    def __exit__(self, *exc):
        for a in reversed(self.around):
            a.__exit__(*exc)


class Q4Weights:
    """A linear layer's weight in 4 bits, laid out once for the products that read it (cakeb200_q4_pack):
    w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group]).

    ``codes``: uint8 CUDA tensor (out_features, ceil(in_features / 2)), two codes to a byte, the even input feature in the
    low half.  ``scales``: float16 or bfloat16, (out_features, ceil(in_features / group)).  ``zeros``: uint8 of the same shape
    with values 0..15, or None for 8 everywhere.  ``group``: 32, 64 or 128.  ``in_features`` tells an odd number of input
    features from the even one above it.  ``Q4Weights.quantize(W)`` makes all of them from a matrix.

    Given zero points are looked at once by the host, in the order of ``stream`` (which it waits for; not while it is captured)."""

    FEW_ROWS = 64  # products of up to this many rows never need a workspace

    def __init__(self, codes, scales, zeros=None, group=128, in_features=None, stream=None, _checked=False):
        import torch
        for t, what in ((codes, "codes"), (scales, "scales")) + (((zeros, "zeros"),) if zeros is not None else ()):
            if not (_is_torch(t) and t.is_cuda):
                raise TypeError("%s must be a CUDA tensor" % what)
            if t.dim() != 2 or not t.is_contiguous():
                raise TypeError("%s must be a contiguous matrix" % what)
            if t.device != codes.device:
                raise ValueError("%s is on %s, the codes are on %s" % (what, t.device, codes.device))
        if codes.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
            raise TypeError("codes and zeros are uint8")
        self.scale_type = _type_code(scales.dtype, "scales", (F16, BF16))
        self.out_features = codes.shape[0]
        self.in_features = 2 * codes.shape[1] if in_features is None else int(in_features)
        if group not in (32, 64, 128):
            raise ValueError("group is 32, 64 or 128, not %r" % (group,))
        if self.out_features < 1 or self.in_features < 1 or (self.in_features + 1) // 2 != codes.shape[1]:
            raise ValueError("codes have shape %s, which does not hold %d input features" % (tuple(codes.shape), self.in_features))
        self.group = int(group)
        groups = -(-self.in_features // self.group)
        _need_shape(scales, (self.out_features, groups), "scales")
        if zeros is not None:
            _need_shape(zeros, (self.out_features, groups), "zeros")
        self.device, self.has_zeros = codes.device, zeros is not None
        n = lib().cakeb200_q4_packed_bytes(self.out_features, self.in_features, self.group, int(zeros is not None))
        with _on_device(self.device, stream) as s:
            # looked at on the stream that they are read on: what wrote them may still be queued there
            if zeros is not None and not _checked and not torch.cuda.is_current_stream_capturing() and int(zeros.max()) > 15:
                raise ValueError("zero points are 0..15")
            self.packed = torch.empty(n, dtype=torch.uint8, device=self.device)
            self._bind()
            _check(lib().cakeb200_q4_pack(_vp(codes.data_ptr()), codes.stride(0), _vp(scales.data_ptr()),
                                          _vp(zeros.data_ptr()) if zeros is not None else None, self.out_features, self.in_features,
                                          self.group, self.scale_type, _vp(self.packed.data_ptr()), s))

    @classmethod
    def from_packed(cls, packed, out_features, in_features, group, scale_type, has_zeros):
        """The weights whose packed form (the ``packed`` tensor of another object of that geometry) is given."""
        n = lib().cakeb200_q4_packed_bytes(out_features, in_features, group, int(has_zeros))
        import torch
        if not (_is_torch(packed) and packed.is_cuda and packed.dtype == torch.uint8 and packed.is_contiguous()):
            raise TypeError("packed weights are a contiguous uint8 CUDA tensor")
        if n == 0:
            _check(-1)
        _need_shape(packed, (n,), "packed")
        self = object.__new__(cls)
        self.out_features, self.in_features, self.group, self.scale_type = int(out_features), int(in_features), int(group), int(scale_type)
        self.has_zeros, self.device, self.packed = bool(has_zeros), packed.device, packed
        self._bind()
        return self

    def _bind(self):
        self._c = _Q4(self.packed.data_ptr(), self.out_features, self.in_features, self.group, self.scale_type, int(self.has_zeros))
        self._ref = ctypes.byref(self._c)

    def __getstate__(self):
        state = dict(self.__dict__)
        del state["_c"], state["_ref"]  # the descriptor holds an address: a copy makes its own
        return state

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.device = self.packed.device
        self._bind()

    @staticmethod
    def quantize_codes(W, group=128, symmetric=True, scale_dtype=None, stream=None):
        """(codes, scales, zeros or None) of a float32, float16 or bfloat16 matrix (cakeb200_q4_quantize)."""
        import torch
        scale_dtype = torch.float16 if scale_dtype is None else scale_dtype
        if not (_is_torch(W) and W.is_cuda):
            raise TypeError("W must be a CUDA tensor")
        if W.dim() != 2 or W.shape[0] < 1 or W.shape[1] < 1:
            raise ValueError("W must be a matrix")
        if group not in (32, 64, 128):
            raise ValueError("group is 32, 64 or 128, not %r" % (group,))
        t = _type_code(W.dtype, "W")
        st = _type_code(scale_dtype, "scales", (F16, BF16))
        p, n, ld = _rows_of(W, W.shape[1], "W", W.device)
        k = W.shape[1]
        with _on_device(W.device, stream) as s:
            codes = torch.empty((n, (k + 1) // 2), dtype=torch.uint8, device=W.device)
            scales = torch.empty((n, -(-k // group)), dtype=scale_dtype, device=W.device)
            zeros = None if symmetric else torch.empty(scales.shape, dtype=torch.uint8, device=W.device)
            _check(lib().cakeb200_q4_quantize(_vp(p), ld, t, n, k, group, st, _vp(codes.data_ptr()), codes.stride(0), _vp(scales.data_ptr()),
                                              _vp(zeros.data_ptr()) if zeros is not None else None, s))
        return codes, scales, zeros

    @classmethod
    def quantize(cls, W, group=128, symmetric=True, scale_dtype=None, stream=None):
        codes, scales, zeros = cls.quantize_codes(W, group, symmetric, scale_dtype, stream)
        return cls(codes, scales, zeros, group=group, in_features=W.shape[1], stream=stream, _checked=True)  # they were allocated on `stream`

    def dequantize(self, dtype=None, out=None, stream=None):
        """The matrix (out_features, in_features) the codes stand for."""
        import torch
        t = _type_code(out.dtype if out is not None else dtype or torch.float32, "out")
        with _on_device(self.device, stream) as s:
            if out is None:
                out = torch.empty((self.out_features, self.in_features), dtype=dtype or torch.float32, device=self.device)
            _need_shape(out, (self.out_features, self.in_features), "out")
            p, _, ld = _rows_of(out, self.in_features, "out", self.device)
            _check(lib().cakeb200_q4_dequantize(self._ref, p, ld, t, s))
        return out


def _need_q4(W4):
    if not isinstance(W4, Q4Weights):
        raise TypeError("the weights must be a Q4Weights object")


def _q4_product(dx, what, src, W4, cols_in, cols_out, bias, out, stream):
    import torch
    p, rows, ld = _rows_of(src, cols_in, what, W4.device)
    t = _type_code(src.dtype, what)
    shape = src.shape[:-1] + (cols_out,)
    pb = po = ldo = None
    if bias is not None:
        pb = _rows_of(bias, cols_out, "bias", W4.device, src.dtype)[0]
        if bias.dim() != 1:
            raise ValueError("bias must be a vector")
    if out is not None:
        _need_shape(out, shape, "out")
        po, _, ldo = _rows_of(out, cols_out, "out", W4.device, src.dtype)

    def run(s):
        nonlocal out, po, ldo
        if out is None:
            out = src.new_empty(shape)
            po, ldo = out.data_ptr(), cols_out
        buf = ws = None
        need = 0
        if rows > W4.FEW_ROWS:
            need = lib().cakeb200_q4_workspace(W4._ref, rows, t, int(dx))
            if need:
                buf, ws = _workspace(need, W4.device)
        if dx:
            _check(lib().cakeb200_q4_linear_dx(W4._ref, p, ld, po, ldo, rows, t, ws, need, s))
        else:
            _check(lib().cakeb200_q4_linear(W4._ref, p, ld, pb, po, ldo, rows, t, ws, need, s))
        return out

    if stream is None and torch.cuda.current_device() == W4.device.index:
        return run(_current_stream(W4.device))
    with _on_device(W4.device, stream) as s:
        return run(s)


def cake_q4_linear(x, W4, bias=None, out=None, stream=None):
    """x @ W.T (+ bias) with W a ``Q4Weights`` (cakeb200_q4_linear), enqueued on the current stream.  x: CUDA tensor
    (..., in_features) in float32, float16 or bfloat16 with contiguous, evenly spaced rows; bias and result have its type."""
    _need_q4(W4)
    return _q4_product(False, "x", x, W4, W4.in_features, W4.out_features, bias, out, stream)


def cake_q4_linear_dx(dy, W4, out=None, stream=None):
    """dy @ W with W a ``Q4Weights`` (cakeb200_q4_linear_dx): the gradient of ``cake_q4_linear`` for its input."""
    _need_q4(W4)
    return _q4_product(True, "dy", dy, W4, W4.out_features, W4.in_features, None, out, stream)


# --------------------------------------------------------- orthogonalised updates

NS_COEFFS = (3.4445, -4.7750, 2.0315)


def _matrix_of(t, what, device=None, shape=None):
    """Checks a CUDA matrix with contiguous rows; returns (address, leading dimension)."""
    if not (_is_torch(t) and t.is_cuda):
        raise TypeError("%s must be a CUDA tensor" % what)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (what, t.device, device))
    if shape is not None:
        _need_shape(t, shape, what)
    rows, cols = t.shape[-2:]
    if rows < 1 or cols < 1:
        raise ValueError("%s has an empty side" % what)
    if cols > 1 and t.stride(-1) != 1:
        raise TypeError("%s must have contiguous rows" % what)
    ld = t.stride(-2) if rows > 1 else cols
    if ld < cols:
        raise TypeError("%s: its rows overlap" % what)
    return t.data_ptr(), ld


def _ns_workspace(rows, cols, batch, t, device):
    """(tensor to keep until the call is enqueued, aligned address, bytes) of the products' scratch planes."""
    need = lib().cakeb200_orthogonalize_workspace(rows, cols, batch, t)
    if need == 0:
        _check(-1)
    return _workspace(need, device) + (need,)


def cake_orthogonalize(G, out=None, steps=5, coeffs=NS_COEFFS, eps=1e-7, stream=None):
    """The orthogonalisation of a matrix, or of every matrix of a batch, by Newton-Schulz products (cakeb200_orthogonalize),
    enqueued on the current stream: X = G / (|G|_F + eps), then ``steps`` times X <- a X + b (X X^T) X + c (X X^T)^2 X.

    G: CUDA tensor (rows, cols) or (batch, rows, cols), float32 or bfloat16, rows contiguous.  ``out`` may be G
    or overlap it."""
    import torch
    if not (_is_torch(G) and G.is_cuda):
        raise TypeError("G must be a CUDA tensor")
    if G.dim() not in (2, 3):
        raise ValueError("G must be a matrix or a batch of matrices")
    t = _type_code(G.dtype, "G", (F32, BF16))
    a, b, c = (float(v) for v in coeffs)
    batch = G.shape[0] if G.dim() == 3 else 1
    rows, cols = G.shape[-2:]
    p, ld = _matrix_of(G, "G")
    if out is not None:
        po, ldo = _matrix_of(out, "out", G.device, G.shape)
        if out.dtype != G.dtype:
            raise TypeError("out is %s, expected %s" % (out.dtype, G.dtype))
    with _on_device(G.device, stream) as s:
        if out is None:
            out = torch.empty(G.shape, dtype=G.dtype, device=G.device)
            po, ldo = out.data_ptr(), cols
        if batch == 0:
            return out
        stride = lambda m: m.stride(0) if m.dim() == 3 else 0
        buf, ws, n = _ns_workspace(rows, cols, batch, t, G.device)
        _check(lib().cakeb200_orthogonalize(p, ld, stride(G), po, ldo, stride(out), rows, cols, batch, t, int(steps), a, b, c, float(eps), ws, n, s))
    return out


def cake_muon_step(W, G, M, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5, coeffs=NS_COEFFS, eps=1e-7, stream=None):
    """One step of an optimiser with orthogonalised updates on the matrix W, in place (cakeb200_muon_step):
    M <- momentum M + (1 - momentum) G;  U = momentum M + (1 - momentum) G, or M without ``nesterov``;
    W <- (1 - lr weight_decay) W - lr scale O(U).  ``scale`` defaults to sqrt(max(1, rows / cols)).

    W and G: float32 or bfloat16 CUDA matrices with contiguous rows, M: the same in float32, in memory of its own.  Returns W."""
    if not (_is_torch(W) and W.is_cuda):
        raise TypeError("W must be a CUDA tensor")
    if W.dim() != 2:
        raise ValueError("W must be a matrix")
    tw, tg = _type_code(W.dtype, "W", (F32, BF16)), _type_code(G.dtype if _is_torch(G) else None, "G", (F32, BF16))
    _type_code(M.dtype if _is_torch(M) else None, "M", (F32,))
    rows, cols = W.shape
    (pw, ldw), (pg, ldg), (pm, ldm) = _matrix_of(W, "W"), _matrix_of(G, "G", W.device, W.shape), _matrix_of(M, "M", W.device, W.shape)
    a, b, c = (float(v) for v in coeffs)
    if scale is None:
        scale = max(1.0, rows / cols) ** 0.5
    with _on_device(W.device, stream) as s:
        buf, ws, n = _ns_workspace(rows, cols, 1, tw, W.device)
        _check(lib().cakeb200_muon_step(pw, ldw, tw, pg, ldg, tg, pm, ldm, rows, cols, float(lr), float(momentum), int(bool(nesterov)),
                                        float(weight_decay), float(scale), int(steps), a, b, c, float(eps), ws, n, s))
    return W


def tune(A, B, C=None, sch=NA, trials=24, stream=None):
    """Search the tile shape of the large-matrix kernel for this product's shape on the device and
    remember the winner (cakeb200_tune).  Returns the winning entry as a dict."""
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if C is None:
        C = _empty_like_kind(A, (M, N))
    _need_shape(C, (M, N), "C")
    _check(lib().cakeb200_tune(_ptr(A), _ptr(B), _ptr(C), M, N, K, sch, trials, _stream_of(C, stream)))
    st = last_stats()
    return dict(tune_get(M, N, K, st["sched"]), evaluated=st["launches"])


def tune_search(M, N, K, cost, sm_count=148, trials=24, seed=1):
    """The search alone with a Python cost function cost(tile_n, band, k_pieces) -> ms (<= 0: invalid point)."""
    cb = TUNE_COST(lambda w, b, p, _user: float(cost(w, b, p)))
    w, b, p, n, ms = _i(), _i(), _i(), _i(), ctypes.c_float()
    _check(lib().cakeb200_tune_search(M, N, K, sm_count, trials, seed, cb, None, ctypes.byref(w), ctypes.byref(b), ctypes.byref(p),
                                      ctypes.byref(ms), ctypes.byref(n)))
    return {"tile_n": w.value, "band": b.value, "k_pieces": p.value, "ms": ms.value, "evaluated": n.value}


def tune_search_shape(M, N, K, cost, sm_count=148, trials=24, seed=1):
    """The search over tile width, cluster shape, band and K pieces with a Python cost function
    cost(tile_n, cluster, band, k_pieces) -> ms (<= 0: invalid point); cluster 1 = pairs of SMs, 2 = single SMs."""
    cb = TUNE_COST_SHAPE(lambda w, c, b, p, _user: float(cost(w, c, b, p)))
    w, c, b, p, n, ms = _i(), _i(), _i(), _i(), _i(), ctypes.c_float()
    _check(lib().cakeb200_tune_search_shape(M, N, K, sm_count, trials, seed, cb, None, ctypes.byref(w), ctypes.byref(c), ctypes.byref(b),
                                            ctypes.byref(p), ctypes.byref(ms), ctypes.byref(n)))
    return {"tile_n": w.value, "cluster": c.value, "band": b.value, "k_pieces": p.value, "ms": ms.value, "evaluated": n.value}


def tune_put(M, N, K, sch, tile_n, band, k_pieces, ms=0.0, cluster=0):
    """Record a choice for a shape; ``cluster`` 0 = the rule, 1 = pairs of SMs, 2 = single SMs."""
    _check(lib().cakeb200_tune_put_shape(M, N, K, sch, tile_n, cluster, band, k_pieces, ms))


def tune_get(M, N, K, sch):
    w, c, b, p, ms = _i(), _i(), _i(), _i(), ctypes.c_float()
    if not lib().cakeb200_tune_get_shape(M, N, K, sch, ctypes.byref(w), ctypes.byref(c), ctypes.byref(b), ctypes.byref(p), ctypes.byref(ms)):
        return None
    return {"tile_n": w.value, "cluster": c.value, "band": b.value, "k_pieces": p.value, "ms": ms.value}


def tune_clear():
    _check(lib().cakeb200_tune_clear())


def tune_save(path):
    n = lib().cakeb200_tune_save(str(path).encode())
    if n < 0:
        _check(n)
    return n


def tune_load(path):
    n = lib().cakeb200_tune_load(str(path).encode())
    if n < 0:
        _check(n)
    return n


def set_option(name, value):
    """Override one choice of the large-matrix kernel (cakeb200_set_option); 0 restores the rule."""
    _check(lib().cakeb200_set_option(name.encode(), int(value)))


def get_option(name):
    return lib().cakeb200_get_option(name.encode())


def profile_begin():
    """Start device-side timing of the asynchronous products that follow (see cakeb200_profile_begin)."""
    _check(lib().cakeb200_profile_begin())


def profile_end():
    """(ms_prepass, ms_kernel, calls) summed over the products since profile_begin()."""
    pre, ker, n = ctypes.c_float(), ctypes.c_float(), ctypes.c_int()
    _check(lib().cakeb200_profile_end(ctypes.byref(pre), ctypes.byref(ker), ctypes.byref(n)))
    return pre.value, ker.value, n.value
