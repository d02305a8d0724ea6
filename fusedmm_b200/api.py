"""Python mirror of the C ABI in ``include/fusedmm_b200.h`` (ctypes; no torch types cross the boundary).

:func:`fusedMM_csr` has the reference's argument list (HipGraph/FusedMM ``fusedMM.h:76-97``) and return
codes.  Arrays may be NumPy arrays (host memory: the library stages them to the GPU and copies Z back) or
torch tensors (CPU or CUDA; CUDA tensors are used in place).  The typed symbol
(``sfusedMM_csr_i32`` ... ``dfusedMM_csr_p64i32``) is picked from the arrays' dtypes, which is what the
reference does at compile time with its VALUETYPE / INDEXTYPE macros.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

import numpy as np

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libfusedmm_b200.so"
_lib = None


class FusedMMError(RuntimeError):
    pass


class SopSpec(C.Structure):
    """``fusedmm_b200_sop`` of include/fusedmm_b200.h."""
    _fields_ = [("kind", C.c_int32), ("reserved", C.c_int32), ("p0", C.c_double), ("p1", C.c_double),
                ("p2", C.c_double)]


class CallInfo(C.Structure):
    """``fusedmm_b200_call_info`` of include/fusedmm_b200.h."""
    _fields_ = [("kernel_launches", C.c_int32), ("pattern", C.c_int32), ("lanes_per_edge", C.c_int32),
                ("vectors_per_lane", C.c_int32), ("h2d_bytes", C.c_int64), ("d2h_bytes", C.c_int64),
                ("hub_rows", C.c_int64), ("hub_chunks", C.c_int64), ("device_ms", C.c_float),
                ("sop_kind", C.c_int32), ("ms_scan", C.c_float), ("ms_rows", C.c_float),
                ("ms_chunks", C.c_float), ("ms_fixup", C.c_float), ("engine", C.c_int32), ("ms_main", C.c_float),
                ("jit_kernel", C.c_int32)]


def lib() -> C.CDLL:
    """Loads ``libfusedmm_b200.so``.  Raises if it is not built: there is no other implementation."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise FusedMMError(f"{LIB_PATH} is missing: build it with `python -m fusedmm_b200.build` "
                               "(nvcc, sm_100a). There is no CPU or PyTorch fallback.")
        _lib = C.CDLL(str(LIB_PATH))
        _lib.fusedmm_b200_status_string.restype = C.c_char_p
        _lib.fusedmm_b200_version.restype = C.c_char_p
        _lib.fusedmm_b200_set_sop.argtypes = [C.c_int32, C.c_double, C.c_double, C.c_double]
        _lib.fusedmm_b200_set_option.argtypes = [C.c_char_p, C.c_int64]
        _lib.fusedmm_b200_get_option.argtypes = [C.c_char_p, C.POINTER(C.c_int64)]
        _lib.fusedmm_b200_last_call_info.argtypes = [C.POINTER(CallInfo)]
        _lib.fusedmm_b200_csr.restype = C.c_int
        _lib.fusedmm_b200_csr.argtypes = (
            [C.c_int32] * 4 + [C.c_int64] * 3 + [C.c_double] + [C.c_int64] * 3 + [C.c_void_p] * 5 +
            [C.c_int64, C.c_void_p, C.c_int64, C.c_double, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p])
    return _lib


def status_string(status: int) -> str:
    return lib().fusedmm_b200_status_string(int(status)).decode()


def set_sop(kind: int, p0: float = 0.0, p1: float = 0.0, p2: float = 0.0) -> int:
    """Process-wide meaning of SOP_UDEF (``fusedmm_b200_set_sop``)."""
    return lib().fusedmm_b200_set_sop(kind, p0, p1, p2)


def set_option(name: str, value: int) -> int:
    return lib().fusedmm_b200_set_option(name.encode(), int(value))


def get_option(name: str) -> int:
    v = C.c_int64(0)
    st = lib().fusedmm_b200_get_option(name.encode(), C.byref(v))
    if st:
        raise FusedMMError(f"unknown option {name!r}")
    return v.value


def jit_prepare(imessage: int, k: int, dtype=np.float32) -> int:
    """``fusedmm_b200_jit_prepare``: build the kernel specialised for a message ahead of its first call."""
    fn = lib().fusedmm_b200_jit_prepare
    fn.argtypes = [C.c_int32, C.c_int32, C.c_int64]
    return fn(0 if np.dtype(dtype) == np.float32 else 1, int(imessage), int(k))


def jit_stats() -> dict:
    out = (C.c_int64 * 5)()
    lib().fusedmm_b200_jit_stats(out)
    return dict(zip(("compiled", "disk_hits", "launches", "failures", "nvrtc_found"), (int(v) for v in out)))


def call_info() -> CallInfo:
    """What the most recent call on this thread did (``fusedmm_b200_last_call_info``)."""
    info = CallInfo()
    lib().fusedmm_b200_last_call_info(C.byref(info))
    return info


_NP = {"float32": np.float32, "float64": np.float64, "int32": np.int32, "int64": np.int64}


def _describe(a):
    """-> (address, numpy dtype) of a NumPy array, a torch tensor or None."""
    if a is None:
        return None, None
    if isinstance(a, np.ndarray):
        if not a.flags["C_CONTIGUOUS"]:
            raise ValueError("arrays must be C-contiguous; use ldx/ldy/ldz for padded rows")
        return a.ctypes.data, a.dtype
    if hasattr(a, "data_ptr"):  # torch tensor, without importing torch here
        if not a.is_contiguous():
            raise ValueError("tensors must be contiguous; use ldx/ldy/ldz for padded rows")
        return a.data_ptr(), np.dtype(_NP[str(a.dtype).replace("torch.", "")])
    raise TypeError(f"unsupported array type {type(a)!r}")


def _symbol(vt, pt, it):
    pre = {np.dtype(np.float32): "s", np.dtype(np.float64): "d"}.get(np.dtype(vt))
    if pre is None:
        raise TypeError("values must be float32 or float64")
    pb, ib = np.dtype(pt).itemsize * 8, np.dtype(it).itemsize * 8
    if np.dtype(pt).kind != "i" or np.dtype(it).kind != "i" or pb not in (32, 64) or ib not in (32, 64):
        raise TypeError("indices must be int32 or int64")
    if pb == ib:
        return pre, f"i{pb}", pb
    if (pb, ib) == (64, 32):
        return pre, "p64i32", 64
    raise TypeError("32-bit row pointers with 64-bit column ids are not supported")


def fusedMM_csr(imessage, m, n, k, alpha, nnz, rows, cols, val, indx, pntrb, pntre, x, ldx, y, ldy, beta,
                z, ldz, sop=None, stream=None, z_peers=None, z_multicast=None):
    """``fusedMM_csr`` with the reference's argument order and return codes.

    ``sop``: ``None`` (process default, see :func:`set_sop`), an ``int`` kind, or ``(kind, p0, p1, p2)``.
    ``stream``: ``None`` for a synchronous call, or a CUDA stream handle (``int``) to enqueue on; every
    array must then be on the device.  With ``sop`` and ``stream`` both ``None`` the call goes through
    the typed symbol (``sfusedMM_csr_i64`` ...), otherwise through ``fusedmm_b200_csr``.
    ``z_peers``: device addresses (``int``) of other GPUs' Z buffers at this call's first row; finished
    rows are then also stored there (``fusedmm_b200_csr_multi``); ``z_multicast``: instead, the NVSwitch
    multicast address of Z at this call's first row (one ``multimem.st`` per row reaches every GPU).
    """
    L = lib()
    ptrs, dts = zip(*[_describe(a) for a in (val, indx, pntrb, pntre, x, y, z)])
    vt = dts[6]
    for d in (dts[0], dts[4], dts[5]):
        if d is not None and d != vt:
            raise TypeError("val, x, y and z must share one floating-point type")
    if dts[3] != dts[2]:
        raise TypeError("pntrb and pntre must share one integer type")
    pre, suffix, size_bits = _symbol(vt, dts[2], dts[1] if dts[1] is not None else dts[2])
    if sop is None and stream is None and not z_peers and not z_multicast:
        VT = C.c_float if pre == "s" else C.c_double
        IT = C.c_int32 if size_bits == 32 else C.c_int64
        fn = getattr(L, f"{pre}fusedMM_csr_{suffix}")
        fn.restype = C.c_int
        fn.argtypes = ([C.c_int32, IT, IT, IT, VT, IT, IT, IT] + [C.c_void_p] * 4 +
                       [C.c_void_p, IT, C.c_void_p, IT, VT, C.c_void_p, IT])
        return fn(imessage, m, n, k, alpha, nnz, rows, cols, ptrs[0], ptrs[1], ptrs[2], ptrs[3], ptrs[4],
                  ldx, ptrs[5], ldy, beta, ptrs[6], ldz)
    spec = None
    if sop is not None:
        kind, *params = (sop,) if isinstance(sop, int) else tuple(sop)
        params = list(params) + [0.0] * (3 - len(params))
        spec = C.byref(SopSpec(int(kind), 0, *map(float, params)))
    pb = np.dtype(dts[2]).itemsize * 8
    ib = np.dtype(dts[1]).itemsize * 8 if dts[1] is not None else pb
    if z_peers or z_multicast:
        z_peers = list(z_peers or [])
        arr = (C.c_void_p * max(1, len(z_peers)))(*[int(q) for q in z_peers])
        fn = L.fusedmm_b200_csr_multi
        fn.restype = C.c_int
        fn.argtypes = list(L.fusedmm_b200_csr.argtypes) + [C.c_int32, C.c_void_p, C.c_void_p]
        return fn(0 if pre == "s" else 1, pb, ib, imessage, m, n, k, alpha, nnz, rows, cols, ptrs[0], ptrs[1],
                  ptrs[2], ptrs[3], ptrs[4], ldx, ptrs[5], ldy, beta, ptrs[6], ldz, spec, stream, len(z_peers), arr,
                  int(z_multicast) if z_multicast else None)
    return L.fusedmm_b200_csr(0 if pre == "s" else 1, pb, ib, imessage, m, n, k, alpha, nnz, rows, cols,
                              ptrs[0], ptrs[1], ptrs[2], ptrs[3], ptrs[4], ldx, ptrs[5], ldy, beta, ptrs[6],
                              ldz, spec, stream)


def gfusedMM_csr(tkern, m, n, k, alpha, nnz, rows, cols, val, indx, pntrb, pntre, a, lda, b, ldb, beta, c,
                 ldc):
    """``sgfusedMM_csr`` / ``dgfusedMM_csr`` (kernels/include/kernels.h:17-37): dispatch by kernel letter."""
    L = lib()
    ptrs, dts = zip(*[_describe(t) for t in (val, indx, pntrb, pntre, a, b, c)])
    pre, suffix, size_bits = _symbol(dts[6], dts[2], dts[1] if dts[1] is not None else dts[2])
    if suffix == "p64i32":
        raise TypeError("the letter dispatcher has a single INDEXTYPE")
    VT = C.c_float if pre == "s" else C.c_double
    IT = C.c_int32 if size_bits == 32 else C.c_int64
    fn = getattr(L, f"{pre}gfusedMM_csr_{suffix}")
    fn.restype = None
    fn.argtypes = ([C.c_char, IT, IT, IT, VT, IT, IT, IT] + [C.c_void_p] * 4 +
                   [C.c_void_p, IT, C.c_void_p, IT, VT, C.c_void_p, IT])
    fn(tkern.encode() if isinstance(tkern, str) else tkern, m, n, k, alpha, nnz, rows, cols, ptrs[0],
       ptrs[1], ptrs[2], ptrs[3], ptrs[4], lda, ptrs[5], ldb, beta, ptrs[6], ldc)


def zero_empty_rows(pntrb, pntre, z, k, ldz, stream=None):
    """``fusedmm_b200_zero_empty_rows``: Z_u = 0 for the rows without edges among the ``len(pntrb)`` rows that
    ``pntrb``/``pntre``/``z`` start at (device tensors); returns the status code."""
    L = lib()
    ptrs, dts = zip(*[_describe(a) for a in (pntrb, pntre, z)])
    if dts[0] != dts[1]:
        raise TypeError("pntrb and pntre must share one integer type")
    fn = L.fusedmm_b200_zero_empty_rows
    fn.restype = C.c_int
    fn.argtypes = [C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    return fn(0 if np.dtype(dts[2]) == np.float32 else 1, np.dtype(dts[0]).itemsize * 8, len(pntrb), k, ptrs[0], ptrs[1],
              ptrs[2], ldz, stream)


def shard_rows(pntrb, pntre, nshards, row_weight=0):
    """Contiguous row ranges of equal cost, a row costing its edges plus ``row_weight``
    (``fusedmm_b200_shard_rows_weighted_*``; 0 = balanced by edges alone); host NumPy row pointers."""
    L = lib()
    pntrb = np.ascontiguousarray(pntrb)
    pntre = np.ascontiguousarray(pntre)
    m = len(pntrb)
    bounds = np.zeros(nshards + 1, dtype=np.int64)
    fn = L.fusedmm_b200_shard_rows_weighted_i32 if pntrb.dtype == np.int32 else L.fusedmm_b200_shard_rows_weighted_i64
    fn.argtypes = [C.c_int64, C.c_int32, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    st = fn(m, nshards, pntrb.ctypes.data, pntre.ctypes.data, int(row_weight), bounds.ctypes.data)
    if st:
        raise FusedMMError(status_string(st))
    return bounds


class Plan:
    """``fusedmm_b200_plan_*``: the CSR kept on the device together with its split-row list, for many calls over
    one graph.  ``indx``, ``pntrb``, ``pntre`` (and optionally ``val``) are NumPy arrays or torch tensors; device
    tensors are borrowed and must outlive the plan."""

    def __init__(self, indx, pntrb, pntre, val=None):
        L = lib()
        ptrs, dts = zip(*[_describe(a) for a in (val, indx, pntrb, pntre)])
        self._keep = (val, indx, pntrb, pntre)
        self.m = len(pntrb)
        pb, ib = np.dtype(dts[2]).itemsize * 8, np.dtype(dts[1]).itemsize * 8
        vd = -1 if val is None else (0 if np.dtype(dts[0]) == np.float32 else 1)
        self._h = C.c_void_p()
        fn = L.fusedmm_b200_plan_create
        fn.restype = C.c_int
        fn.argtypes = [C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32,
                       C.c_void_p, C.POINTER(C.c_void_p)]
        st = fn(pb, ib, self.m, 0, ptrs[1], ptrs[2], ptrs[3], vd, ptrs[0], C.byref(self._h))
        if st:
            raise FusedMMError(status_string(st))

    def csr(self, imessage, n, k, x, ldx, y, ldy, beta, z, ldz, sop=None, stream=None):
        """``fusedmm_b200_plan_csr``: the call without the CSR arguments; returns the status code."""
        L = lib()
        ptrs, dts = zip(*[_describe(a) for a in (x, y, z)])
        dtype = 0 if np.dtype(dts[2]) == np.float32 else 1
        spec = None
        if sop is not None:
            kind, *params = (sop,) if isinstance(sop, int) else tuple(sop)
            params = list(params) + [0.0] * (3 - len(params))
            spec = C.byref(SopSpec(int(kind), 0, *map(float, params)))
        fn = L.fusedmm_b200_plan_csr
        fn.restype = C.c_int
        fn.argtypes = [C.c_void_p, C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_void_p, C.c_int64, C.c_void_p,
                       C.c_int64, C.c_double, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        return fn(self._h, dtype, imessage, n, k, ptrs[0], ldx, ptrs[1], ldy, beta, ptrs[2], ldz, spec, stream)

    def close(self):
        if self._h:
            lib().fusedmm_b200_plan_destroy.argtypes = [C.c_void_p]
            lib().fusedmm_b200_plan_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- attention over the edges of a CSR (torch CUDA tensors only; see include/fusedmm_b200.h) ---------------------------
LEGACY_STREAM = 1  # cudaStreamLegacy: enqueues on the default stream, where NULL would also wait for it
_attn_fns = {}


def _attn_fn(name, restype, *argtypes):
    fn = _attn_fns.get(name)
    if fn is None:
        fn = getattr(lib(), "fusedmm_b200_" + name)
        fn.restype, fn.argtypes = restype, list(argtypes)
        _attn_fns[name] = fn
    return fn


_i, _l, _p, _d = C.c_int32, C.c_int64, C.c_void_p, C.c_double
_ROTARY_IN = (_i, _l, _i, _i, _i, _p, _l, _l, _p, _l, _l, _i, _p, _p, _i, _d, _i, _p, _l, _l, _i, _p, _i, _i)
_ATTN_IN = (_i, _i, _i, _l, _l, _l, _p, _p, _p, _i, _i, _i, _i, _p, _l, _l, _p, _l, _l, _p, _l, _l, _p, _l, _d)


class _Codes(dict):
    """torch dtype -> code of the C ABI or None; filled by the dtypes' names, so that this module needs no torch."""

    def __init__(self, **names):
        super().__init__()
        self._names = names

    def __missing__(self, dtype):
        code = self[dtype] = self._names.get(str(dtype)[6:])
        return code


_DT = _Codes(float32=0, bfloat16=2, float16=3)
_POS = _Codes(int32=0, int64=1, float32=2, float64=3)
_BITS = _Codes(int32=32, int64=64)
_F32 = _Codes(float32=0)
_F64 = _Codes(float64=0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _require(ok, text):
    if not ok:
        raise ValueError(text)


def _rows(t, name):
    """Strides (rows, heads) of a tensor whose axes behind the heads are dense."""
    shape, stride = t.shape, t.stride()
    dense = 1
    for i in range(len(shape) - 1, 1, -1):
        if stride[i] != dense and shape[i] > 1:
            raise ValueError(f"{name}: the axes behind the heads must be dense")
        dense *= shape[i]
    # the stride of an axis of one entry is never used; one that breaks no alignment stands for it
    return (stride[0] if shape[0] > 1 else dense * shape[1]), (stride[1] if shape[1] > 1 else dense)


def _same_place(names, *tensors):
    dev = tensors[0].device
    for name, t in zip(names.split(), tensors):
        if t is not None and (t.device != dev or not t.is_cuda):
            _require(t.is_cuda, f"{name} must be a CUDA tensor")
            _require(False, f"{name} is on {t.device}, the first tensor on {dev}")


def rotary_args(q, k, q_weight, k_weight, pos, freq, eps, interleaved):
    """Checks the arguments of the norm and rotation (ValueError) and lays out what both directions pass to the C ABI."""
    dtype = _DT[q.dtype]
    _require(dtype is not None, "q must be float32, bfloat16 or float16")
    _require(q.dim() == 3, "q must be [rows, heads, d]")
    rows, hq, d = q.shape
    hk = ldk = hsk = 0
    if k is not None:
        _require(k.dtype == q.dtype, "q and k must share one type")
        _require(k.dim() == 3 and k.shape[0] == rows and k.shape[2] == d, "k must be [rows, heads, d] with the rows and d of q")
        hk = k.shape[1]
    _require(1 <= d <= 256, "d must be between 1 and 256")
    _require((pos is None) == (freq is None), "pos and freq come together")
    wt = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        _require(eps is not None, f"{name} without eps: no norm is asked for")
        _require(w.dim() == 1 and w.shape[0] == d and (d == 1 or w.stride(0) == 1), f"{name} must be dense, of d entries")
        _require(w.dtype == q.dtype or _F32[w.dtype] is not None, f"{name} must be float32 or of the type of q")
        _require(wt is None or wt == w.dtype, "q_weight and k_weight must share one type")
        wt = w.dtype
    _require(k_weight is None or k is not None, "k_weight without k")
    _require(eps is None or eps >= 0, "eps must not be negative")
    pt = ldp = asp = axes = pairs = 0
    if pos is not None:
        pt = _POS[pos.dtype]
        _require(pt is not None, "pos must be int32, int64, float32 or float64")
        flat = pos.dim() == 1
        _require(pos.dim() in (1, 2) and pos.shape[0] == rows, "pos must be [rows] or [rows, axes]")
        axes = 1 if flat else pos.shape[1]
        _require(1 <= axes <= 4, "there must be one to four axes")
        _require(_F64[freq.dtype] is not None, "freq must be float64 (angles of far positions need its digits)")
        _require(freq.dim() in (1, 2) and (1 if freq.dim() == 1 else freq.shape[0]) == axes and freq.is_contiguous(),
                 "freq must be dense [axes, pairs], or [pairs] with one axis")
        pairs = freq.shape[-1]
        _require(2 * pairs <= d, "freq has more pairs than half of d")
        ldp, asp = pos.stride(0), 0 if flat else pos.stride(1)
    ldq, hsq = _rows(q, "q")
    if k is not None:
        ldk, hsk = _rows(k, "k")
    _same_place("q k q_weight k_weight pos freq", q, k, q_weight, k_weight, pos, freq)
    return (dtype, rows, hq, hk, d, q.data_ptr(), ldq, hsq, _ptr(k), ldk, hsk, 0 if wt is None else _DT[wt], _ptr(q_weight),
            _ptr(k_weight), 0 if eps is None else 1, 0.0 if eps is None else float(eps), pt, _ptr(pos), ldp, asp, axes, _ptr(freq),
            pairs, 1 if interleaved else 0)


def qk_norm_rotary(args, q_out, k_out, stream=LEGACY_STREAM):
    """``fusedmm_b200_qk_norm_rotary`` with what :func:`rotary_args` laid out, on the current device; returns the status code."""
    return _attn_fn("qk_norm_rotary", C.c_int, *_ROTARY_IN, _p, _p, _p)(*args, _ptr(q_out), _ptr(k_out), stream)


def qk_norm_rotary_backward_workspace(rows, d):
    return _attn_fn("qk_norm_rotary_backward_workspace", _l, _l, _i)(rows, d)


def qk_norm_rotary_backward(args, q, k, dq_out, dk_out, dq, dk, dwq, dwk, workspace, stream=LEGACY_STREAM):
    """``fusedmm_b200_qk_norm_rotary_backward`` likewise; ``dq_out``, ``dk_out`` are the gradients of its results."""
    _require(dq_out.shape == q.shape and dq_out.dtype == q.dtype, "the gradient of q's result must have its shape and type")
    _require(k is None or (dk_out.shape == k.shape and dk_out.dtype == k.dtype), "the gradient of k's result must have its shape and type")
    _same_place("q dq_out dk_out", q, dq_out, dk_out)
    lddq, hsdq = _rows(dq_out, "the gradient of q's result")
    lddk, hsdk = _rows(dk_out, "the gradient of k's result") if k is not None else (0, 0)
    fn = _attn_fn("qk_norm_rotary_backward", C.c_int, *_ROTARY_IN, _p, _l, _l, _p, _l, _l, _p, _p, _p, _p, _p, _l, _p)
    return fn(*args, _ptr(dq_out), lddq, hsdq, _ptr(dk_out) if k is not None else None, lddk, hsdk, _ptr(dq), _ptr(dk), _ptr(dwq),
              _ptr(dwk), _ptr(workspace), 0 if workspace is None else workspace.nbytes, stream)


def _pattern_bits(rowptr, colidx):
    pb, ib = _BITS[rowptr.dtype], _BITS[colidx.dtype]
    _require(pb is not None, "rowptr must be int32 or int64")
    _require(ib is not None, "colidx must be int32 or int64")
    _require(rowptr.dim() == 1 and rowptr.is_contiguous(), "rowptr must be a dense vector")
    _require(colidx.dim() == 1 and colidx.is_contiguous(), "colidx must be a dense vector")
    _require(rowptr.shape[0] >= 1, "rowptr must have rows + 1 entries")
    return pb, ib


def attention_args(rowptr, colidx, bias, q, k, v, lam, scale):
    """Checks the arguments of differential attention (ValueError) and lays out what both directions pass to the C ABI."""
    pb, ib = _pattern_bits(rowptr, colidx)
    dtype = _DT[q.dtype]
    _require(dtype is not None, "q must be float32, bfloat16 or float16")
    _require(k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must share one type")
    _require(q.dim() == 4 and q.shape[2] == 2, "q must be [rows, heads, 2, d]")
    m, heads, _, d = q.shape
    _require(rowptr.shape[0] == m + 1, "rowptr must have one entry more than q has rows")
    _require(k.dim() == 4 and k.shape[2] == 2 and k.shape[3] == d, "k must be [columns, kv_heads, 2, d] with the d of q")
    n, kv_heads = k.shape[0], k.shape[1]
    _require(v.dim() == 3 and v.shape[0] == n and v.shape[1] == kv_heads, "v must be [columns, kv_heads, dv]")
    dv = v.shape[2]
    _require(heads >= 1 and kv_heads >= 1 and heads % kv_heads == 0, "the heads of q must be a multiple of the heads of k")
    _require(1 <= d <= 128 and 1 <= dv <= 256, "d must be between 1 and 128, dv between 1 and 256")
    _require(_F32[lam.dtype] is not None, "lam must be float32")
    if lam.dim() == 1:
        _require(lam.shape[0] == heads and (heads == 1 or lam.stride(0) == 1), "lam must be dense [heads], or [rows, heads]")
        ldlam = 0
    else:
        _require(lam.dim() == 2 and lam.shape[0] == m and lam.shape[1] == heads and (heads == 1 or lam.stride(1) == 1) and
                 (m <= 1 or lam.stride(0) >= heads), "lam must be [heads], or [rows, heads] with dense rows")
        ldlam = lam.stride(0) if m > 1 else heads
    nnz = colidx.shape[0]
    if bias is not None:
        _require(_F32[bias.dtype] is not None and bias.dim() == 1 and bias.is_contiguous() and bias.shape[0] == nnz,
                 "bias must be dense float32 with an entry for each edge")
    ldq, hsq = _rows(q, "q")
    ldk, hsk = _rows(k, "k")
    ldv, hsv = _rows(v, "v")
    _same_place("rowptr colidx bias q k v lam", rowptr, colidx, bias, q, k, v, lam)
    return (dtype, pb, ib, m, n, nnz, rowptr.data_ptr(), colidx.data_ptr(), _ptr(bias), heads, kv_heads, d, dv, q.data_ptr(), ldq, hsq,
            k.data_ptr(), ldk, hsk, v.data_ptr(), ldv, hsv, lam.data_ptr(), ldlam, float(scale))


def diff_attention_workspace(backward, args, *more):
    """Bytes of workspace (``fusedmm_b200_diff_attention_workspace``) of a call with these arguments; ``more``: addresses, and
    strides in elements, of the arrays that come with them (``dout``'s; results of torch are aligned)."""
    fn = _attn_fn("diff_attention_workspace", _l, _i, _i, _i, _l, _l, _l, _i, _i, _i, _i)
    elt = 4 if args[0] == 0 else 2
    # addresses and strides of q, k and v, all in bytes: one multiple of 16 where all are
    bits = args[13] | args[16] | args[19] | (args[14] | args[15] | args[17] | args[18] | args[20] | args[21]) * elt
    if more:
        bits |= more[0] | (more[1] | more[2]) * elt
    return fn(int(backward), int(bits & 15 == 0), args[0], args[3], args[4], args[5], args[9], args[10], args[11], args[12])


def diff_attention(args, out, lse, workspace, stream=LEGACY_STREAM):
    """``fusedmm_b200_diff_attention`` with what :func:`attention_args` laid out, on the current device; returns the status code."""
    fn = _attn_fn("diff_attention", C.c_int, *_ATTN_IN, _p, _p, _p, _l, _p)
    return fn(*args, _ptr(out), _ptr(lse), _ptr(workspace), workspace.nbytes, stream)


def diff_attention_backward(args, q, k, v, lse, dout, transposed, dq, dk, dv, dlam, workspace, stream=LEGACY_STREAM):
    """``fusedmm_b200_diff_attention_backward`` likewise; ``transposed``: what :func:`csr_transpose` wrote."""
    t_rowptr, t_row, t_edge = transposed
    _require(dout.dim() == 3 and dout.shape[0] == q.shape[0] and dout.shape[1] == q.shape[1] and dout.shape[2] == v.shape[2] and
             dout.dtype == q.dtype, "dout must have the shape and type of the result")
    _require(_BITS[t_rowptr.dtype] == args[1] and t_rowptr.shape[0] == k.shape[0] + 1 and t_rowptr.is_contiguous(),
             "the transposed row pointers must have the type of rowptr and an entry more than k has rows")
    for t in (t_row, t_edge):
        _require(t is None or (_BITS[t.dtype] == 32 and t.is_contiguous() and t.shape[0] == args[5]),
                 "the transposed pattern must have an int32 entry for each edge")
    _require(args[8] is None or t_edge is not None, "a bias needs the edges' positions in the transposed pattern")
    _same_place("q dout transposed transposed transposed lse", q, dout, t_rowptr, t_row, t_edge, lse)
    lddo, hsdo = _rows(dout, "dout")
    fn = _attn_fn("diff_attention_backward", C.c_int, *_ATTN_IN, _p, _p, _l, _l, _p, _p, _p, _p, _p, _p, _p, _p, _l, _p)
    return fn(*args, _ptr(lse), _ptr(dout), lddo, hsdo, _ptr(t_rowptr), _ptr(t_row), _ptr(t_edge), _ptr(dq), _ptr(dk), _ptr(dv),
              _ptr(dlam), _ptr(workspace), workspace.nbytes, stream)


def csr_transpose_workspace(m, n, nnz):
    return _attn_fn("csr_transpose_workspace", _l, _l, _l, _l)(m, n, nnz)


def csr_transpose(rowptr, colidx, n, t_rowptr, t_row, t_edge, workspace, stream=LEGACY_STREAM):
    """``fusedmm_b200_csr_transpose`` on torch CUDA tensors of the current device; returns the status code."""
    pb, ib = _pattern_bits(rowptr, colidx)
    _same_place("rowptr colidx", rowptr, colidx)
    fn = _attn_fn("csr_transpose", C.c_int, _i, _i, _l, _l, _l, _p, _p, _p, _p, _p, _p, _l, _p)
    return fn(pb, ib, rowptr.shape[0] - 1, n, colidx.shape[0], _ptr(rowptr), _ptr(colidx), _ptr(t_rowptr), _ptr(t_row),
              _ptr(t_edge), _ptr(workspace), workspace.nbytes, stream)
