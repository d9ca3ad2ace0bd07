"""ctypes binding of include/gern_b200.h.  Device entry points take torch CUDA tensors (used only
as owners of device memory); `_host` entry points take numpy arrays or CPU torch tensors."""
from __future__ import annotations

import ctypes
import itertools
import operator
import os
import struct

import numpy as np

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libgern_b200.so")

if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} is missing: build it with `python -m gern_b200.build` (there is no CPU or "
        "PyTorch fallback for the gern_b200 kernels)")

lib = ctypes.CDLL(LIB_PATH)

_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_int = ctypes.c_int

# name -> argtypes (after the leading ctx pointer); every function returns int unless noted.
SIGNATURES = {
    "gb200_ctx_create": None,
    "gb200_ctx_destroy": None,
    "gb200_device_sync": None,
    "gb200_last_error_string": None,
    "gb200_version": None,
    "gb200_launch_count": None,
    "gb200_gemm_f32": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp],
    "gb200_gemm_f32_variant": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp, _int],
    "gb200_gemm_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp],
    "gb200_gemm_bf16_cluster": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp],
    "gb200_gemm_bf16_splitk": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _int],
    "gb200_gemm_bf16_variant": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _int],
    "gb200_gemm_bf16_splitk_static": None,
    "gb200_softmax_rows_f32": [_vp, _i64, _vp, _i64, _i64, _i64, _vp],
    "gb200_softmax_rows_f32_variant": [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _int],
    "gb200_blur3x3_f32": [_vp, _i64, _i64, _i64, _vp, _i64, _vp],
    "gb200_blur3x3_f32_variant": [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _int],
    "gb200_blur3x3_f32_band": [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp],
    "gb200_attention_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                             ctypes.c_float, _vp],
    "gb200_attention_bf16_cluster": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                     ctypes.c_float, _int, _vp],
    "gb200_attention_bf16_splitkv": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                     ctypes.c_float, _vp, _int],
    "gb200_attention_bf16_variant": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                     ctypes.c_float, _vp, _int],
    "gb200_rmsnorm_f32": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i64, _i64, ctypes.c_float, _vp],
    "gb200_rmsnorm_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i64, _i64, ctypes.c_float, _vp],
    "gb200_rmsnorm_f32_e4m3": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _int,
                               ctypes.c_float, _vp],
    "gb200_rmsnorm_bf16_e4m3": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _int,
                                ctypes.c_float, _vp],
    "gb200_rmsnorm_backward_f32": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp, _int, _i64, _i64,
                                   ctypes.c_float, _vp],
    "gb200_rmsnorm_backward_bf16": [_vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp, _int, _i64, _i64,
                                    ctypes.c_float, _vp],
    "gb200_linear_xent_bf16": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp, _vp],
    "gb200_linear_xent_bf16_backward": [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64,
                                        ctypes.c_float, _vp, _i64, _vp, _i64, _vp],
    "gb200_grad_norm": [_vp, _i64, _vp, _vp],
    "gb200_grad_scale": [_vp, _i64, ctypes.c_float, _vp, _vp],
    "gb200_grad_clip": [_vp, _i64, ctypes.c_float, _vp, _vp],
    "gb200_gemm_f32_host": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _int],
    "gb200_gemm_bf16_host": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64],
    "gb200_softmax_rows_f32_host": [_vp, _i64, _vp, _i64, _i64, _i64],
    "gb200_blur3x3_f32_host": [_vp, _i64, _i64, _i64, _vp, _i64],
    "gb200_attention_bf16_host": [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                  ctypes.c_float],
}

lib.gb200_ctx_create.argtypes = [_int, ctypes.POINTER(_vp)]
lib.gb200_ctx_destroy.argtypes = [_vp]
lib.gb200_device_sync.argtypes = [_vp]
lib.gb200_last_error_string.restype = ctypes.c_char_p
lib.gb200_version.restype = ctypes.c_char_p
lib.gb200_selftest_bounded_wait.argtypes = [_vp, ctypes.c_ulonglong, _vp, _vp]
lib.gb200_selftest_bounded_wait.restype = _int
lib.gb200_selftest_bounded_flag_wait.argtypes = [_vp, ctypes.c_ulonglong, _vp, _vp]
lib.gb200_selftest_bounded_flag_wait.restype = _int
lib.gb200_launch_count.argtypes = [_vp]
lib.gb200_launch_count.restype = _i64
lib.gb200_gemm_bf16_splitk_static.argtypes = [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp]
lib.gb200_gemm_bf16_splitk_static.restype = _int
lib.gb200_static_status.argtypes = [ctypes.POINTER(_int)]
lib.gb200_static_status.restype = _int
SIGNATURES["gb200_static_status"] = None


class KernelResources(ctypes.Structure):
    """gb200_kernel_resources."""
    _fields_ = [("regs_per_thread", _int), ("threads", _int), ("dynamic_smem_bytes", _int), ("cluster_x", _int),
                ("tmem_columns", _int)]


lib.gb200_kernel_resources_query.argtypes = [ctypes.c_char_p, ctypes.POINTER(KernelResources)]
lib.gb200_kernel_resources_query.restype = _int
SIGNATURES["gb200_kernel_resources_query"] = None


def kernel_resources(name: str) -> KernelResources:
    out = KernelResources()
    _check(lib.gb200_kernel_resources_query(name.encode(), ctypes.byref(out)), "gb200_kernel_resources_query")
    return out


class GemmEpilogue(ctypes.Structure):
    """gb200_gemm_epilogue."""
    _fields_ = [("alpha", ctypes.c_float), ("row_sub", _vp), ("apply_exp", _int), ("row_div", _vp),
                ("row_max", _vp), ("row_sum", _vp)]


lib.gb200_gemm_bf16_epilogue.argtypes = [_vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64,
                                         ctypes.POINTER(GemmEpilogue), _vp]
lib.gb200_gemm_bf16_epilogue.restype = _int
lib.gb200_gemm_bf16_epilogue_variant.argtypes = lib.gb200_gemm_bf16_epilogue.argtypes + [_int]
lib.gb200_gemm_bf16_epilogue_variant.restype = _int
SIGNATURES["gb200_gemm_bf16_epilogue"] = None


class Shard(ctypes.Structure):
    """gb200_shard: one device's rows of a sharded call."""
    _fields_ = [("ctx", _vp), ("in_", _vp), ("out", _vp), ("rows", _i64), ("shared0", _vp),
                ("shared1", _vp), ("stream", _vp)]


_shards_p = ctypes.POINTER(Shard)
lib.gb200_gemm_bf16_sharded.argtypes = [_shards_p, _int, _i64, _i64, _i64, _i64, _i64]
lib.gb200_softmax_rows_f32_sharded.argtypes = [_shards_p, _int, _i64, _i64, _i64]
lib.gb200_attention_bf16_sharded.argtypes = [_shards_p, _int, _i64, _i64, _i64, _i64, _i64, _i64,
                                             ctypes.c_float]
lib.gb200_blur3x3_f32_sharded.argtypes = [_shards_p, _int, _i64, _i64, _i64]
for _name in ("gb200_gemm_bf16_sharded", "gb200_softmax_rows_f32_sharded",
              "gb200_attention_bf16_sharded", "gb200_blur3x3_f32_sharded"):
    SIGNATURES[_name] = None
    getattr(lib, _name).restype = _int
for _name, _args in SIGNATURES.items():
    if _args is not None and hasattr(lib, _name):
        getattr(lib, _name).argtypes = [_vp] + _args
        getattr(lib, _name).restype = _int


class GernB200Error(RuntimeError):
    def __init__(self, code: int, what: str):
        self.code = code
        msg = lib.gb200_last_error_string().decode(errors="replace")
        super().__init__(f"{what} failed with status {code}: {msg}")


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise GernB200Error(rc, what)


def _ptr(t) -> int:
    """Address of a torch tensor's / numpy array's first element (None -> NULL)."""
    if t is None:
        return None
    if isinstance(t, np.ndarray):
        return t.ctypes.data
    return t.data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        return None
    return getattr(stream, "cuda_stream", stream)


def _ld(t) -> int:
    if isinstance(t, np.ndarray):
        assert t.strides[1] == t.itemsize, "rows must be contiguous"
        return t.strides[0] // t.itemsize
    assert t.stride(1) == 1, "rows must be contiguous"
    return t.stride(0)


# The training operators' checks.  A call on a few rows takes the GPU 2 us, so what is asked of each tensor
# is asked once, and messages are put together only where a check fails.
_F32, _BF16, _I64 = ("torch.float32",), ("torch.bfloat16",), ("torch.int64",)
_FP8 = ("torch.float8_e4m3fn", "torch.uint8")
_TYPE_CODE = {"torch.float32": 0, "torch.bfloat16": 1}   # gb200_type
_dtype_names: dict = {}   # torch.dtype -> its name; str() of a dtype costs a microsecond
_type_codes: dict = {}    # torch.dtype -> gb200_type, -1 where there is none
_get_dtype = operator.attrgetter("dtype")


def _dtype_name(dtype) -> str:
    name = _dtype_names.get(dtype)
    if name is None:
        name = _dtype_names[dtype] = str(dtype)
    return name


def _mat(t, name, ctx, dtypes, shape) -> int:
    """Checks a matrix operand of a training operator and returns its leading dimension."""
    if t.shape != shape or len(shape) != 2:
        wanted = " x ".join(map(str, shape)) if len(shape) == 2 else "2-D"
        raise ValueError(f"{name}: a {wanted} matrix is wanted, got shape {tuple(t.shape)}")
    if _dtype_names.get(t.dtype) not in dtypes or t.get_device() != ctx.device:
        _explain(t, name, ctx, dtypes)
    ld, inner = t.stride()
    if inner != 1 and shape[1] > 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return ld if shape[0] > 1 else shape[1]


def _vec(t, name, ctx, dtypes, n) -> None:
    """Checks a contiguous vector operand of a training operator."""
    if t.shape != (n,):
        raise ValueError(f"{name}: a vector of {n} is wanted, got shape {tuple(t.shape)}")
    if _dtype_names.get(t.dtype) not in dtypes or t.get_device() != ctx.device:
        _explain(t, name, ctx, dtypes)
    if n > 1 and not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


def _explain(t, name, ctx, dtypes) -> None:
    """Raises what is wrong with a tensor's type or device; returns if the type had only not been seen before."""
    if _dtype_name(t.dtype) not in dtypes:
        raise TypeError(f"{name}: {' or '.join(dtypes)} is wanted, got {t.dtype}")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: must be on cuda:{ctx.device}, the context's device, and is on {t.device}")


def _norm_entry(x, f32, bf16):
    """(entry point, its name, x's type) of a norm by x's type."""
    if _dtype_name(x.dtype) == "torch.float32":
        return f32[0], f32[1], _F32
    return bf16[0], bf16[1], _BF16


def _entry(name):
    return getattr(lib, name), name


_NORM = _entry("gb200_rmsnorm_f32"), _entry("gb200_rmsnorm_bf16")
_NORM_E4M3 = _entry("gb200_rmsnorm_f32_e4m3"), _entry("gb200_rmsnorm_bf16_e4m3")
_NORM_BACKWARD = _entry("gb200_rmsnorm_backward_f32"), _entry("gb200_rmsnorm_backward_bf16")


def gemm_bf16_splitk_static(A, Bt, C, splits=0, stream=None):
    """Context-free, allocation-free split-K GEMM on the current device (see gern_b200.h)."""
    M, K = A.shape
    N = Bt.shape[0]
    _check(lib.gb200_gemm_bf16_splitk_static(_ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C), _ld(C), M, N, K,
                                             int(splits), _stream(stream)), "gb200_gemm_bf16_splitk_static")


def static_status():
    """gb200_static_status: raises GernB200Error(-5) if a kernel of the static entry gave up a wait."""
    code = _int(0)
    _check(lib.gb200_static_status(ctypes.byref(code)), "gb200_static_status")


def _shard_array(parts):
    """parts: list of (Context, in, out, shared0, shared1, stream); rows come from `in`."""
    arr = (Shard * len(parts))()
    for g, (ctx, x, out, s0, s1, stream) in enumerate(parts):
        arr[g] = Shard(ctx.handle, _ptr(x), _ptr(out), x.shape[0], _ptr(s0), _ptr(s1), _stream(stream))
    return arr


def gemm_bf16_sharded(parts):
    """parts: one (Context, A_panel, C_panel, Bt_replica) per device."""
    a0, c0, b0 = parts[0][1], parts[0][2], parts[0][3]
    arr = _shard_array([(c, a, o, b, None, None) for c, a, o, b in parts])
    _check(lib.gb200_gemm_bf16_sharded(arr, len(parts), _ld(a0), _ld(b0), _ld(c0), b0.shape[0],
                                       a0.shape[1]), "gb200_gemm_bf16_sharded")


def softmax_rows_sharded(parts):
    """parts: one (Context, x_rows, out_rows) per device."""
    x0, o0 = parts[0][1], parts[0][2]
    arr = _shard_array([(c, x, o, None, None, None) for c, x, o in parts])
    _check(lib.gb200_softmax_rows_f32_sharded(arr, len(parts), _ld(x0), _ld(o0), x0.shape[1]),
           "gb200_softmax_rows_f32_sharded")


def attention_bf16_sharded(parts, scale):
    """parts: one (Context, Q_rows, O_rows, K_replica, V_replica) per device."""
    q0, o0, k0, v0 = parts[0][1], parts[0][2], parts[0][3], parts[0][4]
    arr = _shard_array([(c, q, o, k, v, None) for c, q, o, k, v in parts])
    _check(lib.gb200_attention_bf16_sharded(arr, len(parts), _ld(q0), _ld(k0), _ld(v0), _ld(o0),
                                            k0.shape[0], q0.shape[1], ctypes.c_float(scale)),
           "gb200_attention_bf16_sharded")


def blur3x3_sharded(parts):
    """parts: one (Context, band, out_band) per device, bands in image order."""
    x0, o0 = parts[0][1], parts[0][2]
    arr = _shard_array([(c, x, o, None, None, None) for c, x, o in parts])
    _check(lib.gb200_blur3x3_f32_sharded(arr, len(parts), _ld(x0), x0.shape[1], _ld(o0)),
           "gb200_blur3x3_f32_sharded")


class Context:
    """Owner of a gb200_ctx (one per process and device)."""

    def __init__(self, device: int = 0):
        h = _vp()
        _check(lib.gb200_ctx_create(int(device), ctypes.byref(h)), "gb200_ctx_create")
        self.handle = h
        self.device = device

    def close(self) -> None:
        if getattr(self, "handle", None):
            lib.gb200_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self) -> None:
        _check(lib.gb200_device_sync(self.handle), "gb200_device_sync")

    def launch_count(self) -> int:
        return int(lib.gb200_launch_count(self.handle))

    # ---- device entry points (torch CUDA tensors) ----
    def gemm_f32(self, A, B, C, accumulate=False, stream=None, variant=None):
        M, K = A.shape
        N = B.shape[1]
        if variant is not None:
            _check(lib.gb200_gemm_f32_variant(self.handle, _ptr(A), _ld(A), _ptr(B), _ld(B), _ptr(C), _ld(C),
                                              M, N, K, int(bool(accumulate)), _stream(stream), int(variant)),
                   "gb200_gemm_f32_variant")
            return
        _check(lib.gb200_gemm_f32(self.handle, _ptr(A), _ld(A), _ptr(B), _ld(B), _ptr(C), _ld(C), M, N, K,
                                  int(bool(accumulate)), _stream(stream)), "gb200_gemm_f32")

    def gemm_bf16(self, A, Bt, C, stream=None, splits=None, variant=None):
        """A: (M,K) bf16; Bt: (N,K) bf16 (column-major B); C: (M,N) bf16."""
        M, K = A.shape
        N = Bt.shape[0]
        if variant is not None:
            _check(lib.gb200_gemm_bf16_variant(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C),
                                               _ld(C), M, N, K, _stream(stream), int(variant)),
                   "gb200_gemm_bf16_variant")
            return
        if splits is not None:
            _check(lib.gb200_gemm_bf16_splitk(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C),
                                              _ld(C), M, N, K, _stream(stream), int(splits)),
                   "gb200_gemm_bf16_splitk")
            return
        _check(lib.gb200_gemm_bf16(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C), _ld(C), M, N,
                                   K, _stream(stream)), "gb200_gemm_bf16")

    def gemm_bf16_epilogue(self, A, Bt, C=None, alpha=1.0, row_sub=None, apply_exp=False, row_div=None,
                           row_max=None, row_sum=None, stream=None, variant=None):
        """C = bf16(epilogue(alpha * A Bt^T)); any of C / row_max / row_sum may be left out."""
        M, K = A.shape
        N = Bt.shape[0]
        e = GemmEpilogue(ctypes.c_float(alpha), _ptr(row_sub), int(bool(apply_exp)), _ptr(row_div),
                         _ptr(row_max), _ptr(row_sum))
        if variant is not None:
            _check(lib.gb200_gemm_bf16_epilogue_variant(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C),
                                                        _ld(C) if C is not None else 0, M, N, K, ctypes.byref(e),
                                                        _stream(stream), int(variant)), "gb200_gemm_bf16_epilogue_variant")
            return
        _check(lib.gb200_gemm_bf16_epilogue(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C),
                                            _ld(C) if C is not None else 0, M, N, K, ctypes.byref(e),
                                            _stream(stream)), "gb200_gemm_bf16_epilogue")

    def softmax_rows(self, x, out, stream=None, variant=None):
        rows, cols = x.shape
        if variant is not None:
            _check(lib.gb200_softmax_rows_f32_variant(self.handle, _ptr(x), _ld(x), _ptr(out), _ld(out),
                                                      rows, cols, _stream(stream), int(variant)),
                   "gb200_softmax_rows_f32_variant")
            return
        _check(lib.gb200_softmax_rows_f32(self.handle, _ptr(x), _ld(x), _ptr(out), _ld(out), rows, cols,
                                          _stream(stream)), "gb200_softmax_rows_f32")

    def blur3x3(self, x, out, stream=None, variant=None):
        rows, cols = x.shape
        if variant is None:
            _check(lib.gb200_blur3x3_f32(self.handle, _ptr(x), _ld(x), rows, cols, _ptr(out), _ld(out),
                                         _stream(stream)), "gb200_blur3x3_f32")
        else:
            _check(lib.gb200_blur3x3_f32_variant(self.handle, _ptr(x), _ld(x), rows, cols, _ptr(out),
                                                 _ld(out), _stream(stream), int(variant)),
                   "gb200_blur3x3_f32_variant")

    def blur3x3_band(self, x, halo, out, stream=None, halo_ptr=None, halo_ld=None):
        """x: this rank's band; halo: tensor with the 2 rows that follow it (or None)."""
        rows, cols = x.shape
        hp = halo_ptr if halo_ptr is not None else _ptr(halo)
        hl = halo_ld if halo_ld is not None else (_ld(halo) if halo is not None else 0)
        _check(lib.gb200_blur3x3_f32_band(self.handle, _ptr(x), _ld(x), rows, cols, hp, hl, _ptr(out),
                                          _ld(out), _stream(stream)), "gb200_blur3x3_f32_band")

    def attention_bf16(self, Q, K, V, O, scale, stream=None, variant=None, splits=None):
        """splits (test hook): 0 = the library's choice, 1 = whole Q tile pairs per thread block,
        n > 1 = that many K/V ranges and a combine pass, -1 = equal runs of (pair, K/V block) units
        per thread block, merged inside the kernel, -9 = whole pairs through the same instantiation
        as the equal runs."""
        nq, d = Q.shape
        nkv = K.shape[0]
        if splits is not None:
            _check(lib.gb200_attention_bf16_splitkv(self.handle, _ptr(Q), _ld(Q), _ptr(K), _ld(K), _ptr(V),
                                                    _ld(V), _ptr(O), _ld(O), nq, nkv, d,
                                                    ctypes.c_float(scale), _stream(stream), int(splits)),
                   "gb200_attention_bf16_splitkv")
            return
        if variant is not None:
            _check(lib.gb200_attention_bf16_variant(self.handle, _ptr(Q), _ld(Q), _ptr(K), _ld(K), _ptr(V),
                                                    _ld(V), _ptr(O), _ld(O), nq, nkv, d,
                                                    ctypes.c_float(scale), _stream(stream), int(variant)),
                   "gb200_attention_bf16_variant")
            return
        _check(lib.gb200_attention_bf16(self.handle, _ptr(Q), _ld(Q), _ptr(K), _ld(K), _ptr(V), _ld(V),
                                        _ptr(O), _ld(O), nq, nkv, d, ctypes.c_float(scale),
                                        _stream(stream)), "gb200_attention_bf16")

    # ---- training operators (torch CUDA tensors on the context's device) ----
    def rmsnorm(self, x, weight, out, eps, residual=None, residual_out=None, stream=None):
        """out = norm(x + residual) * weight by rows; residual_out = x + residual.  All of x's type (fp32 or bf16)."""
        fn, name, dt = _norm_entry(x, *_NORM)
        shape = x.shape
        ldx, ldy = _mat(x, "x", self, dt, shape), _mat(out, "out", self, dt, shape)
        rows, cols = shape
        ldr = ldo = 0
        pr = po = None
        if residual is not None:
            ldr, pr = _mat(residual, "residual", self, dt, shape), residual.data_ptr()
        if residual_out is not None:
            ldo, po = _mat(residual_out, "residual_out", self, dt, shape), residual_out.data_ptr()
        _vec(weight, "weight", self, dt, cols)
        _check(fn(self.handle, x.data_ptr(), ldx, pr, ldr, weight.data_ptr(), out.data_ptr(), ldy, po, ldo, rows, cols, eps,
                  _stream(stream)), name)

    def rmsnorm_e4m3(self, x, weight, out, scales, eps, group=0, residual=None, residual_out=None, stream=None):
        """The norm as e4m3 (out: float8_e4m3fn or uint8) with one fp32 scale per `group` columns (0: per row);
        scales: rows x ceil(cols / group)."""
        fn, name, dt = _norm_entry(x, *_NORM_E4M3)
        shape = x.shape
        ldx, ldq = _mat(x, "x", self, dt, shape), _mat(out, "out", self, _FP8, shape)
        rows, cols = shape
        lds = _mat(scales, "scales", self, _F32, (rows, -(-cols // group) if group > 0 else 1))
        ldr = ldo = 0
        pr = po = None
        if residual is not None:
            ldr, pr = _mat(residual, "residual", self, dt, shape), residual.data_ptr()
        if residual_out is not None:
            ldo, po = _mat(residual_out, "residual_out", self, dt, shape), residual_out.data_ptr()
        _vec(weight, "weight", self, dt, cols)
        _check(fn(self.handle, x.data_ptr(), ldx, pr, ldr, weight.data_ptr(), out.data_ptr(), ldq, scales.data_ptr(), lds, po,
                  ldo, rows, cols, group, eps, _stream(stream)), name)

    def rmsnorm_backward(self, dy, h, weight, dx, dweight, eps, dresidual=None, accumulate=False, stream=None):
        """Gradient of the norm at h, the stored x + residual: dx (of h's type; plus dresidual) and dweight
        (fp32, may be None; added to when `accumulate`)."""
        fn, name, dt = _norm_entry(h, *_NORM_BACKWARD)
        shape = h.shape
        lddy, ldh, lddx = _mat(dy, "dy", self, dt, shape), _mat(h, "h", self, dt, shape), _mat(dx, "dx", self, dt, shape)
        rows, cols = shape
        ldd = 0
        pd = pw = None
        if dresidual is not None:
            ldd, pd = _mat(dresidual, "dresidual", self, dt, shape), dresidual.data_ptr()
        _vec(weight, "weight", self, dt, cols)
        if dweight is not None:
            _vec(dweight, "dweight", self, _F32, cols)
            pw = dweight.data_ptr()
        _check(fn(self.handle, dy.data_ptr(), lddy, h.data_ptr(), ldh, weight.data_ptr(), pd, ldd, dx.data_ptr(), lddx, pw,
                  int(bool(accumulate)), rows, cols, eps, _stream(stream)), name)

    def linear_xent(self, h, w, targets, loss, lse, total=None, ignore_index=-100, stream=None):
        """loss[t] = logsumexp(h[t] w^T) - (h[t] . w[targets[t]]) without keeping the logits.  h: (T, D) bf16; w: (V, D)
        bf16; targets: (T,) int64; loss, lse: (T,) fp32 (either may be None); total: (2,) fp32, the summed loss and the
        number of counted tokens.  Tokens whose target is ignore_index have loss 0."""
        T, D = h.shape
        V = w.shape[0]
        ldh, ldw = _mat(h, "h", self, _BF16, (T, D)), _mat(w, "w", self, _BF16, (V, D))
        _vec(targets, "targets", self, _I64, T)
        ploss = plse = ptotal = None
        if loss is not None:
            _vec(loss, "loss", self, _F32, T)
            ploss = loss.data_ptr()
        if lse is not None:
            _vec(lse, "lse", self, _F32, T)
            plse = lse.data_ptr()
        if total is not None:
            _vec(total, "total", self, _F32, 2)
            ptotal = total.data_ptr()
        _check(lib.gb200_linear_xent_bf16(self.handle, h.data_ptr(), ldh, w.data_ptr(), ldw, targets.data_ptr(), T, V, D,
                                          ignore_index, ploss, plse, ptotal, _stream(stream)), "gb200_linear_xent_bf16")

    def linear_xent_backward(self, h, w, targets, lse, dh, dw, dloss=None, total=None, ignore_index=-100, scale=1.0,
                             stream=None):
        """Gradients dh (T, D) and dw (V, D), bf16 (either may be None), of scale * sum_t dloss[t] loss[t], or with
        total (from linear_xent) in place of dloss of scale * the mean loss of the counted tokens."""
        T, D = h.shape
        V = w.shape[0]
        ldh, ldw = _mat(h, "h", self, _BF16, (T, D)), _mat(w, "w", self, _BF16, (V, D))
        _vec(targets, "targets", self, _I64, T)
        _vec(lse, "lse", self, _F32, T)
        lddh = lddw = 0
        pdh = pdw = pdloss = ptotal = None
        if dh is not None:
            lddh, pdh = _mat(dh, "dh", self, _BF16, (T, D)), dh.data_ptr()
        if dw is not None:
            lddw, pdw = _mat(dw, "dw", self, _BF16, (V, D)), dw.data_ptr()
        if dloss is not None:
            _vec(dloss, "dloss", self, _F32, T)
            pdloss = dloss.data_ptr()
        if total is not None:
            _vec(total, "total", self, _F32, 2)
            ptotal = total.data_ptr()
        _check(lib.gb200_linear_xent_bf16_backward(self.handle, h.data_ptr(), ldh, w.data_ptr(), ldw, targets.data_ptr(),
                                                   lse.data_ptr(), pdloss, ptotal, T, V, D, ignore_index, scale, pdh, lddh,
                                                   pdw, lddw, _stream(stream)), "gb200_linear_xent_bf16_backward")

    def _described(self, tensors, what):
        """Pointers, sizes and gb200_type codes of a list of tensors, each contiguous and on the context's device."""
        if not tensors:
            return (), (), ()
        kinds = list(map(_type_codes.get, map(_get_dtype, tensors)))
        if None in kinds:      # a type that has not come by yet
            for t in tensors:
                _type_codes[t.dtype] = _TYPE_CODE.get(_dtype_name(t.dtype), -1)
            kinds = [_type_codes[t.dtype] for t in tensors]
        tensor = type(tensors[0])
        try:      # one C call per tensor and question instead of an attribute lookup each
            fine = set(map(tensor.get_device, tensors)) == {self.device} and all(map(tensor.is_contiguous, tensors))
            ptrs, sizes = map(tensor.data_ptr, tensors), list(map(tensor.numel, tensors))
        except TypeError:      # a list of several classes of tensors
            fine = all(t.get_device() == self.device and t.is_contiguous() for t in tensors)
            ptrs, sizes = [t.data_ptr() for t in tensors], [t.numel() for t in tensors]
        if not fine or -1 in kinds:
            for i, t in enumerate(tensors):
                if kinds[i] < 0 or t.get_device() != self.device or not t.is_contiguous():
                    raise ValueError(f"{what} {i}: a contiguous fp32 or bf16 tensor on cuda:{self.device} is wanted")
        return ptrs, sizes, kinds

    def _tensors(self, tensors, outs=None):
        """The gb200_tensor array of a list of contiguous tensors (and of as many results)."""
        n = len(tensors)
        if outs is None:
            ptrs, sizes, kinds = self._described(tensors, "tensor")
            fields = zip(ptrs, itertools.repeat(0), sizes, kinds, kinds)
        else:
            ptrs, sizes, kinds = self._described(tensors, "tensor")
            optrs, osizes, okinds = self._described(outs, "result")
            if sizes != osizes:
                raise ValueError(f"{n} tensors and {len(outs)} results, or results of other sizes than their tensors")
            fields = zip(ptrs, optrs, sizes, kinds, okinds)
        return struct.pack("QQqii" * n, *itertools.chain.from_iterable(fields)), n

    def grad_norm(self, grads, norm, stream=None):
        """norm[0] = the 2-norm over all elements of all tensors (fp32 or bf16, mixed as they come)."""
        _vec(norm, "norm", self, _F32, 1)
        buf, n = self._tensors(grads)
        _check(lib.gb200_grad_norm(self.handle, buf, n, _ptr(norm), _stream(stream)), "gb200_grad_norm")

    def grad_scale(self, grads, max_norm, norm, outs=None, stream=None):
        """Scales every tensor by max_norm / norm[0] where norm[0] > max_norm, in place or into `outs`."""
        _vec(norm, "norm", self, _F32, 1)
        buf, n = self._tensors(grads, outs)
        _check(lib.gb200_grad_scale(self.handle, buf, n, max_norm, _ptr(norm), _stream(stream)), "gb200_grad_scale")

    def grad_clip(self, grads, max_norm, norm, outs=None, stream=None):
        """grad_norm and grad_scale: norm[0] receives the norm before clipping."""
        _vec(norm, "norm", self, _F32, 1)
        buf, n = self._tensors(grads, outs)
        _check(lib.gb200_grad_clip(self.handle, buf, n, max_norm, _ptr(norm), _stream(stream)), "gb200_grad_clip")

    # ---- host entry points (numpy arrays / CPU tensors) ----
    def gemm_f32_host(self, A, B, C, accumulate=False):
        M, K = A.shape
        N = B.shape[1]
        _check(lib.gb200_gemm_f32_host(self.handle, _ptr(A), _ld(A), _ptr(B), _ld(B), _ptr(C), _ld(C), M,
                                       N, K, int(bool(accumulate))), "gb200_gemm_f32_host")

    def gemm_bf16_host(self, A, Bt, C):
        M, K = A.shape
        N = Bt.shape[0]
        _check(lib.gb200_gemm_bf16_host(self.handle, _ptr(A), _ld(A), _ptr(Bt), _ld(Bt), _ptr(C), _ld(C),
                                        M, N, K), "gb200_gemm_bf16_host")

    def softmax_rows_host(self, x, out):
        rows, cols = x.shape
        _check(lib.gb200_softmax_rows_f32_host(self.handle, _ptr(x), _ld(x), _ptr(out), _ld(out), rows,
                                               cols), "gb200_softmax_rows_f32_host")

    def blur3x3_host(self, x, out):
        rows, cols = x.shape
        _check(lib.gb200_blur3x3_f32_host(self.handle, _ptr(x), _ld(x), rows, cols, _ptr(out), _ld(out)),
               "gb200_blur3x3_f32_host")

    def attention_bf16_host(self, Q, K, V, O, scale):
        nq, d = Q.shape
        nkv = K.shape[0]
        _check(lib.gb200_attention_bf16_host(self.handle, _ptr(Q), _ld(Q), _ptr(K), _ld(K), _ptr(V),
                                             _ld(V), _ptr(O), _ld(O), nq, nkv, d, ctypes.c_float(scale)),
               "gb200_attention_bf16_host")
