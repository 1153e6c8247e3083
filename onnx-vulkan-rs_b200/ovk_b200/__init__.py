"""ctypes binding of ``libovk_cuda.so`` - the C ABI declared in ``include/ovk_cuda.h``.

The library is the product; this module only loads it, declares the
signatures and wraps device memory held in torch CUDA tensors (torch is the
allocator and the stream provider here, nothing more).  There is no fallback:
if the library is missing or was not built, importing the ops fails loudly.

The wrappers mirror the reference's operator functions
(crates/onnx-vulkan-core/src/interp.rs): ``matmul_nbits`` (:6429),
``dynamic_quantize`` (:1945), ``matmul_integer`` (:2090),
``matmul_integer_scale_bias`` (:2405), ``qlinear_matmul`` (:4845),
``conv_integer`` (:4421), ``qlinear_conv`` (:4796).
"""
from __future__ import annotations

import ctypes as C
import functools
import operator
import os
import struct

FLOAT, UINT8, INT8, INT32, INT64, FLOAT16 = 1, 2, 3, 6, 7, 10
OK, INVALID_ARGUMENT, UNSUPPORTED, BACKEND, TIMEOUT = 0, 1, 2, 3, 4
EPILOGUE_RELU, EPILOGUE_RANGE = 1, 2
NBITS_NO_DECODE_COPY = 1
COMM_HANDLE_BYTES = 64

_PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(_PKG, "libovk_cuda.so")


class OvkError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"[ovk status {status}] {message}")
        self.status = status
        self.message = message


class ConvParams(C.Structure):
    _fields_ = [("n", C.c_int64), ("c_in", C.c_int64), ("h", C.c_int64), ("w", C.c_int64),
                ("pads", C.c_int64 * 4), ("strides", C.c_int64 * 2), ("dilations", C.c_int64 * 2)]


class Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("heads", C.c_int64), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class RotaryParams(C.Structure):
    _fields_ = [("tokens", C.c_int64), ("head_dim", C.c_int64), ("rotary_dim", C.c_int64), ("max_position", C.c_int64),
                ("dtype", C.c_int32), ("table_dtype", C.c_int32), ("positions_dtype", C.c_int32), ("interleaved", C.c_int32),
                ("axes", C.c_int32), ("sections", C.c_int32 * 4)]


class KV4CacheParams(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p),
                ("k_zero_points", C.c_void_p), ("v_zero_points", C.c_void_p), ("pages", C.c_int64), ("kv_heads", C.c_int64),
                ("page_size", C.c_int64), ("head_dim", C.c_int64), ("block_size", C.c_int64)]


class KV4Batch(C.Structure):
    _fields_ = [("tokens", C.c_int64), ("batch", C.c_int64), ("max_pages", C.c_int64), ("cu_tokens", C.c_void_p),
                ("lens", C.c_void_p), ("block_table", C.c_void_p)]


class PromptParams(C.Structure):
    _fields_ = [("q_tokens", C.c_int64), ("k_tokens", C.c_int64), ("batch", C.c_int64), ("head_dim", C.c_int64),
                ("dtype", C.c_int32), ("causal", C.c_int32), ("window", C.c_int64), ("scale", C.c_float), ("max_q", C.c_int32)]


# the same structs as packed bytes
_PACK_HEADS, _PACK_HEADS2 = struct.Struct("@Pqqq").pack, struct.Struct("@PqqqPqqq").pack
_PACK_ROTARY = struct.Struct("@qqqqiiiiiiiii4x").pack
_PACK_BATCH = struct.Struct("@qqqPPP").pack
_PACK_PROMPT = struct.Struct("@qqqqiiqfi").pack


@functools.cache
def _activation_codes() -> dict:
    import torch
    return {torch.float32: FLOAT, torch.float16: FLOAT16}


@functools.cache
def _index_codes() -> dict:
    import torch
    return {torch.int64: INT64, torch.int32: INT32}


@functools.cache
def _int32() -> tuple:
    import torch
    return (torch.int32,)


@functools.cache
def _raw_stream():
    """device -> the handle of torch's current stream there."""
    import torch
    return getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


@functools.cache
def _capturing():
    import torch
    return torch.cuda.is_current_stream_capturing


def _whole(what: str, v, most: int = 2 ** 63 - 1) -> int:
    """A whole number that a signed field holds whose largest value is `most`."""
    try:
        n = operator.index(v)
    except TypeError:
        raise OvkError(INVALID_ARGUMENT, f"{what}: a whole number is needed, not {v!r}") from None
    if not -most - 1 <= n <= most:
        raise OvkError(INVALID_ARGUMENT, f"{what}: {n} is too large")
    return n


def _scale(what: str, scale) -> float:
    """A scale as an f32 field takes it (what is not finite is refused behind the C interface)."""
    try:
        scale = float(scale)
    except (TypeError, ValueError, OverflowError):
        raise OvkError(INVALID_ARGUMENT, f"{what}: scale {scale!r} is no number") from None
    return scale if abs(scale) <= 3.4028234663852886e38 or scale != scale else float("inf")


def _dims(what: str, t, *ranks: int) -> int:
    """How many dimensions a tensor has, one of `ranks`."""
    try:
        n = t.dim()
    except AttributeError:
        raise OvkError(INVALID_ARGUMENT, f"{what}: a tensor is needed, not {type(t).__name__}") from None
    if n not in ranks:
        raise OvkError(INVALID_ARGUMENT, f"{what}: {' or '.join(map(str, ranks))} dimensions are needed, not {list(t.shape)}")
    return n


class _PackedCalls:
    """The attention entry points with their structs as addresses or bytes."""

    def __init__(self):
        for name in ("ovk_rotary", "ovk_kv4_append", "ovk_attention_kv4", "ovk_attention_prompt"):
            fn = lib()[name]
            fn.restype = SIGNATURES[name][0]
            fn.argtypes = [_P if hasattr(t, "_type_") and isinstance(t._type_, type) and issubclass(t._type_, C.Structure) else t
                           for t in SIGNATURES[name][1]]
            setattr(self, name, fn)


@functools.cache
def _packed_calls() -> _PackedCalls:
    return _PackedCalls()


_lib = None

# name -> (restype, argtypes); every symbol ovk_cuda.h declares
_P, _I32, _I64, _U32, _SZ = C.c_void_p, C.c_int32, C.c_int64, C.c_uint32, C.c_size_t
SIGNATURES = {
    "ovk_ctx_create": (_I32, [_I32, _P, C.POINTER(_P)]),
    "ovk_ctx_destroy": (None, [_P]),
    "ovk_last_error": (C.c_char_p, [_P]),
    "ovk_last_kernel": (C.c_char_p, [_P]),
    "ovk_launch_count": (C.c_uint64, [_P]),
    "ovk_stream": (_P, [_P]),
    "ovk_workspace_bytes": (_SZ, [_P]),
    "ovk_selftest_device_timeout": (_I32, [_P]),
    "ovk_probe_mma_rate": (_I32, [_P, _I32, C.POINTER(C.c_double)]),
    "ovk_flush": (_I32, [_P]),
    "ovk_alloc": (_I32, [_P, _SZ, C.POINTER(_P)]),
    "ovk_free": (_I32, [_P, _P]),
    "ovk_upload": (_I32, [_P, _P, _SZ, _P, _SZ]),
    "ovk_download": (_I32, [_P, _P, _SZ, _P, _SZ]),
    "ovk_fill": (_I32, [_P, _P, _SZ, _SZ, _U32]),
    "ovk_timer_start": (_I32, [_P]),
    "ovk_timer_stop": (_I32, [_P, C.POINTER(C.c_float)]),
    "ovk_nbits_prepack": (_I32, [_P, _P, _P, _I32, _P, _I64, _I64, _I64, _I64, _U32, C.POINTER(_P)]),
    "ovk_nbits_weight_destroy": (None, [_P, _P]),
    "ovk_matmul_nbits": (_I32, [_P, _P, _P, _I32, _I64, _P, _I32]),
    "ovk_matmul_nbits_group": (_I32, [_P, _I32, C.POINTER(_P), _P, _I32, _I64, C.POINTER(_P), _I32]),
    "ovk_comm_flag_bytes": (_SZ, []),
    "ovk_comm_alloc": (_I32, [_P, _SZ, C.POINTER(_P)]),
    "ovk_comm_export": (_I32, [_P, _P, _P]),
    "ovk_comm_import": (_I32, [_P, _P, C.POINTER(_P)]),
    "ovk_comm_release": (_I32, [_P, _P]),
    "ovk_comm_init": (_I32, [_P, _I32, _I32, C.POINTER(_P)]),
    "ovk_comm_set_timeout_ms": (_I32, [_P, _I32]),
    "ovk_comm_barrier": (_I32, [_P]),
    "ovk_allgather_cols": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _I64, C.POINTER(_P)]),
    "ovk_matmul_nbits_nsplit": (_I32, [_P, _P, _P, _I32, _I64, _I64, _I64, C.POINTER(_P), _I32]),
    "ovk_matmul_nbits_nsplit_multicast": (_I32, [_P, _P, _P, _I32, _I64, _I64, _I64, C.POINTER(_P), _P, _I32]),
    "ovk_allgather_cols_multicast": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _I64, C.POINTER(_P), _P]),
    "ovk_dynamic_quantize": (_I32, [_P, _P, _I64, _P, _P, _P]),
    "ovk_dynamic_quantize_folded": (_I32, [_P, _P, _I64, _P, _P, _P, _P]),
    "ovk_decomposed_gelu": (_I32, [_P, _P, _I64, C.c_float, C.c_float, C.c_float, _I32, _P]),
    "ovk_decomposed_gelu_quantize": (_I32, [_P, _P, _I64, C.c_float, C.c_float, C.c_float, _I32, _P, _P, _P]),
    "ovk_mmi_prepack": (_I32, [_P, _P, _I32, _I64, _I64, C.POINTER(_P)]),
    "ovk_mmi_weight_destroy": (None, [_P, _P]),
    "ovk_matmul_integer": (_I32, [_P, _P, _P, _I32, _I64, _P, _P, _P]),
    "ovk_matmul_integer_static_scratch": (_I32, [_P, _P, _P, _I32, _I64, _P, _P, _P]),
    "ovk_matmul_integer_scale_bias": (_I32, [_P, _P, _P, _I32, _I64, _P, _P, _P, _I32, _P, _I32, _P,
                                             _I32, _U32, _P, _P]),
    "ovk_integer_scale_bias_unfused": (_I32, [_P, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _U32, _P]),
    "ovk_matmul_integer_group": (_I32, [_P, _I32, C.POINTER(_P), _P, _I32, _I64, _P, _P, C.POINTER(_P)]),
    "ovk_matmul_integer_scale_bias_group": (_I32, [_P, _I32, C.POINTER(_P), _P, _I32, _I64, _P, _P, C.POINTER(_P), _I32,
                                                   _P, _I32, C.POINTER(_P), _I32, _U32, C.POINTER(_P)]),
    "ovk_qlinear_matmul": (_I32, [_P, _P, _P, _I32, _I64, _P, _P, _P, _I64, _I32, _I32, _P]),
    "ovk_qconv_prepack": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _I64, _I64, C.POINTER(_P)]),
    "ovk_qconv_weight_destroy": (None, [_P, _P]),
    "ovk_conv_output_shape": (_I32, [_P, C.POINTER(ConvParams), C.POINTER(_I64), C.POINTER(_I64)]),
    "ovk_conv_integer": (_I32, [_P, _P, _P, _I32, C.POINTER(ConvParams), _I32, _I32, _P]),
    "ovk_conv_integer_scale_bias": (_I32, [_P, _P, _P, _I32, C.POINTER(ConvParams), _I32, _I32, _P, _I32, _P, _I32,
                                           _P, _I32, _U32, _P, _P]),
    "ovk_qlinear_conv": (_I32, [_P, _P, _P, _I32, C.POINTER(ConvParams), _I32, _I32, _P, _P, _I32, _I32, _P]),
    "ovk_qlinear_conv_layout": (_I32, [_P, _P, _P, _I32, _I32, C.POINTER(ConvParams), _I32, _I32, _P, _P, _I32, _I32, _P,
                                       _I32, C.POINTER(_I64)]),
    "ovk_nchw_to_padded_nhwc": (_I32, [_P, _P, _I64, _I64, _I64, _I64, C.POINTER(_I64), _I32, _P]),
    "ovk_padded_nhwc_to_nchw": (_I32, [_P, _P, _I64, _I64, _I64, _I64, C.POINTER(_I64), _P]),
    "ovk_requantize": (_I32, [_P, _P, _I64, _I64, _I64, _P, _P, _I32, _I32, _P]),
    "ovk_gather_block_quantized": (_I32, [_P, _P, _P, _I32, _P, _I64, _I64, _I64, _I64, _P, _I32, _I32, _I64, _P, _I32]),
    "ovk_argmax": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _P]),
    "ovk_qlinear_add": (_I32, [_P, _P, C.POINTER(_I64), _I32, C.c_float, _I32, _P, C.POINTER(_I64), _I32, C.c_float, _I32,
                               C.c_float, _I32, _I32, _P, C.POINTER(_I64), C.POINTER(_I32)]),
    "ovk_maxpool_q": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _I64, C.POINTER(_I64), C.POINTER(_I64), C.POINTER(_I64),
                             C.POINTER(_I64), _P, C.POINTER(_I64), C.POINTER(_I64)]),
    "ovk_quantize_linear": (_I32, [_P, _P, _I64, _I64, _I64, _P, _P, _I32, _P]),
    "ovk_dequantize_linear": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _P, _P, _P]),
    "ovk_rotary": (_I32, [_P, C.POINTER(RotaryParams), _I32, C.POINTER(Heads), C.POINTER(Heads), _P, _P, _P]),
    "ovk_kv4_append": (_I32, [_P, C.POINTER(KV4CacheParams), C.POINTER(KV4Batch), C.POINTER(Heads), C.POINTER(Heads), _I32]),
    "ovk_attention_kv4": (_I32, [_P, C.POINTER(KV4CacheParams), C.POINTER(KV4Batch), C.POINTER(Heads), C.POINTER(Heads), _I32, _I64,
                                 C.c_float, _I64, _P, _SZ]),
    "ovk_attention_kv4_workspace": (_I32, [_P, C.POINTER(KV4CacheParams), _I64, _I64, _I32, C.POINTER(_SZ)]),
    "ovk_attention_prompt": (_I32, [_P, C.POINTER(PromptParams), C.POINTER(Heads), C.POINTER(Heads), C.POINTER(Heads), _P, _P,
                                    C.POINTER(Heads)]),
    "ovk_qlinear_global_average_pool": (_I32, [_P, _P, _I32, _I64, _I64, _I64, C.c_float, _I32, C.c_float, _I32, _P]),
}


def lib() -> C.CDLL:
    """Loads the shared library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise OvkError(BACKEND, f"{LIB_PATH} is missing: run `python onnx-vulkan-rs_b200/build.py` "
                                    "(there is no CPU fallback)")
        _lib = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(_lib, name)
            fn.restype = res
            fn.argtypes = args
    return _lib


def _ptr(t):
    """Device pointer of a torch tensor, an int address, or None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    assert t.is_cuda and t.is_contiguous(), "device tensors must be contiguous CUDA tensors"
    return t.data_ptr()


@functools.cache
def _dtype_codes() -> dict:
    import torch
    return {torch.float32: FLOAT, torch.float16: FLOAT16, torch.uint8: UINT8, torch.int8: INT8,
            torch.int32: INT32, torch.int64: INT64}


def _dtype_code(t) -> int:
    return _dtype_codes()[t.dtype]


class Context:
    """One device, one in-order stream (VkContext, crates/vk-compute/src/context.rs:257)."""

    def __init__(self, device: int = 0, stream: int | None = None):
        import torch
        if not torch.cuda.is_available():
            raise OvkError(BACKEND, "no CUDA device: the quantized-matmul path has no CPU fallback")
        h = _P()
        if stream is None:
            # share torch's current stream so torch allocations, copies and
            # CUDA events are ordered with the kernels
            with torch.cuda.device(device):
                stream = torch.cuda.current_stream().cuda_stream
            if stream == 0:
                stream = 1  # cudaStreamLegacy: the default stream by its explicit handle
        rc = lib().ovk_ctx_create(device, _P(stream) if stream else None, C.byref(h))
        if rc:
            raise OvkError(rc, lib().ovk_last_error(None).decode())
        self.h = h
        self.device = device
        self._stream = lib().ovk_stream(h)
        self._fast = _packed_calls()

    def check(self, rc: int):
        if rc:
            raise OvkError(rc, lib().ovk_last_error(self.h).decode())

    def close(self):
        if getattr(self, "h", None):
            lib().ovk_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def flush(self):
        self.check(lib().ovk_flush(self.h))

    @property
    def last_kernel(self) -> str:
        return lib().ovk_last_kernel(self.h).decode()

    @property
    def launches(self) -> int:
        return int(lib().ovk_launch_count(self.h))

    @property
    def workspace_bytes(self) -> int:
        return int(lib().ovk_workspace_bytes(self.h))

    def probe_mma_rate(self, dtype=INT8) -> float:
        """Multiply-accumulates per clock per SM of back-to-back tcgen05.mma (kind::i8 or kind::f16)."""
        v = C.c_double()
        self.check(lib().ovk_probe_mma_rate(self.h, dtype, C.byref(v)))
        return v.value

    def selftest_device_timeout(self):
        """Enqueues the wait that is meant to run out; the next flush raises with status TIMEOUT."""
        self.check(lib().ovk_selftest_device_timeout(self.h))

    # ---------------------------------------------------------- MatMulNBits
    def nbits_prepack(self, b, scales, zero_points, n, k, block_size, bits=4, flags=0):
        return NBitsWeight(self, b, scales, zero_points, n, k, block_size, bits, flags)

    def matmul_nbits(self, w: "NBitsWeight", a, out=None, out_dtype=None):
        import torch
        m = a.numel() // w.k
        if a.numel() != m * w.k or (a.dim() and a.shape[-1] != w.k):
            raise OvkError(INVALID_ARGUMENT, f"MatMulNBits: A's last dimension {tuple(a.shape)} disagrees with K={w.k}")
        if out is None:
            out = torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=out_dtype or a.dtype, device=a.device)
        self.check(lib().ovk_matmul_nbits(self.h, w.h, _ptr(a), _dtype_code(a), m, _ptr(out), _dtype_code(out)))
        return out

    def matmul_nbits_group(self, ws, a, outs=None, out_dtype=None):
        """Several weights over the same activations (q|k|v, gate|up): one launch where the decode kernel
        applies and the weights share their tile shape, one call per weight otherwise."""
        import torch
        m = a.numel() // ws[0].k
        if outs is None:
            outs = [torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=out_dtype or a.dtype, device=a.device) for w in ws]
        wp = (_P * len(ws))(*[w.h for w in ws])
        yp = (_P * len(ws))(*[_ptr(o) for o in outs])
        self.check(lib().ovk_matmul_nbits_group(self.h, len(ws), wp, _ptr(a), _dtype_code(a), m, yp, _dtype_code(outs[0])))
        return outs

    # --------------------------------------------- several GPUs of one box
    def comm_alloc(self, nbytes: int) -> int:
        """A zero-filled device buffer that other ranks may map (ovk_comm_alloc); returns its address."""
        p = _P()
        self.check(lib().ovk_comm_alloc(self.h, nbytes, C.byref(p)))
        return p.value

    def comm_export(self, ptr: int) -> bytes:
        buf = C.create_string_buffer(COMM_HANDLE_BYTES)
        self.check(lib().ovk_comm_export(self.h, _P(ptr), buf))
        return buf.raw

    def comm_import(self, handle: bytes) -> int:
        p = _P()
        self.check(lib().ovk_comm_import(self.h, C.c_char_p(handle), C.byref(p)))
        return p.value

    def comm_release(self, ptr: int):
        self.check(lib().ovk_comm_release(self.h, _P(ptr)))

    def comm_init(self, rank: int, world: int, flag_blocks):
        arr = (_P * world)(*[int(b) for b in flag_blocks])
        self.check(lib().ovk_comm_init(self.h, rank, world, arr))
        self.rank, self.world = rank, world

    def comm_set_timeout_ms(self, ms: int):
        self.check(lib().ovk_comm_set_timeout_ms(self.h, int(ms)))

    def comm_barrier(self):
        self.check(lib().ovk_comm_barrier(self.h))

    def allgather_cols(self, y_shard, m, n_shard, col0, n_total, y_peers, dtype=FLOAT16, multicast=None):
        """y_shard: a [m, n_shard] tensor, or None when the block already sits in this rank's matrix.
        multicast: a multicast mapping of the ranks' matrices (one store reaches every rank), or None."""
        arr = (_P * len(y_peers))(*[int(p) for p in y_peers])
        self.check(lib().ovk_allgather_cols_multicast(self.h, _ptr(y_shard),
                                                      dtype if y_shard is None else _dtype_code(y_shard),
                                                      m, n_shard, col0, n_total, arr, _P(multicast) if multicast else None))

    def matmul_nbits_nsplit(self, w: "NBitsWeight", a, col0, n_total, y_peers, y_dtype=FLOAT16, multicast=None):
        """This rank's columns [col0, col0 + w.n) of Y = A x dequant(B), stored into every rank's matrix."""
        m = a.numel() // w.k
        arr = (_P * len(y_peers))(*[int(p) for p in y_peers])
        self.check(lib().ovk_matmul_nbits_nsplit_multicast(self.h, w.h, _ptr(a), _dtype_code(a), m, col0, n_total, arr,
                                                           _P(multicast) if multicast else None, y_dtype))

    # ------------------------------------------------- DynamicQuantizeLinear
    def dynamic_quantize(self, x, folded_range=None, out=None):
        """interp::dynamic_quantize (interp.rs:1945).  `folded_range`: the four-u32 slot the producer of x
        folded its range into (then only the quantize pass runs); `out`: (y, scale, zp) tensors to reuse."""
        import torch
        if out is None:
            out = (torch.empty(x.shape, dtype=torch.uint8, device=x.device),
                   torch.empty((), dtype=torch.float32, device=x.device),
                   torch.empty((), dtype=torch.uint8, device=x.device))
        y, scale, zp = out
        if folded_range is None:
            self.check(lib().ovk_dynamic_quantize(self.h, _ptr(x), x.numel(), _ptr(y), _ptr(scale), _ptr(zp)))
        else:
            self.check(lib().ovk_dynamic_quantize_folded(self.h, _ptr(x), x.numel(), _ptr(folded_range), _ptr(y),
                                                         _ptr(scale), _ptr(zp)))
        return y, scale, zp

    def decomposed_gelu(self, x, divisor, offset, factor, factor_first=False):
        """interp::decomposed_gelu (interp.rs:9060): erf(x / divisor) + offset, times x and factor."""
        import torch
        out = torch.empty_like(x)
        self.check(lib().ovk_decomposed_gelu(self.h, _ptr(x), x.numel(), float(divisor), float(offset), float(factor),
                                             int(factor_first), _ptr(out)))
        return out

    def decomposed_gelu_quantize(self, x, divisor, offset, factor, factor_first=False):
        """interp::decomposed_gelu_quantize (interp.rs:9125): DynamicQuantizeLinear of the GELU, which is never stored."""
        import torch
        y = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
        scale = torch.empty((), dtype=torch.float32, device=x.device)
        zp = torch.empty((), dtype=torch.uint8, device=x.device)
        self.check(lib().ovk_decomposed_gelu_quantize(self.h, _ptr(x), x.numel(), float(divisor), float(offset),
                                                      float(factor), int(factor_first), _ptr(y), _ptr(scale), _ptr(zp)))
        return y, scale, zp

    # --------------------------------------------------------- MatMulInteger
    def mmi_prepack(self, b):
        return MmiWeight(self, b)

    def matmul_integer(self, w: "MmiWeight", a, a_zp=None, b_zp=None):
        import torch
        m = a.numel() // max(w.k, 1)
        out = torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.int32, device=a.device)
        self.check(lib().ovk_matmul_integer(self.h, w.h, _ptr(a), int(a.dtype == torch.int8), m,
                                            _ptr(a_zp), _ptr(b_zp), _ptr(out)))
        return out

    def matmul_integer_static_scratch(self, w: "MmiWeight", a, a_zp=None, b_zp=None, out=None):
        """MatMulInteger through the entry point that allocates nothing: for hosts
        that own all device memory themselves.  `out` must be supplied by such a
        caller; it is created here only as a convenience for tests."""
        import torch
        m = a.numel() // max(w.k, 1)
        if out is None:
            out = torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.int32, device=a.device)
        self.check(lib().ovk_matmul_integer_static_scratch(self.h, w.h, _ptr(a), int(a.dtype == torch.int8), m,
                                                           _ptr(a_zp), _ptr(b_zp), _ptr(out)))
        return out

    def matmul_integer_scale_bias(self, w: "MmiWeight", a, a_zp, b_zp, scale, bias, product=None,
                                  relu=False, range_slot=None):
        import torch
        m = a.numel() // max(w.k, 1)
        out = torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.float32, device=a.device)
        step = lambda t: 0 if t is None or t.numel() == 1 else (1 if t.numel() == w.n and t.shape[-1] == w.n else 2)
        flags = (EPILOGUE_RELU if relu else 0) | (EPILOGUE_RANGE if range_slot is not None else 0)
        self.check(lib().ovk_matmul_integer_scale_bias(
            self.h, w.h, _ptr(a), int(a.dtype == torch.int8), m, _ptr(a_zp), _ptr(b_zp),
            _ptr(scale), step(scale), _ptr(product), step(product), _ptr(bias), step(bias), flags,
            _ptr(range_slot), _ptr(out)))
        return out

    def matmul_integer_group(self, ws, a, a_zp=None, b_zp=None):
        """Several weights over the same A (q | k | v): one launch where the tensor-core tiles apply."""
        import torch
        m = a.numel() // max(ws[0].k, 1)
        outs = [torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.int32, device=a.device) for w in ws]
        wp, op = (_P * len(ws))(*[w.h for w in ws]), (_P * len(ws))(*[_ptr(o) for o in outs])
        self.check(lib().ovk_matmul_integer_group(self.h, len(ws), wp, _ptr(a), int(a.dtype == torch.int8), m, _ptr(a_zp),
                                                  _ptr(b_zp), op))
        return outs

    def matmul_integer_scale_bias_group(self, ws, a, a_zp, b_zp, scales, biases, product=None, relu=False):
        """The fused Cast, Mul, Add [, Relu] epilogue for several weights over the same A; scales[j] / biases[j]
        are member j's, all of one value or all of one per column; `product` is one value."""
        import torch
        m = a.numel() // max(ws[0].k, 1)
        outs = [torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.float32, device=a.device) for w in ws]
        n = len(ws)
        step = lambda ts: 0 if all(t.numel() == 1 for t in ts) else (1 if all(t.numel() == w.n for t, w in zip(ts, ws)) else 2)
        arr = lambda ts: (_P * n)(*[_ptr(t) for t in ts])
        self.check(lib().ovk_matmul_integer_scale_bias_group(
            self.h, n, (_P * n)(*[w.h for w in ws]), _ptr(a), int(a.dtype == torch.int8), m, _ptr(a_zp), _ptr(b_zp),
            arr(scales), step(scales), _ptr(product), 0, arr(biases), step(biases), EPILOGUE_RELU if relu else 0, arr(outs)))
        return outs

    def qlinear_matmul(self, w: "MmiWeight", a, a_zp, b_zp, ratio, y_zp, y_signed=False):
        import torch
        m = a.numel() // max(w.k, 1)
        out = torch.empty(tuple(a.shape[:-1]) + (w.n,), dtype=torch.int8 if y_signed else torch.uint8,
                          device=a.device)
        self.check(lib().ovk_qlinear_matmul(self.h, w.h, _ptr(a), int(a.dtype == torch.int8), m,
                                            _ptr(a_zp), _ptr(b_zp), _ptr(ratio), ratio.numel(),
                                            int(y_zp), int(y_signed), _ptr(out)))
        return out

    # ------------------------------------------- ConvInteger / QLinearConv
    def qconv_prepack(self, w, group=1):
        return QConvWeight(self, w, group)

    @staticmethod
    def _conv_params(x, pads, strides, dilations) -> ConvParams:
        n, c, h, wd = x.shape
        return ConvParams(n, c, h, wd, (C.c_int64 * 4)(*pads), (C.c_int64 * 2)(*strides),
                          (C.c_int64 * 2)(*dilations))

    def conv_output_shape(self, w: "QConvWeight", x, pads, strides, dilations):
        p = self._conv_params(x, pads, strides, dilations)
        ho, wo = _I64(), _I64()
        rc = lib().ovk_conv_output_shape(w.h, C.byref(p), C.byref(ho), C.byref(wo))
        if rc:
            raise OvkError(rc, "Conv: degenerate output shape")
        return ho.value, wo.value

    def conv_integer(self, w: "QConvWeight", x, x_zp=0, w_zp=0, pads=(0, 0, 0, 0), strides=(1, 1),
                     dilations=(1, 1)):
        import torch
        ho, wo = self.conv_output_shape(w, x, pads, strides, dilations)
        out = torch.empty((x.shape[0], w.c_out, ho, wo), dtype=torch.int32, device=x.device)
        p = self._conv_params(x, pads, strides, dilations)
        self.check(lib().ovk_conv_integer(self.h, w.h, _ptr(x), int(x.dtype == torch.int8), C.byref(p),
                                          int(x_zp), int(w_zp), _ptr(out)))
        return out

    def conv_integer_scale_bias(self, w: "QConvWeight", x, x_zp, w_zp, scale, bias, product=None, relu=False,
                                range_slot=None, pads=(0, 0, 0, 0), strides=(1, 1), dilations=(1, 1)):
        """scale, bias, product: float32 device tensors of 1 or C_out values."""
        import torch
        ho, wo = self.conv_output_shape(w, x, pads, strides, dilations)
        out = torch.empty((x.shape[0], w.c_out, ho, wo), dtype=torch.float32, device=x.device)
        p = self._conv_params(x, pads, strides, dilations)
        step = lambda t: 0 if t is None or t.numel() == 1 else (1 if t.numel() == w.c_out else 2)
        flags = (EPILOGUE_RELU if relu else 0) | (EPILOGUE_RANGE if range_slot is not None else 0)
        self.check(lib().ovk_conv_integer_scale_bias(
            self.h, w.h, _ptr(x), int(x.dtype == torch.int8), C.byref(p), int(x_zp), int(w_zp),
            _ptr(scale), step(scale), _ptr(product), step(product), _ptr(bias), step(bias), flags,
            _ptr(range_slot), _ptr(out)))
        return out

    def qlinear_conv(self, w: "QConvWeight", x, x_zp, w_zp, ratio, bias, y_zp, y_signed=False,
                     pads=(0, 0, 0, 0), strides=(1, 1), dilations=(1, 1), out=None):
        """ratio: host float32 array of C_out values, (x_scale*w_scale[c])/y_scale."""
        import numpy as np
        import torch
        ho, wo = self.conv_output_shape(w, x, pads, strides, dilations)
        if out is None:
            out = torch.empty((x.shape[0], w.c_out, ho, wo), dtype=torch.int8 if y_signed else torch.uint8,
                              device=x.device)
        ratio = np.ascontiguousarray(ratio, dtype=np.float32)
        if ratio.size == 1:
            ratio = np.repeat(ratio, w.c_out)
        assert ratio.size == w.c_out
        p = self._conv_params(x, pads, strides, dilations)
        self.check(lib().ovk_qlinear_conv(self.h, w.h, _ptr(x), int(x.dtype == torch.int8), C.byref(p),
                                          int(x_zp), int(w_zp), ratio.ctypes.data, _ptr(bias),
                                          int(y_zp), int(y_signed), _ptr(out)))
        return out

    def to_padded_nhwc(self, x, pads, fill, out=None):
        """NCHW u8/i8 -> [n][h + top + bottom][w + left + right][c], the frame set to `fill`; pads = (top, left,
        bottom, right)."""
        import torch
        n, c, h, w = x.shape
        if out is None:
            out = torch.empty((n, h + pads[0] + pads[2], w + pads[1] + pads[3], c), dtype=x.dtype, device=x.device)
        self.check(lib().ovk_nchw_to_padded_nhwc(self.h, _ptr(x.contiguous()), n, c, h, w, (_I64 * 4)(*pads),
                                                 int(fill) & 0xff, _ptr(out)))
        return out

    def from_padded_nhwc(self, xp, pads):
        import torch
        n, hp, wp, c = xp.shape
        h, w = hp - pads[0] - pads[2], wp - pads[1] - pads[3]
        out = torch.empty((n, c, h, w), dtype=xp.dtype, device=xp.device)
        self.check(lib().ovk_padded_nhwc_to_nchw(self.h, _ptr(xp), n, c, h, w, (_I64 * 4)(*pads), _ptr(out)))
        return out

    def qlinear_conv_channels_last(self, w: "QConvWeight", x, x_zp, w_zp, ratio, bias, y_zp, out, out_pads=None,
                                   y_signed=False, pads=(0, 0, 0, 0), dilations=(1, 1), x_nchw=False, strides=(1, 1)):
        """QLinearConv from a padded-NHWC x (frame = `pads`, holding x_zp; or NCHW with x_nchw=True) into the
        interior of the padded-NHWC `out` whose frame is `out_pads` (None: `out` is NCHW)."""
        import numpy as np
        import torch
        if x_nchw:
            n, c, h, wd = x.shape
        else:
            n, hp, wp, c = x.shape
            h, wd = hp - pads[0] - pads[2], wp - pads[1] - pads[3]
        ratio = np.ascontiguousarray(ratio, dtype=np.float32)
        if ratio.size == 1:
            ratio = np.repeat(ratio, w.c_out)
        p = ConvParams(n, c, h, wd, (C.c_int64 * 4)(*pads), (C.c_int64 * 2)(*strides), (C.c_int64 * 2)(*dilations))
        self.check(lib().ovk_qlinear_conv_layout(self.h, w.h, _ptr(x), int(x.dtype == torch.int8), 0 if x_nchw else 1,
                                                 C.byref(p), int(x_zp), int(w_zp), ratio.ctypes.data, _ptr(bias),
                                                 int(y_zp), int(y_signed), _ptr(out), 0 if out_pads is None else 1,
                                                 None if out_pads is None else (_I64 * 4)(*out_pads)))
        return out

    def requantize(self, acc, inner, ratio, y_zp, bias=None, y_signed=False):
        import torch
        out = torch.empty(acc.shape, dtype=torch.int8 if y_signed else torch.uint8, device=acc.device)
        self.check(lib().ovk_requantize(self.h, _ptr(acc), acc.numel(), int(inner), ratio.numel(),
                                        _ptr(bias), _ptr(ratio), int(y_zp), int(y_signed), _ptr(out)))
        return out

    # ------------------------------------- neighbours of the lm_head product
    def gather_block_quantized(self, table, indices, scales, zero_points, block_size, out_dtype=None, out=None):
        """interp::gather_block_quantized (interp.rs:2874).  `indices`: a torch CUDA tensor (read on the
        device), or a CPU tensor / numpy array / list (checked on the host first, as the reference does)."""
        import torch
        if len(table.shape) != 2 and (len(table.shape) < 2 or any(n != 1 for n in table.shape[2:])):
            raise OvkError(INVALID_ARGUMENT, f"GatherBlockQuantized: a table of [rows, bytes] is needed, not {list(table.shape)}")
        rows, half = table.shape[:2]
        cols = half * 2
        on_host = not (isinstance(indices, torch.Tensor) and indices.is_cuda)
        if on_host:
            import numpy as np
            idx = np.ascontiguousarray(np.asarray(indices, dtype=np.int64))
            shape, count, ptr, code = idx.shape, idx.size, idx.ctypes.data, INT64
        else:
            idx = indices if indices.is_contiguous() else indices.contiguous()
            shape, count, ptr, code = idx.shape, idx.numel(), idx.data_ptr(), _dtype_code(idx)
        if out is None:
            out = torch.empty((*shape, cols), dtype=out_dtype or torch.float32, device=table.device)
        self.check(lib().ovk_gather_block_quantized(self.h, _ptr(table), _ptr(scales), _dtype_code(scales),
                                                    _ptr(zero_points), rows, cols, 4, int(block_size), ptr, code,
                                                    1 if on_host else 0, count, _ptr(out), _dtype_code(out)))
        return out

    def argmax(self, x, axis=-1, out=None):
        """interp::arg_extreme_axis (interp.rs:8552): first-occurrence ArgMax over `axis`, int64, on the device."""
        import math
        import torch
        axis = axis % x.dim()
        outer, c, inner = math.prod(x.shape[:axis]), x.shape[axis], math.prod(x.shape[axis + 1:])
        if out is None:
            out = torch.empty(tuple(x.shape[:axis]) + tuple(x.shape[axis + 1:]), dtype=torch.int64, device=x.device)
        self.check(lib().ovk_argmax(self.h, _ptr(x), _dtype_code(x), outer, c, inner, _ptr(out)))
        return out

    # -------------------------------------------- the attention of a decoder layer
    # A decode step makes a few of these calls per layer, each a few microseconds of GPU time, so the wrappers check with
    # few attribute reads and hand the C structs over as packed bytes.
    def _activation(self, what, t, tokens=None, heads=None, head_dim=None, dtype=None):
        """(data, heads, token stride, head stride) of a [tokens, heads, head_dim] tensor whose heads are contiguous; a slice
        of a wider one will do."""
        try:
            n, h, d = t.shape
            st, sh, sd = t.stride()
            if ((sd == 1 or d == 1) and t.get_device() == self.device and t.dtype in _activation_codes()
                    and (tokens is None or n == tokens) and (heads is None or h == heads) and (head_dim is None or d == head_dim)
                    and (dtype is None or t.dtype is dtype)):
                return t.data_ptr(), h, st, sh
        except (AttributeError, TypeError, ValueError):
            pass
        got = f"{list(t.shape)} of {t.dtype} on {t.device} with strides {t.stride()}" if hasattr(t, "stride") else f"{type(t).__name__}"
        raise OvkError(INVALID_ARGUMENT, f"{what}: [{tokens if tokens is not None else 'tokens'}, {heads or 'heads'}, {head_dim or 'head_dim'}] of "
                                         f"{dtype or 'float32 or float16'} on cuda:{self.device} with contiguous heads is needed, not {got}")

    def _indices(self, what, t, shape, dtypes):
        try:
            if t.shape == shape and t.dtype in dtypes and t.is_contiguous() and t.get_device() == self.device:
                return t.data_ptr()
        except AttributeError:
            pass
        got = f"{list(t.shape)} of {t.dtype} on {t.device}" if hasattr(t, "stride") else f"{type(t).__name__}"
        raise OvkError(INVALID_ARGUMENT, f"{what}: a contiguous {list(shape)} tensor of {' or '.join(str(d) for d in dtypes)} on "
                                         f"cuda:{self.device} is needed, not {got}")

    def _foreign_stream(self):
        """None where torch's current stream is this context's, else the latter as a torch stream."""
        if (_raw_stream()(self.device) or 1) == self._stream:
            return None
        import torch
        if self._stream == 1:  # the default stream's handle is not one that torch takes
            return torch.cuda.default_stream(self.device)
        return torch.cuda.ExternalStream(self._stream, device=torch.device("cuda", self.device))

    @staticmethod
    def _new(like, stream):
        """A contiguous tensor of this shape and type, from the pool of the stream that will write it."""
        import torch
        if stream is None:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        with torch.cuda.stream(stream):
            return torch.empty_like(like, memory_format=torch.contiguous_format)

    @staticmethod
    def _keep(stream, *used):
        """Tensors that a call on another stream reads or writes are not reused before it has passed them."""
        if stream is not None:
            for t in used:
                if t is not None:
                    t.record_stream(stream)

    def rotary(self, q, cos, sin, positions, k=None, sections=None, interleaved=False, out=None, k_out=None):
        """Rotary positions of q (and k) [tokens, heads, head_dim]: cos and sin are [positions, rotary_dim / 2] tables,
        positions [tokens] or [axes, tokens], sections the pairs of each axis.  Returns q (and k) turned; out may be q."""
        x = self._activation("Rotary: q", q)
        n, h, d = q.shape
        kind = q.dtype
        try:
            rows, pairs = cos.shape
            flat = positions.dim() == 1
            axes = 1 if flat else positions.shape[0]
        except (AttributeError, ValueError, IndexError, TypeError):
            _dims("Rotary: cos", cos, 2)
            _dims("Rotary: positions", positions, 1, 2)
            raise
        codes = _activation_codes()
        at = self._indices("Rotary: positions", positions, (n,) if flat else (axes, n), _index_codes())
        c = self._indices("Rotary: cos", cos, (rows, pairs), codes)
        s = self._indices("Rotary: sin", sin, (rows, pairs), (cos.dtype,))
        if sections is None:
            sections = (pairs,)
        try:
            if len(sections) != axes or axes > 4:
                raise OvkError(INVALID_ARGUMENT, f"Rotary: {len(sections)} sections for {axes} axes (1 to 4)")
            p = _PACK_ROTARY(n, d, 2 * pairs, rows, codes[kind], codes[cos.dtype], _index_codes()[positions.dtype], 1 if interleaved else 0, axes,
                             *sections, *(0,) * (4 - axes))
        except (TypeError, struct.error):
            if not hasattr(sections, "__len__"):
                raise OvkError(INVALID_ARGUMENT, f"Rotary: sections are pairs per axis, not {sections!r}") from None
            for v in sections:
                _whole("Rotary: sections", v, 2 ** 31 - 1)
            raise
        stream = self._foreign_stream()
        if k is not None:
            x += self._activation("Rotary: k", k, n, None, d, kind)
            if k_out is None:
                k_out = self._new(k, stream)
                y_k = (k_out.data_ptr(), x[5], x[5] * d, d)
            else:
                y_k = self._activation("Rotary: k_out", k_out, n, x[5], d, kind)
        if out is None:
            out = self._new(q, stream)
            y = (out.data_ptr(), h, h * d, d)
        else:
            y = self._activation("Rotary: out", out, n, h, d, kind)
        self._keep(stream, q, k, cos, sin, positions, out, k_out)
        if k is None:
            self.check(self._fast.ovk_rotary(self.h, p, 1, _PACK_HEADS(*x), _PACK_HEADS(*y), at, c, s))
            return out
        self.check(self._fast.ovk_rotary(self.h, p, 2, _PACK_HEADS2(*x), _PACK_HEADS2(*y, *y_k), at, c, s))
        return out, k_out

    def kv4_cache(self, pages, kv_heads, page_size, head_dim, block_size=32, zero_points=True):
        """An empty paged 4-bit cache; with pages = batch and a block table of one column, a [batch, kv_heads, capacity] one."""
        import torch
        pages, kv_heads, page_size, head_dim, block_size = (
            _whole("KV4Cache: " + name, v) for name, v in (("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size), ("head_dim", head_dim),
                                                          ("block_size", block_size)))
        if min(pages, kv_heads, page_size, head_dim) < 0 or block_size < 1:
            raise OvkError(INVALID_ARGUMENT, f"KV4Cache: {pages} pages of {kv_heads} heads x {page_size} places x {head_dim} in blocks of {block_size}")
        blocks = head_dim // block_size
        zeros = lambda last, dtype: torch.zeros((pages, kv_heads, page_size, last), dtype=dtype, device=torch.device("cuda", self.device))  # noqa: E731

        def make():
            code = [zeros(head_dim // 2, torch.uint8) for _ in range(2)]
            scale = [zeros(blocks, torch.float16) for _ in range(2)]
            zero = [zeros((blocks + 1) // 2, torch.uint8) if zero_points else None for _ in range(2)]
            return KV4Cache(*code, *scale, *zero)
        stream = self._foreign_stream()
        if stream is None:
            return make()
        with torch.cuda.stream(stream):
            return make()

    def _kv4_batch(self, what, cache, tokens, block_table, cu_tokens, lens):
        if cache.device != self.device:
            raise OvkError(INVALID_ARGUMENT, f"{what}: the cache is on cuda:{cache.device}, the context on cuda:{self.device}")
        try:
            batch, pages = lens.shape[0], block_table.shape[1]
        except (AttributeError, IndexError):
            _dims(what + ": lens", lens, 1)
            _dims(what + ": block_table", block_table, 2)
            raise
        i32 = _int32()
        return _PACK_BATCH(tokens, batch, pages, self._indices(what + ": cu_tokens", cu_tokens, (batch + 1,), i32),
                           self._indices(what + ": lens", lens, (batch,), i32),
                           self._indices(what + ": block_table", block_table, (batch, pages), i32))

    def kv4_append(self, cache: "KV4Cache", k, v, block_table, cu_tokens, lens):
        """Rounds the new tokens' keys and values [tokens, kv_heads, head_dim] to 4 bits and writes them: sequence b brings rows
        cu_tokens[b] .. cu_tokens[b + 1] - 1, the last of its lens[b] positions; block_table is [batch, max_pages]."""
        if not isinstance(cache, KV4Cache):
            raise OvkError(INVALID_ARGUMENT, f"KV4Append: a KV4Cache is needed, not {type(cache).__name__}")
        hk = self._activation("KV4Append: k", k, None, cache.kv_heads, cache.head_dim)
        n = k.shape[0]
        hv = self._activation("KV4Append: v", v, n, cache.kv_heads, cache.head_dim, k.dtype)
        b = self._kv4_batch("KV4Append", cache, n, block_table, cu_tokens, lens)
        stream = self._foreign_stream()
        if stream is not None:
            self._keep(stream, k, v, block_table, cu_tokens, lens, *cache.tensors)
        self.check(self._fast.ovk_kv4_append(self.h, cache.packed, b, _PACK_HEADS(*hk), _PACK_HEADS(*hv), _activation_codes()[k.dtype]))

    def attention_kv4(self, cache: "KV4Cache", q, block_table, cu_tokens, lens, max_tokens=1, scale=None, window=0, out=None):
        """Causal attention of the new tokens q [tokens, q_heads, head_dim] over the cache, which holds their own rows already.
        max_tokens: the most new tokens a sequence is expected to bring (it chooses how many rows are computed together;
        results hold for any number); scale: 1 / sqrt(head_dim) unless given; window: positions a token reads, its own
        included (0: all before it)."""
        if not isinstance(cache, KV4Cache):
            raise OvkError(INVALID_ARGUMENT, f"AttentionKV4: a KV4Cache is needed, not {type(cache).__name__}")
        hq = self._activation("AttentionKV4: q", q, None, None, cache.head_dim)
        n, h, d = q.shape
        b = self._kv4_batch("AttentionKV4", cache, n, block_table, cu_tokens, lens)
        # ctypes takes any int for a 64-bit field
        if not (type(max_tokens) is int is type(window) and 0 <= max_tokens < 1 << 63 and 0 <= window < 1 << 63):
            max_tokens, window = _whole("AttentionKV4: max_tokens", max_tokens), _whole("AttentionKV4: window", window)
        scale = d ** -0.5 if scale is None else _scale("AttentionKV4", scale)
        code = _activation_codes()[q.dtype]
        stream = self._foreign_stream()
        if out is None:
            out = self._new(q, stream)
            ho = (out.data_ptr(), h, h * d, d)
        else:
            ho = self._activation("AttentionKV4: out", out, n, h, d, q.dtype)
        space, need = None, 0
        if stream is not None:
            self._keep(stream, q, block_table, cu_tokens, lens, out, *cache.tensors)
        elif _capturing()():
            # a graph has a workspace of its own (outside of one, calls on the stream follow each other in the context's)
            import torch
            size = _SZ()
            self.check(lib().ovk_attention_kv4_workspace(self.h, cache.params, h, max_tokens, code, C.byref(size)))
            need = size.value
            space = torch.empty(need, dtype=torch.uint8, device=q.device)
            space[:4096].zero_()
        self.check(self._fast.ovk_attention_kv4(self.h, cache.packed, b, _PACK_HEADS(*hq), _PACK_HEADS(*ho), code, max_tokens,
                                                scale, window,
                                                None if space is None else space.data_ptr(), need))
        return out

    def attention_prompt(self, q, k, v, cu_q, max_q=0, cu_k=None, scale=None, causal=True, window=0, out=None):
        """Attention within packed sequences: q [tokens, q_heads, head_dim], k and v [tokens, kv_heads, head_dim], cu_q the
        sequences' first rows.  With cu_k the keys have rows of their own and the queries are the last tokens of the keys'
        sequence.  max_q: the most queries a sequence has, where the caller knows it (0: not known; rows beyond it are
        left out)."""
        hq = self._activation("AttentionPrompt: q", q)
        n, h, d = q.shape
        kind = q.dtype
        hk = self._activation("AttentionPrompt: k", k, None, None, d, kind)
        hv = self._activation("AttentionPrompt: v", v, k.shape[0], k.shape[1], d, kind)
        try:
            batch = cu_q.shape[0] - 1
        except (AttributeError, IndexError):
            _dims("AttentionPrompt: cu_q", cu_q, 1)
            raise
        pq = self._indices("AttentionPrompt: cu_q", cu_q, (max(batch, 0) + 1,), _int32())
        pk = pq if cu_k is None or cu_k is cu_q else self._indices("AttentionPrompt: cu_k", cu_k, (batch + 1,), _int32())
        scale = d ** -0.5 if scale is None else _scale("AttentionPrompt", scale)
        try:
            p = _PACK_PROMPT(n, k.shape[0], batch, d, _activation_codes()[kind], 1 if causal else 0, window, scale, max_q or 0)
        except struct.error:
            _whole("AttentionPrompt: window", window)
            _whole("AttentionPrompt: max_q", max_q, 2 ** 31 - 1)
            raise
        stream = self._foreign_stream()
        if out is None:
            out = self._new(q, stream)
            ho = (out.data_ptr(), h, h * d, d)
        else:
            ho = self._activation("AttentionPrompt: out", out, n, h, d, kind)
        self._keep(stream, q, k, v, cu_q, cu_k, out)
        self.check(self._fast.ovk_attention_prompt(self.h, p, _PACK_HEADS(*hq), _PACK_HEADS(*hk), _PACK_HEADS(*hv), pq, pk, _PACK_HEADS(*ho)))
        return out

    # ------------------------------------ the QOperator chain around QLinearConv
    def qlinear_add(self, a, a_scale, a_zp, b, b_scale, b_zp, c_scale, c_zp):
        """interp::qlinear_add (interp.rs:4878); a and b are u8 or i8 tensors that broadcast."""
        import torch
        shape = torch.broadcast_shapes(a.shape, b.shape)
        out = torch.empty(shape, dtype=a.dtype, device=a.device)
        a, b = a.contiguous(), b.contiguous()
        sa, sb = (_I64 * max(a.dim(), 1))(*a.shape), (_I64 * max(b.dim(), 1))(*b.shape)
        self.check(lib().ovk_qlinear_add(self.h, _ptr(a), sa, a.dim(), float(a_scale), int(a_zp), _ptr(b), sb, b.dim(),
                                         float(b_scale), int(b_zp), float(c_scale), int(c_zp),
                                         int(a.dtype == torch.int8), _ptr(out), None, None))
        return out

    def maxpool_q(self, x, kernel, strides=None, pads=(0, 0, 0, 0), dilations=(1, 1)):
        """MaxPool in the quantized domain (shaders/qlinear.rs:145); x is [N, C, H, W] u8 or i8."""
        import torch
        n, c, h, w = x.shape
        strides = strides or (1, 1)
        arr = lambda v: (_I64 * len(v))(*[int(i) for i in v])
        dil = arr(dilations)
        ho = (h + pads[0] + pads[2] - (dilations[0] * (kernel[0] - 1) + 1)) // strides[0] + 1
        wo = (w + pads[1] + pads[3] - (dilations[1] * (kernel[1] - 1) + 1)) // strides[1] + 1
        out = torch.empty((n, c, max(ho, 0), max(wo, 0)), dtype=x.dtype, device=x.device)
        self.check(lib().ovk_maxpool_q(self.h, _ptr(x.contiguous()), int(x.dtype == torch.int8), n, c, h, w, arr(kernel),
                                       arr(strides), arr(pads), dil, _ptr(out), None, None))
        return out

    @staticmethod
    def _qdq_layout(shape, scale, axis):
        import math
        if scale.numel() <= 1:
            return 1, 1
        axis = axis % len(shape)
        return max(math.prod(shape[axis + 1:]), 1), scale.numel()

    def quantize_linear(self, x, scale, zero_point=None, axis=1, signed=False):
        """interp::quantize_linear (interp.rs:5117): saturate(rne(x / scale) + zero_point)."""
        import torch
        signed = signed if zero_point is None else zero_point.dtype == torch.int8
        inner, axis_len = self._qdq_layout(x.shape, scale, axis)
        out = torch.empty(x.shape, dtype=torch.int8 if signed else torch.uint8, device=x.device)
        self.check(lib().ovk_quantize_linear(self.h, _ptr(x.contiguous()), x.numel(), inner, axis_len, _ptr(scale),
                                             _ptr(zero_point), int(signed), _ptr(out)))
        return out

    def dequantize_linear(self, x, scale, zero_point=None, axis=1):
        """interp::dequantize_linear (interp.rs:5055): (x - zero_point) * scale, u8 / i8 / i32 input."""
        import torch
        inner, axis_len = self._qdq_layout(x.shape, scale, axis)
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        self.check(lib().ovk_dequantize_linear(self.h, _ptr(x.contiguous()), _dtype_code(x), x.numel(), inner, axis_len,
                                               _ptr(scale), _ptr(zero_point), _ptr(out)))
        return out

    def qlinear_global_average_pool(self, x, x_scale, x_zp, y_scale, y_zp):
        """interp::qlinear_global_average_pool (interp.rs:4975); x is [N, C, ...] u8 or i8."""
        import math
        import torch
        n, c = x.shape[0], x.shape[1]
        out = torch.empty((n, c) + (1,) * (x.dim() - 2), dtype=x.dtype, device=x.device)
        self.check(lib().ovk_qlinear_global_average_pool(self.h, _ptr(x.contiguous()), int(x.dtype == torch.int8), n, c,
                                                         math.prod(x.shape[2:]), float(x_scale), int(x_zp),
                                                         float(y_scale), int(y_zp), _ptr(out)))
        return out


class KV4Cache:
    """A paged key / value cache in 4 bits: codes [pages, kv_heads, page_size, head_dim / 2], fp16 scales [..., blocks] and zero
    points [..., ceil(blocks / 2)] (None: implicit 8), rows as ovk_gather_block_quantized reads them."""

    def __init__(self, k, v, k_scales, v_scales, k_zero_points=None, v_zero_points=None):
        import torch
        for t in (k, v, k_scales, v_scales, *(t for t in (k_zero_points, v_zero_points) if t is not None)):
            if not isinstance(t, torch.Tensor):
                raise OvkError(INVALID_ARGUMENT, f"KV4Cache: tensors are needed, not {type(t).__name__}")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.k_zero_points, self.v_zero_points = k_zero_points, v_zero_points
        self.tensors = tuple(t for t in (k, v, k_scales, v_scales, k_zero_points, v_zero_points) if t is not None)
        if (k_zero_points is None) != (v_zero_points is None) or k.dim() != 4 or k_scales.dim() != 4 or k_scales.shape[3] < 1:
            raise OvkError(INVALID_ARGUMENT, "KV4Cache: four-dimensional tensors, with zero points for both or for neither")
        pages, heads, size, half = k.shape
        blocks = k_scales.shape[3]
        for t, last, dtype in ((k, half, torch.uint8), (v, half, torch.uint8), (k_scales, blocks, torch.float16),
                               (v_scales, blocks, torch.float16), (k_zero_points, (blocks + 1) // 2, torch.uint8),
                               (v_zero_points, (blocks + 1) // 2, torch.uint8)):
            if t is not None and (tuple(t.shape) != (pages, heads, size, last) or t.dtype != dtype or not t.is_cuda
                                  or t.device != k.device or not t.is_contiguous()):
                raise OvkError(INVALID_ARGUMENT, f"KV4Cache: contiguous {[pages, heads, size, last]} of {dtype} on one GPU is needed, "
                                                 f"not {tuple(t.shape)} of {t.dtype} on {t.device}")
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, 2 * half
        if self.head_dim % blocks:
            raise OvkError(INVALID_ARGUMENT, f"KV4Cache: {blocks} scales for {self.head_dim} elements")
        self.block_size = self.head_dim // blocks
        self.device = k.get_device()
        self.params = KV4CacheParams(*[None if t is None else t.data_ptr() for t in (k, v, k_scales, v_scales, k_zero_points, v_zero_points)],
                                     pages, heads, size, self.head_dim, self.block_size)
        self.packed = bytes(self.params)


class NBitsWeight:
    """A MatMulNBits weight prepared once (the role packed_b plays, interp.rs:2712)."""

    def __init__(self, ctx: Context, b, scales, zero_points, n, k, block_size, bits=4, flags=0):
        self.ctx, self.n, self.k, self.block_size = ctx, int(n), int(k), int(block_size)
        self._keep = (b, scales, zero_points)  # the operator-layout buffers must outlive the handle
        h = _P()
        ctx.check(lib().ovk_nbits_prepack(ctx.h, _ptr(b), _ptr(scales), _dtype_code(scales),
                                          _ptr(zero_points), n, k, bits, block_size, flags, C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if self.h and self.ctx.h:
                lib().ovk_nbits_weight_destroy(self.ctx.h, self.h)
        except Exception:
            pass


class MmiWeight:
    """B [K,N] of MatMulInteger in the tensor-core layout (packed_b, interp.rs:2712)."""

    def __init__(self, ctx: Context, b):
        import torch
        assert b.dim() == 2
        self.ctx, self.k, self.n = ctx, int(b.shape[0]), int(b.shape[1])
        self.signed = b.dtype == torch.int8
        h = _P()
        ctx.check(lib().ovk_mmi_prepack(ctx.h, _ptr(b), int(self.signed), self.k, self.n, C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if self.h and self.ctx.h:
                lib().ovk_mmi_weight_destroy(self.ctx.h, self.h)
        except Exception:
            pass


class QConvWeight:
    """A ConvInteger / QLinearConv filter bank [C_out, C_in/group, KH, KW]."""

    def __init__(self, ctx: Context, w, group=1):
        import torch
        if w.dim() == 3:  # 1-D convolution: W = 1
            w = w.unsqueeze(-1)
        self.ctx = ctx
        self.c_out, self.cig, self.kh, self.kw = (int(v) for v in w.shape)
        self.group = int(group)
        h = _P()
        ctx.check(lib().ovk_qconv_prepack(ctx.h, _ptr(w.contiguous()), int(w.dtype == torch.int8),
                                          self.c_out, self.cig, self.kh, self.kw, self.group, C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if self.h and self.ctx.h:
                lib().ovk_qconv_weight_destroy(self.ctx.h, self.h)
        except Exception:
            pass
