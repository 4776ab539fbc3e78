"""ctypes binding of include/abq_b200.h.  Device buffers are torch CUDA tensors (or raw pointers).

There is no fallback: if the shared library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

ROUTE_AUTO, ROUTE_B1_MMA, ROUTE_I8_MMA, ROUTE_I8_UMMA = 0, 1, 2, 3
OUT_INT32, OUT_FP16 = 0, 1
SCALE_NONE, SCALE_TENSOR_COMPAT, SCALE_CHANNEL, SCALE_GROUP = 0, 1, 2, 3
FLAG_PDL = 1
FLAG_WEIGHTS_PREPARED = 2
FLAG_X_HALF = 4

_PKG = Path(__file__).resolve().parent


class AbqError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: abq_status {status} ({_status_string(status)})")


class FusedAllreduce(ctypes.Structure):
    """Mirror of ``abq_fused_allreduce``."""
    _fields_ = [("world", ctypes.c_int), ("rank", ctypes.c_int), ("recv", ctypes.c_void_p * 8), ("flags", ctypes.c_void_p * 8),
                ("counter", ctypes.c_void_p), ("rows_cap", ctypes.c_int)]


class GemmParams(ctypes.Structure):
    """Mirror of ``abq_gemm_params`` (field order is part of the ABI)."""
    _fields_ = [
        ("M", ctypes.c_int), ("N", ctypes.c_int), ("K", ctypes.c_int),
        ("X", ctypes.c_void_p), ("W", ctypes.c_void_p), ("C", ctypes.c_void_p), ("D", ctypes.c_void_p),
        ("bias", ctypes.c_int),
        ("x_bits", ctypes.c_int), ("w_bits", ctypes.c_int),
        ("x_signed", ctypes.c_int), ("w_signed", ctypes.c_int),
        ("out_dtype", ctypes.c_int), ("scale_mode", ctypes.c_int), ("group_size", ctypes.c_int),
        ("w_scale", ctypes.c_void_p), ("w_zero", ctypes.c_void_p), ("x_scale", ctypes.c_void_p),
        ("route", ctypes.c_int), ("flags", ctypes.c_int),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("status_word", ctypes.c_void_p),
        ("x_quant_scale", ctypes.c_void_p),
        ("w_prepared", ctypes.c_void_p),
        ("allreduce", ctypes.POINTER(FusedAllreduce)),
        ("residual", ctypes.c_void_p),
    ]


class GemmState(ctypes.Structure):
    """Mirror of ``abq_gemm_state``."""
    _fields_ = [
        ("p", GemmParams),
        ("init_success", ctypes.c_int), ("route", ctypes.c_int),
        ("grid", ctypes.c_int * 3), ("block", ctypes.c_int * 3), ("cluster", ctypes.c_int),
        ("shared_mem_size", ctypes.c_size_t),
        ("tile", ctypes.c_int * 4),
        ("tmap", (ctypes.c_ulonglong * 16) * 3),
        ("ar", FusedAllreduce),
    ]


HALF_FP16, HALF_BF16 = 0, 1
STATUS_BAD_PAGE = 16


class KVCache(ctypes.Structure):
    """Mirror of ``abq_kv_cache``."""
    _fields_ = [("data", ctypes.c_void_p), ("num_pages", ctypes.c_int), ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("bits", ctypes.c_int), ("half_type", ctypes.c_int)]


_KV_STRIDES = [(n, ctypes.c_longlong) for n in ("k_stride", "k_head_stride", "v_stride", "v_head_stride")]


class KVWriteParams(ctypes.Structure):
    """Mirror of ``abq_kv_write_params``."""
    _fields_ = [("cache", KVCache), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), *_KV_STRIDES, ("slots", ctypes.c_void_p), ("tokens", ctypes.c_int)]


class KVReadParams(ctypes.Structure):
    """Mirror of ``abq_kv_read_params``."""
    _fields_ = [("cache", KVCache), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), *_KV_STRIDES, ("rows", ctypes.c_int), ("batch", ctypes.c_int),
                ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int), ("cu_seqlens", ctypes.c_void_p)]


class CacheAttentionParams(ctypes.Structure):
    """Mirror of ``abq_cache_attention_params``."""
    _fields_ = [("cache", KVCache), ("q", ctypes.c_void_p), ("out", ctypes.c_void_p),
                *[(n, ctypes.c_longlong) for n in ("q_stride", "q_head_stride", "out_stride", "out_head_stride")],
                ("batch", ctypes.c_int), ("rows_per_seq", ctypes.c_int), ("q_heads", ctypes.c_int), ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int),
                ("seq_lens", ctypes.c_void_p), ("tree", ctypes.c_void_p), ("scale", ctypes.c_float), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_size_t), ("status_word", ctypes.c_void_p)]


class PromptAttentionParams(ctypes.Structure):
    """Mirror of ``abq_prompt_attention_params``."""
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("out", ctypes.c_void_p),
                *[(n + s, ctypes.c_longlong) for n in ("q", "k", "v", "out") for s in ("_stride", "_head_stride")],
                ("total_q", ctypes.c_int), ("total_k", ctypes.c_int), ("q_heads", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("half_type", ctypes.c_int), ("batch", ctypes.c_int), ("cu_q", ctypes.c_void_p), ("cu_k", ctypes.c_void_p), ("max_q", ctypes.c_int),
                ("scale", ctypes.c_float), ("status_word", ctypes.c_void_p)]


_lib = None


def lib_path() -> Path:
    return _PKG / "lib" / "libabq_b200.so"


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        path = lib_path()
        if not path.exists():
            raise FileNotFoundError(f"{path} is missing: run `python abq-llm_b200/build.py` (no fallback exists)")
        L = ctypes.CDLL(str(path))
        L.abq_version.restype = ctypes.c_char_p
        L.abq_status_string.restype = ctypes.c_char_p
        L.abq_status_string.argtypes = [ctypes.c_int]
        L.abq_last_cuda_error.restype = ctypes.c_int
        L.abq_gemm_workspace_bytes.restype = ctypes.c_size_t
        L.abq_gemm_workspace_bytes.argtypes = [ctypes.c_int] * 6
        L.abq_gemm_prepared_weight_bytes.restype = ctypes.c_size_t
        L.abq_gemm_prepared_weight_bytes.argtypes = [ctypes.POINTER(GemmParams)]
        L.abq_gemm_init.argtypes = [ctypes.POINTER(GemmParams), ctypes.POINTER(GemmState)]
        L.abq_gemm_exec.argtypes = [ctypes.POINTER(GemmState), ctypes.c_void_p]
        L.abq_gemm_prepare_weights.argtypes = [ctypes.POINTER(GemmState), ctypes.c_void_p]
        L.abq_gemm.argtypes = [ctypes.POINTER(GemmParams), ctypes.c_void_p]
        L.abq_gemm_static_scratch.argtypes = [ctypes.POINTER(GemmParams), ctypes.c_void_p]
        L.abq_pack_int32.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
        L.abq_pack_int4.argtypes = L.abq_pack_int32.argtypes
        L.abq_quantize_pack_half.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                                             ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
        L.abq_quantize_weights_half.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                                                ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        L.abq_swiglu_half.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
        L.abq_add_half.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_long, ctypes.c_void_p]
        L.abq_rmsnorm_quantize_pack_half.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_float] + [ctypes.c_void_p] * 4 + [ctypes.c_int] * 4 + [ctypes.c_void_p]
        L.abq_unpack_int8.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                      ctypes.c_void_p]
        L.abq_kv_cache_bytes.restype = ctypes.c_size_t
        L.abq_kv_cache_bytes.argtypes = [ctypes.POINTER(KVCache)]
        L.abq_kv_cache_write.argtypes = [ctypes.POINTER(KVWriteParams), ctypes.c_void_p]
        L.abq_kv_cache_read.argtypes = [ctypes.POINTER(KVReadParams), ctypes.c_void_p]
        L.abq_cache_attention_workspace_bytes.restype = ctypes.c_size_t
        L.abq_cache_attention_workspace_bytes.argtypes = [ctypes.POINTER(KVCache), ctypes.c_int, ctypes.c_int, ctypes.c_int]
        L.abq_cache_attention.argtypes = [ctypes.POINTER(CacheAttentionParams), ctypes.c_void_p]
        L.abq_prompt_attention.argtypes = [ctypes.POINTER(PromptAttentionParams), ctypes.c_void_p]
        _lib = L
    return _lib


def _status_string(s: int) -> str:
    try:
        return lib().abq_status_string(s).decode()
    except Exception:  # library missing: still give a message
        return "?"


def version() -> str:
    return lib().abq_version().decode()


def _ptr(t) -> int | None:
    """Device address of a torch tensor, an int, or None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    assert t.is_cuda and t.is_contiguous(), "device buffers must be contiguous CUDA tensors"
    return t.data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _check(status: int, what: str) -> None:
    if status != 0:
        extra = ""
        if status == 4:
            extra = f" [cudaError {lib().abq_last_cuda_error()}]"
        raise AbqError(status, what + extra)


def gemm_workspace_bytes(M: int, N: int, K: int, x_bits: int, w_bits: int, route: int = ROUTE_AUTO) -> int:
    return int(lib().abq_gemm_workspace_bytes(M, N, K, x_bits, w_bits, route))


def make_params(M, N, K, X, W, D, *, x_bits, w_bits, x_signed, w_signed, out_dtype=OUT_INT32, scale_mode=SCALE_NONE,
                group_size=0, C=None, w_scale=None, w_zero=None, x_scale=None, route=ROUTE_AUTO, flags=0, workspace=None,
                status_word=None, x_quant_scale=None, w_prepared=None, allreduce=None, residual=None) -> GemmParams:
    p = GemmParams()
    p.M, p.N, p.K = M, N, K
    p.X, p.W, p.C, p.D = _ptr(X), _ptr(W), _ptr(C), _ptr(D)
    p.bias = 0
    p.x_bits, p.w_bits, p.x_signed, p.w_signed = x_bits, w_bits, int(x_signed), int(w_signed)
    p.out_dtype, p.scale_mode, p.group_size = out_dtype, scale_mode, group_size
    p.w_scale, p.w_zero, p.x_scale = _ptr(w_scale), _ptr(w_zero), _ptr(x_scale)
    p.route, p.flags = route, flags
    p.workspace = _ptr(workspace)
    p.workspace_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    p.status_word = _ptr(status_word)
    p.x_quant_scale = _ptr(x_quant_scale)
    p.w_prepared = _ptr(w_prepared)
    p.residual = _ptr(residual)
    # the block carries raw pointers: keep the tensors alive as long as it lives (a temporary passed inline would otherwise
    # be freed, and its memory reused, before the launch)
    p._keep_alive = (X, W, D, C, w_scale, w_zero, x_scale, workspace, status_word, x_quant_scale, w_prepared, residual)
    if allreduce is not None:
        p.allreduce = ctypes.pointer(allreduce)
        p._keep_allreduce = allreduce  # the struct must outlive the call that reads it
    return p


def make_fused_allreduce(world: int, rank: int, recv_ptrs, flag_ptrs, counter, rows_cap: int) -> FusedAllreduce:
    """``recv_ptrs`` / ``flag_ptrs``: every rank's receive buffer / flag array as mapped into this process (ints)."""
    d = FusedAllreduce()
    d.world, d.rank, d.rows_cap = world, rank, rows_cap
    for r in range(world):
        d.recv[r] = int(recv_ptrs[r])
        d.flags[r] = int(flag_ptrs[r])
    d.counter = _ptr(counter)
    return d


def gemm_prepared_weight_bytes(params: GemmParams) -> int:
    """Bytes of the re-ordered weight copy a decode-shape plan reads through ``w_prepared`` (0: no prepared form)."""
    return int(lib().abq_gemm_prepared_weight_bytes(ctypes.byref(params)))


def state_kernel(state: GemmState) -> str:
    """Name of the GEMM kernel a plan launches (for reports): the route, and which of the route's kernels."""
    if state.route == ROUTE_I8_MMA:
        return "stream_kernel" if (state.tmap[1][0] & 0xffffffff) == 0x5354524d else "decode_kernel"
    if state.route == ROUTE_I8_UMMA:  # tc_kernel reads the weights as planes, or (codes) as the int8 expansion in the workspace
        return {0: "umma_kernel", 2: "umma2_kernel", 3: "tc_kernel", 4: "tc_kernel (codes)"}.get(state.tile[2], "?")
    return "b1_kernel" if state.route == ROUTE_B1_MMA else "?"


def gemm_init(params: GemmParams) -> GemmState:
    st = GemmState()
    _check(lib().abq_gemm_init(ctypes.byref(params), ctypes.byref(st)), "abq_gemm_init")
    return st


def gemm_exec(state: GemmState, stream=None) -> None:
    _check(lib().abq_gemm_exec(ctypes.byref(state), _stream(stream)), "abq_gemm_exec")


def gemm_prepare_weights(state: GemmState, stream=None) -> None:
    _check(lib().abq_gemm_prepare_weights(ctypes.byref(state), _stream(stream)), "abq_gemm_prepare_weights")


def peer_allreduce_half(bufs_dev: int, signals_dev: int, rank: int, world: int, signal_offset: int, out, n_halves: int, counter,
                        status_word=None, stream=None, residual=None) -> None:
    """One-shot sum over the ranks' partial buffers (peer-mapped pointers, see abq_peer_allreduce_half), plus ``residual``."""
    f = lib().abq_peer_allreduce_half
    f.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_long, ctypes.c_void_p,
                  ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    _check(f(bufs_dev, signals_dev, rank, world, signal_offset, _ptr(out), n_halves, _ptr(counter), _ptr(status_word), _ptr(residual),
             _stream(stream)), "abq_peer_allreduce_half")


def gemm(params: GemmParams, stream=None) -> None:
    _check(lib().abq_gemm(ctypes.byref(params), _stream(stream)), "abq_gemm")


STATIC_SCRATCH_BYTES = 16 << 20
WORKSPACE_COUNTER_BYTES = 256 << 10


def workspace_sharing_bytes(M: int, N: int, K: int, route: int = ROUTE_AUTO) -> int:
    """The part of gemm_workspace_bytes() that only plans sharing a workspace need (abq_workspace_sharing_bytes in the header)."""
    umma = route == ROUTE_I8_UMMA or (route == ROUTE_AUTO and M > 16)
    return WORKSPACE_COUNTER_BYTES if umma and (M > 128 or N * K < 2 * WORKSPACE_COUNTER_BYTES) else 0


def gemm_static_scratch(params: GemmParams, stream=None) -> None:
    """abq_gemm on the library's built-in device scratch array: allocates nothing, ignores params.workspace."""
    _check(lib().abq_gemm_static_scratch(ctypes.byref(params), _stream(stream)), "abq_gemm_static_scratch")


def pack_int32(values, planes, rows: int, K: int, bits: int, stream=None) -> None:
    _check(lib().abq_pack_int32(_ptr(values), _ptr(planes), rows, K, bits, _stream(stream)), "abq_pack_int32")


def pack_int4(nibbles, planes, rows: int, K: int, bits: int = 4, stream=None) -> None:
    _check(lib().abq_pack_int4(_ptr(nibbles), _ptr(planes), rows, K, bits, _stream(stream)), "abq_pack_int4")


def quantize_pack_half(x_half, scale, planes, rows: int, K: int, bits: int, mode: int = 0, stream=None) -> None:
    _check(lib().abq_quantize_pack_half(_ptr(x_half), _ptr(scale), _ptr(planes), rows, K, bits, mode, _stream(stream)),
           "abq_quantize_pack_half")


def rmsnorm_quantize_pack_half(x_half, gamma, eps: float, rows: int, K: int, bits: int, mode: int, *, residual=None, sum_out=None, scale=None,
                               row_scale_out=None, planes=None, y_out=None, stream=None) -> None:
    """(residual add ->) RMSNorm -> quantiser -> planes in one launch; see abq_rmsnorm_quantize_pack_half in the header."""
    _check(lib().abq_rmsnorm_quantize_pack_half(_ptr(x_half), _ptr(residual), _ptr(sum_out), _ptr(gamma), ctypes.c_float(eps), _ptr(scale),
                                                _ptr(row_scale_out), _ptr(planes), _ptr(y_out), rows, K, bits, mode, _stream(stream)),
           "abq_rmsnorm_quantize_pack_half")


def quantize_weights_half(w_half, planes, scale, zero, N: int, K: int, bits: int, group_size: int = 0, symmetric: bool = False, stream=None) -> None:
    """fp16 weights [N][K] -> bit-planes + fp16 scale + u8 zero point (min/max calibration of the reference's quantiser)."""
    _check(lib().abq_quantize_weights_half(_ptr(w_half), N, K, bits, group_size, int(symmetric), _ptr(planes), _ptr(scale), _ptr(zero), _stream(stream)),
           "abq_quantize_weights_half")


def swiglu_half(gate_up, out, M: int, F: int, stream=None) -> None:
    """out[m][f] = silu(gate_up[m][f]) * gate_up[m][F + f]: one launch, in the GEMMs' dependent-launch chain."""
    _check(lib().abq_swiglu_half(_ptr(gate_up), _ptr(out), M, F, _stream(stream)), "abq_swiglu_half")


def add_half(a, b, out, n: int, stream=None) -> None:
    _check(lib().abq_add_half(_ptr(a), _ptr(b), _ptr(out), n, _stream(stream)), "abq_add_half")


def unpack_int8(planes, out_i8, rows: int, K: int, bits: int, signed: bool, stream=None) -> None:
    _check(lib().abq_unpack_int8(_ptr(planes), _ptr(out_i8), rows, K, bits, int(signed), _stream(stream)), "abq_unpack_int8")


# ---- the quantised key/value cache and attention.  A parameter block is made once and used for many calls (it keeps its tensors alive).

def _half_type(dtype) -> int:
    import torch
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"attention takes fp16 or bf16, not {dtype}")
    return HALF_BF16 if dtype == torch.bfloat16 else HALF_FP16


def _rows_of(t, heads, head_dim: int, half_type: int, what: str):
    """(address, row stride, head stride) of [rows][heads][head_dim] values, any strides that keep a head's values together."""
    if t.dim() != 3 or t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{what} is {tuple(t.shape)}, expected [rows][{heads if heads is not None else 'heads'}][{head_dim}]")
    if not t.is_cuda or _half_type(t.dtype) != half_type:
        raise ValueError(f"{what}: a CUDA tensor of the cache's 16-bit type, not {t.dtype} on {t.device}")
    if t.stride(2) != 1:
        raise ValueError(f"{what}: the values of a head must lie together")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _ints(t, shape, what: str, dtype: str = "int32"):
    import torch
    if t.dtype != getattr(torch, dtype) or not t.is_cuda or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: a contiguous CUDA {dtype} tensor {tuple(shape)}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _one_device(**tensors) -> int:
    """Index of the device that all of them (but None and plain addresses) are on: a kernel must not be handed another GPU's memory."""
    found = {name: t.device.index for name, t in tensors.items() if t is not None and not isinstance(t, int)}
    if len(set(found.values())) > 1:
        raise ValueError("tensors on different devices: " + ", ".join(f"{name} on cuda:{index}" for name, index in found.items()))
    return next(iter(found.values()))


_current_device = _current_raw = None  # index of the current device; address of a device's current stream


def _launch(entry: str, params, stream) -> None:
    """The call on the device its tensors are on, whichever is current; ``stream`` None: that device's current stream.  (Without making a Stream object for it
    where torch has a way to: a call of a few microseconds shows the difference.)"""
    global _current_device, _current_raw
    if _current_device is None:
        import torch
        torch.cuda.init()
        _current_raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        _current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    device = params._device
    if device != _current_device():
        import torch
        with torch.cuda.device(device):
            return _launch(entry, params, stream)
    status = getattr(_lib or lib(), entry)(ctypes.byref(params), _current_raw(device) if stream is None else _stream(stream))
    if status:
        _check(status, entry)


def kv_cache_bytes(num_pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int) -> int:
    """Bytes of one layer's cache (0: no such cache)."""
    return int(lib().abq_kv_cache_bytes(ctypes.byref(KVCache(None, num_pages, page_size, kv_heads, head_dim, bits, HALF_FP16))))


def make_kv_cache(data, *, page_size: int, kv_heads: int, head_dim: int, bits: int, dtype) -> KVCache:
    """A cache of as many whole pages as ``data`` (uint8) has room for, for keys and values of ``dtype``."""
    page = kv_cache_bytes(1, page_size, kv_heads, head_dim, bits)
    pages = data.numel() * data.element_size() // page if page else 0
    if not pages:
        raise ValueError(f"no cache of {bits} bits, {kv_heads} heads of {head_dim}, pages of {page_size} tokens in {data.numel() * data.element_size()} bytes")
    c = KVCache(_ptr(data), pages, page_size, kv_heads, head_dim, bits, _half_type(dtype))
    c._keep_alive = data
    return c


def make_kv_write_params(cache: KVCache, k, v, slots) -> KVWriteParams:
    """k, v [tokens][kv_heads][head_dim] (views with strides are fine), slots int64 [tokens]: page * page_size + place, negative = left out."""
    p = KVWriteParams()
    p.cache, p.tokens = cache, k.shape[0]
    p.k, p.k_stride, p.k_head_stride = _rows_of(k, cache.kv_heads, cache.head_dim, cache.half_type, "k")
    p.v, p.v_stride, p.v_head_stride = _rows_of(v, cache.kv_heads, cache.head_dim, cache.half_type, "v")
    if v.shape[0] != p.tokens:
        raise ValueError(f"{p.tokens} rows of k, {v.shape[0]} of v")
    p.slots = _ints(slots, (p.tokens,), "slots", "int64")
    p._device = _one_device(cache=cache._keep_alive, k=k, v=v, slots=slots)
    p._keep_alive = (cache, k, v, slots)
    return p


def kv_cache_write(params: KVWriteParams, stream=None) -> None:
    _launch("abq_kv_cache_write", params, stream)


def make_kv_read_params(cache: KVCache, k, v, block_table, cu_seqlens) -> KVReadParams:
    """k, v [rows][kv_heads][head_dim] get the sequences packed; block_table int32 [batch][pages], cu_seqlens int32 [batch + 1]."""
    p = KVReadParams()
    p.cache, p.rows = cache, k.shape[0]
    p.k, p.k_stride, p.k_head_stride = _rows_of(k, cache.kv_heads, cache.head_dim, cache.half_type, "k")
    p.v, p.v_stride, p.v_head_stride = _rows_of(v, cache.kv_heads, cache.head_dim, cache.half_type, "v")
    if v.shape[0] != p.rows:
        raise ValueError(f"{p.rows} rows of k, {v.shape[0]} of v")
    p.batch, p.table_stride = block_table.shape
    p.block_table = _ints(block_table, (p.batch, p.table_stride), "block_table")
    p.cu_seqlens = _ints(cu_seqlens, (p.batch + 1,), "cu_seqlens")
    p._device = _one_device(cache=cache._keep_alive, k=k, v=v, block_table=block_table, cu_seqlens=cu_seqlens)
    p._keep_alive = (cache, k, v, block_table, cu_seqlens)
    return p


def kv_cache_read(params: KVReadParams, stream=None) -> None:
    _launch("abq_kv_cache_read", params, stream)


def cache_attention_workspace_bytes(cache: KVCache, batch: int, rows_per_seq: int, q_heads: int) -> int:
    return int(lib().abq_cache_attention_workspace_bytes(ctypes.byref(cache), batch, rows_per_seq, q_heads))


def make_cache_attention_params(cache: KVCache, q, out, block_table, seq_lens, *, scale: float, workspace, tree=None, status_word=None) -> CacheAttentionParams:
    """q, out [batch * n][q_heads][head_dim]: the last n tokens of every sequence; block_table int32 [batch][pages], seq_lens int32 [batch]
    (those tokens included), tree int64 [batch][n]: bit j of a row = it sees draft j (None: each sees those up to itself)."""
    p = CacheAttentionParams()
    p.cache = cache
    p.batch, p.table_stride = block_table.shape
    if q.dim() != 3 or out.shape != q.shape or (q.shape[0] % p.batch if p.batch else q.shape[0]):
        raise ValueError(f"q {tuple(q.shape)} and out {tuple(out.shape)} do not hold the same rows of {p.batch} sequences")
    p.rows_per_seq, p.q_heads = q.shape[0] // p.batch if p.batch else 1, q.shape[1]
    p.q, p.q_stride, p.q_head_stride = _rows_of(q, None, cache.head_dim, cache.half_type, "q")
    p.out, p.out_stride, p.out_head_stride = _rows_of(out, None, cache.head_dim, cache.half_type, "out")
    p.block_table = _ints(block_table, (p.batch, p.table_stride), "block_table")
    p.seq_lens = _ints(seq_lens, (p.batch,), "seq_lens")
    p.tree = None if tree is None else _ints(tree, (p.batch, p.rows_per_seq), "tree", "int64")
    p.scale = scale
    p.workspace, p.workspace_bytes = _ptr(workspace), workspace.numel() * workspace.element_size()
    p.status_word = _ptr(status_word)
    p._device = _one_device(cache=cache._keep_alive, q=q, out=out, block_table=block_table, seq_lens=seq_lens, tree=tree, workspace=workspace, status_word=status_word)
    p._keep_alive = (cache, q, out, block_table, seq_lens, tree, workspace, status_word)
    return p


def cache_attention(params: CacheAttentionParams, stream=None) -> None:
    _launch("abq_cache_attention", params, stream)


def make_prompt_attention_params(q, k, v, out, cu_q, cu_k, *, scale: float, max_q: int = 0, status_word=None) -> PromptAttentionParams:
    """q, out [total_q][q_heads][head_dim], k, v [total_k][kv_heads][head_dim] (views with strides are fine) of sequences packed behind one another;
    cu_q, cu_k int32 [batch + 1]: where each starts.  ``max_q``: rows of the longest, where known."""
    p = PromptAttentionParams()
    if q.dim() != 3 or k.dim() != 3 or out.shape != q.shape or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} and out {tuple(out.shape)} do not belong together")
    p.total_q, p.q_heads, p.head_dim = q.shape
    p.total_k, p.kv_heads = k.shape[:2]
    p.half_type = _half_type(q.dtype)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        at, rows, heads = _rows_of(t, None, p.head_dim, p.half_type, name)
        setattr(p, name, at), setattr(p, name + "_stride", rows), setattr(p, name + "_head_stride", heads)
    p.batch = cu_q.numel() - 1
    p.cu_q, p.cu_k = _ints(cu_q, (p.batch + 1,), "cu_q"), _ints(cu_k, (p.batch + 1,), "cu_k")
    p.scale, p.max_q, p.status_word = scale, max_q, _ptr(status_word)
    p._device = _one_device(q=q, k=k, v=v, out=out, cu_q=cu_q, cu_k=cu_k, status_word=status_word)
    p._keep_alive = (q, k, v, out, cu_q, cu_k, status_word)
    return p


def prompt_attention(params: PromptAttentionParams, stream=None) -> None:
    _launch("abq_prompt_attention", params, stream)
