"""localstack_amd - MI355X (gfx950) Qwen3-MoE expert-FFN path behind a C ABI.

The shared library liblstk_moe.so (built by localstack_amd/build.py from csrc/) holds the HIP
kernels, the HBM expert pool and the C ABI declared in include/lstk_moe.h. This module is a thin
ctypes view of that ABI that mirrors the reference's interface for the path:

  ExpertStore          src/expert_store.h:113-131 (init / acquire / release_all / stats / describe)
  ExpertStore.route    router()    src/qwen3.cpp:175-192
  ExpertStore.ffn      moe_apply() src/qwen3.cpp:197-214 plus the residual add (:250 / :287)
  ExpertStore.block    the resident MoE block of qwen3_build_graph (src/qwen3.cpp:239-250)
  Qwen3Model           the forward pass around it (include/lstk_qwen3.h): Engine::decode
                       (src/engine.cpp:250-278) over qwen3_build_graph (src/qwen3.cpp:223-259)
                       with the KvCache block table (src/kv_cache.cpp:59-150); decode_batch and generate
                       step many sequences at once
  paged_attention, sample, moe_select   the operators of such a step on plain tensors

Device buffers are torch tensors on a ROCm device (or raw integer device pointers); torch is used
only to own device memory and streams. There is no CPU fallback: every compute call runs the HIP
kernels, and a missing library raises.
"""
import ctypes
import gc
import os
import weakref

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
# LSTK_LIBRARY names another build of the library (the sanitizer build of the CPU tests)
LIB_PATH = os.environ.get("LSTK_LIBRARY") or os.path.join(HERE, "liblstk_moe.so")

SCORE_SOFTMAX, SCORE_SIGMOID = 0, 1
TYPE_F32, TYPE_F16, TYPE_Q8_0, TYPE_Q4_K = 0, 1, 8, 12
POOL_STREAMING, POOL_DRY, POOL_DEVICE_LRU, POOL_AUTO_SIZE = 1, 2, 4, 8
E_INVALID, E_NOMEM, E_EXHAUSTED, E_DEVICE, E_IO, E_BADID = -1, -2, -3, -4, -5, -6


class LstkError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(msg)
        self.code = code


class MoeDims(ctypes.Structure):
    _fields_ = [("n_layer", ctypes.c_int32), ("n_embd", ctypes.c_int32), ("n_ff_exp", ctypes.c_int32),
                ("n_expert", ctypes.c_int32), ("n_expert_used", ctypes.c_int32), ("n_batch", ctypes.c_int32)]


class ExpertLayer(ctypes.Structure):
    _fields_ = [("type_up", ctypes.c_int32), ("type_gate", ctypes.c_int32), ("type_down", ctypes.c_int32),
                ("host_up", ctypes.c_void_p), ("host_gate", ctypes.c_void_p), ("host_down", ctypes.c_void_p)]


class PoolStats(ctypes.Structure):
    _fields_ = [("hits", ctypes.c_uint64), ("misses", ctypes.c_uint64), ("bytes_read", ctypes.c_uint64),
                ("acquires", ctypes.c_uint64), ("wait_ms", ctypes.c_double)]


class GgufTensor(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("type", ctypes.c_int32), ("n_dims", ctypes.c_int32),
                ("ne", ctypes.c_int64 * 4), ("offset", ctypes.c_uint64), ("nbytes", ctypes.c_uint64),
                ("data", ctypes.c_void_p)]


class Qwen3HParams(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("n_layer", "n_embd", "n_head", "n_head_kv", "head_dim", "n_vocab",
                                              "n_expert", "n_expert_used", "n_ff_exp", "n_ctx_train")] + \
               [("rms_eps", ctypes.c_float), ("rope_freq_base", ctypes.c_float)]


class Qwen3Layer(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("attn_norm", "wq", "wk", "wv", "wo", "q_norm", "k_norm", "ffn_norm",
                                               "gate_inp")] + [("gate_inp_type", ctypes.c_int32)]


class Qwen3Weights(ctypes.Structure):
    _fields_ = [("tok_embd", ctypes.c_void_p), ("output_norm", ctypes.c_void_p), ("output", ctypes.c_void_p),
                ("layers", ctypes.c_void_p)]


class CRouterRule(ctypes.Structure):
    _fields_ = [("score", ctypes.c_int32), ("n_group", ctypes.c_int32), ("n_group_used", ctypes.c_int32),
                ("group_top", ctypes.c_int32), ("renorm", ctypes.c_int32), ("scale", ctypes.c_float)]


class PagedCache(ctypes.Structure):
    _fields_ = [("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p), ("kv_size", ctypes.c_int64),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("d_cell_seq", ctypes.c_void_p)]


class PagedSeqs(ctypes.Structure):
    _fields_ = [("n_seq", ctypes.c_int32), ("max_len", ctypes.c_int32), ("d_len", ctypes.c_void_p),
                ("d_first", ctypes.c_void_p), ("d_blocks", ctypes.c_void_p), ("n_table", ctypes.c_int32),
                ("d_seq", ctypes.c_void_p)]


class Sampling(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("d_temperature", "d_top_k", "d_top_p", "d_min_p")]


# name -> (restype, argtypes); every function declared in include/lstk_moe.h and include/lstk_qwen3.h
_P, _I, _SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
SIGNATURES = {
    "lstk_last_error": (ctypes.c_char_p, []),
    "lstk_abi_version": (_I, []),
    "lstk_pool_create": (_I, [ctypes.POINTER(MoeDims), _P, _SZ, ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(_P)]),
    "lstk_pool_destroy": (None, [_P]),
    "lstk_pool_default_bytes": (_SZ, [_SZ, _SZ, _SZ, _SZ, _SZ]),
    "lstk_pool_acquire": (_I, [_P, _I, _P, _I, _P, _P]),
    "lstk_pool_acquire_device": (_I, [_P, _I, _P, _I, _P, _P]),
    "lstk_pool_release_all": (_I, [_P, _P]),
    "lstk_pool_stats": (_I, [_P, ctypes.POINTER(PoolStats)]),
    "lstk_pool_total_bytes": (_SZ, [_P]),
    "lstk_pool_total_slots": (ctypes.c_uint32, [_P]),
    "lstk_pool_layer_slots": (_I, [_P, _I]),
    "lstk_pool_describe": (_I, [_P, ctypes.c_char_p, _SZ]),
    "lstk_moe_route": (_I, [_P, _I, _P, _I, _P, _I, _P, _P, _P]),
    "lstk_moe_ffn": (_I, [_P, _I, _P, _P, _P, _P, _P, _I, _P]),
    "lstk_moe_block": (_I, [_P, _I, _P, _P, _I, _P, _P, _P, _P, _I, _P]),
    "lstk_moe_block_noalloc": (_I, [_P, _I, _P, _P, _I, _P, _P, _P, _P, _I, _P]),
    "lstk_moe_permute": (_I, [_P, _P, _I, _I, _P, _P, _P, _P]),
    "lstk_pool_check": (_I, [_P, _P]),
    "lstk_pool_set_timing": (_I, [_P, _I]),
    "lstk_pool_timing": (_I, [_P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_int64)]),
    "lstk_matrix_bytes": (_SZ, [_I, _I, _I]),
    "lstk_repack_matrix": (_I, [_I, _I, _I, _P, _P]),
    "lstk_unpack_matrix": (_I, [_I, _I, _I, _P, _P]),
    "lstk_pool_debug_fail_copies": (_I, [_P, _I]),
    "lstk_model_create": (_I, [ctypes.POINTER(Qwen3HParams), ctypes.POINTER(Qwen3Weights), _P, ctypes.c_uint32,
                               ctypes.c_uint32, ctypes.POINTER(_P)]),
    "lstk_model_destroy": (None, [_P]),
    "lstk_model_decode": (_I, [_P, ctypes.c_int32, _P, _I, _P, _P, _P]),
    "lstk_model_prepare": (_I, [_P, ctypes.c_int32, _P, _I, ctypes.POINTER(ctypes.c_int32), _P]),
    "lstk_model_forward": (_I, [_P, ctypes.c_int32, _I, ctypes.c_int32, _P, _P, _P]),
    "lstk_model_fill_context": (_I, [_P, ctypes.c_int32, _I, ctypes.c_uint64, _P]),
    "lstk_model_set_trace": (_I, [_P, ctypes.c_char_p]),
    "lstk_model_debug_capture": (_I, [_P, _P]),
    "lstk_model_debug_capture_moe_in": (_I, [_P, _P]),
    "lstk_model_remove_seq": (_I, [_P, ctypes.c_int32]),
    "lstk_model_truncate_seq": (_I, [_P, ctypes.c_int32, ctypes.c_int32]),
    "lstk_model_seq_len": (ctypes.c_int32, [_P, ctypes.c_int32]),
    "lstk_gguf_open": (_I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    "lstk_gguf_close": (None, [_P]),
    "lstk_gguf_arch": (ctypes.c_char_p, [_P]),
    "lstk_gguf_version": (_I, [_P]),
    "lstk_gguf_alignment": (_I, [_P]),
    "lstk_gguf_has": (_I, [_P, ctypes.c_char_p]),
    "lstk_gguf_get_int": (ctypes.c_int64, [_P, ctypes.c_char_p, ctypes.c_int64]),
    "lstk_gguf_get_float": (ctypes.c_double, [_P, ctypes.c_char_p, ctypes.c_double]),
    "lstk_gguf_get_str": (ctypes.c_char_p, [_P, ctypes.c_char_p, ctypes.c_char_p]),
    "lstk_gguf_n_tensors": (_I, [_P]),
    "lstk_gguf_tensor_at": (_I, [_P, _I, ctypes.POINTER(GgufTensor)]),
    "lstk_gguf_find_tensor": (_I, [_P, ctypes.c_char_p, ctypes.POINTER(GgufTensor)]),
    "lstk_gguf_qwen3_hparams": (_I, [_P, ctypes.POINTER(Qwen3HParams)]),
    "lstk_gguf_qwen3_experts": (_I, [_P, ctypes.POINTER(Qwen3HParams), _P]),
    "lstk_dequant_f16": (_I, [_I, _P, ctypes.c_size_t, _P]),
    "lstk_model_set_timing": (_I, [_P, _I]),
    "lstk_moe_select": (_I, [ctypes.POINTER(CRouterRule), _P, ctypes.c_int64, _P, _I, _I, _I, _P, _P, _P]),
    "lstk_moe_route_by": (_I, [_P, _I, ctypes.POINTER(CRouterRule), _P, _I, _P, _I, _P, _P, _P, _P]),
    "lstk_attn_paged_work_bytes": (_SZ, [_I] * 7),
    "lstk_attn_paged": (_I, [ctypes.POINTER(PagedCache), ctypes.POINTER(PagedSeqs), _P, _I, _I, _I, ctypes.c_float, _P, _P, _SZ,
                             _P]),
    "lstk_sample_work_bytes": (_SZ, [_I, _I]),
    "lstk_sample": (_I, [_P, ctypes.c_int64, _I, _I, ctypes.POINTER(Sampling), _P, _P, _P, _P, _SZ, _P]),
    "lstk_model_decode_batch": (_I, [_P, _I, _P, _P, _I, _I, _P, _P, _P]),
    "lstk_model_prepare_batch": (_I, [_P, _I, _P, _P, ctypes.POINTER(ctypes.c_int32), _P]),
    "lstk_model_forward_batch": (_I, [_P, _I, ctypes.c_int32, _I, _I, _P, _P, _P]),
    "lstk_debug_attn_plan": (_I, [_I, _I, _I, _I, _I, _I, _I, _I, _P]),
    "lstk_debug_attn_split": (_I, [_I, _I, _I, _I, _I, _I, _I, _I, ctypes.POINTER(ctypes.c_int32)]),
    "lstk_debug_moe_plan": (_I, [ctypes.POINTER(MoeDims), _I, _I, _I, _I, _P]),
    "lstk_model_debug_options": (_I, [_P, _I]),
    "lstk_model_timing": (_I, [_P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_int64)]),
}

_lib = None


def lib():
    """Loads liblstk_moe.so; raises if it has not been built (there is no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python localstack_amd/build.py`")
        # torch ships its own HIP runtime (SONAME libamdhip64.so.7). Loading it first makes the
        # library's libamdhip64.so.7 dependency bind to that same runtime, so the library and torch
        # share one device context and torch's streams are valid handles for the library.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(rc):
    if rc != 0:
        raise LstkError(rc, lib().lstk_last_error().decode())
    return rc


def _ptr(x):
    """Device/host pointer of a torch tensor, numpy array or integer."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)}")


def _stream(stream):
    if stream is None:
        try:
            import torch
            if torch.cuda.is_available():
                return torch.cuda.current_stream().cuda_stream
        except ImportError:
            pass
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _current_device():
    """torch's current GPU, -1 without one."""
    try:
        import torch
    except ImportError:
        return -1
    return torch.cuda.current_device() if torch.cuda.is_available() else -1


def matrix_bytes(type_, rows, cols):
    return lib().lstk_matrix_bytes(type_, rows, cols)


def default_pool_bytes(table_bytes, weight_bytes, kv_bytes, device_total, device_free):
    """Engine::init's pool budget (src/engine.cpp:84-117) for HBM: min(table, total - weights - kv - 1.5 GiB,
    free - 3 GiB), at least 16 KiB."""
    return lib().lstk_pool_default_bytes(int(table_bytes), int(weight_bytes), int(kv_bytes), int(device_total),
                                         int(device_free))


def attn_plan(n_tokens, n_head, n_kv, head_dim, kv_size, n_cells, cell_begin=0, rope_in=False):
    """The attention launch plan the library takes for a step (host arithmetic, no device call):
    (rows per work-group, row blocks, cells per chunk, chunks, RoPE inside the launch, work-groups)."""
    out = (ctypes.c_int32 * 6)()
    _check(lib().lstk_debug_attn_plan(int(n_tokens), int(n_head), int(n_kv), int(head_dim), int(kv_size), int(n_cells),
                                      int(cell_begin), 1 if rope_in else 0, ctypes.cast(out, ctypes.c_void_p)))
    return out[0], out[1], out[2], out[3], bool(out[4]), out[5]


def attn_split(n_tokens, n_head, n_kv, head_dim, kv_size, n_cells, cell_begin=0, n_live=0):
    """Whether a step's attention splits the cells over a work-group's wavefronts (host arithmetic, no device call); n_live =
    cells of the range that belong to the sequence (0: all)."""
    out = ctypes.c_int32()
    _check(lib().lstk_debug_attn_split(int(n_tokens), int(n_head), int(n_kv), int(head_dim), int(kv_size), int(n_cells),
                                       int(cell_begin), int(n_live), ctypes.byref(out)))
    return bool(out.value)


def moe_plan(types, n_embd, n_ff_exp, n_expert, n_expert_used, n_tokens, n_slots=None):
    """How an expert call of n_tokens runs (host arithmetic, no device call): (grouped path, register-streaming kernels,
    pairs per work item, non-temporal weights, grouped in block_noalloc too). types = (up, gate, down)."""
    d = MoeDims(1, int(n_embd), int(n_ff_exp), int(n_expert), int(n_expert_used), int(n_tokens))
    out = (ctypes.c_int32 * 5)()
    _check(lib().lstk_debug_moe_plan(ctypes.byref(d), int(types[1]), int(types[2]), int(n_slots or n_expert), int(n_tokens),
                                     ctypes.cast(out, ctypes.c_void_p)))
    return bool(out[0]), bool(out[1]), out[2], bool(out[3]), bool(out[4])


def repack_matrix(type_, rows, cols, gguf):
    gguf = np.ascontiguousarray(gguf, dtype=np.uint8)
    out = np.empty(matrix_bytes(type_, rows, cols), np.uint8)
    _check(lib().lstk_repack_matrix(type_, rows, cols, gguf.ctypes.data, out.ctypes.data))
    return out


def unpack_matrix(type_, rows, cols, packed):
    packed = np.ascontiguousarray(packed, dtype=np.uint8)
    out = np.empty(matrix_bytes(type_, rows, cols), np.uint8)
    _check(lib().lstk_unpack_matrix(type_, rows, cols, packed.ctypes.data, out.ctypes.data))
    return out


# ---- operators of a step over many sequences -------------------------------------------------------
_MOST = 2 ** 31 - 1


def _i32(v, name):
    """v as a number that the library's 32-bit arguments hold (ctypes would drop its upper bits)."""
    try:
        i = int(v)
    except (TypeError, ValueError, OverflowError):
        raise LstkError(E_INVALID, f"{name} must be a whole number, got {v!r}") from None
    if not -_MOST - 1 <= i <= _MOST:
        raise LstkError(E_INVALID, f"{name} must fit 32 bits, got {i}")
    return i


def _check_i32(**named):
    for name, v in named.items():
        _i32(v, name)


def _ids32(a, name):
    """An int32 array of these host numbers; numpy would drop their upper bits or fractions."""
    try:
        v = np.asarray(a)
        with np.errstate(invalid="ignore"):
            i = np.ascontiguousarray(v, dtype=np.int32).ravel()
    except (TypeError, ValueError, OverflowError):
        i = None
    if i is None or not np.array_equal(i, v.ravel()):
        raise LstkError(E_INVALID, f"{name} must be whole numbers of 32 bits")
    return i


# A call that takes the device a few microseconds is bound by what Python does around it, so the checks below look at each
# tensor once, in the cheapest order, and build a message only when one fails.

def _tensor(t, name, dtype, shape, dev=None):
    """Pointer of a contiguous tensor of this dtype and shape (None: any size) on device `dev` (None: any GPU)."""
    try:
        s = t.shape
        if t.dtype is dtype and (s == shape or (len(s) == len(shape) and all(w is None or n == w for n, w in zip(s, shape)))) and \
                t.is_contiguous():
            d = t.get_device()
            if d == dev or (dev is None and d >= 0):
                return t.data_ptr()
    except AttributeError:
        raise LstkError(E_INVALID, f"{name} must be a tensor, got {type(t)}") from None
    if t.is_contiguous() and t.dtype is dtype and len(s) == len(shape) and all(w is None or n == w for n, w in zip(s, shape)):
        raise LstkError(E_INVALID, f"{name} is on {t.device}" + ("" if dev is None else f", not on GPU {dev}"))
    want = "x".join("n" if w is None else str(w) for w in shape)
    raise LstkError(E_INVALID, f"{name} must be a contiguous {dtype} tensor of shape {want}, got {t.dtype} {tuple(s)}")


def _rows(t, name, dtype):
    """A 2-D tensor on a GPU whose rows are contiguous: (pointer, row stride, rows, row length, device)."""
    try:
        n, m = t.shape
        ld, one = t.stride()
        dev = t.get_device()
    except (AttributeError, ValueError):
        raise LstkError(E_INVALID, f"{name} must be a 2-D tensor") from None
    if t.dtype is not dtype:
        raise LstkError(E_INVALID, f"{name} must be a 2-D {dtype} tensor, got {t.dtype}")
    if dev < 0:
        raise LstkError(E_INVALID, f"{name} is on {t.device}")
    if (m > 1 and one != 1) or (n > 1 and ld < m):
        raise LstkError(E_INVALID, f"{name} must have contiguous rows that do not overlap")
    return t.data_ptr(), ld if n > 1 else m, n, m, dev


def _buffer(t, name, dtype, least, dev):
    """Pointer of a contiguous tensor on GPU `dev` with at least `least` elements of this dtype (None: bytes of any), for calls
    that also take raw device pointers (integers) and None."""
    if t is None or isinstance(t, int):
        return t
    try:
        fits = (dtype is None or t.dtype is dtype) and t.is_contiguous()
        room = t.numel() * (t.element_size() if dtype is None else 1)
        on = t.get_device()
    except AttributeError:
        raise LstkError(E_INVALID, f"{name} must be a tensor or a device pointer, got {type(t)}") from None
    if not fits or room < least:
        raise LstkError(E_INVALID, f"{name} must be a contiguous tensor of at least {least} " +
                        (f"bytes, got {room}" if dtype is None else f"{dtype} elements, got {t.dtype} {tuple(t.shape)}"))
    if on < 0 or on != dev:
        raise LstkError(E_INVALID, f"{name} is on {t.device}" + (f", not on GPU {dev}" if dev >= 0 else ", not on the GPU"))
    return t.data_ptr()


def _on_device(dev, stream, call):
    """call(stream handle) with device `dev` current; the handle is `stream`'s, or that of the device's current stream."""
    import torch
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(dev)
    else:
        handle = stream if isinstance(stream, int) else stream.cuda_stream
        if getattr(stream, "device_index", dev) != dev:
            raise LstkError(E_INVALID, f"the stream is of GPU {stream.device_index}, the tensors of GPU {dev}")
    if torch.cuda.current_device() == dev:
        return call(handle)
    with torch.cuda.device(dev):
        return call(handle)


def _empty(shape, dtype, dev, stream):
    """A new tensor for the work of `stream`: of that stream's memory, since what the current stream has freed may still be in use
    by what it has queued."""
    import torch
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=dev)


def _work(given, nbytes, dev, stream):
    """(tensor, pointer, bytes) of the caller's workspace, or of a new one."""
    if given is None:
        import torch
        given = _empty(nbytes, torch.uint8, dev, stream)
    elif not hasattr(given, "data_ptr") or given.get_device() != dev or not given.is_contiguous():
        raise LstkError(E_INVALID, f"work must be a contiguous tensor on GPU {dev}")
    return given, given.data_ptr(), given.numel() * given.element_size()


class RouterRule:
    """How a router chooses experts from its logits (lstk_router_rule, include/lstk_moe.h): score "softmax" or "sigmoid";
    n_group groups of which the n_group_used with the largest sum of their group_top best choice values stay; weights divided
    by their sum (renorm) and scaled."""

    def __init__(self, score="softmax", n_group=1, n_group_used=None, group_top=1, renorm=True, scale=1.0):
        if score not in ("softmax", "sigmoid"):
            raise LstkError(E_INVALID, f"unknown score function {score!r}")
        self.c = CRouterRule(SCORE_SIGMOID if score == "sigmoid" else SCORE_SOFTMAX, _i32(n_group, "n_group"),
                             _i32(n_group if n_group_used is None else n_group_used, "n_group_used"), _i32(group_top, "group_top"),
                             1 if renorm else 0, float(scale))


def moe_select(logits, n_expert_used, rule, bias=None, ids=None, weights=None, stream=None):
    """The experts a rule chooses from router logits [T][n_expert] (f32, rows may be strided): (ids int32, weights f32), each
    [T][n_expert_used], in descending order of choice. bias: f32 [n_expert], added to the scores for the choice only."""
    import torch
    p, ld, T, E, dev = _rows(logits, "logits", torch.float32)
    b = None if bias is None else _tensor(bias, "bias", torch.float32, (E,), dev)
    k = int(n_expert_used)
    if not (T <= _MOST and E <= _MOST and 0 <= k <= _MOST):
        _check_i32(n_tokens=T, n_expert=E, n_expert_used=k)
    shape = (T, k)
    if ids is None:
        ids = _empty((T, max(k, 0)), torch.int32, dev, stream)
    if weights is None:
        weights = _empty((T, max(k, 0)), torch.float32, dev, stream)
    ip, wp = _tensor(ids, "ids", torch.int32, shape, dev), _tensor(weights, "weights", torch.float32, shape, dev)
    _check(_on_device(dev, stream, lambda st: lib().lstk_moe_select(ctypes.byref(rule.c), p, ld, b, T, E, k, ip, wp, st)))
    return ids, weights


def paged_attention_work_bytes(n_seq, n_head, n_head_kv, head_dim, max_len, window=0, n_sink=0):
    return lib().lstk_attn_paged_work_bytes(_i32(n_seq, "n_seq"), _i32(n_head, "n_head"), _i32(n_head_kv, "n_head_kv"),
                                            _i32(head_dim, "head_dim"), _i32(max_len, "max_len"), _i32(window, "window"),
                                            _i32(n_sink, "n_sink"))


def paged_attention(q, k_cache, v_cache, lens, first, blocks, max_len, window=0, n_sink=0, scale=None, cell_seq=None, seqs=None,
                    out=None, work=None, stream=None):
    """Attention of one new token per sequence over a paged cache (lstk_attn_paged, include/lstk_qwen3.h).

    q: fp16 [n_seq][n_head][head_dim]. k_cache: fp16 [n_head_kv][head_dim / 4][kv_size][4], v_cache: fp16
    [n_head_kv][kv_size / 4][head_dim][4]. lens, first: int32 [n_seq]; blocks: int32, the 32-cell block numbers of row b from
    first[b] on. max_len bounds the lengths (it sizes the launch). window > 0: only the last `window` cells and the first
    n_sink. cell_seq (int32 [kv_size]) with seqs (int32 [n_seq]): cells of other owners are not visible. Returns out, like q."""
    import torch
    i32, f16 = torch.int32, torch.float16
    max_len, window, n_sink = int(max_len), int(window), int(n_sink)
    qp = _tensor(q, "q", f16, (None, None, None))
    dev = q.get_device()
    n, H, hd = shape = q.shape
    kp = _tensor(k_cache, "k_cache", f16, (None, hd // 4, None, 4), dev)
    kv, _, size, _ = k_cache.shape
    cache = PagedCache(kp, _tensor(v_cache, "v_cache", f16, (kv, size // 4, hd, 4), dev), size, kv, hd,
                       None if cell_seq is None else _tensor(cell_seq, "cell_seq", i32, (size,), dev))
    table = _tensor(blocks, "blocks", i32, (None,), dev)
    # (the other sizes are those of tensors that would not fit the device)
    if not (0 <= max_len <= _MOST and 0 <= window <= _MOST and 0 <= n_sink <= _MOST and blocks.numel() <= _MOST):
        _check_i32(max_len=max_len, window=window, n_sink=n_sink, n_table=blocks.numel())
    s = PagedSeqs(n, max_len, _tensor(lens, "lens", i32, (n,), dev), _tensor(first, "first", i32, (n,), dev), table,
                  blocks.numel(), None if seqs is None else _tensor(seqs, "seqs", i32, (n,), dev))
    if out is None:
        out = _empty(shape, f16, dev, stream)
    op = _tensor(out, "out", f16, shape, dev)
    need = 0 if work is not None else lib().lstk_attn_paged_work_bytes(n, H, kv, hd, max_len, window, n_sink)
    wt, wp, wn = (None, None, 0) if work is None and need == 0 else _work(work, need, dev, stream)
    f = float(hd ** -0.5 if scale is None else scale)
    _check(_on_device(dev, stream, lambda st: lib().lstk_attn_paged(ctypes.byref(cache), ctypes.byref(s), qp, H, window, n_sink, f,
                                                                    op, wp, wn, st)))
    return out


def sample_work_bytes(n_rows, n_vocab):
    return lib().lstk_sample_work_bytes(_i32(n_rows, "n_rows"), _i32(n_vocab, "n_vocab"))


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, probs=None, work=None, stream=None):
    """The next token of each row of logits (f32 [n][n_vocab], rows may be strided), drawn with the random numbers u (f32 [n],
    in [0, 1)): lstk_sample, include/lstk_qwen3.h. temperature, top_p, min_p (f32) and top_k (int32) are [n] device tensors;
    None means temperature 1 / no cut. Returns (tokens int32 [n], probabilities f32 [n])."""
    import torch
    f32, i32 = torch.float32, torch.int32
    p, ld, n, V, dev = _rows(logits, "logits", f32)
    if not (n <= _MOST and V <= _MOST):
        _check_i32(n_rows=n, n_vocab=V)
    shape = (n,)
    how = Sampling(None if temperature is None else _tensor(temperature, "temperature", f32, shape, dev),
                   None if top_k is None else _tensor(top_k, "top_k", i32, shape, dev),
                   None if top_p is None else _tensor(top_p, "top_p", f32, shape, dev),
                   None if min_p is None else _tensor(min_p, "min_p", f32, shape, dev))
    up = _tensor(u, "u", f32, shape, dev)
    if tokens is None:
        tokens = _empty(n, i32, dev, stream)
    if probs is None:
        probs = _empty(n, f32, dev, stream)
    tp, pp = _tensor(tokens, "tokens", i32, shape, dev), _tensor(probs, "probs", f32, shape, dev)
    wt, wp, wn = _work(work, lib().lstk_sample_work_bytes(n, V) if work is None else 0, dev, stream)
    _check(_on_device(dev, stream, lambda st: lib().lstk_sample(p, ld, n, V, ctypes.byref(how), up, tp, pp, wp, wn, st)))
    return tokens, probs


_stores = weakref.WeakSet()  # stores not yet freed


class ExpertStore:
    """The HBM expert pool (ExpertStore, src/expert_store.h:113-131) and the MoE calls that read it.

    layers: one (types, up, gate, down) per layer; types = (type_up, type_gate, type_down), and
    up/gate/down are the layer's stacked expert tensors as GGUF bytes (numpy uint8, expert-major).
    """

    def __init__(self, n_layer, n_embd, n_ff_exp, n_expert, n_expert_used, n_batch, layers, pool_bytes=0,
                 min_slots=0, streaming=False, dry=False, device_lru=False, auto_size=False):
        self.dims = MoeDims(n_layer, n_embd, n_ff_exp, n_expert, n_expert_used, n_batch)
        arr = (ExpertLayer * n_layer)()
        self._keep = []
        for l, (types, up, gate, down) in enumerate(layers):
            ptrs = []
            for a in (up, gate, down):
                if a is None or isinstance(a, int):
                    ptrs.append(a)
                else:
                    a = np.ascontiguousarray(a)
                    self._keep.append(a)
                    ptrs.append(a.ctypes.data)
            arr[l] = ExpertLayer(types[0], types[1], types[2], *ptrs)
        # A store dropped in a reference cycle, and the graphs that replay it, stay until Python's cyclic collector runs. Their
        # HBM is wanted now; and a collection that falls into a later stream capture would free device memory and destroy
        # graphs there, which HIP refuses (torch ends the process). 65 ms beside torch, and only where another store is left.
        if not dry and _stores:
            gc.collect()
        flags = ((POOL_STREAMING if streaming else 0) | (POOL_DRY if dry else 0) | (POOL_DEVICE_LRU if device_lru else 0) |
                 (POOL_AUTO_SIZE if auto_size else 0))
        h = ctypes.c_void_p()
        _check(lib().lstk_pool_create(ctypes.byref(self.dims), ctypes.cast(arr, ctypes.c_void_p), int(pool_bytes),
                                      int(min_slots), flags, ctypes.byref(h)))
        self._h = h
        self._dev = -1 if dry else _current_device()  # the pool lives on it
        self._keep = None  # the pool copied what it needs
        self._destroy = lib().lstk_pool_destroy  # held, so that closing works during interpreter shutdown
        _stores.add(self)

    def close(self):
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()

    # -- ExpertStore bookkeeping ------------------------------------------------------------
    def acquire(self, layer, experts, stream=None):
        e = np.ascontiguousarray(experts, dtype=np.int32).ravel()
        slots = np.zeros(e.size, np.int32)
        _check(lib().lstk_pool_acquire(self._h, layer, e.ctypes.data, e.size, slots.ctypes.data, _stream(stream)))
        return slots.reshape(np.shape(experts))

    def acquire_device(self, layer, experts, slots, n=None, stream=None):
        """Device-side acquire + release of one segment (pools made with device_lru=True): experts and
        slots are int32 device tensors."""
        n = experts.numel() if n is None else n
        _check(lib().lstk_pool_acquire_device(self._h, layer, _ptr(experts), n, _ptr(slots), _stream(stream)))

    def release_all(self, stream=None):
        _check(lib().lstk_pool_release_all(self._h, _stream(stream)))

    def stats(self):
        s = PoolStats()
        _check(lib().lstk_pool_stats(self._h, ctypes.byref(s)))
        return dict(hits=s.hits, misses=s.misses, bytes_read=s.bytes_read, acquires=s.acquires, wait_ms=s.wait_ms)

    def total_bytes(self):
        return lib().lstk_pool_total_bytes(self._h)

    def total_slots(self):
        return lib().lstk_pool_total_slots(self._h)

    def layer_slots(self, layer):
        n = lib().lstk_pool_layer_slots(self._h, layer)
        if n < 0:
            _check(n)
        return n

    def describe(self):
        buf = ctypes.create_string_buffer(1 << 16)
        _check(lib().lstk_pool_describe(self._h, buf, len(buf)))
        return buf.value.decode()

    def debug_fail_copies(self, n):
        _check(lib().lstk_pool_debug_fail_copies(self._h, n))

    # -- compute ----------------------------------------------------------------------------
    def route(self, layer, hnorm, gate_inp, gate_type, ids, weights, n_tokens=None, stream=None):
        T = hnorm.shape[0] if n_tokens is None else n_tokens
        _check(lib().lstk_moe_route(self._h, layer, _ptr(hnorm), T, _ptr(gate_inp), gate_type, _ptr(ids), _ptr(weights),
                                    _stream(stream)))

    def route_by(self, layer, rule, hnorm, gate_inp, gate_type, ids, weights, bias=None, n_tokens=None, stream=None):
        """route() by a RouterRule; bias: f32 [n_expert] or None. Tensors are checked for their type, size and device."""
        import torch
        T = _i32(hnorm.shape[0] if n_tokens is None else n_tokens, "n_tokens")
        layer, gate_type = _i32(layer, "layer"), _i32(gate_type, "gate_type")
        d, dev, rows = self.dims, self._dev, max(T, 0)
        x = _buffer(hnorm, "hnorm", torch.float32, rows * d.n_embd, dev)
        gate = _buffer(gate_inp, "gate_inp", None, d.n_expert * d.n_embd * (4 if gate_type == TYPE_F32 else 2), dev)
        b = _buffer(bias, "bias", torch.float32, d.n_expert, dev)
        i = _buffer(ids, "ids", torch.int32, rows * d.n_expert_used, dev)
        w = _buffer(weights, "weights", torch.float32, rows * d.n_expert_used, dev)
        call = lambda st: lib().lstk_moe_route_by(self._h, layer, ctypes.byref(rule.c), x, T, gate, gate_type, b, i, w, st)
        _check(_on_device(dev, stream, call) if dev >= 0 else call(None))

    def ffn(self, layer, hnorm, slots, weights, resid, out, n_tokens=None, stream=None):
        T = hnorm.shape[0] if n_tokens is None else n_tokens
        _check(lib().lstk_moe_ffn(self._h, layer, _ptr(hnorm), _ptr(slots), _ptr(weights), _ptr(resid), _ptr(out), T,
                                  _stream(stream)))

    def block(self, layer, hnorm, gate_inp, gate_type, resid, out, ids, weights, n_tokens=None, stream=None):
        T = hnorm.shape[0] if n_tokens is None else n_tokens
        _check(lib().lstk_moe_block(self._h, layer, _ptr(hnorm), _ptr(gate_inp), gate_type, _ptr(resid), _ptr(out),
                                    _ptr(ids), _ptr(weights), T, _stream(stream)))

    def block_noalloc(self, layer, hnorm, gate_inp, gate_type, resid, out, ids, weights, n_tokens=None, stream=None):
        """block() with the call's scratch in the library's fixed per-device array (allocates nothing)."""
        T = hnorm.shape[0] if n_tokens is None else n_tokens
        _check(lib().lstk_moe_block_noalloc(self._h, layer, _ptr(hnorm), _ptr(gate_inp), gate_type, _ptr(resid),
                                            _ptr(out), _ptr(ids), _ptr(weights), T, _stream(stream)))

    def permute(self, bins, n_bins, counts, offsets, perm, n_tokens=None, stream=None):
        """Stable grouping of the (token, slot) pairs by bin, as ggml's CPU mul_mat_id walks them."""
        T = bins.shape[0] if n_tokens is None else n_tokens
        _check(lib().lstk_moe_permute(self._h, _ptr(bins), T, n_bins, _ptr(counts), _ptr(offsets), _ptr(perm),
                                      _stream(stream)))

    def check(self, stream=None):
        _check(lib().lstk_pool_check(self._h, _stream(stream)))

    def set_timing(self, on):
        _check(lib().lstk_pool_set_timing(self._h, 1 if on else 0))

    def timing(self):
        """(ms, launches) per stage: router (+ top-k), gate_up, down, combine."""
        ms = (ctypes.c_double * 4)()
        n = (ctypes.c_int64 * 4)()
        _check(lib().lstk_pool_timing(self._h, ms, n))
        return list(ms), list(n)


class Qwen3Model:
    """The Qwen3-MoE forward pass on the device (include/lstk_qwen3.h), mirroring Engine::decode.

    hp: dict of the lstk_qwen3_hparams fields. weights: dict with numpy arrays tok_embd (fp16
    [n_vocab][n_embd]), output_norm (f32), optional output (fp16), and layers, a list of dicts with
    attn_norm, wq, wk, wv, wo, q_norm, k_norm (or None), ffn_norm and gate_inp (fp16 [n_expert][n_embd]).
    The dense tensors are uploaded to `device` here (torch owns that memory); the experts live in
    `store`, an ExpertStore of matching dims created by the caller (resident or streaming).
    """

    def __init__(self, hp, weights, store, kv_size, n_batch, device="cuda", join_qkv=True):
        import torch
        self.hp = dict(hp)
        self.n_batch = int(n_batch)
        self.store = store
        self.device = torch.device(device)
        self._keep = []

        def up(a, dtype):
            if a is None:
                return None
            a = np.ascontiguousarray(a)
            if not a.flags.writeable:  # a view of a read-only file mapping: torch wants a writable source
                a = a.copy()
            t = torch.from_numpy(a.view(dtype)).to(self.device)
            self._keep.append(t)
            return t.data_ptr()

        def up_joined(arrs, dtype):
            """The arrays one after the other in one device buffer (Q, K and V weights, so the model can
            multiply all three in one product); returns each one's device pointer."""
            flat = [np.ascontiguousarray(a).view(dtype).ravel() for a in arrs]
            t = torch.from_numpy(np.concatenate(flat)).to(self.device)
            self._keep.append(t)
            offs = np.cumsum([0] + [a.size for a in flat[:-1]])
            return [t.data_ptr() + int(o) * t.element_size() for o in offs]

        f16, f32 = np.uint16, np.float32
        self._hp = Qwen3HParams(*(int(self.hp[n]) for n in ("n_layer", "n_embd", "n_head", "n_head_kv", "head_dim",
                                                             "n_vocab", "n_expert", "n_expert_used", "n_ff_exp")),
                                int(self.hp.get("n_ctx_train", 0)), float(self.hp["rms_eps"]),
                                float(self.hp["rope_freq_base"]))
        n_layer = self.hp["n_layer"]
        self._layers = (Qwen3Layer * n_layer)()
        for l, L in enumerate(weights["layers"]):
            if join_qkv:
                wq, wk, wv = up_joined((L["wq"], L["wk"], L["wv"]), f16)
            else:
                wq, wk, wv = up(L["wq"], f16), up(L["wk"], f16), up(L["wv"], f16)
            self._layers[l] = Qwen3Layer(up(L["attn_norm"], f32), wq, wk, wv,
                                         up(L["wo"], f16), up(L.get("q_norm"), f32), up(L.get("k_norm"), f32),
                                         up(L["ffn_norm"], f32),
                                         up(L["gate_inp"], f32 if L["gate_inp"].dtype == np.float32 else f16),
                                         TYPE_F32 if L["gate_inp"].dtype == np.float32 else TYPE_F16)
        self._w = Qwen3Weights(up(weights["tok_embd"], f16), up(weights["output_norm"], f32),
                               up(weights.get("output"), f16), ctypes.cast(self._layers, ctypes.c_void_p))
        h = ctypes.c_void_p()
        _check(lib().lstk_model_create(ctypes.byref(self._hp), ctypes.byref(self._w), store._h, int(kv_size),
                                       int(n_batch), ctypes.byref(h)))
        self._h = h
        self._destroy = lib().lstk_model_destroy
        self.logits = torch.empty(self.hp["n_vocab"], dtype=torch.float32, device=self.device)

    def close(self):
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()

    def decode(self, seq, tokens, trace=None, logits=None, stream=None):
        """Appends tokens to sequence seq; returns the device logits [n_vocab] of the last token.

        trace: optional device int32 tensor [n_layer, n_step_tokens, n_expert_used] for the router ids
        of the last step (-1 for rows the last layer skips)."""
        tok = np.ascontiguousarray(tokens, dtype=np.int32).ravel()
        out = self.logits if logits is None else logits
        _check(lib().lstk_model_decode(self._h, int(seq), tok.ctypes.data, tok.size, _ptr(out), _ptr(trace),
                                       _stream(stream)))
        return out

    def prepare(self, seq, tokens, stream=None):
        """First half of a step: KV cells and input upload; returns the attended cell count."""
        tok = np.ascontiguousarray(tokens, dtype=np.int32).ravel()
        n = ctypes.c_int32()
        _check(lib().lstk_model_prepare(self._h, int(seq), tok.ctypes.data, tok.size, ctypes.byref(n), _stream(stream)))
        return n.value

    def forward(self, seq, n_tokens, n_cells, trace=None, logits=None, stream=None):
        """Second half of a step: the kernels (capturable in a HIP graph with a resident pool)."""
        out = self.logits if logits is None else logits
        _check(lib().lstk_model_forward(self._h, int(seq), int(n_tokens), int(n_cells), _ptr(out), _ptr(trace),
                                        _stream(stream)))
        return out

    def _batch_call(self, n, logits, trace, stream, call):
        """The step's logits; call(logits pointer, trace pointer, stream handle) on the model's device, after a look at what the
        kernels will write to."""
        import torch
        dev, hp = self.logits.get_device(), self.hp
        rows = max(n, 0)
        tr = _buffer(trace, "trace", torch.int32, hp["n_layer"] * rows * hp["n_expert_used"], dev)
        if logits is None:
            logits = _empty((rows, hp["n_vocab"]), torch.float32, self.logits.device, stream)
        out = _buffer(logits, "logits", torch.float32, rows * hp["n_vocab"], dev)
        _check(_on_device(dev, stream, lambda st: call(out, tr, st)))
        return logits

    def decode_batch(self, seqs, tokens, window=0, n_sink=0, trace=None, logits=None, stream=None):
        """Appends tokens[i] to sequence seqs[i] (distinct), all in one step; returns the device logits [n_seq][n_vocab].
        window > 0: each token attends its sequence's last `window` cells and first n_sink. trace: as decode's, with a row for
        every sequence."""
        s, tok = _ids32(seqs, "sequences"), _ids32(tokens, "tokens")
        if s.size != tok.size:
            raise LstkError(E_INVALID, "one token per sequence")
        window, n_sink = _i32(window, "window"), _i32(n_sink, "n_sink")
        return self._batch_call(s.size, logits, trace, stream, lambda out, tr, st: lib().lstk_model_decode_batch(
            self._h, s.size, s.ctypes.data, tok.ctypes.data, window, n_sink, out, tr, st))

    def prepare_batch(self, seqs, tokens, stream=None):
        """First half of a batch step; returns the longest sequence's cells."""
        s, tok = _ids32(seqs, "sequences"), _ids32(tokens, "tokens")
        if s.size != tok.size:
            raise LstkError(E_INVALID, "one token per sequence")
        n = ctypes.c_int32()
        _check(_on_device(self.logits.get_device(), stream, lambda st: lib().lstk_model_prepare_batch(
            self._h, s.size, s.ctypes.data, tok.ctypes.data, ctypes.byref(n), st)))
        return n.value

    def forward_batch(self, n_seq, max_len, window=0, n_sink=0, trace=None, logits=None, stream=None):
        """Second half of a batch step (capturable; replays after each prepare_batch of n_seq sequences up to max_len)."""
        n_seq, max_len, window, n_sink = (_i32(v, n) for v, n in ((n_seq, "n_seq"), (max_len, "max_len"), (window, "window"),
                                                                  (n_sink, "n_sink")))
        return self._batch_call(n_seq, logits, trace, stream, lambda out, tr, st: lib().lstk_model_forward_batch(
            self._h, n_seq, max_len, window, n_sink, out, tr, st))

    def generate(self, prompts, n_new, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, generator=None, window=0, n_sink=0):
        """Continues several sequences together: prompts is {seq: token ids}, each is decoded (appended to what seq holds), then
        n_new tokens are sampled for all of them, a batch step each. Returns {seq: the n_new tokens}; the last is not appended.
        The settings are numbers, or sequences with one per prompt; generator: a torch generator on the model's device. Arguments
        are checked before anything is appended; where a later step fails (no room in the cache, a sequence without a finite
        logit) every sequence is cut back to what it held before."""
        import torch
        seqs = _ids32(list(prompts), "sequences").tolist()
        n, V = len(seqs), self.hp["n_vocab"]
        if n == 0 or n_new <= 0:
            return {s: [] for s in seqs}
        if n > self.n_batch:
            raise LstkError(E_INVALID, f"{n} sequences in a model of {self.n_batch} tokens a step")
        if min(seqs) < 0:
            raise LstkError(E_INVALID, "a sequence below 0")
        window, n_sink = _i32(window, "window"), _i32(n_sink, "n_sink")
        if n_sink < 0:
            raise LstkError(E_INVALID, "n_sink must be >= 0")
        tokens = {s: _ids32(prompts[s], f"the tokens of sequence {s}") for s in seqs}
        for s, t in tokens.items():
            if t.size == 0:
                raise LstkError(E_INVALID, f"sequence {s}: an empty prompt")
            if t.min() < 0 or t.max() >= V:
                raise LstkError(E_INVALID, f"sequence {s}: token id out of range")

        def setting(v, dtype):
            v = torch.as_tensor(v).flatten()
            if v.numel() not in (1, n):
                raise LstkError(E_INVALID, "a setting is one number, or one per prompt")
            w = v.to(dtype)
            if dtype is torch.int32 and not torch.equal(w.to(v.dtype), v):
                raise LstkError(E_INVALID, "top_k must be whole numbers of 32 bits")
            return w.expand(n).contiguous().to(self.device)

        how = dict(temperature=setting(temperature, torch.float32), top_k=setting(top_k, torch.int32),
                   top_p=setting(top_p, torch.float32), min_p=setting(min_p, torch.float32))
        before = {s: self.seq_len(s) for s in seqs}
        try:
            with torch.cuda.device(self.logits.device):
                logits = torch.empty(n, V, dtype=torch.float32, device=self.device)
                for i, s in enumerate(seqs):
                    self.decode(s, tokens[s], logits=logits[i])
                got = []
                for i in range(n_new):
                    u = torch.rand(n, device=self.device, generator=generator)
                    t = sample(logits, u, **how)[0].cpu().numpy()
                    if t.min() < 0:
                        raise LstkError(E_INVALID, f"sequence {seqs[int(t.argmin())]} has no finite logit at new token {i}")
                    got.append(t)
                    if i + 1 < n_new:
                        self.decode_batch(seqs, t, window=window, n_sink=n_sink, logits=logits)
        except BaseException:
            for s, length in before.items():
                try:
                    if self.seq_len(s) > length:
                        self.truncate_seq(s, length)
                except LstkError:
                    pass  # the first error is the one to report
            raise
        return {s: [int(t[i]) for t in got] for i, s in enumerate(seqs)}

    def fill_context(self, seq, n_cells, seed=0, stream=None):
        """Appends n_cells synthetic positions (seeded random K/V, no tokens run) to sequence seq."""
        _check(lib().lstk_model_fill_context(self._h, int(seq), int(n_cells), int(seed), _stream(stream)))

    def debug_capture(self, states):
        """Test hook: every forward copies the residual stream after each layer into the device tensor
        states ([n_layer][T][n_embd] f32, T the step's tokens); None turns it off."""
        self._capture = states
        _check(lib().lstk_model_debug_capture(self._h, None if states is None else _ptr(states)))

    def debug_capture_moe_in(self, states):
        """Test hook: every forward copies the residual stream entering each layer's MoE block (the router's
        input before ffn_norm) into the device tensor states ([n_layer][T][n_embd] f32); None turns it off."""
        self._capture_moe = states
        _check(lib().lstk_model_debug_capture_moe_in(self._h, None if states is None else _ptr(states)))

    def debug_options(self, rope_apart=False):
        """Test hook: rope_apart runs a single-token step's RoPE in its own launch (multi-pass attention
        chunks) instead of inside the attention launch (one-pass chunks)."""
        _check(lib().lstk_model_debug_options(self._h, 1 if rope_apart else 0))

    def set_trace(self, path):
        """Routing trace to `path` (LSTKRTE1, read by localstack_amd.trace); None closes it."""
        _check(lib().lstk_model_set_trace(self._h, None if path is None else os.fsencode(path)))

    def remove_seq(self, seq):
        _check(lib().lstk_model_remove_seq(self._h, int(seq)))

    def truncate_seq(self, seq, keep):
        _check(lib().lstk_model_truncate_seq(self._h, int(seq), int(keep)))

    def seq_len(self, seq):
        return lib().lstk_model_seq_len(self._h, int(seq))

    def set_timing(self, on):
        _check(lib().lstk_model_set_timing(self._h, 1 if on else 0))

    def timing(self):
        """(ms, launches) per stage: norms, Q/K/V + RoPE, attention, o-proj, output head."""
        ms = (ctypes.c_double * 5)()
        n = (ctypes.c_int64 * 5)()
        _check(lib().lstk_model_timing(self._h, ms, n))
        return list(ms), list(n)


_GGML_NP = {0: np.float32, 1: np.float16}
_GGML_NAME = {0: "F32", 1: "F16", 8: "Q8_0", 10: "Q2_K", 11: "Q3_K", 12: "Q4_K", 13: "Q5_K", 14: "Q6_K", 15: "Q8_K", 30: "BF16"}
# types lstk_dequant_f16 expands, with (values, bytes) per block
DEQUANT_TYPES = {0: (1, 4), 1: (1, 2), 8: (32, 34), 10: (256, 84), 11: (256, 110), 12: (256, 144), 13: (256, 176),
                 14: (256, 210)}


def dequant_f16(type_, data, n):
    """n values of ggml type type_ (bytes-like or uint8 array) to a float16 numpy array (lstk_dequant_f16)."""
    if type_ not in DEQUANT_TYPES:
        raise LstkError(E_INVALID, f"no dequantizer for {_GGML_NAME.get(type_, type_)}")
    per, nb = DEQUANT_TYPES[type_]
    src = np.ascontiguousarray(np.frombuffer(data, np.uint8) if not isinstance(data, np.ndarray) else data.view(np.uint8).ravel())
    if n % per or src.nbytes < n // per * nb:
        raise LstkError(E_INVALID, f"{n} values of {_GGML_NAME[type_]} need {-(-n // per) * nb} bytes, got {src.nbytes}")
    out = np.empty(n, np.float16)
    _check(lib().lstk_dequant_f16(type_, src.ctypes.data, n, out.ctypes.data))
    return out


class GgufFile:
    """A memory-mapped GGUF file (include/lstk_gguf.h), mirroring GgufModel (src/gguf_model.h:31-60).

    The mapping lives as long as this object or any array view taken from it (tensor_bytes /
    tensor_array keep the object alive), so a view never outlives the memory it reads."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        _check(lib().lstk_gguf_open(os.fsencode(path), ctypes.byref(h)))
        self._h = h
        self._destroy = lib().lstk_gguf_close
        self.path = path

    def __del__(self):
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    @property
    def arch(self):
        return lib().lstk_gguf_arch(self._h).decode()

    @property
    def version(self):
        return lib().lstk_gguf_version(self._h)

    @property
    def alignment(self):
        return lib().lstk_gguf_alignment(self._h)

    def has(self, key):
        return bool(lib().lstk_gguf_has(self._h, key.encode()))

    def get_int(self, key, default=0):
        return lib().lstk_gguf_get_int(self._h, key.encode(), int(default))

    def get_float(self, key, default=0.0):
        return lib().lstk_gguf_get_float(self._h, key.encode(), float(default))

    def get_str(self, key, default=""):
        r = lib().lstk_gguf_get_str(self._h, key.encode(), None)
        return default if r is None else r.decode()

    def _info(self, t):
        return {"name": t.name.decode(), "type": t.type, "ne": tuple(t.ne[:t.n_dims]), "offset": t.offset,
                "nbytes": t.nbytes, "data": t.data}

    def tensors(self):
        out = []
        for i in range(lib().lstk_gguf_n_tensors(self._h)):
            t = GgufTensor()
            _check(lib().lstk_gguf_tensor_at(self._h, i, ctypes.byref(t)))
            out.append(self._info(t))
        return out

    def tensor_info(self, name):
        t = GgufTensor()
        _check(lib().lstk_gguf_find_tensor(self._h, name.encode(), ctypes.byref(t)))
        return self._info(t)

    def tensor_bytes(self, name):
        """A read-only uint8 view of the tensor's bytes in the mapping (valid while the file is open)."""
        info = self.tensor_info(name)
        buf = (ctypes.c_uint8 * info["nbytes"]).from_address(info["data"])
        buf._owner = self  # the view keeps the mapping alive
        a = np.ctypeslib.as_array(buf)
        a.flags.writeable = False
        return a

    def tensor_array(self, name):
        """F32 / F16 tensors as numpy arrays shaped [ne[n-1]]...[ne[0]] (a view of the mapping)."""
        info = self.tensor_info(name)
        if info["type"] not in _GGML_NP:
            raise LstkError(E_INVALID, f"tensor {name} is {_GGML_NAME.get(info['type'], info['type'])}, not F32/F16")
        return self.tensor_bytes(name).view(_GGML_NP[info["type"]]).reshape(tuple(reversed(info["ne"])))

    def tensor_f16(self, name):
        """Any type lstk_dequant_f16 expands (F32, F16, Q8_0, Q2_K .. Q6_K) as a float16 array shaped
        [ne[n-1]]...[ne[0]]; F16 stays a view of the mapping, the others are dequantized copies."""
        info = self.tensor_info(name)
        if info["type"] == 1:
            return self.tensor_array(name)
        n = int(np.prod(info["ne"]))
        return dequant_f16(info["type"], self.tensor_bytes(name), n).reshape(tuple(reversed(info["ne"])))

    def qwen3_hparams(self):
        hp = Qwen3HParams()
        _check(lib().lstk_gguf_qwen3_hparams(self._h, ctypes.byref(hp)))
        return {n: getattr(hp, n) for n, _ in Qwen3HParams._fields_}

    def qwen3_experts(self, hp):
        c = Qwen3HParams(*(hp[n] for n, _ in Qwen3HParams._fields_))
        arr = (ExpertLayer * hp["n_layer"])()
        _check(lib().lstk_gguf_qwen3_experts(self._h, ctypes.byref(c), ctypes.cast(arr, ctypes.c_void_p)))
        return [((L.type_up, L.type_gate, L.type_down), L.host_up, L.host_gate, L.host_down) for L in arr]


def qwen3_dense_weights(g, hp):
    """The non-expert tensors of a qwen3moe GGUF as the forward pass takes them (qwen3_map_weights,
    src/qwen3.cpp:52-89): {"tok_embd", "output_norm", "output" (None when the head is tied), "layers": [...]}.
    Norms must be F32; the router is taken as F16 or F32 as stored; the matrices the forward pass multiplies
    in F16 (embedding, attention, output) are taken as stored when F16 and dequantized to F16 from F32, Q8_0,
    Q2_K, Q3_K, Q4_K, Q5_K or Q6_K (lstk_dequant_f16); other types are rejected with the tensor's name."""
    names = {t["name"] for t in g.tensors()}

    def dense(name, types=tuple(DEQUANT_TYPES), optional=False):
        if optional and name not in names:
            return None
        t = g.tensor_info(name)
        if t["type"] not in types:
            want = "/".join(_GGML_NAME[x] for x in types)
            raise LstkError(E_INVALID, f"tensor {name} is {_GGML_NAME.get(t['type'], t['type'])}; the forward pass takes {want}")
        if types == (0,) or (types == (0, 1) and t["type"] in types):
            return g.tensor_array(name)
        return g.tensor_f16(name)

    w = {"tok_embd": dense("token_embd.weight"), "output_norm": dense("output_norm.weight", (0,)),
         "output": dense("output.weight", optional=True), "layers": []}
    for l in range(hp["n_layer"]):
        p = f"blk.{l}."
        w["layers"].append({
            "attn_norm": dense(p + "attn_norm.weight", (0,)), "wq": dense(p + "attn_q.weight"),
            "wk": dense(p + "attn_k.weight"), "wv": dense(p + "attn_v.weight"), "wo": dense(p + "attn_output.weight"),
            "q_norm": dense(p + "attn_q_norm.weight", (0,), optional=True),
            "k_norm": dense(p + "attn_k_norm.weight", (0,), optional=True),
            "ffn_norm": dense(p + "ffn_norm.weight", (0,)), "gate_inp": dense(p + "ffn_gate_inp.weight", (0, 1))})
    return w


def load_qwen3_gguf(path, n_batch=64, kv_size=4096, device="cuda", pool_bytes=None, min_slots=None, streaming=False,
                    device_lru=False):
    """qwen3_load_hparams + qwen3_map_weights + the expert pool (src/qwen3.cpp:16-109,
    src/engine.cpp:31-173) from a qwen3moe GGUF: returns (hparams, ExpertStore, Qwen3Model, GgufFile).
    The experts go to the pool straight from the mapping; the dense tensors as qwen3_dense_weights takes them."""
    g = GgufFile(path)
    hp = g.qwen3_hparams()
    experts = g.qwen3_experts(hp)
    w = qwen3_dense_weights(g, hp)
    if min_slots is None:
        # a pool class never has fewer slots than one layer's experts (src/engine.cpp:114-116)
        min_slots = max(hp["n_expert"], 2 * hp["n_expert_used"] + 2) if streaming else 0
    if pool_bytes is None:
        pool_bytes = 0
        if streaming:
            # Engine::init's budget (src/engine.cpp:84-117) from this device's memory, the dense weights and
            # the KV cache
            import torch
            free_now, total = torch.cuda.mem_get_info(torch.device(device))
            table = sum((matrix_bytes(t[0], hp["n_ff_exp"], hp["n_embd"]) + matrix_bytes(t[1], hp["n_ff_exp"], hp["n_embd"]) +
                         matrix_bytes(t[2], hp["n_embd"], hp["n_ff_exp"])) * hp["n_expert"] for t, *_ in experts)
            dense_bytes = sum(a.nbytes for a in (w["tok_embd"], w["output_norm"], w["output"]) if a is not None)
            dense_bytes += sum(a.nbytes for lw in w["layers"] for a in lw.values() if a is not None)
            kv = hp["n_layer"] * ((kv_size + 255) // 256 * 256) * hp["n_head_kv"] * hp["head_dim"] * 2 * 2
            pool_bytes = default_pool_bytes(table, dense_bytes, kv, total, free_now)
    store = ExpertStore(hp["n_layer"], hp["n_embd"], hp["n_ff_exp"], hp["n_expert"], hp["n_expert_used"], n_batch,
                        experts, pool_bytes=pool_bytes, min_slots=min_slots, streaming=streaming,
                        device_lru=device_lru)
    model = Qwen3Model(hp, w, store, kv_size, n_batch, device=device)
    return hp, store, model, g
