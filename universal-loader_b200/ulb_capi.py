"""ctypes binding of libulb_cuda.so (include/ulb.h).

This is the binding a Python caller of the C ABI uses (the reference's own FFI for this
path is pybind11; see vulkangguf for that surface).  Device memory is handled through the
library itself (ulb_malloc / ulb_memcpy_*), so no other GPU framework is involved.
"""
import ctypes as C
import os
import re

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libulb_cuda.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "ulb.h")

OK, EINVAL, ENOMEM, ECUDA, ENCCL, ETIMEOUT, EFORMAT, EUNSUPPORTED = 0, -1, -2, -3, -4, -5, -6, -7
T_F32, T_F16, T_Q4_0, T_Q4_1, T_Q8_0, T_Q4_K, T_BF16 = 0, 1, 2, 3, 8, 12, 30
RNG_DRAFT, RNG_ACCEPT, RNG_RESID, RNG_FIRST = 1, 2, 3, 4

P = C.c_void_p


class AttnDesc(C.Structure):
    _fields_ = [("n_head", C.c_int), ("n_head_kv", C.c_int), ("head_dim", C.c_int),
                ("capacity", C.c_int), ("n_seq", C.c_int), ("scale", C.c_float)]


class Warp(C.Structure):
    _fields_ = [("temperature", C.c_float), ("top_k", C.c_int), ("top_p", C.c_float)]


class ModelDesc(C.Structure):
    _fields_ = [("n_layer", C.c_int), ("d_model", C.c_int), ("n_head", C.c_int),
                ("n_head_kv", C.c_int), ("head_dim", C.c_int), ("d_ff", C.c_int),
                ("n_vocab", C.c_int), ("rms_eps", C.c_float), ("rope_base", C.c_float),
                ("max_rows", C.c_int)]


class SpecDesc(C.Structure):
    _fields_ = [("n_seq", C.c_int), ("k", C.c_int), ("max_prompt", C.c_int),
                ("max_new", C.c_int), ("warp", Warp), ("seed", C.c_uint64),
                ("use_graphs", C.c_int), ("kv_pages", C.c_int), ("tree_width", C.c_int)]


class CacheDesc(C.Structure):
    _fields_ = [("dtype", C.c_int), ("n_layer", C.c_int), ("n_head_kv", C.c_int), ("head_dim", C.c_int),
                ("page", C.c_int), ("n_pages", C.c_int), ("n_seq", C.c_int), ("max_pages", C.c_int),
                ("layer_stride", C.c_int64), ("page_stride", C.c_int64), ("head_stride", C.c_int64),
                ("pos_stride", C.c_int64)]


class RopeDesc(C.Structure):
    _fields_ = [("head_dim", C.c_int), ("rot_dim", C.c_int), ("layout", C.c_int), ("scaling", C.c_int),
                ("base", C.c_double), ("factor", C.c_double), ("orig_len", C.c_double), ("beta_fast", C.c_double),
                ("beta_slow", C.c_double), ("low_freq", C.c_double), ("high_freq", C.c_double),
                ("attn_scale", C.c_double)]


class TreeDesc(C.Structure):
    _fields_ = [("n_head", C.c_int), ("rows", C.c_int), ("max_rows", C.c_int), ("max_len", C.c_int),
                ("mask_words", C.c_int), ("scale", C.c_float)]


class LogitsArgs(C.Structure):
    _fields_ = ([(n, C.c_int) for n in ("dtype", "V", "n_seq", "rows", "max_rows", "ld_in", "ld_out", "mask_words",
                                        "n_allow")] +
                [(n, P) for n in ("in_", "out", "row_start", "params", "history", "history_start", "prompt",
                                  "node_tokens", "mask", "bias_start", "bias_tokens", "bias_values", "allow",
                                  "row_allow")])


class NormRopeArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("M", C.c_int), ("n_head", C.c_int), ("n_head_kv", C.c_int), ("eps", C.c_float),
                ("q_row", C.c_int64), ("q_head", C.c_int64), ("k_row", C.c_int64), ("k_head", C.c_int64), ("q", P), ("k", P),
                ("q_weight", P), ("k_weight", P), ("pos", P)]


class QuantDesc(C.Structure):
    """A paged cache in 8 or 4 bits: format T_Q8_0 or T_Q4_1, dtype of q and outputs."""
    _fields_ = [(n, C.c_int) for n in ("format", "dtype", "n_head_kv", "head_dim", "page", "n_pages", "n_seq", "max_pages")]

    @property
    def row_bytes(self):
        n = C.c_int()
        check(lib().ulb_quant_row_bytes(C.byref(self), C.byref(n)))
        return n.value

    def pages_view(self, n_layer=1):
        """The pools as a CacheDesc of 16-bit elements, for page moves and the page book."""
        d = CacheDesc()
        check(lib().ulb_quant_pages(C.byref(self), n_layer, C.byref(d)))
        return d


class QuantAppendArgs(C.Structure):
    _fields_ = [("in_dtype", C.c_int), ("M", C.c_int), ("n_head", C.c_int), ("eps", C.c_float), ("q_row", C.c_int64),
                ("k_row", C.c_int64), ("v_row", C.c_int64)] + [
                (n, P) for n in ("q", "k", "v", "q_weight", "k_weight", "pos", "row_seq", "slot", "block_table", "q_out", "k_pool",
                                 "v_pool")]


class PromptDesc(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("dtype", "n_head", "n_head_kv", "head_dim", "n_seq", "q_rows", "k_rows", "max_q", "max_k")] + [
                ("scale", C.c_float), ("q_row", C.c_int64), ("k_row", C.c_int64), ("v_row", C.c_int64)]


ROPE_LAYOUTS = {"interleaved": 0, "half": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "wavelength": 4}
_DTYPE_IDS = {"f32": T_F32, "f16": T_F16, "bf16": T_BF16}


def dtype_id(name):
    """The type id of "f32", "f16" or "bf16"."""
    return _DTYPE_IDS[name]


_SIGS = {
    "ulb_last_error": (C.c_char_p, []),
    "ulb_version": (C.c_char_p, []),
    "ulb_init": (C.c_int, [C.c_int, C.POINTER(P)]),
    "ulb_destroy": (C.c_int, [P]),
    "ulb_stream": (P, [P]),
    "ulb_stream_sync": (C.c_int, [P]),
    "ulb_use_stream": (C.c_int, [P, P]),
    "ulb_rope_create": (C.c_int, [P, C.POINTER(RopeDesc), P, C.POINTER(P)]),
    "ulb_rope_free": (C.c_int, [P]),
    "ulb_rope_apply": (C.c_int, [P, P, C.c_int, P, C.c_int64, C.c_int64, P, C.c_int, C.c_int, C.c_int, P,
                                 C.c_int64, C.c_int64]),
    "ulb_rope_append": (C.c_int, [P, P, P, C.c_int, P, C.c_int64, P, C.c_int64, P, C.c_int64, C.c_int, P, P, P, P,
                                  C.c_int, P, P, P]),
    "ulb_tree_attention": (C.c_int, [P, P, P, P, P, P, P, P, P, P, P, P, P]),
    "ulb_norm_rope_apply": (C.c_int, [P, P, P, P, P]),
    "ulb_norm_rope_grad": (C.c_int, [P, P, P, P, P, P, P, P, P]),
    "ulb_quant_row_bytes": (C.c_int, [P, C.POINTER(C.c_int)]),
    "ulb_quant_pages": (C.c_int, [P, C.c_int, P]),
    "ulb_quant_append": (C.c_int, [P, P, P, P]),
    "ulb_quant_read": (C.c_int, [P, P, C.c_int, P, P, P, P, P, C.c_int, P, P]),
    "ulb_quant_attention": (C.c_int, [P, P, P, P, P, P, P, P, P, P, P, P, P]),
    "ulb_prompt_attention": (C.c_int, [P, P, P, P, P, P, P, P, P]),
    "ulb_pages_copy": (C.c_int, [P, P, P, P, P, C.c_int]),
    "ulb_pages_compact": (C.c_int, [P, P, P, P, P, P, P, P, C.c_int]),
    "ulb_pages_create": (C.c_int, [P, P, P, P, C.POINTER(P)]),
    "ulb_pages_free": (C.c_int, [P]),
    "ulb_pages_reserve": (C.c_int, [P, C.c_int, C.c_int, C.c_int]),
    "ulb_pages_fork": (C.c_int, [P, C.c_int, C.c_int, C.c_int]),
    "ulb_pages_truncate": (C.c_int, [P, C.c_int, C.c_int]),
    "ulb_pages_defrag": (C.c_int, [P, C.POINTER(C.c_int)]),
    "ulb_pages_info": (C.c_int, [P, C.POINTER(P), C.POINTER(C.c_int), C.c_int, C.POINTER(C.c_int)]),
    "ulb_logits_process": (C.c_int, [P, P]),
    "ulb_mem_used": (C.c_int, [P, C.POINTER(C.c_size_t)]),
    "ulb_malloc": (C.c_int, [P, C.c_size_t, C.POINTER(P)]),
    "ulb_free": (C.c_int, [P, P]),
    "ulb_memcpy_h2d": (C.c_int, [P, P, P, C.c_size_t]),
    "ulb_memcpy_d2h": (C.c_int, [P, P, P, C.c_size_t]),
    "ulb_event_create": (C.c_int, [P, C.POINTER(P)]),
    "ulb_event_record": (C.c_int, [P, P]),
    "ulb_event_elapsed_ms": (C.c_int, [P, P, C.POINTER(C.c_float)]),
    "ulb_event_destroy": (C.c_int, [P]),
    "ulb_tp_unique_id": (C.c_int, [P]),
    "ulb_tp_init": (C.c_int, [P, C.c_int, C.c_int, P]),
    "ulb_tp_set_timeout": (C.c_int, [P, C.c_int]),
    "ulb_wait_flag": (C.c_int, [P, P, C.c_int32, C.c_uint64]),
    "ulb_model_set_tp": (C.c_int, [P, C.c_int, C.c_int]),
    "ulb_capture_begin": (C.c_int, [P]),
    "ulb_capture_end": (C.c_int, [P, C.POINTER(P)]),
    "ulb_graph_launch": (C.c_int, [P, P]),
    "ulb_graph_free": (C.c_int, [P]),
    "ulb_tensor_upload": (C.c_int, [P, C.c_int, C.POINTER(C.c_uint64), P, C.c_size_t, C.POINTER(P)]),
    "ulb_tensor_free": (C.c_int, [P]),
    "ulb_tensor_info": (C.c_int, [P, C.POINTER(C.c_int), C.POINTER(C.c_uint64), C.POINTER(C.c_size_t)]),
    "ulb_dequant": (C.c_int, [P, P, P]),
    "ulb_qgemm": (C.c_int, [P, P, P, C.c_int, P, C.c_int]),
    "ulb_attention": (C.c_int, [P, C.POINTER(AttnDesc), P, P, P, P, P, C.c_int, C.c_int, P]),
    "ulb_attention_noalloc": (C.c_int, [P, C.POINTER(AttnDesc), P, P, P, P, P, C.c_int, C.c_int, P]),
    "ulb_attention_set_form": (C.c_int, [P, C.c_int]),
    "ulb_attention_paged": (C.c_int, [P, C.POINTER(AttnDesc), P, P, P, P, C.c_int, P, P, C.c_int, C.c_int, P]),
    "ulb_sample": (C.c_int, [P, P, C.c_int, C.c_int, C.c_int, C.POINTER(Warp), C.c_uint64,
                             C.c_uint32, C.c_uint32, C.c_uint32, P]),
    "ulb_spec_accept": (C.c_int, [P, P, P, P, C.c_int, C.c_int, C.c_int, C.POINTER(Warp),
                                  C.c_uint64, C.c_uint32, P, P]),
    "ulb_spec_tree_accept": (C.c_int, [P, P, P, P, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(Warp),
                                       C.c_uint64, C.c_uint32, P, P, P]),
    "ulb_model_create": (C.c_int, [P, C.POINTER(ModelDesc), C.POINTER(P)]),
    "ulb_model_set_weight": (C.c_int, [P, C.c_char_p, C.c_int, C.POINTER(C.c_uint64), P, C.c_size_t]),
    "ulb_model_finalize": (C.c_int, [P]),
    "ulb_model_free": (C.c_int, [P]),
    "ulb_model_weight_bytes": (C.c_int, [P, C.POINTER(C.c_size_t)]),
    "ulb_kv_alloc": (C.c_int, [P, P, C.c_int, C.c_int, C.POINTER(P)]),
    "ulb_kv_alloc_paged": (C.c_int, [P, P, C.c_int, C.c_int, C.c_int, C.POINTER(P)]),
    "ulb_kv_map": (C.c_int, [P, C.c_int, C.c_int, C.c_int, P]),
    "ulb_kv_free": (C.c_int, [P]),
    "ulb_model_forward": (C.c_int, [P, P, P, C.c_int, C.c_int, P, P, P, C.c_int, P, C.c_int]),
    "ulb_spec_create": (C.c_int, [P, P, P, C.POINTER(SpecDesc), C.POINTER(P)]),
    "ulb_spec_prefill": (C.c_int, [P, P, P]),
    "ulb_spec_run": (C.c_int, [P, C.c_int, C.POINTER(C.c_int)]),
    "ulb_spec_read": (C.c_int, [P, P, P, P]),
    "ulb_spec_free": (C.c_int, [P]),
    "ulb_spec_profile_round": (C.c_int, [P, C.POINTER(C.c_float)]),
    "ulb_spec_profile_round_ex": (C.c_int, [P, C.POINTER(C.c_float)]),
    "ulb_spec_read_rounds": (C.c_int, [P, C.c_int, C.c_int, P, C.POINTER(C.c_int)]),
    "ulb_spec_admit": (C.c_int, [P, C.c_int, P, C.c_int]),
    "ulb_spec_launch_count": (C.c_int, [P, C.POINTER(C.c_uint64)]),
}

_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("libulb_cuda.so is not built (run __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def header_functions():
    """Names of every function include/ulb.h declares."""
    with open(HEADER) as f:
        text = f.read()
    return sorted(set(re.findall(r"^ULB_API\s+[\w\s\*]+?\b(ulb_\w+)\s*\(", text, flags=re.M)))


class UlbError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__("ULB error %d: %s" % (code, msg))
        self.code = code


def check(rc):
    if rc != OK:
        raise UlbError(rc, lib().ulb_last_error().decode())
    return rc


def _ptr(a):
    return a.ctypes.data_as(P)


class DeviceBuffer:
    def __init__(self, ctx, nbytes):
        self.ctx = ctx
        self.nbytes = int(nbytes)
        p = P()
        check(lib().ulb_malloc(ctx.h, self.nbytes, C.byref(p)))
        self.ptr = p

    @property
    def value(self):
        return self.ptr.value

    def upload(self, arr):
        arr = np.ascontiguousarray(arr)
        assert arr.nbytes <= self.nbytes
        check(lib().ulb_memcpy_h2d(self.ctx.h, self.ptr, _ptr(arr), arr.nbytes))
        return self

    def download(self, dtype, shape):
        out = np.empty(shape, dtype)
        assert out.nbytes <= self.nbytes
        check(lib().ulb_memcpy_d2h(self.ctx.h, _ptr(out), self.ptr, out.nbytes))
        return out

    def free(self):
        if self.ptr is not None and self.ptr.value:
            lib().ulb_free(self.ctx.h, self.ptr)
        self.ptr = None


class Context:
    def __init__(self, device=0):
        h = P()
        check(lib().ulb_init(device, C.byref(h)))
        self.h = h
        self._stream = None

    def close(self):
        if self.h:
            lib().ulb_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def sync(self):
        check(lib().ulb_stream_sync(self.h))

    def use_stream(self, handle):
        """Enqueue later calls on another stream: a cudaStream_t as an integer, 0 the legacy default
        stream (as torch's current_stream().cuda_stream names it), None the context's own."""
        if handle != self._stream:
            check(lib().ulb_use_stream(self.h, None if handle is None else handle or 1))
            self._stream = handle

    # Paged cache operators (include/ulb.h).  Arrays are device addresses (integers, c_void_p, or
    # None where the header allows NULL); everything is enqueued, nothing is waited for.
    def tree_attention(self, cache, n_head, rows, max_rows, max_len, scale, q, k_pool, v_pool, block_table, row_start,
                       prefix, length, mask, mask_words, out, lse=None):
        d = TreeDesc(n_head, rows, max_rows, max_len, mask_words, scale)
        check(lib().ulb_tree_attention(self.h, C.byref(cache), C.byref(d), q, k_pool, v_pool, block_table, row_start, prefix,
                                       length, mask, out, lse))

    def quant_read(self, cache, dtype, k_pool, v_pool, block_table, row_seq, slot, M, k_out, v_out):
        check(lib().ulb_quant_read(self.h, C.byref(cache), dtype, k_pool, v_pool, block_table, row_seq, slot, M, k_out, v_out))

    def quant_attention(self, cache, n_head, rows, max_rows, max_len, scale, q, k_pool, v_pool, block_table, row_start, prefix,
                        length, mask, mask_words, out, lse=None):
        d = TreeDesc(n_head, rows, max_rows, max_len, mask_words, scale)
        check(lib().ulb_quant_attention(self.h, C.byref(cache), C.byref(d), q, k_pool, v_pool, block_table, row_start, prefix,
                                        length, mask, out, lse))

    def prompt_attention(self, dtype, n_head, n_head_kv, head_dim, n_seq, q_rows, k_rows, max_q, max_k, scale, q, k, v, q_start,
                         k_start, out, lse=None, q_row=0, k_row=0, v_row=0):
        d = PromptDesc(dtype, n_head, n_head_kv, head_dim, n_seq, q_rows, k_rows, max_q, max_k, scale, q_row, k_row, v_row)
        check(lib().ulb_prompt_attention(self.h, C.byref(d), q, k, v, q_start, k_start, out, lse))

    def pages_copy(self, cache, k_pool, v_pool, moves, n):
        check(lib().ulb_pages_copy(self.h, C.byref(cache), k_pool, v_pool, moves, n))

    def pages_compact(self, cache, k_pool, v_pool, block_table, base, count, src, max_src):
        check(lib().ulb_pages_compact(self.h, C.byref(cache), k_pool, v_pool, block_table, base, count, src, max_src))

    def logits_process(self, dtype, logits, out, V, n_seq, rows, row_start, max_rows=None, ld_in=None, ld_out=None,
                       params=None, history=None, history_start=None, prompt=None, node_tokens=None, words=None,
                       n_words=0, bias_start=None, bias_tokens=None, bias_values=None, allow=None, row_allow=None,
                       n_allow=0):
        a = LogitsArgs(dtype, V, n_seq, rows, rows if max_rows is None else max_rows, V if ld_in is None else ld_in,
                       V if ld_out is None else ld_out, n_words, n_allow, logits, out, row_start, params, history,
                       history_start, prompt, node_tokens, words, bias_start, bias_tokens, bias_values, allow, row_allow)
        check(lib().ulb_logits_process(self.h, C.byref(a)))

    def buffer(self, arr=None, nbytes=None):
        if arr is not None:
            arr = np.ascontiguousarray(arr)
            return DeviceBuffer(self, max(arr.nbytes, 16)).upload(arr)
        return DeviceBuffer(self, max(int(nbytes), 16))

    def upload_tensor(self, ggml_type, ne, raw):
        raw = np.ascontiguousarray(raw, np.uint8)
        ne4 = (C.c_uint64 * 4)(*(list(ne) + [1] * (4 - len(ne))))
        t = P()
        check(lib().ulb_tensor_upload(self.h, ggml_type, ne4, _ptr(raw), raw.nbytes, C.byref(t)))
        return t

    def free_tensor(self, t):
        lib().ulb_tensor_free(t)

    def dequant(self, t, n_rows, n_cols):
        out = self.buffer(nbytes=n_rows * n_cols * 4)
        check(lib().ulb_dequant(self.h, t, out.ptr))
        r = out.download(np.float32, (n_rows, n_cols))
        out.free()
        return r

    def qgemm(self, t, x16, N):
        x16 = np.ascontiguousarray(x16, np.float16)
        M = x16.shape[0]
        xb = self.buffer(x16)
        yb = self.buffer(nbytes=max(M, 1) * N * 4)
        check(lib().ulb_qgemm(self.h, t, xb.ptr, M, yb.ptr, N))
        y = yb.download(np.float32, (M, N))
        xb.free()
        yb.free()
        return y

    def event(self):
        e = P()
        check(lib().ulb_event_create(self.h, C.byref(e)))
        return e

    def record(self, e):
        check(lib().ulb_event_record(self.h, e))

    def capture(self, fn):
        """Record the device work of fn() into a CUDA graph (returns the graph handle)."""
        check(lib().ulb_capture_begin(self.h))
        try:
            fn()
        finally:
            g = P()
            rc = lib().ulb_capture_end(self.h, C.byref(g))
        check(rc)
        return g

    def time_graph(self, g, reps=10):
        """Device milliseconds of one replay of g (CUDA events, after one warm replay)."""
        check(lib().ulb_graph_launch(self.h, g))
        a, b = self.event(), self.event()
        self.record(a)
        for _ in range(reps):
            check(lib().ulb_graph_launch(self.h, g))
        self.record(b)
        self.sync()
        ms = self.elapsed_ms(a, b) / reps
        lib().ulb_event_destroy(a)
        lib().ulb_event_destroy(b)
        return ms

    def elapsed_ms(self, a, b):
        ms = C.c_float()
        check(lib().ulb_event_elapsed_ms(a, b, C.byref(ms)))
        return ms.value


class Rope:
    """Rotary positions of one model (ulb_rope): the handle a program keeps beside its weights."""

    def __init__(self, ctx, head_dim, rot_dim=None, layout="interleaved", base=10000.0, scaling="none", factor=1.0,
                 orig_len=0, beta_fast=32.0, beta_slow=1.0, low_freq=1.0, high_freq=4.0, attn_scale=0.0,
                 freq_factors=None):
        self.ctx = ctx
        rot = head_dim if rot_dim is None else rot_dim
        d = RopeDesc(head_dim, rot, ROPE_LAYOUTS[layout], ROPE_SCALINGS[scaling], base, factor, orig_len, beta_fast,
                     beta_slow, low_freq, high_freq, attn_scale)
        if freq_factors is not None:
            freq_factors = np.ascontiguousarray(freq_factors, np.float32)
            if freq_factors.shape != (rot // 2,):
                raise ValueError("freq_factors holds one value a pair (%d)" % (rot // 2))
        h = P()
        check(lib().ulb_rope_create(ctx.h, C.byref(d), None if freq_factors is None else _ptr(freq_factors), C.byref(h)))
        self.h = h

    def apply(self, dtype, x, M, n_head, pos, out, x_row=0, x_head=0, out_row=0, out_head=0, inverse=False):
        check(lib().ulb_rope_apply(self.ctx.h, self.h, dtype, x, x_row, x_head, pos, M, n_head, int(inverse), out, out_row,
                                   out_head))

    def append(self, cache, in_dtype, q, k, v, n_head, pos, row_seq, slot, block_table, M, q_out, k_pool, v_pool, q_row=0,
               k_row=0, v_row=0):
        check(lib().ulb_rope_append(self.ctx.h, self.h, C.byref(cache), in_dtype, q, q_row, k, k_row, v, v_row, n_head, pos,
                                    row_seq, slot, block_table, M, q_out, k_pool, v_pool))

    def norm_apply(self, dtype, q, k, M, n_head, n_head_kv, q_weight, k_weight, eps, pos, q_out, k_out, q_row=0, q_head=0, k_row=0,
                   k_head=0):
        """q and k heads normed, weighted and turned."""
        a = NormRopeArgs(dtype, M, n_head, n_head_kv, eps, q_row, q_head, k_row, k_head, q, k, q_weight, k_weight, pos)
        check(lib().ulb_norm_rope_apply(self.ctx.h, self.h, C.byref(a), q_out, k_out))

    def norm_grad(self, dtype, q, k, dq_out, dk_out, M, n_head, n_head_kv, q_weight, k_weight, eps, pos, dq, dk, dq_weight,
                  dk_weight, q_row=0, q_head=0, k_row=0, k_head=0):
        """norm_apply's gradient with respect to q, k and the weights."""
        a = NormRopeArgs(dtype, M, n_head, n_head_kv, eps, q_row, q_head, k_row, k_head, q, k, q_weight, k_weight, pos)
        check(lib().ulb_norm_rope_grad(self.ctx.h, self.h, C.byref(a), dq_out, dk_out, dq, dk, dq_weight, dk_weight))

    def quant_append(self, cache, in_dtype, q, k, v, n_head, pos, row_seq, slot, block_table, M, q_out, k_pool, v_pool, q_row=0,
                     k_row=0, v_row=0, q_weight=None, k_weight=None, eps=1e-6):
        """append into a quantised cache, q and k normed first where their weights are given."""
        a = QuantAppendArgs(in_dtype, M, n_head, eps, q_row, k_row, v_row, q, k, v, q_weight, k_weight, pos, row_seq, slot,
                            block_table, q_out, k_pool, v_pool)
        check(lib().ulb_quant_append(self.ctx.h, self.h, C.byref(cache), C.byref(a)))

    def close(self):
        if self.h:
            lib().ulb_rope_free(self.h)
            self.h = None


class Pages:
    """The book of a cache's pages (ulb_pages): who holds which page, shared pages, the block table."""

    def __init__(self, ctx, cache, k_pool, v_pool):
        self.ctx = ctx
        h = P()
        check(lib().ulb_pages_create(ctx.h, C.byref(cache), k_pool, v_pool, C.byref(h)))
        self.h = h

    def reserve(self, seq, start, to):
        check(lib().ulb_pages_reserve(self.h, seq, start, to))

    def fork(self, src, dst, n):
        check(lib().ulb_pages_fork(self.h, src, dst, n))

    def truncate(self, seq, n):
        check(lib().ulb_pages_truncate(self.h, seq, n))

    def defrag(self):
        n = C.c_int()
        check(lib().ulb_pages_defrag(self.h, C.byref(n)))
        return n.value

    @property
    def table(self):
        """Device address of the block table."""
        t = P()
        check(lib().ulb_pages_info(self.h, C.byref(t), None, -1, None))
        return t.value

    @property
    def free(self):
        n = C.c_int()
        check(lib().ulb_pages_info(self.h, None, C.byref(n), -1, None))
        return n.value

    def mapped(self, seq):
        n = C.c_int()
        check(lib().ulb_pages_info(self.h, None, None, seq, C.byref(n)))
        return n.value

    def close(self):
        if self.h:
            lib().ulb_pages_free(self.h)
            self.h = None
