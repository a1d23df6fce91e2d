"""MI355X (gfx950) full-attention hot path of the qwen35moe engine.

Python host mirror of the C ABI in include/sqattn.h, named after the ggml ops
and the engine objects it stands in for (reference: src/backend/ffi.rs:363-405,
src/engine/kv.rs). Device memory and streams come from PyTorch; every kernel
runs from libsqattn.so, which sits next to this file. If the library is
missing the first call fails: there is no CPU fallback. Calls that give their
output and workspace and use the current stream go through _sqahost.so
(binding/host.cpp) where it was built, the others build their descriptors here.

Tensor conventions (torch shapes, C order, all on the GPU):
  q       float32 (n_q, H, D)             the engine's [D, H, n_q] Q
  cache   uint8   (rows, Hkv, D//32*18)   one q4_0 K or V cache (kv.rs:95-148)
  mask    float16 (n_q_pad, n_kv)         0 / -inf, or None
  out     float32 (n_q, H, D)             [D, H, n_q] attention output
  pool    uint8   (n_pages, page, Hkv, D//32*18)  one paged q4_0 K or V cache of a batch
  table   int32   (B, W)                  page ids of every request
"""
import collections
import ctypes
import importlib.machinery
import importlib.util
import math
import struct
import os

import torch

__all__ = [
    "Tensor", "lib", "last_error", "SqaError", "set_rows_q4_0", "flash_attn_ext",
    "flash_attn_ext_causal", "flash_attn_ext_static", "sigmoid_mul", "fill_causal_mask", "supports_flash_attn_ext",
    "flash_attn_workspace_size", "out_proj", "out_proj_workspace_size", "KvCache", "cache_view", "row_bytes", "profile_begin", "profile_end",
    "profile_get", "Rope", "rope_params", "rope_norm_set_rows_q4_0", "rope_norm_f32",
    "paged_plan", "paged_attn", "paged_attn_workspace_size", "supports_paged_attn", "PagedStep", "PagedKvCache",
    "lora_add", "supports_lora_add", "get_rows_q4_0", "move_rows_q4_0",
    "paged_share", "paged_attn_shared", "paged_attn_shared_workspace_size", "supports_paged_attn_shared", "PagedShare",
]

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsqattn.so")
HOST_PATH = os.path.join(HERE, "_sqahost.so")

TYPE_F32, TYPE_F16, TYPE_Q4_0, TYPE_Q4_K, TYPE_I32, TYPE_I64 = 0, 1, 2, 12, 26, 27
Q4_K_BLOCK = 144  # bytes per 256-value Q4_K super-block
QK4_0 = 32
Q4_0_BLOCK = 18
KV_PAD = 256
STATUS = {0: "ok", 1: "invalid argument", 2: "unsupported configuration", 3: "workspace too small",
          4: "HIP runtime error", 5: "KV cache overflow", 6: "argument out of range"}


class SqaError(RuntimeError):
    def __init__(self, status, msg):
        super().__init__(f"{STATUS.get(status, status)}: {msg}")
        self.status = status


_TENSOR_LAYOUT = struct.Struct("<ii4q4QQ")  # type, pad_, ne[4], nb[4], data


class Tensor(ctypes.Structure):
    """sqa_tensor: ggml's {type, ne[4], nb[4], data} (reference ffi.rs:22-39)."""

    _fields_ = [
        ("type", ctypes.c_int32),
        ("pad_", ctypes.c_int32),
        ("ne", ctypes.c_int64 * 4),
        ("nb", ctypes.c_uint64 * 4),
        ("data", ctypes.c_void_p),
    ]

    @staticmethod
    def make(ttype, ne, nb, ptr):
        """Fields packed in one go: a decode step builds five of these per call."""
        ne = tuple(ne) + (1,) * (4 - len(ne))
        nb = list(nb)
        while len(nb) < 4:
            nb.append(nb[-1] * ne[len(nb) - 1])
        return Tensor.from_buffer_copy(_TENSOR_LAYOUT.pack(ttype, 0, *ne, *nb, ptr))


class Rope(ctypes.Structure):
    """sqa_rope: the ggml_rope_multi parameters of RopeParams (reference attn.rs:30-65)."""

    _fields_ = [
        ("n_rot", ctypes.c_int32),
        ("sections", ctypes.c_int32 * 4),
        ("freq_base", ctypes.c_float),
        ("freq_scale", ctypes.c_float),
        ("ext_factor", ctypes.c_float),
        ("attn_factor", ctypes.c_float),
    ]


def rope_params(n_rot, sections, freq_base, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0):
    """RopeParams::text (reference attn.rs:46-64): no YaRN ramp, attn_factor 1."""
    r = Rope()
    r.n_rot = int(n_rot)
    for i in range(4):
        r.sections[i] = int(sections[i])
    r.freq_base, r.freq_scale, r.ext_factor, r.attn_factor = freq_base, freq_scale, ext_factor, attn_factor
    return r


_lib = None


def lib():
    """The loaded libsqattn.so (raises if it was never built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: run __graft_entry__.build() first")
        L = ctypes.CDLL(LIB_PATH)
        P = ctypes.POINTER(Tensor)
        vp, sz, i64, f32, i32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int64, ctypes.c_float, ctypes.c_int32
        sigs = {
            "sqa_version": (ctypes.c_char_p, []),
            "sqa_last_error": (ctypes.c_char_p, []),
            "sqa_status_string": (ctypes.c_char_p, [ctypes.c_int]),
            "sqa_set_rows_q4_0": (ctypes.c_int, [P, P, P, vp]),
            "sqa_supports_set_rows": (ctypes.c_int, [P, P, P]),
            "sqa_rope_norm_set_rows_q4_0": (ctypes.c_int, [P, P, P, f32, P, ctypes.POINTER(Rope), P, vp]),
            "sqa_rope_norm_f32": (ctypes.c_int, [P, P, P, f32, P, ctypes.POINTER(Rope), vp]),
            "sqa_supports_rope_norm": (ctypes.c_int, [P, P, P, P, ctypes.POINTER(Rope), P]),
            "sqa_flash_attn_ext": (ctypes.c_int, [P, P, P, P, f32, f32, f32, P, vp, sz, vp]),
            "sqa_flash_attn_ext_workspace_size": (sz, [P, P, P, P]),
            "sqa_supports_flash_attn_ext": (ctypes.c_int, [P, P, P, P, f32, f32, f32, P]),
            "sqa_flash_attn_ext_causal": (ctypes.c_int, [P, P, P, i64, P, f32, P, vp, sz, vp]),
            "sqa_flash_attn_ext_static": (ctypes.c_int, [P, P, P, P, f32, f32, f32, P, vp]),
            "sqa_sigmoid_mul": (ctypes.c_int, [P, P, P, vp]),
            "sqa_out_proj_workspace_size": (sz, [P, P]),
            "sqa_supports_out_proj": (ctypes.c_int, [P, P, P, P]),
            "sqa_out_proj": (ctypes.c_int, [P, P, P, P, vp, sz, vp]),
            "sqa_fill_causal_mask": (ctypes.c_int, [P, i64, vp]),
            "sqa_kv_cache_layer_bytes": (sz, [i64, i64, i64]),
            "sqa_kv_cache_create": (vp, [i32, i64, i64, i64, ctypes.POINTER(vp), ctypes.POINTER(vp)]),
            "sqa_kv_cache_destroy": (None, [vp]),
            "sqa_kv_cache_n_used": (i64, [vp]),
            "sqa_kv_cache_step_start": (i64, [vp]),
            "sqa_kv_cache_n_kv_padded": (i64, [vp]),
            "sqa_kv_cache_n_kv_padded_after": (i64, [vp, i64]),
            "sqa_kv_cache_begin_step": (ctypes.c_int, [vp, i64]),
            "sqa_kv_cache_rewind_to": (ctypes.c_int, [vp, i64]),
            "sqa_kv_cache_reset": (None, [vp]),
            "sqa_kv_cache_k_view": (ctypes.c_int, [vp, i32, P]),
            "sqa_kv_cache_v_view": (ctypes.c_int, [vp, i32, P]),
            "sqa_kv_cache_append": (ctypes.c_int, [vp, i32, P, P, P, vp]),
            "sqa_paged_plan": (ctypes.c_int, [P, P, P, P, P, i32, P, P, P, P, P, P, vp]),
            "sqa_paged_attn": (ctypes.c_int, [P, P, P, P, P, P, P, i64, f32, f32, f32, P, P, vp, sz, vp]),
            "sqa_paged_attn_workspace_size": (sz, [P, P, P, i64]),
            "sqa_supports_paged_attn": (ctypes.c_int, [P, P, P, P, i64, f32, f32, f32, P]),
            "sqa_get_rows_q4_0": (ctypes.c_int, [P, P, P, vp]),
            "sqa_supports_get_rows": (ctypes.c_int, [P, P, P]),
            "sqa_move_rows_q4_0": (ctypes.c_int, [P, P, P, P, P, ctypes.POINTER(Rope), vp]),
            "sqa_supports_move_rows": (ctypes.c_int, [P, P, P, P, P, ctypes.POINTER(Rope)]),
            "sqa_paged_share": (ctypes.c_int, [P] * 9 + [vp]),
            "sqa_paged_attn_shared": (ctypes.c_int, [P] * 13 + [i64, f32, f32, f32, P, P, vp, sz, vp]),
            "sqa_paged_attn_shared_workspace_size": (sz, [P, P, P, P, i64]),
            "sqa_supports_paged_attn_shared": (ctypes.c_int, [P, P, P, P, P, i64, f32, f32, f32, P]),
            "sqa_lora_add": (ctypes.c_int, [P, P, P, P, P, P, P, P, vp]),
            "sqa_supports_lora_add": (ctypes.c_int, [P, P, P, P, P, P]),
            "sqa_profile_begin": (ctypes.c_int, [i32]),
            "sqa_profile_end": (ctypes.c_int, []),
            "sqa_profile_get": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_double),
                                               ctypes.POINTER(i64)]),
        }
        for name, (res, args) in sigs.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


_FLOATS = {torch.float32: (TYPE_F32, 4), torch.float16: (TYPE_F16, 2)}
_host = None


class _General:
    """Stands in for the native binding where it was not built: leaves every call
    to the ctypes path."""

    def __getattr__(self, name):
        return lambda *args: None


def _load_host():
    """The native binding of the hot entry points. A build without torch's headers
    has none; one that is there has to load."""
    global _host
    lib()  # the binding links against the library beside it
    if not os.path.exists(HOST_PATH):
        _host = _General()
        return _host
    loader = importlib.machinery.ExtensionFileLoader("_sqahost", HOST_PATH)
    mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_sqahost", loader))
    loader.exec_module(mod)
    _host = mod
    return mod


def last_error():
    return lib().sqa_last_error().decode()


def _check(rc):
    if rc != 0:
        raise SqaError(rc, last_error())


def _stream(stream):
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


def _stream_of(stream, device):
    """Makes a call's stream (None: the device's current one) and its device the current ones."""
    if stream is None:
        return torch.cuda.device(device)
    if not isinstance(stream, torch.cuda.Stream):
        handle = _stream(stream)
        handle = getattr(handle, "value", handle)
        stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream)


def _make(stream, device, make):
    """make() on the stream that a call runs on, for the tensors that it makes itself: what fills one is
    then in order with the kernels, and freed memory goes to tensors of that stream, behind them."""
    if stream is None:
        return make()
    with _stream_of(stream, device):
        t = make()
    if t is not None:  # the caller's own stream may read it until it is freed
        t.record_stream(torch.cuda.current_stream(t.device))
    return t


def _ref(t):
    return ctypes.byref(t) if t is not None else None


def row_bytes(D, Hkv=1):
    return D // QK4_0 * Q4_0_BLOCK * Hkv


# ------------------------------------------------------------ descriptors ---

def q_desc(q):
    """(n_q, H, D) float32 -> ggml view [D, n_q, H] (the permute of attn.rs:232)."""
    n_q, H, D = q.shape
    s = q.stride()
    return Tensor.make(TYPE_F32, [D, n_q, H, 1], [4, s[0] * 4, s[1] * 4], q.data_ptr())


def cache_view(cache, n_kv):
    """(rows, Hkv, D//32*18) uint8 -> q4_0 view [D, n_kv, Hkv] (kv.rs:401-447 permuted)."""
    rows, Hkv, rb = cache.shape
    D = rb // Q4_0_BLOCK * QK4_0
    assert cache.dtype == torch.uint8 and cache.is_contiguous() and n_kv <= rows
    return Tensor.make(TYPE_Q4_0, [D, n_kv, Hkv, 1], [Q4_0_BLOCK, Hkv * rb, rb], cache.data_ptr())


def out_desc(out):
    n_q, H, D = out.shape
    assert out.is_contiguous()
    return Tensor.make(TYPE_F32, [D, H, n_q, 1], [4, D * 4, H * D * 4], out.data_ptr())


def mask_desc(mask):
    if mask is None:
        return None
    n_rows, n_kv = mask.shape
    assert mask.dtype == torch.float16 and mask.stride(1) == 1
    return Tensor.make(TYPE_F16, [n_kv, n_rows, 1, 1], [2, mask.stride(0) * 2], mask.data_ptr())


# ---------------------------------------------------------------------- ops --

def set_rows_q4_0(cache, src, idx, stream=None):
    """cache[idx[i]] = quantize_row_q4_0(src[i]) (GGML_OP_SET_ROWS, kv.rs:356-396).

    cache: uint8 (rows, ..., row_bytes) contiguous; src: float32 (n, ne0); idx: int64 (n,)."""
    if stream is None:
        rc = (_host or _load_host()).set_rows(cache, src, idx)
        if rc is not None:
            if rc:
                _check(rc)
            return cache
    rows = cache.shape[0]
    rb = cache[0].numel()
    ne0 = src.shape[1]
    assert rb == ne0 // QK4_0 * Q4_0_BLOCK, "row length mismatch"
    td = Tensor.make(TYPE_Q4_0, [ne0, rows], [Q4_0_BLOCK, rb], cache.data_ptr())
    ts = Tensor.make(TYPE_F32, [ne0, src.shape[0]], [4, src.stride(0) * 4], src.data_ptr())
    ti = Tensor.make(TYPE_I64, [idx.shape[0]], [idx.stride(0) * 8], idx.data_ptr())
    _check(lib().sqa_set_rows_q4_0(ctypes.byref(td), ctypes.byref(ts), ctypes.byref(ti), _stream(stream)))
    return cache


def get_rows_q4_0(cache, idx, out=None, dtype=torch.float32, stream=None):
    """out[i] = the values of cache row idx[i] (GGML_OP_GET_ROWS of a q4_0 cache): set_rows_q4_0's counterpart.

    cache: uint8 (rows, ..., row_bytes) contiguous, rows of whole blocks; idx: int64 (n,), an index outside the cache
    reads as zeros; out: float32 or float16 (n, ne0) with contiguous elements, made here of dtype where it is not given."""
    if stream is None and out is not None:
        rc = (_host or _load_host()).get_rows(cache, idx, out)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    _need(cache.dim() >= 2 and cache.dtype == torch.uint8 and cache.is_contiguous() and
          math.prod(cache.shape[1:]) % Q4_0_BLOCK == 0, "cache must be contiguous uint8 (rows, ...), rows of whole 18-byte blocks")
    with _on(cache.device, idx=idx, out=out):
        _need(idx.dim() == 1 and idx.dtype == torch.int64, "idx must be int64 (n,)")
        rb, n = math.prod(cache.shape[1:]), idx.shape[0]
        ne0 = rb // Q4_0_BLOCK * QK4_0
        if out is None:
            _need(dtype in _FLOATS, "dtype must be float32 or float16")
            out = _make(stream, cache.device, lambda: torch.empty((n, ne0), dtype=dtype, device=cache.device))
        _need(out.dim() == 2 and out.dtype in _FLOATS and (out.shape[1] <= 1 or out.stride(1) == 1),
              "out must be float32 or float16 (n, ne0) with contiguous elements")
        code, size = _FLOATS[out.dtype]
        to = Tensor.make(code, [out.shape[1], out.shape[0]], [size, out.stride(0) * size], out.data_ptr())
        ts = Tensor.make(TYPE_Q4_0, [ne0, cache.shape[0]], [Q4_0_BLOCK, rb], cache.data_ptr())
        ti = Tensor.make(TYPE_I64, [n], [idx.stride(0) * 8], idx.data_ptr())
        _check(lib().sqa_get_rows_q4_0(ctypes.byref(to), ctypes.byref(ts), ctypes.byref(ti), _stream(stream)))
    return out


def _heads_desc(cache, name):
    _need(cache.dim() == 3 and cache.dtype == torch.uint8 and cache.is_contiguous() and cache.shape[2] % Q4_0_BLOCK == 0,
          f"{name} must be contiguous uint8 (rows, n_head, D // 32 * 18)")
    rows, heads, rb = cache.shape
    return Tensor.make(TYPE_Q4_0, [rb // Q4_0_BLOCK * QK4_0, heads, rows], [Q4_0_BLOCK, rb, heads * rb], cache.data_ptr())


def move_rows_q4_0(dst, src, to, from_, delta=None, rope=None, stream=None):
    """dst[to[i]] = src[from_[i]], with a rope the heads' first n_rot dims rotated on by delta and quantized again: cached
    keys at other positions (a context that drops its oldest part, a cached passage behind another prompt).

    dst, src: uint8 (rows, n_head, D//32*18) contiguous, dst may be src; to, from_: int64 (n,), entries outside a cache
    are skipped; delta: int32 (4*n,), how far the positions t, h, w, e move; without delta and rope rows are copied (V).
    In place a row that one entry reads must be no other entry's to (from_ == to is fine)."""
    if stream is None and (rope is None or isinstance(rope, Rope)):
        rc = (_host or _load_host()).move_rows(dst, src, to, from_, delta, rope)
        if rc is not None:
            if rc:
                _check(rc)
            return dst
    with _on(dst.device, src=src, to=to, from_=from_, delta=delta):
        td, ts = _heads_desc(dst, "dst"), _heads_desc(src, "src")
        for t, name in ((to, "to"), (from_, "from_")):
            _need(t.dim() == 1 and t.dtype == torch.int64, f"{name} must be int64 (n,)")
        tt, tf = (Tensor.make(TYPE_I64, [t.shape[0]], [t.stride(0) * 8], t.data_ptr()) for t in (to, from_))
        tl = None if delta is None else _vec(delta, torch.int32, "delta")
        _check(lib().sqa_move_rows_q4_0(ctypes.byref(td), ctypes.byref(ts), ctypes.byref(tt), ctypes.byref(tf), _ref(tl),
                                        _ref(rope), _stream(stream)))
    return dst


def _producer_descs(src, norm_w, pos):
    n_tok, n_head, D = src.shape
    ts = Tensor.make(TYPE_F32, [D, n_head, n_tok], [4, src.stride(1) * 4, src.stride(0) * 4], src.data_ptr())
    tw = None if norm_w is None else Tensor.make(TYPE_F32, [D], [4], norm_w.data_ptr())
    tp = Tensor.make(TYPE_I32, [pos.shape[0]], [4], pos.data_ptr())
    return ts, tw, tp


def rope_norm_set_rows_q4_0(cache, src, norm_w, eps, pos, rope, idx, stream=None):
    """K producer (reference attn.rs:166-200 + kv.rs:313-399): per-head RMSNorm times
    norm_w, IMROPE with positions pos, q4_0 quantize-on-write into cache rows idx.

    cache: uint8 (rows, ..., n_head*D//32*18) contiguous; src: float32 (n_tok, n_head, D)
    with contiguous rows; norm_w: float32 (D,) or None; pos: int32 (4*n_tok,);
    idx: int64 (n_tok,)."""
    if stream is None and idx is not None and isinstance(rope, Rope):
        rc = (_host or _load_host()).rope_norm(cache, src, norm_w, eps, pos, rope, idx)
        if rc is not None:
            if rc:
                _check(rc)
            return cache
    n_tok, n_head, D = src.shape
    rows = cache.shape[0]
    rb = cache[0].numel()
    assert rb == n_head * D // QK4_0 * Q4_0_BLOCK, "row length mismatch"
    ts, tw, tp = _producer_descs(src, norm_w, pos)
    td = Tensor.make(TYPE_Q4_0, [n_head * D, rows], [Q4_0_BLOCK, rb], cache.data_ptr())
    ti = Tensor.make(TYPE_I64, [idx.shape[0]], [idx.stride(0) * 8], idx.data_ptr())
    _check(lib().sqa_rope_norm_set_rows_q4_0(ctypes.byref(td), ctypes.byref(ts), _ref(tw), eps, ctypes.byref(tp),
                                             ctypes.byref(rope), ctypes.byref(ti), _stream(stream)))
    return cache


def rope_norm_f32(out, src, norm_w, eps, pos, rope, stream=None):
    """Q producer (reference attn.rs:166-199): out float32 (n_tok, n_head, D) contiguous."""
    if stream is None and isinstance(rope, Rope):
        rc = (_host or _load_host()).rope_norm(out, src, norm_w, eps, pos, rope, None)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    n_tok, n_head, D = src.shape
    ts, tw, tp = _producer_descs(src, norm_w, pos)
    to = Tensor.make(TYPE_F32, [D, n_head, n_tok], [4, D * 4, n_head * D * 4], out.data_ptr())
    _check(lib().sqa_rope_norm_f32(ctypes.byref(to), ctypes.byref(ts), _ref(tw), eps, ctypes.byref(tp),
                                   ctypes.byref(rope), _stream(stream)))
    return out


def flash_attn_workspace_size(q, k_cache, n_kv):
    n_q, H, D = q.shape
    tq, tk = q_desc(q), cache_view(k_cache, n_kv)
    to = Tensor.make(TYPE_F32, [D, H, n_q, 1], [4, D * 4, H * D * 4], 16)
    return int(lib().sqa_flash_attn_ext_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tk),
                                                       ctypes.byref(to)))


def supports_flash_attn_ext(q, k_cache, n_kv, mask=None, scale=None, max_bias=0.0, softcap=0.0):
    n_q, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    tq, tk = q_desc(q), cache_view(k_cache, n_kv)
    to = Tensor.make(TYPE_F32, [D, H, n_q, 1], [4, D * 4, H * D * 4], 16)
    tm = mask_desc(mask)
    return bool(lib().sqa_supports_flash_attn_ext(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tk),
                                                  _ref(tm), scale, max_bias, softcap, ctypes.byref(to)))


def _workspace(nbytes, device):
    if nbytes == 0:
        return None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, nbytes


def flash_attn_ext(q, k_cache, v_cache, n_kv, mask=None, scale=None, max_bias=0.0, softcap=0.0,
                   out=None, workspace=None, stream=None):
    """ggml_flash_attn_ext(q, k, v, mask, scale, max_bias, softcap) over q4_0 caches."""
    if stream is None and out is not None and workspace is not None:
        rc = (_host or _load_host()).fa(q, k_cache, v_cache, n_kv, mask, scale, max_bias, softcap, out, workspace)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    n_q, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    if out is None:
        out = _make(stream, q.device, lambda: torch.empty((n_q, H, D), dtype=torch.float32, device=q.device))
    tq, tk, tv = q_desc(q), cache_view(k_cache, n_kv), cache_view(v_cache, n_kv)
    to, tm = out_desc(out), mask_desc(mask)
    if workspace is None:  # a given workspace is checked by the library
        need = int(lib().sqa_flash_attn_ext_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv),
                                                           ctypes.byref(to)))
        workspace = _make(stream, q.device, lambda: _workspace(need, q.device)[0])
    wptr = workspace.data_ptr() if workspace is not None else None
    wbytes = workspace.numel() if workspace is not None else 0
    _check(lib().sqa_flash_attn_ext(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), _ref(tm), scale,
                                    max_bias, softcap, ctypes.byref(to), wptr, wbytes, _stream(stream)))
    return out


def flash_attn_ext_static(q, k_cache, v_cache, n_kv, mask=None, scale=None, max_bias=0.0, softcap=0.0,
                          out=None, stream=None):
    """flash_attn_ext for decode/verify shapes with the library's own device scratch:
    no workspace, no allocation inside the call (out must be given for that)."""
    n_q, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    if out is None:
        out = _make(stream, q.device, lambda: torch.empty((n_q, H, D), dtype=torch.float32, device=q.device))
    tq, tk, tv = q_desc(q), cache_view(k_cache, n_kv), cache_view(v_cache, n_kv)
    to, tm = out_desc(out), mask_desc(mask)
    _check(lib().sqa_flash_attn_ext_static(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), _ref(tm), scale,
                                           max_bias, softcap, ctypes.byref(to), _stream(stream)))
    return out


def flash_attn_ext_causal(q, k_cache, v_cache, n_kv, q_pos0, gate=None, scale=None, out=None,
                          workspace=None, stream=None):
    """Mask-free causal FA (query t at position q_pos0 + t) with optional fused sigmoid gate."""
    if stream is None and out is not None and workspace is not None:
        rc = (_host or _load_host()).fa_causal(q, k_cache, v_cache, n_kv, q_pos0, gate, scale, out, workspace)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    n_q, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    if out is None:
        out = _make(stream, q.device, lambda: torch.empty((n_q, H, D), dtype=torch.float32, device=q.device))
    tq, tk, tv = q_desc(q), cache_view(k_cache, n_kv), cache_view(v_cache, n_kv)
    to = out_desc(out)
    tg = None
    if gate is not None:
        s = gate.stride()
        tg = Tensor.make(TYPE_F32, [D, H, n_q, 1], [4, s[1] * 4, s[0] * 4], gate.data_ptr())
    if workspace is None:  # a given workspace is checked by the library
        need = int(lib().sqa_flash_attn_ext_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv),
                                                           ctypes.byref(to)))
        workspace = _make(stream, q.device, lambda: _workspace(need, q.device)[0])
    wptr = workspace.data_ptr() if workspace is not None else None
    wbytes = workspace.numel() if workspace is not None else 0
    _check(lib().sqa_flash_attn_ext_causal(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), q_pos0,
                                           _ref(tg), scale, ctypes.byref(to), wptr, wbytes, _stream(stream)))
    return out


def sigmoid_mul(x, gate, out=None, stream=None):
    """out = x * sigmoid(gate) over 2-D float32 [n_tok, n] (attn.rs:282-283)."""
    if out is None:
        out = _make(stream, x.device, lambda: torch.empty_like(x))
    n1, n0 = x.shape
    d = [Tensor.make(TYPE_F32, [n0, n1], [4, t.stride(0) * 4], t.data_ptr()) for t in (out, x, gate)]
    _check(lib().sqa_sigmoid_mul(ctypes.byref(d[0]), ctypes.byref(d[1]), ctypes.byref(d[2]), _stream(stream)))
    return out


def _out_proj_descs(w, x, gate, out):
    """w: uint8 (N, K // 256 * 144) Q4_K rows; x, gate: float32 (M, K); out: float32 (M, N)."""
    M, K = x.shape
    N = w.shape[0]
    tw = Tensor.make(TYPE_Q4_K, [K, N], [Q4_K_BLOCK, w.stride(0)], w.data_ptr())
    tx = Tensor.make(TYPE_F32, [K, M], [4, x.stride(0) * 4], x.data_ptr())
    tg = None if gate is None else Tensor.make(TYPE_F32, [K, M], [4, gate.stride(0) * 4], gate.data_ptr())
    to = None if out is None else Tensor.make(TYPE_F32, [N, M], [4, out.stride(0) * 4], out.data_ptr())
    return tw, tx, tg, to


def out_proj_workspace_size(w, x):
    tw, tx, _, _ = _out_proj_descs(w, x, None, None)
    return int(lib().sqa_out_proj_workspace_size(ctypes.byref(tw), ctypes.byref(tx)))


def out_proj(w, x, gate=None, out=None, workspace=None, stream=None):
    """W_o projection (attn.rs:281-285): out (M, N) = (x * sigmoid(gate)) @ W^T with
    W the Q4_K weight rows w (N, K // 256 * 144) and x, gate (M, K) float32."""
    if stream is None and out is not None and workspace is not None:
        rc = (_host or _load_host()).out_proj(w, x, gate, out, workspace)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    M, K = x.shape
    if out is None:
        out = _make(stream, x.device, lambda: torch.empty((M, w.shape[0]), dtype=torch.float32, device=x.device))
    tw, tx, tg, to = _out_proj_descs(w, x, gate, out)
    need = int(lib().sqa_out_proj_workspace_size(ctypes.byref(tw), ctypes.byref(tx)))
    if workspace is None:
        workspace = _make(stream, x.device, lambda: _workspace(need, x.device)[0])
    _check(lib().sqa_out_proj(ctypes.byref(tw), ctypes.byref(tx), _ref(tg), ctypes.byref(to),
                              workspace.data_ptr() if workspace is not None else None,
                              workspace.numel() if workspace is not None else 0, _stream(stream)))
    return out


def fill_causal_mask(mask, step_start, stream=None):
    """Device fill of the F16 mask (n_q, n_kv): row t allows keys <= step_start + t."""
    if stream is None:
        rc = (_host or _load_host()).fill_mask(mask, step_start)
        if rc is not None:
            if rc:
                _check(rc)
            return mask
    tm = mask_desc(mask)
    _check(lib().sqa_fill_causal_mask(ctypes.byref(tm), step_start, _stream(stream)))
    return mask


# ------------------------------------------- a batch over one paged pool --

def _need(ok, msg):
    if not ok:
        raise SqaError(1, msg)


def _on(device, **tensors):
    """The tensors (None left out) are on one GPU; what follows runs with it as the current device."""
    for name, t in tensors.items():
        if t is not None:
            _need(isinstance(t, torch.Tensor) and t.device == device, f"{name} must be a tensor on {device}")
    _need(device.type == "cuda", "tensors must be on the GPU")
    return torch.cuda.device(device)


def _vec(t, dtype, name):
    _need(t.dim() == 1 and t.dtype == dtype and t.is_contiguous(), f"{name} must be a contiguous 1-D {dtype} tensor")
    code, size = (TYPE_I64, 8) if dtype == torch.int64 else (TYPE_F32 if dtype == torch.float32 else TYPE_I32, 4)
    return Tensor.make(code, [t.shape[0]], [size], t.data_ptr())


def _table_desc(table):
    _need(table.dim() == 2 and table.dtype == torch.int32 and (table.shape[1] <= 1 or table.stride(1) == 1),
          "table must be int32 (B, W) with contiguous rows")
    return Tensor.make(TYPE_I32, [table.shape[1], table.shape[0]], [4, table.stride(0) * 4], table.data_ptr())


def _pool_desc(pool, name):
    _need(pool.dim() == 4 and pool.dtype == torch.uint8 and pool.shape[3] % Q4_0_BLOCK == 0 and
          (pool.shape[0] <= 1 or pool.stride(0) > 0) and (pool.numel() == 0 or pool[0].is_contiguous()),
          f"{name} must be uint8 (n_pages, page, Hkv, D // 32 * 18) with contiguous pages")
    n_pages, page, Hkv, rb = pool.shape
    step = pool.stride(0) if n_pages > 1 else page * Hkv * rb
    return Tensor.make(TYPE_Q4_0, [rb // Q4_0_BLOCK * QK4_0, Hkv, page, n_pages], [Q4_0_BLOCK, rb, Hkv * rb, step],
                       pool.data_ptr())


def _tokens_desc(t, name):
    """(n_tok, H, D) float32 -> [D, n_tok, H], any strides with contiguous elements."""
    _need(t.dim() == 3 and t.dtype == torch.float32, f"{name} must be float32 (n_tok, H, D)")
    return q_desc(t)


def paged_plan(state, ring, table, n_past, n_new, page, slots, pos=None, state_out=None, n_past_out=None, q_start=None,
               kv_len=None, stream=None):
    """One step's plan for a batch, on the GPU: pages of ended requests (n_new < 0) return
    to the ring of free ones, new tokens get their pages, every token its pool row
    (slots, -1: none) and rotary positions. table and ring are updated in place; the
    other results are (state_out, n_past_out, q_start, kv_len, slots, pos), made here
    where they are not given, and returned as a PagedStep.

    state: int32 (4,) {first free place of the ring, free pages, ., .}; ring: int32
    (n_pages,); table: int32 (B, W); n_past, n_new: int32 (B,); slots: int64 (T,);
    pos: int32 (4 * T,), a token's place in its request four times (text; write over it for
    images). A request that finds too few pages, too little room in its table row or in
    slots is refused whole: state_out[2] counts them. Places are served in order and a
    refused one's wants stay counted, so those behind it that need a page are refused too:
    plan it with n_new = 0 until state_out[1], the free pages, covers it."""
    if state_out is None or n_past_out is None or q_start is None or kv_len is None or pos is None:
        def new(t, n):
            if t is not None:
                return t
            return _make(stream, slots.device, lambda: torch.empty(n, dtype=torch.int32, device=slots.device))

        _need(stream is None or slots.is_cuda, "tensors must be on the GPU")

        B, T = table.shape[0], slots.shape[0]
        state_out, n_past_out, q_start = new(state_out, 4), new(n_past_out, B), new(q_start, B + 1)
        kv_len, pos = new(kv_len, B), new(pos, 4 * T)
    step = PagedStep(state_out, n_past_out, q_start, kv_len, slots, pos)
    if stream is None:
        rc = (_host or _load_host()).plan(state, ring, table, n_past, n_new, page, state_out, n_past_out, q_start, kv_len,
                                          slots, pos)
        if rc is not None:
            if rc:
                _check(rc)
            return step
    i32 = torch.int32
    with _on(slots.device, state=state, ring=ring, table=table, n_past=n_past, n_new=n_new, state_out=step.state,
             n_past_out=step.n_past, q_start=step.q_start, kv_len=step.kv_len, pos=step.pos):
        d = [_vec(n_past, i32, "n_past"), _vec(n_new, i32, "n_new"), _table_desc(table), _vec(ring, i32, "ring"),
             _vec(state, i32, "state")]
        o = [_vec(step.state, i32, "state_out"), _vec(step.n_past, i32, "n_past_out"), _vec(step.q_start, i32, "q_start"),
             _vec(step.kv_len, i32, "kv_len"), _vec(slots, torch.int64, "slots"), _vec(step.pos, i32, "pos")]
        _check(lib().sqa_paged_plan(*[ctypes.byref(t) for t in d], int(page), *[ctypes.byref(t) for t in o],
                                    _stream(stream)))
    return step


class PagedStep(collections.namedtuple("PagedStep", "state n_past q_start kv_len slots pos")):
    """What paged_plan gives for one step (q_start, kv_len, slots and pos are the
    operands of paged_attn, set_rows_q4_0 and the producers)."""

    __slots__ = ()


def paged_attn_workspace_size(q, k_pool, table, max_q):
    """Workspace bytes of paged_attn for these shapes (a smaller one takes fewer splits)."""
    tq, tk, tt = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _table_desc(table)
    return int(lib().sqa_paged_attn_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tt), int(max_q)))


def supports_paged_attn(q, k_pool, table, max_q, scale=None, max_bias=0.0, softcap=0.0):
    n_tok, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    tq, tk, tt = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _table_desc(table)
    to = Tensor.make(TYPE_F32, [D, H, n_tok, 1], [4, D * 4, H * D * 4], 16)
    return bool(lib().sqa_supports_paged_attn(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tk), ctypes.byref(tt),
                                              int(max_q), scale, max_bias, softcap, ctypes.byref(to)))


def paged_attn(q, k_pool, v_pool, table, q_start, kv_len, max_q, scale=None, max_bias=0.0, softcap=0.0, prefix=None,
               gate=None, out=None, workspace=None, stream=None):
    """Causal attention of every request's new tokens over its pages of one q4_0 pool.

    q: float32 (n_tok, H, 256), request b's tokens in rows q_start[b] .. q_start[b + 1] - 1
    at positions kv_len[b] - n .. kv_len[b] - 1; table, q_start, kv_len: int32 as
    paged_plan writes them; max_q: the most new tokens of a request; prefix: int32 (B,),
    keys that every token of the request sees; softcap, max_bias: tanh cap and distance
    bias of the logits; gate: float32 like q, out *= sigmoid(gate). Rows of no request
    are left as they were (zeros in an out made here)."""
    if stream is None and out is not None and workspace is not None:
        rc = (_host or _load_host()).paged_attn(q, k_pool, v_pool, table, q_start, kv_len, prefix, max_q, scale,
                                                max_bias, softcap, gate, out, workspace)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    with _on(q.device, k_pool=k_pool, v_pool=v_pool, table=table, q_start=q_start, kv_len=kv_len, prefix=prefix,
             gate=gate, out=out, workspace=workspace):
        tq, tk, tv = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _pool_desc(v_pool, "v_pool")
        n_tok, H, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        if out is None:
            out = _make(stream, q.device, lambda: torch.zeros((n_tok, H, D), dtype=torch.float32, device=q.device))
        _need(out.dtype == torch.float32 and out.dim() == 3 and out.is_contiguous(), "out must be contiguous float32 (n_tok, H, D)")
        tt, to = _table_desc(table), out_desc(out)
        ts, tl = _vec(q_start, torch.int32, "q_start"), _vec(kv_len, torch.int32, "kv_len")
        tp = None if prefix is None else _vec(prefix, torch.int32, "prefix")
        tg = None
        if gate is not None:
            _need(gate.dim() == 3 and gate.dtype == torch.float32 and gate.shape == q.shape and
                  (gate.shape[2] <= 1 or gate.stride(2) == 1), "gate must be float32 like q")
            tg = Tensor.make(TYPE_F32, [D, H, n_tok, 1], [4, gate.stride(1) * 4, gate.stride(0) * 4], gate.data_ptr())
        _need(q.shape[2] <= 1 or q.stride(2) == 1, "q rows must have unit element stride")
        if workspace is None:
            need = int(lib().sqa_paged_attn_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tt), int(max_q)))
            workspace = _make(stream, q.device, lambda: _workspace(need, q.device)[0])
        _need(workspace is None or workspace.is_contiguous(), "workspace must be contiguous")
        _check(lib().sqa_paged_attn(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), ctypes.byref(tt), ctypes.byref(ts),
                                    ctypes.byref(tl), _ref(tp), int(max_q), scale, max_bias, softcap, _ref(tg),
                                    ctypes.byref(to), workspace.data_ptr() if workspace is not None else None,
                                    workspace.numel() * workspace.element_size() if workspace is not None else 0,
                                    _stream(stream)))
    return out


class PagedShare(collections.namedtuple("PagedShare", "members m_start m_pos token_group")):
    """What paged_share gives for one step: the operands of paged_attn_shared."""

    __slots__ = ()


def paged_share(q_start, kv_len, group, shared_len, members, m_start=None, m_pos=None, token_group=None, pos=None, stream=None):
    """Which of a step's tokens go with which shared prefix, on the GPU, once per step: request b continues the first
    shared_len[group[b]] keys of its group (group: int32 (B,), outside [0, G) for none; shared_len: int32 (G,)).

    members: int32 (T,), made into the members' token rows by group, request and token; m_start: int32 (G + 1,) where a
    group's begin; m_pos: int32 (T,) their positions behind the shared keys; token_group: int32 (T,) the group of every
    token row, -1 for none. Those not given are made here; all are returned as a PagedShare. pos: int32 (4 * T,) as
    paged_plan wrote it: the members' rotary positions are moved behind the shared keys (None: left alone). Requests with
    kv_len <= 0 (refused ones) and groups of no keys have no members."""
    if m_start is None or m_pos is None or token_group is None:
        _need(stream is None or members.is_cuda, "tensors must be on the GPU")

        def new(t, n):
            if t is not None:
                return t
            return _make(stream, members.device, lambda: torch.empty(n, dtype=torch.int32, device=members.device))

        T = members.shape[0]
        m_start, m_pos, token_group = new(m_start, shared_len.shape[0] + 1), new(m_pos, T), new(token_group, T)
    share = tuple.__new__(PagedShare, (members, m_start, m_pos, token_group))
    if stream is None:
        rc = (_host or _load_host()).share(q_start, kv_len, group, shared_len, members, m_start, m_pos, token_group, pos)
        if rc is not None:
            if rc:
                _check(rc)
            return share
    names = ("q_start", "kv_len", "group", "shared_len", "members", "m_start", "m_pos", "token_group", "pos")
    ts = dict(zip(names, (q_start, kv_len, group, shared_len, *share, pos)))
    with _on(members.device, **ts):
        d = [None if t is None else _vec(t, torch.int32, name) for name, t in ts.items()]
        _check(lib().sqa_paged_share(*[_ref(t) for t in d], _stream(stream)))
    return share


def paged_attn_shared_workspace_size(q, k_pool, table, shared_table, max_q):
    """Workspace bytes of paged_attn_shared for these shapes (a smaller one takes fewer splits)."""
    tq, tk, tt, ts = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _table_desc(table), _table_desc(shared_table)
    return int(lib().sqa_paged_attn_shared_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tt),
                                                          ctypes.byref(ts), int(max_q)))


def supports_paged_attn_shared(q, k_pool, table, shared_table, max_q, scale=None, max_bias=0.0, softcap=0.0):
    n_tok, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    tq, tk, tt, ts = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _table_desc(table), _table_desc(shared_table)
    to = Tensor.make(TYPE_F32, [D, H, n_tok, 1], [4, D * 4, H * D * 4], 16)
    return bool(lib().sqa_supports_paged_attn_shared(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tk), ctypes.byref(tt),
                                                     ctypes.byref(ts), int(max_q), scale, max_bias, softcap, ctypes.byref(to)))


def paged_attn_shared(q, k_pool, v_pool, table, q_start, kv_len, shared_table, shared_len, share, max_q, scale=None,
                      max_bias=0.0, softcap=0.0, prefix=None, gate=None, out=None, workspace=None, stream=None):
    """paged_attn of requests that continue shared prefixes: the tokens of group g see the first shared_len[g] keys of
    the pages in shared_table[g], read once for all of them, and their own keys as in paged_attn, under one softmax.

    shared_table: int32 (G, W'), may be table itself with a place of the batch as the group; shared_len: int32 (G,);
    share: paged_share's PagedShare of this step (T == n_tok); the rest as in paged_attn."""
    if stream is None and out is not None and workspace is not None and isinstance(share, tuple) and len(share) == 4:
        rc = (_host or _load_host()).attn_shared(q, k_pool, v_pool, table, q_start, kv_len, prefix, shared_table, shared_len,
                                                 *share, max_q, scale, max_bias, softcap, gate, out, workspace)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    members, m_start, m_pos, token_group = share
    with _on(q.device, k_pool=k_pool, v_pool=v_pool, table=table, q_start=q_start, kv_len=kv_len, prefix=prefix,
             shared_table=shared_table, shared_len=shared_len, members=members, m_start=m_start, m_pos=m_pos,
             token_group=token_group, gate=gate, out=out, workspace=workspace):
        tq, tk, tv = _tokens_desc(q, "q"), _pool_desc(k_pool, "k_pool"), _pool_desc(v_pool, "v_pool")
        n_tok, H, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        if out is None:
            out = _make(stream, q.device, lambda: torch.zeros((n_tok, H, D), dtype=torch.float32, device=q.device))
        _need(out.dtype == torch.float32 and out.dim() == 3 and out.is_contiguous(), "out must be contiguous float32 (n_tok, H, D)")
        tt, tst, to = _table_desc(table), _table_desc(shared_table), out_desc(out)
        i32 = torch.int32
        tp = None if prefix is None else _vec(prefix, i32, "prefix")
        d = [_vec(t, i32, name) for t, name in ((q_start, "q_start"), (kv_len, "kv_len"))]
        e = [_vec(t, i32, name) for t, name in ((shared_len, "shared_len"), (members, "members"), (m_start, "m_start"),
                                                (m_pos, "m_pos"), (token_group, "token_group"))]
        tg = None
        if gate is not None:
            _need(gate.dim() == 3 and gate.dtype == torch.float32 and gate.shape == q.shape and
                  (gate.shape[2] <= 1 or gate.stride(2) == 1), "gate must be float32 like q")
            tg = Tensor.make(TYPE_F32, [D, H, n_tok, 1], [4, gate.stride(1) * 4, gate.stride(0) * 4], gate.data_ptr())
        _need(q.shape[2] <= 1 or q.stride(2) == 1, "q rows must have unit element stride")
        if workspace is None:
            need = int(lib().sqa_paged_attn_shared_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tt),
                                                                  ctypes.byref(tst), int(max_q)))
            workspace = _make(stream, q.device, lambda: _workspace(need, q.device)[0])
        _need(workspace is None or workspace.is_contiguous(), "workspace must be contiguous")
        _check(lib().sqa_paged_attn_shared(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), ctypes.byref(tt),
                                           *[ctypes.byref(t) for t in d], _ref(tp), ctypes.byref(tst),
                                           *[ctypes.byref(t) for t in e], int(max_q), scale, max_bias, softcap, _ref(tg),
                                           ctypes.byref(to), workspace.data_ptr() if workspace is not None else None,
                                           workspace.numel() * workspace.element_size() if workspace is not None else 0,
                                           _stream(stream)))
    return out


def _lora_descs(base, x, a, b, gate, out):
    for t, name in ((base, "base"), (x, "x"), (gate, "gate"), (out, "out")):
        _need(t is None or (t.dim() == 2 and t.dtype == torch.float32 and (t.shape[1] <= 1 or t.stride(1) == 1)),
              f"{name} must be float32 rows with contiguous elements")
    for t, name in ((a, "a"), (b, "b")):
        _need(t.dim() == 3 and t.dtype == torch.float16 and t.is_contiguous(), f"{name} must be contiguous float16 of 3 dims")

    def rows(t):
        return None if t is None else Tensor.make(TYPE_F32, [t.shape[1], t.shape[0]], [4, t.stride(0) * 4], t.data_ptr())

    ta, tb = (Tensor.make(TYPE_F16, [t.shape[2], t.shape[1], t.shape[0]],
                          [2, 2 * t.shape[2], 2 * t.shape[2] * t.shape[1]], t.data_ptr()) for t in (a, b))
    return rows(base), rows(x), rows(gate), ta, tb, rows(out)


def supports_lora_add(base, x, a, b, gate=None, out=None):
    td, tx, tg, ta, tb, to = _lora_descs(base, x, a, b, gate, base if out is None else out)
    return bool(lib().sqa_supports_lora_add(_ref(td), _ref(tx), _ref(tg), _ref(ta), _ref(tb), _ref(to)))


def lora_add(base, x, a, b, ids, scale=None, gate=None, out=None, stream=None):
    """out = base + scale[i] * (x * sigmoid(gate)) @ a[i]^T @ b[i]^T with i = ids[m] for token m:
    the low-rank adapters of a batch's requests beside a shared projection (out_proj).

    base: float32 (M, N), may be out; x, gate: float32 (M, K); a: float16 (n, r, K);
    b: float16 (n, N, r); ids: int32 (M,), an id outside [0, n) is a token without
    adapter; scale: float32 (n,) or None. out may be base, and overlaps nothing else.
    Up to 512 tokens (and K of 16384) all is float32; more tokens take x * sigmoid(gate)
    and scale * A x at 22 bits, an absolute 2^-36 below 2^-13."""
    if stream is None and out is not None:
        rc = (_host or _load_host()).lora(base, x, a, b, ids, scale, gate, out)
        if rc is not None:
            if rc:
                _check(rc)
            return out
    with _on(x.device, base=base, a=a, b=b, ids=ids, scale=scale, gate=gate, out=out):
        if out is None:
            out = _make(stream, x.device, lambda: torch.empty_like(base, memory_format=torch.contiguous_format))
        td, tx, tg, ta, tb, to = _lora_descs(base, x, a, b, gate, out)
        ti = _vec(ids, torch.int32, "ids")
        ts = None if scale is None else _vec(scale, torch.float32, "scale")
        _check(lib().sqa_lora_add(_ref(td), _ref(tx), _ref(tg), _ref(ta), _ref(tb), _ref(ti), _ref(ts), _ref(to),
                                  _stream(stream)))
    return out


def profile_begin(max_records=4096):
    """Bracket every kernel launch with HIP events until profile_end()."""
    _check(lib().sqa_profile_begin(max_records))


def profile_end():
    lib().sqa_profile_end()


def profile_get(kernel):
    """(total_ms, launches) recorded for one kernel since profile_begin()."""
    ms, n = ctypes.c_double(), ctypes.c_int64()
    _check(lib().sqa_profile_get(kernel.encode(), ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value


# ---------------------------------------------------------------- KvCache ---

class KvCache:
    """Single-sequence append-only q4_0 KV cache (mirror of kv.rs:67-448).

    Owns one K and one V uint8 buffer per full-attention layer, each of shape
    (cap_alloc, Hkv, D//32*18); bookkeeping runs in the C++ library."""

    def __init__(self, n_layers, head_dim, n_head_kv, kv_cap, device="cuda"):
        L = lib()
        self.head_dim, self.n_head_kv, self.kv_cap = head_dim, n_head_kv, kv_cap
        nbytes = int(L.sqa_kv_cache_layer_bytes(head_dim, n_head_kv, kv_cap))
        if nbytes == 0:
            raise SqaError(1, "invalid KV cache geometry")
        self.kv_cap_alloc = (kv_cap + KV_PAD - 1) // KV_PAD * KV_PAD
        shape = (self.kv_cap_alloc, n_head_kv, row_bytes(head_dim))
        self.k = [torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(n_layers)]
        kp = (ctypes.c_void_p * n_layers)(*[t.data_ptr() for t in self.k])
        vp = (ctypes.c_void_p * n_layers)(*[t.data_ptr() for t in self.v])
        self._h = L.sqa_kv_cache_create(n_layers, head_dim, n_head_kv, kv_cap, kp, vp)
        if not self._h:
            raise SqaError(1, last_error())

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib().sqa_kv_cache_destroy(h)
            self._h = None

    def zero_caches(self):
        """Zero every layer once at load (kv.rs:150-170): padded rows then contribute 0."""
        for t in self.k + self.v:
            t.zero_()

    @property
    def n_used(self):
        return int(lib().sqa_kv_cache_n_used(self._h))

    @property
    def step_start(self):
        return int(lib().sqa_kv_cache_step_start(self._h))

    def n_kv_padded(self):
        return int(lib().sqa_kv_cache_n_kv_padded(self._h))

    def n_kv_padded_after(self, n_tokens):
        return int(lib().sqa_kv_cache_n_kv_padded_after(self._h, n_tokens))

    def begin_step(self, n_tokens):
        _check(lib().sqa_kv_cache_begin_step(self._h, n_tokens))

    def rewind_to(self, pos):
        _check(lib().sqa_kv_cache_rewind_to(self._h, pos))

    def reset(self):
        lib().sqa_kv_cache_reset(self._h)

    def view(self, slot, which="k"):
        t = Tensor()
        fn = lib().sqa_kv_cache_k_view if which == "k" else lib().sqa_kv_cache_v_view
        _check(fn(self._h, slot, ctypes.byref(t)))
        return t

    def append(self, slot, k_cur, v_cur, idx, stream=None):
        """Quantize this step's K/V rows, float32 (n_tokens, Hkv*D), into layer `slot`."""
        if stream is None:
            rc = (_host or _load_host()).append(self._h, slot, k_cur, v_cur, idx)
            if rc is not None:
                return _check(rc)
        n_tok, ne0 = k_cur.shape
        tk = Tensor.make(TYPE_F32, [ne0, n_tok], [4, k_cur.stride(0) * 4], k_cur.data_ptr())
        tv = Tensor.make(TYPE_F32, [ne0, n_tok], [4, v_cur.stride(0) * 4], v_cur.data_ptr())
        ti = Tensor.make(TYPE_I64, [n_tok], [8], idx.data_ptr())
        _check(lib().sqa_kv_cache_append(self._h, slot, ctypes.byref(tk), ctypes.byref(tv), ctypes.byref(ti),
                                         _stream(stream)))

    def read(self, slot, idx, which="k", out=None, dtype=torch.float32, stream=None):
        """Layer `slot`'s cached K or V of rows idx (int64) as values (n, Hkv*D), float32 or float16."""
        return get_rows_q4_0((self.k if which == "k" else self.v)[slot], idx, out=out, dtype=dtype, stream=stream)

    def move(self, slot, to, from_, delta, rope, stream=None):
        """Rows from_ of layer `slot` to rows to, K rotated on by delta (int32 (4*n,)) and V as it is; a row of from_
        must be no other entry's to (a long move down goes in pieces of at most its own distance, lowest first)."""
        move_rows_q4_0(self.k[slot], self.k[slot], to, from_, delta, rope, stream=stream)
        move_rows_q4_0(self.v[slot], self.v[slot], to, from_, stream=stream)

    def workspace_size(self, slot, q):
        """Workspace bytes of attend() for q over the current [0, n_kv_padded) views."""
        n_q, H, D = q.shape
        tq, tk, tv = q_desc(q), self.view(slot, "k"), self.view(slot, "v")
        to = Tensor.make(TYPE_F32, [D, H, n_q, 1], [4, D * 4, H * D * 4], 16)
        return int(lib().sqa_flash_attn_ext_workspace_size(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv),
                                                           ctypes.byref(to)))

    def attend(self, slot, q, mask=None, scale=None, out=None, workspace=None, stream=None):
        """flash_attn_ext over this layer's [0, n_kv_padded) views, taken from the
        library's k_view/v_view (the permuted views of kv.rs:401-447 that
        attn.rs:228-251 hands to ggml_flash_attn_ext)."""
        n_q, H, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        if out is None:
            out = _make(stream, q.device, lambda: torch.empty((n_q, H, D), dtype=torch.float32, device=q.device))
        tq, tk, tv = q_desc(q), self.view(slot, "k"), self.view(slot, "v")
        to, tm = out_desc(out), mask_desc(mask)
        if workspace is None:
            need = self.workspace_size(slot, q)
            workspace = _make(stream, q.device, lambda: _workspace(need, q.device)[0])
        wptr = workspace.data_ptr() if workspace is not None else None
        wbytes = workspace.numel() if workspace is not None else 0
        _check(lib().sqa_flash_attn_ext(ctypes.byref(tq), ctypes.byref(tk), ctypes.byref(tv), _ref(tm), scale,
                                        0.0, 0.0, ctypes.byref(to), wptr, wbytes, _stream(stream)))
        return out


# ----------------------------------------------------------- PagedKvCache ---

class PagedKvCache:
    """q4_0 KV cache of many requests in pages of one pool, KvCache's counterpart for a batch.

    Owns one K and one V pool per layer, uint8 (n_pages, page, Hkv, D//32*18), the page
    table (max_requests, max_pages) and the lengths; a request is a place of the batch.
    All bookkeeping runs on the GPU: plan() then append() and attend() of every layer
    make up a step that can be captured into a graph and replayed with other n_new."""

    def __init__(self, n_layers, head_dim, n_head_kv, n_pages, page, max_requests, max_pages, device="cuda"):
        _need(n_layers >= 1 and n_pages >= 1 and max_requests >= 1 and max_pages >= 1 and n_head_kv >= 1 and
              head_dim % QK4_0 == 0 and page >= 16 and page & (page - 1) == 0, "invalid paged KV cache geometry")
        self.head_dim, self.n_head_kv, self.page = head_dim, n_head_kv, page
        shape = (n_pages, page, n_head_kv, row_bytes(head_dim))
        self.k = [torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(n_layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.full((max_requests, max_pages), -1, **i32)
        self.ring = torch.arange(n_pages, **i32)
        # {first, free, refused, tokens} and the lengths, and the same after the step being planned
        self._now, self._next = torch.zeros(4 + max_requests, **i32), torch.zeros(4 + max_requests, **i32)
        self._now[1] = n_pages

    @property
    def state(self):
        """int32 (4,) on the GPU: first free place of the ring, free pages, requests the last plan refused, its tokens."""
        return self._now[:4]

    @property
    def n_past(self):
        """int32 (max_requests,) on the GPU: tokens of every request."""
        return self._now[4:]

    def new_step(self, n_rows):
        """Buffers of a step of up to n_rows tokens (kept by the caller, reused step after step). state and
        n_past are the cache's own: every step's show what plan() made last."""
        i32, B, dev = torch.int32, self.table.shape[0], self.table.device
        return PagedStep(self._next[:4], self._next[4:], torch.zeros(B + 1, dtype=i32, device=dev),
                         torch.zeros(B, dtype=i32, device=dev), torch.zeros(n_rows, dtype=torch.int64, device=dev),
                         torch.zeros(4 * n_rows, dtype=i32, device=dev))

    def plan(self, n_new, step, stream=None):
        """Gives the step's new tokens (n_new: int32 (max_requests,), < 0 ends a request) their pages."""
        with _stream_of(stream, self.table.device):
            paged_plan(self.state, self.ring, self.table, self.n_past, n_new, self.page, step.slots, step.pos,
                       step.state, step.n_past, step.q_start, step.kv_len)
            self._now.copy_(self._next)
        return step

    def rows(self, layer, which="k"):
        """Layer's K or V pool as cache rows (n_pages * page, Hkv, bytes): where slots point."""
        return (self.k if which == "k" else self.v)[layer].view(-1, self.n_head_kv, row_bytes(self.head_dim))

    def append(self, layer, k_cur, v_cur, step, stream=None):
        """Quantize the step's K and V rows, float32 (n_rows, Hkv*D), into the layer's pages."""
        with _stream_of(stream, self.table.device):
            set_rows_q4_0(self.rows(layer, "k"), k_cur, step.slots)
            set_rows_q4_0(self.rows(layer, "v"), v_cur, step.slots)

    def read(self, layer, slots, which="k", out=None, dtype=torch.float32, stream=None):
        """The layer's cached K or V at pool rows slots (int64, -1 reads as zeros) as values (n, Hkv*D)."""
        return get_rows_q4_0(self.rows(layer, which), slots, out=out, dtype=dtype, stream=stream)

    def move(self, layer, to, from_, delta, rope, stream=None):
        """Pool rows from_ of the layer to rows to, K rotated on by delta (int32 (4*n,)) and V as it is; a row of from_
        must be no other entry's to."""
        move_rows_q4_0(self.rows(layer, "k"), self.rows(layer, "k"), to, from_, delta, rope, stream=stream)
        move_rows_q4_0(self.rows(layer, "v"), self.rows(layer, "v"), to, from_, stream=stream)

    def new_share(self, n_rows):
        """Buffers of share() for steps of up to n_rows tokens (kept by the caller, reused step after step)."""
        dev = self.table.device
        return PagedShare(*(torch.zeros(n, dtype=torch.int32, device=dev)
                            for n in (n_rows, self.table.shape[0] + 1, n_rows, n_rows)))

    def share(self, parent, step, share, stream=None):
        """After plan(): request b of this step continues all cached keys of place parent[b] (int32 (max_requests,),
        -1 for none), which holds a prompt for several requests; its own pages and lengths count its own tokens only.
        The members' positions in step.pos move behind the parent's keys. A parent has no parent that counts, and must
        not end or grow while others continue it."""
        return paged_share(step.q_start, step.kv_len, parent, step.n_past, *share, pos=step.pos, stream=stream)

    def workspace_size(self, q, max_q, share=None):
        if share is not None:
            return paged_attn_shared_workspace_size(q, self.k[0], self.table, self.table, max_q)
        return paged_attn_workspace_size(q, self.k[0], self.table, max_q)

    def attend(self, layer, q, step, max_q, share=None, **options):
        """paged_attn of the step's tokens over the layer's pages, with share() paged_attn_shared (options: scale,
        max_bias, softcap, prefix, gate, out, workspace, stream)."""
        if share is not None:
            return paged_attn_shared(q, self.k[layer], self.v[layer], self.table, step.q_start, step.kv_len, self.table,
                                     step.n_past, share, max_q, **options)
        return paged_attn(q, self.k[layer], self.v[layer], self.table, step.q_start, step.kv_len, max_q, **options)
