"""eyebrowse_b200 -- B200 (sm_100a) attention path for eyebrowse, behind a C ABI.

The product is libeyebrowse_attn.so (include/eyebrowse_attn.h). This module
binds it with ctypes for Python callers (tests, bench.py, the head-sharded
multi-GPU driver in eyebrowse_b200.sharded). Tensors are torch CUDA tensors;
only their device pointers cross the boundary. There is no CPU fallback:
importing works without a GPU, but every call needs the CUDA library and an
sm_100 device, and a non-OK status raises EbError.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libeyebrowse_attn.so")

EB_F32, EB_F16, EB_BF16, EB_E4M3, EB_E5M2 = 0, 1, 2, 3, 4
STATUS = {0: "EB_OK", 1: "EB_ERR_INVALID_ARGUMENT", 2: "EB_ERR_UNSUPPORTED", 3: "EB_ERR_CUDA",
          4: "EB_ERR_WORKSPACE", 5: "EB_ERR_NO_DEVICE", 6: "EB_ERR_DEVICE_TIMEOUT"}

# Every symbol include/eyebrowse_attn.h declares.
EXPORTS = (
    "eb_status_string", "eb_version", "eb_attn_prefill", "eb_attn_prefill_workspace_bytes",
    "eb_attn_decode", "eb_attn_decode_workspace_bytes", "eb_rope", "eb_kv_write", "eb_rmsnorm",
    "eb_rope_tables", "eb_attention_prefill", "eb_attention_prefill_workspace_bytes",
    "eb_attention_prefill_kv", "eb_attention_prefill_attend",
    "eb_attention_prefill_gather", "eb_attention_prefill_attend_gather",
    "eb_attention_decode", "eb_attention_decode_batched", "eb_attention_decode_workspace_bytes",
    "eb_workspace_init", "eb_head_concat", "eb_get_device_error",
    "eb_attention_decode_noalloc", "eb_head_broadcast", "eb_linear_f16w",
    "eb_linear_f16w_workspace_bytes", "eb_selftest_wait_timeout",
    "eb_attention_decode_batched_gather", "eb_w4_weight_bytes", "eb_w4_pack", "eb_w4_quantize",
    "eb_linear_w4_workspace_bytes", "eb_linear_w4", "eb_kv8_write",
    "eb_attention_decode_kv8_workspace_bytes", "eb_attention_decode_kv8",
    "eb_sample_workspace_bytes", "eb_sample",
)


class HeadGather(ctypes.Structure):
    """eb_head_gather: where a head-sharded prefill stores its heads (dst is a
    host array of device addresses, one per rank)."""
    _fields_ = [("n_dst", ctypes.c_int32), ("head_offset", ctypes.c_int32),
                ("n_heads_total", ctypes.c_int64), ("dst", ctypes.POINTER(ctypes.c_uint64))]


class EbError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {STATUS.get(status, status)} ({_lib.eb_status_string(status).decode()})")


class AttnDesc(ctypes.Structure):
    """eb_attn_desc (include/eyebrowse_attn.h)."""
    _fields_ = [("n_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("max_seq", ctypes.c_int32),
                ("dtype_qkv", ctypes.c_int32), ("dtype_cache", ctypes.c_int32),
                ("dtype_out", ctypes.c_int32), ("q_stride", ctypes.c_int32),
                ("kv_stride", ctypes.c_int32), ("o_stride", ctypes.c_int32),
                ("eps", ctypes.c_float), ("scale", ctypes.c_float),
                ("window", ctypes.c_int32)]


class AttnLayer(ctypes.Structure):
    """eb_attn_layer (include/eyebrowse_attn.h)."""
    _fields_ = [("q_norm_w", ctypes.c_void_p), ("k_norm_w", ctypes.c_void_p),
                ("v_norm_w", ctypes.c_void_p), ("rope_cos", ctypes.c_void_p),
                ("rope_sin", ctypes.c_void_p)]


class W4(ctypes.Structure):
    """eb_w4: 4-bit weights with group scales."""
    _fields_ = [("in_f", ctypes.c_int64), ("out_f", ctypes.c_int64), ("group", ctypes.c_int32),
                ("dtype_scale", ctypes.c_int32), ("q", ctypes.c_void_p),
                ("scale", ctypes.c_void_p), ("zero", ctypes.c_void_p)]


class Kv8(ctypes.Structure):
    """eb_kv8: an 8-bit KV cache with block scales."""
    codes = scales = 1 << 62  # elements from the first on that k and v, and their scales, hold
    axes = scale_axes = None  # the tensors' own: [(batch,) rows, kv_heads, head_dim], [(batch,) blocks, kv_heads]
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("batch_stride", ctypes.c_int64),
                ("scale_batch_stride", ctypes.c_int64), ("block", ctypes.c_int32)]

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.plans = {}  # what calls expect of their tensors, by descriptor and batch


class SampleParams(ctypes.Structure):
    """eb_sample_params: per-row temperature, top-k, top-p and min-p arrays."""
    rows = 1 << 24  # that the arrays hold
    _fields_ = [("temperature", ctypes.c_void_p), ("top_k", ctypes.c_void_p),
                ("top_p", ctypes.c_void_p), ("min_p", ctypes.c_void_p)]


_lib = None
_vp, _i64, _f, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


def lib() -> ctypes.CDLL:
    """Load libeyebrowse_attn.so (built by eyebrowse_b200.build). Raises if absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: run `python -m eyebrowse_b200.build` "
                           "(there is no fallback path)")
    L = ctypes.CDLL(LIB_PATH)
    L.eb_status_string.restype = ctypes.c_char_p
    L.eb_status_string.argtypes = [ctypes.c_int]
    L.eb_version.restype = ctypes.c_char_p
    L.eb_attn_prefill.argtypes = [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _f, _vp, _sz, _vp]
    L.eb_attn_prefill_workspace_bytes.restype = _sz
    L.eb_attn_prefill_workspace_bytes.argtypes = [_i64, _i64, _i64, _i64]
    L.eb_attn_decode.argtypes = [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _f, _vp, _sz, _vp]
    L.eb_attn_decode_workspace_bytes.restype = _sz
    L.eb_attn_decode_workspace_bytes.argtypes = [_i64, _i64, _i64, _i64]
    L.eb_rope.argtypes = [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp]
    L.eb_kv_write.argtypes = [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp]
    L.eb_rmsnorm.argtypes = [_vp, _vp, _vp, _i64, _i64, _f, _vp]
    L.eb_linear_f16w.argtypes = [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _sz, _vp]
    L.eb_linear_f16w_workspace_bytes.restype = _sz
    L.eb_linear_f16w_workspace_bytes.argtypes = [_i64, _i64, _i64]
    L.eb_rope_tables.argtypes = [_vp, _vp, _i64, _i64, _i64, _f]
    dp, lp = ctypes.POINTER(AttnDesc), ctypes.POINTER(AttnLayer)
    L.eb_attention_prefill.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp]
    L.eb_attention_prefill_kv.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, _sz, _vp]
    L.eb_attention_prefill_attend.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, _sz, _vp]
    L.eb_head_broadcast.argtypes = [_vp, _vp, _i64, _i64, ctypes.c_int32, ctypes.c_int32, _i64,
                                    ctypes.c_int32, _vp]
    gp = ctypes.POINTER(HeadGather)
    L.eb_attention_prefill_gather.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, gp, _vp, _sz,
                                              _vp]
    L.eb_attention_prefill_attend_gather.argtypes = [dp, lp, _i64, _vp, _vp, _vp, gp, _vp, _sz,
                                                     _vp]
    L.eb_attention_prefill_workspace_bytes.restype = _sz
    L.eb_attention_prefill_workspace_bytes.argtypes = [dp, _i64]
    L.eb_attention_decode.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp]
    L.eb_attention_decode_batched.argtypes = [dp, lp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp,
                                              _i64, _vp, _vp, _sz, _vp]
    L.eb_attention_decode_batched_gather.argtypes = [dp, lp, _i64, _vp, _i64, _vp, _vp, _vp, _vp,
                                                     _vp, _i64, gp, _vp, _vp, _sz, _vp]
    L.eb_attention_decode_workspace_bytes.restype = _sz
    L.eb_attention_decode_workspace_bytes.argtypes = [dp, _i64, _i64]
    L.eb_attention_decode_noalloc.argtypes = [dp, lp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp]
    wp, kp, i32 = ctypes.POINTER(W4), ctypes.POINTER(Kv8), ctypes.c_int32
    L.eb_w4_weight_bytes.restype = _sz
    L.eb_w4_weight_bytes.argtypes = [_i64, _i64]
    L.eb_w4_pack.argtypes = [_vp, _i64, _i64, _vp]
    L.eb_w4_quantize.argtypes = [_vp, _i64, _i64, i32, i32, _vp, _vp, _vp]
    L.eb_linear_w4_workspace_bytes.restype = _sz
    L.eb_linear_w4_workspace_bytes.argtypes = [_i64, _i64, _i64]
    L.eb_linear_w4.argtypes = [wp, _vp, i32, _i64, _vp, i32, _i64, _i64, _vp, _sz, _vp]
    L.eb_kv8_write.argtypes = [dp, lp, kp, _i64, _i64, _vp, _vp, _vp]
    L.eb_attention_decode_kv8_workspace_bytes.restype = _sz
    L.eb_attention_decode_kv8_workspace_bytes.argtypes = [dp, _i64, _i64]
    L.eb_attention_decode_kv8.argtypes = [dp, lp, kp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _sz,
                                          _vp]
    L.eb_sample_workspace_bytes.restype = _sz
    L.eb_sample_workspace_bytes.argtypes = [_i64, _i64]
    L.eb_sample.argtypes = [_vp, i32, _i64, _i64, _i64, ctypes.POINTER(SampleParams), _vp, _vp, _vp,
                            _sz, _vp]
    L.eb_workspace_init.argtypes = [_vp, _sz, _vp]
    L.eb_head_concat.argtypes = [_vp, _vp, _i64, _i64, _i64, _i64, ctypes.c_int32, _vp]
    L.eb_get_device_error.argtypes = [ctypes.POINTER(ctypes.c_uint32)]
    L.eb_selftest_wait_timeout.argtypes = [ctypes.c_uint32, _vp]
    _lib = L
    return L


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = _device = None  # torch's, once a call has needed them


def _stream(stream) -> int | None:
    global _raw_stream, _device
    if stream is None:
        if _raw_stream is None:
            import torch
            torch.cuda.init()
            _device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        # torch.cuda.current_stream() without the Stream object around it
        return _raw_stream(_device())
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _check(status: int, what: str) -> None:
    if status != 0:
        raise EbError(status, what)


_dtype_codes = {}


def _codes() -> dict:
    if not _dtype_codes:
        import torch
        _dtype_codes.update({torch.float32: EB_F32, torch.float16: EB_F16, torch.bfloat16: EB_BF16})
    return _dtype_codes


def torch_dtype_code(dt) -> int:
    return _codes()[dt]


# ---------------------------------------------------------------- kernel level
def attn_prefill(q, k, v, o, h, hkv, s, hd, scale, workspace=None, stream=None):
    """eb_attn_prefill: drop-in for eyebrowse-kernels attn_prefill (f32)."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attn_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(o), h, hkv, s, hd, scale,
                                 _ptr(workspace), ws_bytes, _stream(stream)), "eb_attn_prefill")


def attn_prefill_workspace_bytes(h, hkv, s, hd) -> int:
    return lib().eb_attn_prefill_workspace_bytes(h, hkv, s, hd)


def attn_decode(q, kcache, vcache, o, h, hkv, pos, hd, max_seq, scale, workspace=None,
                stream=None):
    """eb_attn_decode: drop-in for eyebrowse-kernels attn_decode (f32)."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attn_decode(_ptr(q), _ptr(kcache), _ptr(vcache), _ptr(o), h, hkv, pos, hd,
                                max_seq, scale, _ptr(workspace), ws_bytes, _stream(stream)),
           "eb_attn_decode")


def attn_decode_workspace_bytes(h, hkv, pos, hd) -> int:
    return lib().eb_attn_decode_workspace_bytes(h, hkv, pos, hd)


def rope(x, cos, sin, out, seq, n_heads, head_dim, base_pos, stream=None):
    _check(lib().eb_rope(_ptr(x), _ptr(cos), _ptr(sin), _ptr(out), seq, n_heads, head_dim,
                         base_pos, _stream(stream)), "eb_rope")


def kv_write(cache, src, hkv, count, hd, max_seq, dst_start, stream=None):
    _check(lib().eb_kv_write(_ptr(cache), _ptr(src), hkv, count, hd, max_seq, dst_start,
                             _stream(stream)), "eb_kv_write")


def rmsnorm(x, weight, out, rows, dim, eps, stream=None):
    _check(lib().eb_rmsnorm(_ptr(x), _ptr(weight), _ptr(out), rows, dim, eps, _stream(stream)),
           "eb_rmsnorm")


def linear_f16w_workspace_bytes(m, in_f, out_f) -> int:
    return lib().eb_linear_f16w_workspace_bytes(m, in_f, out_f)


def linear_f16w(x, w, y, m, in_f, out_f, workspace=None, stream=None):
    """eb_linear_f16w: y [m, out_f] = x [m, in_f] (f32) @ w[out_f, in_f]^T (f16),
    f32 accumulation (linear_f16w, crates/eyebrowse-kernels/src/matmul.rs:128-149).
    m > 8 needs linear_f16w_workspace_bytes of workspace."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_linear_f16w(_ptr(x), _ptr(w), _ptr(y), m, in_f, out_f, _ptr(workspace),
                                ws_bytes, _stream(stream)), "eb_linear_f16w")


# ---------------------------------------------------------------- 4-bit weights
def w4_weight_bytes(in_f, out_f) -> int:
    return lib().eb_w4_weight_bytes(in_f, out_f)


def w4_pack(codes):
    """eb_w4_pack (host): codes [out_f, in_f] (numpy, 0..15) -> packed uint8 rows
    [out_f, ceil(in_f / 128) * 64]."""
    import numpy as np
    given = np.asarray(codes)
    codes = np.ascontiguousarray(given, dtype=np.uint8)
    if given.dtype != np.uint8 and not np.array_equal(codes, given):
        _refuse("w4_pack: codes that are not whole numbers of 0..15")
    out_f, in_f = codes.shape
    q = np.empty((out_f, (in_f + 127) // 128 * 64), np.uint8)
    _check(lib().eb_w4_pack(codes.ctypes.data, in_f, out_f, q.ctypes.data), "eb_w4_pack")
    return q


def w4_quantize(w, group=128, zero_point=False, dtype_scale=EB_F16):
    """eb_w4_quantize (host): weights [out_f, in_f] -> (packed rows, scales [groups, out_f],
    zero points [groups, out_f] or None) as numpy arrays. bf16 scales come back as their uint16
    bits (numpy has no bf16), f16 scales as float16."""
    import numpy as np
    w = np.ascontiguousarray(w, dtype=np.float32)
    out_f, in_f = w.shape
    groups = (in_f + group - 1) // group if group > 0 else 0
    q = np.empty((out_f, (in_f + 127) // 128 * 64), np.uint8)
    scale = np.empty((groups, out_f), np.uint16)
    zero = np.empty((groups, out_f), np.uint8) if zero_point else None
    _check(lib().eb_w4_quantize(w.ctypes.data, in_f, out_f, group, dtype_scale, q.ctypes.data,
                                scale.ctypes.data, zero.ctypes.data if zero_point else None),
           "eb_w4_quantize")
    return q, scale.view(np.float16) if dtype_scale == EB_F16 else scale, zero


def make_w4(q, scale, zero, in_f, out_f, group, dtype_scale=None):
    """eb_w4 over dense device tensors (kept alive by the object): q as w4_pack lays it out, scale
    (2 bytes an element) and zero [ceil(in_f / group), out_f]. The scale type is the scale tensor's
    unless dtype_scale says otherwise."""
    _dtype(q, "u8", "make_w4: q")
    _dtype(zero, "u8", "make_w4: zero")
    if dtype_scale is None:
        dtype_scale = torch_dtype_code(scale.dtype)
    if hasattr(scale, "element_size") and scale.element_size() != 2:
        _refuse(f"make_w4: scales of {scale.dtype}")
    groups = -(-in_f // group) if group > 0 else 0
    for t, n, name in ((q, w4_weight_bytes(in_f, out_f), "q"), (scale, groups * out_f, "scale"),
                       (zero, groups * out_f, "zero")):
        if hasattr(t, "numel") and not (t.is_contiguous() and t.numel() >= n):
            _refuse(f"make_w4: {name} of shape {tuple(t.shape)}, strides {t.stride()}, for {in_f} inputs and "
                    f"{out_f} outputs in groups of {group}")
    for name, t in (("scale", scale), ("zero", zero)):
        if getattr(t, "ndim", 0) == 2 and groups and tuple(t.shape) != (groups, out_f):
            _refuse(f"make_w4: {name} of shape {tuple(t.shape)}, not {(groups, out_f)}")
    w = W4(in_f, out_f, group, dtype_scale, _ptr(q), _ptr(scale), _ptr(zero))
    w._keepalive = (q, scale, zero)
    return w


def linear_w4_workspace_bytes(m, in_f, out_f) -> int:
    return lib().eb_linear_w4_workspace_bytes(m, in_f, out_f)


def _refuse(what):
    lib()
    raise EbError(1, what)


def _row_stride(t, shape, what) -> int:
    """Stride of the rows of [rows, n] or of one row [n]; other layouts have none, nor do rows that
    are one (an expanded tensor)."""
    st = t.stride()
    if len(st) == 2 and (st[1] == 1 or shape[1] < 2):
        if shape[0] < 2:
            return 0
        if st[0] >= shape[1]:
            return st[0]
    elif len(st) == 1 and (st[0] == 1 or shape[0] < 2):
        return 0
    _refuse(f"{what}: rows of a tensor of shape {tuple(shape)}, strides {st}")


_names = {}  # dtype -> its name


def _dtype(t, name, what):
    """Refuses a tensor of another type (u8: any of one byte)."""
    if not hasattr(t, "element_size"):
        return
    have = _names.get(t.dtype)
    if have is None:
        have = _names[t.dtype] = "u8" if t.element_size() == 1 else str(t.dtype)[6:]
    if have != name:
        _refuse(f"{what}: {t.dtype}, not {name}")


def linear_w4(w: W4, x, y, m, workspace=None, stream=None):
    """eb_linear_w4: y [m, out_f] = x [m, in_f] @ W^T with 4-bit weights; x and y are tensors in
    f32, f16 or bf16 of [m, n] or, of one row, [n], whose rows may be strided."""
    xs, ys = x.shape, y.shape
    if (m > (xs[0] if len(xs) > 1 else 1) or m > (ys[0] if len(ys) > 1 else 1)
            or xs[-1] < w.in_f or ys[-1] < w.out_f):
        _refuse(f"linear_w4: {m} rows of {tuple(xs)} and {tuple(ys)}")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_linear_w4(w, _ptr(x), torch_dtype_code(x.dtype),
                              _row_stride(x, xs, "linear_w4"), _ptr(y),
                              torch_dtype_code(y.dtype),
                              _row_stride(y, ys, "linear_w4"), m, _ptr(workspace), ws_bytes,
                              _stream(stream)), "eb_linear_w4")


def rope_tables(max_seq: int, head_dim: int, theta: float, rope_angles: int | None = None):
    """Rope::build / build_partial tables (host, f64 math) as numpy f32 arrays."""
    import numpy as np
    if rope_angles is None:
        rope_angles = head_dim // 2
    cos = np.empty(max_seq * (head_dim // 2), np.float32)
    sin = np.empty_like(cos)
    _check(lib().eb_rope_tables(cos.ctypes.data, sin.ctypes.data, max_seq, head_dim, rope_angles,
                                theta), "eb_rope_tables")
    return cos, sin


# ---------------------------------------------------------------- fused primitive
def make_desc(n_heads, n_kv_heads, head_dim, max_seq, *, dtype_qkv=EB_F32, dtype_cache=EB_F32,
              dtype_out=EB_F32, eps=1e-6, scale=None, q_stride=0, kv_stride=0, o_stride=0,
              window=0):
    """eb_attn_desc. window > 0 restricts each query row i to key rows
    i - window < j <= i (sliding-window layers); 0 attends the whole causal
    context."""
    if scale is None:
        scale = head_dim ** -0.5
    return AttnDesc(n_heads, n_kv_heads, head_dim, max_seq, dtype_qkv, dtype_cache, dtype_out,
                    q_stride, kv_stride, o_stride, eps, scale, window)


def make_layer(q_norm_w=None, k_norm_w=None, v_norm_w=None, rope_cos=None, rope_sin=None):
    """eb_attn_layer over device tensors. The struct keeps references to the
    tensors, so they stay allocated for as long as the layer object lives."""
    layer = AttnLayer(_ptr(q_norm_w), _ptr(k_norm_w), _ptr(v_norm_w), _ptr(rope_cos),
                      _ptr(rope_sin))
    layer._keepalive = (q_norm_w, k_norm_w, v_norm_w, rope_cos, rope_sin)
    return layer


def attention_prefill_workspace_bytes(desc, seq) -> int:
    return lib().eb_attention_prefill_workspace_bytes(ctypes.byref(desc), seq)


def attention_prefill(desc, layer, seq, q, k, v, kcache, vcache, o, workspace=None, stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_prefill(ctypes.byref(desc), ctypes.byref(layer), seq, _ptr(q),
                                      _ptr(k), _ptr(v), _ptr(kcache), _ptr(vcache), _ptr(o),
                                      _ptr(workspace), ws_bytes, _stream(stream)),
           "eb_attention_prefill")


def attention_prefill_kv(desc, layer, seq, k, v, kcache, vcache, workspace=None, stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_prefill_kv(ctypes.byref(desc), ctypes.byref(layer), seq, _ptr(k),
                                         _ptr(v), _ptr(kcache), _ptr(vcache), _ptr(workspace),
                                         ws_bytes, _stream(stream)), "eb_attention_prefill_kv")


def attention_prefill_attend(desc, layer, seq, q, kcache, vcache, o, workspace=None,
                             stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_prefill_attend(ctypes.byref(desc), ctypes.byref(layer), seq,
                                             _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(o),
                                             _ptr(workspace), ws_bytes, _stream(stream)),
           "eb_attention_prefill_attend")


def attention_prefill_gather(desc, layer, seq, q, k, v, kcache, vcache, gather: HeadGather,
                             workspace=None, stream=None):
    """eb_attention_prefill with the head gather fused into the attention kernel."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_prefill_gather(ctypes.byref(desc), ctypes.byref(layer), seq,
                                             _ptr(q), _ptr(k), _ptr(v), _ptr(kcache),
                                             _ptr(vcache), ctypes.byref(gather), _ptr(workspace),
                                             ws_bytes, _stream(stream)),
           "eb_attention_prefill_gather")


def attention_prefill_attend_gather(desc, layer, seq, q, kcache, vcache, gather: HeadGather,
                                    workspace=None, stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_prefill_attend_gather(ctypes.byref(desc), ctypes.byref(layer), seq,
                                                    _ptr(q), _ptr(kcache), _ptr(vcache),
                                                    ctypes.byref(gather), _ptr(workspace),
                                                    ws_bytes, _stream(stream)),
           "eb_attention_prefill_attend_gather")


def head_broadcast(local, multicast_ptr: int, rows, n_heads_total, head_offset, n_heads,
                   head_dim, dtype, stream=None):
    """eb_head_broadcast: this rank's heads of `local` into every rank's buffer
    through the multicast address."""
    _check(lib().eb_head_broadcast(_ptr(local), multicast_ptr, rows, n_heads_total, head_offset,
                                   n_heads, head_dim, dtype, _stream(stream)),
           "eb_head_broadcast")


def attention_decode_workspace_bytes(desc, batch, max_pos) -> int:
    return lib().eb_attention_decode_workspace_bytes(ctypes.byref(desc), batch, max_pos)


def attention_decode(desc, layer, pos, q, k, v, kcache, vcache, o, workspace=None, stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_decode(ctypes.byref(desc), ctypes.byref(layer), pos, _ptr(q),
                                     _ptr(k), _ptr(v), _ptr(kcache), _ptr(vcache), _ptr(o),
                                     _ptr(workspace), ws_bytes, _stream(stream)),
           "eb_attention_decode")


def attention_decode_batched(desc, layer, batch, positions, max_pos, q, k, v, kcache, vcache,
                             cache_batch_stride, o, workspace=None, stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_decode_batched(ctypes.byref(desc), ctypes.byref(layer), batch,
                                             _ptr(positions), max_pos, _ptr(q), _ptr(k), _ptr(v),
                                             _ptr(kcache), _ptr(vcache), cache_batch_stride,
                                             _ptr(o), _ptr(workspace), ws_bytes, _stream(stream)),
           "eb_attention_decode_batched")


def attention_decode_batched_gather(desc, layer, batch, positions, max_pos, q, k, v, kcache,
                                    vcache, cache_batch_stride, gather: HeadGather,
                                    seq_index=None, workspace=None, stream=None):
    """eb_attention_decode_batched_gather: batched decode whose kernel stores
    each output row into every rank's gathered buffer (row seq_index[b] or b,
    heads gather.head_offset + h) instead of o."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_decode_batched_gather(
        ctypes.byref(desc), ctypes.byref(layer), batch, _ptr(positions), max_pos, _ptr(q),
        _ptr(k), _ptr(v), _ptr(kcache), _ptr(vcache), cache_batch_stride, ctypes.byref(gather),
        _ptr(seq_index), _ptr(workspace), ws_bytes, _stream(stream)),
        "eb_attention_decode_batched_gather")


def attention_decode_noalloc(desc, layer, pos, q, k, v, kcache, vcache, o, stream=None):
    """eb_attention_decode_noalloc: the decode step using the library's own
    fixed device scratch instead of a caller workspace (for callers that
    cannot allocate; calls on one device must not overlap)."""
    _check(lib().eb_attention_decode_noalloc(ctypes.byref(desc), ctypes.byref(layer), pos,
                                             _ptr(q), _ptr(k), _ptr(v), _ptr(kcache),
                                             _ptr(vcache), _ptr(o), _stream(stream)),
           "eb_attention_decode_noalloc")


# ---------------------------------------------------------------- 8-bit cache
def _batches(a, b, inner, stride, what):
    """Elements that two tensors of one layout hold from their first on, and the stride between
    sequences: `stride`, or what their leading axis (in front of `inner` others) has if it is not
    dense. Sequences are dense in themselves."""
    if a.shape != b.shape or a.stride() != b.stride():
        _refuse(f"{what}: shapes {tuple(a.shape)} and {tuple(b.shape)}, strides {a.stride()} and {b.stride()}")
    if a.is_contiguous():
        return a.numel(), stride
    st = a.stride()
    if a.ndim != inner + 1 or a.numel() == 0 or not a[0].is_contiguous() or st[0] < a[0].numel() or (stride and stride != st[0]):
        _refuse(f"{what}: shape {tuple(a.shape)}, strides {st}")
    return (a.shape[0] - 1) * st[0] + a[0].numel(), st[0]


def make_kv8(k, v, k_scale, v_scale, block, batch_stride=0, scale_batch_stride=0):
    """eb_kv8 over device tensors (kept alive by the object): codes [(batch,) max_seq, kv_heads,
    head_dim] of one byte, scales f32 [(batch,) ceil(max_seq / block), kv_heads]. Sequences may lie
    apart, as a slice of a longer cache has them."""
    for t, name in ((k, "u8"), (v, "u8"), (k_scale, "float32"), (v_scale, "float32")):
        _dtype(t, name, "make_kv8")
    tensors = hasattr(k, "numel") and hasattr(v, "numel")
    if tensors:
        codes, batch_stride = _batches(k, v, 3, batch_stride, "make_kv8")
    if hasattr(k_scale, "numel") and hasattr(v_scale, "numel"):
        scales, scale_batch_stride = _batches(k_scale, v_scale, 2, scale_batch_stride, "make_kv8: scales")
    c = Kv8(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), batch_stride, scale_batch_stride, block)
    if tensors:
        c.codes, c.axes = codes, tuple(k.shape)
    if hasattr(k_scale, "numel") and hasattr(v_scale, "numel"):
        c.scales, c.scale_axes = scales, tuple(k_scale.shape)
    c._keepalive = (k, v, k_scale, v_scale)
    return c


def _kv8_plan(desc, c, batch, what):
    """What a call over `batch` sequences as desc describes them expects of its tensors: types, widths
    and strides of the rows, once per descriptor and batch. A cache that does not hold the
    sequences is refused."""
    key = bytes(desc), batch
    plan = c.plans.get(key)
    if plan:
        return plan
    rows, heads, hd = desc.max_seq, desc.n_kv_heads, desc.head_dim
    blocks = -(-rows // max(1, c.block))
    # tensors with an axis for the sequences, for the rows or blocks, and for the rest
    for have, want, stride in ((c.axes, (rows, heads, hd), c.batch_stride),
                               (c.scale_axes, (blocks, heads), c.scale_batch_stride)):
        if have is None or len(have) < len(want):
            continue
        own = have[-len(want):]
        if own[1:] != want[1:] or own[0] < want[0] or (batch > 1 and len(have) > len(want) and own[0] != want[0] and not stride):
            _refuse(f"{what}: a cache of {have}, {want} a sequence in the descriptor")
    n, s = rows * heads * hd, blocks * heads
    if (n + ((batch - 1) * (c.batch_stride or n) if batch > 1 else 0) > c.codes
            or s + ((batch - 1) * (c.scale_batch_stride or s) if batch > 1 else 0) > c.scales):
        _refuse(f"{what}: a cache of {c.codes} codes and {c.scales} scales")
    q, kv = desc.n_heads * hd, heads * hd
    types = {code: dt for dt, code in _codes().items()}
    plan = (types.get(desc.dtype_qkv), types.get(desc.dtype_out), q, desc.q_stride or q, kv, desc.kv_stride or kv,
            desc.o_stride or q)
    if len(c.plans) >= 64:
        c.plans.clear()
    c.plans[key] = plan
    return plan


def _rows(t, dtype, rows, width, stride, what):
    """Pointer of a tensor that holds `rows` rows of `width` elements, `stride` apart; others are
    refused. Pointers and None pass as they are."""
    try:
        have = t.dtype
    except AttributeError:
        return _ptr(t)
    if have is dtype and t.numel() == rows * width and (stride == width or rows == 1) and t.is_contiguous():
        return t.data_ptr()
    shape, st = t.shape, t.stride()
    if have is dtype:
        if len(shape) == 2 and st[1] == 1 and shape[1] >= width and shape[0] >= rows and (st[0] == stride or rows == 1):
            return t.data_ptr()
        if (len(shape) > 1 and shape[0] >= rows and (st[0] == stride or rows == 1) and t[0].is_contiguous()
                and t[0].numel() >= width):
            return t.data_ptr()
        # one run of elements, without an axis for the rows
        if (rows == 1 or len(shape) == 1) and t.is_contiguous() and t.numel() >= (rows - 1) * stride + width:
            return t.data_ptr()
    _refuse(f"{what}: {have}, shape {tuple(shape)}, strides {st} for {rows} rows of {width}, {stride} apart, in {dtype}")


def kv8_write(desc, layer, cache: Kv8, start, count, k, v, stream=None):
    """eb_kv8_write: rows [start, start + count) of one sequence's 8-bit cache; layer None writes
    the rows as they are."""
    dt, _, _, _, width, stride, _ = (cache.plans.get((bytes(desc), 1))
                                     or _kv8_plan(desc, cache, 1, "kv8_write"))
    _check((_lib or lib()).eb_kv8_write(desc, layer, cache, start, count,
                                        _rows(k, dt, count, width, stride, "kv8_write: k"),
                                        _rows(v, dt, count, width, stride, "kv8_write: v"), _stream(stream)),
           "eb_kv8_write")


def attention_decode_kv8_workspace_bytes(desc, batch, max_pos) -> int:
    return lib().eb_attention_decode_kv8_workspace_bytes(desc, batch, max_pos)


def attention_decode_kv8(desc, layer, cache: Kv8, batch, positions, max_pos, q, k, v, o,
                         workspace=None, stream=None):
    """eb_attention_decode_kv8: one decode step per sequence over an 8-bit cache; positions None
    puts every sequence at max_pos, k and v None append nothing."""
    what = "attention_decode_kv8"
    dt, dt_o, nq, sq, nkv, skv, so = _kv8_plan(desc, cache, batch, what)
    if hasattr(positions, "numel"):
        _dtype(positions, "int32", what)
        if positions.numel() < batch or not positions.is_contiguous():
            _refuse(f"{what}: {positions.numel()} positions for {batch} sequences, or strided")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_attention_decode_kv8(desc, layer, cache, batch, _ptr(positions), max_pos,
                                         _rows(q, dt, batch, nq, sq, what), _rows(k, dt, batch, nkv, skv, what),
                                         _rows(v, dt, batch, nkv, skv, what), _rows(o, dt_o, batch, nq, so, what),
                                         _ptr(workspace), ws_bytes, _stream(stream)), "eb_attention_decode_kv8")


# ---------------------------------------------------------------- sampling
def make_sample_params(temperature=None, top_k=None, top_p=None, min_p=None):
    """eb_sample_params over device arrays of one value per row (f32, top_k int32; None leaves a
    filter out), kept alive by the object."""
    for t, name in ((temperature, "float32"), (top_k, "int32"), (top_p, "float32"), (min_p, "float32")):
        _dtype(t, name, "make_sample_params")
    given = [t for t in (temperature, top_k, top_p, min_p) if hasattr(t, "numel")]
    if not all(t.is_contiguous() for t in given):
        _refuse("make_sample_params: strided")
    p = SampleParams(_ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p))
    p._keepalive = (temperature, top_k, top_p, min_p)
    p.rows = min((t.numel() for t in given), default=1 << 24)
    return p


def sample_workspace_bytes(rows, vocab) -> int:
    return lib().eb_sample_workspace_bytes(rows, vocab)


def sample(logits, params: SampleParams | None, u, ids, workspace=None, stream=None):
    """eb_sample: ids [rows] (int32) drawn from logits [rows, vocab] (or one row [vocab]) with the
    uniform numbers u [rows] (f32)."""
    shape = logits.shape
    rows, vocab = shape if len(shape) == 2 else (1, shape[0])
    if (u.numel() < rows or ids.numel() < rows or (params is not None and params.rows < rows)
            or not (u.is_contiguous() and ids.is_contiguous())):
        _refuse(f"sample: {rows} rows, {u.numel()} uniform numbers, {ids.numel()} ids, or strided")
    _dtype(u, "float32", "sample: u")
    _dtype(ids, "int32", "sample: ids")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().eb_sample(_ptr(logits), torch_dtype_code(logits.dtype), rows, vocab,
                           _row_stride(logits, shape, "sample"), params, _ptr(u), _ptr(ids), _ptr(workspace),
                           ws_bytes, _stream(stream)), "eb_sample")


def workspace_init(workspace, stream=None):
    _check(lib().eb_workspace_init(_ptr(workspace), workspace.numel() * workspace.element_size(),
                                   _stream(stream)), "eb_workspace_init")


def head_concat(src, dst, shards, rows, heads_per, head_dim, dtype_code, stream=None):
    _check(lib().eb_head_concat(_ptr(src), _ptr(dst), shards, rows, heads_per, head_dim,
                                dtype_code, _stream(stream)), "eb_head_concat")


def device_error() -> int:
    """Device error word (bounded-wait timeouts) of the current device; clears it."""
    bits = ctypes.c_uint32(0)
    st = lib().eb_get_device_error(ctypes.byref(bits))
    if st not in (0, 6):
        raise EbError(st, "eb_get_device_error")
    return bits.value


DEVICE_ERROR_TMA = 1 << 0       # bits of the device error word (EB_DEVICE_ERROR_*)
DEVICE_ERROR_MMA = 1 << 1
DEVICE_ERROR_SOFTMAX = 1 << 2
DEVICE_ERROR_EPILOGUE = 1 << 3
DEVICE_ERROR_SELFTEST = 1 << 5


def selftest_wait_timeout(timeout_us: int, stream=None):
    """eb_selftest_wait_timeout: a kernel whose bounded wait never completes
    gives up after timeout_us and sets DEVICE_ERROR_SELFTEST in the device
    error word (read and cleared by device_error())."""
    _check(lib().eb_selftest_wait_timeout(timeout_us, _stream(stream)),
           "eb_selftest_wait_timeout")


def alloc_workspace(nbytes: int, device=None):
    """A zeroed, 256-byte-aligned workspace tensor of at least nbytes (torch owns it)."""
    import torch
    n = max(1, (nbytes + 255) // 256 * 256)
    return torch.zeros(n, dtype=torch.uint8, device=device or "cuda")
