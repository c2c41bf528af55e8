"""CPU checks of the quantised decode step's calls: the host functions that lay 4-bit weights out,
workspace sizes, and the argument checks, which come before any device work."""
import ctypes

import numpy as np
import pytest

import _quant_oracle as qo


@pytest.mark.parametrize("in_f,out_f", [(1, 1), (31, 3), (128, 5), (129, 2), (300, 7), (4096, 4)])
def test_w4_pack_layout(eb, in_f, out_f):
    codes = np.random.default_rng(in_f).integers(0, 16, (out_f, in_f)).astype(np.uint8)
    q = eb.w4_pack(codes)
    assert q.nbytes == eb.w4_weight_bytes(in_f, out_f)
    assert np.array_equal(q, qo.w4_pack(codes))
    assert np.array_equal(qo.w4_unpack(q, in_f), codes)


def _bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def _to_bf16(x):
    """f64 -> nearest bf16 (ties to even) as f64, for normal magnitudes."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 1e-30)))
    unit = 2.0 ** (e - 7)
    return np.round(x / unit) * unit


@pytest.mark.parametrize("zero_point", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("bf16", [False, True])
def test_w4_quantize(eb, zero_point, group, bf16):
    """Codes, scales and zero points are the definition's, ragged last group included."""
    rng = np.random.default_rng(group)
    out_f, in_f = 6, 300
    w = (0.02 * rng.standard_normal((out_f, in_f))).astype(np.float32)
    w[0, :group] = 0            # a group of zeros
    w[1] = np.abs(w[1])         # one sign only
    w[2, 5] = 3.0               # an outlier
    q, scale, zero = eb.w4_quantize(w, group, zero_point, eb.EB_BF16 if bf16 else eb.EB_F16)
    codes = qo.w4_unpack(q, in_f)
    s = (_bf16(scale) if bf16 else scale).astype(np.float64)
    for g in range(-(-in_f // group)):
        part = w[:, g * group:(g + 1) * group].astype(np.float64)
        lo, hi = np.minimum(part.min(1), 0), np.maximum(part.max(1), 0)
        want = (hi - lo) / 15 if zero_point else np.maximum(hi, -lo) / 7
        want = _to_bf16(want) if bf16 else want.astype(np.float16).astype(np.float64)
        assert np.array_equal(s[g], want)
        safe = np.where(want > 0, want, 1.0)
        z = np.clip(np.round(-lo / safe), 0, 15) if zero_point else np.full(out_f, 8)
        if zero_point:
            assert np.array_equal(zero[g], z)
        t = np.where(want[:, None] > 0, np.round(part / safe[:, None]), 0) + z[:, None]
        assert np.array_equal(codes[:, g * group:(g + 1) * group], np.clip(t, 0, 15))


def test_w4_quantize_refusals(eb):
    ok = np.zeros((2, 40), np.float32)
    for bad in (np.nan, np.inf, -np.inf):
        w = ok.copy()
        w[1, 39] = bad
        with pytest.raises(eb.EbError):
            eb.w4_quantize(w)
    w = ok.copy()
    w[0, 0] = 1e6  # 1e6 / 7 passes f16
    with pytest.raises(eb.EbError):
        eb.w4_quantize(w)
    eb.w4_quantize(w, dtype_scale=eb.EB_BF16)
    for group in (0, 16, 48, 256):
        with pytest.raises(eb.EbError):
            eb.w4_quantize(ok, group)
    with pytest.raises(eb.EbError):
        eb.w4_quantize(ok, 32, False, eb.EB_F32)
    with pytest.raises(eb.EbError):
        eb.w4_pack(np.full((1, 8), 16, np.uint8))
    L = eb.lib()
    assert L.eb_w4_pack(None, 8, 1, 16) == 1 and L.eb_w4_pack(16, 0, 1, 16) == 1
    assert L.eb_w4_quantize(None, 8, 1, 32, 1, 16, 16, None) == 1
    assert eb.w4_weight_bytes(0, 4) == 0 and eb.w4_weight_bytes(4, -1) == 0


def test_linear_w4_refusals(eb):
    L = eb.lib()

    def call(w=None, x=16, dx=0, xs=0, y=16, dy=0, ys=0, m=1, **kw):
        w = eb.W4(**{**dict(in_f=256, out_f=64, group=64, dtype_scale=1, q=256, scale=256, zero=None),
                     **kw}) if w is None else w
        return L.eb_linear_w4(w, x, dx, xs, y, dy, ys, m, None, 0, None)

    assert call(m=0) == 0                       # nothing to do, no device needed
    assert L.eb_linear_w4(None, 16, 0, 0, 16, 0, 0, 1, None, 0, None) == 1
    for kw in (dict(in_f=0), dict(out_f=-1), dict(group=16), dict(group=0), dict(dtype_scale=0),
               dict(dtype_scale=3), dict(q=None), dict(q=264), dict(scale=None), dict(x=None),
               dict(y=None), dict(m=-1), dict(dx=3), dict(dy=7), dict(xs=255), dict(ys=63),
               dict(xs=-1), dict(in_f=1 << 25)):
        assert call(**kw) == 1, kw
    assert eb.linear_w4_workspace_bytes(0, 64, 64) == 0
    assert eb.linear_w4_workspace_bytes(8, 4096, 4096) == 0
    assert eb.linear_w4_workspace_bytes(8, 0, 64) == 0


def _desc(eb, **kw):
    d = eb.make_desc(8, 4, 128, 100, dtype_cache=eb.EB_E4M3)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _kv8(eb, **kw):
    return eb.Kv8(**{**dict(k=256, v=256, k_scale=256, v_scale=256, batch_stride=0,
                            scale_batch_stride=0, block=16), **kw})


def test_kv8_refusals(eb):
    L = eb.lib()

    def write(d=None, c=None, start=0, count=1, k=16, v=16, layer=None):
        return L.eb_kv8_write(d or _desc(eb), layer, c or _kv8(eb), start, count, k, v, None)

    def decode(d=None, c=None, batch=1, pos=16, max_pos=5, q=16, k=16, v=16, o=16, layer=None):
        return L.eb_attention_decode_kv8(d or _desc(eb), layer, c or _kv8(eb), batch, pos, max_pos,
                                         q, k, v, o, None, 0, None)

    assert write(count=0) == 0 and decode(batch=0) == 0
    half = eb.make_layer()
    half.rope_cos = 16  # cos without sin
    for call in (write, decode):
        for d in (dict(dtype_cache=eb.EB_F16), dict(dtype_cache=5), dict(head_dim=127), dict(n_heads=7),
                  dict(head_dim=258), dict(max_seq=0), dict(window=-1), dict(kv_stride=-1),
                  dict(dtype_qkv=3), dict(dtype_out=4)):
            assert call(d=_desc(eb, **d)) == 1, d
        for c in (dict(block=0), dict(block=8), dict(block=48), dict(block=256), dict(k=None),
                  dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=264), dict(v=257),
                  dict(batch_stride=-16), dict(scale_batch_stride=-1)):
            assert call(c=_kv8(eb, **c)) == 1, c
        assert call(layer=half) == 1
    for kw in (dict(start=-1), dict(count=-1), dict(start=100), dict(start=90, count=11),
               dict(start=(1 << 62), count=(1 << 62)), dict(k=None), dict(v=None)):
        assert write(**kw) == 1, kw
    assert write(d=_desc(eb, kv_stride=511)) == 1
    for kw in (dict(batch=-1), dict(batch=32768), dict(max_pos=-1), dict(max_pos=100), dict(q=None),
               dict(o=None), dict(k=None), dict(v=None)):
        assert decode(**kw) == 1, kw
    dense = 100 * 4 * 128
    for c in (dict(batch_stride=dense - 16), dict(batch_stride=dense + 8),
              dict(scale_batch_stride=27)):
        assert decode(batch=2, c=_kv8(eb, **c)) == 1, c
    for d in (dict(q_stride=1023), dict(kv_stride=511), dict(o_stride=1023)):
        assert decode(batch=2, d=_desc(eb, **d)) == 1, d
    # the other calls do not take the 8-bit cache types
    d8 = _desc(eb)
    assert L.eb_attention_decode(ctypes.byref(d8), None, 4, 16, 16, 16, 16, 16, 16, None, 0, None) == 1
    assert eb.attention_decode_kv8_workspace_bytes(_desc(eb, dtype_cache=0), 1, 5) == 0
    assert eb.attention_decode_kv8_workspace_bytes(_desc(eb), 0, 5) == 0
    assert eb.attention_decode_kv8_workspace_bytes(_desc(eb), 1, 100) == 0


def test_sample_refusals(eb):
    L = eb.lib()

    def call(logits=16, dtype=0, rows=1, vocab=100, stride=0, u=16, ids=16):
        return L.eb_sample(logits, dtype, rows, vocab, stride, None, u, ids, None, 0, None)

    assert call(rows=0) == 0
    for kw in (dict(logits=None), dict(u=None), dict(ids=None), dict(dtype=3), dict(dtype=-1),
               dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(stride=99),
               dict(stride=-1)):
        assert call(**kw) == 1, kw
    assert eb.sample_workspace_bytes(0, 100) == 0 and eb.sample_workspace_bytes(4, 0) == 0


def test_valid_calls_without_a_device_are_refused(eb):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    L = eb.lib()
    w = eb.W4(in_f=256, out_f=64, group=64, dtype_scale=1, q=256, scale=256, zero=None)
    assert L.eb_linear_w4(w, 16, 0, 0, 16, 0, 0, 1, None, 0, None) == 5
    assert L.eb_kv8_write(_desc(eb), None, _kv8(eb), 0, 1, 16, 16, None) == 5
    assert L.eb_attention_decode_kv8(_desc(eb), None, _kv8(eb), 1, 16, 5, 16, 16, 16, 16, None, 0,
                                     None) == 5
    assert L.eb_sample(16, 0, 1, 100, 0, None, 16, 16, None, 0, None) == 5


def test_binding_refuses_layouts_it_would_misread(eb):
    """Tensors whose rows have no stride, are too short or too few, or are of another type: refused
    before their pointers are taken."""
    import torch
    t = torch.zeros
    w = eb.make_w4(t(64, 128, dtype=torch.uint8), t(4, 64, dtype=torch.float16), None, 256, 64, 64)
    x, y = t(4, 256), t(4, 64)
    for bad_x, bad_y, m in ((x, y, 5), (x[0], y, 2), (x, y[0], 2), (x[:1].expand(4, 256), y, 4), (x.t(), y, 4),
                            (t(4, 512)[:, ::2], y, 4), (t(512)[::2], y, 1), (t(2, 2, 256), t(2, 2, 64), 2),
                            (x[:, 1:], y, 4), (x, y[:, :63], 4), (x[0, :255], y[0], 1), (x, t(64, 4).t(), 4)):
        with pytest.raises(eb.EbError) as e:
            eb.linear_w4(w, bad_x, bad_y, m)
        assert e.value.status == 1
    logits, u, ids = t(4, 100), t(4), t(4, dtype=torch.int32)
    short = eb.make_sample_params(t(3))
    for args in ((logits.t(), None, t(100), t(100, dtype=torch.int32)), (logits[:1].expand(4, 100), None, u, ids),
                 (t(4, 200)[:, ::2], None, u, ids), (logits, None, u[:3], ids), (logits, None, u, ids[:3]),
                 (logits, None, u.double(), ids), (logits, None, u, ids.long()), (logits, short, u, ids),
                 (logits, None, t(8)[::2], ids)):
        with pytest.raises(eb.EbError) as e:
            eb.sample(*args)
        assert e.value.status == 1
    for kw in (dict(temperature=t(4).double()), dict(top_k=t(4, dtype=torch.int64)), dict(top_p=t(4).half()),
               dict(min_p=t(8)[::2])):
        with pytest.raises(eb.EbError):
            eb.make_sample_params(**kw)
    k, s = t(64, 2, 64, dtype=torch.uint8), t(4, 2)
    for args in ((k.float(), k, s, s), (k, k.half(), s, s), (k, k, s.half(), s), (k, k, s, s.double())):
        with pytest.raises(eb.EbError):
            eb.make_kv8(*args, 16)
    with pytest.raises(eb.EbError):
        eb.make_w4(t(64, 128), t(4, 64, dtype=torch.float16), None, 256, 64, 64)
