"""CPU checks: calls of the quantised decode step that the library or its binding refuses before any
device work, because the kernels would read or write elsewhere than the caller means."""
import pytest


def test_contexts_that_pass_32_bits_are_refused(eb):
    """The kernels step over a context's rows in 32 bits: 2^30 rows at most."""
    L = eb.lib()
    cache = eb.Kv8(k=256, v=256, k_scale=256, v_scale=256, batch_stride=0, scale_batch_stride=0, block=128)
    for rows, want in (((1 << 30) + 1, 1), ((1 << 31) - 1, 1)):
        for hd in (2, 64):
            d = eb.make_desc(1, 1, hd, rows, dtype_cache=eb.EB_E4M3)
            assert L.eb_attention_decode_kv8(d, None, cache, 1, None, rows - 1, 16, 16, 16, 16, None, 0, None) == want
            assert L.eb_kv8_write(d, None, cache, 0, 1, 16, 16, None) == want
            assert eb.attention_decode_kv8_workspace_bytes(d, 1, rows - 1) == 0
    d = eb.make_desc(1, 1, 64, 1 << 30, dtype_cache=eb.EB_E4M3)
    assert eb.attention_decode_kv8_workspace_bytes(d, 1, (1 << 30) - 1) > 0


def _refused(eb, call, *args, **kw):
    with pytest.raises(eb.EbError) as e:
        call(*args, **kw)
    assert e.value.status == 1, e.value


def test_w4_weights_the_kernel_would_misread(eb):
    """Tensors that are too small, not dense, of another element size or the other way round."""
    import torch
    in_f, out_f, group = 300, 48, 64  # five groups, three blocks
    q, s, z = (torch.zeros(out_f, 192, dtype=torch.uint8), torch.zeros(5, out_f).half(),
               torch.zeros(5, out_f, dtype=torch.uint8))
    make = lambda q=q, s=s, z=z, **kw: eb.make_w4(q, s, z, in_f, out_f, group, **kw)  # noqa: E731
    for ok in (make(), make(z=None), make(s=s.bfloat16()), make(q=q.flatten(), s=s.flatten(), z=z.flatten()),
               make(s=torch.zeros(5, out_f, dtype=torch.int16), dtype_scale=eb.EB_BF16)):
        assert (ok.in_f, ok.out_f, ok.group) == (in_f, out_f, group)
    for bad in (dict(q=q[:, :191]), dict(q=q[:47]), dict(q=torch.zeros(192, out_f, dtype=torch.uint8).t()),
                dict(q=torch.zeros(out_f, 384, dtype=torch.uint8)[:, ::2]), dict(s=s[:4]), dict(s=s.t()),
                dict(s=torch.zeros(out_f, 5).half().t()), dict(s=s.t().contiguous()), dict(s=s[:1].expand(5, out_f)),
                dict(s=s.float()), dict(s=s.float(), dtype_scale=eb.EB_F16), dict(z=z[:4]), dict(z=z.t().contiguous()),
                dict(z=torch.zeros(out_f, 5, dtype=torch.uint8).t()), dict(z=z.float()), dict(s=s.flatten()[:-1])):
        _refused(eb, make, **bad)


def _cache(eb, B=2, S=96, h=2, hd=64, block=32, make=None):
    import torch
    t = [torch.zeros(B, S, h, hd, dtype=torch.uint8) for _ in "kv"] + [torch.zeros(B, -(-S // block), h) for _ in "kv"]
    return eb.make_kv8(*(make(t) if make else t), block)


def test_kv8_caches_the_kernels_would_misread(eb):
    """Sequences that are not dense in themselves, K and V of different layouts, scales that are too
    few; a slice of a longer cache has a stride of its own."""
    import torch
    c = _cache(eb)
    assert c.batch_stride == 0 and c.scale_batch_stride == 0
    c = _cache(eb, make=lambda t: [x[:, :64] for x in t[:2]] + [x[:, :2] for x in t[2:]])
    assert c.batch_stride == 96 * 2 * 64 and c.scale_batch_stride == 3 * 2
    for make in (lambda t: [x.transpose(1, 2) for x in t[:2]] + t[2:],          # [B, heads, rows, hd]
                 lambda t: [x[..., ::2] for x in t[:2]] + t[2:],
                 lambda t: [x[:, ::2] for x in t[:2]] + t[2:],
                 lambda t: [x[:1].expand(2, -1, -1, -1) for x in t[:2]] + t[2:],
                 lambda t: [t[0], t[1][:, :64]] + t[2:],
                 lambda t: t[:2] + [x.transpose(1, 2) for x in t[2:]],
                 lambda t: t[:2] + [t[2], t[3][:, :2]]):
        _refused(eb, _cache, eb, make=make)
    k, s = torch.zeros(2, 96, 2, 64, dtype=torch.uint8), torch.zeros(2, 3, 2)
    _refused(eb, eb.make_kv8, k[:, :64], k[:, :64], s, s, 32, batch_stride=64 * 2 * 64)  # they lie further apart


def _desc(eb, **kw):
    return eb.make_desc(4, 2, 64, 96, dtype_cache=eb.EB_E4M3, **kw)


def test_kv8_caches_smaller_than_the_descriptor_are_refused(eb):
    import torch
    k, q, o = torch.zeros(2, 2 * 64), torch.zeros(2, 4 * 64), torch.zeros(2, 4 * 64)
    pos = torch.zeros(2, dtype=torch.int32)
    decode = lambda c, batch=2, d=None: eb.attention_decode_kv8(  # noqa: E731
        d or _desc(eb), None, c, batch, pos, 95, q, k, k, o, None, 0)
    write = lambda c, d=None: eb.kv8_write(d or _desc(eb), None, c, 0, 0, k, k, 0)  # noqa: E731
    write(_cache(eb))  # no rows: nothing to do, no device needed
    for c in (_cache(eb, S=95), _cache(eb, h=1), _cache(eb, hd=32), _cache(eb, make=lambda t: t[:2] + [x[:, :2] for x in t[2:]]),
              _cache(eb, make=lambda t: [x.flatten()[:2 * 96 * 128 - 1] for x in t[:2]] + t[2:])):
        _refused(eb, decode, c)
    for c in (_cache(eb, S=95), _cache(eb, h=1), _cache(eb, hd=32), _cache(eb, make=lambda t: t[:2] + [x[0, :2] for x in t[2:]])):
        _refused(eb, write, c)
    _refused(eb, decode, _cache(eb, B=1))
    _refused(eb, decode, _cache(eb, S=100))  # dense sequences of 100 rows, read as of 96
    longer, few = _cache(eb, S=130)._keepalive[2:], _cache(eb, h=3)._keepalive[2:]
    for scales in (longer, few):             # five blocks a sequence, read as three; three heads, as two
        _refused(eb, decode, _cache(eb, make=lambda t: t[:2] + list(scales)))  # noqa: B023
    write(_cache(eb, make=lambda t: t[:2] + list(longer)))
    both = _cache(eb, make=lambda t: [x.flatten(0, 1) for x in t])  # no axis for the sequences: dense
    eb.attention_decode_kv8(_desc(eb), None, both, 0, None, 95, q, k, k, o, None, 0)
    eb._kv8_plan(_desc(eb), both, 2, "dense")
    write(_cache(eb, S=100))                 # one sequence: the first 96 of its rows
    write(_cache(eb, make=lambda t: [x.flatten() for x in t[:2]] + t[2:]))


@pytest.mark.parametrize("dtype", ["float64", "int64", "float32", "int16"])
def test_kv8_positions_are_int32(eb, dtype):
    """int64, torch's default, would be read as pairs of int32 and rows appended elsewhere."""
    import torch
    t = torch.zeros(2, 4 * 64)
    _refused(eb, eb.attention_decode_kv8, _desc(eb), None, _cache(eb), 2, torch.zeros(2, dtype=getattr(torch, dtype)), 95,
             t, t[:, :128], t[:, :128], t, None, 0)


def test_kv8_positions_are_dense_and_enough(eb):
    import torch
    t = torch.zeros(2, 4 * 64)
    for pos in (torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        _refused(eb, eb.attention_decode_kv8, _desc(eb), None, _cache(eb), 2, pos, 95, t, t[:, :128], t[:, :128], t, None, 0)


def test_kv8_rows_the_kernels_would_misread(eb):
    """Rows of another type, too few, too short, strided or further apart than the descriptor says."""
    import torch
    t = torch.zeros
    q, k, o = t(2, 256), t(2, 128), t(2, 256)
    fused = t(2, 512)
    pos = t(2, dtype=torch.int32)

    def decode(q=q, k=k, v=k, o=o, d=None):
        eb.attention_decode_kv8(d or _desc(eb), None, _cache(eb), 2, pos, 95, q, k, v, o, None, 0)

    def write(k=k, v=k, count=2, d=None):
        eb.kv8_write(d or _desc(eb), None, _cache(eb), 0, count, k, v, 0)

    strided = _desc(eb, q_stride=512, kv_stride=512)
    wide = _desc(eb, dtype_out=eb.EB_BF16)
    for kw in (dict(q=q.half()), dict(k=k.half()), dict(v=k.bfloat16()), dict(o=o.half()), dict(d=wide), dict(q=q[:1]),
               dict(q=q[:, :255]), dict(k=k[:, :127]), dict(v=k[:1]), dict(o=o[:, :255]), dict(q=fused[:, :256]),
               dict(q=fused), dict(k=fused[:, 256:384]), dict(d=strided), dict(q=fused[:, ::2]), dict(q=t(256, 2).t()),
               dict(q=q[:1].expand(2, 256)), dict(o=fused[:, :256]), dict(q=t(511))):
        _refused(eb, decode, **kw)
    for kw in (dict(k=k.half()), dict(v=k.half()), dict(k=k[:1]), dict(v=k[:, :127]), dict(k=fused[:, :128]), dict(k=fused),
               dict(d=strided), dict(k=fused[:, ::4]), dict(count=3), dict(k=t(128, 2).t()), dict(k=t(255))):
        _refused(eb, write, **kw)


def test_w4_pack_takes_codes_as_they_are(eb):
    """Codes past a byte are refused as those past 15 are, not wrapped into its range."""
    import numpy as np
    ok = np.arange(16)[None]
    assert np.array_equal(eb.w4_pack(ok), eb.w4_pack(ok.astype(np.uint8)))
    for bad in (256, 261, -251, 16, -1):
        codes = ok.copy()
        codes[0, 3] = bad
        _refused(eb, eb.w4_pack, codes)
    _refused(eb, eb.w4_pack, ok + 0.5)
