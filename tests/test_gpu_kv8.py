"""GPU parity of the 8-bit KV cache: eb_kv8_write and eb_attention_decode_kv8 against their
definitions in 64 bits.

Tolerances, from the arithmetic. A code may be off the value it stands for by half a step of the type
(2^-4 or 2^-3 relative, less for subnormals) and by what f32 makes of the norm and the rotation before
it, (head_dim + 8) * 2^-23 of the row's largest value. Rows that are neither normalised nor rotated
give the definition's codes and scales exactly. Attention in f32: _quant_oracle.attend's bound; a
16-bit o adds half a step."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
EPS = 1e-6


def _randn(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def _f8(eb, f8):
    return {"e4m3": eb.EB_E4M3, "e5m2": eb.EB_E5M2}[f8]


class _Cache:
    """A batch of caches on the GPU; its definition's side as numpy arrays."""

    def __init__(self, batch, max_seq, heads, hd, block, f8, seed, pad=0, dirty=True):
        import torch
        self.block, self.f8, self.max_seq, self.heads, self.hd = block, f8, max_seq, heads, hd
        rng = np.random.default_rng(seed)
        blocks = -(-max_seq // block)
        self.np = {}
        for n in "kv":
            # what earlier calls left: any code (NaN too) unless a test fills rows
            codes = rng.integers(0, 256, (batch, max_seq, heads, hd)).astype(np.uint8)
            scale = 2.0 ** rng.integers(-12, -5, (batch, blocks, heads))
            if not dirty:
                codes[:] = 0
            self.np[n] = [codes, scale]
        self.pad = pad

    def fill(self, b, rows, seed, spread=1.0):
        """Rows [0, rows) of sequence b as a write leaves them."""
        for i, n in enumerate("kv"):
            x = spread * _randn(seed + i, rows, self.heads, self.hd).astype(np.float64)
            x *= 2.0 ** np.random.default_rng(seed + i).integers(-2, 3, (1, self.heads, 1))
            if rows:
                qo.kv8_write(self.np[n][0][b], self.np[n][1][b], 0, x, self.block, self.f8)

    def upload(self, eb):
        import torch
        self.dev = {}
        for n, (codes, scale) in self.np.items():
            row = codes[0].size
            stride = row + self.pad if self.pad else row
            flat = torch.full((codes.shape[0] * stride + 16,), 0x55, dtype=torch.uint8, device="cuda")
            for b in range(codes.shape[0]):
                flat[b * stride:b * stride + row] = torch.from_numpy(codes[b].reshape(-1).copy()).cuda()
            self.dev[n] = [flat, torch.from_numpy(scale.astype(np.float32)).cuda(), stride]
        k, v = self.dev["k"], self.dev["v"]
        return eb.make_kv8(k[0], v[0], k[1], v[1], self.block, k[2] if self.pad else 0)

    def download(self):
        out = {}
        for n, (codes, scale) in self.np.items():
            flat, s, stride = self.dev[n]
            row = codes[0].size
            f = flat.cpu().numpy()
            got = np.stack([f[b * stride:b * stride + row] for b in range(codes.shape[0])]).reshape(codes.shape)
            if self.pad:
                for b in range(codes.shape[0]):
                    assert (f[b * stride + row:(b + 1) * stride] == 0x55).all()
            out[n] = (got, s.double().cpu().numpy())
        return out


def _tables(max_seq, hd, theta=1e4):
    t = np.arange(max_seq)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(t).astype(np.float32), np.sin(t).astype(np.float32)


def _dev(x, dtype="f32"):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(getattr(torch, DT[dtype])).cuda()


def _near(got, scale, want, f8, err):
    """Codes `got` at `scale` stand for `want` within half a step and err (both per value)."""
    val = qo.f8_decode(got, f8) * scale
    off = np.abs(val - want)
    assert (off <= qo.f8_step(want, scale, f8) / 2 + err).all(), float((off - err).max())


# ---------------------------------------------------------------- rows in
@pytest.mark.parametrize("f8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,heads", [(64, 3), (128, 2), (256, 1), (80, 2), (2, 1)])
@pytest.mark.parametrize("start,count", [(0, 1), (0, 300), (37, 1), (31, 65), (127, 130), (64, 64)])
def test_write_exact(eb, f8, block, hd, heads, start, count):
    """Rows as they are: codes, scales and untouched bytes are the definition's."""
    c = _Cache(1, 400, heads, hd, block, f8, hd + block + start)
    c.fill(0, start, 5)
    cache = c.upload(eb)
    rows = {n: _randn(i + count, count, heads, hd) * np.float32(4.0 ** (i + 1)) for i, n in enumerate("kv")}
    rows["k"][0, 0, 0], rows["v"][-1, -1, -1] = np.nan, -np.inf
    rows["k"][:, -1, 1:] *= np.float32(2.0 ** -20)
    if count > 100:
        rows["v"][70] = 0
    desc = eb.make_desc(heads, heads, hd, 400, dtype_cache=_f8(eb, f8))
    eb.kv8_write(desc, None, cache, start, count, _dev(rows["k"]), _dev(rows["v"]))
    got = c.download()
    for n in "kv":
        codes, scale = c.np[n]
        qo.kv8_write(codes[0], scale[0], start, rows[n].astype(np.float64), block, f8)
        assert np.array_equal(got[n][1], scale), n
        nan = (codes & 0x7F) == 0x7F
        assert np.array_equal(np.where(nan, codes & 0x7F, codes),
                              np.where(nan, got[n][0] & 0x7F, got[n][0])), n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,block", [(64, 32), (128, 64), (128, 16), (256, 128), (96, 64)])
@pytest.mark.parametrize("start,count", [(0, 150), (45, 3)])
def test_write_norm_rope_strided(eb, dtype, hd, block, start, count):
    """Rows of a fused projection, normalised and rotated."""
    heads, max_seq = 3, 200
    c = _Cache(1, max_seq, heads, hd, block, "e4m3", 1)
    c.fill(0, start, 5, 0.5)
    cache = c.upload(eb)
    wide = _randn(2, count, 4 * heads * hd)
    dev = _dev(wide, dtype)
    wide = dev.double().cpu().numpy()
    kw, vw = 1 + 0.1 * _randn(3, hd), np.ones(hd, np.float32)
    cos, sin = _tables(max_seq, hd)
    desc = eb.make_desc(heads, heads, hd, max_seq, dtype_qkv=eb.torch_dtype_code(dev.dtype),
                        dtype_cache=eb.EB_E4M3, eps=EPS, kv_stride=4 * heads * hd)
    layer = eb.make_layer(None, _dev(kw), _dev(vw), _dev(cos), _dev(sin))
    eb.kv8_write(desc, layer, cache, start, count, dev[:, heads * hd:], dev[:, 2 * heads * hd:])
    got = c.download()
    at = slice(start, start + count)
    k = qo.row_rope(qo.row_norm(wide[:, heads * hd:2 * heads * hd].reshape(count, heads, hd), kw, EPS),
                    cos[at, None].astype(np.float64), sin[at, None].astype(np.float64))
    v = qo.row_norm(wide[:, 2 * heads * hd:3 * heads * hd].reshape(count, heads, hd), vw, EPS)
    for n, x in (("k", k), ("v", v)):
        codes, scale = c.np[n]
        qo.kv8_write(codes[0], scale[0], start, x, block, "e4m3")
        assert np.array_equal(got[n][1], scale), n
        s = scale[0][np.arange(start, start + count) // block][:, :, None]
        _near(got[n][0][0, at], s, x, "e4m3", (hd + 8) * 2.0 ** -23 * np.abs(x).max(-1, keepdims=True))
        rest = np.r_[0:start, start + count:max_seq]
        assert np.array_equal(got[n][0][0, rest], codes[0, rest])


@pytest.mark.parametrize("hd,heads", [(64, 3), (128, 2), (256, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift,stride", [(1, 0), (0, 1), (3, 2)])
def test_write_unaligned(eb, hd, heads, dtype, shift, stride):
    """Rows that begin at any element, tables too: the same codes and scales, twice in a row."""
    import torch
    start, count, block, max_seq, row = 21, 60, 32, 100, heads * hd + stride
    c = _Cache(1, max_seq, heads, hd, block, "e4m3", 3)
    c.fill(0, start, 5, 0.25)
    cache = c.upload(eb)
    buf = [_dev(_randn(8 + i, shift + max_seq * row), dtype) for i in range(2)]
    rows = [t[shift:shift + count * row].reshape(count, row) for t in buf]
    cos, sin = (_dev(np.concatenate([np.zeros(shift, np.float32), t.ravel()]))[shift:] for t in _tables(max_seq, hd))
    desc = eb.make_desc(heads, heads, hd, max_seq, dtype_qkv=eb.torch_dtype_code(buf[0].dtype),
                        dtype_cache=eb.EB_E4M3, eps=EPS, kv_stride=row)
    layer = eb.make_layer(None, None, None, cos, sin)
    x = [t[:, :heads * hd].double().cpu().numpy().reshape(count, heads, hd) for t in rows]
    ct, st = (t[start:start + count, None].astype(np.float64) for t in _tables(max_seq, hd))
    x[0] = qo.row_rope(x[0], ct, st)
    for _ in range(2):
        eb.kv8_write(desc, layer, cache, start, count, rows[0], rows[1])
    torch.cuda.synchronize()
    got = c.download()
    for n, t in zip("kv", x):
        codes, scale = c.np[n]
        qo.kv8_write(codes[0], scale[0], start, t, block, "e4m3")
        assert np.array_equal(got[n][1], scale), n
        s = scale[0][np.arange(start, start + count) // block][:, :, None]
        _near(got[n][0][0, start:start + count], s, t, "e4m3", (hd + 8) * 2.0 ** -23 * np.abs(t).max(-1, keepdims=True))
        rest = np.r_[0:start, start + count:max_seq]
        assert np.array_equal(got[n][0][0, rest], codes[0, rest])


# ---------------------------------------------------------------- decode
def _decode(eb, *, positions, H, heads, hd, block, f8="e4m3", dtype="f32", o_dtype=None, max_seq=None,
            window=0, norm=False, rope=True, append=True, pad=0, fused=False, max_pos=None, scale=None,
            spread=1.0, seed=0):
    """One call, checked: the appended rows and their scales, the rest of the cache, o, and empty
    slots left as they were."""
    import torch
    o_dtype = o_dtype or dtype
    B = len(positions)
    max_pos = max(positions) if max_pos is None else max_pos
    max_seq = max_seq or max_pos + 1
    c = _Cache(B, max_seq, heads, hd, block, f8, seed, pad)
    for b, p in enumerate(positions):
        if 0 <= p <= max_pos:
            c.fill(b, p if append else p + 1, 100 + b, spread)
    cache = c.upload(eb)
    width = (H + 2 * heads) * hd
    qkv = _dev(_randn(seed + 7, B, width), dtype)
    parts = qkv.split([H * hd, heads * hd, heads * hd], 1)
    q, k, v = parts if fused else [t.contiguous() for t in parts]
    qw, kw = (1 + 0.1 * _randn(3, hd), 1 + 0.1 * _randn(4, hd)) if norm else (None, None)
    cos, sin = _tables(max_seq, hd) if rope else (None, None)
    scale = hd ** -0.5 if scale is None else scale
    desc = eb.make_desc(H, heads, hd, max_seq, dtype_qkv=eb.torch_dtype_code(qkv.dtype), dtype_cache=_f8(eb, f8),
                        dtype_out=eb.torch_dtype_code(getattr(torch, DT[o_dtype])), eps=EPS, scale=scale,
                        q_stride=width if fused else 0, kv_stride=width if fused else 0, window=window)
    layer = eb.make_layer(_dev(qw), _dev(kw), None, _dev(cos), _dev(sin))
    o = torch.full((B, H * hd), 3.0, device="cuda", dtype=getattr(torch, DT[o_dtype]))
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, B, max_pos))
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    for _ in range(2):  # the second call finds the same rows, scales and workspace
        eb.attention_decode_kv8(desc, layer, cache, B, pos, max_pos, q, k if append else None,
                                v if append else None, o, ws)
    assert eb.device_error() == 0
    got, out = c.download(), o.double().cpu().numpy().reshape(B, H, hd)
    qn, kn, vn = (t.double().cpu().numpy().reshape(B, -1, hd) for t in (q, k, v))
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[o_dtype]
    for b, p in enumerate(positions):
        if not 0 <= p <= max_pos:
            assert (out[b] == 3.0).all()
            for n in "kv":
                assert np.array_equal(got[n][0][b], c.np[n][0][b]) and np.array_equal(got[n][1][b], c.np[n][1][b])
            continue
        cr, sr = (cos[p].astype(np.float64), sin[p].astype(np.float64)) if rope else (None, None)
        if append:
            new = {"k": qo.row_rope(qo.row_norm(kn[b], kw, EPS), cr, sr), "v": vn[b]}
            for n in "kv":
                codes, s = c.np[n]
                qo.kv8_write(codes[b], s[b], p, new[n][None], block, f8)
                assert np.array_equal(got[n][1][b], s[b]), (b, n)
                _near(got[n][0][b, p], s[b, p // block][:, None], new[n], f8,
                      (hd + 8) * 2.0 ** -23 * np.abs(new[n]).max(-1, keepdims=True))
                keep = np.arange(max_seq) != p
                assert np.array_equal(got[n][0][b, keep], codes[b, keep]), (b, n)
        else:
            for n in "kv":
                assert np.array_equal(got[n][0][b], c.np[n][0][b])
        lo = max(0, p + 1 - window) if window else 0
        rows = np.arange(lo, p + 1)
        K, V = (qo.f8_decode(got[n][0][b, rows], f8) * got[n][1][b, rows // block][:, :, None] for n in "kv")
        want, bound = qo.attend(qo.row_rope(qo.row_norm(qn[b], qw, EPS), cr, sr), K, V, scale)
        off = np.abs(out[b] - want)
        lim = bound + (half + 2.0 ** -24) * np.abs(want) + (2.0 ** -25 if o_dtype == "f16" else 0)
        assert (off <= lim).all(), (b, p, float((off / lim).max()))


@pytest.mark.parametrize("pos", [0, 1, 15, 16, 17, 63, 64, 127, 128, 129, 255, 300, 1000, 2047, 2048])
@pytest.mark.parametrize("hd", [64, 128, 256, 80])
def test_decode_lengths(eb, pos, hd):
    _decode(eb, positions=[pos], H=4, heads=2, hd=hd, block=16, norm=True)


@pytest.mark.parametrize("f8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_types(eb, f8, block, dtype, hd):
    _decode(eb, positions=[130, 5, 77, 400], H=6, heads=2, hd=hd, block=block, f8=f8, dtype=dtype)


@pytest.mark.parametrize("H,heads", [(1, 1), (2, 2), (3, 1), (5, 1), (7, 1), (8, 1), (16, 2), (20, 2), (32, 1),
                                     (33, 1), (64, 1), (96, 1)])
@pytest.mark.parametrize("hd,dtype", [(64, "f32"), (128, "f16"), (128, "f32"), (256, "bf16")])
def test_decode_head_layouts(eb, H, heads, hd, dtype):
    _decode(eb, positions=[200, 9], H=H, heads=heads, hd=hd, block=32, dtype=dtype, o_dtype="f32")


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 500, 10000])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
def test_decode_window(eb, window, hd):
    _decode(eb, positions=[700, 130, 128, 0, 99], H=4, heads=2, hd=hd, block=64, window=window)


@pytest.mark.parametrize("hd", [64, 128, 256, 24])
def test_decode_empty_slots_and_strides(eb, hd):
    """Positions outside [0, max_pos] mark empty slots; caches lie apart, q, k, v in fused rows."""
    _decode(eb, positions=[-1, 40, 300, 1 << 30, -(1 << 31), 0, 299], H=4, heads=2, hd=hd, block=32,
            max_pos=299, max_seq=303, pad=48, fused=True, dtype="f16")


@pytest.mark.parametrize("hd", [64, 128, 256, 100])
def test_decode_reads_only(eb, hd):
    _decode(eb, positions=[63, 500, 0], H=4, heads=2, hd=hd, block=64, append=False, rope=False)


@pytest.mark.parametrize("hd", [128, 256])
def test_decode_many_rows_split(eb, hd):
    """Contexts long enough to be split, unequal lengths in a batch."""
    _decode(eb, positions=[9000, 17, 4095, 8191], H=8, heads=2, hd=hd, block=128, max_pos=9001, max_seq=9100)


@pytest.mark.parametrize("hd,pos,H,heads", [(64, 131000, 3, 1), (128, 40000, 2, 1), (256, 40000, 6, 2), (64, 33000, 6, 3)])
def test_decode_many_chunks(eb, hd, pos, H, heads):
    """One long context in a hundred chunks and more, 256 of them in the first case."""
    _decode(eb, positions=[pos], H=H, heads=heads, hd=hd, block=128, rope=False)


@pytest.mark.parametrize("hd", [64, 128, 256, 16])
def test_decode_large_scores(eb, hd):
    """Scores of hundreds: one row takes nearly all the weight, wherever it stands."""
    _decode(eb, positions=[400, 20], H=4, heads=2, hd=hd, block=16, scale=1.0, spread=8.0)


def test_decode_block_scale_grows(eb):
    """A small row, then rows 2^3 and 2^9 times as large in the same block: earlier rows are rounded
    again, step by step as the definition says."""
    import torch
    heads, hd, block, f8 = 2, 128, 16, "e4m3"
    c = _Cache(1, 64, heads, hd, block, f8, 3)
    cache = c.upload(eb)
    desc = eb.make_desc(4, heads, hd, 64, dtype_cache=eb.EB_E4M3)
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, 1, 63))
    o = torch.empty(4 * hd, device="cuda")
    for p in range(20):
        x = {n: _randn(p + 50 * i, 1, heads, hd) * np.float32({3: 8, 9: 512}.get(p, 1)) for i, n in enumerate("kv")}
        eb.attention_decode_kv8(desc, None, cache, 1, torch.tensor([p], dtype=torch.int32, device="cuda"), p,
                                _dev(_randn(9, 4, hd)), _dev(x["k"]), _dev(x["v"]), o, ws)
        got = c.download()
        for n in "kv":
            qo.kv8_write(c.np[n][0][0], c.np[n][1][0], p, x[n].astype(np.float64), block, f8)
            assert np.array_equal(got[n][0], c.np[n][0]) and np.array_equal(got[n][1], c.np[n][1]), (p, n)


@pytest.mark.parametrize("H,heads", [(3, 3), (10, 5), (35, 7), (24, 3), (40, 4), (27, 3), (8, 8)])
@pytest.mark.parametrize("f8,dtype", [("e4m3", "bf16"), ("e5m2", "f32")])
def test_decode_neighbouring_heads(eb, H, heads, f8, dtype):
    """head_dim 64, where two KV heads share a tile: odd numbers of them, one to ten query heads each."""
    _decode(eb, positions=[333, 9, 128], H=H, heads=heads, hd=64, block=32, f8=f8, dtype=dtype, norm=True)


@pytest.mark.parametrize("heads", [1, 2, 5])
def test_decode_neighbouring_heads_split(eb, heads):
    """As many rows as make several chunks, unequal lengths, a window that begins in the middle."""
    for window in (0, 5000):
        _decode(eb, positions=[9000, 17, 4095, 8191], H=4 * heads, heads=heads, hd=64, block=128, max_pos=9001,
                max_seq=9100, window=window)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_decode_nan_stays_in_its_head(eb, hd, bad):
    """NaN in the rows of one KV head reaches the query heads of that one alone."""
    import torch
    heads, G, p = 3, 2, 200
    c = _Cache(1, p + 1, heads, hd, 16, "e4m3", 1)
    c.fill(0, p + 1, 2, 1.0)
    desc = eb.make_desc(G * heads, heads, hd, p + 1, dtype_cache=eb.EB_E4M3)
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, 1, p))
    q, outs = _dev(_randn(3, G * heads, hd)), []
    for nan in (False, True):
        if nan:
            c.np["k"][0][0, 50, bad, 3] = 0x7F
            c.np["v"][0][0, 60, bad] = 0x7F
        o = torch.empty(G * heads, hd, device="cuda")
        eb.attention_decode_kv8(desc, None, c.upload(eb), 1, torch.tensor([p], dtype=torch.int32, device="cuda"), p,
                                q, None, None, o, ws)
        outs.append(o.cpu().numpy().reshape(heads, G, hd))
    rest = np.arange(heads) != bad
    assert np.isnan(outs[1][bad]).all()
    assert np.array_equal(outs[0][rest], outs[1][rest]) and np.isfinite(outs[0]).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 40])
def test_decode_garbage_behind_the_context(eb, hd):
    """Rows past the position hold NaN codes and NaN scales: nothing of them reaches o."""
    import torch
    max_seq, p = 300, 133
    c = _Cache(1, max_seq, 2, hd, 16, "e4m3", 1)
    c.fill(0, p + 1, 4)
    for n in "kv":
        c.np[n][0][0, p + 1:] = 0x7F
        c.np[n][1][0, p // 16 + 1:] = np.nan
    cache = c.upload(eb)
    desc = eb.make_desc(4, 2, hd, max_seq, dtype_cache=eb.EB_E4M3)
    q, o = _randn(2, 4, hd), torch.empty(4 * hd, device="cuda")
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, 1, max_seq - 1))
    eb.attention_decode_kv8(desc, None, cache, 1, torch.tensor([p], dtype=torch.int32, device="cuda"),
                            max_seq - 1, _dev(q), None, None, o, ws)
    rows = np.arange(p + 1)
    K, V = (qo.f8_decode(c.np[n][0][0, rows], "e4m3") * c.np[n][1][0, rows // 16][:, :, None] for n in "kv")
    want, bound = qo.attend(q.astype(np.float64), K, V, hd ** -0.5)
    assert (np.abs(o.double().cpu().numpy().reshape(4, hd) - want) <= bound + 2.0 ** -23 * np.abs(want)).all()


def test_decode_any_scales(eb):
    """A cache written elsewhere: scales that are no powers of two, read and appended to."""
    import torch
    heads, hd, block, n_rows = 2, 128, 32, 90
    rng = np.random.default_rng(3)
    c = _Cache(1, 128, heads, hd, block, "e4m3", 3)
    c.fill(0, n_rows, 4)
    for n in "kv":
        c.np[n][1][:] = (0.003 * (1 + rng.random(c.np[n][1].shape))).astype(np.float32)
    cache = c.upload(eb)
    desc = eb.make_desc(2, heads, hd, 128, dtype_cache=eb.EB_E4M3)
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, 1, 127))
    q, o = _randn(2, 2, hd), torch.empty(2 * hd, device="cuda")
    rows = np.arange(n_rows)
    K, V = (qo.f8_decode(c.np[n][0][0, rows], "e4m3") * c.np[n][1][0, rows // block][:, :, None] for n in "kv")
    eb.attention_decode_kv8(desc, None, cache, 1, None, n_rows - 1, _dev(q), None, None, o, ws)
    want, bound = qo.attend(q.astype(np.float64), K, V, hd ** -0.5)
    assert (np.abs(o.double().cpu().numpy().reshape(2, hd) - want) <= bound + 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize("hd", [128, 256])
def test_decode_streams_and_graphs(eb, hd):
    """A captured step replays with positions, rows and caches that changed since; two streams with a
    workspace each run side by side."""
    import torch
    B, H, heads, block, max_seq = 3, 8, 2, 64, 1500
    desc = eb.make_desc(H, heads, hd, max_seq, dtype_cache=eb.EB_E4M3)
    n = eb.attention_decode_kv8_workspace_bytes(desc, B, max_seq - 1)
    sets = []
    for i in range(2):
        c = _Cache(B, max_seq, heads, hd, block, "e4m3", i)
        for b in range(B):
            c.fill(b, 1400, 20 * i + b)
        sets.append(dict(c=c, cache=c.upload(eb), ws=eb.alloc_workspace(n), q=_dev(_randn(i, B, H * hd)),
                         k=_dev(_randn(i + 5, B, heads * hd)), v=_dev(_randn(i + 9, B, heads * hd)),
                         o=torch.zeros(B, H * hd, device="cuda"),
                         pos=torch.tensor([5, 700 + i, 1399], dtype=torch.int32, device="cuda")))

    def step(s):
        eb.attention_decode_kv8(desc, None, s["cache"], B, s["pos"], max_seq - 1, s["q"], s["k"], s["v"], s["o"],
                                s["ws"])

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                step(s)
    torch.cuda.synchronize()
    for s in sets:
        first = s["o"].clone()
        step(s)
        assert torch.equal(first, s["o"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for s in sets:
            step(s)
    for s in sets:
        s["pos"].copy_(torch.tensor([1023, 64, 0], dtype=torch.int32))
        s["k"].mul_(2.0)
    g.replay()
    torch.cuda.synchronize()
    for s in sets:
        replayed = s["o"].clone()
        step(s)
        assert torch.equal(replayed, s["o"]) and bool(torch.isfinite(replayed).all())


def test_decode_offsets_past_32_bits(eb):
    """A cache of more than 2^32 bytes: the last sequence's rows are the ones read and written."""
    import torch
    B, heads, hd, max_seq, block = 3, 8, 128, 1 << 21, 128
    size = max_seq * heads * hd
    k = torch.zeros(B * size, dtype=torch.uint8, device="cuda")
    v = torch.zeros(B * size, dtype=torch.uint8, device="cuda")
    ks = torch.zeros(B, max_seq // block, heads, device="cuda")
    vs = torch.zeros(B, max_seq // block, heads, device="cuda")
    cache = eb.make_kv8(k, v, ks, vs, block)
    desc = eb.make_desc(heads, heads, hd, max_seq, dtype_cache=eb.EB_E4M3, window=300)
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, B, max_seq - 1))
    o = torch.zeros(B, heads * hd, device="cuda")
    new = [torch.randn(B, heads * hd, generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]
    pos = torch.tensor([3, max_seq // 2, max_seq - 1], dtype=torch.int32, device="cuda")
    eb.attention_decode_kv8(desc, None, cache, B, pos, max_seq - 1, *new, o, ws)
    # one block holds something: rows of zeros have scores of zero; the new row has its own
    for b, p in enumerate(pos.tolist()):
        rows = min(p + 1, 300)
        for h in range(heads):
            at = (b * max_seq + p) * heads * hd + h * hd
            kk, vv = (t[at:at + hd].view(torch.float8_e4m3fn).double() * s[b, p // block, h].double()
                      for t, s in ((k, ks), (v, vs)))
            assert float(vv.abs().max()) > 0
            s = (new[0][b].view(heads, hd)[h].double() @ kk) * hd ** -0.5
            w = torch.exp(s) / (torch.exp(s) + rows - 1)
            got = o[b].view(heads, hd)[h].double()
            assert float((got - w * vv).abs().max()) <= (300 + 4 * hd) * 2.0 ** -23 * float(vv.abs().max())
    assert int((k != 0).view(B, -1).any(1).sum()) == B
