"""attention_decode_kv8 over the range of scales that it promises: K scales of any size whose scores are
finite, V scales of 2^-64 to 2^95, and blocks of very different ones side by side.

Tolerance: _quant_oracle.attend's bound of what f32 arithmetic may make, half a step of o's type, and for
q and the weights in the products 2^-20 (f32 outputs) or 2^-16 of each, the weights 2^-31 or 2^-27 of the
largest at least: with E the extra relative error of a product of one of each, scores move by E |q| |k| and
o by that times 2, and by (E + rows * floor) of the weighted magnitudes."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu


def _case(eb, hd, o_dtype, ks, vs, seed=0, spread=1.0):
    import torch
    H, heads, block = 4, 2, 32
    rows = len(ks) * block
    rng = np.random.default_rng(seed)
    codes = [qo.f8_encode(spread * rng.standard_normal((rows, heads, hd)), "e4m3") for _ in "kv"]
    scale = [np.repeat(np.asarray(s, np.float64)[:, None], heads, 1) for s in (ks, vs)]
    q = (rng.standard_normal((H, hd)) / max(ks)).astype(np.float32)
    dev = lambda a, t=None: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    cache = eb.make_kv8(*(dev(c) for c in codes), *(dev(s.astype(np.float32)) for s in scale), block)
    dt = getattr(torch, o_dtype)
    desc = eb.make_desc(H, heads, hd, rows, dtype_cache=eb.EB_E4M3, dtype_out=eb.torch_dtype_code(dt))
    o = torch.empty(H * hd, device="cuda", dtype=dt)
    ws = eb.alloc_workspace(eb.attention_decode_kv8_workspace_bytes(desc, 1, rows - 1))
    eb.attention_decode_kv8(desc, None, cache, 1, None, rows - 1, dev(q), None, None, o, ws)
    K, V = (qo.f8_decode(c, "e4m3") * np.repeat(s, block, 0)[..., None] for c, s in zip(codes, scale))
    want, bound = qo.attend(q.astype(np.float64), K, V, hd ** -0.5)
    wide = o_dtype == "float32"
    E, floor = (2.0 ** -20, 2.0 ** -31) if wide else (2.0 ** -16, 2.0 ** -27)
    half = 2.0 ** -24 if wide else 2.0 ** -8
    extra = np.empty_like(want)
    for h in range(H):
        k, v = K[:, h // 2], V[:, h // 2]
        s = k @ q[h].astype(np.float64) * hd ** -0.5
        p = np.exp(s - s.max())
        p /= p.sum()
        ds = E * (np.abs(k) @ np.abs(q[h].astype(np.float64))).max() * hd ** -0.5
        extra[h] = (2 * ds + E) * (p @ np.abs(v)) + floor * (p[:, None] * np.abs(v)).max() * rows
    off = np.abs(o.double().cpu().numpy().reshape(H, hd) - want)
    assert (off <= bound + extra + half * np.abs(want)).all(), float((off / (bound + extra + half * np.abs(want))).max())


@pytest.mark.parametrize("hd", [64, 128, 256, 80])
@pytest.mark.parametrize("o_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e", [-64, -40, 0, 60, 95])
def test_v_scales(eb, hd, o_dtype, e):
    _case(eb, hd, o_dtype, [1.0] * 12, [2.0 ** e] * 12, seed=e + 100)


@pytest.mark.parametrize("hd", [64, 128, 256, 80])
@pytest.mark.parametrize("e", [-90, -30, 30, 90])
def test_k_scales(eb, hd, e):
    _case(eb, hd, "float32", [2.0 ** e] * 12, [0.25] * 12, seed=e + 100)


@pytest.mark.parametrize("hd", [64, 128, 256, 80])
@pytest.mark.parametrize("o_dtype", ["float32", "bfloat16"])
def test_v_scales_of_every_size(eb, hd, o_dtype):
    _case(eb, hd, o_dtype, [1.0] * 20, list(2.0 ** np.random.default_rng(1).integers(-64, 96, 20)), seed=7)
    _case(eb, hd, o_dtype, [1.0] * 20, [2.0 ** -64, 1.0] * 10, seed=8, spread=3.0)
