"""GPU parity of eb_linear_w4 against f64 sums over the same codes, scales and zero points.

Tolerance, from the arithmetic: products are exact and summed in f32, in runs of at most 8 sums
within a group and one more per group and per part of a row; each sum is off by at most 2^-23 of its
value (the tensor core truncates), partial sums stay near the size of the result, so the relative
2-norm error is below 2^-23 * (16 + in_f / 32). A 16-bit y adds half a step (finfo.eps / 2)."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _make(eb, in_f, out_f, group, zero, s_dtype, seed):
    import torch
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (out_f, in_f)).astype(np.uint8)
    groups = -(-in_f // group)
    scale = torch.from_numpy((0.01 * np.exp(0.3 * rng.standard_normal((groups, out_f)))).astype(np.float32))
    scale = scale.to(getattr(torch, DT[s_dtype]))
    z = rng.integers(0, 16, (groups, out_f)).astype(np.uint8) if zero else None
    w4 = eb.make_w4(torch.from_numpy(eb.w4_pack(codes)).cuda(), scale.cuda(),
                    torch.from_numpy(z).cuda() if zero else None, in_f, out_f, group)
    return w4, qo.w4_weights(codes, scale.double().numpy(), z, group)


def _call(eb, w4, x, y_dtype, m, out_f, y=None):
    import torch
    y = torch.full((m, out_f), float("nan"), device="cuda", dtype=getattr(torch, DT[y_dtype])) if y is None else y
    n = eb.linear_w4_workspace_bytes(m, w4.in_f, out_f)
    eb.linear_w4(w4, x, y, m, eb.alloc_workspace(n) if n else None)
    return y


def _tol(in_f, y_dtype):
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[y_dtype]
    return 2.0 ** -23 * (16 + in_f / 32) + half


def _check(got, want, in_f, y_dtype, what=""):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= _tol(in_f, y_dtype), f"{what}: rel {rel:.3e} > {_tol(in_f, y_dtype):.3e}"


@pytest.mark.parametrize("in_f,out_f", [(1, 1), (33, 7), (128, 16), (1000, 61), (1024, 4096), (4100, 333),
                                        (8192, 130)])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 17, 64, 65])
def test_sizes(eb, in_f, out_f, m):
    import torch
    w4, W = _make(eb, in_f, out_f, 64, True, "f16", in_f + m)
    x = torch.randn(m, in_f, generator=torch.Generator().manual_seed(m)).cuda()
    _check(_call(eb, w4, x, "f32", m, out_f), x.double().cpu().numpy() @ W.T, in_f, "f32")
    assert eb.device_error() == 0


@pytest.mark.parametrize("m,in_f,out_f", [(8, 2304, 19000), (8, 14336, 4096), (1, 14336, 4096), (24, 5000, 9000)])
def test_long_rows(eb, m, in_f, out_f):
    """Rows whose inputs are staged in several pieces, over row counts that split them differently."""
    import torch
    w4, _ = _make(eb, in_f, out_f, 128, True, "f16", in_f)
    x = torch.randn(m, in_f, generator=torch.Generator().manual_seed(m)).cuda()
    codes = torch.from_numpy(qo.w4_unpack(w4._keepalive[0].cpu().numpy(), in_f)).cuda()
    g = torch.arange(in_f, device="cuda") // 128
    scale, zero = w4._keepalive[1], w4._keepalive[2]
    W = (codes.double() - zero[g].T.double()) * scale[g].T.double()
    _check(_call(eb, w4, x, "f32", m, out_f), (x.double() @ W.T).cpu().numpy(), in_f, "f32")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("x_dtype,y_dtype,s_dtype", [("f32", "f32", "bf16"), ("f16", "f16", "f16"),
                                                     ("f16", "f32", "bf16"), ("bf16", "bf16", "bf16"),
                                                     ("bf16", "f32", "f16"), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("m", [1, 4, 23])
def test_types(eb, group, zero, x_dtype, y_dtype, s_dtype, m):
    import torch
    in_f, out_f = 736, 250  # five blocks and three quarters
    w4, W = _make(eb, in_f, out_f, group, zero, s_dtype, group + m)
    x = torch.randn(m, in_f, generator=torch.Generator().manual_seed(m)).to(getattr(torch, DT[x_dtype])).cuda()
    _check(_call(eb, w4, x, y_dtype, m, out_f), x.double().cpu().numpy() @ W.T, in_f, y_dtype)


@pytest.mark.parametrize("m", [1, 7, 40])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_strides_and_alignment(eb, m, offset):
    """Rows with gaps, starting at any element; the gaps of y stay as they are."""
    import torch
    in_f, out_f = 300, 77
    w4, W = _make(eb, in_f, out_f, 32, False, "f16", 3)
    xb = torch.randn(m * 331 + 8, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    yb = torch.full((m * 91 + 8,), 7.0, device="cuda")
    x = xb[offset:offset + m * 331].view(m, 331)[:, :in_f]
    y = yb[offset:offset + m * 91].view(m, 91)[:, :out_f]
    _call(eb, w4, x, "f32", m, out_f, y)
    _check(y, x.double().cpu().numpy() @ W.T, in_f, "f32")
    y.fill_(7.0)
    assert bool((yb == 7.0).all())


def test_f32_activations_keep_their_bits(eb):
    """Values over the whole f32 range: nothing overflows or is lost in a narrower type."""
    import torch
    w4, W = _make(eb, 256, 40, 128, False, "f16", 11)
    for e in (-30, -12, 0, 17, 100):
        x = (torch.randn(2, 256, generator=torch.Generator().manual_seed(1)) * 2.0 ** e).cuda()
        _check(_call(eb, w4, x, "f32", 2, 40), x.double().cpu().numpy() @ W.T, 256, "f32", str(e))


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16"])
def test_non_finite_rows(eb, x_dtype):
    """An infinity or a NaN spoils its own row and no other."""
    import torch
    in_f, out_f, m = 260, 48, 4
    w4, W = _make(eb, in_f, out_f, 64, True, "f16", 2)
    x = torch.randn(m, in_f, generator=torch.Generator().manual_seed(1)).to(getattr(torch, DT[x_dtype])).cuda()
    x[1, 7], x[2, 100] = float("inf"), float("nan")
    y = _call(eb, w4, x, "f32", m, out_f)
    assert not bool(torch.isfinite(y[1]).any()) or bool((~torch.isfinite(y[1])).sum() >= out_f - (W[:, 7] == 0).sum())
    assert bool(torch.isnan(y[2]).all())
    rows = [0, 3]
    _check(y[rows], x[rows].double().cpu().numpy() @ W.T, in_f, "f32")


def test_quantised_weights_come_back(eb):
    """w4_quantize's packed rows through the kernel: unit vectors read W's columns, exactly."""
    import torch
    rng = np.random.default_rng(0)
    w = (0.05 * rng.standard_normal((50, 192))).astype(np.float32)
    for zero_point in (False, True):
        q, scale, zero = eb.w4_quantize(w, 64, zero_point)
        dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
        w4 = eb.make_w4(dev(q), dev(scale), dev(zero), 192, 50, 64)
        y = _call(eb, w4, torch.eye(192, device="cuda"), "f32", 192, 50)
        W = qo.w4_weights(qo.w4_unpack(q, 192), scale, zero, 64)
        assert np.array_equal(y.double().cpu().numpy().T, W)
        step = scale.astype(np.float64)[np.arange(192) // 64].T  # the half step the rounding may be off
        assert (np.abs(W - w) <= step * (0.5 + 1e-3) + 7 * 2.0 ** -11 * step).all()


@pytest.mark.parametrize("m", [1, 20])
def test_streams_graphs_and_repeats(eb, m):
    """The same call gives the same bits on another stream, in a replayed graph and beside others."""
    import torch
    w4, W = _make(eb, 2048, 512, 128, True, "f16", 9)
    x = torch.randn(m, 2048, device="cuda")
    y = _call(eb, w4, x, "f32", m, 512)
    n = eb.linear_w4_workspace_bytes(m, 2048, 512)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2, ws2 = torch.empty_like(y), eb.alloc_workspace(n) if n else None
        eb.linear_w4(w4, x, y2, m, ws2)
    y3, ws3 = torch.empty_like(y), eb.alloc_workspace(n) if n else None
    eb.linear_w4(w4, x, y3, m, ws3)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(y, y3)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eb.linear_w4(w4, x, y3, m, ws3)
    for seed in (1, 2):
        x.copy_(torch.randn(m, 2048, generator=torch.Generator().manual_seed(seed)))
        y3.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(y3, x.double().cpu().numpy() @ W.T, 2048, "f32")


def test_workspace_check(eb):
    import torch
    w4, _ = _make(eb, 256, 64, 64, False, "f16", 1)
    n = eb.linear_w4_workspace_bytes(33, 256, 64)
    x, y = torch.randn(33, 256, device="cuda"), torch.empty(33, 64, device="cuda")
    if n:
        for ws in (None, torch.empty(n - 1, dtype=torch.uint8, device="cuda")):
            with pytest.raises(eb.EbError) as e:
                eb.linear_w4(w4, x, y, 33, ws)
            assert e.value.status == 4
