"""eb_linear_w4 against the error its arithmetic allows, and what it gives exactly.

An activation is a whole number of units, a power of two per (row, block of 128 inputs): with m the
block's largest magnitude the unit is 2^(floor(log2 m) - 21), 2^-121 at least, and the activation is off
by half a unit at most (2^-22 of m). Rounding errors of different activations are independent and even
over the unit, so an output's error from them has variance sum (unit^2 / 12) W^2 =: q^2. A group's sum is
whole; what follows is f32: at most n = groups + 32 sums in a row (one per group where a warp has all of
them; the join of the planes, the warps and the cluster after that), each off by at most 2^-24 of a partial
sum, evenly (variance 1/3 of the square), and partial sums of independent products grow in the mean square
to W^2 x^2 summed, half of it on average: f^2 = 2^-48 n / 6 * sum W^2 x^2. Zero points subtracted after the
join would break this: they cancel sums far larger than the result. The 2-norm of the errors over many
outputs is within half again of sqrt(q^2 + f^2) summed (it is a mean over hundreds), and none of a few
thousand outputs passes 7 of its own. The largest y in f32 is f^2's too."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu


def _make(eb, in_f, out_f, group, zero, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (out_f, in_f), device="cuda", generator=g, dtype=torch.uint8)
    groups = -(-in_f // group)
    scale = (0.01 * torch.exp(0.3 * torch.randn(groups, out_f, device="cuda", generator=g))).half()
    z = torch.randint(0, 16, (groups, out_f), device="cuda", generator=g, dtype=torch.uint8) if zero else None
    w4 = eb.make_w4(torch.from_numpy(eb.w4_pack(codes.cpu().numpy())).cuda(), scale, z, in_f, out_f, group)
    at = torch.arange(in_f, device="cuda") // group
    return w4, (codes.double() - (z[at].T.double() if zero else 8.0)) * scale[at].T.double()


def _call(eb, w4, x):
    import torch
    m = x.shape[0]
    y = torch.full((m, w4.out_f), float("nan"), device="cuda")
    n = eb.linear_w4_workspace_bytes(m, w4.in_f, w4.out_f)
    eb.linear_w4(w4, x, y, m, eb.alloc_workspace(n) if n else None)
    return y


def _within(y, x, W, group):
    import torch
    x = x.double()
    m, in_f = x.shape
    blocks = -(-in_f // 128)
    pad = torch.zeros(m, blocks * 128, device="cuda", dtype=torch.float64)
    pad[:, :in_f] = x.abs()
    top = pad.view(m, blocks, 128).amax(2)
    unit = torch.exp2((torch.floor(torch.log2(top.clamp_min(2.0 ** -140))) - 21).clamp_min(-121))
    unit = unit.repeat_interleave(128, 1)[:, :in_f]
    W2 = (W * W).T
    var = unit.square() @ W2 / 12 + 2.0 ** -48 * (-(-in_f // group) + 32) / 6 * (x.square() @ W2)
    err = y.double() - x @ W.T
    assert bool(torch.isfinite(err).all())
    norm = float(err.norm() / var.sum().sqrt())
    far = float((err.abs() / var.sqrt().clamp_min(1e-300)).max())
    assert norm <= 1.5 and far <= 7, (norm, far)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("m,in_f,out_f", [(1, 1024, 4096), (1, 14336, 1000), (4, 4100, 700), (5, 8192, 130), (6, 3000, 500),
                                          (8, 14336, 1024), (8, 384, 2000), (9, 4096, 333), (37, 4100, 503), (64, 8192, 64)])
def test_error_is_what_the_arithmetic_allows(eb, group, zero, m, in_f, out_f):
    import torch
    w4, W = _make(eb, in_f, out_f, group, zero, m + in_f)
    x = torch.randn(m, in_f, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m))
    _within(_call(eb, w4, x), x, W, group)


@pytest.mark.parametrize("m", [1, 5, 8, 20])
@pytest.mark.parametrize("group", [32, 128])
def test_large_and_small_values_in_a_block(eb, m, group):
    """Values over 2^20 within each block of 128, and blocks of very different sizes: every one is rounded
    at its own block's unit. 2^-110 and 2^-140 lie below the smallest unit."""
    import torch
    in_f, out_f = 2000, 640
    w4, W = _make(eb, in_f, out_f, group, True, 5)
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, in_f, device="cuda", generator=g)
    x *= torch.exp2(torch.randint(-20, 1, (m, in_f), device="cuda", generator=g).float())
    x *= torch.exp2(torch.randint(-9, 10, (m, -(-in_f // 128)), device="cuda", generator=g).float()).repeat_interleave(128, 1)[:, :in_f]
    _within(_call(eb, w4, x), x, W, group)
    for e in (-140, -110, -60, 100):
        t = torch.randn(m, in_f, device="cuda", generator=g) * 2.0 ** e
        _within(_call(eb, w4, t), t, W, group)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 6, 7, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_codes_at_their_zero_point_give_zero(eb, m, group):
    """Weights of exactly zero: no share of a zero point is left over, whatever the number of rows."""
    import torch
    in_f, out_f = 1100, 96
    groups = -(-in_f // group)
    rng = np.random.default_rng(group)
    z = rng.integers(0, 16, (groups, out_f)).astype(np.uint8)
    codes = z[np.arange(in_f) // group].T
    w4 = eb.make_w4(torch.from_numpy(eb.w4_pack(codes)).cuda(), torch.full((groups, out_f), 0.37, device="cuda").half(),
                    torch.from_numpy(z).cuda(), in_f, out_f, group)
    x = torch.rand(m, in_f, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)) + 0.5
    assert bool((_call(eb, w4, x) == 0).all())


@pytest.mark.parametrize("m", [8, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_do_not_depend_on_their_number(eb, m, group):
    """Positive activations (their sums cancel against zero points): a row among `m` is as exact as alone."""
    import torch
    w4, W = _make(eb, 2048, 512, group, True, 3)
    x = torch.rand(m, 2048, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)) + 0.5
    want = x.double() @ W.T
    errs = [float((_call(eb, w4, t).double() - w).norm() / w.norm()) for t, w in ((x, want), (x[:1], want[:1]))]
    assert errs[0] <= 2 * errs[1] + 2.0 ** -24, errs


@pytest.mark.parametrize("m", [1, 3, 4, 8, 20])
@pytest.mark.parametrize("x_dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_value_that_is_not_finite_makes_its_row_nan(eb, m, x_dtype, bad):
    import torch
    w4, W = _make(eb, 700, 130, 64, True, 2)
    x = torch.randn(m, 700, generator=torch.Generator().manual_seed(1)).to(getattr(torch, x_dtype)).cuda()
    x[m // 2, 650] = bad
    y = _call(eb, w4, x)
    rest = [r for r in range(m) if r != m // 2]
    assert bool(torch.isnan(y[m // 2]).all()) and bool(torch.isfinite(y[rest]).all())
