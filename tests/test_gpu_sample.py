"""GPU parity of eb_sample: ids equal the definition's in 64 bits (tests/_quant_oracle.py). Kernel and
definition sum in f64, in different orders; the ids could differ only where u times the total falls
within about 2^-48 of a running sum."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
F32_MAX = 3.4028234e38


def _run(eb, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    import torch
    rows, vocab = logits.shape
    arr = lambda v, dt: None if v is None else torch.tensor(  # noqa: E731
        np.broadcast_to(np.asarray(v), (rows,)).copy(), dtype=dt, device="cuda")
    p = eb.make_sample_params(arr(temperature, torch.float32), arr(top_k, torch.int32), arr(top_p, torch.float32),
                              arr(min_p, torch.float32))
    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    n = eb.sample_workspace_bytes(rows, vocab)
    ws = eb.alloc_workspace(n) if n else None
    u = arr(u, torch.float32)
    for _ in range(2):
        eb.sample(logits, p, u, ids, ws)
    assert eb.device_error() == 0
    return ids.cpu().numpy()


def _check(eb, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]
    got = _run(eb, logits, u, temperature, top_k, top_p, min_p)
    l = logits.double().cpu().numpy()
    b = [np.broadcast_to(np.asarray(v), (rows,)) for v in (u, temperature, top_k, top_p, min_p)]
    want = [qo.sample(l[r], *(v[r] for v in b)) for r in range(rows)]
    assert got.tolist() == want


def _logits(rows, vocab, seed, dtype="f32", spread=3.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, vocab, generator=g)).to(getattr(torch, DT[dtype])).cuda()


U = np.linspace(0, 1, 12, endpoint=False) + 0.013


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1024, 1025, 4097, 32003, 151936, 200001])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05),
                                dict(top_k=40, top_p=0.95, min_p=0.02, temperature=0.7)])
def test_vocabularies(eb, vocab, kw):
    _check(eb, _logits(12, vocab, vocab), U, **kw)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), 1e-30, 0.01, 0.5, 1.0, 3.0, 1e4, float("inf")])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_p=0.8)])
def test_temperatures(eb, dtype, temperature, kw):
    _check(eb, _logits(12, 5000, 1, dtype), U, temperature=temperature, **kw)


@pytest.mark.parametrize("top_k", [-3, 0, 1, 2, 31, 32, 33, 500, 1023, 1024, 1025, 3000, 19999, 20000, 20001, 1 << 30])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top_p", [1.0, 0.7])
def test_top_k(eb, top_k, dtype, top_p):
    _check(eb, _logits(12, 20000, 2, dtype), U, top_k=top_k, top_p=top_p)


@pytest.mark.parametrize("top_p", [-1.0, 0.0, 1e-9, 0.1, 0.5, 0.9, 0.99, 0.999, 0.999999, 1.0, 2.0, float("nan")])
@pytest.mark.parametrize("dtype,spread", [("f32", 3.0), ("bf16", 3.0), ("f32", 0.3), ("f16", 8.0)])
def test_top_p(eb, top_p, dtype, spread):
    _check(eb, _logits(12, 50257, 3, dtype, spread), U, top_p=top_p)


@pytest.mark.parametrize("min_p", [-1.0, 0.0, 1e-6, 0.05, 0.5, 1.0, 2.0, float("nan")])
def test_min_p(eb, min_p):
    _check(eb, _logits(12, 9000, 4), U, min_p=min_p)
    _check(eb, _logits(12, 9000, 4), U, min_p=min_p, top_k=100, top_p=0.9)


@pytest.mark.parametrize("vocab", [5, 3000, 70000])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_k=1500), dict(top_p=0.37), dict(min_p=1.0),
                                dict(top_k=60000, top_p=0.9)])
def test_ties(eb, vocab, kw):
    """Equal logits everywhere, and two values: the first indexes come first."""
    import torch
    flat = torch.zeros(12, vocab, device="cuda")
    _check(eb, flat, U, **kw)
    flat[:, ::3] = 1.0
    _check(eb, flat, U, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                                dict(top_k=2, top_p=0.5, temperature=2.0)])
def test_masked_and_odd_logits(eb, kw):
    """Masked tokens (-inf, the type's lowest value), NaN, +inf, rows with nothing left."""
    import torch
    rows = _logits(9, 3000, 5)
    rows[0, :] = float("-inf")
    rows[1, :] = float("nan")
    rows[2, 5:] = float("-inf")
    rows[3, 1:] = -F32_MAX
    rows[4, 17] = rows[4, 2900] = float("inf")
    rows[5, ::2] = float("nan")
    rows[6, :] = float("-inf")
    rows[6, 2999] = -50.0
    rows[7, :] = -F32_MAX
    rows[8, 3] = F32_MAX
    for u in (0.0, 0.3, 0.77, 0.999):
        _check(eb, rows, u, **kw)


@pytest.mark.parametrize("u", [0.0, -1.0, 1.0, 2.0, float("nan"), float("inf"), 1 - 2.0 ** -24, 2.0 ** -24])
def test_odd_uniforms(eb, u):
    _check(eb, _logits(12, 3333, 6), u)
    _check(eb, _logits(12, 3333, 6), u, top_k=20)
    _check(eb, _logits(12, 3333, 6, spread=40.0), u)


@pytest.mark.parametrize("rows", [1, 3, 40, 100, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.97, temperature=1.3),
                                dict(top_k=5000, temperature=2.0), dict(top_k=3000, top_p=0.95),
                                dict(min_p=0.001, temperature=1.5), dict(top_p=0.99, min_p=0.0001)])
def test_row_counts_and_wide_cuts(eb, rows, dtype, kw):
    """Few rows share a cluster of CTAs, many have one each; cuts behind some tokens and behind tens of
    thousands."""
    rng = np.random.default_rng(rows)
    _check(eb, _logits(rows, 60013, rows, dtype, 2.0), rng.random(rows).astype(np.float32), **kw)


def test_rows_with_settings_of_their_own(eb):
    rng = np.random.default_rng(0)
    rows = 60
    _check(eb, _logits(rows, 32000, 8, "bf16"), rng.random(rows).astype(np.float32),
           temperature=rng.choice([0.0, 0.3, 0.8, 1.5], rows), top_k=rng.choice([0, 1, 5, 40, 2000], rows),
           top_p=rng.choice([0.2, 0.9, 0.99, 1.0], rows), min_p=rng.choice([0.0, 0.02, 0.3], rows))


def test_strided_rows_and_no_parameters(eb):
    import torch
    wide = _logits(12, 5003, 9)
    view = wide[:, 1:4000]
    _check(eb, view, U)
    ids = torch.empty(12, dtype=torch.int32, device="cuda")
    u = torch.tensor(U, dtype=torch.float32, device="cuda")
    n = eb.sample_workspace_bytes(12, 3999)
    eb.sample(view, None, u, ids, eb.alloc_workspace(n) if n else None)
    want = [qo.sample(view[r].double().cpu().numpy(), U[r]) for r in range(12)]
    assert ids.cpu().tolist() == want


def test_frequencies(eb):
    """Over many uniforms the ids come as often as their probabilities say (stratified draws: off by at
    most one each)."""
    import torch
    n = 4096
    row = torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0], device="cuda")
    ids = _run(eb, row.repeat(n, 1), (np.arange(n) + 0.5) / n)
    p = torch.softmax(row.double(), 0).cpu().numpy()
    assert (np.abs(np.bincount(ids, minlength=5) - n * p) <= 1).all()


def test_many_rows_streams_and_graphs(eb):
    import torch
    rows, vocab = 700, 6000
    logits = _logits(rows, vocab, 10)
    rng = np.random.default_rng(1)
    u = rng.random(rows).astype(np.float32)
    _check(eb, logits, u, top_k=rng.integers(0, 60, rows), top_p=0.9)
    want = _run(eb, logits, u, top_k=50)
    p = eb.make_sample_params(top_k=torch.full((rows,), 50, dtype=torch.int32, device="cuda"))
    ud = torch.from_numpy(u).cuda()
    n = eb.sample_workspace_bytes(rows, vocab)
    outs, torch_streams = [], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for st in torch_streams:
        with torch.cuda.stream(st):
            ids, ws = torch.empty(rows, dtype=torch.int32, device="cuda"), eb.alloc_workspace(n) if n else None
            eb.sample(logits, p, ud, ids, ws)
            outs.append((ids, ws))
    torch.cuda.synchronize()
    assert all(np.array_equal(o.cpu().numpy(), want) for o, _ in outs)
    ids, ws = outs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eb.sample(logits, p, ud, ids, ws)
    ud.copy_(torch.from_numpy(u[::-1].copy()))
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(ids.cpu().numpy(), _run(eb, logits, u[::-1].copy(), top_k=50))
