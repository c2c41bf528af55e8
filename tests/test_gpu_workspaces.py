"""One decode workspace, zeroed once, serves calls of every batch, head count and entry point: the
split-K tickets of a call never lie where another call's partial results went. Each output equals,
bit by bit, that of the same call with a workspace of its own."""
import pytest

pytestmark = pytest.mark.gpu


class _Kv8:
    """attention_decode_kv8 over `batch` sequences of `rows` rows; every context is split."""

    def __init__(self, eb, batch, H, heads, hd=64, rows=4096, seed=0):
        import torch
        self.eb, self.batch, self.max_pos = eb, batch, rows - 1
        g = torch.Generator(device="cuda").manual_seed(seed)
        codes = [torch.randint(0, 0x70, (batch, rows, heads, hd), device="cuda", dtype=torch.uint8, generator=g)
                 for _ in "kv"]
        self.cache = eb.make_kv8(*codes, *(torch.full((batch, rows // 64, heads), 2.0 ** -8, device="cuda") for _ in "kv"),
                                 64)
        self.desc = eb.make_desc(H, heads, hd, rows, dtype_cache=eb.EB_E4M3)
        self.q = torch.randn(batch, H * hd, device="cuda", generator=g)
        self.bytes = eb.attention_decode_kv8_workspace_bytes(self.desc, batch, self.max_pos)
        assert self.bytes > 0

    def __call__(self, ws):
        import torch
        o = torch.full_like(self.q, float("nan"))
        self.eb.attention_decode_kv8(self.desc, None, self.cache, self.batch, None, self.max_pos, self.q, None, None, o, ws)
        return o


class _Batched:
    """attention_decode_batched over f16 caches."""

    def __init__(self, eb, batch, H, heads, hd=128, rows=2048, seed=0):
        import torch
        self.eb, self.batch, self.rows = eb, batch, rows
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
        self.cache = [rand(batch, rows, heads, hd) for _ in "kv"]
        self.desc = eb.make_desc(H, heads, hd, rows, dtype_qkv=eb.EB_F16, dtype_cache=eb.EB_F16)
        self.q, self.new = rand(batch, H * hd), [rand(batch, heads * hd) for _ in "kv"]
        self.pos = torch.full((batch,), rows - 1, device="cuda", dtype=torch.int32)
        self.bytes = eb.attention_decode_workspace_bytes(self.desc, batch, rows - 1)
        assert self.bytes > 0

    def __call__(self, ws):
        import torch
        o = torch.full((self.batch, self.q.shape[1]), float("nan"), device="cuda")
        self.eb.attention_decode_batched(self.desc, self.eb.make_layer(), self.batch, self.pos, self.rows - 1, self.q, *self.new,
                                         *self.cache, self.cache[0].stride(0), o, ws)
        return o


def _together(eb, calls):
    import torch
    want = [c(eb.alloc_workspace(c.bytes)) for c in calls]
    assert all(bool(torch.isfinite(w).all()) for w in want)
    ws = eb.alloc_workspace(max(c.bytes for c in calls))
    for turn in range(2):
        for i in list(range(len(calls))) + [0]:
            assert torch.equal(calls[i](ws), want[i]), (turn, i)
    assert eb.device_error() == 0


def test_kv8_batches_share_a_workspace(eb):
    """40 sequences, then one, then 40, then 17 of another head count."""
    _together(eb, [_Kv8(eb, 40, 16, 8), _Kv8(eb, 1, 8, 8), _Kv8(eb, 40, 16, 8, seed=1), _Kv8(eb, 17, 32, 2)])


def test_kv8_head_counts_share_a_workspace(eb):
    _together(eb, [_Kv8(eb, 1, 96, 48), _Kv8(eb, 1, 8, 8), _Kv8(eb, 2, 128, 64), _Kv8(eb, 1, 16, 2, 256)])


def test_kv8_many_sequences_share_a_workspace(eb):
    """More (sequence, head) pairs than the fixed part of the workspace has tickets for."""
    _together(eb, [_Kv8(eb, 520, 32, 32, 128, 4224), _Kv8(eb, 1, 8, 8), _Kv8(eb, 40, 16, 8)])


def test_batched_decode_shares_a_workspace(eb):
    _together(eb, [_Batched(eb, 20, 32, 8), _Batched(eb, 1, 8, 8), _Batched(eb, 3, 64, 64), _Kv8(eb, 40, 16, 8),
                   _Kv8(eb, 1, 8, 8)])


def test_noalloc_head_counts(eb):
    """The library's own scratch under eb_attention_decode_noalloc: 8 heads, then 128."""
    import torch
    rows, hd = 2048, 128
    calls = []
    for H, heads in ((8, 8), (128, 128), (16, 8)):
        g = torch.Generator(device="cuda").manual_seed(H)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731,B023
        desc = eb.make_desc(H, heads, hd, rows, dtype_qkv=eb.EB_F16, dtype_cache=eb.EB_F16)
        calls.append((desc, rand(H * hd), rand(heads * hd), rand(heads * hd), rand(rows, heads, hd), rand(rows, heads, hd)))
    want = []
    for desc, q, k, v, kc, vc in calls:
        o = torch.empty(q.shape[0], device="cuda")
        n = eb.attention_decode_workspace_bytes(desc, 1, rows - 1)
        eb.attention_decode(desc, eb.make_layer(), rows - 1, q, k, v, kc, vc, o, eb.alloc_workspace(n))
        want.append(o)
    for _ in range(2):
        for (desc, q, k, v, kc, vc), w in zip(calls, want):
            o = torch.full_like(w, float("nan"))
            eb.attention_decode_noalloc(desc, eb.make_layer(), rows - 1, q, k, v, kc, vc, o)
            assert torch.equal(o, w)
    assert eb.device_error() == 0
