"""What is measured of the operators of a quantised decode step, and their plain forms.

Four operators, each in the plain form (elementary torch operations in 32 bits,
64 where a border or a long sum needs it) and as the library's calls:

  linear_w4             y = x W^T with W in 4 bits, one scale (and zero point) per group of inputs
  kv8_write             k/v rows -> RMSNorm -> RoPE -> 8-bit cache with a scale per (block of rows, head)
  attention_decode_kv8  one decode step per sequence over such a cache: append, then attention
  sample                one token per row of logits: temperature, top-k, top-p, min-p, given uniforms

Formats (the library's header states them in full):

  4-bit weights: a row of W is cut into blocks of 128 inputs, 64 bytes each. Byte 16 c + 4 i + b of a
  block holds inputs 32 i + 8 c + 2 b (low nibble) and + 1 (high nibble); inputs past in_f hold 0.
  scale and zero are [groups, out_f]; W = scale * (code - zero), zero = 8 where there is none.

  8-bit cache: codes [max_seq, heads, head_dim], scales f32 [blocks, heads] for K and for V; a value is
  code * scale. A write keeps a block's scale, or raises it to the smallest power of two that holds the
  new rows; the block's earlier rows are then rounded again at the new scale. A write of a block's first
  row starts the block anew.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP_EXP = {"e4m3": 8, "e5m2": 15}  # the largest value of either type is 1.75 * 2^this
MIN_EXP = -64                      # no scale is below 2^this
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's fused q/k/v rows of a small decoder (hidden 1024, 16 + 2 * 8 heads of 128): latency
        dict(name="w4_token_small", op="linear_w4", m=1, in_f=1024, out_f=4096, group=128, zero=False,
             x="f32", y="f32", s="f16"),
        # one token through a gate/up pair of an 8-billion-parameter decoder, zero points
        dict(name="w4_token_gate_up", op="linear_w4", m=1, in_f=4096, out_f=28672, group=128, zero=True,
             x="bf16", y="bf16", s="bf16"),
        # eight sequences' tokens through the down projection of that decoder
        dict(name="w4_batch8_down", op="linear_w4", m=8, in_f=14336, out_f=4096, group=64, zero=False,
             x="f32", y="f32", s="f16"),
        # a batch of tokens, ragged in every size, small groups with zero points
        dict(name="w4_batch37_ragged", op="linear_w4", m=37, in_f=4100, out_f=5003, group=32, zero=True,
             x="f16", y="f32", s="f16"),
        # a prompt's rows into the cache, as the fused projection leaves them, keys rotated
        dict(name="kv8_write_prompt", op="kv8_write", start=0, count=8192, heads=8, head_dim=128,
             block=64, f8="e4m3", x="bf16", norm=False, rope=True, fused=True),
        # a piece of a prompt that begins and ends inside a block, head_dim 256, keys and values normalised
        dict(name="kv8_write_piece", op="kv8_write", start=1013, count=93, heads=4, head_dim=256,
             block=16, f8="e4m3", x="f32", norm=True, rope=True, fused=False),
        # one sequence, 2048 tokens, QK-norm and RoPE: latency
        dict(name="kv8_decode_one", op="kv8_decode", batch=1, low=2047, high=2047, max_seq=4096, q_heads=16,
             heads=8, head_dim=128, block=32, f8="e4m3", x="f32", o="f32", norm=True, window=0, fused=False),
        # a serving batch with contexts of 512 to 16384 tokens, 32/8 heads of 128
        dict(name="kv8_decode_batch", op="kv8_decode", batch=64, low=511, high=16383, max_seq=16384,
             q_heads=32, heads=8, head_dim=128, block=64, f8="e4m3", x="f16", o="f16", norm=False,
             window=0, fused=True),
        # sliding-window layers of 8/4 heads of 256, the other 8-bit type
        dict(name="kv8_decode_window", op="kv8_decode", batch=24, low=99, high=4095, max_seq=4096, q_heads=8,
             heads=4, head_dim=256, block=128, f8="e5m2", x="bf16", o="bf16", norm=True, window=1024,
             fused=True),
        # one sequence's next token, usual settings, a vocabulary of 151936: latency
        dict(name="sample_one", op="sample", rows=1, vocab=151936, x="f32", mix="usual", spread=3.0),
        # a serving batch, every row with settings of its own (greedy, each filter alone, all of them)
        dict(name="sample_batch64", op="sample", rows=64, vocab=151936, x="bf16", mix="mixed", spread=2.5),
        # a large batch, an odd vocabulary, temperature alone: every token counts
        dict(name="sample_batch256_open", op="sample", rows=256, vocab=128257, x="f32", mix="open",
             spread=2.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear_w4", "linear_w4", "kv8_write", "kv8_decode", "kv8_decode", "sample"])
    if op == "linear_w4":
        in_f, out_f = _log(rng, 96, 14336), _log(rng, 64, 28672)
        while in_f * out_f > 4096 * 28672:
            in_f, out_f = _log(rng, 96, 14336), _log(rng, 64, 28672)
        if rng.random() < 0.6:  # most real sizes are round
            in_f, out_f = max(128, in_f // 128 * 128), max(64, out_f // 64 * 64)
        x = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, m=_log(rng, 1, 64) if rng.random() < 0.7 else 1, in_f=in_f, out_f=out_f,
                    group=rng.choice([32, 64, 128]), zero=rng.random() < 0.5, x=x,
                    y=rng.choice([x, "f32"]), s=rng.choice(["f16", "bf16"]))
    if op == "kv8_write":
        return dict(op=op, start=rng.choice([0, rng.randrange(1, 3000)]), count=_log(rng, 1, 8192),
                    heads=rng.choice([1, 2, 4, 5, 8]), head_dim=rng.choice([64, 128, 256]),
                    block=rng.choice([16, 32, 64, 128]), f8=rng.choice(["e4m3", "e5m2"]),
                    x=rng.choice(["f32", "f16", "bf16"]), norm=rng.random() < 0.5,
                    rope=rng.random() < 0.7, fused=rng.random() < 0.5)
    if op == "kv8_decode":
        head_dim = rng.choice([64, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        most = 64 * 8192 * 8 * 128 // (batch * heads * head_dim)
        high = min(_log(rng, 1, 32768), most) - 1
        x = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, batch=batch, low=min(high, _log(rng, 1, 2048) - 1), high=high,
                    max_seq=high + 1 + rng.randrange(0, 100), q_heads=heads * rng.choice([1, 2, 3, 4, 5, 8]),
                    heads=heads, head_dim=head_dim, block=rng.choice([16, 32, 64, 128]),
                    f8=rng.choice(["e4m3", "e4m3", "e5m2"]), x=x, o=x, norm=rng.random() < 0.5,
                    window=rng.choice([0, 0, 0, _log(rng, 1, 2048)]), fused=rng.random() < 0.5)
    return dict(op=op, rows=_log(rng, 1, 200), vocab=_log(rng, 1000, 160000),
                x=rng.choice(["f32", "f16", "bf16"]), mix=rng.choice(["usual", "mixed", "open"]),
                spread=round(rng.uniform(1.5, 4.0), 2))


# ------------------------------------------------------------------ inputs
def _positions(case):
    """The sequences' positions: from the case alone, so that the work is the same for every seed."""
    rng = random.Random(case["batch"] * 1000003 + case["high"] * 101 + case["low"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]


def _rope_tables(rows, head_dim, theta):
    freq = theta ** (-2.0 * torch.arange(head_dim // 2, device="cuda", dtype=torch.float64) / head_dim)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _scale_exp(amax, f8):
    """Exponent of the smallest power of two that holds amax (f64 tensor, >= 0)."""
    m, e = torch.frexp(amax)
    e = e - 1 - TOP_EXP[f8] + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp_min(MIN_EXP)


def _fill_cache(g, batch, max_seq, heads, head_dim, block, f8):
    """An 8-bit cache as earlier writes leave it: codes and scales of N(0, 1) rows whose size differs
    by head and by block."""
    blocks = -(-max_seq // block)
    codes = torch.empty(batch, max_seq, heads, head_dim, device="cuda", dtype=F8[f8])
    scale = torch.empty(batch, blocks, heads, device="cuda")
    for b in range(batch):
        v = torch.randn(blocks * block, heads, head_dim, device="cuda", generator=g)
        v *= torch.exp2(torch.randn(heads, 1, device="cuda", generator=g))
        v = v.view(blocks, block, heads, head_dim)
        v *= 0.6 + torch.rand(blocks, 1, 1, 1, device="cuda", generator=g)
        s = torch.exp2(_scale_exp(v.abs().amax((1, 3)).double(), f8).float())
        scale[b] = s
        codes[b] = (v / s[:, None, :, None]).to(F8[f8]).view(-1, heads, head_dim)[:max_seq]
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = dict(case=case)
    if case["op"] == "linear_w4":
        m, in_f, out_f, group = case["m"], case["in_f"], case["out_f"], case["group"]
        blocks, groups = -(-in_f // 128), -(-in_f // group)
        codes = torch.randint(0, 16, (out_f, blocks * 128), device="cuda", generator=g, dtype=torch.uint8)
        if not case["zero"]:  # near a bell, as rounded weights are
            codes = (codes + torch.randint(0, 16, codes.shape, device="cuda", generator=g,
                                           dtype=torch.uint8) + 1) // 2
            codes = codes.clamp(0, 15)
        codes[:, in_f:] = 0
        c = codes.view(out_f, blocks, 4, 4, 4, 2).permute(0, 1, 3, 2, 4, 5)  # [.., c, i, b, nibble]
        s["q"] = (c[..., 0] | (c[..., 1] << 4)).contiguous().view(out_f, blocks * 64)
        s["scale"] = (0.01 * torch.exp(0.3 * rand(groups, out_f))).to(DT[case["s"]])
        s["zero"] = (torch.randint(5, 11, (groups, out_f), device="cuda", generator=g, dtype=torch.uint8)
                     if case["zero"] else None)
        s["x"] = rand(m, in_f).to(DT[case["x"]])
        s["y"] = torch.empty(m, out_f, device="cuda", dtype=DT[case["y"]])
    elif case["op"] == "kv8_write":
        rows, heads, hd, block = case["start"] + case["count"], case["heads"], case["head_dim"], case["block"]
        s["kc"], s["ks"] = _fill_cache(g, 1, rows + 7, heads, hd, block, case["f8"])
        s["vc"], s["vs"] = _fill_cache(g, 1, rows + 7, heads, hd, block, case["f8"])
        n, pad = case["count"], heads * hd if case["fused"] else 0
        kv = rand(n, pad + 2 * heads * hd).to(DT[case["x"]])  # [q | k | v] where fused
        s["k"], s["v"] = kv[:, pad:pad + heads * hd], kv[:, pad + heads * hd:]
        if not case["fused"]:
            s["k"], s["v"] = s["k"].contiguous(), s["v"].contiguous()
        s["kw"] = 1 + 0.1 * rand(hd) if case["norm"] else None
        s["vw"] = torch.ones(hd, device="cuda") if case["norm"] else None
        s["cos"], s["sin"] = _rope_tables(rows + 7, hd, 5e5) if case["rope"] else (None, None)
    elif case["op"] == "kv8_decode":
        batch, heads, hd, H = case["batch"], case["heads"], case["head_dim"], case["q_heads"]
        s["kc"], s["ks"] = _fill_cache(g, batch, case["max_seq"], heads, hd, case["block"], case["f8"])
        s["vc"], s["vs"] = _fill_cache(g, batch, case["max_seq"], heads, hd, case["block"], case["f8"])
        qkv = rand(batch, (H + 2 * heads) * hd).to(DT[case["x"]])
        s["q"], s["k"], s["v"] = qkv.split([H * hd, heads * hd, heads * hd], 1)
        if not case["fused"]:
            s["q"], s["k"], s["v"] = s["q"].contiguous(), s["k"].contiguous(), s["v"].contiguous()
        s["qw"], s["kw"] = (1 + 0.1 * rand(hd), 1 + 0.1 * rand(hd)) if case["norm"] else (None, None)
        s["cos"], s["sin"] = _rope_tables(case["max_seq"], hd, 1e6)
        s["pos"] = torch.tensor(_positions(case), device="cuda", dtype=torch.int32)
        s["o"] = torch.empty(batch, H * hd, device="cuda", dtype=DT[case["o"]])
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = case["spread"] * rand(rows, vocab)
        # a few tokens that stand out, as a trained model's do
        n = min(vocab, 24)
        at = torch.randint(0, vocab, (rows, n), device="cuda", generator=g)
        logits.scatter_add_(1, at, 2.0 * case["spread"] + 2.0 * rand(rows, n))
        s["logits"] = logits.to(DT[case["x"]])
        s["u"] = torch.rand(rows, device="cuda", generator=g)
        i = torch.arange(rows, device="cuda")
        t = 0.6 + 0.8 * torch.rand(rows, device="cuda", generator=g)
        if case["mix"] == "usual":
            k, p, q = torch.full_like(i, 50), torch.full_like(t, 0.95), torch.zeros_like(t)
        elif case["mix"] == "open":
            k, p, q = torch.zeros_like(i), torch.ones_like(t), torch.zeros_like(t)
        else:
            kind = i % 6  # greedy, top-k, top-p, min-p, top-k and top-p, all
            t = torch.where(kind == 0, torch.zeros_like(t), t)
            k = torch.where((kind == 1) | (kind >= 4), 1 + (37 * i) % 200, torch.zeros_like(i))
            p = torch.where((kind == 2) | (kind >= 4), 0.8 + 0.19 * torch.rand(rows, device="cuda", generator=g),
                            torch.ones_like(t))
            q = torch.where((kind == 3) | (kind == 5), torch.full_like(t, 0.05), torch.zeros_like(t))
        s["t"], s["top_k"], s["top_p"], s["min_p"] = t.float(), k.int(), p.float(), q.float()
        s["ids"] = torch.empty(rows, device="cuda", dtype=torch.int32)
    return s


# ------------------------------------------------------------------ plain forms
def _unpack_w4(q, in_f):
    blocks = q.shape[1] // 64
    q = q.view(-1, blocks, 4, 4, 4)                       # [o, block, c, i, b]
    codes = torch.stack((q & 15, q >> 4), -1)             # [o, block, c, i, b, nibble]
    return codes.permute(0, 1, 3, 2, 4, 5).reshape(-1, blocks * 128)[:, :in_f]


def _linear_w4(s):
    c = s["case"]
    codes = _unpack_w4(s["q"], c["in_f"]).float()
    spread = lambda t: t.float().T.repeat_interleave(c["group"], 1)[:, :c["in_f"]]  # noqa: E731
    w = (codes - (spread(s["zero"]) if c["zero"] else 8.0)) * spread(s["scale"])
    return (s["x"].float() @ w.T).to(DT[c["y"]])


def _norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rope(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _requantise(codes, old, new, f8):
    """codes at scale `old` rounded at scale `new` (powers of two times the old one)."""
    return (codes.float() * (old / new)).to(F8[f8])


def _append(x, pos, codes, scale, case):
    """Rows x [B, heads, hd] into row pos[b] of sequence b's cache (codes and scale change in place)."""
    f8, block = case["f8"], case["block"]
    b = torch.arange(len(pos), device=pos.device)
    blk, r = pos // block, pos % block
    need = torch.exp2(_scale_exp(x.abs().amax(-1).double(), f8).float())          # [B, heads]
    old = scale[b, blk]
    new = torch.where((r == 0)[:, None], need, torch.maximum(old, need))
    at = (blk * block)[:, None] + torch.arange(block, device=pos.device)          # [B, block]
    earlier = at < pos[:, None]
    at = torch.where(earlier, at, pos[:, None])
    raw = codes.view(torch.uint8)
    rows = raw[b[:, None], at].view(F8[f8])
    again = _requantise(rows, old[:, None, :, None], new[:, None, :, None], f8)
    put = torch.where(earlier[..., None, None], again.view(torch.uint8),
                      (x / new[..., None]).to(F8[f8]).view(torch.uint8)[:, None])
    raw[b[:, None], at] = put
    scale[b, blk] = new


def _kv8_write(s):
    c = s["case"]
    n, heads, hd, block, start = c["count"], c["heads"], c["head_dim"], c["block"], c["start"]
    k = _norm(s["k"].float().reshape(n, heads, hd), s["kw"])
    v = _norm(s["v"].float().reshape(n, heads, hd), s["vw"])
    if c["rope"]:
        k = _rope(k, s["cos"][start:start + n, None], s["sin"][start:start + n, None])
    first, last = start // block, (start + n - 1) // block
    for x, codes, scale in ((k, s["kc"], s["ks"]), (v, s["vc"], s["vs"])):
        pad = torch.zeros((last - first + 1) * block, heads, hd, device=x.device)
        pad[start - first * block:start - first * block + n] = x
        pad = pad.view(-1, block, heads, hd)
        need = torch.exp2(_scale_exp(pad.abs().amax((1, 3)).double(), c["f8"]).float())
        old = scale[0, first].clone()
        if start % block:
            need[0] = torch.maximum(need[0], old)
            codes[0, first * block:start] = _requantise(codes[0, first * block:start], old[:, None],
                                                        need[0][:, None], c["f8"])
        scale[0, first:last + 1] = need
        codes[0, start:start + n] = (pad / need[:, None, :, None]).to(F8[c["f8"]]).view(
            -1, heads, hd)[start - first * block:start - first * block + n]
    return s["kc"], s["ks"], s["vc"], s["vs"]


def _kv8_decode(s):
    c = s["case"]
    B, H, heads, hd = c["batch"], c["q_heads"], c["heads"], c["head_dim"]
    pos = s["pos"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rope(_norm(s["q"].float().reshape(B, H, hd), s["qw"]), cos, sin)
    k = _rope(_norm(s["k"].float().reshape(B, heads, hd), s["kw"]), cos, sin)
    _append(k, pos, s["kc"], s["ks"], c)
    _append(s["v"].float().reshape(B, heads, hd), pos, s["vc"], s["vs"], c)
    rows = int(c["high"]) + 1
    spread = lambda t: t.repeat_interleave(c["block"], 1)[:, :rows, :, None]  # noqa: E731
    K = s["kc"][:, :rows].float() * spread(s["ks"])
    score = torch.einsum("bgih,btgh->bgit", q.view(B, heads, H // heads, hd), K) * hd ** -0.5
    del K
    t = torch.arange(rows, device=pos.device)
    seen = t <= pos[:, None]
    if c["window"]:
        seen &= t > pos[:, None] - c["window"]
    score = score.masked_fill(~seen[:, None, None], -torch.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    V = s["vc"][:, :rows].float() * spread(s["vs"])
    o = torch.einsum("bgit,btgh->bgih", p, V).reshape(B, H * hd).to(DT[c["o"]])
    return o, s["kc"], s["ks"], s["vc"], s["vs"]


def _sample(s):
    l = s["logits"].double()
    rows, vocab = l.shape
    t = s["t"].double()[:, None]
    top = l.amax(1, keepdim=True)
    w = torch.where(t > 0, torch.exp((l - top) / torch.where(t > 0, t, 1.0)), (l == top).double())
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=l.device)
    k = s["top_k"].long()[:, None]
    keep = torch.where(t > 0, (k <= 0) | (rank < k), rank < 1)
    ws = ws * keep
    before = ws.cumsum(1) - ws
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (before < p * ws.sum(1, keepdim=True)) | (rank < 1)
    keep &= ws >= s["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, ws * keep)
    run_ = kept.cumsum(1)
    target = s["u"].double()[:, None] * run_[:, -1:]
    return ((run_ > target) & (kept > 0)).int().argmax(1).int()


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"linear_w4": _linear_w4, "kv8_write": _kv8_write, "kv8_decode": _kv8_decode,
                "sample": _sample}[op](s)
    import eyebrowse_b200 as eb
    c = s["case"]
    if op == "linear_w4":
        if "ws" not in s:
            n = eb.linear_w4_workspace_bytes(c["m"], c["in_f"], c["out_f"])
            s["w"] = eb.make_w4(s["q"], s["scale"], s["zero"], c["in_f"], c["out_f"], c["group"])
            s["ws"] = eb.alloc_workspace(n) if n else None
        eb.linear_w4(s["w"], s["x"], s["y"], c["m"], s["ws"])
        return s["y"]
    if op == "sample":
        if "params" not in s:
            n = eb.sample_workspace_bytes(c["rows"], c["vocab"])
            s["params"] = eb.make_sample_params(s["t"], s["top_k"], s["top_p"], s["min_p"])
            s["ws"] = eb.alloc_workspace(n) if n else None
        eb.sample(s["logits"], s["params"], s["u"], s["ids"], s["ws"])
        return s["ids"]
    if "desc" not in s:
        x, f8 = eb.torch_dtype_code(DT[c["x"]]), {"e4m3": eb.EB_E4M3, "e5m2": eb.EB_E5M2}[c["f8"]]
        s["kv8"] = eb.make_kv8(s["kc"], s["vc"], s["ks"], s["vs"], c["block"])
        if op == "kv8_write":
            s["desc"] = eb.make_desc(c["heads"], c["heads"], c["head_dim"], s["kc"].shape[1], dtype_qkv=x,
                                     dtype_cache=f8, eps=EPS, kv_stride=s["k"].stride(0))
            s["layer"] = eb.make_layer(None, s["kw"], s["vw"], s["cos"], s["sin"])
        else:
            s["desc"] = eb.make_desc(c["q_heads"], c["heads"], c["head_dim"], c["max_seq"], dtype_qkv=x,
                                     dtype_cache=f8, dtype_out=eb.torch_dtype_code(DT[c["o"]]), eps=EPS,
                                     q_stride=s["q"].stride(0), kv_stride=s["k"].stride(0),
                                     window=c["window"])
            s["layer"] = eb.make_layer(s["qw"], s["kw"], None, s["cos"], s["sin"])
            n = eb.attention_decode_kv8_workspace_bytes(s["desc"], c["batch"], c["high"])
            s["ws"] = eb.alloc_workspace(n) if n else None
    if op == "kv8_write":
        eb.kv8_write(s["desc"], s["layer"], s["kv8"], c["start"], c["count"], s["k"], s["v"])
        return s["kc"], s["ks"], s["vc"], s["vs"]
    eb.attention_decode_kv8(s["desc"], s["layer"], s["kv8"], c["batch"], s["pos"], c["high"], s["q"],
                            s["k"], s["v"], s["o"], s["ws"])
    return s["o"], s["kc"], s["ks"], s["vc"], s["vs"]


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "linear_w4":
        m, n, k = case["m"], case["out_f"], case["in_f"]
        groups = -(-k // case["group"])
        return dict(bytes=n * k / 2 + n * groups * (3 if case["zero"] else 2) + m * k * size[case["x"]]
                    + m * n * size[case["y"]], flops=2.0 * m * n * k)
    if case["op"] == "kv8_write":
        n = case["count"] * case["heads"] * case["head_dim"]
        return dict(bytes=2 * n * (size[case["x"]] + 1), flops=12.0 * n)
    if case["op"] == "kv8_decode":
        rows = sum(min(p + 1, case["window"] or p + 1) for p in _positions(case))
        e = case["heads"] * case["head_dim"]
        return dict(bytes=2.0 * rows * e + 8.0 * rows * case["heads"] / case["block"]
                    + case["batch"] * ((case["q_heads"] * case["head_dim"] + 2 * e) * size[case["x"]]
                                       + case["q_heads"] * case["head_dim"] * size[case["o"]]),
                    flops=4.0 * rows * case["q_heads"] * case["head_dim"])
    return dict(bytes=case["rows"] * (case["vocab"] * size[case["x"]] + 24.0),
                flops=4.0 * case["rows"] * case["vocab"])


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear_w4":
        return _exact_linear(s, case)
    if case["op"] == "sample":
        return _exact_sample(s, case)
    n = 1 if case["op"] == "kv8_write" else case["batch"]
    pos = [None] if case["op"] == "kv8_write" else _positions(case)
    heads, hd = case["heads"], case["head_dim"]
    if case["op"] == "kv8_write":
        k = s["k"].double().reshape(case["count"], heads, hd)
        v = s["v"].double().reshape(case["count"], heads, hd)
        at = case["start"] + torch.arange(case["count"], device="cuda")
        _exact_rows(s, case, 0, case["start"], _exact_turn(_exact_unit(k, s["kw"]), s["cos"], s["sin"], at),
                    _exact_unit(v, s["vw"]))
        return s["kc"], s["ks"], s["vc"], s["vs"]
    out = torch.empty(n, case["q_heads"] * hd, device="cuda", dtype=torch.float64)
    group = case["q_heads"] // heads
    for b in range(n):
        at = torch.tensor([pos[b]], device="cuda")
        q = s["q"][b].double().reshape(1, case["q_heads"], hd)
        k = s["k"][b].double().reshape(1, heads, hd)
        q = _exact_turn(_exact_unit(q, s["qw"]), s["cos"], s["sin"], at)[0]
        k = _exact_turn(_exact_unit(k, s["kw"]), s["cos"], s["sin"], at)
        _exact_rows(s, case, b, pos[b], k, s["v"][b].double().reshape(1, heads, hd))
        lo = max(0, pos[b] + 1 - case["window"]) if case["window"] else 0
        blocks = torch.arange(lo, pos[b] + 1, device="cuda") // case["block"]
        for h in range(heads):
            K = s["kc"][b, lo:pos[b] + 1, h].double() * s["ks"][b, blocks, h].double()[:, None]
            V = s["vc"][b, lo:pos[b] + 1, h].double() * s["vs"][b, blocks, h].double()[:, None]
            z = (q[h * group:(h + 1) * group] @ K.T) / math.sqrt(hd)
            out[b].view(-1, hd)[h * group:(h + 1) * group] = torch.softmax(z, 1) @ V
    return out, s["kc"], s["ks"], s["vc"], s["vs"]


def _exact_linear(s, case):
    out_f, in_f = case["out_f"], case["in_f"]
    raw = s["q"].view(out_f, -1, 64)
    k = torch.arange(in_f, device="cuda")
    inner = k % 128
    byte = (inner % 32) // 8 * 16 + inner // 32 * 4 + inner % 8 // 2
    y = torch.empty(case["m"], out_f, device="cuda", dtype=torch.float64)
    for at in range(0, out_f, 4096):
        rows = slice(at, min(out_f, at + 4096))
        code = (raw[rows][:, k // 128, byte] >> (4 * (inner % 2)).to(torch.uint8)) & 15
        g = k // case["group"]
        zero = s["zero"][g][:, rows].T.double() if case["zero"] else 8.0
        y[:, rows] = s["x"].double() @ ((code.double() - zero) * s["scale"][g][:, rows].T.double()).T
    return y


def _exact_unit(x, w):
    return x if w is None else x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()


def _exact_turn(x, cos, sin, at):
    if cos is None:
        return x
    c, n = cos[at].double()[:, None], sin[at].double()[:, None]
    h = x.shape[-1] // 2
    y = torch.empty_like(x)
    y[..., :h] = x[..., :h] * c - x[..., h:] * n
    y[..., h:] = x[..., h:] * c + x[..., :h] * n
    return y


def _exact_rows(s, case, b, start, *kv):
    """Rows start.. of sequence b's K and V caches, block by block."""
    block, lim = case["block"], 1.75 * 2.0 ** TOP_EXP[case["f8"]]
    for x, codes, scale in zip(kv, (s["kc"], s["vc"]), (s["ks"], s["vs"])):
        n = x.shape[0]
        row = start
        while row < start + n:
            j = row // block
            end = min((j + 1) * block, start + n)
            part = x[row - start:end - start]
            e = torch.ceil(torch.log2(part.abs().amax((0, 2)) / lim).clamp_min(MIN_EXP))
            new = torch.exp2(e).float()
            if row % block:
                new = torch.maximum(new, scale[b, j])
                old = codes[b, j * block:row].double() * scale[b, j].double()[:, None]
                codes[b, j * block:row] = _round8(old / new.double()[:, None], case["f8"])
            scale[b, j] = new
            codes[b, row:end] = _round8(part / new.double()[:, None], case["f8"])
            row = end


def _round8(x, f8):
    """f64 to the nearest value of the 8-bit type, ties to even, by its definition."""
    bits, low = (3, -6) if f8 == "e4m3" else (2, -14)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** low)))
    unit = torch.exp2(e - bits)
    return (torch.round(x / unit) * unit).float().to(F8[f8])  # a value of the type: this cast is exact


def _exact_sample(s, case):
    l = s["logits"].double().cpu().numpy()
    ids = np.empty(case["rows"], np.int32)
    for r in range(case["rows"]):
        t, k = float(s["t"][r]), int(s["top_k"][r])
        p, q, u = float(s["top_p"][r]), float(s["min_p"][r]), float(s["u"][r])
        if t <= 0:
            ids[r] = int(np.argmax(l[r]))
            continue
        order = np.argsort(-l[r], kind="stable")
        order = order[:k] if k > 0 else order
        w = np.exp((l[r][order] - l[r][order[0]]) / t)
        if p < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))]
        order = order[w[:len(order)] >= q]
        order = np.sort(order)
        run_ = np.cumsum(np.exp((l[r][order] - l[r].max()) / t))
        ids[r] = order[min(len(order) - 1, int(np.searchsorted(run_, u * run_[-1], side="right")))]
    return torch.from_numpy(ids)
