"""The quantised operators together, as a model uses them: a decoder with 4-bit projections, an 8-bit
cache and sampled tokens (eyebrowse_b200.decoder), against the same decoder in f64 numpy over the
dequantised weights, with the cache rounded as the definition says.

Tolerance of single-token steps: both sides round values to 8 bits that are alike to f32's accuracy, in
front of which stand at most four products of 320 terms (sqrt(320) 2^-24 of a row's size each) and their
norms: 2^-16 of a row's largest value. A value that near to the middle of two codes may get either. Such
codes are not rare (2 * 2^-20, the usual error, over the step of 2^-4 to 2^-3 is one value in 30,000 to
60,000, and forty tokens store 41,000), and one is felt: a step of 2^-3 of one of hd values of K moves its
row's score by 2^-3 |q k| / sqrt(hd), up to 0.1 where the two are of size 3, so that a row of weight w moves
the output by up to 0.1 w. So the f64 decoder checks that the value lies in the middle to 2^-16 and takes
the code that was stored; all else is f32's error, far below 1e-3.

Tolerance after a prompt of several rows: eb_attention_prefill rounds its softmax weights to f16, so what
the first layer hands on is off by e = 2^-11 of its size. The next layer's cached values then cross a
rounding border with probability e / (2 h), h the type's half step (2^-4, 2^-3), and move by 2 h where
they do: an rms error of sqrt(e / (2 h)) * 2 h = sqrt(2 e h) of the cached rows (2^-7, 2^-6.5), which bounds
what it does to the logits."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu


def _config(arch, hd):
    return dict(model_type=arch, num_attention_heads=4, num_key_value_heads=2, head_dim=hd, hidden_size=192,
                num_hidden_layers=2, intermediate_size=320, vocab_size=777, rms_norm_eps=1e-6, rope_theta=1e4)


def _weights(c, seed):
    rng = np.random.default_rng(seed)
    H, Hkv, hd, D, I = (c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], c["hidden_size"],
                        c["intermediate_size"])
    lin = lambda o, i: (0.08 * rng.standard_normal((o, i))).astype(np.float16).astype(np.float32)  # noqa: E731
    norm = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    w = {"model.embed_tokens.weight": lin(c["vocab_size"], D), "model.norm.weight": norm(D)}
    for i in range(c["num_hidden_layers"]):
        p = f"model.layers.{i}."
        w |= {p + "input_layernorm.weight": norm(D), p + "post_attention_layernorm.weight": norm(D),
              p + "self_attn.q_norm.weight": norm(hd), p + "self_attn.k_norm.weight": norm(hd),
              p + "self_attn.q_proj.weight": lin(H * hd, D), p + "self_attn.k_proj.weight": lin(Hkv * hd, D),
              p + "self_attn.v_proj.weight": lin(Hkv * hd, D), p + "self_attn.o_proj.weight": lin(D, H * hd),
              p + "mlp.gate_proj.weight": lin(I, D), p + "mlp.up_proj.weight": lin(I, D),
              p + "mlp.down_proj.weight": lin(D, I)}
    return w


class _Reference:
    def __init__(self, eb, w, c, max_seq, group, zero_point, f8, block):
        self.w, self.c, self.f8, self.block = w, c, f8, block
        H, Hkv, hd = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"]
        self.dims = H, Hkv, hd
        self.cos, self.sin = (t.reshape(max_seq, hd // 2).astype(np.float64)
                              for t in eb.rope_tables(max_seq, hd, c["rope_theta"]))
        self.lin = []
        for i in range(c["num_hidden_layers"]):
            p = f"model.layers.{i}."
            cat = dict(qkv=("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), o=("self_attn.o_proj",),
                       gu=("mlp.gate_proj", "mlp.up_proj"), down=("mlp.down_proj",))
            d = {}
            for n, names in cat.items():
                m = np.concatenate([w[p + x + ".weight"] for x in names])
                if group:
                    q, s, z = eb.w4_quantize(m, group, zero_point)
                    m = qo.w4_weights(qo.w4_unpack(q, m.shape[1]), s, z, group)
                d[n] = m.astype(np.float64)
            d["cache"] = {n: [np.zeros((max_seq, Hkv, hd), np.uint8), np.zeros((-(-max_seq // block), Hkv))]
                          for n in "kv"}
            self.lin.append(d)

    def follow(self, layer, d, pos, new):
        """Stored codes of row `pos` other than this decoder's: checked and taken over."""
        for n, x in new.items():
            codes, scale = d["cache"][n][0][pos], d["cache"][n][1][pos // self.block]
            got = layer[n + "c"].cpu().numpy().reshape(d["cache"][n][0].shape)[pos]
            middle = (qo.f8_decode(codes, self.f8) + qo.f8_decode(got, self.f8)) / 2 * scale[:, None]
            near = np.abs(x - middle) <= 2.0 ** -16 * np.abs(x).max(-1, keepdims=True)
            assert near[got != codes].all(), (n, pos)
            codes[:] = got

    def logits(self, ids, pos, model=None):
        w, c = self.w, self.c
        H, Hkv, hd = self.dims
        norm = lambda x, n: qo.row_norm(x, w[n].astype(np.float64), c["rms_norm_eps"])  # noqa: E731
        x = w["model.embed_tokens.weight"][ids].astype(np.float64)
        rows = len(ids)
        cos, sin = self.cos[pos:pos + rows, None], self.sin[pos:pos + rows, None]
        for i, d in enumerate(self.lin):
            p = f"model.layers.{i}."
            y = norm(x, p + "input_layernorm.weight") @ d["qkv"].T
            q, k, v = (t.reshape(rows, -1, hd) for t in np.split(y, [H * hd, (H + Hkv) * hd], 1))
            if c["model_type"] == "qwen3":
                q, k = norm(q, p + "self_attn.q_norm.weight"), norm(k, p + "self_attn.k_norm.weight")
            q, k = qo.row_rope(q, cos, sin), qo.row_rope(k, cos, sin)
            for n, t in (("k", k), ("v", v)):
                qo.kv8_write(d["cache"][n][0], d["cache"][n][1], pos, t, self.block, self.f8)
            if model is not None:
                self.follow(model.L[i], d, pos, {"k": k[0], "v": v[0]})
            out = np.empty((rows, H * hd))
            for r in range(rows):
                if rows > 1:  # a prompt attends its own rows as they are
                    K, V = k[:r + 1], v[:r + 1]
                else:
                    at = np.arange(pos + 1)
                    K, V = (qo.f8_decode(d["cache"][n][0][at], self.f8) * d["cache"][n][1][at // self.block][..., None]
                            for n in "kv")
                out[r] = qo.attend(q[r], K, V, hd ** -0.5)[0].ravel()
            x = x + out @ d["o"].T
            y = norm(x, p + "post_attention_layernorm.weight") @ d["gu"].T
            g, u = np.split(y, 2, 1)
            x = x + (g / (1 + np.exp(-g)) * u) @ d["down"].T
        return norm(x[-1:], "model.norm.weight")[0] @ w["model.embed_tokens.weight"].astype(np.float64).T


@pytest.mark.parametrize("arch,hd,group,zero_point,f8,block,prompt", [
    ("qwen3", 128, 128, False, "e4m3", 64, 70), ("mistral", 64, 32, True, "e5m2", 16, 33),
    ("qwen3", 256, 64, True, "e4m3", 32, 1), ("mistral", 48, 64, False, "e4m3", 128, 130)])
def test_quantised_decoder(eb, arch, hd, group, zero_point, f8, block, prompt):
    from eyebrowse_b200.decoder import DecoderModel
    c = _config(arch, hd)
    w = _weights(c, hd)
    max_seq = 160
    model = DecoderModel(w, c, max_seq, w4_group=group, w4_zero_point=zero_point, cache=f8, kv_block=block)
    ref = _Reference(eb, w, c, max_seq, group, zero_point, f8, block)
    rng = np.random.default_rng(1)
    ids, pos = rng.integers(0, c["vocab_size"], prompt).tolist(), 0
    tol = 1e-3 if prompt == 1 else (2 * 2.0 ** -11 * {"e4m3": 2.0 ** -4, "e5m2": 2.0 ** -3}[f8]) ** 0.5
    for step in range(12):
        got = model.logits(ids, pos).double().cpu().numpy()
        want = ref.logits(ids, pos, model if prompt == 1 else None)
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= tol, (step, rel)
        pos += len(ids)
        ids = [int(np.argmax(want))]
    assert eb.device_error() == 0


@pytest.mark.parametrize("f8,block,hd", [("e4m3", 16, 128), ("e5m2", 64, 64)])
def test_token_by_token(eb, f8, block, hd):
    """Forty tokens one at a time: every row is appended and read in 8 bits, f32 throughout."""
    from eyebrowse_b200.decoder import DecoderModel
    c = _config("qwen3", hd)
    w = _weights(c, 7)
    model = DecoderModel(w, c, 64, w4_group=64, cache=f8, kv_block=block)
    ref = _Reference(eb, w, c, 64, 64, False, f8, block)
    for pos, t in enumerate(np.random.default_rng(2).integers(0, c["vocab_size"], 40).tolist()):
        got, want = model.logits([t], pos).double().cpu().numpy(), ref.logits([t], pos, model)
        assert np.linalg.norm(got - want) <= 1e-3 * np.linalg.norm(want), pos
    assert eb.device_error() == 0


def test_prompt_rows_reach_the_cache(eb):
    """After a prompt the last layer's 8-bit rows are its f32 rows, rounded by the definition."""
    from eyebrowse_b200.decoder import DecoderModel
    c = _config("qwen3", 128)
    model = DecoderModel(_weights(c, 9), c, 128, cache="e4m3", kv_block=32)
    model.logits(list(range(77)), 0)
    ly = model.L[-1]
    for n, codes, rows, scale in zip("kv", (ly["kc"], ly["vc"]), model.shared[128], ly["kv8"]._keepalive[2:]):
        want, s = np.zeros((128, 2, 128), np.uint8), np.zeros((4, 2))
        qo.kv8_write(want, s, 0, rows[:77].double().cpu().numpy(), 32, "e4m3")
        assert np.array_equal(codes.cpu().numpy()[:77], want[:77]) and np.array_equal(scale.double().cpu().numpy()[:3], s[:3]), n


def test_sampled_generation(eb):
    """generate with uniforms: each id is the definition's draw from that step's logits, and the same
    uniforms give the same ids; uniforms of a greedy temperature give the greedy ids."""
    from eyebrowse_b200.decoder import DecoderModel
    c = _config("qwen3", 128)
    model = DecoderModel(_weights(c, 3), c, 64, w4_group=64, cache="e4m3")
    prompt = [5, 700, 3, 42]
    kw = dict(temperature=0.9, top_k=40, top_p=0.9, min_p=0.01)
    u = np.random.default_rng(0).random(20).astype(np.float32)
    ids = model.generate(prompt, 20, uniforms=u, **kw)
    assert ids == model.generate(prompt, 20, uniforms=u, **kw)
    model.reset()
    pos, last = 0, prompt
    for i, t in enumerate(ids):
        logits = model.logits(last, pos).double().cpu().numpy()
        assert t == qo.sample(logits, u[i], **kw), i
        pos, last = pos + len(last), [t]
    assert model.generate(prompt, 20) == model.generate(prompt, 20, uniforms=u, temperature=0.0)
    with pytest.raises(ValueError):
        model.generate(prompt, 20, uniforms=u[:19])


def test_cache_names_are_checked(eb):
    from eyebrowse_b200.decoder import DecoderModel
    c = _config("qwen3", 128)
    with pytest.raises(ValueError):
        DecoderModel(_weights(c, 3), c, 64, cache="int8")
    with pytest.raises(eb.EbError):
        DecoderModel(_weights(c, 3), c, 64, w4_group=48)
