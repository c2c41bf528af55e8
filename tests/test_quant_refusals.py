"""CPU checks: calls of the quantised decode step that the library or its binding refuses before any
device work, because the kernels would read or write elsewhere than the caller means."""


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
