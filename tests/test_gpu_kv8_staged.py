"""eb_kv8_write's kernel for head dims without one of their own, and for unaligned rows, at the sizes
of shared memory where a launch needs leave for more than 48 KB: 49152 bytes of rows (the kernel has
static shared memory beside them) and above. In a process of its own, as the leave is given once."""
import os
import subprocess
import sys

import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def write_exact(eb, hd, block, count, shift=0):
    """One write of rows as they are into a fresh cache; codes and scales are the definition's."""
    import torch
    heads, max_seq = 2, 2 * block + 40
    rng = np.random.default_rng(hd)
    rows = [rng.standard_normal((count, heads, hd)).astype(np.float32) for _ in "kv"]
    codes = [torch.zeros(max_seq, heads, hd, dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.zeros(-(-max_seq // block), heads, device="cuda") for _ in "kv"]
    dev = []
    for r in rows:
        flat = torch.zeros(r.size + shift, device="cuda")
        flat[shift:] = torch.from_numpy(r.ravel()).cuda()
        dev.append(flat[shift:].view(count, heads, hd))
    desc = eb.make_desc(heads, heads, hd, max_seq, dtype_cache=eb.EB_E4M3)
    eb.kv8_write(desc, None, eb.make_kv8(*codes, *scales, block), 0, count, *dev)
    torch.cuda.synchronize()
    for c, s, r in zip(codes, scales, rows):
        want, ws = np.zeros((max_seq, heads, hd), np.uint8), np.zeros((-(-max_seq // block), heads))
        qo.kv8_write(want, ws, 0, r.astype(np.float64), block, "e4m3")
        assert np.array_equal(c.cpu().numpy(), want) and np.array_equal(s.double().cpu().numpy(), ws), (hd, block)


@pytest.mark.parametrize("hd,block,count,shift", [(96, 128, 128, 0), (192, 64, 64, 0), (192, 64, 100, 0),
                                                  (128, 128, 96, 1), (256, 128, 48, 1)])
def test_write_at_48_kb_in_a_new_process(eb, hd, block, count, shift):
    code = (f"import sys; sys.path[:0] = [{HERE!r}, {os.path.dirname(HERE)!r}]\n"
            "import eyebrowse_b200 as eb, test_gpu_kv8_staged as t\n"
            f"t.write_exact(eb, {hd}, {block}, {count}, {shift})\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("hd,block,count,shift", [(96, 128, 128, 0), (160, 128, 128, 0), (254, 128, 200, 0),
                                                  (256, 128, 128, 1), (192, 64, 64, 3)])
def test_write_past_48_kb(eb, hd, block, count, shift):
    write_exact(eb, hd, block, count, shift)
