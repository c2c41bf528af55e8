"""eb_sample where filters meet ties and odd settings: ids equal the definition's (tests/_quant_oracle.py)."""
import numpy as np
import pytest

import _quant_oracle as qo

pytestmark = pytest.mark.gpu


def _check(eb, logits, u, **kw):
    import torch
    rows = logits.shape[0]
    dt = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    p = eb.make_sample_params(**{n: torch.full((rows,), v, dtype=dt[n], device="cuda") for n, v in kw.items()})
    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    eb.sample(logits, p, torch.tensor(u, dtype=torch.float32, device="cuda"), ids)
    l = logits.double().cpu().numpy()
    assert ids.cpu().tolist() == [qo.sample(l[r], u[r], **kw) for r in range(rows)]
    assert eb.device_error() == 0


@pytest.mark.parametrize("min_p", [0.9999, 1.0, 1.5, 2.0, float("inf")])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=100), dict(top_p=0.8), dict(top_k=50, top_p=0.9), dict(top_k=3000),
                                dict(top_k=2500, top_p=0.9)])
@pytest.mark.parametrize("vocab", [40, 6000])
def test_min_p_past_one_keeps_all_of_the_largest(eb, min_p, kw, vocab):
    """Several tokens share the largest logit: all of them are kept, on every path."""
    import torch
    logits = torch.randn(8, vocab, generator=torch.Generator().manual_seed(1)).cuda()
    logits[:, 3::7] = 6.0
    logits[4:] = 0.25
    _check(eb, logits, (np.arange(8) / 8 + 0.05).astype(np.float32), min_p=min_p, **kw)
