"""Verification over rows so long that fp32 sums of them are off by more than next to nothing: 64 bits decide there."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight,aside", [(0.319988, -7e-5), (0.314778, 7e-5)], ids=["accepted", "refused"])
def test_sums_of_many_additions(weight, aside):
    """One logit of four is 0, the others ln(weight): a lane adds the same number again and again, so that its roundings go the same way.  Probabilities
    are off by 2e-4 then; the random numbers lie less than half of that from the border."""
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    vocab, k = 1 << 27, 15
    low = np.float32(np.log(weight))
    target = torch.tensor([0.0, low, low, low], device="cuda").repeat(vocab // 4)[None].expand(k + 1, -1).contiguous()
    p = 4.0 / (vocab * (1.0 + 3.0 * np.exp(np.float64(low))))
    u = torch.full((1, k + 1), p * (1.0 + aside), device="cuda")
    u[0, k] = 0.0
    tokens = (torch.arange(k, device="cuda", dtype=torch.int32) * 4444)[None]
    out = torch.zeros(k + 2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert abs(float(u[0, 0]) / p - 1.0 - aside) < 2e-7
    rt = Runtime()
    for name, t in (("target", target), ("tokens", tokens), ("u", u), ("out", out)):
        rt.bind(name, t.data_ptr(), t.numel(), t.element_size())
    kept = rt.verify("target", None, "tokens", "u", vocab, 1, k, out="out")
    # (refused: the token behind comes from p without the draft's)
    assert kept == [[*tokens[0].tolist(), 0]] if aside < 0 else kept == [[1]]
    rt.close()
