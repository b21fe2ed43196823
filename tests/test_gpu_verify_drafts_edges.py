"""Verification of drafted tokens where its sums and temperatures can go wrong, against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_decoding import DTYPES
from tests.test_gpu_drafts import check_verify

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 5002, 60001])
def test_small_temperatures(dtype, V):
    """Rows whose largest logit lies below, at and above zero, alone at the top or not, and rows as small as the temperature itself."""
    dt = DTYPES[dtype]
    rng = np.random.RandomState(V)
    base = torch.from_numpy(rng.randn(V)).float() * 2
    twice = base - base.max() - 1
    twice[[1, V - 2]] = -0.5
    for k, temp in enumerate((1e-3, 1e-6, 2e-7, 1.5e-7, 1e-7, 8e-11, 1e-11, 1e-20, 1e-30, 1e-34, 1.2e-36, 1e-36, 1e-37, 1e-40, 1e-44)):
        rows = [torch.log_softmax(base, -1), base - base.max(), base, base.clamp(max=0.0), twice, base - 60, base + 60, base * temp, -base.abs() * (30 * temp),
                torch.where(base > 1, base, torch.full_like(base, -math.inf)), torch.zeros(V)]
        x = torch.stack([torch.stack([r, base, -base.abs()]) for r in rows]).to(dt).cuda()
        B = len(rows)
        best = x[:, 0].float().argmax(1).cpu().numpy()
        drafts = rng.randint(0, V, (B, 3))
        drafts[::2, 1] = best[::2]                         # the largest, which stands, or one that hardly ever does
        check_verify(x, drafts, np.array([[-1, 0, 1]] * B), rng.rand(B, 3).astype(np.float32), [temp] * B)
        check_verify(x, drafts, np.array([[-1, 0, 0]] * B), rng.rand(B, 3).astype(np.float32), [temp] * B)
