"""Rows that are sure of their word beside rows with far larger scores: what the many other words keep together still counts, although each of them
lies far below the other rows' scores.

The scores are bias-free products of one hidden value s and one weight per word, 1 for the row's word and 0 for the others: a row has the scores s
and 0, and its loss is log(1 + (V - 1) exp(-s)), 1.7e-4 for s = 19 and V = 30000. Tolerances: 4e-6 for a loss and, times the weight of 1, for the
hidden states' gradient, which is the difference of two fp32 numbers around 1; the bf16 gradient is rounded twice on top (2 x 2^-8 of itself)."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,d,v", [(3, 64, 30000), (40, 64, 30000), (300, 64, 5000), (500, 512, 30000), (700, 520, 30000)])
@pytest.mark.parametrize("high", [30.0, 62.0, 75.0, 88.0, 120.0])
@pytest.mark.parametrize("distil", [False, True])
def test_confident_rows_beside_rows_of_larger_scores(n, d, v, dtype, high, layout, distil):
    word = v // 3
    h, w = torch.zeros(n, d, device=DEV), torch.zeros(v, d, device=DEV)
    h[:, 5] = torch.where(torch.arange(n, device=DEV) % 2 == 0, 19.0, high)
    w[word, 5] = 1.0
    h, w = h.to(dtype).requires_grad_(), w.to(dtype)
    w = w if layout == "vd" else w.t().contiguous().t()
    if distil:
        loss = VL.linear_topk_distillation(h, w, torch.full((n, 1), word, device=DEV), torch.zeros(n, 1, device=DEV))
    else:
        loss = VL.linear_cross_entropy(h, w, torch.full((n,), word, device=DEV))
    dh, = torch.autograd.grad(loss.sum(), h)
    s = h.detach()[:, 5].double()
    rest = (v - 1) * torch.exp(-s)
    assert float((loss.detach().double() - torch.log1p(rest)).abs().max()) <= 4e-6
    want = -rest / (1 + rest)
    err = (dh[:, 5].double() - want).abs()
    assert bool((err <= 4e-6 + (0.0 if dtype == torch.float32 else 2 * 2.0 ** -8) * want.abs()).all())
    assert math.isfinite(float(loss.detach().sum()))
