"""Teacher entries outside the vocabulary make their row NaN however small their weight, in both distillation losses alike; with a logit of -inf
they count as none."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("logit,nan", [(0.0, True), (-40.0, True), (-1e4, True), (-3e38, True), (-math.inf, False)])
def test_entries_outside_the_vocabulary(dtype, temperature, logit, nan):
    n, d, v, k = 9, 64, 300, 5
    g = torch.Generator(device=DEV).manual_seed(0)
    h, w = torch.randn(n, d, generator=g, device=DEV).to(dtype), torch.randn(v, d, generator=g, device=DEV).to(dtype)
    z = (h.float() @ w.float().t()).to(dtype).requires_grad_()
    h.requires_grad_()
    idx, t = torch.randint(0, v, (n, k), generator=g, device=DEV), torch.randn(n, k, generator=g, device=DEV)
    idx[4, 2], t[4, 2] = v, logit
    idx[7, 0], t[7, 0] = 2 ** 40, logit
    want = torch.zeros(n, dtype=torch.bool, device=DEV)
    want[[4, 7]] = nan
    for plain in (False, True):
        for loss, x in ((VL.topk_distillation(z, idx, t, temperature, plain=plain), z), (VL.linear_topk_distillation(h, w, idx, t, None, temperature, plain=plain), h)):
            assert torch.equal(loss.isnan(), want)
            grad, = torch.autograd.grad(loss.sum(), x)
            assert torch.equal(grad.isnan().any(1), want) and torch.equal(grad.isnan().all(1), want)
