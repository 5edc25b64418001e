"""Teacher entries outside the vocabulary make their row NaN however small their weight; with a logit of -inf they count as none (plain forms)."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL


@pytest.mark.parametrize("logit,nan", [(0.0, True), (-40.0, True), (-1e4, True), (-1e300, True), (-math.inf, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_entries_outside_the_vocabulary(dtype, logit, nan):
    if dtype == torch.float32 and logit == -1e300:
        logit = -3e38
    g = torch.Generator().manual_seed(0)
    z = torch.randn(3, 7, generator=g, dtype=dtype).requires_grad_()
    w = torch.eye(7, dtype=dtype)
    idx, t = torch.tensor([[0, 1], [2, 7], [3, 4]]), torch.tensor([[0.0, 1.0], [0.5, logit], [1.0, 1.0]], dtype=dtype)
    for loss in (VL.topk_distillation(z, idx, t, 0.5), VL.linear_topk_distillation(z, w, idx, t, None, 0.5)):
        assert loss.isnan().tolist() == [False, nan, False]
        dz, = torch.autograd.grad(loss.sum(), z)
        assert dz.isnan().all(1).tolist() == [False, nan, False] and dz.isnan().any(1).tolist() == [False, nan, False]
