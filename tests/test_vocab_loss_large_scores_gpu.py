"""Rows whose scores are so large that a rounding of the score is many units: the largest score still has probability 1 at most, losses and
gradients are those of the definition in 64 bits.

Tolerances: a score's error is relative to its size, so a loss is held to 4e-6 of the row's largest |score| (sums of up to 520 fp32 products). The
words' scores lie 2^-8 and more of their size apart, the softmax is 0 or 1 in 64 bits and here, and the gradients carry their own rounding and that
of the scores' gradient alone: two roundings of half a step, 4e-6 in fp32."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"
LIMIT = {torch.bfloat16: 2 * 2.0 ** -8, torch.float16: 2 * 2.0 ** -11, torch.float32: 4e-6}


def _grads(fn, leaves):
    leaves = [x.detach().requires_grad_() for x in leaves]
    loss = fn(*leaves)
    return loss.detach(), torch.autograd.grad(loss.sum(), leaves)


def _close(got, want, limit, what):
    assert torch.isfinite(got).all(), what
    assert float((got.double() - want).norm()) <= limit * float(want.norm()), what


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", [(1, 64, 20000), (40, 64, 900), (500, 512, 4000), (700, 520, 30000)])
@pytest.mark.parametrize("dtype,factor", [(torch.float32, 1e10), (torch.float32, 1e25), (torch.bfloat16, 1e10), (torch.bfloat16, 1e25)])
@pytest.mark.parametrize("loss", ["cross entropy", "smoothed", "distillation"])
def test_linear_losses_of_rows_with_large_scores(n, d, v, dtype, factor, loss, layout):
    g = torch.Generator(device=DEV).manual_seed(n + v)
    # the scores are +-factor times the words' first weights, up to the rest's part
    h = torch.zeros(n, d, device=DEV)
    h[:, 0] = factor * (1 - 2 * (torch.arange(n, device=DEV) % 2))
    h[:, 1:] = torch.randn(n, d - 1, generator=g, device=DEV)
    w = torch.randn(v, d, generator=g, device=DEV) * 0.1
    w[:, 0] = 0.5
    w[v // 2, 0], w[v // 3, 0] = 1.0, 0.25                                # the largest of even rows, of odd rows
    h, w = h.to(dtype), w.to(dtype)
    w = w if layout == "vd" else w.t().contiguous().t()
    y = torch.randint(0, v, (n,), generator=g, device=DEV)
    y[::3] = v // 2
    idx, t = torch.randint(0, v, (n, 5), generator=g, device=DEV), torch.randn(n, 5, generator=g, device=DEV)

    def fn(plain):
        if loss == "distillation":
            return lambda h, w: VL.linear_topk_distillation(h, w, idx, t, temperature=1.7, plain=plain)
        return lambda h, w: VL.linear_cross_entropy(h, w, y, label_smoothing=0.1 if loss == "smoothed" else 0.0, plain=plain)
    got, (dh, dw) = _grads(fn(False), [h, w])
    want, (edh, edw) = _grads(fn(True), [h.double(), w.double()])
    size = (h[:, 0].double().abs() * (1.7 if loss == "distillation" else 1.0)).clamp(min=1.0)
    assert torch.isfinite(got).all() and float(((got.double() - want).abs() / size).max()) <= 4e-6
    _close(dh, edh, LIMIT[dtype], "hidden")
    _close(dw, edw, LIMIT[dtype], "weights")


@pytest.mark.parametrize("v", [7, 1000, 65537])
@pytest.mark.parametrize("dtype,factor", [(torch.float32, 1e10), (torch.float32, 1e30), (torch.bfloat16, 1e10), (torch.bfloat16, 1e30), (torch.float16, 3e4)])
def test_distillation_on_large_logits(v, dtype, factor):
    n = 33
    g = torch.Generator(device=DEV).manual_seed(v)
    z = torch.rand(n, v, generator=g, device=DEV) * 0.5
    z[torch.arange(n), torch.arange(n) % v] = 1.0
    z = (z * factor * (1 - 1.75 * (torch.arange(n, device=DEV) % 2))[:, None]).to(dtype)
    z[1::2] = torch.where(torch.arange(v, device=DEV) == 3, z[1::2] * 0, z[1::2].abs() * -1 - factor / 100)    # odd rows: one word far above the others
    idx, t = torch.randint(0, v, (n, 5), generator=g, device=DEV), torch.randn(n, 5, generator=g, device=DEV)
    got, (dz,) = _grads(lambda z: VL.topk_distillation(z, idx, t, temperature=1.7), [z])
    want, (edz,) = _grads(lambda z: VL.topk_distillation(z, idx, t, temperature=1.7, plain=True), [z.double()])
    assert torch.isfinite(got).all() and float(((got.double() - want).abs() / (1.7 * factor)).max()) <= 4e-6
    _close(dz, edz, LIMIT[dtype], "logits")
