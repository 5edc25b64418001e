"""Training steps of the vocabulary losses whose saved tensors come back as others (recomputation, offload to the host) on the GPU kernels: the
gradients are those of the step without hooks, bit for bit, although the memory of the forward call's tensors holds something else by then."""
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"

# sizes: fp32 cores, 16-bit, fp32 in halves (128 x 128 and 256 x 256 tiles), copied operands (odd width, odd vocabulary in [D, V])
CASES = [(40, 64, 900, torch.float32, "vd"), (300, 128, 5000, torch.bfloat16, "vd"), (600, 520, 30011, torch.bfloat16, "dv"), (500, 512, 4000, torch.float32, "vd"),
         (700, 528, 30000, torch.float32, "dv"), (77, 101, 1003, torch.float16, "dv"), (77, 101, 1003, torch.float32, "vd")]


def _inputs(n, d, v, dtype, layout):
    g = torch.Generator(device=DEV).manual_seed(n + v)
    x = torch.randn(n, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(v, d, generator=g, device=DEV) * (2.5 / math.sqrt(d))).to(dtype)
    if layout == "dv":
        w = w.t().contiguous()
    b = torch.randn(v, generator=g, device=DEV).to(dtype)
    y = torch.randint(0, v, (n,), generator=g, device=DEV)
    y[::4] = -100
    idx, t = torch.randint(0, v, (n, 7), generator=g, device=DEV), torch.randn(n, 7, generator=g, device=DEV)
    return x, w, b, y, idx, t, torch.rand(n, generator=g, device=DEV) + 0.5


def _blocks(layout, y, idx, t):
    """The losses behind something that makes their operands inside the block (so that they are not leaves)."""
    wv = (lambda w: w * 1.0) if layout == "vd" else (lambda w: (w * 1.0).t())
    return [lambda x, w, b: VL.linear_cross_entropy(torch.tanh(x), wv(w), y, b * 1.0, label_smoothing=0.1),
            lambda x, w, b: VL.linear_topk_distillation(torch.tanh(x), wv(w), idx, t, b * 1.0, temperature=1.5),
            lambda x, w, b: VL.topk_distillation(torch.tanh(x), idx % x.shape[1], t * 1.0, temperature=1.5)]


def _overwrite(*like):
    """Takes the memory that freed tensors of these shapes left and fills it with NaN."""
    return [torch.full_like(t, math.nan) for t in like for _ in range(4)]


@pytest.mark.parametrize("n,d,v,dtype,layout", CASES)
@pytest.mark.parametrize("kind", ["recomputed", "offloaded", "cloned"])
def test_saved_tensors_may_come_back_as_others(n, d, v, dtype, layout, kind):
    x, w, b, y, idx, t, dl = _inputs(n, d, v, dtype, layout)
    for block in _blocks(layout, y, idx, t):
        leaves = [a.detach().clone().requires_grad_() for a in (x, w, b)]
        want = torch.autograd.grad(block(*leaves), leaves, dl, allow_unused=True)
        if kind == "recomputed":
            loss = checkpoint(block, *leaves, use_reentrant=False)
        elif kind == "offloaded":
            with torch.autograd.graph.save_on_cpu(pin_memory=False):
                loss = block(*leaves)
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda a: a.detach().clone(), lambda a: a):
                loss = block(*leaves)
        junk = _overwrite(x, w, b)
        got = torch.autograd.grad(loss, leaves, dl, allow_unused=True)
        del junk
        for a, e in zip(got, want):
            assert (a is None and e is None) or torch.equal(a, e)
