"""Calls of so many rows that the [V, D] table is transposed for the hidden states' gradient, over one and several pieces of the vocabulary, and
calls of as many rows of which too few take part for that. Against the definition in 64 bits, with the tolerances of test_vocab_loss_gpu.py.

The rows' weights are those of a mean, some 1 / n, and the hidden states' gradients in fp16 then lie below 2^-14 (a weight of 1.6e-4 times words of
0.1 is 1.6e-5), where fp16 has a step of 2^-24 whatever the value: a value is off by up to 2^-25 from that, a tensor of m values by up to
2^-25 sqrt(m) in the 2-norm (6144 x 512: 5.3e-5, beside a norm of 0.031). That is added to fp16's limit."""
import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL
from test_vocab_loss_gpu import LIMIT, _grads, _labels, _linear_inputs, _losses_close, _teacher

pytestmark = pytest.mark.gpu


def _both(fn, ref, leaves, dloss):
    loss, grads = _grads(fn, leaves, dloss)
    want, wgrads = _grads(ref, [x.double() for x in leaves], dloss)
    _losses_close(loss, want)
    for a, e, x, what in zip(grads, wgrads, leaves, ("hidden", "weights", "bias")):
        assert a.dtype == x.dtype and a.shape == x.shape and torch.isfinite(a).all(), what
        limit = LIMIT[leaves[0].dtype] * float(e.norm()) + (2.0 ** -25 * x.numel() ** 0.5 if x.dtype == torch.float16 else 0.0)
        assert float((a.double() - e).norm()) <= limit, what


@pytest.mark.parametrize("ignored", [0.0, 0.3, 0.9])
@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "vd"), (torch.bfloat16, "dv"), (torch.float16, "vd"), (torch.float32, "vd")])
@pytest.mark.parametrize("n,d,v", [(6144, 512, 9001), (6500, 521, 45001)])
def test_cross_entropy_of_many_rows(n, d, v, dtype, layout, ignored):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n, True, layout)
    y = _labels(n, v, ignored, n)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b, label_smoothing=0.1),
          lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b, label_smoothing=0.1), [h, w, b], dl / n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ignored", [0.0, 0.5])
def test_distillation_of_many_rows(dtype, ignored):
    n, d, v = 6200, 520, 45001
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n, True, "vd")
    idx, t = _teacher(n, v, 9, n)
    idx[torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") < ignored] = -1
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b, temperature=1.7),
          lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b, temperature=1.7), [h, w, b], dl / n)
