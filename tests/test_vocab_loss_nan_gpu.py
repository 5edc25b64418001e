"""Rows without a sound loss: a label or an entry outside the vocabulary makes the row's loss NaN, and with it every gradient that the row
enters, on every tile and in both layouts, exactly where the definition in 64 bits has NaN."""
import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL
from test_vocab_loss_gpu import DEV, LIMIT, _close, _grads, _labels, _linear_inputs, _losses_close, _teacher

pytestmark = pytest.mark.gpu

# 64 x 64 tiles with and without shares of the sum, 128 x 128 tiles, 256 x 256 tiles
SIZES = [(64, 64, 1000), (1000, 64, 1000), (300, 520, 5000), (700, 520, 30011)]


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_nan_rows_make_the_gradients_nan(n, d, v, dtype, layout):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n, True, layout)
    y = _labels(n, v, 0.3, n)
    y[n // 2] = v
    idx, t = _teacher(n, v, 9, n)
    idx[n // 3, 2], t[n // 3, 2] = v + 7, 1.0
    for fn, ref in ((lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b)),
                    (lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b), lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b))):
        loss, grads = _grads(fn, [h, w, b], dl)
        want, wgrads = _grads(ref, [x.double() for x in (h, w, b)], dl)
        _losses_close(loss, want)
        assert wgrads[1].isnan().all() and wgrads[2].isnan().all()
        for a, e, what in zip(grads, wgrads, ("hidden", "weights", "bias")):
            _close(a, e, LIMIT[dtype], what)
