"""The linear vocabulary losses on values of very different size: rows, words and row weights that lie many powers of ten apart must not
disturb one another. Against the definition in 64 bits; sizes reach the fp32 cores, the products of halves on both tiles and both layouts.

Tolerances. Losses of single rows: 4e-6 of the row's own size (at least of 1), as the sum of D = 512 fp32 products and a normaliser of V terms
gives it. Gradients of single rows in the 2-norm: fp32 4e-6 (2e-6 for a whole tensor; a row of 64 or more values spreads around that by less than
a factor of two), fp16 two roundings of 2^-11."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROW = {torch.float32: 4e-6, torch.float16: 2 * 2.0 ** -11}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inputs(n, d, v, dtype, layout, seed=0):
    g = _gen(seed + n + v)
    h = torch.randn(n, d, generator=g, device=DEV)
    w = torch.randn(v, d, generator=g, device=DEV) * (2.5 / math.sqrt(d))
    b = torch.randn(v, generator=g, device=DEV)
    y = torch.randint(0, v, (n,), generator=g, device=DEV)
    idx, t = torch.randint(0, v, (n, 9), generator=g, device=DEV), torch.randn(n, 9, generator=g, device=DEV) * 2
    return h.to(dtype), w.to(dtype), b.to(dtype), y, idx, t, torch.rand(n, generator=g, device=DEV) + 0.5


def _step(distil, h, w, b, y, idx, t, dl, layout, plain=False):
    if layout == "dv":
        w = w.t().contiguous().t()
    h, w, b = [x.detach().requires_grad_() for x in (h, w, b)]
    if distil:
        loss = VL.linear_topk_distillation(h, w, idx, t, b, temperature=1.5, plain=plain)
    else:
        loss = VL.linear_cross_entropy(h, w, y, b, plain=plain)
    return (loss.detach(),) + torch.autograd.grad(loss, [h, w, b], dl.to(loss.dtype))


def _both(distil, h, w, b, y, idx, t, dl, layout):
    return _step(distil, h, w, b, y, idx, t, dl, layout), _step(distil, h.double(), w.double(), b.double(), y, idx, t, dl, layout, plain=True)


def _rows_close(got, want, limit, what):
    err, ref = (got.double() - want).norm(dim=1), want.norm(dim=1)
    worst = int((err - limit * ref).argmax())
    assert bool((err <= limit * ref + 1e-300).all()), "%s: row %d is off by %.3g of its size" % (what, worst, float(err[worst] / ref[worst]))


def _losses_close(got, want):
    bad = (got.double() - want).abs() / want.abs().clamp(min=1.0)
    assert float(bad.max()) <= 4e-6, "loss of row %d is off by %.3g" % (int(bad.argmax()), float(bad.max()))


# fp32 cores; halves on 128 x 128 tiles; halves on 256 x 256 tiles with both layouts of the gradient
SIZES = [(40, 64, 900), (500, 512, 4000), (700, 520, 30000)]


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("factor", [1e6, 1e9, 1e12])
@pytest.mark.parametrize("distil", [False, True])
def test_one_huge_row_leaves_the_others_alone(n, d, v, factor, layout, distil):
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    h[n // 3] *= factor
    (loss, dh, _, _), (eloss, edh, _, _) = _both(distil, h, w, b, y, idx, t, dl, layout)
    others = torch.arange(n, device=DEV) != n // 3
    _losses_close(loss[others], eloss[others])
    _rows_close(dh[others], edh[others], ROW[torch.float32], "hidden")


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("factor", [1e6, 1e9])
@pytest.mark.parametrize("distil", [False, True])
def test_one_huge_word_leaves_the_others_alone(n, d, v, factor, layout, distil):
    """A word whose weights are far larger than the others', with scores so low that it has no probability anywhere."""
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    h[:, 0] = h[:, 0].abs() + 0.5
    j = v // 2
    w[j] = 0.0
    w[j, 0] = -factor * 0.4
    y[y == j] = 0
    idx[idx == j] = 0
    (loss, dh, dw, db), (eloss, edh, edw, edb) = _both(distil, h, w, b, y, idx, t, dl, layout)
    _losses_close(loss, eloss)
    _rows_close(dh, edh, ROW[torch.float32], "hidden")
    others = torch.arange(v, device=DEV) != j
    assert (dw[j] == 0).all() and float((dw[others].double() - edw[others]).norm()) <= 2e-6 * float(edw[others].norm())
    assert float((db.double() - edb).norm()) <= 2e-6 * float(edb.norm())


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("distil", [False, True])
def test_words_of_very_different_size(n, d, v, layout, distil):
    """Words of zeros, and words down to 1e-12 of the largest: their scores hardly count, their gradients are as large as any."""
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    w *= 10.0 ** (-12 * torch.rand(v, 1, generator=_gen(5), device=DEV))
    w[::7] = 0.0
    got, want = _both(distil, h, w, b, y, idx, t, dl, layout)
    _losses_close(got[0], want[0])
    for a, e, what in zip(got[1:], want[1:], ("hidden", "weights", "bias")):
        assert float((a.double() - e).norm()) <= 2e-6 * float(e.norm()), what
    labelled = y.unique() if not distil else idx.reshape(-1).unique()
    _rows_close(got[2][labelled], want[2][labelled], ROW[torch.float32], "weights")


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("distil", [False, True])
def test_row_weights_from_1_to_1e_8(n, d, v, layout, distil):
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    dl *= 10.0 ** -(torch.arange(n, device=DEV) % 9).float()
    dl[5] = 0.0
    got, want = _both(distil, h, w, b, y, idx, t, dl, layout)
    assert (got[1][5] == 0).all()
    _rows_close(got[1], want[1], ROW[torch.float32], "hidden")
    for a, e, what in zip(got[2:], want[2:], ("weights", "bias")):
        assert float((a.double() - e).norm()) <= 2e-6 * float(e.norm()), what


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", [(300, 64, 900), (700, 520, 30000), (300, 101, 1003)])
@pytest.mark.parametrize("distil", [False, True])
def test_row_weights_from_1_to_1e_7_in_half_precision(n, d, v, layout, distil):
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    # (weights of some 10 and hidden states of some 0.1, and a loss scale: the small rows' gradients are then normal fp16 numbers)
    h, w = (h * (0.25 / math.sqrt(d))).half(), (w * (10 / 2.5 * math.sqrt(d))).half()
    dl *= 1e3 * 10.0 ** -(torch.arange(n, device=DEV) % 8).float()
    got, want = _both(distil, h, w, b.half(), y, idx, t, dl, layout)
    _rows_close(got[1], want[1], ROW[torch.float16], "hidden")
    for a, e, what in zip(got[2:], want[2:], ("weights", "bias")):
        assert float((a.double() - e).norm()) <= ROW[torch.float16] * float(e.norm()), what


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("scale", [0.0, 1e-34, 1e30])
def test_all_row_weights_tiny_huge_or_zero(n, d, v, scale, layout):
    """One row's huge hidden states count for nothing where its weight is zero."""
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    h[n // 2] *= 1e6
    dl *= scale
    dl[n // 2] = 0.0
    got, want = _both(False, h, w, b, y, idx, t, dl, layout)
    for a, e, what in zip(got[1:], want[1:], ("hidden", "weights", "bias")):
        assert torch.isfinite(a).all() and float((a.double() - e).norm()) <= 2e-6 * float(e.norm()), what


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("distil", [False, True])
def test_each_gradient_alone_is_that_of_the_whole_step(n, d, v, dtype, layout, distil):
    """With words and row weights far enough apart for factors and copies: what is not asked for is left out, the rest has the same bits."""
    h, w, b, y, idx, t, dl = _inputs(n, d, v, torch.float32, layout)
    if dtype == torch.float32:
        w *= 10.0 ** (-6 * torch.rand(v, 1, generator=_gen(5), device=DEV))
    dl *= 10.0 ** -(torch.arange(n, device=DEV) % 6).float()
    h, w, b = h.to(dtype), w.to(dtype), b.to(dtype)
    w = w if layout == "vd" else w.t().contiguous().t()

    def grads(wanted):
        x = [a.detach().requires_grad_(k in wanted) for k, a in enumerate((h, w, b))]
        if distil:
            loss = VL.linear_topk_distillation(x[0], x[1], idx, t, x[2], temperature=1.5)
        else:
            loss = VL.linear_cross_entropy(x[0], x[1], y, x[2])
        return dict(zip(wanted, torch.autograd.grad(loss, [x[k] for k in wanted], dl)))
    whole = grads((0, 1, 2))
    for wanted in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        for k, g in grads(wanted).items():
            assert torch.equal(g, whole[k]), (wanted, k)
