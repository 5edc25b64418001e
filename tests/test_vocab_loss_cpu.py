"""Losses over a large vocabulary (ops/vocab_loss.py): argument checks, the plain forms against the definition, gradients against differences,
and the ops' surfaces (Nd4j.loss(), sd.loss, gradient graph) on the CPU."""
import math

import pytest
import torch

from deeplearning4j_amd.autodiff.samediff import SameDiff
from deeplearning4j_amd.nd4j.exceptions import ND4JIllegalArgumentException
from deeplearning4j_amd.nd4j.factory import Nd4j
from deeplearning4j_amd.ops import vocab_loss as VL


def _inputs(seed=0, n=7, d=6, v=11, k=4):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                    # noqa: E731
    y = torch.randint(0, v, (n,), generator=g)
    y[2] = -100
    idx = torch.randint(0, v, (n, k), generator=g)
    idx[1], idx[3, 2] = -1, -1
    idx[4, 1] = idx[4, 0]
    return r(n, d), r(v, d), r(v), y, idx, r(n, k)


def _tensor(a):
    f = getattr(a, "tensor", None)
    return a if f is None else (f() if callable(f) else f)


def test_plain_forms_follow_the_definition():
    h, w, b, y, idx, t = _inputs()
    z = h @ w.t() + b
    logq = torch.log_softmax(z, 1)
    eps = 0.2
    for n in range(len(y)):
        want = 0.0 if y[n] < 0 else float(-(1 - eps) * logq[n, y[n]] - eps * logq[n].mean())
        assert abs(float(VL.linear_cross_entropy(h, w, y, b, label_smoothing=eps)[n]) - want) < 1e-12
        T = 1.7
        at = [k for k in range(idx.shape[1]) if idx[n, k] >= 0]
        p = torch.softmax(t[n, at] / T, 0) if at else torch.zeros(0, dtype=torch.float64)
        lq = torch.log_softmax(z[n] / T, 0)
        want = T * T * float(sum(p[j] * (p[j].log() - lq[idx[n, k]]) for j, k in enumerate(at))) if at else 0.0
        assert abs(float(VL.linear_topk_distillation(h, w, idx, t, b, T)[n]) - want) < 1e-12
        assert abs(float(VL.topk_distillation(z, idx, t, T)[n]) - want) < 1e-12


def test_gradients_against_differences():
    h, w, b, y, idx, t = _inputs(1)
    for x in (h, w, b):
        x.requires_grad_()
    assert torch.autograd.gradcheck(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b, label_smoothing=0.1), (h, w, b))
    assert torch.autograd.gradcheck(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b, temperature=2.0), (h, w, b))
    z = (h.detach() @ w.detach().t()).requires_grad_()
    assert torch.autograd.gradcheck(lambda z: VL.topk_distillation(z, idx, t, temperature=0.5), (z,))


def test_ignored_rows_and_bad_labels():
    h, w, b, y, idx, t = _inputs(2)
    bad = h.clone()
    bad[2] = math.nan
    bad.requires_grad_()
    w.requires_grad_()
    loss = VL.linear_cross_entropy(bad, w, y, b)
    dh, dw = torch.autograd.grad(loss.sum(), [bad, w])
    assert loss[2] == 0 and (dh[2] == 0).all() and torch.isfinite(dw).all()
    y[0], y[5] = 11, -3
    assert VL.linear_cross_entropy(h, w, y, b).isnan().nonzero().squeeze(1).tolist() == [0, 5]
    idx[6, 0] = 11
    assert VL.linear_topk_distillation(h, w, idx, t).isnan().nonzero().squeeze(1).tolist() == [6]
    none = torch.full_like(y, -100)
    assert (VL.linear_cross_entropy(h, w, none) == 0).all()


@pytest.mark.parametrize("name,call", [
    ("types differ", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w.float(), y)),
    ("hidden is integral", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h.long(), w.long(), y)),
    ("widths differ", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h[:, :5], w, y)),
    ("weights 1-D", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w[0], y)),
    ("empty vocabulary", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w[:0], y)),
    ("bias length", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y, b[:4])),
    ("bias type", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y, b.half())),
    ("float labels", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y.double())),
    ("label count", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y[:3])),
    ("label rank", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y[:, None])),
    ("smoothing 1", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y, label_smoothing=1.0)),
    ("smoothing < 0", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y, label_smoothing=-0.1)),
    ("smoothing NaN", lambda h, w, b, y, i, t: VL.linear_cross_entropy(h, w, y, label_smoothing=math.nan)),
    ("float indices", lambda h, w, b, y, i, t: VL.linear_topk_distillation(h, w, i.double(), t)),
    ("teacher shapes", lambda h, w, b, y, i, t: VL.linear_topk_distillation(h, w, i, t[:, :2])),
    ("teacher rows", lambda h, w, b, y, i, t: VL.topk_distillation(h, i[:2], t[:2])),
    ("no entries", lambda h, w, b, y, i, t: VL.topk_distillation(h, i[:, :0], t[:, :0])),
    ("too many entries", lambda h, w, b, y, i, t: VL.topk_distillation(h, i.repeat(1, 300), t.repeat(1, 300))),
    ("integral teacher", lambda h, w, b, y, i, t: VL.topk_distillation(h, i, i)),
    ("temperature 0", lambda h, w, b, y, i, t: VL.topk_distillation(h, i, t, 0.0)),
    ("temperature inf", lambda h, w, b, y, i, t: VL.topk_distillation(h, i, t, math.inf)),
    ("temperature NaN", lambda h, w, b, y, i, t: VL.linear_topk_distillation(h, w, i, t, temperature=math.nan)),
])
def test_refusals(name, call):
    with pytest.raises(ND4JIllegalArgumentException):
        call(*_inputs())


def test_namespaces_and_gradient_graph():
    h, w, b, y, idx, t = _inputs(3)
    e = Nd4j.loss().linearSoftmaxCrossEntropy(h, w, y, b, 0.1)
    torch.testing.assert_close(_tensor(e), VL.linear_cross_entropy(h, w, y, b, label_smoothing=0.1))
    e = Nd4j.loss().linearSoftmaxCrossEntropy(h, w.t().contiguous(), y, None, 0.0, 3, True)
    torch.testing.assert_close(_tensor(e), VL.linear_cross_entropy(h, w, y, ignore_index=3), equal_nan=True)   # -100 is a bad label here: NaN
    torch.testing.assert_close(_tensor(Nd4j.loss().linearTopKDistillation(h, w, idx, t, b, 2.0)), VL.linear_topk_distillation(h, w, idx, t, b, 2.0))
    torch.testing.assert_close(_tensor(Nd4j.loss().topKDistillation(h, idx % 6, t, 2.0)), VL.topk_distillation(h, idx % 6, t, 2.0))
    sd = SameDiff.create("cpu")
    H, W, B = sd.var("h", h), sd.var("w", w.t().contiguous()), sd.var("b", b)
    ce = sd.loss.linearSoftmaxCrossEntropy(H, W, sd.constant("y", y), B, 0.1, -100, True)
    kd = sd.loss.linearTopKDistillation(H, W, sd.constant("i", idx), sd.constant("t", t), None, 1.5, True)
    kl = sd.loss.topKDistillation(H, sd.constant("i2", torch.where(idx < 0, idx, idx % 6)), sd.constant("t2", t), 3.0)
    (ce.mean() + kd.sum() + kl.mean()).rename("loss").markAsLoss()
    x, m, c = h.clone().requires_grad_(), w.t().contiguous().requires_grad_(), b.clone().requires_grad_()
    loss = (VL.linear_cross_entropy(x, m.t(), y, c, label_smoothing=0.1).mean() + VL.linear_topk_distillation(x, m.t(), idx, t, None, 1.5).sum()
            + VL.topk_distillation(x, torch.where(idx < 0, idx, idx % 6), t, 3.0).mean())
    want = dict(zip("hwb", torch.autograd.grad(loss, [x, m, c])))
    got = sd.calculateGradients({}, ["h", "w", "b"])
    for n in "hwb":
        torch.testing.assert_close(_tensor(got[n]), want[n])
    graph = sd.createGradFunction().sd.output({}, [n + "-grad" for n in "hwb"])
    for n in "hwb":
        torch.testing.assert_close(_tensor(graph[n + "-grad"]), want[n])


def test_gradients_are_differentiable_once_only_on_request():
    h, w, b, y, idx, t = _inputs(4)
    h.requires_grad_()
    g, = torch.autograd.grad(VL.linear_cross_entropy(h, w, y, b).sum(), h, create_graph=True)     # the plain form differentiates twice
    assert torch.autograd.grad(g.sum(), h)[0].shape == h.shape
