"""Losses over a large vocabulary (ops/vocab_loss.py) on the GPU kernels against the definition in 64 bits.

Tolerances count roundings. The rows' losses come from fp32 sums over D products and V exponentials: an error of some 2^-24 sqrt(D) in a score
of size |z| and as much again in the normaliser; 4e-6 of the largest |loss| (at least of 1) covers D = 4096. A gradient has its own rounding
(half a step: u = eps / 2, relative) and the rounding of the scores' gradient, also u relative to each of the terms that are summed; with
terms of both signs the sums' errors are u times the root of the sum of squares, which the 2-norm over the whole tensor averages. So each
gradient is held to 2 u in the 2-norm (two independent roundings of at most u each), fp32 to 2e-6 (sums of up to 2^13 terms)."""
import math

import pytest
import torch

from deeplearning4j_amd.nd4j.exceptions import ND4JIllegalArgumentException
from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"
LIMIT = {torch.bfloat16: 2 * 2.0 ** -8, torch.float16: 2 * 2.0 ** -11, torch.float32: 2e-6}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _close(got, want, limit, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), what
    ok = ~want.isnan()
    err, ref = float((got[ok] - want[ok]).norm()), float(want[ok].norm())
    assert err <= limit * ref + 1e-30, "%s: off by %.3g of %.3g (limit %.3g)" % (what, err, ref, limit * ref)


def _losses_close(got, want):
    assert got.dtype == torch.float32
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    if ok.any():
        assert float((got[ok] - want[ok]).abs().max()) <= 4e-6 * max(1.0, float(want[ok].abs().max()))


def _linear_inputs(n, d, v, dtype, seed, bias, layout, bias_dtype=None):
    g = _gen(seed)
    h = torch.randn(n, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(v, d, generator=g, device=DEV) * (2.5 / math.sqrt(d))).to(dtype)
    if layout == "dv":
        w = w.t().contiguous().t()
    b = torch.randn(v, generator=g, device=DEV).to(bias_dtype or dtype) if bias else None
    return h, w, b, torch.rand(n, generator=g, device=DEV) + 0.5


def _grads(fn, leaves, dloss):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in leaves]
    loss = fn(*leaves)
    return loss.detach(), torch.autograd.grad(loss, [t for t in leaves if t is not None], grad_outputs=dloss.to(loss.dtype))


def _both(fn, ref, leaves, dloss, limit=None, names=("hidden", "weights", "bias")):
    loss, grads = _grads(fn, leaves, dloss)
    want, wgrads = _grads(ref, [None if t is None else t.double() for t in leaves], dloss)
    _losses_close(loss, want)
    there = [(n, t) for n, t in zip(names, leaves) if t is not None]
    for (name, t), a, e in zip(there, grads, wgrads):
        assert a.dtype == t.dtype and a.shape == t.shape
        _close(a, e, limit or LIMIT[t.dtype] if t.dtype != torch.float32 or leaves[0].dtype == torch.float32 else LIMIT[leaves[0].dtype], name)
    return loss, grads


def _labels(n, v, ignored, seed, dtype=torch.int64):
    g = _gen(seed + 1)
    y = torch.randint(0, v, (n,), generator=g, device=DEV)
    y[torch.rand(n, generator=g, device=DEV) < ignored] = -100
    return y.to(dtype)


def _teacher(n, v, k, seed, padded=0.2, dtype=torch.float32):
    g = _gen(seed + 2)
    idx = torch.randint(0, v, (n, k), generator=g, device=DEV)          # now and then the same index twice
    t = (torch.randn(n, k, generator=g, device=DEV) * 2).to(dtype)
    idx[torch.rand(n, k, generator=g, device=DEV) < padded] = -1
    if n > 2:
        idx[n // 2] = -1                                                # a row without entries
        t[n // 3] = -math.inf
    return idx, t


SIZES = [(1, 8, 2), (1, 768, 1000), (2, 64, 129), (7, 100, 98), (127, 72, 255), (128, 128, 128), (129, 136, 257), (300, 520, 1031), (513, 1000, 4099),
         (1000, 96, 20001)]


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_cross_entropy_matches_the_definition(n, d, v, dtype, layout):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n + d + v, True, layout)
    y = _labels(n, v, 0.3 if n > 1 else 0.0, n)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b), [h, w, b], dl)


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_linear_distillation_matches_the_definition(n, d, v, dtype, layout):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n + d + v, True, layout)
    idx, t = _teacher(n, v, 1 + (n * 7) % 70, n)
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b, temperature=1.7),
          lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b, temperature=1.7), [h, w, b], dl)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 7, 3), (3, 9, 1024), (5, 1000, 16), (64, 1031, 64), (33, 30522, 65), (257, 4099, 200), (2, 65537, 128)])
def test_distillation_on_logits_matches_the_definition(n, v, k, dtype):
    z = (torch.randn(n, v, generator=_gen(n + v), device=DEV) * 2.5).to(dtype)
    idx, t = _teacher(n, v, k, n)
    dl = torch.rand(n, generator=_gen(9), device=DEV) + 0.5
    _both(lambda z: VL.topk_distillation(z, idx, t, temperature=2.0), lambda z: VL.topk_distillation_reference(z, idx, t, temperature=2.0), [z], dl,
          limit=max(2.0 ** -8 if dtype == torch.bfloat16 else 0, 2.0 ** -11 if dtype == torch.float16 else 0, 2e-6), names=("logits",))
