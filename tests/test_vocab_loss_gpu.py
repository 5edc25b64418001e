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


# the 256 x 256 tiles (K-contiguous operands, gradient laid out both ways), one and several pieces of the vocabulary
@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "vd"), (torch.bfloat16, "dv"), (torch.float16, "vd"), (torch.float32, "vd"), (torch.float32, "dv")])
@pytest.mark.parametrize("n,d,v,eps", [(700, 264, 40001, 0.0), (1025, 513, 30522, 0.1), (4100, 64, 70001, 0.0)])
def test_large_tiles_match_the_definition(n, d, v, eps, dtype, layout):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n + d, True, layout)
    y = _labels(n, v, 0.4, n)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b, label_smoothing=eps),
          lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b, label_smoothing=eps), [h, w, b], dl / n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_tiles_of_the_distillation_match_the_definition(dtype):
    n, d, v = 900, 256, 30011
    h, w, _, dl = _linear_inputs(n, d, v, dtype, 5, False, "vd")
    idx, t = _teacher(n, v, 33, 4)
    _both(lambda h, w: VL.linear_topk_distillation(h, w, idx, t, temperature=3.0),
          lambda h, w: VL.linear_topk_distillation_reference(h, w, idx, t, temperature=3.0), [h, w], dl / n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 40, 300, 2000])
def test_ignored_rows_take_no_part_whatever_they_hold(n, dtype):
    """NaN and infinities in the hidden states of ignored rows: losses and all gradients are those of the other rows, bit for bit."""
    h, w, b, dl = _linear_inputs(n, 72, 300, dtype, n, True, "vd")
    y = _labels(n, 300, 0.5, n)
    y[0] = 7
    clean = _grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), [h, w, b], dl)
    bad = h.clone()
    bad[y == -100] = math.nan
    if n > 2:
        bad[(y == -100).nonzero().squeeze(1)[::2]] = math.inf
    dirty = _grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), [bad, w, b], dl)
    assert torch.equal(clean[0], dirty[0]) and (clean[0][y == -100] == 0).all()
    for a, e in zip(dirty[1], clean[1]):
        assert torch.equal(a, e)
    assert (dirty[1][0][y == -100] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [5, 600])
def test_a_batch_without_labels_gives_zeros(n, dtype):
    h, w, b, dl = _linear_inputs(n, 64, 40000, dtype, 1, True, "vd")
    y = torch.full((n,), -100, device=DEV)
    loss, grads = _grads(lambda h, w, b: VL.linear_cross_entropy(h * math.nan, w, y, b), [h, w, b], dl)
    assert (loss == 0).all() and (grads[1] == 0).all() and (grads[2] == 0).all()
    idx = torch.full((n, 4), -1, device=DEV)
    loss, grads = _grads(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, torch.zeros(n, 4, device=DEV), b), [h, w, b], dl)
    assert (loss == 0).all() and all((g == 0).all() for g in grads)


def test_no_rows():
    w = torch.randn(11, 8, device=DEV, requires_grad=True)
    h = torch.randn(0, 8, device=DEV, requires_grad=True)
    loss = VL.linear_cross_entropy(h, w, torch.zeros(0, dtype=torch.int64, device=DEV))
    assert loss.shape == (0,)
    dh, dw = torch.autograd.grad(loss.sum(), [h, w])
    assert dh.shape == (0, 8) and (dw == 0).all()


@pytest.mark.parametrize("n", [3, 200, 1000])
def test_banned_words_and_rows_of_very_different_scale(n):
    """Words banned by a bias of -inf or the type's lowest value have probability 0; rows whose scores lie 10^4 apart share a tile (the sums of
    exponentials need a reference of their own there)."""
    d, v = 64, 1500
    h, w, b, dl = _linear_inputs(n, d, v, torch.bfloat16, n, True, "vd", bias_dtype=torch.float32)
    b[::3] = -math.inf
    b[1::3] = torch.finfo(torch.float32).min
    b[1400:] = -math.inf                                                # whole column strips without a finite score
    h[0] *= 1000.0
    h[n // 2] *= -300.0
    h[n - 1] *= 1e-3
    y = (torch.randint(0, 400, (n,), generator=_gen(n), device=DEV) * 3 + 2)
    loss, grads = _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b), [h, w, b], dl)
    assert torch.isfinite(loss).all()
    assert (grads[2][::3] == 0).all() and (grads[2][1::3] == 0).all()
    y[1] = 0                                                            # a banned label: infinite loss, finite gradient
    loss, grads = _grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), [h, w, b], dl)
    assert math.isinf(float(loss[1])) and torch.isfinite(grads[0]).all() and torch.isfinite(grads[1]).all()


def test_nan_stays_in_its_row_and_bad_labels_are_nan():
    n, v = 300, 700
    h, w, _, dl = _linear_inputs(n, 64, v, torch.bfloat16, 3, False, "vd")
    h[17, 5] = math.nan
    y = _labels(n, v, 0.0, 3)
    y[40], y[41] = v, -1
    loss = VL.linear_cross_entropy(h, w, y)
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[[17, 40, 41]] = True
    assert torch.equal(loss.isnan(), bad)
    dh = torch.autograd.grad(VL.linear_cross_entropy(h.requires_grad_(), w, y), h, dl)[0]
    assert torch.equal(dh.isnan().any(1), bad)
    idx, t = _teacher(n, v, 9, 3, padded=0.0)
    idx[5, 3], t[6, 1], t[7, 2] = v, math.nan, math.inf
    loss = VL.linear_topk_distillation(h.detach().nan_to_num(0.0), w, idx, t)
    assert loss.isnan().nonzero().squeeze(1).tolist() == [5, 6, 7]
    z = torch.randn(n, v, device=DEV, requires_grad=True)
    loss = VL.topk_distillation(z, idx, t)
    assert loss.isnan().nonzero().squeeze(1).tolist() == [5, 6, 7]
    dz = torch.autograd.grad(loss, z, dl)[0]
    assert dz.isnan().any(1).nonzero().squeeze(1).tolist() == [5, 6, 7]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_offsets_and_index_types(dtype):
    """Hidden states cut out of [B, T, D], weights cut out of a larger table (offset rows, odd row starts), INT32 labels, a bias in fp32."""
    B, T, D, V = 6, 33, 80, 333
    g = _gen(8)
    full = torch.randn(B, T + 1, D + 5, generator=g, device=DEV).to(dtype)
    table = (torch.randn(V + 9, D + 3, generator=g, device=DEV) * 0.3).to(dtype)
    bias = torch.randn(V, generator=g, device=DEV)
    y = torch.randint(0, V, (B, T), generator=g, device=DEV).to(torch.int32)
    y[2, 4:] = -1
    dl = torch.rand(B, T, generator=g, device=DEV)

    def run(fn, full, table, bias):
        full, table, bias = [x.detach().requires_grad_() for x in (full, table, bias)]
        loss = fn(full[:, :-1, 3:3 + D], table[4:4 + V, 1:1 + D], y, bias, ignore_index=-1)
        return loss.detach(), torch.autograd.grad(loss, [full, table, bias], dl.to(loss.dtype))

    loss, grads = run(VL.linear_cross_entropy, full, table, bias)
    want, wgrads = run(VL.linear_cross_entropy_reference, full.double(), table.double(), bias.double())
    assert loss.shape == (B, T)
    _losses_close(loss, want)
    for a, e, name in zip(grads, wgrads, ("hidden", "weights", "bias")):
        _close(a, e, LIMIT[dtype], name)
    big = torch.randn(50, 4, 120, generator=g, device=DEV).to(dtype).requires_grad_()
    idx, t = torch.randint(0, 100, (50, 4, 7), generator=g, device=DEV).to(torch.int32), torch.randn(50, 4, 7, generator=g, device=DEV).half()
    lo = VL.topk_distillation(big[..., 3:103], idx, t, temperature=2.0)
    ref = big.detach().double().requires_grad_()
    lw = VL.topk_distillation_reference(ref[..., 3:103], idx, t, temperature=2.0)
    _losses_close(lo.detach(), lw.detach())
    _close(torch.autograd.grad(lo.sum(), big)[0], torch.autograd.grad(lw.sum(), ref)[0], LIMIT[dtype], "logits")


@pytest.mark.parametrize("n,d,v,dtype", [(64, 128, 1000, torch.bfloat16), (900, 256, 40000, torch.bfloat16), (300, 100, 2000, torch.float32)])
def test_results_do_not_change_from_run_to_run(n, d, v, dtype):
    h, w, b, dl = _linear_inputs(n, d, v, dtype, 2, True, "vd")
    y = _labels(n, v, 0.3, 1)
    idx, t = _teacher(n, v, 20, 1)
    for fn in (lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b)):
        first = _grads(fn, [h, w, b], dl)
        for _ in range(4):
            again = _grads(fn, [h, w, b], dl)
            assert torch.equal(first[0], again[0]) and all(torch.equal(a, e) for a, e in zip(first[1], again[1]))


def test_gradients_that_nobody_asks_for_are_left_out():
    h, w, b, dl = _linear_inputs(50, 64, 200, torch.bfloat16, 6, True, "vd")
    y = _labels(50, 200, 0.1, 2)
    _, (dh, dw, db) = _grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), [h, w, b], dl)
    for k, want in enumerate((dh, dw, db)):
        leaves = [x.detach().requires_grad_(j == k) for j, x in enumerate((h, w, b))]
        got = torch.autograd.grad(VL.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2]), leaves[k], dl)[0]
        assert torch.equal(got, want)
    loss = VL.linear_cross_entropy(h.requires_grad_(), w, y, b)
    one = torch.autograd.grad(loss, h, dl, retain_graph=True)[0]
    assert torch.equal(one, torch.autograd.grad(loss, h, 1.0 * dl)[0])                  # the same graph walked twice
    loss = VL.linear_cross_entropy(h, w, y, b)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, h, dl)


def test_captured_step_replays_with_new_data():
    """A forward + backward pass recorded into a graph (fresh leaves, no other graph of theirs alive) gives the eager results on every replay."""
    n, d, v = 300, 128, 5000
    h, w, b, dl = _linear_inputs(n, d, v, torch.bfloat16, 1, True, "vd")
    y, (idx, t) = _labels(n, v, 0.3, 1), _teacher(n, v, 8, 1)
    z = torch.randn(n, v, generator=_gen(4), device=DEV).bfloat16()

    def step(h, w, b, z):
        a = VL.linear_cross_entropy(h, w, y, b)
        k = VL.linear_topk_distillation(h, w, idx, t, b, temperature=2.0)
        m = VL.topk_distillation(z, idx, t, temperature=2.0)
        return (a, k, m) + torch.autograd.grad([a, k, m], [h, w, b, z], [dl, dl, dl])

    def fresh():
        return [x.detach().clone().requires_grad_() for x in (h, w, b, z)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(*fresh())
    torch.cuda.current_stream().wait_stream(s)
    leaves = fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*leaves)
    gen = _gen(77)
    for round_ in range(3):
        with torch.no_grad():
            for x in leaves:
                x.copy_(torch.randn(x.shape, generator=gen, device=DEV) * 0.3)
            y.copy_(torch.where(torch.rand(n, generator=gen, device=DEV) < 0.2 * round_, -100, torch.randint(0, v, (n,), generator=gen, device=DEV)))
            idx[round_ * 7] = -1
        g.replay()
        torch.cuda.synchronize()
        want = step(*[x.detach().clone().requires_grad_() for x in leaves])
        for a, e in zip(out, want):
            assert torch.equal(a, e)


def test_two_streams_at_once():
    n, d, v = 400, 128, 3000
    h, w, b, dl = _linear_inputs(n, d, v, torch.bfloat16, 1, True, "vd")
    ys = [_labels(n, v, 0.3, k) for k in (1, 2)]
    want = [_grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), [h, w, b], dl) for y in ys]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(_grads(lambda h, w, b: VL.linear_cross_entropy(h, w, ys[k], b), [h, w, b], dl))
    torch.cuda.synchronize()
    for k in range(2):
        for loss, grads in got[k]:
            assert torch.equal(loss, want[k][0]) and all(torch.equal(a, e) for a, e in zip(grads, want[k][1]))


def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements, a table of more than 2^32 bytes: the last rows come out as on their own."""
    n, v = 36000, 65536
    z = torch.empty(n, v, dtype=torch.bfloat16, device=DEV)
    z[-64:] = torch.randn(64, v, generator=_gen(1), device=DEV).bfloat16()
    idx = torch.full((n, 5), -1, device=DEV)
    idx[-64:] = torch.randint(0, v, (64, 5), generator=_gen(2), device=DEV)
    t = torch.randn(n, 5, generator=_gen(3), device=DEV)
    dl = torch.ones(n, device=DEV)
    loss, (dz,) = _grads(lambda z: VL.topk_distillation(z, idx, t), [z], dl)
    tail, (dtail,) = _grads(lambda z: VL.topk_distillation(z, idx[-64:], t[-64:]), [z[-64:].clone()], dl[-64:])
    assert torch.equal(loss[-64:], tail) and torch.equal(dz[-64:], dtail) and (loss[:-64] == 0).all() and not dz[n // 2].any()
    del z, dz
    v, d = 1_100_000, 2048
    w = torch.empty(v, d, dtype=torch.bfloat16, device=DEV).uniform_(-0.05, 0.05, generator=_gen(5))
    h = torch.randn(3, d, generator=_gen(6), device=DEV).bfloat16()
    y = torch.tensor([v - 1, 5, v - 77], device=DEV)
    b = torch.zeros(v, device=DEV)
    b[:v - 5000] = -math.inf                                            # what is left lies behind 4 GiB
    b[5] = 0.0
    loss, (dh, dw) = _grads(lambda h, w: VL.linear_cross_entropy(h, w, y, b), [h, w], torch.ones(3, device=DEV))
    keep = torch.cat([torch.tensor([5], device=DEV), torch.arange(v - 5000, v, device=DEV)])
    sub = torch.tensor([5000, 0, 5001 - 77], device=DEV)
    want, (dhe, dwe) = _grads(lambda h, w: VL.linear_cross_entropy_reference(h, w, sub), [h.double(), w[keep].double()], torch.ones(3, device=DEV))
    _losses_close(loss, want)
    _close(dh, dhe, LIMIT[torch.bfloat16], "hidden")
    _close(dw[keep], dwe, LIMIT[torch.bfloat16], "weights")
    assert not dw[6:v - 5000].any()


@pytest.mark.parametrize("k", [1, 64, 1024])
def test_one_index_many_times_and_weightless_entries(k):
    """All of a row's entries on one word; entries whose logit is -inf count as none."""
    n, d, v = 70, 64, 500
    h, w, b, dl = _linear_inputs(n, d, v, torch.bfloat16, k, True, "vd")
    idx = (torch.arange(n, device=DEV) % v).unsqueeze(1).expand(n, k).contiguous()
    t = torch.randn(n, k, generator=_gen(k), device=DEV)
    if k > 1:
        idx[:, 1::2] = 3
        t[:, 3::4] = -math.inf
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b), lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b), [h, w, b], dl)
    z = torch.randn(n, v, generator=_gen(1), device=DEV).bfloat16()
    _both(lambda z: VL.topk_distillation(z, idx, t), lambda z: VL.topk_distillation_reference(z, idx, t), [z], dl, names=("logits",))


def test_ops_run_on_the_kernels_and_train_together():
    """The three ops through SameDiff: one student graph with tied word embedding, cross entropy on the labels, distillation on the unkept and on
    kept logits. Gradients of the training session (autograd) and of the gradient graph (_bp ops) agree with the plain forms in fp64."""
    from deeplearning4j_amd.autodiff.samediff import SameDiff
    from deeplearning4j_amd.nd4j.ops.custom import OpExecutioner
    n, d, v, k = 96, 64, 1000, 8
    g = torch.Generator().manual_seed(0)
    emb0, b0, w0 = torch.randn(v, d, generator=g) * 0.3, torch.randn(v, generator=g) * 0.1, torch.randn(d, d, generator=g) * 0.2
    tok = torch.randint(0, v, (n,), generator=g)
    lab = torch.randint(0, v, (n,), generator=g)
    lab[::5] = -100
    idx, t = torch.randint(0, v, (n, k), generator=g), torch.randn(n, k, generator=g)
    sd = SameDiff.create(DEV)
    emb, bias, W = sd.var("emb", emb0), sd.var("bias", b0), sd.var("W", w0)
    x = sd.nn.tanh(sd.nn.embeddingLookup(emb, sd.placeHolder("tok", "INT64", -1)).mmul(W))
    y, ti, tl = sd.placeHolder("lab", "INT64", -1), sd.placeHolder("ti", "INT64", -1, k), sd.placeHolder("tl", "FLOAT", -1, k)
    ce = sd.loss.linearSoftmaxCrossEntropy(x, emb, y, bias, 0.1)
    kd = sd.loss.linearTopKDistillation(x, emb, ti, tl, bias, 2.0)
    kl = sd.loss.topKDistillation(x, sd.constant("ti2", (idx % d).to(DEV)), tl, 1.5)
    (ce.mean() + kd.mean() + kl.mean()).rename("loss").markAsLoss()
    ph = {"tok": tok.to(DEV), "lab": lab.to(DEV), "ti": idx.to(DEV), "tl": t.to(DEV)}
    OpExecutioner.resetHelperStatistics()
    got = {m: _tensor(a) for m, a in sd.calculateGradients(ph, ["emb", "bias", "W"]).items()}
    hit = OpExecutioner.helperStatistics()["hit"]
    assert all(hit.get(o, 0) > 0 for o in ("linear_softmax_cross_entropy_loss", "linear_topk_distillation_loss", "topk_distillation_loss")), hit
    E, B, M = [a.double().to(DEV).requires_grad_() for a in (emb0, b0, w0)]
    X = torch.tanh(E[tok.to(DEV)] @ M)
    ref = (VL.linear_cross_entropy_reference(X, E, lab.to(DEV), B, label_smoothing=0.1).mean()
           + VL.linear_topk_distillation_reference(X, E, idx.to(DEV), t.to(DEV), B, 2.0).mean()
           + VL.topk_distillation_reference(X, (idx % d).to(DEV), t.to(DEV), 1.5).mean())
    want = dict(zip(("emb", "bias", "W"), torch.autograd.grad(ref, [E, B, M])))
    for m in want:
        # fp32 all the way, products and sums of up to 1000 terms behind one another: a few 2^-24 sqrt(1000) each
        _close(got[m], want[m], 1e-5, m)
    grads = sd.createGradFunction().sd.output(ph, [m + "-grad" for m in want])
    for m in want:
        _close(_tensor(grads[m + "-grad"]), want[m], 1e-5, m + "-grad")


def _tensor(a):
    f = getattr(a, "tensor", None)
    return a if f is None else (f() if callable(f) else f)


def test_refusals():
    h, w = torch.randn(4, 8, device=DEV), torch.randn(11, 8, device=DEV)
    y = torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: VL.linear_cross_entropy(h, w.half(), y), lambda: VL.linear_cross_entropy(h, w.cpu(), y), lambda: VL.linear_cross_entropy(h, w, y.cpu()),
                 lambda: VL.linear_cross_entropy(h, w, y[:3]), lambda: VL.linear_cross_entropy(h, w, y.float()),
                 lambda: VL.linear_topk_distillation(h, w, torch.zeros(4, 1025, dtype=torch.int64, device=DEV), torch.zeros(4, 1025, device=DEV))):
        with pytest.raises(ND4JIllegalArgumentException):
            call()


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 17, 32])
def test_few_rows_against_a_wide_vocabulary(n, dtype, layout):
    d, v = 137, 16399
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n, True, layout)
    y = _labels(n, v, 0.2, n)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b), [h, w, b], dl)
    idx, t = _teacher(n, v, 33, n)
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b, 1.5),
          lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b, 1.5), [h, w, b], dl)


def test_one_row_without_a_row_axis():
    h, w, b, dl = _linear_inputs(1, 72, 300, torch.float32, 5, True, "vd")
    h, dl, y = h[0], dl[0], torch.tensor(7, device=DEV)
    idx, t = torch.tensor([3, 299, -1], device=DEV), torch.tensor([0.5, 1.5, 9.0], device=DEV)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b), [h, w, b], dl)
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b), lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b), [h, w, b], dl)
    _both(lambda z: VL.topk_distillation(z, idx, t), lambda z: VL.topk_distillation_reference(z, idx, t), [b], dl, names=("logits",))


@pytest.mark.parametrize("exponent", [-70, -110])
def test_tiny_hidden_states_beside_a_large_bias(exponent):
    """fp32 operands in scaled halves: the bias, up to some 10^5, is scaled with them."""
    n, d, v = 600, 512, 1000
    h, w, b, dl = _linear_inputs(n, d, v, torch.float32, 4, True, "vd")
    h, b = h * 2.0 ** exponent, b * 3e4
    y = b.argsort(descending=True)[:3].repeat(n // 3)
    loss, grads = _grads(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b, label_smoothing=0.1), [h, w, b], dl)
    want, wgrads = _grads(lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b, label_smoothing=0.1), [t.double() for t in (h, w, b)], dl)
    _losses_close(loss, want)
    for k, (a, e) in enumerate(zip(grads, wgrads)):
        if k == 1 and exponent < -100:                                  # products of the hidden states alone: 2^-24 of the scaled range is gone
            assert torch.isfinite(a).all()
        else:
            _close(a, e, LIMIT[torch.float32], ("hidden", "weights", "bias")[k])


def test_the_loss_and_the_labels_may_be_changed_before_the_backward_pass():
    h, w, b, dl = _linear_inputs(50, 64, 500, torch.bfloat16, 6, True, "vd")
    y = _labels(50, 500, 0.2, 6)
    idx, t = _teacher(50, 500, 9, 6)
    for fn, held in ((lambda *p: VL.linear_cross_entropy(p[0], p[1], y, p[2]), (y,)),
                     (lambda *p: VL.linear_topk_distillation(p[0], p[1], idx, t, p[2]), (idx, t))):
        want = _grads(fn, [h, w, b], dl * 0.5)[1]
        leaves = [x.detach().requires_grad_() for x in (h, w, b)]
        loss = fn(*leaves)
        loss.mul_(0.5)
        kept = [x.clone() for x in held]
        for x in held:
            x.zero_()
        got = torch.autograd.grad(loss, leaves, dl)
        for x, k in zip(held, kept):
            x.copy_(k)
        assert all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [129, 256])
def test_gradient_halves_on_large_tiles(n, dtype, layout):
    """Up to 256 rows the scores' gradient comes in two halves, whatever the tile that forms it. What is left of its rounding is u^2, so the
    weights' and hidden states' gradients are off by their own rounding alone."""
    d, v = 72, 45057
    h, w, b, dl = _linear_inputs(n, d, v, dtype, n, True, layout)
    y = _labels(n, v, 0.1, n)
    _both(lambda h, w, b: VL.linear_cross_entropy(h, w, y, b), lambda h, w, b: VL.linear_cross_entropy_reference(h, w, y, b), [h, w, b], dl,
          limit=LIMIT[dtype] / 2)
    idx, t = _teacher(n, v, 17, n)
    _both(lambda h, w, b: VL.linear_topk_distillation(h, w, idx, t, b), lambda h, w, b: VL.linear_topk_distillation_reference(h, w, idx, t, b), [h, w, b], dl,
          limit=LIMIT[dtype] / 2)


@pytest.mark.parametrize("n,d,v", [(1, 64, 17001), (3, 1, 16387), (27, 1085, 16595), (32, 33, 20000), (30, 130, 1003), (64, 257, 5001), (33, 31, 2)])
@pytest.mark.parametrize("layout", ["vd", "dv"])
def test_forward_of_few_rows_reads_weights_off_16_bytes(n, d, v, layout):
    """fp32 weights cut out of a larger table at an odd place: every row starts and ends on 4 bytes only; what lies around them is NaN."""
    h, w, b, _ = _linear_inputs(n, d, v, torch.float32, n, True, "vd")
    rows, cols = (v, d) if layout == "vd" else (d, v)
    table = torch.full((rows + 2, cols + 3), math.nan, device=DEV)
    part = table[1:1 + rows, 1:1 + cols]
    part.copy_(w if layout == "vd" else w.t())
    w = part if layout == "vd" else part.t()
    y = _labels(n, v, 0.2, n)
    _losses_close(VL.linear_cross_entropy(h, w, y, b), VL.linear_cross_entropy_reference(h.double(), w.double(), y, b.double()))
    k = min(9, v)
    idx, t = _teacher(n, v, k, n)
    _losses_close(VL.linear_topk_distillation(h, w, idx, t, b), VL.linear_topk_distillation_reference(h.double(), w.double(), idx, t, b.double()))
