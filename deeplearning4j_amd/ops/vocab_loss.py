"""Losses over a large vocabulary: cross entropy and distillation from a teacher's top logits, straight from the hidden states (the logits
``hidden . weights^T + bias`` are never kept, neither in forward nor for backward), and the distillation loss on given logits.

    linear_cross_entropy(hidden, weights, labels)                      loss_n = lse_n - (1 - e) z[n, y_n] - (e / V) sum_j z[n, j]
    linear_topk_distillation(hidden, weights, indices, logits)         loss_n = T^2 KL(softmax(teacher_n / T) || softmax(z_n / T))
    topk_distillation(z, indices, logits)                              the same on logits that are there already

All return the loss of every row in fp32 (fp64 for fp64 operands), shaped like the rows, so that weights, masks and means are the caller's;
all are differentiable once. GPU path: native/csrc/vocab_loss.hip and topk_distill.hip for bf16 / fp16 / fp32; CPU and fp64 operands take the
plain form (``*_reference``), which is also what the tests compare with.

They stand beside ``ops/softmax.py`` (LossMCXENT on kept logits) and the declarable ``sparse_softmax_cross_entropy_loss_with_logits``
(libnd4j/include/ops/declarable/generic/loss/sparseSoftmaxCrossEntropyWithLogits.cpp), which need the [N, V] logits in memory.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from ..native import lib as L
from ..nd4j.exceptions import ND4JIllegalArgumentException

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}      # operand codes of the GEMM core
MAX_TEACHER = 1024                                                  # entries per row the kernels keep on chip
PIECE_BYTES = 256 << 20                                             # gradient of the scores held at a time: fits the last-level cache


def _need(ok, what):
    if not ok:
        raise ND4JIllegalArgumentException(what)


def _floating(t):
    return t.dtype in (torch.float32, torch.bfloat16, torch.float16, torch.float64)


def _check_linear(hidden, weights, bias, name):
    _need(hidden.dim() >= 1 and _floating(hidden), "%s: hidden must be a floating point tensor [..., D]" % name)
    _need(weights.dim() == 2 and weights.dtype == hidden.dtype, "%s: weights must be [V, D] in the type of hidden (%s)" % (name, hidden.dtype))
    _need(weights.shape[1] == hidden.shape[-1], "%s: weights are [V, %d], hidden is [..., %d]" % (name, weights.shape[1], hidden.shape[-1]))
    _need(weights.shape[0] > 0 and weights.shape[1] > 0, "%s: an empty vocabulary or hidden axis" % name)
    _need(weights.device == hidden.device, "%s: weights and hidden are on different devices" % name)
    if bias is not None:
        _need(bias.shape == (weights.shape[0],), "%s: bias must be [V] = [%d]" % (name, weights.shape[0]))
        _need(bias.dtype in (hidden.dtype, torch.float32) and bias.device == hidden.device, "%s: bias must be in the type of weights or fp32, on their device" % name)


def _check_teacher(rows, device, indices, logits, temperature, name):
    _need(indices.dtype in (torch.int32, torch.int64), "%s: teacher indices must be INT32 or INT64" % name)
    _need(_floating(logits), "%s: teacher logits must be floating point" % name)
    _need(indices.dim() == len(rows) + 1 and tuple(indices.shape[:-1]) == tuple(rows), "%s: teacher indices must be %s + [K]" % (name, list(rows)))
    _need(logits.shape == indices.shape, "%s: teacher logits %s and indices %s differ in shape" % (name, list(logits.shape), list(indices.shape)))
    _need(1 <= indices.shape[-1] <= MAX_TEACHER, "%s: 1 to %d teacher entries per row" % (name, MAX_TEACHER))
    _need(indices.device == device and logits.device == device, "%s: teacher entries are on another device" % name)
    _need(math.isfinite(temperature) and temperature > 0, "%s: temperature must be positive" % name)


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _teacher_weights(indices, logits, temperature, dtype):
    t = torch.where(indices >= 0, logits.detach().to(dtype) / temperature, -math.inf)
    p = torch.softmax(t, dim=-1)
    return torch.where((t == -math.inf).all(-1, keepdim=True), torch.zeros_like(p), p)


def linear_cross_entropy_reference(hidden, weights, labels, bias=None, ignore_index=-100, label_smoothing=0.0):
    """Plain form (elementary operations, 32 bits or 64 for fp64): the CPU path and the oracle of the kernels."""
    rows = labels.reshape(-1)
    keep = (rows != ignore_index).nonzero().squeeze(1)
    y = rows[keep].long()
    z = _wide(hidden).reshape(-1, hidden.shape[-1])[keep] @ _wide(weights).t()
    if bias is not None:
        z = z + bias.to(z.dtype)
    V = weights.shape[0]
    lse = torch.logsumexp(z, 1)
    inside = (y >= 0) & (y < V)
    loss = lse - (1.0 - label_smoothing) * z.gather(1, y.clamp(0, V - 1).unsqueeze(1)).squeeze(1)
    if label_smoothing:
        loss = loss - (z * (label_smoothing / V)).sum(1)
    loss = loss * torch.where(inside, 1.0, math.nan)
    return torch.zeros(rows.shape[0], dtype=z.dtype, device=z.device).index_copy(0, keep, loss).reshape(labels.shape)


def _distill_rows(z, indices, teacher_logits, temperature):
    p = _teacher_weights(indices, teacher_logits, temperature, z.dtype)
    V = z.shape[1]
    z = z / temperature
    at = z.gather(1, indices.long().clamp(0, V - 1))
    at = torch.where(p != 0, at, torch.zeros_like(at))                 # a score of -inf that the teacher gives no weight
    cross = (p * (torch.logsumexp(z, 1, keepdim=True) - at)).sum(1)
    outside = ((indices >= V) & (p != 0)).any(1)
    return temperature * temperature * (torch.xlogy(p, p).sum(1) + cross) * torch.where(outside, math.nan, 1.0)


def topk_distillation_reference(logits, teacher_indices, teacher_logits, temperature=1.0):
    """Plain form of :func:`topk_distillation`."""
    K, V = teacher_indices.shape[-1], logits.shape[-1]
    z, idx, t = _wide(logits).reshape(-1, V), teacher_indices.reshape(-1, K), teacher_logits.reshape(-1, K)
    keep = ((idx >= 0) & (t != -math.inf)).any(1).nonzero().squeeze(1)
    loss = _distill_rows(z[keep], idx[keep], t[keep], temperature)
    return torch.zeros(z.shape[0], dtype=z.dtype, device=z.device).index_copy(0, keep, loss).reshape(logits.shape[:-1])


def linear_topk_distillation_reference(hidden, weights, teacher_indices, teacher_logits, bias=None, temperature=1.0):
    """Plain form of :func:`linear_topk_distillation`."""
    K = teacher_indices.shape[-1]
    idx, t = teacher_indices.reshape(-1, K), teacher_logits.reshape(-1, K)
    keep = ((idx >= 0) & (t != -math.inf)).any(1).nonzero().squeeze(1)
    z = _wide(hidden).reshape(-1, hidden.shape[-1])[keep] @ _wide(weights).t()
    if bias is not None:
        z = z + bias.to(z.dtype)
    loss = _distill_rows(z, idx[keep], t[keep], temperature)
    return torch.zeros(idx.shape[0], dtype=z.dtype, device=z.device).index_copy(0, keep, loss).reshape(hidden.shape[:-1])


# ------------------------------------------------------------------------------------------------------------------ kernel calls
def _i64(*v):
    return (ctypes.c_int64 * len(v))(*[int(x) for x in v])


def _up(n, m):
    return (n + m - 1) // m * m


def _rows16(t):
    """[R, C] with contiguous rows that start on 16 bytes and are readable in whole 16-byte chunks (zeros behind C): ``t`` itself where it
    is laid out so, else a padded copy."""
    ch = 16 // t.element_size()
    R, C = t.shape
    if t.stride(1) == 1 and C % ch == 0 and (R == 1 or (t.stride(0) % ch == 0 and t.stride(0) >= C)) and t.data_ptr() % 16 == 0:
        return t
    out = torch.zeros(R, _up(C, ch), dtype=t.dtype, device=t.device) if C % ch else torch.empty(R, C, dtype=t.dtype, device=t.device)
    out[:, :C].copy_(t)
    return out[:, :C]


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else _up(t.shape[1], 16 // t.element_size())


def _weights16(w):
    """(operand, is_dv): W [V, D] row by row, or as the rows of its [D, V] transpose where that is how it lies in memory."""
    if w.stride(1) != 1 and w.stride(0) == 1:
        return _rows16(w.t()), 1
    return _rows16(w), 0


def _label_ptrs(labels):
    return (L.ptr(labels), L.ptr(None)) if labels.dtype == torch.int64 else (L.ptr(None), L.ptr(labels))


class _Rows:
    """What both losses know about their rows: the list of those that take part, their number (on the device), and the loss' own terms."""
    __slots__ = ("N", "rows", "count", "labels", "ignore", "keep", "smooth_v", "T", "idx", "p", "psum", "ent", "mass", "zk", "cross", "K")


def _f32(n, like):
    return torch.empty(n, dtype=torch.float32, device=like.device)


def _cross_entropy_rows(labels, ignore, smoothing, V, loss):
    r = _Rows()
    r.N, r.labels, r.ignore, r.keep, r.smooth_v, r.T = labels.numel(), labels, ignore, 1.0 - smoothing, smoothing / V, 1.0
    r.idx = r.p = r.psum = r.ent = r.mass = r.zk = r.cross = None
    r.K = 0
    buf = torch.empty(r.N + 1, dtype=torch.int32, device=labels.device)
    r.rows, r.count = buf[1:], buf[:1]
    l64, l32 = _label_ptrs(labels)
    L.check(L.hip().dl4j_vl_rows(l64, l32, L.c_int64(ignore), L.ptr(None), L.c_int(r.N), L.ptr(r.rows), L.ptr(r.count), L.ptr(loss), L.stream()), "vl_rows")
    return r


def _distillation_rows(idx, t, temperature, loss):
    r = _Rows()
    N, K = idx.shape
    r.N, r.K, r.labels, r.ignore, r.keep, r.smooth_v, r.T = N, K, None, 0, 0.0, 0.0, temperature
    buf = torch.empty(N + 1, dtype=torch.int32, device=idx.device)
    r.rows, r.count, r.idx = buf[1:], buf[:1], idx
    r.p, r.psum, r.zk = _f32(N * K, idx), _f32(N * K, idx), _f32(N * K, idx)
    r.ent, r.mass, r.cross = _f32(N, idx), _f32(N, idx), _f32(N, idx)
    L.check(L.hip().dl4j_vl_teacher(L.ptr(idx), L.c_int(idx.dtype == torch.int64), L.ptr(t), L.c_int(_DT[t.dtype]), L.c_int(N), L.c_int(K),
                                    L.c_float(1.0 / temperature), L.ptr(r.p), L.ptr(r.psum), L.ptr(r.ent), L.ptr(r.mass), L.stream()), "vl_teacher")
    L.check(L.hip().dl4j_vl_rows(L.ptr(None), L.ptr(None), L.c_int64(0), L.ptr(r.mass), L.c_int(N), L.ptr(r.rows), L.ptr(r.count), L.ptr(loss), L.stream()),
            "vl_rows")
    return r


def _scores(grad, r, h, w, dv, bias, v0, v1, part=None, tz=None, zs=None, lse=None, coef=None, G=None):
    l64, l32 = _label_ptrs(r.labels) if r.labels is not None else (L.ptr(None), L.ptr(None))
    V = w.shape[1] if dv else w.shape[0]
    d = _i64(r.N, h.shape[1], V, v0, v1, _ld(h), _ld(w), G.stride(0) if G is not None else 0, _DT[h.dtype], dv, _DT[bias.dtype] if bias is not None else 0)
    f = (ctypes.c_float * 3)(1.0 / r.T, r.smooth_v, r.keep)
    L.check(L.hip().dl4j_vl_scores(L.c_int(grad), L.ptr(h), L.ptr(w), L.ptr(bias), L.ptr(r.rows), L.ptr(r.count), l64, l32, L.ptr(part), L.ptr(tz),
                                   L.ptr(zs), L.ptr(lse), L.ptr(coef), L.ptr(r.mass), L.ptr(G), d, f, L.stream()), "vl_scores")


def _forward(r, h, w, dv, bias, loss):
    V = w.shape[1] if dv else w.shape[0]
    N = r.N
    tiles = L.hip().dl4j_vl_tiles(L.c_int(V), L.c_int(_DT[h.dtype]))
    part, tz = _f32(tiles * N * 2, h), _f32(N, h)
    zs = _f32(tiles * N, h) if r.smooth_v else None
    lse = _f32(N, h)
    if r.idx is not None:
        g = _i64(N, h.shape[1], V, _ld(h), 1 if dv else _ld(w), _ld(w) if dv else 1, _DT[h.dtype], _DT[bias.dtype] if bias is not None else 0,
                 r.idx.dtype == torch.int64, r.K)
        L.check(L.hip().dl4j_vl_gather(L.ptr(h), L.ptr(w), L.ptr(bias), L.ptr(r.idx), L.ptr(r.p), L.ptr(r.rows), L.ptr(r.count), L.c_float(1.0 / r.T),
                                       L.ptr(r.zk), L.ptr(r.cross), g, L.stream()), "vl_gather")
    _scores(0, r, h, w, dv, bias, 0, V, part=part, tz=tz, zs=zs)
    l64, l32 = _label_ptrs(r.labels) if r.labels is not None else (L.ptr(None), L.ptr(None))
    L.check(L.hip().dl4j_vl_combine(L.ptr(part), L.ptr(zs), L.ptr(tz), L.ptr(r.rows), L.ptr(r.count), l64, l32, L.ptr(r.ent), L.ptr(r.cross),
                                    L.ptr(r.mass), L.c_int(N), L.c_int(V), L.c_int(tiles), L.c_float(r.keep), L.c_float(r.T), L.ptr(lse),
                                    L.ptr(loss), L.stream()), "vl_combine")
    return lse


def _pieces(V, rows, esz):
    """Column ranges of the vocabulary whose score gradients fit PIECE_BYTES, of equal size up to a tile."""
    most = max(256, PIECE_BYTES // (rows * esz) // 256 * 256)
    n = (V + most - 1) // most
    step = _up((V + n - 1) // n, 256)
    return [(a, min(V, a + step)) for a in range(0, V, step)]


def _backward(r, h, w, dv, bias, lse, dloss, shape, want_h, want_w, want_b):
    N, D, V, dt = r.N, h.shape[1], (w.shape[1] if dv else w.shape[0]), h.dtype
    dev, esz, code = h.device, h.element_size(), _DT[h.dtype]
    coef, scale = _f32(N, h), _f32(1, h)
    L.check(L.hip().dl4j_vl_coef(L.ptr(dloss), L.ptr(r.rows), L.ptr(r.count), L.c_float(r.T), L.c_int(dt == torch.float16), L.ptr(coef), L.ptr(scale),
                                 L.stream()), "vl_coef")
    Np = _up(N, 256)
    pieces = _pieces(V, Np, esz)
    G = torch.empty(Np, _up(pieces[0][1] - pieces[0][0], 256), dtype=dt, device=dev)
    dh = dw = db = packed = slab = None
    if want_w:
        Dp = _up(D, 16 // esz)
        packed = torch.empty(Np, Dp, dtype=dt, device=dev)
        L.check(L.hip().dl4j_vl_pack(L.ptr(h), L.c_int64(_ld(h) * esz), L.ptr(r.rows), L.ptr(r.count), L.ptr(packed), L.c_int64(Dp * esz), L.c_int(N),
                                     L.stream()), "vl_pack")
        dw = torch.empty((D, V) if dv else (V, D), dtype=dt, device=dev)
    if want_h:
        units = L.hip().dl4j_vl_dh_units(L.c_int(N), L.c_int(D))
        slab = _f32(units * 128 * 128, h)
        dh = torch.empty(N, D, dtype=dt, device=dev)
    if want_b:
        db = torch.empty(V, dtype=bias.dtype, device=dev)
    for k, (a, b) in enumerate(pieces):
        _scores(1, r, h, w, dv, bias, a, b, lse=lse, coef=coef, G=G)
        if r.idx is not None:
            L.check(L.hip().dl4j_vl_entries(L.ptr(r.idx), L.c_int(r.idx.dtype == torch.int64), L.c_int(r.K), L.ptr(r.p), L.ptr(r.psum), L.ptr(r.zk), L.ptr(lse),
                                            L.ptr(coef), L.ptr(r.mass), L.ptr(r.rows), L.ptr(r.count), L.c_int(N), L.c_int(a), L.c_int(b), L.ptr(G),
                                            L.c_int64(G.stride(0)), L.c_int(code), L.stream()), "vl_entries")
        if want_b:
            L.check(L.hip().dl4j_vl_colsum(L.ptr(G), L.c_int64(G.stride(0)), L.c_int(code), L.c_int(b - a), L.ptr(r.count), L.ptr(scale), L.ptr(db[a:b]),
                                           L.c_int(_DT[db.dtype]), L.stream()), "vl_colsum")
        if want_h:
            wp = w[:, a:b] if dv else w[a:b]
            L.check(L.hip().dl4j_vl_dh(L.ptr(G), L.ptr(wp), L.ptr(r.count), L.ptr(slab), _i64(N, D, b - a, G.stride(0), _ld(w), code, dv, k > 0, units),
                                       L.stream()), "vl_dh")
        if want_w:
            out = dw[:, a:b] if dv else dw[a:b]
            L.check(L.hip().dl4j_vl_dw(L.ptr(G), L.ptr(packed), L.ptr(r.count), L.ptr(scale), L.ptr(out),
                                       _i64(D, b - a, G.stride(0), packed.stride(0), dw.stride(0), code, dv), L.stream()), "vl_dw")
    if want_h:
        L.check(L.hip().dl4j_vl_dh_rows(L.ptr(slab), L.ptr(r.rows), L.ptr(r.count), L.ptr(scale), L.c_int(N), L.c_int(D), L.ptr(dh), L.c_int64(D),
                                        L.c_int(code), L.stream()), "vl_dh_rows")
        dh = dh.view(shape)
    return dh, (dw.t() if dw is not None and dv else dw), db


class _LinearLoss(torch.autograd.Function):
    """hidden [..., D], weights [V, D], bias [V] or None; the rest describes the rows (labels, or teacher entries)."""

    @staticmethod
    def forward(ctx, hidden, weights, bias, first, second, ignore, smoothing, temperature):
        h = _rows16(hidden.reshape(-1, hidden.shape[-1]))
        w, dv = _weights16(weights)
        loss = _f32(h.shape[0], h)
        if second is None:
            r = _cross_entropy_rows(first, ignore, smoothing, weights.shape[0], loss)
        else:
            r = _distillation_rows(first, second, temperature, loss)
        lse = _forward(r, h, w, dv, bias, loss)
        ctx.save_for_backward(h, w, bias, lse, first, second)
        ctx.r, ctx.dv, ctx.shape = r, dv, hidden.shape
        return loss.view(hidden.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        h, w, bias, lse, _, _ = ctx.saved_tensors
        with torch.cuda.device(h.device):
            g = dloss.reshape(-1)
            g = g if g.dtype == torch.float32 and g.is_contiguous() else g.float().contiguous()
            dh, dw, db = _backward(ctx.r, h, w, ctx.dv, bias, lse, g, ctx.shape, *ctx.needs_input_grad[:3])
        return dh, dw, db, None, None, None, None, None


class _TopkDistillation(torch.autograd.Function):
    CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

    @staticmethod
    def forward(ctx, logits, idx, t, temperature):
        z = logits.reshape(-1, logits.shape[-1])
        z = z if z.stride(1) == 1 and z.stride(0) >= z.shape[1] else z.contiguous()
        loss, lse = _f32(z.shape[0], z), _f32(z.shape[0], z)
        c = _TopkDistillation.CODE
        L.check(L.hip().dl4j_topk_distill_fwd(L.ptr(z), L.c_int64(z.stride(0)), L.ptr(idx), L.c_int(idx.dtype == torch.int64), L.ptr(t), L.c_int(c[t.dtype]),
                                              L.c_int(z.shape[0]), L.c_int(z.shape[1]), L.c_int(idx.shape[1]), L.c_int(c[z.dtype]),
                                              L.c_float(temperature), L.ptr(loss), L.ptr(lse), L.stream()), "topk_distill_fwd")
        ctx.save_for_backward(z, idx, t, lse)
        ctx.temperature, ctx.shape = temperature, logits.shape
        return loss.view(logits.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        z, idx, t, lse = ctx.saved_tensors
        c = _TopkDistillation.CODE
        with torch.cuda.device(z.device):
            g = dloss.reshape(-1)
            g = g if g.dtype == torch.float32 and g.is_contiguous() else g.float().contiguous()
            dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
            L.check(L.hip().dl4j_topk_distill_bwd(L.ptr(z), L.c_int64(z.stride(0)), L.ptr(idx), L.c_int(idx.dtype == torch.int64), L.ptr(t),
                                                  L.c_int(c[t.dtype]), L.c_int(z.shape[0]), L.c_int(z.shape[1]), L.c_int(idx.shape[1]),
                                                  L.c_int(c[z.dtype]), L.c_float(ctx.temperature), L.ptr(lse), L.ptr(g), L.ptr(dz), L.stream()),
                    "topk_distill_bwd")
        return dz.view(ctx.shape), None, None, None


# ------------------------------------------------------------------------------------------------------------------ entry points
def usable(operand, *others):
    """True where the kernels take the call (GPU operands in bf16 / fp16 / fp32, at least one row); else the plain form does."""
    if not L.use_hip(operand, *others) or operand.dtype not in _DT or operand.numel() == 0:
        return False
    _need(operand.numel() // operand.shape[-1] < 2 ** 31 - 512, "more than 2^31 rows")
    return True


def _teacher_operands(indices, logits):
    K = indices.shape[-1]
    t = logits.detach()
    t = t.float() if t.dtype not in _DT else t
    return indices.reshape(-1, K).contiguous(), t.reshape(-1, K).contiguous()


def linear_cross_entropy(hidden, weights, labels, bias=None, ignore_index=-100, label_smoothing=0.0):
    """Softmax cross entropy of the logits ``hidden . weights^T + bias`` against integer labels, without keeping the logits.

    hidden [..., D]; weights [V, D] in hidden's type (an embedding table, or ``w.t()`` of a dense layer's [nIn, nOut] weights: both layouts
    are read in place); labels [...] INT32 / INT64; bias [V]. Rows whose label is ``ignore_index`` have loss 0, take no part in any product
    and get no gradient, whatever their hidden states hold. A row with another label outside [0, V) has loss and gradients NaN.
    Returns the rows' losses (fp32; fp64 for fp64 operands). Differentiable in hidden, weights and bias.

    16-bit operands: scores, softmax and all sums in fp32, the scores' gradient is rounded to the operands' type for the two gradient
    products (fp16: scaled to its range first)."""
    name = "linear_cross_entropy"
    _check_linear(hidden, weights, bias, name)
    _need(labels.dtype in (torch.int32, torch.int64), "%s: labels must be INT32 or INT64" % name)
    _need(labels.shape == hidden.shape[:-1], "%s: labels %s must have the shape of hidden's rows %s" % (name, list(labels.shape), list(hidden.shape[:-1])))
    _need(labels.device == hidden.device, "%s: labels are on another device" % name)
    _need(0.0 <= label_smoothing < 1.0, "%s: label smoothing must be in [0, 1)" % name)
    if not usable(hidden, weights, labels, bias):
        return linear_cross_entropy_reference(hidden, weights, labels, bias, ignore_index, label_smoothing)
    with torch.cuda.device(hidden.device):
        return _LinearLoss.apply(hidden, weights, None if bias is None else bias.contiguous(), labels.reshape(-1).contiguous(), None, int(ignore_index),
                                 float(label_smoothing), 1.0)


def linear_topk_distillation(hidden, weights, teacher_indices, teacher_logits, bias=None, temperature=1.0):
    """Distillation from a teacher's top logits: T^2 KL(softmax(teacher_logits / T) || softmax(z / T)) per row for the student's logits
    ``z = hidden . weights^T + bias``, which are not kept.

    teacher_indices [..., K] INT32 / INT64 and teacher_logits [..., K] name the teacher's K best words of every row in any order; the
    teacher's softmax runs over them alone. Entries with a negative index are padding; a logit of -inf counts as none; an index that comes
    twice counts twice. A row without entries has loss 0 and no gradient. A row with an index >= V, or a teacher logit that is NaN or +inf,
    has loss and gradients NaN. No gradient goes to the teacher. Other arguments, types and result as :func:`linear_cross_entropy`."""
    name = "linear_topk_distillation"
    _check_linear(hidden, weights, bias, name)
    _check_teacher(hidden.shape[:-1], hidden.device, teacher_indices, teacher_logits, temperature, name)
    if not usable(hidden, weights, teacher_indices, teacher_logits, bias):
        return linear_topk_distillation_reference(hidden, weights, teacher_indices, teacher_logits, bias, temperature)
    with torch.cuda.device(hidden.device):
        idx, t = _teacher_operands(teacher_indices, teacher_logits)
        return _LinearLoss.apply(hidden, weights, None if bias is None else bias.contiguous(), idx, t, 0, 0.0, float(temperature))


def topk_distillation(logits, teacher_indices, teacher_logits, temperature=1.0):
    """:func:`linear_topk_distillation` for a student whose logits [..., V] are there already. Differentiable in the logits."""
    name = "topk_distillation"
    _need(logits.dim() >= 1 and _floating(logits) and logits.shape[-1] > 0, "%s: logits must be a floating point tensor [..., V]" % name)
    _check_teacher(logits.shape[:-1], logits.device, teacher_indices, teacher_logits, temperature, name)
    if not usable(logits, teacher_indices, teacher_logits):
        return topk_distillation_reference(logits, teacher_indices, teacher_logits, temperature)
    with torch.cuda.device(logits.device):
        idx, t = _teacher_operands(teacher_indices, teacher_logits)
        return _TopkDistillation.apply(logits, idx, t, float(temperature))
