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
import threading

import torch
from torch.autograd.function import once_differentiable

from ..native import lib as L
from ..nd4j.exceptions import ND4JIllegalArgumentException

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}      # operand codes of the GEMM core
MAX_TEACHER = 1024                                                  # entries per row the kernels keep on chip


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
    outside = ((indices >= V) & (teacher_logits.detach() != -math.inf)).any(1)
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
# the fields of struct Args in native/csrc/vocab_loss.hip, in order
_ARGS = ("N D V dt split wt bdt ldh ldw lab64 ignore idx64 tdt K want_h want_w want_b pad_h pad_w "
         "H W bias labels idx t loss state ws dloss dh dw db").split()
_AT = {n: k for k, n in enumerate(_ARGS)}
_Block = ctypes.c_int64 * len(_ARGS)
_Floats = ctypes.c_float * 2
_Sizes = ctypes.c_int64 * 3
_STATE, _WS = _AT["state"], _AT["ws"]
_H, _W, _BIAS, _LDH, _LDW, _SPLIT, _PAD_H, _PAD_W = (_AT[n] for n in "H W bias ldh ldw split pad_h pad_w".split())
# struct DistillArgs in native/csrc/topk_distill.hip: N V K ldz dt idx64 tdt z idx t loss lse dloss dz
_TopkBlock = ctypes.c_int64 * 14


def _up(n, m):
    return (n + m - 1) // m * m


def _rows(t):
    """[R, C] with contiguous rows, ``t`` itself where they are. (Rows that do not start or end on 16 bytes are copied by the native call.)"""
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _ld(t):
    """From one row of ``_rows(t)`` to the next; the stride of a single row says nothing."""
    return t.stride(0) if t.shape[0] > 1 else _up(t.shape[1], 16 // t.element_size())


def _split(rows, hidden, vocabulary, training):
    """fp32 operands as pairs of halves on the 16-bit matrix cores: three products there take a quarter of one on the fp32 cores, once the rows
    pay for the conversion of the weights (12 bytes an element) and the call for its two launches. Step of 96 rows x 768 against 30522 words:
    261 us in fp32, 204 us in halves, of 40 rows: 186 and 189 us; 64 rows x 512 against 8000 words: 147 and 152 us; one forward of 512 rows x 768
    against 30522 words: 221 and 121 us, of 128 rows: 74 and 91 us."""
    work = hidden * vocabulary
    return (rows - 40) * work > 150e6 if training else (rows - 150) * work > 600e6


def _as_before(t, ld, any_start):
    """``t``, or its values with rows ``ld`` apart and on 16 bytes (unless any start will do). Saved tensors come back from hooks (recomputation,
    offload) in other memory, and the forward call's choices hold for its own row distance and alignment."""
    if (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] == 1 or t.stride(0) == ld) and (any_start or t.data_ptr() % 16 == 0):
        return t
    return torch.empty_strided(t.shape, (ld, 1), dtype=t.dtype, device=t.device).copy_(t)


def _launch(fn, what, dev, *args):
    """One native call on the current stream of ``dev``, with ``dev`` as the current device."""
    if dev.index == torch.cuda.current_device():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if code:
        L.check(code, what)


_LIB, _LOCK = None, threading.Lock()


def _lib():
    """The kernel library with the calls' signatures declared, for every thread alike."""
    global _LIB
    if _LIB is None:
        with _LOCK:
            if _LIB is None:
                lib = L.hip()
                for fn in (lib.dl4j_linear_loss_fwd, lib.dl4j_linear_loss_bwd, lib.dl4j_topk_distill):
                    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
                lib.dl4j_linear_loss_bytes.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
                _LIB = lib
    return _LIB


def _dloss(g):
    g = g.reshape(-1)
    return g if g.dtype == torch.float32 and g.is_contiguous() else g.float().contiguous()


def _linear_forward(hidden, weights, bias, first, second, ignore, smoothing, temperature, want=(False, False, False)):
    """(loss, what the backward pass needs: tensors, call) - the latter None where no gradient is wanted."""
    lib = _lib()
    h = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    dv = weights.stride(1) != 1 and weights.stride(0) == 1              # [V, D] row by row, or as the rows of its [D, V] transpose
    w = weights.t() if dv else weights
    training = any(want)
    N, D = h.shape
    split = h.dtype == torch.float32 and _split(N, D, weights.shape[0], training)
    h, w = _rows(h), _rows(w)
    dev = h.device
    loss = torch.empty(hidden.shape[:-1], dtype=torch.float32, device=dev)
    teacher = second is not None
    is64, at = first.dtype == torch.int64, first.data_ptr()
    a = _Block(N, D, weights.shape[0], _DT[h.dtype], split, dv, 0 if bias is None else _DT[bias.dtype], _ld(h), _ld(w), is64, ignore, is64,
               _DT[second.dtype] if teacher else 0, first.shape[1] if teacher else 0, *want, 0, 0,
               h.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if teacher else at, at if teacher else 0,
               second.data_ptr() if teacher else 0, loss.data_ptr(), 0, 0, 0, 0, 0, 0)
    f = _Floats(temperature, smoothing)
    size = _Sizes()
    lib.dl4j_linear_loss_bytes(a, size)
    if training:
        state, ws = torch.empty(size[0], dtype=torch.uint8, device=dev), torch.empty(size[1], dtype=torch.uint8, device=dev)
        a[_STATE], a[_WS] = state.data_ptr(), ws.data_ptr()
    else:
        both = torch.empty(size[0] + size[1], dtype=torch.uint8, device=dev)
        a[_STATE] = both.data_ptr()
        a[_WS] = a[_STATE] + size[0]
    _launch(lib.dl4j_linear_loss_fwd, "linear_loss_fwd", dev, a, f)
    return loss, ((h, w, state), (a, f, size[0], size[2], dv)) if training else None


class _LinearLoss(torch.autograd.Function):
    """hidden [..., D], weights [V, D], bias [V] or None; first / second: labels and None, or the teacher's indices and logits."""

    @staticmethod
    def forward(ctx, hidden, weights, bias, first, second, ignore, smoothing, temperature):
        loss, ((h, w, state), call) = _linear_forward(hidden, weights, bias, first, second, ignore, smoothing, temperature, ctx.needs_input_grad[:3])
        ctx.save_for_backward(h, w, bias, state)                       # (labels and teacher are in the state: their tensors may change)
        ctx.call, ctx.shape = call, hidden.shape
        return loss

    @staticmethod
    def apply_or_run(hidden, weights, bias, *rest):
        if torch.is_grad_enabled() and (hidden.requires_grad or weights.requires_grad or (bias is not None and bias.requires_grad)):
            return _LinearLoss.apply(hidden, weights, bias, *rest)
        return _linear_forward(hidden, weights, bias, *rest)[0]

    @staticmethod
    def backward(ctx, dloss):
        return _once(_linear_backward, ctx, dloss) if torch.is_grad_enabled() else _linear_backward(ctx, dloss)


def _linear_backward(ctx, dloss):
    h, w, bias, state = ctx.saved_tensors                               # (the forward call's own, or what hooks make of them)
    a, f, state_size, size, dv = ctx.call
    a = _Block.from_buffer_copy(a)                                      # (a graph kept alive may be walked from two threads)
    _need(state.numel() == state_size, "linear loss: the saved state is another call's (%d bytes for %d)" % (state.numel(), state_size))
    split = a[_SPLIT]
    h, w = _as_before(h, a[_LDH], split or a[_PAD_H]), _as_before(w, a[_LDW], split or a[_PAD_W])
    a[_H], a[_W] = h.data_ptr(), w.data_ptr()
    if bias is not None:
        bias = bias.contiguous()
        a[_BIAS] = bias.data_ptr()
    dev = h.device
    g = _dloss(dloss)
    want_h, want_w, want_b = ctx.needs_input_grad[:3]
    dh = torch.empty(ctx.shape, dtype=h.dtype, device=dev) if want_h else None
    dw = torch.empty(w.shape, dtype=h.dtype, device=dev) if want_w else None
    db = torch.empty_like(bias) if want_b else None
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    for name, t in (("state", state), ("ws", ws), ("dloss", g), ("dh", dh), ("dw", dw), ("db", db)):
        if t is not None:
            a[_AT[name]] = t.data_ptr()
    _launch(_lib().dl4j_linear_loss_bwd, "linear_loss_bwd", dev, a, f)
    return dh, (dw.t() if want_w and dv else dw), db, None, None, None, None, None


def _once(fn, ctx, dloss):
    """``fn`` where the caller asked for a graph of the gradients: differentiating them raises."""
    class Once:
        call = once_differentiable(lambda c, g: fn(c, g))
    return Once.call(ctx, dloss)


_TOPK_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _topk_forward(logits, idx, t, temperature):
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    z = _rows(z)
    N, dev = z.shape[0], z.device
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    lse = torch.empty(N, dtype=torch.float32, device=dev)
    a = _TopkBlock(N, z.shape[1], idx.shape[1], _ld(z), _TOPK_DT[z.dtype], idx.dtype == torch.int64, _TOPK_DT[t.dtype], z.data_ptr(), idx.data_ptr(),
                   t.data_ptr(), loss.data_ptr(), lse.data_ptr(), 0, 0)
    f = _Floats(temperature, 0.0)
    _launch(_lib().dl4j_topk_distill, "topk_distill", dev, a, f)
    return loss, z, lse, (a, f)


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, t, temperature):
        loss, z, lse, ctx.call = _topk_forward(logits, idx, t, temperature)
        ctx.save_for_backward(z, idx, t, lse)
        ctx.shape = logits.shape
        return loss

    @staticmethod
    def backward(ctx, dloss):
        return _once(_topk_backward, ctx, dloss) if torch.is_grad_enabled() else _topk_backward(ctx, dloss)


def _topk_backward(ctx, dloss):
    z, idx, t, lse = ctx.saved_tensors                                  # (the forward call's own, or what hooks make of them)
    z, idx, t, lse = _rows(z), idx.contiguous(), t.contiguous(), lse.contiguous()
    a, f = ctx.call
    a = _TopkBlock.from_buffer_copy(a)
    g = _dloss(dloss)
    dz = torch.empty(ctx.shape, dtype=z.dtype, device=z.device)
    a[3], a[7], a[8], a[9], a[11] = _ld(z), z.data_ptr(), idx.data_ptr(), t.data_ptr(), lse.data_ptr()
    a[10], a[12], a[13] = 0, g.data_ptr(), dz.data_ptr()
    _launch(_lib().dl4j_topk_distill, "topk_distill", z.device, a, f)
    return dz, None, None, None


# ------------------------------------------------------------------------------------------------------------------ entry points
def usable(operand, *others):
    """True where the kernels take the call (GPU operands in bf16 / fp16 / fp32, at least one row); else the plain form does."""
    if not L.use_hip(operand, *others) or operand.dtype not in _DT or operand.numel() == 0:
        return False
    _need(operand.numel() // operand.shape[-1] < 2 ** 31 - 512, "more than 2^31 rows")
    return True


def _teacher_operands(indices, logits):
    K = indices.shape[-1]
    t = logits.detach() if logits.requires_grad else logits
    t = t.float() if t.dtype not in _DT else t
    if t.dim() != 2:
        indices, t = indices.reshape(-1, K), t.reshape(-1, K)
    return indices.contiguous(), t.contiguous()


def linear_cross_entropy(hidden, weights, labels, bias=None, ignore_index=-100, label_smoothing=0.0, plain=False):
    """Softmax cross entropy of the logits ``hidden . weights^T + bias`` against integer labels, without keeping the logits.

    hidden [..., D]; weights [V, D] in hidden's type (an embedding table, or ``w.t()`` of a dense layer's [nIn, nOut] weights: both layouts
    are read in place); labels [...] INT32 / INT64; bias [V]. Rows whose label is ``ignore_index`` have loss 0, take no part in any product
    and get no gradient, whatever their hidden states hold. A row with another label outside [0, V) has loss and gradients NaN.
    Returns the rows' losses (fp32; fp64 for fp64 operands). Differentiable in hidden, weights and bias.

    16-bit operands: scores, softmax and all sums in fp32, the scores' gradient is rounded to the operands' type for the two gradient
    products (fp16: scaled to its range first; up to 256 rows it is kept in two halves). fp32 operands may run as scaled pairs of fp16 halves, which
    hold 2^-24 of a value, or 2^-40 of the largest value of the row of hidden states, of the words within 2^8 of the largest one, of the row's
    gradient. ``plain``: the plain form, whatever the operands."""
    name = "linear_cross_entropy"
    _check_linear(hidden, weights, bias, name)
    _need(labels.dtype in (torch.int32, torch.int64), "%s: labels must be INT32 or INT64" % name)
    _need(labels.shape == hidden.shape[:-1], "%s: labels %s must have the shape of hidden's rows %s" % (name, list(labels.shape), list(hidden.shape[:-1])))
    _need(labels.device == hidden.device, "%s: labels are on another device" % name)
    _need(0.0 <= label_smoothing < 1.0, "%s: label smoothing must be in [0, 1)" % name)
    if plain or not usable(hidden, weights, labels, bias):
        return linear_cross_entropy_reference(hidden, weights, labels, bias, ignore_index, label_smoothing)
    return _LinearLoss.apply_or_run(hidden, weights, None if bias is None else bias.contiguous(), labels.reshape(-1).contiguous(), None,
                                    int(ignore_index), float(label_smoothing), 1.0)


def linear_topk_distillation(hidden, weights, teacher_indices, teacher_logits, bias=None, temperature=1.0, plain=False):
    """Distillation from a teacher's top logits: T^2 KL(softmax(teacher_logits / T) || softmax(z / T)) per row for the student's logits
    ``z = hidden . weights^T + bias``, which are not kept.

    teacher_indices [..., K] INT32 / INT64 and teacher_logits [..., K] name the teacher's K best words of every row in any order; the
    teacher's softmax runs over them alone. Entries with a negative index are padding; a logit of -inf counts as none; an index that comes
    twice counts twice. A row without entries has loss 0 and no gradient. A row with an index >= V, or a teacher logit that is NaN or +inf,
    has loss and gradients NaN, however little the teacher gives it. No gradient goes to the teacher. Other arguments, types and result as :func:`linear_cross_entropy`."""
    name = "linear_topk_distillation"
    _check_linear(hidden, weights, bias, name)
    _check_teacher(hidden.shape[:-1], hidden.device, teacher_indices, teacher_logits, temperature, name)
    if plain or not usable(hidden, weights, teacher_indices, teacher_logits, bias):
        return linear_topk_distillation_reference(hidden, weights, teacher_indices, teacher_logits, bias, temperature)
    idx, t = _teacher_operands(teacher_indices, teacher_logits)
    return _LinearLoss.apply_or_run(hidden, weights, None if bias is None else bias.contiguous(), idx, t, 0, 0.0, float(temperature))


def topk_distillation(logits, teacher_indices, teacher_logits, temperature=1.0, plain=False):
    """:func:`linear_topk_distillation` for a student whose logits [..., V] are there already. Differentiable in the logits."""
    name = "topk_distillation"
    _need(logits.dim() >= 1 and _floating(logits) and logits.shape[-1] > 0, "%s: logits must be a floating point tensor [..., V]" % name)
    _check_teacher(logits.shape[:-1], logits.device, teacher_indices, teacher_logits, temperature, name)
    if plain or not usable(logits, teacher_indices, teacher_logits):
        return topk_distillation_reference(logits, teacher_indices, teacher_logits, temperature)
    idx, t = _teacher_operands(teacher_indices, teacher_logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TopkDistillation.apply(logits, idx, t, float(temperature))
    return _topk_forward(logits, idx, t, float(temperature))[0]
