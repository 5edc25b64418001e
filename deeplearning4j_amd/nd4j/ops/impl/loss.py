"""GENERATED by deeplearning4j_amd.codegen from codegen/ops/loss.py -- do not edit; change the definition and run
``python -m deeplearning4j_amd.codegen``. (Reference counterpart: the generated nd4j-api linalg/api/ops/impl/** classes used by NDLoss / SDLoss.)"""
from __future__ import annotations

import torch

from . import _core as _b
from ._core import _t


def _dims(d):
    return list(d[0]) if len(d) == 1 and isinstance(d[0], (list, tuple)) else list(d)


class AbsoluteDifference(_b.GeneratedCustomOp):
    """Absolute difference loss: sum_i |label_i - predictions_i|.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'absolute_difference_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', outputs=None):
        super().__init__('absolute_difference_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])


class CosineDistance(_b.GeneratedCustomOp):
    """Cosine distance loss: 1 - sum(label * predictions) along a dimension (inputs are expected normalised).
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param dimension: Dimension along which the cosine distance is taken (INT, default -1)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'cosine_distance_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', dimension=-1, outputs=None):
        super().__init__('cosine_distance_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce), dimension])


class HingeLoss(_b.GeneratedCustomOp):
    """Hinge loss: max(0, 1 - t * predictions) with t = 2 * label - 1.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'hinge_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', outputs=None):
        super().__init__('hinge_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])


class HuberLoss(_b.GeneratedCustomOp):
    """Huber loss: quadratic below delta, linear above.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param delta: Switch point between the quadratic and the linear part (FLOATING_POINT, default 1.0)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'huber_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', delta=1.0, outputs=None):
        super().__init__('huber_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[delta])


class LogLoss(_b.GeneratedCustomOp):
    """Binary cross entropy on probabilities.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param epsilon: Added inside the logarithms (FLOATING_POINT, default 1e-07)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'log_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', epsilon=1e-07, outputs=None):
        super().__init__('log_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[epsilon])


class LogPoisson(_b.GeneratedCustomOp):
    """Log-Poisson loss: exp(predictions) - label * predictions (+ Stirling term when full).
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param full: Add the Stirling approximation term (BOOL, default False)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'log_poisson_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', full=False, outputs=None):
        super().__init__('log_poisson_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce), int(full)])


class MeanPairwiseSquaredError(_b.GeneratedCustomOp):
    """Mean pairwise squared error over all pairs of elements of an example.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'mean_pairwssqerr_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', outputs=None):
        super().__init__('mean_pairwssqerr_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])


class MeanSquaredError(_b.GeneratedCustomOp):
    """Mean squared error.
    :param label: Label array (NUMERIC)
    :param predictions: Predictions (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'mean_sqerr_loss', 'loss', 1

    def __init__(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', outputs=None):
        super().__init__('mean_sqerr_loss', [_t(v) for v in [predictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])


class SigmoidCrossEntropy(_b.GeneratedCustomOp):
    """Sigmoid cross entropy on logits, with optional label smoothing.
    :param label: Label array (NUMERIC)
    :param predictionLogits: Logits (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param labelSmoothing: Label smoothing factor (FLOATING_POINT, default 0.0)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'sigm_cross_entropy_loss', 'loss', 1

    def __init__(self, label, predictionLogits, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', labelSmoothing=0.0, outputs=None):
        super().__init__('sigm_cross_entropy_loss', [_t(v) for v in [predictionLogits, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[labelSmoothing])


class SoftmaxCrossEntropy(_b.GeneratedCustomOp):
    """Softmax cross entropy on logits against one-hot labels.
    :param label: Label array (NUMERIC)
    :param logitPredictions: Logits (NUMERIC)
    :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
    :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
    :param labelSmoothing: Label smoothing factor (FLOATING_POINT, default 0.0)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'softmax_cross_entropy_loss', 'loss', 1

    def __init__(self, label, logitPredictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', labelSmoothing=0.0, outputs=None):
        super().__init__('softmax_cross_entropy_loss', [_t(v) for v in [logitPredictions, (weights if weights is not None else torch.tensor(1.0)), label]], outputs, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[labelSmoothing])


class SparseSoftmaxCrossEntropy(_b.GeneratedCustomOp):
    """Softmax cross entropy against integer class labels.
    :param logits: Logits [..., nClasses] (NUMERIC)
    :param labels: Class indices [...] (INT)
    :return output: Per-example loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'sparse_softmax_cross_entropy_loss_with_logits', 'loss', 1

    def __init__(self, logits, labels, outputs=None):
        super().__init__('sparse_softmax_cross_entropy_loss_with_logits', [_t(v) for v in [labels, logits]], outputs)


class LinearSoftmaxCrossEntropy(_b.GeneratedCustomOp):
    """Softmax cross entropy of the logits hidden . weights^T + bias against integer class labels; the logits are not kept.
    :param hidden: Hidden states [..., D] (FLOATING_POINT)
    :param weights: Output weights [V, D] (an embedding table), or [D, V] with transposeWeights, in the type of hidden (FLOATING_POINT)
    :param labels: Class indices [...]; a row labelled ignoreIndex has loss 0 and no gradient, one labelled otherwise outside [0, V) gives NaN (INT)
    :param bias: Output bias [V] (FLOATING_POINT, optional)
    :param labelSmoothing: Label smoothing factor in [0, 1) (FLOATING_POINT, default 0.0)
    :param ignoreIndex: Label of the rows that take no part (INT, default -100)
    :param transposeWeights: Weights are [D, V], as a dense layer holds them (BOOL, default False)
    :return output: Per-row loss [...], FLOAT (DOUBLE for DOUBLE operands) (FLOATING_POINT)
    """
    OP, NAMESPACE, N_OUT = 'linear_softmax_cross_entropy_loss', 'loss', 1

    def __init__(self, hidden, weights, labels, bias=None, labelSmoothing=0.0, ignoreIndex=-100, transposeWeights=False, outputs=None):
        super().__init__('linear_softmax_cross_entropy_loss', [_t(v) for v in [hidden, weights, labels] + ([bias] if bias is not None else [])], outputs, iArgs=[ignoreIndex, int(transposeWeights)], tArgs=[labelSmoothing])


class LinearTopKDistillation(_b.GeneratedCustomOp):
    """Distillation from a teacher's top logits, T^2 KL(softmax(teacher / T) || softmax(student / T)), for student logits hidden . weights^T + bias that are not kept.
    :param hidden: Hidden states [..., D] (FLOATING_POINT)
    :param weights: Output weights [V, D], or [D, V] with transposeWeights (FLOATING_POINT)
    :param teacherIndices: Words of the teacher's K best logits [..., K], negative: padding (INT)
    :param teacherLogits: Their logits [..., K] (FLOATING_POINT)
    :param bias: Output bias [V] (FLOATING_POINT, optional)
    :param temperature: Temperature T (FLOATING_POINT, default 1.0)
    :param transposeWeights: Weights are [D, V], as a dense layer holds them (BOOL, default False)
    :return output: Per-row loss [...] (FLOATING_POINT)
    """
    OP, NAMESPACE, N_OUT = 'linear_topk_distillation_loss', 'loss', 1

    def __init__(self, hidden, weights, teacherIndices, teacherLogits, bias=None, temperature=1.0, transposeWeights=False, outputs=None):
        super().__init__('linear_topk_distillation_loss', [_t(v) for v in [hidden, weights, teacherIndices, teacherLogits] + ([bias] if bias is not None else [])], outputs, iArgs=[int(transposeWeights)], tArgs=[temperature])


class TopKDistillation(_b.GeneratedCustomOp):
    """Distillation from a teacher's top logits, T^2 KL(softmax(teacher / T) || softmax(student / T)), on student logits.
    :param logits: Student logits [..., V] (FLOATING_POINT)
    :param teacherIndices: Words of the teacher's K best logits [..., K], negative: padding (INT)
    :param teacherLogits: Their logits [..., K] (FLOATING_POINT)
    :param temperature: Temperature T (FLOATING_POINT, default 1.0)
    :return output: Per-row loss [...] (FLOATING_POINT)
    """
    OP, NAMESPACE, N_OUT = 'topk_distillation_loss', 'loss', 1

    def __init__(self, logits, teacherIndices, teacherLogits, temperature=1.0, outputs=None):
        super().__init__('topk_distillation_loss', [_t(v) for v in [logits, teacherIndices, teacherLogits]], outputs, tArgs=[temperature])


class L2Loss(_b.GeneratedCustomOp):
    """Half the sum of squares: sum(x^2) / 2.
    :param var: Input (NUMERIC)
    :return output: Scalar loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'l2_loss', 'loss', 1

    def __init__(self, var, outputs=None):
        super().__init__('l2_loss', [_t(v) for v in [var]], outputs)


class CtcLoss(_b.GeneratedCustomOp):
    """Connectionist temporal classification loss.
    :param targetLabels: Label sequences [batch, maxLabelLength] (INT)
    :param logitInput: Logits [batch, time, nClasses] (NUMERIC)
    :param targetLabelLengths: Label lengths [batch] (INT)
    :param logitInputLengths: Logit sequence lengths [batch] (INT)
    :param blankIndex: Index of the blank class (INT, default 0)
    :return output: Per-example loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'ctc_loss', 'loss', 1

    def __init__(self, targetLabels, logitInput, targetLabelLengths, logitInputLengths, blankIndex=0, outputs=None):
        super().__init__('ctc_loss', [_t(v) for v in [targetLabels, logitInput, targetLabelLengths, logitInputLengths]], outputs, iArgs=[blankIndex])


class WeightedCrossEntropyWithLogits(_b.GeneratedCustomOp):
    """Sigmoid cross entropy with a weight on the positive term.
    :param targets: Targets (NUMERIC)
    :param inputs: Logits (NUMERIC)
    :param weights: Positive-class weights (NUMERIC)
    :return output: Loss (NUMERIC)
    """
    OP, NAMESPACE, N_OUT = 'weighted_cross_entropy_with_logits', 'loss', 1

    def __init__(self, targets, inputs, weights, outputs=None):
        super().__init__('weighted_cross_entropy_with_logits', [_t(v) for v in [targets, inputs, weights]], outputs)


CLASSES = (AbsoluteDifference, CosineDistance, HingeLoss, HuberLoss, LogLoss, LogPoisson, MeanPairwiseSquaredError, MeanSquaredError, SigmoidCrossEntropy, SoftmaxCrossEntropy, SparseSoftmaxCrossEntropy, LinearSoftmaxCrossEntropy, LinearTopKDistillation, TopKDistillation, L2Loss, CtcLoss, WeightedCrossEntropyWithLogits, )
