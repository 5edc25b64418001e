"""GENERATED by deeplearning4j_amd.codegen from codegen/ops/loss.py -- do not edit; change the definition and run
``python -m deeplearning4j_amd.codegen``. (Reference counterpart: the generated nd4j-api autodiff/samediff/ops/SDLoss.java.)"""
from __future__ import annotations

def _dims(d):
    return list(d[0]) if len(d) == 1 and isinstance(d[0], (list, tuple)) else list(d)


class GenSDLoss:
    """Loss functions. Every weighted loss takes optional broadcastable weights (default 1.0) and a reduction mode.

    Mixin: the concrete namespace class provides ``self.sd`` and ``self._o(opName, inputs, name, nOut, **argVectors)``."""

    def absoluteDifference(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', name=None):
        """Absolute difference loss: sum_i |label_i - predictions_i|.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :return output: Loss (NUMERIC)
        """
        return self._o('absolute_difference_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])

    def cosineDistance(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', dimension=-1, name=None):
        """Cosine distance loss: 1 - sum(label * predictions) along a dimension (inputs are expected normalised).
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param dimension: Dimension along which the cosine distance is taken (INT, default -1)
        :return output: Loss (NUMERIC)
        """
        return self._o('cosine_distance_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce), dimension])

    def hingeLoss(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', name=None):
        """Hinge loss: max(0, 1 - t * predictions) with t = 2 * label - 1.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :return output: Loss (NUMERIC)
        """
        return self._o('hinge_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])

    def huberLoss(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', delta=1.0, name=None):
        """Huber loss: quadratic below delta, linear above.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param delta: Switch point between the quadratic and the linear part (FLOATING_POINT, default 1.0)
        :return output: Loss (NUMERIC)
        """
        return self._o('huber_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[delta])

    def logLoss(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', epsilon=1e-07, name=None):
        """Binary cross entropy on probabilities.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param epsilon: Added inside the logarithms (FLOATING_POINT, default 1e-07)
        :return output: Loss (NUMERIC)
        """
        return self._o('log_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[epsilon])

    def logPoisson(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', full=False, name=None):
        """Log-Poisson loss: exp(predictions) - label * predictions (+ Stirling term when full).
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param full: Add the Stirling approximation term (BOOL, default False)
        :return output: Loss (NUMERIC)
        """
        return self._o('log_poisson_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce), int(full)])

    def meanPairwiseSquaredError(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', name=None):
        """Mean pairwise squared error over all pairs of elements of an example.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :return output: Loss (NUMERIC)
        """
        return self._o('mean_pairwssqerr_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])

    def meanSquaredError(self, label, predictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', name=None):
        """Mean squared error.
        :param label: Label array (NUMERIC)
        :param predictions: Predictions (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :return output: Loss (NUMERIC)
        """
        return self._o('mean_sqerr_loss', [predictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)])

    def sigmoidCrossEntropy(self, label, predictionLogits, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', labelSmoothing=0.0, name=None):
        """Sigmoid cross entropy on logits, with optional label smoothing.
        :param label: Label array (NUMERIC)
        :param predictionLogits: Logits (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param labelSmoothing: Label smoothing factor (FLOATING_POINT, default 0.0)
        :return output: Loss (NUMERIC)
        """
        return self._o('sigm_cross_entropy_loss', [predictionLogits, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[labelSmoothing])

    def softmaxCrossEntropy(self, label, logitPredictions, weights=None, lossReduce='MEAN_BY_NONZERO_WEIGHT_COUNT', labelSmoothing=0.0, name=None):
        """Softmax cross entropy on logits against one-hot labels.
        :param label: Label array (NUMERIC)
        :param logitPredictions: Logits (NUMERIC)
        :param weights: Weights, broadcastable to the loss shape (NUMERIC, optional)
        :param lossReduce: Reduction of the per-example losses (ENUM, one of NONE/SUM/MEAN_BY_WEIGHT/MEAN_BY_NONZERO_WEIGHT_COUNT, default 'MEAN_BY_NONZERO_WEIGHT_COUNT')
        :param labelSmoothing: Label smoothing factor (FLOATING_POINT, default 0.0)
        :return output: Loss (NUMERIC)
        """
        return self._o('softmax_cross_entropy_loss', [logitPredictions, (weights if weights is not None else self.sd.constant(None, 1.0)), label], name, 1, iArgs=[['NONE', 'SUM', 'MEAN_BY_WEIGHT', 'MEAN_BY_NONZERO_WEIGHT_COUNT'].index(lossReduce) if isinstance(lossReduce, str) else int(lossReduce)], tArgs=[labelSmoothing])

    def sparseSoftmaxCrossEntropy(self, logits, labels, name=None):
        """Softmax cross entropy against integer class labels.
        :param logits: Logits [..., nClasses] (NUMERIC)
        :param labels: Class indices [...] (INT)
        :return output: Per-example loss (NUMERIC)
        """
        return self._o('sparse_softmax_cross_entropy_loss_with_logits', [labels, logits], name, 1)

    def linearSoftmaxCrossEntropy(self, hidden, weights, labels, bias=None, labelSmoothing=0.0, ignoreIndex=-100, transposeWeights=False, name=None):
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
        return self._o('linear_softmax_cross_entropy_loss', [hidden, weights, labels] + ([bias] if bias is not None else []), name, 1, iArgs=[ignoreIndex, int(transposeWeights)], tArgs=[labelSmoothing])

    def linearTopKDistillation(self, hidden, weights, teacherIndices, teacherLogits, bias=None, temperature=1.0, transposeWeights=False, name=None):
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
        return self._o('linear_topk_distillation_loss', [hidden, weights, teacherIndices, teacherLogits] + ([bias] if bias is not None else []), name, 1, iArgs=[int(transposeWeights)], tArgs=[temperature])

    def topKDistillation(self, logits, teacherIndices, teacherLogits, temperature=1.0, name=None):
        """Distillation from a teacher's top logits, T^2 KL(softmax(teacher / T) || softmax(student / T)), on student logits.
        :param logits: Student logits [..., V] (FLOATING_POINT)
        :param teacherIndices: Words of the teacher's K best logits [..., K], negative: padding (INT)
        :param teacherLogits: Their logits [..., K] (FLOATING_POINT)
        :param temperature: Temperature T (FLOATING_POINT, default 1.0)
        :return output: Per-row loss [...] (FLOATING_POINT)
        """
        return self._o('topk_distillation_loss', [logits, teacherIndices, teacherLogits], name, 1, tArgs=[temperature])

    def l2Loss(self, var, name=None):
        """Half the sum of squares: sum(x^2) / 2.
        :param var: Input (NUMERIC)
        :return output: Scalar loss (NUMERIC)
        """
        return self._o('l2_loss', [var], name, 1)

    def ctcLoss(self, targetLabels, logitInput, targetLabelLengths, logitInputLengths, blankIndex=0, name=None):
        """Connectionist temporal classification loss.
        :param targetLabels: Label sequences [batch, maxLabelLength] (INT)
        :param logitInput: Logits [batch, time, nClasses] (NUMERIC)
        :param targetLabelLengths: Label lengths [batch] (INT)
        :param logitInputLengths: Logit sequence lengths [batch] (INT)
        :param blankIndex: Index of the blank class (INT, default 0)
        :return output: Per-example loss (NUMERIC)
        """
        return self._o('ctc_loss', [targetLabels, logitInput, targetLabelLengths, logitInputLengths], name, 1, iArgs=[blankIndex])

    def weightedCrossEntropyWithLogits(self, targets, inputs, weights, name=None):
        """Sigmoid cross entropy with a weight on the positive term.
        :param targets: Targets (NUMERIC)
        :param inputs: Logits (NUMERIC)
        :param weights: Positive-class weights (NUMERIC)
        :return output: Loss (NUMERIC)
        """
        return self._o('weighted_cross_entropy_with_logits', [targets, inputs, weights], name, 1)
