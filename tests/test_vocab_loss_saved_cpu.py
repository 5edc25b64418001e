"""The vocabulary losses' backward pass works on the tensors that autograd hands back, which need not be the forward call's: hooks of saved
tensors (recomputation, offload to the host) replace them. Without a GPU: the native call is replaced by a recorder of its argument block."""
import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL


class _Recorder:
    """Stands for the native calls: keeps each block's fields by name; the gradients stay as allocated."""

    def __init__(self):
        self.calls = []

    def __call__(self, fn, what, dev, a, f):
        fields = VL._ARGS if "linear" in what else "N V K ldz dt idx64 tdt z idx t loss lse dloss dz".split()
        self.calls.append((what, dict(zip(fields, list(a)))))


@pytest.fixture
def calls(monkeypatch):
    rec = _Recorder()
    monkeypatch.setattr(VL, "_launch", rec)
    monkeypatch.setattr(VL, "usable", lambda *t: True)
    return rec.calls


class _Clones:
    """Hooks that keep clones, as an offload does; ``change`` alters what is handed back."""

    def __init__(self, change=lambda t: t):
        self.back, self.change = [], change

    def __enter__(self):
        def unpack(t):
            t = self.change(t)
            self.back.append(t)
            return t
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack)
        self.hooks.__enter__()
        return self

    def __exit__(self, *e):
        return self.hooks.__exit__(*e)

    def addresses(self):
        return {t.data_ptr() for t in self.back}


def _leaves(*shapes, dtype=torch.bfloat16):
    return [torch.randn(*s).to(dtype).requires_grad_() for s in shapes]


def _backward(loss):
    loss.backward(torch.ones_like(loss))


@pytest.mark.parametrize("layout", ["vd", "dv"])
@pytest.mark.parametrize("distil", [False, True])
def test_linear_losses_read_what_was_saved(calls, distil, layout):
    h, w, b = _leaves((5, 16), (24, 16) if layout == "vd" else (16, 24), (24,))
    wv = w if layout == "vd" else w.t()
    with _Clones() as hooks:
        if distil:
            loss = VL.linear_topk_distillation(h, wv, torch.zeros(5, 3, dtype=torch.int64), torch.zeros(5, 3), b)
        else:
            loss = VL.linear_cross_entropy(h, wv, torch.zeros(5, dtype=torch.int64), b)
    _backward(loss)
    (_, fwd), (what, bwd) = calls
    assert what == "linear_loss_bwd"
    for name in ("H", "W", "bias", "state"):
        assert bwd[name] in hooks.addresses() and bwd[name] != fwd[name], name
    same = [n for n in VL._ARGS[:VL._AT["H"]]]
    assert [bwd[n] for n in same] == [fwd[n] for n in same]               # sizes, layouts and choices are the forward call's


def test_the_on_logits_loss_reads_what_was_saved(calls):
    z, = _leaves((5, 24))
    with _Clones() as hooks:
        loss = VL.topk_distillation(z, torch.zeros(5, 3, dtype=torch.int64), torch.zeros(5, 3))
    _backward(loss)
    (_, fwd), (_, bwd) = calls
    for name in ("z", "idx", "t", "lse"):
        assert bwd[name] in hooks.addresses() and bwd[name] != fwd[name], name


def test_recomputation_hands_over_the_second_pass(calls):
    """Non-reentrant checkpointing frees the first pass's hidden states: the backward call must not hold their address."""
    from torch.utils.checkpoint import checkpoint
    x, w = _leaves((6, 16), (24, 16))
    made = []

    def block(x, w):
        h = torch.tanh(x)
        made.append(h.data_ptr())
        keep.append(h)                                                     # (so that the second pass lies elsewhere)
        return VL.linear_cross_entropy(h, w, torch.zeros(6, dtype=torch.int64))

    keep = []
    _backward(checkpoint(block, x, w, use_reentrant=False))
    bwd = [c for c in calls if c[0] == "linear_loss_bwd"][-1][1]
    assert len(made) == 2 and made[0] != made[1] and bwd["H"] == made[1]


def test_other_strides_and_alignments_are_brought_back(calls):
    """The forward call's choices rest on rows that start on 16 bytes and lie ``ld`` apart: what comes back otherwise is laid out so again."""
    def odd(t):                                                            # same values, rows 3 further apart, off 16 bytes
        if t.dim() != 2 or t.dtype == torch.uint8:
            return t
        big = torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype)
        big[:, 1:1 + t.shape[1]] = t
        return big[:, 1:1 + t.shape[1]]
    h, w = _leaves((5, 16), (24, 16))
    with _Clones(odd):
        loss = VL.linear_cross_entropy(h, w, torch.zeros(5, dtype=torch.int64))
    _backward(loss)
    (_, fwd), (_, bwd) = calls
    assert bwd["H"] % 16 == 0 and bwd["W"] % 16 == 0
    for n in VL._ARGS[:VL._AT["H"]]:
        assert bwd[n] == fwd[n], n
    del calls[:]
    z, = _leaves((5, 24))
    with _Clones(odd):
        loss = VL.topk_distillation(z, torch.zeros(5, 3, dtype=torch.int64), torch.zeros(5, 3))
    _backward(loss)
    assert calls[1][1]["ldz"] == 27                                        # (any stride is fine there, if it is the tensor's)


def test_a_state_of_another_call_is_refused(calls):
    h, w = _leaves((5, 16), (24, 16))
    with _Clones(lambda t: t[:-256] if t.dtype == torch.uint8 else t):
        loss = VL.linear_cross_entropy(h, w, torch.zeros(5, dtype=torch.int64))
    with pytest.raises(VL.ND4JIllegalArgumentException, match="state"):
        _backward(loss)


@pytest.mark.parametrize("v", [1, 7, 24])
@pytest.mark.parametrize("row", [lambda v: torch.randn(v, 1).t(), lambda v: torch.randn(v).expand(3, v)[1:2], lambda v: torch.randn(v, 3).t()[1:2]])
def test_one_row_of_logits_has_a_row_distance_whatever_its_stride(calls, v, row):
    z = row(v).requires_grad_()
    _backward(VL.topk_distillation(z, torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, 3)))
    for _, c in calls:
        assert c["ldz"] >= v


@pytest.mark.parametrize("rows", [2, 5])
def test_rows_of_one_logit_lie_as_far_apart_as_they_do(calls, rows):
    z = torch.randn(rows, 4)[:, 1:2].requires_grad_()                      # strides (4, 1)
    _backward(VL.topk_distillation(z, torch.zeros(rows, 3, dtype=torch.int64), torch.zeros(rows, 3)))
    assert [c["ldz"] for _, c in calls] == [4, 4]
    del calls[:]
    z = torch.randn(3, rows).t()[:, 1:2].requires_grad_()                  # strides (1, rows): the inner one says nothing
    _backward(VL.topk_distillation(z, torch.zeros(rows, 3, dtype=torch.int64), torch.zeros(rows, 3)))
    assert [c["ldz"] for _, c in calls] == [1, 1]
