"""One row of logits whose leading stride says nothing (a row of length-1 axes keeps whatever stride it came with)."""
import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _one_row(kind, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(v)
    if kind == "transposed column":                                        # strides (1, 1)
        return (torch.randn(v, 1, generator=g, device=DEV) * 2).to(dtype).t()
    if kind == "expanded":                                                 # strides (0, 1)
        return (torch.randn(v, generator=g, device=DEV) * 2).to(dtype).expand(3, v)[1:2]
    return (torch.randn(v, 3, generator=g, device=DEV) * 2).to(dtype).t()[1:2]      # strides (1, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [1, 7, 1000])
@pytest.mark.parametrize("kind", ["transposed column", "expanded", "strided"])
def test_one_row_of_logits_of_any_stride(kind, v, dtype):
    z = _one_row(kind, v, dtype)
    idx, t = torch.tensor([[0, v - 1, -1]], device=DEV), torch.tensor([[0.5, -0.25, 9.0]], device=DEV)
    plain = z.detach().clone(memory_format=torch.contiguous_format).reshape(-1).clone().reshape(1, v)
    assert plain.stride() == (v, 1)
    want_leaf, leaf = plain.requires_grad_(), z.detach().requires_grad_()
    want = VL.topk_distillation(want_leaf, idx, t, temperature=2.0)
    got = VL.topk_distillation(leaf, idx, t, temperature=2.0)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), leaf)[0], torch.autograd.grad(want.sum(), want_leaf)[0])
    with torch.no_grad():
        assert torch.equal(VL.topk_distillation(z, idx, t, temperature=2.0), want)
