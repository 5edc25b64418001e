"""Training steps in fp32 (halves) and fp16 recorded into a graph: every replay gives the eager results bit for bit, with rows, words and row weights
whose sizes, and so the kernels' factors and copies, change from replay to replay; and two such steps run at once on two streams."""
import math

import pytest
import torch

from deeplearning4j_amd.ops import vocab_loss as VL

pytestmark = pytest.mark.gpu
DEV = "cuda"
CASES = [(500, 512, 4000, torch.float32, "vd"), (700, 520, 30000, torch.float32, "vd"), (700, 520, 30000, torch.float32, "dv"), (1300, 260, 3001, torch.float32, "dv"),
         (300, 101, 903, torch.float16, "vd"), (1100, 520, 30000, torch.float16, "dv")]


def _data(n, d, v, dtype, layout, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(n, d, generator=g, device=DEV)
    w = torch.randn(v, d, generator=g, device=DEV) * (2.5 / math.sqrt(d))
    dl = torch.rand(n, generator=g, device=DEV) + 0.5
    if seed % 3 == 1:                                                      # a huge row, words far apart, row weights far apart
        if dtype == torch.float32:
            h[n // 2] *= 1e7
            w *= 10.0 ** (-8 * torch.rand(v, 1, generator=g, device=DEV))
        dl *= 10.0 ** -(torch.arange(n, device=DEV) % 7).float()
    y = torch.randint(0, v, (n,), generator=g, device=DEV)
    y[torch.rand(n, generator=g, device=DEV) < 0.3 * (seed % 4)] = -100
    idx, t = torch.randint(0, v, (n, 6), generator=g, device=DEV), torch.randn(n, 6, generator=g, device=DEV)
    return [h.to(dtype), (w if layout == "vd" else w.t()).to(dtype).contiguous(), torch.randn(v, generator=g, device=DEV).to(dtype)], y, idx, t, dl


def _step(layout, leaves, y, idx, t, dl):
    h, w, b = leaves
    wv = w if layout == "vd" else w.t()
    a, k = VL.linear_cross_entropy(h, wv, y, b, label_smoothing=0.1), VL.linear_topk_distillation(h, wv, idx, t, b, temperature=2.0)
    return (a.detach(), k.detach()) + torch.autograd.grad([a, k], leaves, [dl, dl])


def _eager(layout, data):
    leaves, *rest = data
    return _step(layout, [x.detach().clone().requires_grad_() for x in leaves], *rest)


@pytest.mark.parametrize("n,d,v,dtype,layout", CASES)
def test_replays_follow_their_data(n, d, v, dtype, layout):
    leaves, *rest = _data(n, d, v, dtype, layout, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _eager(layout, (leaves, *rest))
    torch.cuda.current_stream().wait_stream(s)
    static = [x.detach().clone().requires_grad_() for x in leaves]
    held = [x.clone() for x in rest]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(layout, static, *held)
    for seed in (3, 1, 2, 4, 6):
        data = _data(n, d, v, dtype, layout, seed)
        with torch.no_grad():
            for x, new in zip(static + held, data[0] + list(data[1:])):
                x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, _eager(layout, data)):
            assert torch.equal(a, e) or (a.isnan().any() and torch.equal(a.nan_to_num(), e.nan_to_num()))


@pytest.mark.parametrize("n,d,v,dtype,layout", CASES)
def test_two_streams_at_once(n, d, v, dtype, layout):
    data = [_data(n, d, v, dtype, layout, seed) for seed in (1, 2)]
    want = [_eager(layout, x) for x in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k, _eager(layout, data[k])))
    torch.cuda.synchronize()
    for k, out in got:
        for a, e in zip(out, want[k]):
            assert torch.equal(a, e)
