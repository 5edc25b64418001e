"""Workspace sizes of the linear losses, as the library gives them for a call (no GPU needed)."""
import pytest

from deeplearning4j_amd.ops import vocab_loss as VL

MIB = 2 ** 20


def _sizes(n, d, v, dt, wt=False, k=0, bias=True):
    """bytes of the state, the forward and the backward workspace; dt 0 bf16, 1 fp16, 2 fp32"""
    a = VL._Block()
    fields = dict(N=n, D=d, V=v, dt=dt, split=dt == 2 and VL._split(n, d, v, True), wt=wt, ldh=d, ldw=v if wt else d, K=k, want_h=1, want_w=1, want_b=bias,
                  H=4096, W=4096)
    for name, x in fields.items():
        a[VL._AT[name]] = int(x)
    out = VL._Sizes()
    VL._lib().dl4j_linear_loss_bytes(a, out)
    return list(out)


@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("n,d,v", [(1, 768, 30522), (256, 1024, 128256), (512, 1024, 262144), (4096, 768, 30522), (4096, 256, 128256), (8192, 2048, 65536),
                                   (32768, 4096, 128256), (131072, 512, 32000), (131072, 64, 32000)])
def test_the_scores_gradient_takes_640_mib_at_most_in_all_its_copies(n, d, v, dt, wt):
    size = 4 if dt == 2 else 2
    up = lambda x, m: (x + m - 1) // m * m                                 # noqa: E731
    rows, words, width = up(n, 256), up(v, 256), up(d, 256)
    rest = (rows * width * (4 + 2 * size)                                  # dh in fp32, the packed or transposed rows
            + width * words * size                                        # the transposed table
            + 2 * 1024 * 128 * 128 * 4                                     # tiles of calls with few of them
            + (rows // 32 + 64) * 4 * v + 1024 * n)                        # column sums, side arrays
    gradient = max(640 * MIB, rows * 256 * size * 2)                       # (256 words at a time where the rows are that many)
    assert _sizes(n, d, v, dt, wt)[2] <= gradient + rest


def test_a_large_step_takes_less_than_its_logits():
    assert _sizes(8192, 2048, 65536, 0, bias=False)[2] < 8192 * 65536 * 2
