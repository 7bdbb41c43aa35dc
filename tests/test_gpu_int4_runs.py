"""Expert products with four-bit weights whose K is cut into runs that do not divide it, against 64
bits.  Tolerances are those of test_gpu_int4.py."""
import pytest
import torch

import host_ops as H
from test_gpu_int4 import gated, gen, matrix, near, ops

pytestmark = pytest.mark.gpu


def uneven(rows, experts, g):
    """Offsets of `experts` ragged ranges over rows; with three or more one of them is empty."""
    share = torch.rand(experts, generator=g, device="cuda") + 0.5
    if experts > 2:
        share[1] = 0.0
    ends = (share.cumsum(0) / share.sum() * rows).round().to(torch.int32)
    ends[-1] = rows
    return torch.nn.functional.pad(ends, (1, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("experts,rows,hidden,inner,group", [
    (8, 2000, 2560, 128, 128),      # 20 chunks: runs of 3
    (8, 2000, 2560, 128, 32),
    (2, 1000, 2304, 512, 64),       # 18
    (1, 1024, 2176, 512, 128),      # 17
    (1, 700, 4608, 512, 128),       # 36: runs of 3 or 5
    (4, 1200, 4224, 128, 64),       # 33
])
def test_gate_and_up_in_runs(dtype, experts, rows, hidden, inner, group):
    g = gen(hidden + experts)
    w = H.quantize_int4(matrix((experts, 2 * inner, hidden), g) * 2, group, 2)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, group, halves=2)
    x = torch.randn((rows, hidden), generator=g, device="cuda").to(dtype)
    offsets, order = uneven(rows, experts, g), torch.randperm(rows, generator=g, device="cuda")
    named = order.to(torch.int32)
    got = ops().grouped_gate_up_swiglu(x, named, offsets, q)
    ops().check_async_errors()
    bounds = offsets.tolist()
    for e in range(experts):
        a, b = bounds[e], bounds[e + 1]
        near(got[a:b], *gated(x[order[a:b]], w[e].dense(torch.float64)))
    assert torch.equal(got, ops().grouped_gate_up_swiglu(x, named, offsets, q))
    ops().check_async_errors()
