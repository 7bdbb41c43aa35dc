"""Expert products with four-bit weights whose K is cut into runs that do not divide it, with several
items to a pair of SMs, against 64 bits.  Tolerances are those of test_gpu_int4.py."""
import pytest
import torch

import host_ops as H
from test_gpu_int4 import gated, gen, matrix, near, ops, sums_error

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
    (1, 700, 4608, 512, 128),       # 36
    (4, 1200, 4224, 128, 64),       # 33
    (3, 1500, 3328, 300, 128),      # 26
    (5, 4096, 1160, 130, 128),      # 9 and a part: the last run is the short chunk alone
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("experts,rows,inner,hidden,group", [
    (1, 1024, 2560, 1024, 128), (1, 1024, 2560, 1024, 64), (2, 900, 3200, 1024, 128),
    (4, 1200, 4224, 256, 32), (8, 2000, 2560, 256, 128), (2, 4096, 2304, 515, 64)])
def test_down_in_runs(dtype, experts, rows, inner, hidden, group):
    g = gen(inner + experts)
    w = H.quantize_int4(matrix((experts, hidden, inner), g), group)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, group)
    x = torch.randn((rows, inner), generator=g, device="cuda").to(dtype)
    offsets = uneven(rows, experts, g)
    got = ops().grouped_down(x, offsets, q)
    ops().check_async_errors()
    bounds = offsets.tolist()
    for e in range(experts):
        a, b = bounds[e], bounds[e + 1]
        dense = w[e].dense(torch.float64)
        near(got[a:b], x[a:b].double() @ dense.t(), sums_error(x[a:b], dense))


@pytest.mark.parametrize("hidden,inner", [(3328, 384), (3200, 300), (3328, 300)])
def test_codes_are_read_before_the_next_ones_land(hidden, inner):
    """Items that follow one another quickly on a pair, with results of single numbers going out
    beside them: every call gives the same bits, and they are the product's."""
    g = gen(hidden + inner)
    experts, rows = 3, 1500
    w = H.quantize_int4(matrix((experts, 2 * inner, hidden), g) * 2, 128, 2)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, 128, halves=2)
    x = torch.randn((rows, hidden), generator=g, device="cuda").to(torch.bfloat16)
    named = torch.arange(rows, device="cuda", dtype=torch.int32)
    offsets = torch.tensor([0, 677, 677, rows], dtype=torch.int32, device="cuda")
    got = [ops().grouped_gate_up_swiglu(x, named, offsets, q) for _ in range(25)]
    ops().check_async_errors()
    for y in got[1:]:
        assert torch.equal(y, got[0])
    for e, a, b in ((0, 0, 677), (2, 677, rows)):
        near(got[0][a:b], *gated(x[a:b], w[e].dense(torch.float64)))
