"""A product that is recorded before any has run."""
import pytest
import torch

from test_gpu_int4 import gen, matrix, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4, 300])
def test_the_first_product_is_a_recorded_one(rows, monkeypatch):
    o = ops()
    monkeypatch.setattr(o, "_TC_STATUS", {})
    g = gen(rows)
    q = o.quantize_int4(matrix((264, 520), g), 128)
    x = torch.randn((rows, 520), generator=g, device="cuda").to(torch.bfloat16)
    # what the allocator hands out next is not zero
    junk = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (1, 128, 1 << 18)]
    del junk
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = o.linear(x, q)
    o.check_async_errors()                  # nothing has run, so nothing has waited too long
    word = o._tc_status(x.device)
    word.fill_(52)                          # as a kernel's warp would
    graph.replay()
    with pytest.raises(o.KernelError, match="the MMA issuer"):
        o.check_async_errors()
    graph.replay()
    o.check_async_errors()
    assert torch.equal(y, o.linear(x, q))
