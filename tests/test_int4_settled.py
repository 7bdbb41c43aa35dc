"""Products with four-bit weights may fetch codes ahead of the kernel before them only where nothing
still writes them."""
import copy
import types

import pytest
import torch

from inferx_b200.kernels import ops
from inferx_b200.parts.base import BuildContext, hold_in_int4


def empty():
    return ops._int4_empty("here", (32, 128), 64, 1, "cpu")


def test_a_new_weight_is_not_settled():
    q = empty()
    assert not q.settled and q._record.settled == 0
    assert q.settle() is q and q.settled and q._record.settled == 1
    # what a copy's codes were written by is another launch
    assert not copy.deepcopy(q).settled


def test_a_loaded_model_settles_what_it_holds():
    made = []
    fake = types.SimpleNamespace(quantize_int4=lambda w, g, h: made.append(empty()) or made[-1])

    class Part:
        int4_weights = {"a": 1, "b": 1, "none": 1}
        a, b, none = torch.ones(32, 128), torch.ones(32, 128), None
    part = Part()
    assert hold_in_int4(part, BuildContext(torch.float32, torch.device("cpu"), fake, 64)) == 2
    assert [part.a, part.b] == made and all(q.settled for q in made)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_right_behind_the_weights(dtype):
    """Quantised and multiplied with at once, into the same memory again and again, with launches
    that overlap."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    ws = [torch.randn((1024, 1024), generator=g, device="cuda").to(dtype) for _ in range(4)]
    x = torch.randn((3, 1024), generator=g, device="cuda").to(dtype)
    want = []
    for w in ws:
        q = ops.quantize_int4(w, 128)
        torch.cuda.synchronize()
        want.append(ops.linear(x, q))
        del q
    try:
        ops.set_dependent_launch(True)
        for i in range(40):
            q = ops.quantize_int4(ws[i % 4], 128)
            got = [ops.linear(x, q), ops.linear(x, q), ops.linear(x, q.settle())]
            del q
            assert all(torch.equal(y, want[i % 4]) for y in got)
    finally:
        ops.set_dependent_launch(False)
