"""The clamped gated unit over a matrix held in four bits, against 64 bits.

a(v) = v sigmoid(alpha v) has a slope within 1.1 in magnitude for every alpha > 0 (it is silu's at alpha v),
so |error| <= 1.1 |u + s| dg + |a(g)| du + 1.1 dg du with dg, du the products' (test_gpu_int4.py), and
the exponential and the quotient cost what they cost there: (6 + 1.2 alpha |g|) 2^-23 of the result.
In bfloat16 a few rows are rounded once; many rows are rounded before the activation too, which adds
2^-8 |g| to dg and 2^-8 |u| to du."""
import pytest
import torch

import host_ops as H
from test_gpu_int4 import gen, kernel, matrix, near, ops, sums_error  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,i", [(1, 264, 40), (3, 1000, 130), (16, 520, 64), (17, 520, 64),
                                   (150, 264, 72)])
@pytest.mark.parametrize("limit,alpha,shift", [(0.9, 1.702, 1.0), (7.0, 1.0, 0.0)])
def test_clamped_unit(dtype, m, k, i, limit, alpha, shift):
    g_ = gen(m + k)
    w = H.quantize_int4(matrix((2 * i, k), g_) * 3, 64)
    x = torch.randn((m, k), generator=g_, device="cuda").to(dtype)
    got = ops().gate_up_glu_clamped(x, ops().pack_int4(w.codes, w.scales, w.zeros, 64), limit,
                                    alpha, shift)
    assert got.dtype == dtype and got.shape == (m, i)
    dense = w.dense(torch.float64)
    g, u = x.double() @ dense[:i].t(), x.double() @ dense[i:].t()
    dg, du = sums_error(x, dense[:i]), sums_error(x, dense[i:])
    if dtype == torch.bfloat16 and m > ops().SMALL_M_DENSE_ROWS:
        dg, du = dg + 2.0 ** -8 * g.abs(), du + 2.0 ** -8 * u.abs()
    g, u = g.clamp(max=limit), u.clamp(-limit, limit) + shift
    a = g * torch.sigmoid(alpha * g)
    slack = 1.1 * u.abs() * dg + a.abs() * du + 1.1 * dg * du \
        + (a * u).abs() * (6.0 + 1.2 * alpha * g.abs()) * 2.0 ** -23
    near(got, a * u, slack)


def test_the_types_that_go_in_and_out():
    o = ops()
    gu = torch.randn((3, 48), device="cuda")
    want = o.glu_clamped(gu, 0.9, 1.702, 1.0)
    assert torch.equal(o.glu_clamped(gu, 0.9, 1.702, 1.0, out_dtype=torch.bfloat16),
                       want.to(torch.bfloat16))
    with pytest.raises(o.KernelError):
        o.glu_clamped(gu.to(torch.bfloat16), 0.9, 1.702, 1.0, out_dtype=torch.float32)
    with pytest.raises(o.KernelError):
        o.glu_clamped(gu, 0.9, 1.702, 1.0, out_dtype=torch.float16)
