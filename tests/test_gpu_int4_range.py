"""Products with four-bit weights at the ends of the types' ranges.  Powers of two change no bits of a
result as long as every term of every sum is a number that fp32 holds whole:

* from above: a group's sum is less than the greatest activation, so activations up to the type's
  greatest number give what 64 bits give wherever that is a number;
* from below: an activation of e bits times a code has its last bit at 2^(its exponent - e - 11), which is
  to be 2^-149 or more.  Activations of N(0, 1) in bfloat16 are multiples of 2^-30 here (the smallest are
  set to 0), in fp32 of 2^-40: times 2^-100 and 2^-90 they stay so.
"""
import pytest
import torch

import host_ops as H
from test_gpu_int4 import gen, kernel, matrix, near, ops, sums_error  # noqa: F401

pytestmark = pytest.mark.gpu


def rows(dtype, k, g):
    x = torch.randn((1, k), generator=g, device="cuda")
    x = torch.where(x.abs() < 2.0 ** -15, 0.0, x)
    return x.to(dtype)


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype,least", [(torch.bfloat16, -100), (torch.float32, -90)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [4, 96])
def test_activations_from_end_to_end_of_the_range(dtype, least, group, m):
    g = gen(group)
    q = ops().quantize_int4(matrix((64, 512), g), group)
    x = rows(dtype, 512, g)
    powers = [0, least, 100, 124]
    x = torch.cat([x * 2.0 ** p for p in powers] + [x.new_zeros((m - len(powers), 512))])
    y = ops().linear(x, q, out_dtype=torch.float32)
    for i, p in enumerate(powers):
        assert torch.equal(y[i].double(), y[0].double() * 2.0 ** p), p


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [3, 90])
def test_the_greatest_activations(dtype, m):
    """Rows of the type's greatest number, of either sign: small where they cancel."""
    g = gen(m)
    w = H.quantize_int4(matrix((40, 256), g), 128)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, 128)
    sign = torch.where(torch.rand((m, 256), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x = (sign * torch.finfo(dtype).max).to(dtype)
    dense = w.dense(torch.float64)
    want = x.double() @ dense.t()
    # 32-bit sums pass through the two groups' own sums: where one of those is no number of 32 bits
    # (3.4e38; 1 % is more than the bound below allows) no sum of it is, though the other may bring it back
    parts = [x[:, k:k + 128].double() @ dense[:, k:k + 128].t() for k in (0, 128)]
    inside = torch.stack([want, *parts]).abs().amax(0) < 3.36e38
    assert inside.float().mean() > 0.5
    got = ops().linear(x, q, out_dtype=torch.float32)
    assert torch.isfinite(got[inside]).all()
    off = (got.double() - want)[inside].abs()
    assert (off <= sums_error(x, dense)[inside] + want[inside].abs() * 2.0 ** -24).all()


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [2, 80])
@pytest.mark.parametrize("power", [-130, -120, 0, 110, 116, 117, 122])
def test_scales_from_end_to_end_of_the_range(dtype, m, power):
    g = gen(m)
    codes = torch.randint(0, 16, (48, 384), generator=g, device="cuda", dtype=torch.uint8)
    zeros = torch.randint(0, 16, (48, 6), generator=g, device="cuda", dtype=torch.uint8)
    sign = torch.where(torch.rand((48, 6), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    # (bfloat16's subnormal scales: whole multiples of 2^-133)
    scales = (sign * torch.randint(1, 9, (48, 6), generator=g, device="cuda") * 2.0 ** power) \
        .to(torch.bfloat16)
    q = ops().pack_int4(codes, scales, zeros, 64)
    for a, b in zip(ops().unpack_int4(q), (codes, scales, zeros)):
        assert torch.equal(a, b)
    x = (rows(dtype, 384, g) * 2.0 ** -(power // 2)).expand(m, 384).contiguous()
    at = torch.arange(384, device="cuda") // 64
    dense = scales.double()[:, at] * (codes.double() - zeros.double()[:, at])
    near(ops().linear(x, q, out_dtype=torch.float32), x.double() @ dense.t(),
         sums_error(x, dense))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_scale_comes_back(group):
    """All 65,536 bit patterns of a scale, with every zero point."""
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16)
    scales = bits.view(torch.bfloat16).view(4096, 16)
    codes = torch.full((4096, 16 * group), 9, dtype=torch.uint8, device="cuda")
    for zero in range(16):
        zeros = torch.full((4096, 16), zero, dtype=torch.uint8, device="cuda")
        back = ops().unpack_int4(ops().pack_int4(codes, scales, zeros, group))
        assert torch.equal(back[0], codes) and torch.equal(back[2], zeros)
        assert torch.equal(back[1].view(torch.int16), scales.contiguous().view(torch.int16))
