"""Weights in four bits: quantising, laying out, and the products that read them, against plain
statements in 64 bits.

Tolerances, counted before the first run.  A product of n terms is summed in fp32: every partial
sum is off by at most half a step of 2^-23 of the sum of magnitudes below it (a whole step where
the tensor cores cut off), n + 8 of them with the joins, so |error| <= (n + 8) 2^-23 sum |x w|.
fp32 activations are three exact terms: three times as many.  A result in bfloat16 adds 2^-8 of
itself, one in fp32 2^-24.  silu(g) u moves by at most 1.1 |u| dg + |silu(g)| du + 1.1 dg du (the
slope of silu lies between -0.1 and 1.1), and the exponential is good to 2 + 1.2 |g| steps of 2^-23
(the fast one), its quotient to two more.
"""
import pytest
import torch

import host_ops as H

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def ops():
    from inferx_b200.kernels import ops as o
    return o


@pytest.fixture(params=["chosen", "few rows", "many rows"])
def kernel(request, monkeypatch):
    """The products as the rules choose their kernel, and each kernel for calls of either's sizes."""
    if request.param != "chosen":
        most = 0 if request.param == "many rows" else 1 << 62
        each = {torch.bfloat16: most, torch.float32: most}
        monkeypatch.setattr(ops(), "INT4_STREAM_ROWS", most)
        monkeypatch.setattr(ops(), "INT4_STREAM_MOST_ROWS", each)
        monkeypatch.setattr(ops(), "INT4_STREAM_ROW_BYTES", each)
        monkeypatch.setattr(ops(), "INT4_STREAM_ROWS_PER_EXPERT", each)
    return request.param


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(shape, g, dtype=torch.float32):
    w = torch.randn(shape, generator=g, device="cuda") * 0.02
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.01, 6 * w, w).to(dtype)


def sums_error(x, w):
    """What summing in fp32 may cost: x [M, K], w [N, K] in 64 bits."""
    n = x.shape[1] + 8
    if x.dtype == torch.float32:
        n *= 3
    return n * 2.0 ** -23 * (x.double().abs() @ w.abs().t())


def near(got, want, slack):
    """|got - want| <= slack + a rounding of the result, entry by entry."""
    off = (got.double() - want).abs()
    room = slack + want.abs() * STEP[got.dtype] + 1e-37
    worst = (off / room).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"off by {worst:.3f} of what is allowed"


def gated(x, w, scale=None):
    """(silu(g) u, slack) in 64 bits."""
    n = w.shape[0] // 2
    g, u = x.double() @ w[:n].t(), x.double() @ w[n:].t()
    dg, du = sums_error(x, w[:n]), sums_error(x, w[n:])
    if scale is not None:
        s = scale.double()[:, None]
        g, u, dg, du = g * s, u * s, dg * s.abs() + g.abs() * s.abs() * 2.0 ** -23, \
            du * s.abs() + u.abs() * s.abs() * 2.0 ** -23
    a = g * torch.sigmoid(g)
    y = a * u
    slack = 1.1 * u.abs() * dg + a.abs() * du + 1.1 * dg * du \
        + y.abs() * (6.0 + 1.2 * g.abs()) * 2.0 ** -23
    return y, slack


# -- quantising and the layout -----------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape,halves", [((16, 128), 1), ((1, 1), 1), ((17, 33), 1),
                                          ((3, 50, 200), 1), ((2, 34, 1000), 2), ((515, 72), 1),
                                          ((130, 257), 2)])
def test_quantize_is_the_definition_bit_for_bit(dtype, group, shape, halves):
    w = matrix(shape, gen(1), dtype)
    got = ops().unpack_int4(ops().quantize_int4(w, group, halves))
    want = H.quantize_int4(w, group, halves)
    for a, b in zip(got, (want.codes, want.scales, want.zeros)):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_groups_at_the_edges_of_the_type(dtype):
    """Groups of zeros, of one sign, of one value, next to a border between two codes, of the
    type's least and greatest numbers, with an infinity or a NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    w = torch.zeros((12, 64), device="cuda")
    w[1] = 0.75
    w[2] = -0.75
    w[3, ::2] = 3.0
    w[4] = torch.linspace(-1, 1, 64, device="cuda")
    w[5] = torch.arange(64, device="cuda") * 0.5 - 7.5        # quotients on the half
    w[6, 0], w[6, 1] = big, -big
    w[7, 0] = tiny
    w[8, 0], w[8, 1] = 15.0, 1e-30
    w[9, 3] = 1.0
    w[10, 5] = 1.0
    w = w.to(dtype)
    w[9, 40], w[10, 41], w[10, 2] = float("inf"), float("nan"), -float("inf")
    w[11, :2] = torch.tensor([15.0, 0.5], device="cuda", dtype=dtype)
    if dtype == torch.float32:
        w[11, 2] = torch.nextafter(torch.tensor(0.5), torch.tensor(1.0))
        w[11, 3] = torch.nextafter(torch.tensor(0.5), torch.tensor(0.0))
    got = ops().unpack_int4(ops().quantize_int4(w, 32))
    want = H.quantize_int4(w, 32)
    assert torch.equal(got[0], want.codes) and torch.equal(got[2], want.zeros)
    assert torch.equal(got[1].nan_to_num(-1.0), want.scales.nan_to_num(-1.0))
    if dtype == torch.float32:
        assert got[0][11, 1:4].tolist() == [0, 1, 0]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape,halves", [((48, 256), 1), ((2, 34, 77), 2), ((1, 5), 1)])
def test_pack_and_unpack_are_inverse(group, shape, halves):
    g = gen(2)
    groups = (*shape[:-1], -(-shape[-1] // group))
    codes = torch.randint(0, 16, shape, generator=g, device="cuda", dtype=torch.uint8)
    zeros = torch.randint(0, 16, groups, generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randn(groups, generator=g, device="cuda").to(torch.bfloat16)
    back = ops().unpack_int4(ops().pack_int4(codes, scales, zeros, group, halves))
    for a, b in zip(back, (codes, scales, zeros)):
        assert torch.equal(a, b)


# -- one matrix --------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 128, 16), (2, 40, 15), (3, 129, 17), (7, 1000, 515), (8, 2048, 64),
         (9, 64, 33), (16, 333, 100), (17, 640, 96), (31, 256, 1030), (33, 1000, 515),
         (64, 2048, 130), (65, 72, 256), (130, 520, 129), (257, 1408, 300), (1, 20480, 48)]


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16),
                                       (torch.bfloat16, torch.float32),
                                       (torch.float32, torch.float32)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(dtype, out, group, m, k, n):
    g = gen(m * 7 + k)
    w = H.quantize_int4(matrix((n, k), g), group)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, group)
    got = ops().linear(x, q, out_dtype=out)
    assert got.dtype == out and got.shape == (m, n)
    dense = w.dense(torch.float64)
    near(got, x.double() @ dense.t(), sums_error(x, dense))
    assert torch.equal(got, ops().linear(x, q, out_dtype=out))


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", [(1, 128, 16), (2, 40, 15), (8, 2048, 88), (13, 333, 65),
                                   (33, 1000, 130), (70, 256, 515), (300, 640, 129)])
def test_gated(dtype, group, m, k, n):
    g = gen(m * 11 + n)
    w = H.quantize_int4(matrix((2 * n, k), g) * 3, group, 2)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, group, halves=2)
    got = ops().gate_up_swiglu(x, q)
    assert got.dtype == dtype and got.shape == (m, n)
    near(got, *gated(x, w.dense(torch.float64)))


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation", ["gelu", "relu_squared"])
@pytest.mark.parametrize("m", [3, 150])
def test_linear_act(dtype, activation, m):
    g = gen(m)
    w = H.quantize_int4(matrix((100, 264), g) * 3, 64)
    x = torch.randn((m, 264), generator=g, device="cuda").to(dtype)
    got = ops().linear_act(x, ops().pack_int4(w.codes, w.scales, w.zeros, 64), activation)
    dense = w.dense(torch.float64)
    y, d = x.double() @ dense.t(), sums_error(x, dense)
    if activation == "gelu":
        # the slope of gelu lies within 1.13; the error function of bfloat16 results is good to
        # 3e-7 and that of fp32 ones to two steps
        want = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
        near(got, want, 1.13 * d + 0.5 * y.abs() * (4e-7 if dtype == torch.bfloat16 else 2.0 ** -21))
    else:
        near(got, y.clamp(min=0) ** 2, 2 * y.abs() * d + d * d + y * y * 2.0 ** -23)


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("m", [2, 40, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan_stay_in_their_rows(m, dtype):
    g = gen(5)
    w = H.quantize_int4(matrix((70, 200), g), 64)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, 64)
    x = torch.randn((m, 200), generator=g, device="cuda").to(dtype)
    clean = ops().linear(x, q, out_dtype=torch.float32)
    bad = x.clone()
    bad[0, 3] = float("inf")
    bad[1, 199] = float("nan")
    got = ops().linear(bad, q, out_dtype=torch.float32)
    assert torch.equal(got[2:], clean[2:])
    dense = w.dense(torch.float64)
    want = bad[:2].double() @ dense.t()
    assert torch.equal(torch.isnan(got[:2]), torch.isnan(want))
    assert torch.equal(got[0].double()[~torch.isnan(want[0])], want[0][~torch.isnan(want[0])])


@pytest.mark.usefixtures("kernel")
def test_weights_that_hold_an_infinity_say_so():
    w = matrix((40, 256), gen(6), torch.bfloat16)
    w[7, 130] = float("inf")
    q = ops().quantize_int4(w, 128)
    for m in (3, 100):
        y = ops().linear(torch.ones((m, 256), device="cuda", dtype=torch.bfloat16), q)
        assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, :7]).all()
        assert torch.isfinite(y[:, 8:]).all()


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_great_and_small_activations_keep_their_bits(dtype):
    """Rows scaled by powers of two give results scaled by them, bit for bit."""
    g = gen(8)
    q = ops().quantize_int4(matrix((64, 512), g), 128)
    x = torch.randn((4, 512), generator=g, device="cuda").to(dtype)
    x[1], x[2], x[3] = x[0] * 2.0 ** -60, x[0] * 2.0 ** 60, x[0] * 2.0 ** 100
    for m in (4, 96):
        rows = torch.cat([x, x.new_zeros((m - 4, 512))])
        y = ops().linear(rows, q, out_dtype=torch.float32)
        assert torch.equal(y[1], y[0] * 2.0 ** -60)
        assert torch.equal(y[2], y[0] * 2.0 ** 60)
        assert torch.equal(y[3], y[0] * 2.0 ** 100)


@pytest.mark.usefixtures("kernel")
def test_misaligned_rows():
    """A contiguous view that starts in the middle of a buffer."""
    g = gen(9)
    w = H.quantize_int4(matrix((50, 64), g), 32)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, 32)
    for m in (3, 90):
        x = torch.randn(m * 64 + 1, generator=g, device="cuda").to(torch.bfloat16)[1:].view(m, 64)
        assert torch.equal(ops().linear(x, q), ops().linear(x.clone(), q))


@pytest.mark.usefixtures("kernel")
def test_no_rows():
    q = ops().quantize_int4(matrix((50, 64), gen(1)), 32)
    y = ops().linear(torch.empty((0, 64), device="cuda"), q)
    assert y.shape == (0, 50) and y.dtype == torch.float32


# -- experts -----------------------------------------------------------------------------
def routed(tokens, experts, top, g, skew=0.0):
    score = torch.randn((tokens, experts), generator=g, device="cuda")
    score[:, 0] += skew
    chosen = score.topk(top, dim=-1).indices.flatten()
    order = torch.sort(chosen, stable=True).indices
    counts = torch.bincount(chosen, minlength=experts)
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
    return (order // top).to(torch.int32), offsets


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,experts,top,hidden,inner,skew", [
    (1, 4, 2, 64, 32, 0.0), (1, 60, 4, 256, 48, 0.0), (5, 8, 3, 104, 40, 0.0),
    (8, 60, 4, 512, 136, 0.0), (33, 16, 2, 200, 100, 0.0), (100, 4, 4, 264, 72, 0.0),
    (150, 8, 2, 136, 65, 9.0), (700, 3, 2, 128, 40, 9.0)])
def test_experts_up_and_down(dtype, group, tokens, experts, top, hidden, inner, skew):
    """The routed products one after the other: gate and up, then down from what they gave."""
    g = gen(tokens + experts)
    rows, offsets = routed(tokens, experts, top, g, skew)
    gu = H.quantize_int4(matrix((experts, 2 * inner, hidden), g) * 3, group, 2)
    dn = H.quantize_int4(matrix((experts, hidden, inner), g), group)
    x = torch.randn((tokens, hidden), generator=g, device="cuda").to(dtype)
    qg = ops().pack_int4(gu.codes, gu.scales, gu.zeros, group, halves=2)
    qd = ops().pack_int4(dn.codes, dn.scales, dn.zeros, group)
    for scale in (None, torch.rand(rows.numel(), generator=g, device="cuda") + 0.5):
        act = ops().grouped_gate_up_swiglu(x, rows, offsets, qg, row_scale=scale)
        y = ops().grouped_down(act, offsets, qd)
        bounds = offsets.tolist()
        for e in range(experts):
            a, b = bounds[e], bounds[e + 1]
            mine = x[rows[a:b].long()]
            near(act[a:b], *gated(mine, gu[e].dense(torch.float64),
                                  None if scale is None else scale[a:b]))
            w = dn[e].dense(torch.float64)
            near(y[a:b], act[a:b].double() @ w.t(), sums_error(act[a:b], w))


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [2, 90])
def test_experts_without_a_gate(dtype, tokens):
    g = gen(tokens)
    rows, offsets = routed(tokens, 6, 2, g)
    w = H.quantize_int4(matrix((6, 50, 136), g) * 3, 32)
    x = torch.randn((tokens, 136), generator=g, device="cuda").to(dtype)
    got = ops().grouped_up(x, rows, offsets, ops().pack_int4(w.codes, w.scales, w.zeros, 32),
                           "relu_squared")
    bounds = offsets.tolist()
    for e in range(6):
        a, b = bounds[e], bounds[e + 1]
        mine, dense = x[rows[a:b].long()], w[e].dense(torch.float64)
        y, d = mine.double() @ dense.t(), sums_error(mine, dense)
        near(got[a:b], y.clamp(min=0) ** 2, 2 * y.abs() * d + d * d + y * y * 2.0 ** -23)


@pytest.mark.usefixtures("kernel")
def test_rows_behind_the_last_expert_are_left_alone():
    """Rows of experts that are not there (a router's identity outputs) get no product, and
    what stands there does not reach the others."""
    g = gen(3)
    rows, offsets = routed(40, 5, 2, g)
    q = ops().quantize_int4(matrix((4, 64, 128), g), 64, halves=2)
    x = torch.randn((40, 128), generator=g, device="cuda").to(torch.bfloat16)
    last = int(offsets[4])
    part = ops().grouped_gate_up_swiglu(x, rows, offsets[:5].contiguous(), q)
    assert part.shape == (80, 32)
    alone = ops().grouped_gate_up_swiglu(x, rows[:last].contiguous(), offsets[:5].contiguous(), q)
    # (how the work is cut may follow the number of rows: equal up to the last bit of a result)
    assert torch.allclose(part[:last].float(), alone.float(), rtol=2.0 ** -7, atol=1e-6)


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("kernel", ["many rows"], indirect=True)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n,halves", [
    (193, 5632, 260, 1),       # runs of K that are joined
    (2500, 384, 777, 2),       # more tiles than pairs of SMs, a short last one
    (700, 2048, 2048, 1), (4100, 136, 520, 1), (385, 640, 1409, 2)])
def test_many_rows(dtype, group, m, k, n, halves):
    """Tiles of each height, several of them to a pair, more rows than one run of K serves."""
    g = gen(m + n)
    q = ops().quantize_int4(matrix((halves * n, k), g), group, halves=halves)
    codes, scales, zeros = ops().unpack_int4(q)
    at = torch.arange(k, device="cuda") // group
    w = scales.double()[:, at] * (codes.double() - zeros.double()[:, at])
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    if halves == 2:
        near(ops().gate_up_swiglu(x, q), *gated(x, w))
    else:
        near(ops().linear(x, q), x.double() @ w.t(), sums_error(x, w))


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("experts", [1, 1024, 1030])
def test_as_many_experts_as_there_may_be(dtype, experts):
    """The same expert for all rows, with all others empty, and rows that are named twice."""
    g = gen(experts)
    w = H.quantize_int4(matrix((experts, 40, 96), g), 32)
    q = ops().pack_int4(w.codes, w.scales, w.zeros, 32)
    for here, count in ((0, 37), (experts - 1, 37), (experts // 2, 700)):
        x = torch.randn((count, 96), generator=g, device="cuda").to(dtype)
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        offsets[here + 1:] = count
        dense = w[here].dense(torch.float64)
        near(ops().grouped_down(x, offsets, q), x.double() @ dense.t(), sums_error(x, dense))
        twice = torch.arange(count, device="cuda", dtype=torch.int32) // 2
        mine = x[twice.long()]
        y, d = mine.double() @ dense.t(), sums_error(mine, dense)
        near(ops().grouped_up(x, twice, offsets, q, "relu_squared"), y.clamp(min=0) ** 2,
             2 * y.abs() * d + d * d + y * y * 2.0 ** -23)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("hidden,inner", [(2048, 520), (1408, 264)])
def test_codes_that_land_out_of_order(group, hidden, inner):
    """Long prompts over weights that are not in the second-level cache: a chunk's codes may land
    after the next one's.  Every call gives the same bits, and they are the product's."""
    g = gen(hidden + group)
    experts, tokens = 24, 1100
    rows, offsets = routed(tokens, experts, 4, g, 1.0)
    q = ops().quantize_int4(matrix((experts, 2 * inner, hidden), g), group, halves=2)
    x = torch.randn((tokens, hidden), generator=g, device="cuda").to(torch.bfloat16)
    other = torch.empty(160 << 20, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(12):
        other.fill_(i)
        got = ops().grouped_gate_up_swiglu(x, rows, offsets, q)
        first = got if first is None else first
        assert torch.equal(got, first)
    ops().check_async_errors()
    codes, scales, zeros = ops().unpack_int4(q)
    at = torch.arange(hidden, device="cuda") // group
    bounds = offsets.tolist()
    for e in (0, 7, experts - 1):
        w = scales[e].double()[:, at] * (codes[e].double() - zeros[e].double()[:, at])
        a, b = bounds[e], bounds[e + 1]
        near(first[a:b], *gated(x[rows[a:b].long()], w))


# -- streams, graphs, refusals -----------------------------------------------------------
@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("m", [4, 120])
def test_recorded_calls_follow_their_inputs(m):
    g = gen(12)
    q = ops().quantize_int4(matrix((2 * 96, 264), g), 64, halves=2)
    d = ops().quantize_int4(matrix((264, 96), g), 32)
    x = torch.randn((m, 264), generator=g, device="cuda").to(torch.bfloat16)

    def block(v):
        return ops().linear(ops().gate_up_swiglu(v, q), d)
    block(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(x)
        graphs.append((graph, y))
    for seed in (1, 2):
        x.copy_(torch.randn((m, 264), generator=gen(seed), device="cuda"))
        want = block(x)
        for graph, y in graphs + graphs[::-1]:
            graph.replay()
            assert torch.equal(y, want)


@pytest.mark.usefixtures("kernel")
def test_calls_on_two_streams():
    g = gen(13)
    q = ops().quantize_int4(matrix((512, 1024), g), 128)
    xs = [torch.randn((m, 1024), generator=g, device="cuda").to(torch.bfloat16) for m in (5, 130)]
    want = [ops().linear(x, q) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops().linear(xs[i], q))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_a_row_does_not_depend_on_its_company():
    g = gen(14)
    for dtype in (torch.bfloat16, torch.float32):
        q = ops().quantize_int4(matrix((200, 1000), g), 64)
        x = torch.randn((14, 1000), generator=g, device="cuda").to(dtype)
        whole = ops().linear(x, q)
        for i in (0, 5, 13):
            assert torch.equal(whole[i:i + 1], ops().linear(x[i:i + 1], q))


def test_refusals():
    o = ops()
    w = matrix((64, 128), gen(1))
    q = o.quantize_int4(w, 32)
    x = torch.ones((2, 128), device="cuda")
    offsets = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for call in (
            lambda: o.quantize_int4(w.half()),                       # element type
            lambda: o.quantize_int4(w.cpu()),                        # device
            lambda: o.quantize_int4(w.t()),                          # order
            lambda: o.quantize_int4(w, 48),                          # group
            lambda: o.quantize_int4(w[0]),                           # a vector
            lambda: o.quantize_int4(w[:0]),                          # no rows
            lambda: o.quantize_int4(w[:63].contiguous(), 32, 2),     # an odd number in halves
            lambda: o.quantize_int4(w, 32, 3),
            lambda: o.linear(x.half(), q),
            lambda: o.linear(x.cpu(), q),
            lambda: o.linear(x[:, ::2], q),
            lambda: o.linear(x[:, :64].contiguous(), q),             # inner size
            lambda: o.linear(x, q, out_dtype=torch.bfloat16),        # narrower than the input
            lambda: o.gate_up_swiglu(x, q),                          # one half
            lambda: o.linear(x, o.quantize_int4(w, 32, 2)),          # two halves
            lambda: o.grouped_down(x, offsets, q),                   # not per expert
            lambda: o.linear(x, o.quantize_int4(w.view(1, 64, 128), 32)),
            lambda: o.grouped_down(x, offsets, o.quantize_int4(w.view(2, 32, 128), 32)),
            lambda: o.unpack_int4(w),
            lambda: o.linear_act(x, q, "silu")):
        with pytest.raises((o.KernelError, KeyError)):
            call()
    codes, scales, zeros = o.unpack_int4(q)
    for args in ((codes + 16, scales, zeros), (codes, scales, zeros + 16),
                 (codes.int(), scales, zeros), (codes, scales.float(), zeros),
                 (codes, scales[:, :1].contiguous(), zeros)):
        with pytest.raises(o.KernelError):
            o.pack_int4(*args, 32)
