"""Products with weights held in four bits, as cases that can be timed and checked.

A weight matrix is cut along its inner size into groups of 32, 64 or 128 entries (the last one
may be shorter).  A group keeps one code of four bits per entry, a bfloat16 scale and a zero
point of four bits: an entry stands for ``scale * (code - zero)``.  Four operators:

* ``quantize``: a matrix into codes, scales and zero points.  With lo = min(0, the group's least
  entry) and hi = max(0, its greatest), scale = (hi - lo) / 15 rounded to bfloat16,
  zero = -lo / scale and code = entry / scale + zero, both quotients rounded to the nearest whole
  number (ties to even) and kept within 0..15.
* ``linear``: x . W^T.
* ``gated``: silu(x . Wg^T) * (x . Wu^T), the front of a gated feed-forward.
* ``experts``: the same two products and the way back down for the rows that a router gave to
  each expert, ``act[r] = silu(x[rows[r]] . Wg[e]^T) * (x[rows[r]] . Wu[e]^T)`` and
  ``y[r] = act[r] . Wd[e]^T``.

Sizes are those of the models that ``bench.py`` runs (hidden 2048 with 60 experts of 1408, a
shared expert of 5632; hidden 3584 with a shared expert of 20480), and generic odd ones.
"""
import math

import torch

own = False

BF16, F32 = "bfloat16", "float32"


def listed():
    return [
        # loading a model: the attention's projections of one layer
        dict(name="quantize_projections", op="quantize", dtype=BF16, n=6144, k=2048, group=128),
        # loading a 32-bit model of odd sizes: the last group is shorter than the others
        dict(name="quantize_odd_fp32", op="quantize", dtype=F32, n=1030, k=1000, group=32),
        # one sequence decoding: attention's output projection; launch latency counts
        dict(name="linear_one_token", op="linear", dtype=BF16, tokens=1, k=2048, n=2048,
             group=128, out=BF16),
        # eight sequences decoding: the shared expert's way down, widened for the stream
        dict(name="linear_eight_tokens", op="linear", dtype=BF16, tokens=8, k=5632, n=2048,
             group=128, out=F32),
        # a short prompt through an odd 32-bit layer
        dict(name="linear_odd_fp32", op="linear", dtype=F32, tokens=33, k=1000, n=515,
             group=32, out=F32),
        # a prompt portion: the attention's projections
        dict(name="linear_prompt", op="linear", dtype=BF16, tokens=2048, k=2048, n=6144,
             group=64, out=BF16),
        # the largest: a long prompt portion through the large shared expert's way down
        dict(name="linear_long_prompt", op="linear", dtype=BF16, tokens=4096, k=20480, n=3584,
             group=128, out=BF16),
        # one sequence decoding: the shared expert's front
        dict(name="gated_one_token", op="gated", dtype=BF16, tokens=1, k=2048, n=5632, group=128),
        # a ragged prompt portion through the same
        dict(name="gated_prompt", op="gated", dtype=BF16, tokens=613, k=2048, n=5632, group=128),
        # one sequence decoding in 32 bits: the routed experts
        dict(name="experts_one_token_fp32", op="experts", dtype=F32, tokens=1, k=2048, n=1408,
             group=64, experts=60, top=4),
        # eight sequences decoding: the routed experts
        dict(name="experts_eight_tokens", op="experts", dtype=BF16, tokens=8, k=2048, n=1408,
             group=128, experts=60, top=4),
        # a prompt portion: the routed experts
        dict(name="experts_prompt", op="experts", dtype=BF16, tokens=2048, k=2048, n=1408,
             group=128, experts=60, top=4),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A matrix size: mostly a multiple of 64, now and then any number."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, (n + 32) // 64 * 64)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gated", "experts"])
    case = dict(op=op, dtype=BF16 if rng.random() < 0.75 else F32,
                group=rng.choice([32, 64, 128, 128]))
    if op == "quantize":
        case.update(n=_size(rng, 64, 12000), k=_size(rng, 200, 6000))
    elif op == "linear":
        case.update(tokens=_spread(rng, 1, 4096), k=_size(rng, 200, 20480), n=_size(rng, 64, 12000),
                    out=rng.choice([BF16, F32]) if case["dtype"] == BF16 else F32)
    elif op == "gated":
        case.update(tokens=_spread(rng, 1, 4096), k=_size(rng, 200, 4096), n=_size(rng, 64, 8000))
    else:
        experts = rng.choice([8, 16, 32, 60, 64])
        case.update(tokens=_spread(rng, 1, 2048), k=_size(rng, 256, 2560), n=_size(rng, 64, 2048),
                    experts=experts, top=rng.choice([1, 2, 4, 6, 8]))
    # no more work than the largest listed case (products of 32-bit numbers are dearer)
    most = max(work(c)["flops"] for c in listed()) / (8 if case["dtype"] == F32 else 1)
    while "tokens" in case and case["tokens"] > 1 and work(case)["flops"] > most:
        case["tokens"] = case["tokens"] // 2
    return case


def _groups(case, k=None):
    return -(-(k or case["k"]) // case["group"])


def _weight_bytes(case, n, k):
    """Codes of half a byte, scales of two, zero points of half a byte."""
    return n * k // 2 + n * _groups(case, k) * 2.5


def _active(case):
    """Experts that rows are expected to reach."""
    e, picks = case["experts"], case["tokens"] * case["top"]
    return min(e, e * (1.0 - (1.0 - 1.0 / e) ** picks))


def work(case):
    n, k, size = case["n"], case["k"], 2 if case["dtype"] == BF16 else 4
    if case["op"] == "quantize":
        # codes and zero points come back as bytes, scales in bfloat16
        return dict(bytes=n * k * (size + 1) + n * _groups(case) * 3, flops=4 * n * k)
    t = case["tokens"]
    if case["op"] == "linear":
        o = 2 if case["out"] == BF16 else 4
        return dict(bytes=_weight_bytes(case, n, k) + t * k * size + t * n * o, flops=2 * t * n * k)
    if case["op"] == "gated":
        return dict(bytes=_weight_bytes(case, 2 * n, k) + t * k * size + t * n * size,
                    flops=4 * t * n * k)
    rows = t * case["top"]
    weights = _weight_bytes(case, 2 * n, k) + _weight_bytes(case, k, n)
    return dict(bytes=int(_active(case) * weights) + t * k * size + rows * (n + k) * size,
                flops=6 * rows * n * k)


# -- the plain forms ---------------------------------------------------------------------
def _cut(w, group):
    """[..., k] -> [..., groups, group], zeros behind the last entry."""
    g = -(-w.shape[-1] // group)
    return torch.nn.functional.pad(w, (0, g * group - w.shape[-1])).unflatten(-1, (g, group))


def _to_bf16(t):
    """float64 (not negative) to bfloat16 in one rounding: to 32 bits towards zero first, with
    the last bit set where something was left, then to nearest."""
    f = t.to(torch.float32)
    f = torch.where(f.double() > t, torch.nextafter(f, torch.zeros_like(f)), f)
    odd = (f.double() != t).to(torch.int32)
    return (f.view(torch.int32) | odd).view(torch.float32).to(torch.bfloat16)


def _quantize(w, group):
    """Codes, scales and zero points.  In 64 bits: a quotient next to a border between two codes
    must fall on its own side."""
    cut = _cut(w, group).double()
    lo, hi = cut.amin(-1).clamp(max=0.0), cut.amax(-1).clamp(min=0.0)
    scale = _to_bf16((hi - lo) / 15.0)
    step = scale.double()
    some = step > 0
    step = torch.where(some, step, torch.ones_like(step))
    zero = torch.where(some, torch.round(-lo / step).clamp(0, 15), torch.zeros_like(step))
    code = (torch.round(cut / step[..., None]) + zero[..., None]).clamp(0, 15)
    code = torch.where(some[..., None], code, torch.zeros_like(code))
    return (code.flatten(-2)[..., :w.shape[-1]].to(torch.uint8).contiguous(), scale,
            zero.to(torch.uint8))


def _entries(packed, group, dtype=torch.float32):
    """What codes stand for: a small whole number times eight bits, exact in 32 bits."""
    codes, scales, zeros = packed
    cut = _cut(codes, group).to(dtype) - zeros.to(dtype)[..., None]
    return (cut * scales.to(dtype)[..., None]).flatten(-2)[..., :codes.shape[-1]]


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _expert_products(st, x, gate_up, down, round_to):
    """Rows of one expert side by side, [experts with rows, most rows, .]; back in the rows'
    order at the end."""
    rows_of, place = st["rows_of"], st["place"]
    n = st["case"]["n"]
    front = torch.bmm(x[rows_of.flatten()].view(*rows_of.shape, -1), gate_up.transpose(1, 2))
    act = (_silu(front[..., :n]) * front[..., n:]).to(round_to)
    y = torch.bmm(act.to(gate_up.dtype), down.transpose(1, 2))
    return act.flatten(0, 1)[place], y.flatten(0, 1)[place]


# -- inputs ------------------------------------------------------------------------------
def _weights(shape, gen):
    """Entries as trained matrices have them: small, rows of differing size, a few far out."""
    w = torch.randn(shape, generator=gen, device="cuda") * 0.02
    w *= 0.5 + torch.rand((*shape[:-1], 1), generator=gen, device="cuda")
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 1e-3, w * 5.0, w)


def _rows(tokens, k, gen):
    """Normed activations: unit size, a few channels much larger."""
    x = torch.randn((tokens, k), generator=gen, device="cuda")
    return torch.where(torch.arange(k, device="cuda") % 89 == 7, x * 8.0, x)


def _handle(packed, case, halves=1):
    """The laid out weights that a program keeps."""
    from inferx_b200.kernels import ops
    return ops.pack_int4(*packed, case["group"], halves=halves)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, n, k, group = case["op"], case["n"], case["k"], case["group"]
    dtype = torch.bfloat16 if case["dtype"] == BF16 else torch.float32
    st = dict(case=case)
    if op == "quantize":
        st["w"] = _weights((n, k), gen).to(dtype)
        return st
    st["x"] = _rows(case["tokens"], k, gen).to(dtype)
    if op == "linear":
        w = _quantize(_weights((n, k), gen).to(dtype), group)
        st["w"] = _handle(w, case) if own else w
        st["out"] = torch.bfloat16 if case["out"] == BF16 else torch.float32
        return st
    if op == "gated":
        w = _quantize(_weights((2 * n, k), gen).to(dtype), group)
        st["w"] = _handle(w, case, halves=2) if own else w
        return st
    # routed rows: every token's experts are distinct, some experts more liked than others
    e, top, tokens = case["experts"], case["top"], case["tokens"]
    score = torch.randn((tokens, e), generator=gen, device="cuda")
    score += 0.5 * torch.randn((1, e), generator=gen, device="cuda")
    chosen = score.topk(top, dim=-1).indices.flatten()
    order = torch.sort(chosen, stable=True).indices
    counts = torch.bincount(chosen, minlength=e)
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
    st["rows"] = (order // top).to(torch.int32)
    st["offsets"] = offsets
    gate_up = _quantize(_weights((e, 2 * n, k), gen).to(dtype), group)
    down = _quantize(_weights((e, k, n), gen).to(dtype), group)
    if own:
        st["gate_up"] = _handle(gate_up, case, halves=2)
        st["down"] = _handle(down, case)
        return st
    # the plain form's view of the routing: the experts with rows, and for each the tokens
    # of its rows (the first token where it has fewer than the most)
    st["gate_up"], st["down"] = gate_up, down
    active = counts.nonzero().flatten()
    most = int(counts.max())
    place = torch.arange(most, device="cuda")
    at = offsets[active].long()[:, None] + place
    inside = place < counts[active][:, None]
    st["active"] = active
    st["rows_of"] = torch.where(inside, st["rows"].long()[at.clamp(max=order.numel() - 1)], 0)
    st["place"] = inside.flatten().nonzero().flatten()
    return st


# -- one pass ----------------------------------------------------------------------------
def run(st):
    case = st["case"]
    op, group = case["op"], case["group"]
    if own:
        from inferx_b200.kernels import ops
        if op == "quantize":
            return ops.unpack_int4(ops.quantize_int4(st["w"], group))
        if op == "linear":
            return ops.linear(st["x"], st["w"], out_dtype=st["out"])
        if op == "gated":
            return ops.gate_up_swiglu(st["x"], st["w"])
        act = ops.grouped_gate_up_swiglu(st["x"], st["rows"], st["offsets"], st["gate_up"])
        return act, ops.grouped_down(act, st["offsets"], st["down"])
    if op == "quantize":
        return _quantize(st["w"], group)
    x = st["x"].float()
    if op == "linear":
        return torch.mm(x, _entries(st["w"], group).t()).to(st["out"])
    if op == "gated":
        front = torch.mm(x, _entries(st["w"], group).t())
        return (_silu(front[:, :case["n"]]) * front[:, case["n"]:]).to(st["x"].dtype)
    pick = [tuple(t[st["active"]] for t in st[name]) for name in ("gate_up", "down")]
    act, y = _expert_products(st, x, _entries(pick[0], group), _entries(pick[1], group),
                              st["x"].dtype)
    return act, y.to(st["x"].dtype)


# -- the definition in 64 bits -----------------------------------------------------------
def _exact_scale(spread):
    """spread / 15 rounded to eight significant bits, ties to even."""
    quotient = spread / 15.0
    mantissa, exponent = torch.frexp(quotient)                 # in [1/2, 1)
    return torch.ldexp(torch.round(mantissa * 256.0) / 256.0, exponent)


def _exact_codes(w, group):
    """Group by group of whole rows, each entry's group named by its place."""
    n, k = w.shape
    of = torch.arange(k, device=w.device) // group
    g = int(of[-1]) + 1
    zeros = torch.zeros((n, g), dtype=torch.float64, device=w.device)
    low = zeros.scatter_reduce(1, of.expand(n, k), w, "amin", include_self=True)
    high = zeros.scatter_reduce(1, of.expand(n, k), w, "amax", include_self=True)
    scale = _exact_scale(high - low)
    zero = torch.round(-low / scale).clamp(0, 15)
    code = (torch.round(w / scale[:, of]) + zero[:, of]).clamp(0, 15)
    return code, scale, zero


def _exact_matrix(w, group):
    flat = w.double().flatten(0, -2)
    code, scale, zero = _exact_codes(flat, group)
    of = torch.arange(flat.shape[1], device=w.device) // group
    return ((code - zero[:, of]) * scale[:, of]).view(w.shape)


def exact(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, n, k, group = case["op"], case["n"], case["k"], case["group"]
    dtype = torch.bfloat16 if case["dtype"] == BF16 else torch.float32
    if op == "quantize":
        code, scale, zero = _exact_codes(_weights((n, k), gen).to(dtype).double(), group)
        return code.to(torch.uint8), scale, zero.to(torch.uint8)
    x = _rows(case["tokens"], k, gen).to(dtype).double()
    if op == "linear":
        return x @ _exact_matrix(_weights((n, k), gen).to(dtype), group).t()
    if op == "gated":
        w = _exact_matrix(_weights((2 * n, k), gen).to(dtype), group)
        gate, up = x @ w[:n].t(), x @ w[n:].t()
        return gate * torch.sigmoid(gate) * up
    e, top, tokens = case["experts"], case["top"], case["tokens"]
    score = torch.randn((tokens, e), generator=gen, device="cuda")
    score += 0.5 * torch.randn((1, e), generator=gen, device="cuda")
    chosen = score.topk(top, dim=-1).indices.flatten()
    order = torch.sort(chosen, stable=True).indices
    bounds = [0] + torch.bincount(chosen, minlength=e).cumsum(0).tolist()
    gate_up = _weights((e, 2 * n, k), gen).to(dtype)
    down = _weights((e, k, n), gen).to(dtype)
    act = torch.empty((tokens * top, n), dtype=torch.float64, device="cuda")
    y = torch.empty((tokens * top, k), dtype=torch.float64, device="cuda")
    for i in range(e):
        a, b = bounds[i], bounds[i + 1]
        if a == b:
            continue
        w = _exact_matrix(gate_up[i], group)
        mine = x[order[a:b] // top]
        gate, up = mine @ w[:n].t(), mine @ w[n:].t()
        act[a:b] = gate * torch.sigmoid(gate) * up
        y[a:b] = act[a:b] @ _exact_matrix(down[i], group).t()
    return act, y
