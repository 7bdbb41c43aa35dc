"""Weights held in four bits, on the CPU: which matrices of a model are, what the options take and
refuse, and that a model held so is the model whose matrices are what the codes stand for.  The
kernels are replaced by their plain statements (tests/host_ops.py)."""

import pytest
import torch

import biguzen_cases as bk
import fudulix_cases as fk
import host_ops as H
import model_cases as mc
import traces
from conftest import TINY_A, TINY_B
from inferx_b200.engine.engine import Engine, EngineConfig, Request
from inferx_b200.engine.replay import ReplaySession
from inferx_b200.engine.runtime import load_model
from inferx_b200.kernels import ops as kernel_ops
from inferx_b200.sampling.params import SamplingParams
from inferx_b200.weights.loader import CheckpointSource, RandomSource


class Rounded(CheckpointSource):
    """The folder's tensors; the matrices that go into four bits as what their codes stand for."""

    def __init__(self, folder, group, names):
        super().__init__(folder)
        self.group, self.held = group, names

    def fetch(self, decl):
        t = super().fetch(decl)
        if decl.name.endswith(self.held):
            return H.quantize_int4(t.float(), self.group).dense()
        return t


HELD = ("q_proj.weight", "k_proj.weight", "v_proj.weight", "o_proj.weight", "gate_proj.weight",
        "up_proj.weight", "down_proj.weight")


@pytest.mark.parametrize("cfg,group", [(TINY_A, 32), (TINY_B, 64), (TINY_B, 128)])
def test_a_model_in_four_bits_is_the_model_of_its_codes(tmp_path, cfg, group):
    folder = mc.make_model_dir(cfg, tmp_path / "m", 3)
    reqs = mc.make_requests(cfg, [5, 17, 33], 3)
    steps = mc.TRACE_KINDS["mixed"](reqs)
    peak = traces.peak_tokens(steps)
    held = ReplaySession(folder, "float32", peak, page_size=4, max_live=4, device="cpu", ops=H,
                         int4_group=group)
    rows = mc.run_trace(held, steps)
    _, plain = load_model(folder, dtype="float32", device="cpu", ops=H,
                          source=Rounded(folder, group, HELD))
    other = ReplaySession(folder, "float32", peak, page_size=4, max_live=4, device="cpu", ops=H)
    for mine, theirs in zip(other.runtime.model.blocks, plain.blocks):
        for a, b in zip(mine.parts(), theirs.parts()):
            a.__dict__.update(b.__dict__)
    want = mc.run_trace(other, steps)
    assert rows.keys() == want.keys() and rows
    for k in rows:
        # the same statements of the same fp32 numbers
        assert torch.equal(rows[k], want[k])


@pytest.mark.parametrize("cfg", [TINY_A, TINY_B])
def test_which_matrices_are_held(cfg):
    _, model = load_model(config_json=cfg, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H, int4_group=32)
    assert isinstance(model.embed, torch.Tensor) and isinstance(model.head, torch.Tensor)
    for block in model.blocks:
        for part in block.parts():
            for name, halves in getattr(part, "int4_weights", {}).items():
                w = getattr(part, name)
                assert isinstance(w, H.HostInt4) and w.halves == halves and w.group_size == 32
            if hasattr(part, "router_w"):
                assert isinstance(part.router_w, torch.Tensor)
                assert isinstance(part.shared.gate_up_w, H.HostInt4)
                assert part._shared_bytes == (part.shared.gate_up_w.nbytes
                                              + part.shared.down_w.nbytes)


@pytest.mark.parametrize("cfg", [fk.FA, bk.BA])
def test_other_designs_run(cfg):
    """Experts without a gate, biased units, prepared attention: what names matrices has them
    held, what does not keeps them."""
    _, model = load_model(config_json=cfg, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H, int4_group=32)
    held = [getattr(p, n) for b in model.blocks for p in b.parts()
            for n in getattr(p, "int4_weights", {})]
    assert held and all(isinstance(w, H.HostInt4) for w in held)


def test_generation_through_the_engine(tmp_path):
    folder = mc.make_model_dir(TINY_A, tmp_path / "m", 5)
    engine = Engine.create(EngineConfig(model=folder, dtype="float32", device="cpu",
                                        max_model_len=64, max_num_seqs=2, block_size=4,
                                        enforce_eager=True, quantization="int4",
                                        quantization_group=32), ops=H)
    done = engine.generate([Request([1, 2, 3], SamplingParams(max_tokens=5)),
                            Request([7] * 20, SamplingParams(max_tokens=3))])
    assert [len(c.output_tokens) for c in done] == [5, 3]


def test_options():
    assert EngineConfig().int4_group() == 0
    assert EngineConfig(quantization="none").int4_group() == 0
    assert EngineConfig(quantization="int4").int4_group() == 128
    for bad in (dict(quantization="int8"), dict(quantization="int4", quantization_group=48)):
        with pytest.raises(ValueError):
            EngineConfig(**bad).int4_group()
    with pytest.raises(ValueError):
        Engine.create(EngineConfig(config_json=TINY_A, device="cpu", quantization="fp8"), ops=H)


def test_command_line(capsys):
    from inferx_b200.engine import cli
    assert cli.main(["x", "--prompt-ids", "1", "--quantization", "fp8"]) == 2
    assert "--quantization" in capsys.readouterr().err
    args = cli.build_parser().parse_args(["x", "-q", "int4", "--quantization-group", "64"])
    assert not cli._refusals(args) and args.quantization_group == 64
    with pytest.raises(SystemExit):
        cli.build_parser().parse_args(["x", "--quantization-group", "48"])
    capsys.readouterr()


# -- the faces, as far as they go without a device ----------------------------------------
def test_refusals_without_a_device():
    w = torch.zeros((4, 64))
    with pytest.raises(kernel_ops.KernelError, match="CUDA"):
        kernel_ops.quantize_int4(w)
    with pytest.raises(kernel_ops.KernelError, match="CUDA"):
        kernel_ops.pack_int4(w.to(torch.uint8), w, w.to(torch.uint8))
    with pytest.raises(kernel_ops.KernelError, match="Int4Weight"):
        kernel_ops.unpack_int4(w)
    for shape, group, halves in (((64,), 32, 1), ((0, 64), 32, 1), ((4, 64), 16, 1),
                                 ((3, 64), 32, 2), ((4, 64), 32, 0)):
        with pytest.raises(kernel_ops.KernelError):
            kernel_ops._int4_empty("quantize_int4", shape, group, halves, "cpu")


def test_the_layout_has_whole_strips_and_chunks():
    q = kernel_ops._int4_empty("quantize_int4", (3, 34, 200), 64, 2, "cpu")
    assert tuple(q.data.shape) == (6, 2, 2, 256 + 32)     # 17 rows a half, 200 columns
    assert (q.experts, q.cols, q.inner, q.numel()) == (3, 17, 200, 3 * 34 * 200)
    assert "halves=2" in repr(q) and q.nbytes == q.data.nbytes
    one = kernel_ops._int4_empty("quantize_int4", (16, 128), 128, 1, "cpu")
    assert tuple(one.data.shape) == (1, 1, 1, 272)


def test_the_plain_statement_of_quantising():
    """Against the definition written out entry by entry."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn((3, 70), generator=g)
    q = H.quantize_int4(w, 32)
    for r in range(3):
        for i, k0 in enumerate((0, 32, 64)):
            part = w[r, k0:k0 + 32].double()
            lo, hi = min(0.0, part.min().item()), max(0.0, part.max().item())
            # nearest of the bfloat16 numbers about the quotient
            near = torch.tensor((hi - lo) / 15, dtype=torch.float32).bfloat16()
            bits = near.view(torch.int16)
            around = torch.stack([(bits + d).view(torch.bfloat16) for d in (-1, 0, 1)]).double()
            s = around[(around - (hi - lo) / 15).abs().argmin()].item()
            assert q.scales[r, i].item() == s
            zero = min(15, max(0, round(-lo / s)))
            assert q.zeros[r, i].item() == zero
            for j, v in enumerate(part.tolist()):
                assert q.codes[r, k0 + j].item() == min(15, max(0, round(v / s) + zero))
    # an entry is off by half a step, or, at the range's ends, by what the scale's rounding took
    step = q.scales.float()[:, torch.arange(70) // 32]
    assert ((q.dense() - w).abs() <= step * (0.5 + 16 * 2.0 ** -8)).all()




def test_a_weight_keeps_the_tensor_that_its_record_names():
    import copy
    import pickle
    q = kernel_ops._int4_empty("here", (4, 96, 200), 64, 2, "cpu")
    q.data.random_(-2 ** 31, 2 ** 31 - 1)
    assert q._record.data == q.data.data_ptr() and q._record.cols == 48
    with pytest.raises(AttributeError):
        q.data = q.data.clone()
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert other._record.data == other.data.data_ptr() != q.data.data_ptr()
        assert torch.equal(other.data, q.data) and other.shape == q.shape
        assert (other.halves, other.group_size, other.cols, other.inner, other.experts) == \
            (2, 64, 48, 200, 4)
    assert copy.copy(q).data is q.data


def test_a_model_whose_parts_name_no_matrices_is_refused(monkeypatch):
    from inferx_b200.parts import block
    monkeypatch.setattr(block, "hold_in_int4", lambda part, ctx: 0)
    with pytest.raises(ValueError, match="no part of this model"):
        load_model(config_json=TINY_A, source=RandomSource(1), dtype="float32", device="cpu", ops=H,
                   int4_group=32)


@pytest.mark.parametrize("rows,k,n,dtype,want", [
    (1, 20480, 3584, torch.bfloat16, "few"), (16, 20480, 3584, torch.bfloat16, "few"),
    (64, 20480, 3584, torch.bfloat16, "many"), (64, 512, 512, torch.bfloat16, "few"),
    (65, 512, 512, torch.bfloat16, "many"), (1024, 128, 16, torch.bfloat16, "many"),
    (48, 512, 512, torch.float32, "few"), (49, 512, 512, torch.float32, "many"),
    (17, 20480, 3584, torch.float32, "many"), (0, 64, 64, torch.float32, "none")])
def test_which_kernel_takes_a_call(monkeypatch, rows, k, n, dtype, want):
    taken = []
    monkeypatch.setattr(kernel_ops, "_int4_operands", lambda *a: None)
    monkeypatch.setattr(kernel_ops, "_int4_stream", lambda *a, **kw: taken.append("few"))
    monkeypatch.setattr(kernel_ops, "_int4_tc", lambda *a, **kw: taken.append("many"))
    q = kernel_ops._int4_empty("here", (n, k), 128, 1, "meta")
    out = kernel_ops.linear(torch.empty((rows, k), dtype=dtype, device="meta"), q)
    assert taken == ([] if want == "none" else [want])
    assert want != "none" or tuple(out.shape) == (0, n)
