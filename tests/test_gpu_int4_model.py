"""Models whose matrices are held in four bits: replayed against the plain model whose matrices are
what the codes stand for, in 32 bits and in bfloat16, eagerly and from recorded steps, and generated
from.  Bounds are those of the models that are not held so (tests/model_cases.py): the codes are
exact there, so nothing is added to them."""
import pytest
import torch

import host_ops as H
import model_cases as mc
import traces
from conftest import TINY_A, TINY_B
from inferx_b200.engine.engine import Engine, EngineConfig, Request
from inferx_b200.engine.replay import ReplaySession
from inferx_b200.kernels import ops
from inferx_b200.sampling.params import SamplingParams
from inferx_b200.weights.random_model import write_random_model

pytestmark = pytest.mark.gpu

HELD = ("q_proj.weight", "k_proj.weight", "v_proj.weight", "o_proj.weight", "gate_proj.weight",
        "up_proj.weight", "down_proj.weight")


def folders(cfg, path, seed, group, dtype):
    """A model, and the one that a run of it holds: what the codes stand for (made from entries of
    the run's type), the embedding and the head in the run's type."""
    mine = mc.make_model_dir(cfg, path / "m", seed)

    def rounded(name, t):
        t = mc.sharpen(name, t)
        if name.endswith(HELD):
            return H.quantize_int4(t.to(dtype), group).dense()
        if name.endswith(("embed_tokens.weight", "lm_head.weight")):
            return t.to(dtype).float()
        return t
    write_random_model(cfg, str(path / "r"), seed=seed, dtype="float32", adjust=rounded)
    return mine, str(path / "r")


@pytest.mark.parametrize("cfg,group,page", [(TINY_A, 32, 4), (TINY_B, 64, 8), (TINY_B, 128, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,graphs", [("mixed", False), ("whole", False), ("tail", True)])
def test_replay(tmp_path, cfg, group, page, dtype, kind, graphs):
    mine, rounded = folders(cfg, tmp_path, 7, group, dtype)
    reqs = mc.make_requests(cfg, [5, 33, 70, 2], 7)
    steps = mc.TRACE_KINDS[kind](reqs)
    sess = ReplaySession(mine, str(dtype)[6:], traces.peak_tokens(steps), page_size=page,
                         max_live=4, int4_group=group, use_graphs=graphs)
    rows = mc.run_trace(sess, steps)
    bound = 2e-5 if dtype == torch.float32 else mc.bf16_bound(rounded, reqs)
    mc.compare(rows, mc.reference_rows(rounded, reqs), bound, f"{kind}/{group}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_is_the_same_from_recorded_steps(dtype):
    def run(eager):
        engine = Engine.create(EngineConfig(config_json=TINY_B, dtype=dtype, max_model_len=96,
                                            max_num_seqs=3, block_size=8, enforce_eager=eager,
                                            quantization="int4", quantization_group=64))
        done = engine.generate([Request([3, 1, 4, 1, 5], SamplingParams(max_tokens=20)),
                                Request([9] * 40, SamplingParams(max_tokens=12)),
                                Request([2, 6], SamplingParams(max_tokens=20))])
        stats = engine.stats()
        return [c.output_tokens for c in done], stats
    eager, _ = run(True)
    recorded, stats = run(False)
    assert stats["graph_replays"] > 0
    assert recorded == eager


def test_held_weights_take_a_quarter():
    """Codes of half a byte, a word for every 64 entries: 4.5 of 16 bits, and padding to whole
    strips and chunks."""
    w = torch.randn((4, 512, 1024), device="cuda").to(torch.bfloat16)
    q = ops.quantize_int4(w, 64, halves=2)
    assert q.nbytes == w.nbytes * 4.5 / 16
