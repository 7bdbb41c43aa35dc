"""How much of a model four bits hold, and that a user hears of it."""
import pytest

import host_ops as H
import zuzisun_cases as zk
from conftest import TINY_A, TINY_B
from inferx_b200.engine.engine import Engine, EngineConfig
from inferx_b200.engine.runtime import load_model
from inferx_b200.weights.loader import RandomSource


@pytest.mark.parametrize("cfg", [TINY_A, TINY_B])
def test_every_matrix_of_the_layers_is_held(cfg):
    _, model = load_model(config_json=cfg, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H, int4_group=32)
    assert model.int4_share == 1.0
    _, plain = load_model(config_json=cfg, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H)
    assert plain.int4_share == 0.0


def test_mixers_that_keep_their_matrices_are_counted():
    """Latent attention keeps its projections; the feed-forwards beside it are held."""
    _, model = load_model(config_json=zk.ZA, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H, int4_group=32)
    held = sum(p.gate_up_w.numel() + p.down_w.numel() for b in model.blocks for p in b.parts()
               if hasattr(p, "gate_up_w"))
    kept = sum(d.shape[0] * d.shape[1] for b in model.blocks for p in b.parts()
               for d in p.tensors() if d.keep == "param" and len(d.shape) == 2
               and min(d.shape) > 1 and not hasattr(p, "gate_up_w"))
    assert held and kept
    assert model.int4_share == pytest.approx(held / (held + kept))


def test_the_engine_says_so():
    def stats(**kw):
        return Engine.create(EngineConfig(config_json=zk.ZA, dtype="float32", device="cpu",
                                          max_model_len=32, max_num_seqs=1, block_size=4,
                                          enforce_eager=True, **kw), ops=H).stats()
    assert 0.0 < stats(quantization="int4", quantization_group=32)["int4_share"] < 1.0
    assert "int4_share" not in stats()
