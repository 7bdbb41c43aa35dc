"""Every design with its matrices held in four bits where its parts name them, replayed against its plain
model of what the codes stand for, in 32 bits and in bfloat16, eagerly and from recorded steps.  Bounds
are those of the designs' own tests: codes are exact, so nothing is added to them."""
import pytest
import torch

import biguzen_cases as bk
import dominex_cases as dk
import fudulix_cases as fk
import int4_models
import mapovik_cases as mk
import model_cases as mc
import tinapel_cases as tk
import traces
import zuzisun_cases as zk
from inferx_b200.engine.replay import ReplaySession

pytestmark = pytest.mark.gpu

CASES = {"ZA": (zk, zk.ZA, 32), "ZB": (zk, zk.ZB, 64), "TA": (tk, tk.TA, 32), "TC": (tk, tk.TC, 64),
         "MA": (mk, mk.MA, 32), "MC": (mk, mk.MC, 128), "FA": (fk, fk.FA, 32), "FB": (fk, fk.FB, 64),
         "FC": (fk, fk.FC, 128), "DA": (dk, dk.DA, 32), "DC": (dk, dk.DC, 64),
         "BA": (bk, bk.BA, 32), "BB": (bk, bk.BB, 64), "BC": (bk, bk.BC, 128)}


def bound_for(cases, dtype, folder, reqs):
    name = str(dtype)[6:]
    if hasattr(cases, "bound_for"):
        return cases.bound_for(name, folder, reqs)
    return (cases.f32_bound if name == "float32" else cases.bf16_bound)(folder, reqs)


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,graphs", [("mixed", False), ("tail", True)])
def test_replay(tmp_path, name, dtype, kind, graphs):
    cases, cfg, group = CASES[name]
    mine, of_codes = int4_models.folders(cfg, tmp_path, 11, group, dtype, cases.sharpen)
    reqs = cases.make_requests(cfg, [5, 37, 45, 2], 11)
    steps = mc.TRACE_KINDS[kind](reqs)
    sess = ReplaySession(mine, str(dtype)[6:], traces.peak_tokens(steps), page_size=8, max_live=4,
                         int4_group=group, use_graphs=graphs)
    assert sess.runtime.model.int4_share > 0
    rows = mc.run_trace(sess, steps)
    sess.executor.poll_errors()
    if dtype == torch.bfloat16 and hasattr(cases, "decisive_rows"):
        keep = cases.decisive_rows(of_codes, reqs)
        rows = {k: v for k, v in rows.items() if k in keep}
    if rows:
        mc.compare(rows, cases.reference_rows(of_codes, reqs),
                   bound_for(cases, dtype, of_codes, reqs), f"{name}/{kind}")


# nine chunks of K and a short one, experts with enough rows for the tensor cores
WIDE = {
    "architectures": ["Qwen2MoeForCausalLM"], "model_type": "qwen2_moe",
    "num_hidden_layers": 2, "hidden_size": 1160, "num_attention_heads": 9,
    "num_key_value_heads": 3, "head_dim": 64, "num_experts": 4, "num_experts_per_tok": 2,
    "moe_intermediate_size": 648, "shared_expert_intermediate_size": 1096,
    "decoder_sparse_step": 1, "mlp_only_layers": [], "norm_topk_prob": True, "vocab_size": 300,
    "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "use_sliding_window": False,
    "tie_word_embeddings": False, "torch_dtype": "float32",
}


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,graphs", [("whole", False), ("mixed", False), ("tail", True)])
def test_many_chunks(tmp_path, group, dtype, kind, graphs):
    mine, of_codes = int4_models.folders(WIDE, tmp_path, 5, group, dtype, mc.sharpen_wide)
    reqs = mc.make_requests(WIDE, [150, 3, 60], 5)
    steps = mc.TRACE_KINDS[kind](reqs)
    sess = ReplaySession(mine, str(dtype)[6:], traces.peak_tokens(steps), page_size=16, max_live=3,
                         int4_group=group, use_graphs=graphs)
    rows = mc.run_trace(sess, steps)
    sess.executor.poll_errors()
    mc.compare(rows, mc.reference_rows(of_codes, reqs),
               mc.bound_for(str(dtype)[6:], of_codes, reqs), f"{kind}/{group}")
