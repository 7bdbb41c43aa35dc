"""What a model held in four bits leaves of the device's memory: in a process of its own, whose allocator
holds nothing of other tests."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def check():
    import torch

    from conftest import TINY_A
    from inferx_b200.engine.engine import EngineConfig, autosize_pages
    from inferx_b200.engine.runtime import load_model
    from inferx_b200.weights.loader import RandomSource
    # experts of 100 MB a layer in bfloat16
    wide = dict(TINY_A, hidden_size=1024, num_experts=32, moe_intermediate_size=512,
                shared_expert_intermediate_size=512, torch_dtype="bfloat16")
    # (the kernels themselves take some 140 MB of the device once: a first load is not counted)
    load_model(config_json=TINY_A, source=RandomSource(1, device="cuda"), int4_group=128)
    torch.cuda.empty_cache()
    held0, free0 = torch.cuda.memory_allocated(), torch.cuda.mem_get_info()[0]
    _, model = load_model(config_json=wide, source=RandomSource(1, device="cuda"), int4_group=128)
    held = torch.cuda.memory_allocated() - held0
    matrices = 2 * 32 * 3 * 512 * 1024 * 2                   # bytes in bfloat16
    assert held < 0.45 * matrices                            # 4.25 of 16 bits, and what is not held
    # the allocator keeps pieces of 2 and of 20 MB: a few of them, not a layer's matrices
    assert free0 - torch.cuda.mem_get_info()[0] < held + 0.3 * matrices
    assert torch.cuda.memory_reserved() - torch.cuda.memory_allocated() < 0.3 * matrices
    cfg = EngineConfig(config_json=wide, max_model_len=1 << 20, max_num_seqs=4096, block_size=16)
    before = autosize_pages(cfg, model, "cuda")
    torch.cuda.empty_cache()
    after = autosize_pages(cfg, model, "cuda")
    assert before >= 0.999 * after


def test_replaced_matrices_are_given_back():
    child = subprocess.run(
        [sys.executable, "-c", "import test_gpu_int4_memory as t; t.check()"], timeout=300,
        cwd=HERE, env=dict(os.environ, PYTHONPATH=os.pathsep.join([HERE, os.path.dirname(HERE)])),
        stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert child.returncode == 0, child.stdout[-3000:]
