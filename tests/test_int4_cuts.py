"""Into how many runs of K the tensor-core products with four-bit weights are cut (no GPU needed:
the library's functions only compute)."""
import itertools

import pytest
import torch

from inferx_b200.kernels import ops


def runs_of(experts, halves, cols, chunks, rows, grouped, terms):
    """(runs, chunks of a run) of a call: the scratch holds one set of sums a run."""
    w = ops._Int4Record(None, cols, experts, 128, halves - 1)
    need = ops._int4_entry("ix_int4_tc_scratch")(ops.ctypes.addressof(w), rows, chunks * 128,
                                                 grouped, terms)
    per = rows * cols * halves
    assert need % per == 0
    runs = max(1, need // per)
    return runs, -(-chunks // runs)


def covers(runs, run, chunks):
    """Every run has a chunk at least and one after the other they are the whole of K."""
    ends = [(z * run, min(chunks, (z + 1) * run)) for z in range(runs)]
    return ends[-1][1] == chunks and all(0 < b - a <= run for a, b in ends)


@pytest.mark.parametrize("experts", [1, 2, 3, 4, 5, 8, 16, 33, 64])
def test_no_run_of_an_expert_product_is_empty(experts):
    cut = 0
    for chunks, cols, rows, halves in itertools.product(
            range(1, 161), (1, 100, 128, 256, 300, 512, 1024, 2048),
            (1, 30, 129, 700, 2000, 4096, 4097), (1, 2)):
        for terms in (1, 3):
            runs, run = runs_of(experts, halves, cols, chunks, rows, 1, terms)
            assert 1 <= runs <= 16
            assert covers(runs, run, chunks), (experts, chunks, cols, rows, halves, runs)
            cut += runs > 1
    assert cut


@pytest.mark.parametrize("rows", [1, 17, 64, 200, 613, 2048, 4096, 5000])
def test_no_run_of_one_matrix_is_empty(rows):
    for chunks, cols, halves, terms in itertools.product(range(1, 161, 3), (16, 515, 2048, 6144),
                                                         (1, 2), (1, 3)):
        runs, run = runs_of(1, halves, cols, chunks, rows, 0, terms)
        assert covers(runs, run, chunks), (chunks, cols, rows, halves, runs)


@pytest.mark.parametrize("rows,experts,dtype,want", [
    (1, 60, torch.bfloat16, "few"), (720, 60, torch.bfloat16, "few"),
    (721, 60, torch.bfloat16, "many"), (420, 60, torch.float32, "few"),
    (421, 60, torch.float32, "many"), (12, 1, torch.bfloat16, "few"),
    (13, 1, torch.bfloat16, "many"), (100000, 1025, torch.bfloat16, "few"),
    (100000, 1024, torch.bfloat16, "many"), (0, 4, torch.float32, "none")])
def test_which_kernel_takes_an_expert_product(monkeypatch, rows, experts, dtype, want):
    taken = []
    monkeypatch.setattr(ops, "_chk", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "_int4_operands", lambda *a: None)
    monkeypatch.setattr(ops, "_int4_stream", lambda *a, **kw: taken.append("few"))
    monkeypatch.setattr(ops, "_int4_tc", lambda *a, **kw: taken.append("many"))
    q = ops._int4_empty("here", (experts, 32, 128), 128, 1, "meta")
    out = ops.grouped_down(torch.empty((rows, 128), dtype=dtype, device="meta"),
                           torch.empty(experts + 1, dtype=torch.int32, device="meta"), q)
    assert taken == ([] if want == "none" else [want])
    assert want != "none" or tuple(out.shape) == (0, 32)
