"""Models held in four bits beside the models of their codes: two folders with the same numbers, the
second one's held matrices being what the first one's codes stand for."""
import host_ops as H
from inferx_b200.engine.runtime import load_model
from inferx_b200.weights.loader import RandomSource
from inferx_b200.weights.random_model import write_random_model


def held_names(cfg):
    """The tensors whose entries a run with matrices in four bits holds that way."""
    _, model = load_model(config_json=cfg, source=RandomSource(1), dtype="float32", device="cpu",
                          ops=H, int4_group=32)
    return {d.name for b in model.blocks for p in b.parts() if hasattr(p, "int4_weights")
            for d in p.tensors() if d.keep == "param" and len(d.shape) == 2 and min(d.shape) > 1}


def folders(cfg, path, seed, group, dtype, adjust):
    names = held_names(cfg)
    assert names
    write_random_model(cfg, str(path / "m"), seed=seed, dtype=str(dtype)[6:], adjust=adjust)

    def of_codes(name, t):
        t = adjust(name, t).to(dtype).float()
        return H.quantize_int4(t, group).dense() if name in names else t
    write_random_model(cfg, str(path / "r"), seed=seed, dtype="float32", adjust=of_codes)
    return str(path / "m"), str(path / "r")
