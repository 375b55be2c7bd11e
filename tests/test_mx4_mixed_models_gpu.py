"""Models of which only some parts keep their matrices in 4 bits, in every arrangement that holds such a part, against the same models whose
matrices are tensors of the same values (4 bits and a power of two are exact in bfloat16 and float32)."""
import json

import numpy as np
import pytest
import torch

import model_helpers as mh
import tiny_configs
import tiny_dokulorn
import tiny_gasetar
import tiny_kitonex
import tiny_ligirax
import tiny_paditar
import tiny_revepel
from rust_deeplearning_b200 import Engine, Generator, cli, random_model
from rust_deeplearning_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIGS = {**tiny_dokulorn.CONFIGS, **tiny_gasetar.CONFIGS, **tiny_kitonex.CONFIGS, **tiny_paditar.CONFIGS, **tiny_revepel.CONFIGS}
MATRICES = ("w_qkv", "w_q", "w_o", "w_gate_up", "w_up", "w_down")
# the parts with the offer, by layer, from the configurations
PACKED = {"DA": ["feed_forward 0", "feed_forward 2"], "DC": ["feed_forward 1"],
          "GA": ["feed_forward 1", "mixer 1", "mixer 2"], "GB": ["feed_forward 1", "mixer 0", "mixer 2"],
          "KA": ["feed_forward 2", "mixer 0", "mixer 1", "mixer 2", "mixer 3"], "KC": ["feed_forward 0", "mixer 0", "mixer 1", "mixer 2"],
          "PA": ["feed_forward 0", "feed_forward 2"], "PB": ["feed_forward 0", "feed_forward 1", "feed_forward 3"],
          "PC": ["feed_forward 0", "feed_forward 2"], "PD": ["feed_forward 0", "feed_forward 1"],
          "RA": ["mixer 0", "mixer 3"], "RB": ["mixer 1", "mixer 3"], "RC": ["mixer 1", "mixer 3"]}


def pair(name, dtype):
    """(the model in 4 bits, the same with tensors of the values 4 bits leave, those tensors)"""
    cfg, seed = CONFIGS[name]
    packed, plain = (random_model(cfg, seed, dtype, DEV, weight_format=f) for f in ("mx4", None))
    values, seen = [], []
    for i, (a, b) in enumerate(zip(packed.layers, plain.layers)):
        for role in ("mixer", "feed_forward"):
            for m in MATRICES:
                w = getattr(getattr(a, role, None), m, None)
                if type(w) is ops.Mx4Weight:
                    assert w.shape == tuple(getattr(getattr(b, role), m).shape)
                    values.append(ops.expand_mx4(w, plain.dtype))
                    setattr(getattr(b, role), m, values[-1])
                    seen.append(f"{role} {i}")
    assert sorted(set(seen)) == PACKED[name]
    return packed, plain, values


def near(got, want, dtype, what):
    """Two results that are each within the model tests' tolerance of the true one."""
    want = want.double().cpu().numpy()
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all() and np.abs(got - want).max() <= 2 * mh.tolerance(dtype, want), (what, np.abs(got - want).max(), np.abs(want).max())


def run(models, ids, steps, want="all"):
    """Every model's logits of a prompt and of single tokens behind it."""
    out = []
    for m in models:
        eng = Engine(m, max_tokens=1024, use_graphs=False)
        slot = eng.new_sequence()
        out.append([eng.step([slot], [ids], want)] + [eng.step([slot], [[t]], "last") for t in steps])
        eng.check_status()
    return out


@pytest.mark.parametrize("name", sorted(PACKED))
def test_float32(name):
    packed, plain, _ = pair(name, "float32")
    ids = mh.prompt(910, 43, packed.vocab_size)
    for i, (got, want) in enumerate(zip(*run((packed, plain), ids[:40], ids[40:]))):
        near(got, want, "float32", f"{name}, step {i}")


@pytest.mark.parametrize("name", ["DA", "DC", "PA", "PB", "PC", "PD"])
def test_bfloat16(name, monkeypatch):
    """A prompt of more rows than enter as they are: the tensors' side rounds the inputs of the same products to 8 bits, after a rounding to
    bfloat16 that the packed side does not make, which turns some codes by a step (2^-3 to 2^-4 of a value): 8 % of the largest logit, as the
    tests of whole models in 4 bits have it.  Then single tokens and a prompt of 16, where nothing but the weights is rounded."""
    packed, plain, values = pair(name, "bfloat16")
    real, real_gated = ops.linear, ops.linear_gated
    ours = lambda x, w: (ops.pack_mx8(x).dequantise(torch.bfloat16)
                         if type(x) is torch.Tensor and x.shape[0] > 16 and any(w is v for v in values) else x)
    monkeypatch.setattr(ops, "linear", lambda x, w, *a, **kw: real(ours(x, w), w, *a, **kw))
    monkeypatch.setattr(ops, "linear_gated", lambda x, w, *a, **kw: real_gated(ours(x, w), w, *a, **kw))
    ids = mh.prompt(911, 60, packed.vocab_size)
    got, want = run((packed, plain), ids[:57], [])
    got, want = got[0].double(), want[0].double()
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 0.08 * want.abs().max()
    for i, (got, want) in enumerate(zip(*run((packed, plain), ids[:16], ids[16:19]))):
        near(got, want, "bfloat16", f"{name}, step {i}")


@pytest.mark.parametrize("name", sorted(tiny_ligirax.CONFIGS))
def test_a_model_without_such_a_part(name):
    """Latent attention and routed experts keep their matrices: 4 bits are refused rather than left out without a word."""
    cfg, seed = tiny_ligirax.CONFIGS[name]
    with pytest.raises(ValueError, match="none of its parts keeps its matrices in 4 bits"):
        random_model(cfg, seed, "bfloat16", DEV, weight_format="mx4")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["as-stored", "mx4", "mx4+head"])
def test_the_command_line_runs_the_model_it_names(fmt, dtype, tmp_path, capsys):
    cfg = tiny_configs.config("D")[0]
    path = tmp_path / "config.json"
    path.write_text(json.dumps(cfg))
    prompt = mh.prompt(912, 20, cfg["vocab_size"])
    model = random_model(cfg, 5, dtype, DEV, weight_format=None if fmt == "as-stored" else fmt)
    want = Generator(model, max_batch=1, max_context=64).with_temperature(0.0).with_stop_tokens(None).generate_batch([prompt], 6)[0][len(prompt):]
    argv = ["--random-config", str(path), "--weights-seed", "5", "--prompt-ids", ",".join(map(str, prompt)), "--max-tokens", "6", "--temperature", "0",
            "--dtype", dtype, "--weights", fmt, "--stop-ids", "", "--max-context", "64"]
    assert cli.main(argv) == 0
    got = [int(t) for t in capsys.readouterr().out.replace(",", " ").split()]
    assert len(got) == 6 and got == want
