"""Whole models with 4-bit weights: weights that are packed as a model is built, steps of up to 16 rows (activations as they are) and
larger ones (activations in 8 bits), against the plain implementation with the same 4-bit values."""
import json

import numpy as np
import pytest
import torch

import model_helpers as mh
import plain_gemma2 as plain
import plain_microscaling as mx
import tiny_configs
from rust_deeplearning_b200 import Engine, Generator, cli, load_model, random_model
from rust_deeplearning_b200.kernels import library, ops
from rust_deeplearning_b200.parts.model import Model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain_weights(name, head):
    """The folder's tensors with the packed matrices replaced by the values 4 bits leave of them."""
    cfg, w = mh.plain_model(name)
    out = dict(w)
    for n, v in w.items():
        if n.endswith("_proj.weight") or (head and n == "lm_head.weight"):
            out[n] = mx.quantise(v, mx.E2M1)[0]
    return cfg, out


def to_bf16(v):
    return torch.from_numpy(np.asarray(v)).to(torch.bfloat16).double().numpy()


def packed_forward(cfg, w, ids, keep=lambda v: v):
    """`plain.forward` with the inputs of all packed products rounded to 8 bits; keep: what happens to what a bfloat16 model keeps in
    bfloat16 (products' results, the attention's)."""
    q8 = lambda v: mx.quantise(v, mx.E4M3)[0]
    eps, T, nh, nkv, hd = cfg["rms_norm_eps"], len(ids), cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
    x = plain.embed(w["model.embed_tokens.weight"], ids, cfg["hidden_size"])
    cos, sin = plain.rope_tables(hd, T, cfg["rope_theta"])
    pick = np.split(np.eye((nh + 2 * nkv) * hd), [nh * hd, (nh + nkv) * hd])             # q, k and v of their rows side by side
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        n = q8(plain.rms_norm(x, w[p + "input_layernorm.weight"], eps))
        qkv = np.concatenate([keep(n @ w[p + f"self_attn.{m}_proj.weight"].T) for m in "qkv"], axis=1)
        a = keep(plain.attention(qkv, *pick, np.eye(nh * hd), cos, sin, n_heads=nh, n_kv_heads=nkv, head_dim=hd,
                                 query_pre_attn_scalar=cfg["query_pre_attn_scalar"], softcap=cfg.get("attn_logit_softcapping"), window=plain.layer_window(cfg, i)))
        x = x + plain.rms_norm(keep(q8(a) @ w[p + "self_attn.o_proj.weight"].T), w[p + "post_attention_layernorm.weight"], eps)
        n = q8(plain.rms_norm(x, w[p + "pre_feedforward_layernorm.weight"], eps))
        f = keep(q8(plain.gelu_tanh(n @ w[p + "mlp.gate_proj.weight"].T) * (n @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T)
        x = x + plain.rms_norm(f, w[p + "post_feedforward_layernorm.weight"], eps)
    n = keep(plain.rms_norm(x, w["model.norm.weight"], eps))
    return plain.lm_head(n, w["model.embed_tokens.weight"], cfg.get("final_logit_softcapping"))


def engine(name, dtype, fmt, **kw):
    return Engine(load_model(mh.model_folder(name), dtype, DEV, weight_format=fmt), max_tokens=2048, **kw)


@pytest.mark.parametrize("fmt", ["mx4", "mx4+head"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_float32(name, fmt):
    """In 32 bits nothing but the weights is rounded, whatever the step's size: the tolerance of every float32 model test."""
    cfg, w = plain_weights(name, False)
    table = w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings", True) else w["lm_head.weight"]
    if fmt == "mx4+head":
        table = mx.quantise(table, mx.E2M1)[0]
    ids = mh.prompt(900, 40, cfg["vocab_size"])
    h = dict(cfg, tie_word_embeddings=False)
    want = plain.forward(h, dict(w, **{"lm_head.weight": table}), ids)
    eng = engine(name, "float32", fmt, use_graphs=False)
    slot = eng.new_sequence()
    mh.assert_logits(eng.step([slot], [ids[:30]], "all"), want[:30], "float32", "prompt")
    for t in range(30, 33):
        mh.assert_logits(eng.step([slot], [[ids[t]]], "last"), want[t:t + 1], "float32", f"position {t}")
    mh.assert_logits(eng.step([slot], [ids[33:]], "all"), want[33:], "float32", "a few more")
    eng.check_status()


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
def test_bfloat16_few_rows(name, graphs):
    """Steps of up to 16 rows round nothing but the weights: the tolerance of every bfloat16 model test."""
    cfg, w = plain_weights(name, False)
    ids = mh.prompt(901, 24, cfg["vocab_size"])
    want = plain.forward(cfg, w, ids)
    eng = engine(name, "bfloat16", "mx4", use_graphs=graphs)
    slot = eng.new_sequence()
    mh.assert_logits(eng.step([slot], [ids[:16]], "all"), want[:16], "bfloat16", "16 rows")
    for t in range(16, 24):
        mh.assert_logits(eng.step([slot], [[ids[t]]], "last"), want[t:t + 1], "bfloat16", f"position {t}")
    assert eng.graph_replays > 0 or not graphs


@pytest.mark.parametrize("name,n", [("A", 17), ("B", 60), ("C", 130), ("D", 200), ("D", 300)])
def test_bfloat16_prompts(name, n):
    """Larger steps round activations to 8 bits, where bfloat16 roundings before that turn some codes by a whole step (2^-3 to 2^-4 of a value):
    logits within 8 % of the largest, and in the mean no further from the plain ones than one and a half times what the bfloat16
    roundings alone, put into the plain implementation, move them."""
    cfg, w = plain_weights(name, False)
    ids = mh.prompt(902, n, cfg["vocab_size"])
    want = packed_forward(cfg, w, ids)
    eng = engine(name, "bfloat16", "mx4", use_graphs=False)
    got = eng.step([eng.new_sequence()], [ids], "all").double().cpu().numpy()
    rms = lambda v: np.sqrt(np.mean(v ** 2))
    assert np.abs(got - want).max() <= 0.08 * np.abs(want).max()
    assert rms(got - want) <= 1.5 * rms(packed_forward(cfg, w, ids, to_bf16) - want)
    eng.check_status()


def test_prompt_uses_the_packed_norm(monkeypatch):
    seen = []
    real = ops.norm_mx8
    monkeypatch.setattr(ops, "norm_mx8", lambda x, **kw: (seen.append((x.shape[0], sorted(kw))), real(x, **kw))[1])
    eng = engine("A", "bfloat16", "mx4", use_graphs=False)
    eng.step([eng.new_sequence()], [mh.prompt(903, 40, 256)], "last")
    # per layer: the norm before the mixer (with the branch before it from the second layer on), the context, the norm before the feed-forward
    fused = [k for rows, k in seen if "residual" in k and rows == 40]
    assert len(fused) == 3 and len(seen) == 6
    seen.clear()
    eng.step([eng.new_sequence()], [[5]], "last")
    assert not seen


def test_several_prompts_in_one_step_and_generation():
    name = "D"
    cfg, w = plain_weights(name, False)
    prompts = [mh.prompt(904 + i, n, cfg["vocab_size"]) for i, n in enumerate((3, 50, 17))]
    eng = engine(name, "bfloat16", "mx4")
    got = eng.step([eng.new_sequence() for _ in prompts], prompts, "last").double().cpu().numpy()
    for g, p in zip(got, prompts):
        want = packed_forward(cfg, w, p)[-1]
        assert np.abs(g - want).max() <= 0.08 * np.abs(want).max()
    model = load_model(mh.model_folder(name), "float32", DEV, weight_format="mx4")
    out = Generator(model, max_batch=4, max_context=128).with_temperature(0.0).with_stop_tokens(None).generate_batch(prompts, 5)
    assert [o[len(p):] for o, p in zip(out, prompts)] == [plain.generate_greedy(cfg, w, p, 5) for p in prompts]


def test_an_architecture_whose_mixers_keep_their_matrices():
    """Parts without the offer run as they were; a model without any is refused."""
    import tiny_ligirax
    cfg = tiny_ligirax.config(sorted(tiny_ligirax.CONFIGS)[0])[0]
    a = random_model(cfg, 3, "bfloat16", DEV)
    try:
        b = random_model(cfg, 3, "bfloat16", DEV, weight_format="mx4")
    except ValueError as e:
        assert "4 bits" in str(e)
        return
    ids = mh.prompt(905, 20, a.vocab_size)
    la, lb = (Engine(m, max_tokens=512, use_graphs=False) for m in (a, b))
    ya, yb = (e.step([e.new_sequence()], [ids], "all").float() for e in (la, lb))
    assert torch.isfinite(yb).all() and not torch.equal(ya, yb)


def test_the_first_rows_of_a_weight():
    w = torch.randn(300, 200, generator=torch.Generator().manual_seed(1)).to(DEV)
    packed = ops.pack_mx4(w)
    x = torch.randn(40, 200, generator=torch.Generator().manual_seed(2)).to(DEV)
    for n in (1, 128, 130, 300):
        for rows in (x[:5].contiguous(), ops.pack_mx8(x)):
            assert torch.equal(ops.linear_mx4(rows, packed.first(n)), ops.linear_mx4(rows, packed)[:, :n])
    with pytest.raises(library.KernelError):
        packed.first(301)


def test_unknown_formats_and_the_command_line(tmp_path, capsys):
    with pytest.raises(ValueError, match="weight format"):
        load_model(mh.model_folder("A"), "bfloat16", DEV, weight_format="q4")
    path = tmp_path / "config.json"
    path.write_text(json.dumps(tiny_configs.config("A")[0]))
    argv = ["--random-config", str(path), "--prompt-ids", "2,5,9", "--max-tokens", "4", "--temperature", "0"]
    outs = []
    for extra in (["--weights", "mx4"], ["--weights", "mx4+head"]):
        assert cli.main(argv + extra) == 0
        outs.append(capsys.readouterr().out.split())
    assert all(len(o) <= 4 for o in outs)


def test_rows_of_the_split_form():
    """How many rows take the norms apart follows from the sizes: as many as every part's product can keep in shared memory."""
    small = ops.pack_mx4(torch.zeros((2 * 64, 128), device=DEV), gated=True)
    tall = ops.pack_mx4(torch.zeros((2 * 10000, 4608), device=DEV), gated=True)          # 157 tiles, 36 blocks of columns
    taller = ops.pack_mx4(torch.zeros((20000, 8320), device=DEV))                        # 65 blocks
    assert (small.deferred_rows, tall.deferred_rows, taller.deferred_rows) == (8, 8, 0)
    model = load_model(mh.model_folder("A"), "bfloat16", DEV, weight_format="mx4")
    assert model.deferred_rows == 8
    h = torch.randn((5, 4608), device=DEV)
    norm = ops.NormParams(torch.zeros(4608, device=DEV), 1e-6, 1.0)
    w = ops.pack_mx4(torch.randn((4608, 2048), device=DEV))
    operand = ops.scaled_rows(h, norm)
    branch = ops.linear_branch(torch.randn((5, 2048), device=DEV).bfloat16(), w, ops.BranchSink(h, norm, norm, operand))
    d = ops.DeferredRows(branch, torch.empty_like(h), norm, torch.empty_like(operand))
    rows = ops.linear_gated(d, tall, "silu")             # five rows: made into a tensor first
    assert d.consumed and torch.equal(rows, ops.linear_gated_mx4(d.materialise(), tall, "silu"))
