"""The Llama decoder with its layers' matrices in 8 bits: every layer against plain arithmetic with the same roundings, and
generation through the entry point."""
import pytest
import torch

import fp8_util as fu
import plain_llama as pl
from conftest import TINY

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rounded(x):
    q, s = fu.quantize_rows(x)
    return fu.row_values(q, s).float()


def weight(w):
    q, s = fu.quantize_weight(w.to(torch.bfloat16))
    return fu.weight_values(q, s).float()


def plain_layer(cfg, w, i, x):
    """One layer of the plain decoder on float32 rows `x`: branch inputs rounded to 8 bits, matrices too (queries, keys and values
    are one matrix), what the engine stores in bfloat16 rounded to that."""
    p, hd = f"model.layers.{i}.", cfg.get("head_dim") or cfg["hidden_size"] // cfg["num_attention_heads"]
    nq, nkv, t = cfg["num_attention_heads"], cfg["num_key_value_heads"], x.shape[0]
    cos, sin = pl.rope_tables(cfg["max_position_embeddings"], hd, cfg["rope_theta"])
    h = rounded(pl.rms_norm(x, w[p + "input_layernorm.weight"], cfg["rms_norm_eps"]))
    qkv = pl.bf16_quant(h @ weight(torch.cat([w[p + f"self_attn.{n}_proj.weight"] for n in "qkv"])).T)
    q, k, v = (y.view(t, -1, hd) for y in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    pos = torch.arange(t)
    q, k = (pl.bf16_quant(pl.apply_rope(y, cos, sin, pos)) for y in (q, k))
    o = pl.bf16_quant(pl.attention(q, k, v, pos, quant=pl.bf16_quant)).reshape(t, nq * hd)
    x = x + rounded(o) @ weight(w[p + "self_attn.o_proj.weight"]).T
    h = rounded(pl.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg["rms_norm_eps"]))
    m = rounded(pl.silu(h @ weight(w[p + "mlp.gate_proj.weight"]).T) * (h @ weight(w[p + "mlp.up_proj.weight"]).T))
    return x + m @ weight(w[p + "mlp.down_proj.weight"]).T


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_every_layer_is_near_plain_arithmetic(model_dirs, name):
    """A layer's change of the stream against the plain layer on the engine's own stream.  What enters a rounding to 8 bits differs by
    the bfloat16 roundings before it, 2^-8 of the value; a value so moved falls to the other side of a border with a probability of at
    most 2^-8 / 2^-4, and then moves by 2^-3: 2^-5 in the mean square, on four inputs of products, beside the bfloat16 roundings
    themselves: 2 * 2^-5 in all, and twice that for the sizes' spread."""
    from tiny_llm_b200.engine import StepEntry
    from tiny_llm_b200.engine.loading import load_model, make_runner
    cfg, w = pl.load_config(model_dirs[name]), pl.load_weights(model_dirs[name])
    cfg.setdefault("head_dim", cfg["hidden_size"] // cfg["num_attention_heads"])
    _, model = load_model(model_dirs[name], "bfloat16", DEV, weights="fp8")
    seen = []
    model.probe = lambda pos, resid: seen.append(resid.clone().cpu())
    runner = make_runner(model, "bfloat16", DEV, max_tokens=512, max_requests=4)
    runner.use_graphs = runner.use_tapes = False
    toks = torch.randint(3, cfg["vocab_size"], (57,), generator=torch.Generator().manual_seed(3)).tolist()
    runner.cache.add_request("r")
    runner.step([StepEntry("r", toks, [56])])
    x = w["model.embed_tokens.weight"].to(torch.bfloat16).float()[torch.tensor(toks)]
    for i, got in enumerate(seen):
        change = plain_layer(cfg, w, i, x) - x
        assert float((got - x - change).norm() / change.norm()) <= 2.0 ** -3, i
        x = got
    assert len(seen) == cfg["num_hidden_layers"]


@pytest.mark.parametrize("name", ["A", "C"])
def test_generation_with_8_bit_weights(model_dirs, name):
    """Prompts in portions beside decoded tokens: steps run as graphs and tapes give what the same steps give without either."""
    from tiny_llm_b200 import Pipeline
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(8, TINY[name][0]["vocab_size"], (n,), generator=g).tolist() for n in (1, 7, 16, 33)]
    kw = dict(dtype="bfloat16", weights="fp8", device=0, page_size=TINY[name][1], max_tokens=512, max_requests=4)
    pipe = Pipeline(model_dirs[name], max_tokens_per_step=24, chunk=5, **kw)
    out = pipe.apply(prompts, max_new_tokens=12, do_sample=False, ignore_eos=True)
    assert [len(o) for o in out] == [12] * 4 and pipe.runner.graph_replays > 0
    again = pipe.apply(prompts, max_new_tokens=12, do_sample=False, ignore_eos=True)
    assert again == out
    plain = Pipeline(model_dirs[name], max_tokens_per_step=24, chunk=5, **kw)
    plain.runner.use_graphs = plain.runner.use_tapes = False
    assert plain.apply(prompts, max_new_tokens=12, do_sample=False, ignore_eos=True) == out


def test_the_command_line_with_8_bit_weights(model_dirs, tmp_path):
    import subprocess
    import sys
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-m", "tiny_llm_b200", f"--model_path={model_dirs['A']}", "--weights=fp8", "--nodo_sample",
                        "--max_new_tokens=5", "--max_tokens=256"], input="9 10 11\n\n", capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0, r.stderr
    line = r.stdout.split("[Output] >\n")[1].split("\n")[0]
    assert 1 <= len(line.split()) <= 5
    r = subprocess.run([sys.executable, "-m", "tiny_llm_b200", f"--model_path={model_dirs['A']}", "--weights=fp8", "--dtype=float32"],
                       input="", capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 1 and "bfloat16 engine" in r.stderr
