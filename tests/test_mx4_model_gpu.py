"""Models whose layers' matrices are in microscaled 4-bit floats, through the engine and the
library's entry points, and layers whose sublayers end with a residual scale."""
import json
import os
import tempfile

import numpy as np
import pytest
import torch

import plain_qwen3 as plain
from helpers import model_dir, rel_err, run_trace, trace_tail, trace_whole
from test_mx4_gpu import plain_blocks
from tiny import SEEDS, TINY, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
PACKED = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")
U32 = torch.finfo(F32).eps / 2


def ops():
    from janas_b200.csrc import ops as o
    return o


def engine(d, **kw):
    from janas_b200.engine import Engine
    return Engine.open(d, dtype="bfloat16", max_tokens=1024, max_seqs=8, **kw)


def values(x):
    return plain_blocks(x)[2].float()


_VALUES = {}


def values_dir(name):
    """The model's folder with every matrix of its layers replaced by what it stands for in 4 bits."""
    if name not in _VALUES:
        from safetensors.torch import load_file
        from janas_b200.weights import write_safetensors
        src, d = model_dir(name), tempfile.mkdtemp(prefix="janas_b200_mx4_")
        w = load_file(os.path.join(src, "model.safetensors"))
        w = {k: values(v).to(BF16) if any(p in k for p in PACKED) else v for k, v in w.items()}
        with open(os.path.join(src, "config.json")) as f, open(os.path.join(d, "config.json"), "w") as g:
            g.write(f.read())
        write_safetensors(os.path.join(d, "model.safetensors"), w.items())
        _VALUES[name] = d
    return _VALUES[name]


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "F"])
def test_model_is_what_its_values_are(name):
    """A matrix and its own 4-bit values give the same codes, so the two folders give the same bits, whole and token by
    token; and fewer bytes of weights than as stored."""
    rng = np.random.default_rng(3)
    reqs = [tokens(rng, n, TINY[name]["vocab_size"]) for n in (1, 9, 70)]
    a, b, c = engine(model_dir(name), weights="mx4"), engine(values_dir(name), weights="mx4"), engine(model_dir(name))
    i = a.info()
    assert i["weights"] == "mx4" and i["packed_matrices"] == 4 * TINY[name]["num_hidden_layers"]
    assert c.info()["weights"] == "stored" and c.info()["packed_matrices"] == 0
    assert i["weight_bytes"] < c.info()["weight_bytes"]
    differs = False
    for trace in (trace_whole(reqs), trace_tail(reqs, 5)):
        x, y, z = run_trace(a, trace), run_trace(b, trace), run_trace(c, trace)
        for r in x:
            for p in x[r]:
                assert np.array_equal(x[r][p], y[r][p]) and np.isfinite(x[r][p]).all()
                differs |= not np.array_equal(x[r][p], z[r][p])
    assert differs
    for e in (a, b, c):
        e.close()


def plain_mx4_logits(c, w, toks):
    """The plain forward with both operands of every packed product in 4 bits and the engine's roundings to bfloat16."""
    r = lambda t: t.to(BF16).float()    # noqa: E731
    mm = lambda a, m: values(a) @ values(m).T    # noqa: E731
    eps, nh, nkv, hd = c["rms_norm_eps"], c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"]
    x = plain.embedding(w["model.embed_tokens.weight"], toks)
    n = len(toks)
    for i in range(c["num_hidden_layers"]):
        p = f"model.layers.{i}."
        window = c["sliding_window"] if c["layer_types"][i] == "sliding_attention" else 0
        h = r(plain.rms_norm(x, w[p + "input_layernorm.weight"], eps))
        s = p + "self_attn."
        q, k, v = (mm(h, w[s + n_ + "_proj.weight"]) for n_ in "qkv")
        q = plain.rms_norm(q.view(n, nh, hd), w[s + "q_norm.weight"], eps)
        k = plain.rms_norm(k.view(n, nkv, hd), w[s + "k_norm.weight"], eps)
        cs, sn = plain.rope_table(range(n), hd, c["rope_theta"])
        a = r(plain.attention(r(plain.rope_neox(q, cs, sn)), r(plain.rope_neox(k, cs, sn)), r(v.view(n, nkv, hd)), window))
        x = x + mm(a.reshape(n, nh * hd), w[s + "o_proj.weight"])
        h = r(plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], eps))
        f = p + "mlp."
        g, u = mm(h, w[f + "gate_proj.weight"]), mm(h, w[f + "up_proj.weight"])
        x = x + mm(g / (1.0 + torch.exp(-g)) * u, w[f + "down_proj.weight"])
    h = r(plain.rms_norm(x, w["model.norm.weight"], eps))
    return (h @ w.get("lm_head.weight", w["model.embed_tokens.weight"]).T).numpy()


@pytest.mark.parametrize("name", ["B", "D", "F"])
def test_logits_against_plain(name):
    """A value that lies at a border may round to the other side of it in one of the two, and what follows then differs by
    a step of its block; so the yardstick is the change that the 4 bits themselves make to the logits: the engine must be
    at least twice closer to the plain 4-bit model than the plain model in bfloat16 is.

    How far it may be: attention's result is off by two roundings to bfloat16 (the softmax weights', the result's), 2^-7
    of its value.  Neighbouring 4-bit numbers lie a third of their value apart or more, so up to 3 2^-7 = 2.4% of the
    values round to the other one, a half of the value away at most: the product's input is off by sqrt(0.024) / 2 = 8% of
    its norm.  Two layers of that, each carried on by a feed-forward that rounds again: sqrt(4) 8% = 16% of the logits,
    where the 4 bits themselves make 31% (measured on D)."""
    d = model_dir(name)
    c, w = plain.read_config(d), plain.read_weights(d)
    toks = tokens(np.random.default_rng(5), 40, TINY[name]["vocab_size"])
    want = plain_mx4_logits(c, w, toks)
    full = plain.forward(c, w, toks, "bfloat16").numpy()
    e = engine(d, weights="mx4")
    got = run_trace(e, trace_whole([toks]))["r0"]
    got = np.stack([got[p] for p in range(len(toks))])
    e.close()
    assert np.linalg.norm(got - want) <= 0.5 * np.linalg.norm(full - want), \
        (np.linalg.norm(got - want) / np.linalg.norm(want), np.linalg.norm(full - want) / np.linalg.norm(want))


@pytest.mark.parametrize("n", [1, 5, 40, 200])
def test_feed_forwards_are_their_operators(n):
    """Each dense feed-forward in 4 bits, bit for bit the library's operators one after the other."""
    from janas_b200.config import PartSpec
    from test_parts_gpu import build, context, give
    o = ops()
    hidden, inter = 96, 328
    h = torch.randn(n, hidden, generator=torch.Generator().manual_seed(n)).to(BF16).to(DEV)
    sizes = {"hidden_size": hidden, "intermediate_size": inter}
    for kind, params in (("swiglu", sizes), ("swiglu", {**sizes, "unit": {"alpha": 1.702, "limit": 7.0, "shift": 1.0}}),
                         ("dense", {**sizes, "activation": "relu2"}), ("polynorm", {**sizes, "eps": 1e-6})):
        part = build("feed_forward", PartSpec(kind, params), BF16)
        w = {k: v.to(BF16).to(DEV) for k, v in give(part, "f", 2, BF16).items()}
        before = part.forward(context([0], [n], BF16), h).sum(0)
        assert part.pack() == 2
        got = part.forward(context([0], [n], BF16), h)
        down = o.mx4_quantize(w["f.down_proj.weight"])
        if kind == "swiglu":
            z = o.linear_mx4(h, o.mx4_quantize(torch.cat([w["f.gate_proj.weight"], w["f.up_proj.weight"]])))
            u = params.get("unit", {"alpha": 1.0, "limit": 0.0, "shift": 0.0})
            act = o.mx4_gated_unit(z, u["alpha"], u["limit"], u["shift"])
        else:
            z = o.linear_mx4(h, o.mx4_quantize(w["f.up_proj.weight"]))
            act = o.activation(z, "relu2", BF16) if kind == "dense" else \
                o.polynorm(z, w["f.act.weight"].float(), 1e-6, BF16)
        assert got.shape == (1, n, hidden) and torch.equal(got[0], o.linear_mx4(act, down))
        assert not torch.equal(got[0], before)


def test_generate_in_4_bits():
    """The library's entry point: captured decode steps give the tokens that eager ones do; one batch and one by one."""
    import janas_b200
    from janas_b200 import lib
    rng = np.random.default_rng(7)
    prompts = [tokens(rng, n, TINY["D"]["vocab_size"]) for n in (3, 17, 80)]
    llm = janas_b200.open(model_dir("D"), janas_b200.LLMParams(n_ctx=256, max_batch=4, max_tokens=1024, weights="mx4"))
    outs, _ = llm.generate_batch(prompts, 20)
    assert llm.engine.info()["graph_captures"] > 0
    lib.call("llm.set", llm=llm.engine._h.value, use_graphs=False)
    again, _ = llm.generate_batch(prompts, 20)
    assert outs == again
    llm.close()


def test_weights_refusals():
    import janas_b200
    from janas_b200 import lib
    from janas_b200.engine import Engine
    from kefesun_models import CONFIGS
    with pytest.raises(lib.LLMError) as e:
        Engine.open(model_dir("A"), dtype="float32", weights="mx4")
    assert e.value.code == lib.EINVAL and "BF16" in str(e.value)
    with pytest.raises(ValueError):
        Engine.open(model_dir("A"), weights="int4")
    with pytest.raises(lib.LLMError) as e:
        Engine.open_random(CONFIGS["KA"], weights="mx4")
    assert e.value.code == lib.EMODEL and "4 bits" in str(e.value)
    p = janas_b200.engine.engine._params("bfloat16", 128, 1, "cuda:0", None)
    p.weights = 2
    import ctypes
    h = ctypes.c_void_p()
    assert lib.lib().jb_llm_open(model_dir("A").encode(), ctypes.byref(p), ctypes.byref(h)) == lib.EINVAL


# ------------------------------------------------------------ residual scales
def scaled_spec(kind, gates, ffn=True):
    """Two sandwich layers whose sublayers' results are scaled per feature, with the norms of one kind."""
    from janas_b200.config import LayerSpec, ModelSpec, PartSpec, RunEntry
    H, F = 96, 160
    norm = PartSpec("rmsnorm", {"size": H, "eps": 1e-5, "one_plus": True}) if kind == "rms" else \
        PartSpec("layernorm", {"size": H, "eps": 1e-5})
    mixer = PartSpec("gqa_attention", {"hidden_size": H, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16, "window": 0,
                                       "position": {"kind": "rope_neox", "params": {"rotary_dim": 16, "theta": 1000.0, "max_positions": 256}}})
    ff = PartSpec("swiglu", {"hidden_size": H, "intermediate_size": F})
    bp = {"hidden_size": H, "mixer_scale": "mixer_scale", "ffn_scale": "ffn_scale"}
    if gates:
        bp.update(mixer_gate="mixer_gate", ffn_gate="ffn_gate", gate_bias=".bias")
    layers = tuple(LayerSpec("sandwich", mixer, ff if ffn or i == 0 else None, norm, norm if ffn or i == 0 else None,
                             f"layers.{i}", post_mixer_norm=norm, post_ffn_norm=norm if ffn or i == 0 else None,
                             block_params=bp) for i in range(2))
    return ModelSpec("toy", H, 130, 256, layers, (RunEntry(0), RunEntry(1)), norm, True)


def plain_scaled(spec, w, kind, gates, toks):
    H, nh, nkv, hd = 96, 4, 2, 16

    def norm(x, name):
        if kind == "rms":
            return x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * (1 + w[name + ".weight"])
        d = x - x.mean(-1, keepdim=True)
        return d / (d.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w[name + ".weight"] + w[name + ".bias"]

    x = w["model.embed_tokens.weight"][torch.tensor(toks)]
    n = len(toks)
    for i, l in enumerate(spec.layers):
        p = f"layers.{i}."

        def end(y, h, which, post):
            if gates:
                y = y * torch.sigmoid(h @ w[p + which + "_gate"].T + w[p + which + "_gate.bias"])
            return x + w[p + which + "_scale"] * norm(y, p + post)

        h = norm(x, p + "input_layernorm")
        s = p + "self_attn."
        q, k, v = (h @ w[s + t + "_proj.weight"].T for t in "qkv")
        cs, sn = plain.rope_table(range(n), hd, 1000.0)
        cs, sn = cs.double(), sn.double()
        a = plain.attention(plain.rope_neox(q.view(n, nh, hd), cs, sn), plain.rope_neox(k.view(n, nkv, hd), cs, sn),
                            v.view(n, nkv, hd), 0)
        x = end(a.reshape(n, -1) @ w[s + "o_proj.weight"].T, h, "mixer", "post_mixer_norm")
        if l.feed_forward:
            h = norm(x, p + "post_attention_layernorm")
            g, u = h @ w[p + "mlp.gate_proj.weight"].T, h @ w[p + "mlp.up_proj.weight"].T
            x = end((g * torch.sigmoid(g) * u) @ w[p + "mlp.down_proj.weight"].T, h, "ffn", "post_ffn_norm")
    return (norm(x, "model.norm") @ w["model.embed_tokens.weight"].T).numpy()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gates", [False, True])
@pytest.mark.parametrize("ffn", [True, False])
def test_residual_scales(kind, gates, ffn):
    """Against 64 bits.  float32: four sublayers, each two products over up to 160 values and two norms, off by about
    160 U of the sums of magnitudes at most, which the norms' division can make ten times as much of the result.  bfloat16:
    each of a sublayer's inputs, q, k, v, attention's result and the unit off by 2^-8, about six a sublayer, and as many
    sublayers (their squares add up at best, and at worst they themselves: 24 2^-8)."""
    from janas_b200.engine import Engine
    spec = scaled_spec(kind, gates, ffn)
    tensors = {}
    probe = Engine.from_spec(spec, seed=1, dtype="float32", max_tokens=256)
    probe.close()
    g = torch.Generator().manual_seed(4)
    H, F = 96, 160
    rnd = lambda *s, scale=1.0: torch.randn(*s, generator=g) * scale    # noqa: E731

    def norm(name):
        tensors[name + ".weight"] = rnd(H, scale=0.2) + (0.0 if kind == "rms" else 1.0)
        if kind != "rms":
            tensors[name + ".bias"] = rnd(H, scale=0.1)

    tensors["model.embed_tokens.weight"] = rnd(130, H)
    for i, l in enumerate(spec.layers):
        p = f"layers.{i}."
        norm(p + "input_layernorm"), norm(p + "post_mixer_norm")
        for t, rows in (("q", 64), ("k", 32), ("v", 32)):
            tensors[p + f"self_attn.{t}_proj.weight"] = rnd(rows, H, scale=H ** -0.5)
        tensors[p + "self_attn.o_proj.weight"] = rnd(H, 64, scale=0.125)
        which = ["mixer"]
        if l.feed_forward:
            which.append("ffn")
            norm(p + "post_attention_layernorm"), norm(p + "post_ffn_norm")
            for t in ("gate", "up"):
                tensors[p + f"mlp.{t}_proj.weight"] = rnd(F, H, scale=H ** -0.5)
            tensors[p + "mlp.down_proj.weight"] = rnd(H, F, scale=F ** -0.5)
        for t in which:
            tensors[p + t + "_scale"] = 0.5 + rnd(H, scale=0.2)
            if gates:
                tensors[p + t + "_gate"], tensors[p + t + "_gate.bias"] = rnd(H, H, scale=H ** -0.5), rnd(H, scale=0.2)
    norm("model.norm")
    tensors = {k: v.to(BF16).float() if "proj" in k or k.endswith("_gate") or "embed" in k else v for k, v in tensors.items()}
    w = {k: v.double() for k, v in tensors.items()}
    toks = tokens(np.random.default_rng(2), 50, 130)
    want = plain_scaled(spec, w, kind, gates, toks)
    for dtype, tol in (("float32", 10 * 160 * U32 * 4), ("bfloat16", 24 * 2.0 ** -8)):
        e = Engine.from_spec(spec, tensors={k: v.to(DEV) for k, v in tensors.items()}, dtype=dtype, max_tokens=256)
        for trace in (trace_whole([toks]), trace_tail([toks], 8)):
            got = run_trace(e, trace)["r0"]
            assert rel_err(np.stack([got[p] for p in range(len(toks))]), want) <= tol
        e.close()


def test_residual_scale_refusals():
    """A norm on the result whose parameters the kernel does not take."""
    from dataclasses import replace
    from janas_b200 import lib
    from janas_b200.config import PartSpec
    from janas_b200.engine import Engine
    spec = scaled_spec("rms", False)
    for bad in (PartSpec("dynamic_tanh", {"size": 96}), PartSpec("rmsnorm", {"size": 96, "eps": 1e-5})):
        layers = tuple(replace(l, post_mixer_norm=bad) for l in spec.layers)
        with pytest.raises(lib.LLMError) as e:
            Engine.from_spec(replace(spec, layers=layers), seed=1, dtype="bfloat16", max_tokens=256)
        assert "residual scale" in str(e.value)
