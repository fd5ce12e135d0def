"""Layers whose parts are held in 4 bits: what goes to 4 bits and what stays, and the same steps run one by one."""
import numpy as np
import pytest
import torch

from helpers import run_trace, trace_tail, trace_whole
from test_mx4_gpu import plain_blocks
from tiny import tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
H, F, VOCAB = 96, 160, 130


def norm_spec(kind):
    from janas_b200.config import PartSpec
    return PartSpec("rmsnorm", {"size": H, "eps": 1e-5}) if kind == "rms" else PartSpec("layernorm", {"size": H, "eps": 1e-5})


def sandwich(ffn_kind="polynorm", kind="rms", gates=True, scales=False, fuse=True):
    """Two sandwich layers: grouped attention and a feed-forward, norms around both."""
    from janas_b200.config import LayerSpec, ModelSpec, PartSpec, RunEntry
    norm = norm_spec(kind)
    mixer = PartSpec("gqa_attention", {"hidden_size": H, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16, "window": 0,
                                       "position": {"kind": "rope_neox", "params": {"rotary_dim": 16, "theta": 1000.0,
                                                                                   "max_positions": 256}}})
    params = {"hidden_size": H, "intermediate_size": F}
    ffn = PartSpec(ffn_kind, {**params, "eps": 1e-6} if ffn_kind == "polynorm" else params)
    bp = {"hidden_size": H, "fuse": fuse}
    if scales:
        bp.update(mixer_scale="mixer_scale", ffn_scale="ffn_scale")
    if gates:
        bp.update(mixer_gate="mixer_gate", ffn_gate="ffn_gate", gate_bias=".bias")
    layers = tuple(LayerSpec("sandwich", mixer, ffn, norm, norm, f"layers.{i}", post_mixer_norm=norm, post_ffn_norm=norm,
                             block_params=bp) for i in range(2))
    return ModelSpec("toy", H, VOCAB, 256, layers, (RunEntry(0), RunEntry(1)), norm, True)


def weights_of(spec, seed=3):
    """Random tensors for the model, by name."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: torch.randn(*s, generator=g) * scale    # noqa: E731
    t = {"model.embed_tokens.weight": r(VOCAB, H)}
    biased = spec.layers[0].mixer_norm.kind == "layernorm"

    def norm(name):
        t[name + ".weight"] = 1.0 + r(H, scale=0.2)
        if biased:
            t[name + ".bias"] = r(H, scale=0.1)

    norm("model.norm")
    for i, l in enumerate(spec.layers):
        p = f"layers.{i}."
        for n in ("input_layernorm", "post_mixer_norm", "post_attention_layernorm", "post_ffn_norm"):
            norm(p + n)
        for n, rows in (("q", 64), ("k", 32), ("v", 32)):
            t[p + f"self_attn.{n}_proj.weight"] = r(rows, H, scale=H ** -0.5)
        t[p + "self_attn.o_proj.weight"] = r(H, 64, scale=0.125)
        names = ("up", "gate") if l.feed_forward.kind == "swiglu" else ("up",)
        for n in names:
            t[p + f"mlp.{n}_proj.weight"] = r(F, H, scale=H ** -0.5)
        t[p + "mlp.down_proj.weight"] = r(H, F, scale=F ** -0.5)
        if l.feed_forward.kind == "polynorm":
            t[p + "mlp.act.weight"] = 0.3 + r(4, scale=0.2)
        for n in ("mixer", "ffn"):
            if l.block_params.get(n + "_gate"):
                t[p + n + "_gate"], t[p + n + "_gate.bias"] = r(H, H, scale=H ** -0.5), r(H, scale=0.2)
            if l.block_params.get(n + "_scale"):
                t[p + n + "_scale"] = 0.5 + r(H, scale=0.2)
    return {n: v.to(BF16) if v.dim() == 2 else v for n, v in t.items()}


def opened(spec, tensors, **kw):
    from janas_b200.engine import Engine
    kw = {"dtype": "bfloat16", "weights": "mx4", **kw}
    return Engine.from_spec(spec, tensors={n: v.to(DEV) for n, v in tensors.items()}, max_tokens=256, **kw)


def logits(e, toks, tail=0):
    got = run_trace(e, trace_tail([toks], tail) if tail else trace_whole([toks]))["r0"]
    return np.stack([got[p] for p in range(len(toks))])


TOKENS = tokens(np.random.default_rng(2), 40, VOCAB)


def test_gates_stay_as_stored():
    """A gate is no matrix of attention or of a feed-forward: it stays in bfloat16, whether its product would have gone
    into the feed-forward's (fuse) or not.  With norms that are always steps of their own the two give the same bits."""
    a, b = sandwich(fuse=True), sandwich(fuse=False)
    w = weights_of(a)
    fused, steps = opened(a, w), opened(b, w)
    for key in ("weight_bytes", "packed_matrices"):
        assert fused.info()[key] == steps.info()[key]
    assert fused.info()["packed_matrices"] == 2 * 4
    x = logits(fused, TOKENS)
    for tail in (0, 6):
        assert np.array_equal(logits(fused, TOKENS, tail), logits(steps, TOKENS, tail))
    for which in ("mixer_gate", "ffn_gate"):
        # the gate's 4-bit values in its place would give the same bits if it went to 4 bits
        other = {n: plain_blocks(v)[2].to(BF16) if n.endswith(which) else v for n, v in w.items()}
        e = opened(a, other)
        assert not np.array_equal(logits(e, TOKENS), x), which
        e.close()
    fused.close(), steps.close()


def test_a_stored_model_has_its_gates_in_the_product():
    """As before for weights as stored: one product for the feed-forward's rows and its gate's."""
    from janas_b200 import lib
    launches = lambda: lib.call("llm.launches")["launches"]    # noqa: E731
    count = {}
    for fuse in (True, False):
        spec = sandwich(fuse=fuse)
        e = opened(spec, weights_of(spec), weights="stored")
        logits(e, TOKENS)
        at = launches()
        logits(e, TOKENS)
        count[fuse] = launches() - at
        e.close()
    assert count[True] < count[False]


@pytest.mark.parametrize("name", ["ZA", "ZC"])
def test_zuzelorn_in_4_bits(name):
    """A registered design with gated polynorm feed-forwards: these go to 4 bits, and nothing else does."""
    from janas_b200.engine import Engine
    from test_zuzelorn_gpu import model, requests
    folder, c, w = model(name)
    toks = requests(name)[3][:50]
    e = Engine.open(folder, dtype="bfloat16", max_tokens=1024, weights="mx4")
    ffns = [i for i, l in enumerate(c["layers"]) if l["mlp"]]
    assert e.info()["packed_matrices"] == 2 * len(ffns)
    got = logits(e, toks)
    e.close()
    # the same bits from a folder of the values that those matrices stand for
    vals = {n: plain_blocks(v)[2] if n.split(".")[-1] in ("up", "down") else v for n, v in w.items()}
    vals = {n: v.to(BF16) if v.dim() == 2 else v.float() for n, v in vals.items()}
    from janas_b200.config import config_from_dict
    same = Engine.from_spec(config_from_dict(c).to_model_spec(), tensors={n: v.to(DEV) for n, v in vals.items()},
                            dtype="bfloat16", max_tokens=1024, weights="mx4")
    assert np.array_equal(got, logits(same, toks)) and np.isfinite(got).all()
    same.close()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gates", [False, True])
def test_residual_scales_step_by_step(kind, gates):
    """fuse false: gate, norm, and scale and add, each a kernel of its own.  Each way is off from the sublayers in 64 bits
    by at most 10 x 160 roundings a sublayer (products over up to 160 values, norms that can make their error ten times as
    much of the result), four sublayers; so the two differ by twice that at most."""
    from helpers import rel_err
    from janas_b200 import lib
    got, count = {}, {}
    for fuse in (True, False):
        spec = sandwich("swiglu", kind, gates, scales=True, fuse=fuse)
        e = opened(spec, weights_of(spec), weights="stored", dtype="float32")
        logits(e, TOKENS)
        at = lib.call("llm.launches")["launches"]
        got[fuse] = logits(e, TOKENS)
        count[fuse] = lib.call("llm.launches")["launches"] - at
        tail = logits(e, TOKENS, 5)
        assert rel_err(tail, got[fuse]) <= 2 * 10 * 160 * 4 * torch.finfo(torch.float32).eps / 2
        e.close()
    # a step's kernels: a norm for each of the four sublayers' results, three norms that wait for the next sublayer (the
    # last one the model's), and with gates four gates
    assert count[False] > count[True] + 4
    assert rel_err(got[False], got[True]) <= 2 * 10 * 160 * 4 * torch.finfo(torch.float32).eps / 2


def test_a_residual_scale_of_too_many_features():
    """Longer rows than the kernel takes: refused when the model is opened, not in its first step."""
    from dataclasses import replace
    from janas_b200 import lib
    from janas_b200.csrc import ops
    from janas_b200.engine import Engine
    spec = sandwich("swiglu", "layer", False, scales=True)
    wide = ops.lib().jb_norm_residual_norm_most() + 4

    def sized(part):
        key = "size" if "size" in part.params else "hidden_size"
        return replace(part, params={**part.params, key: wide})

    layers = tuple(replace(l, mixer=sized(l.mixer), feed_forward=sized(l.feed_forward), mixer_norm=sized(l.mixer_norm),
                           ffn_norm=sized(l.ffn_norm), post_mixer_norm=sized(l.post_mixer_norm),
                           post_ffn_norm=sized(l.post_ffn_norm), block_params={**l.block_params, "hidden_size": wide})
                   for l in spec.layers)
    spec = replace(spec, hidden_size=wide, layers=layers, final_norm=sized(spec.final_norm))
    with pytest.raises(lib.LLMError) as err:
        Engine.from_spec(spec, seed=1, dtype="bfloat16", max_tokens=64)
    assert "residual scale" in str(err.value)


def test_the_refusal_names_the_parts():
    """A design with attention of another kind and routed experts alone: none of its parts takes 4 bits, and the message
    says which do."""
    from janas_b200 import lib
    from janas_b200.engine import Engine
    from kefesun_models import CONFIGS
    with pytest.raises(lib.LLMError) as err:
        Engine.open_random(CONFIGS["KA"], weights="mx4")
    assert err.value.code == lib.EMODEL
    assert all(kind in str(err.value) for kind in ("gqa_attention", "swiglu", "polynorm", "dense"))
