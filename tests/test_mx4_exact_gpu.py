"""Products in 4 bits on numbers whose sums are exact in float32, in any order: a part, a chunk or a block of k that is
lost or counted twice, or meets another's scale, shows in nearly every result.  And what follows from them: attention in 4
bits against its operators, rows alone and among others, tokens alone and in captured steps."""
import numpy as np
import pytest
import torch

from test_mx4_gpu import plain_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
U32 = torch.finfo(F32).eps / 2
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def ops():
    from janas_b200.csrc import ops as o
    return o


def numbers(rows, k, seed, exponents=False):
    """Signed 4-bit numbers, in each block of 32 at least one of the two largest, so that they stand for themselves; with
    exponents, each chunk of 256 of k times one of 1/2, 1 and 2, another one than its neighbours' (as for each row)."""
    g = torch.Generator().manual_seed(seed)
    v = GRID[torch.randint(0, 8, (rows, k), generator=g)]
    first = GRID[6 + torch.randint(0, 2, (rows, (k + 31) // 32), generator=g)]
    v[:, ::32] = first
    v *= torch.randint(0, 2, (rows, k), generator=g) * 2 - 1
    if exponents:
        chunk = torch.arange(k) // 256
        v *= torch.exp2(((chunk[None, :] + torch.arange(rows)[:, None]) % 3 - 1).float())
    return v


def exact_case(n, m, k, seed=0):
    """Rows, a weight and their product, exact: every sum, whole or of a part of k in any order, is a multiple of 1/8 (two
    numbers' halves, and a chunk's half) below 2^24 eighths, where float32 holds each."""
    a, w = numbers(n, k, seed + 1, exponents=True), numbers(m, k, seed + 2)
    ad, wd = a.to(DEV).double(), w.to(DEV).double()
    assert float((ad.abs() @ wd.abs().T).max()) * 8 < 2 ** 24
    # every chunk of k counts: without it most results differ
    for c in range(0, k, 256):
        part = ad[:, c:c + 256] @ wd[:, c:c + 256].T
        assert (part != 0).double().mean() > 0.5
    return a, w, (ad @ wd.T).cpu()


def test_numbers_stand_for_themselves():
    for k in (1, 33, 300, 1037):
        a = numbers(5, k, 1, exponents=True)
        assert torch.equal(plain_blocks(a)[2], a.double())
        assert torch.equal(plain_blocks(a.to(BF16))[2], a.double())


# one token; few long rows, through several rounds of a product's stages; tiles of 16, 32, 64 and 128 rows with k in
# parts; rows packed ahead; pairs' tiles, whole, shared out along k, and both
SHAPES = [(1, 300, 30000), (5, 300, 30000), (16, 140, 26624), (20, 260, 30000), (32, 128, 30464), (3, 70, 29999),
          (1, 6144, 2560), (8, 2560, 9728), (33, 300, 512), (40, 1003, 1000), (64, 140, 2048), (77, 1003, 1037),
          (97, 500, 264), (128, 256, 9728), (128, 260, 768), (127, 130, 3001), (100, 6000, 700), (128, 3000, 2560),
          (70, 1280, 2560), (129, 385, 320), (140, 257, 40000), (300, 700, 9728), (513, 300, 1000), (2048, 2560, 4096),
          (600, 20000, 3000)]


@pytest.mark.parametrize("n,m,k", SHAPES)
def test_every_chunk_of_k_counts(n, m, k):
    o = ops()
    a, w, want = exact_case(n, m, k)
    qw = o.mx4_quantize(w.to(DEV))
    for rows in (a.to(DEV), a.to(DEV, BF16), o.mx4_quantize(a.to(DEV))):
        got = o.linear_mx4(rows, qw)
        assert torch.equal(got.cpu().double(), want)
        assert torch.equal(o.linear_mx4(rows, qw, BF16).cpu(), want.to(F32).to(BF16))
    assert o.gemm_tc_error() == 0


@pytest.mark.parametrize("n,m,k,c", [(1, 200, 30000, 117), (16, 140, 26624, 50), (64, 140, 2048, 3), (128, 256, 9728, 37),
                                     (140, 257, 40000, 156), (300, 700, 9728, 20)])
def test_one_chunk_alone(n, m, k, c):
    """All of k zero but for one chunk."""
    o = ops()
    a, w = numbers(n, k, 3), numbers(m, k, 4)
    a[:, :256 * c] = 0.0
    a[:, 256 * (c + 1):] = 0.0
    want = a.double() @ w.double().T
    got = o.linear_mx4(a.to(DEV), o.mx4_quantize(w.to(DEV)))
    assert (want != 0).double().mean() > 0.5 and torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("n,m,k", [(300, 700, 9728), (2048, 2560, 4096), (77, 1003, 1037), (600, 1280, 2560)])
def test_rows_alone_and_among_others(n, m, k):
    """A row's results do not depend on how many rows there are beyond the rounding of its sums, whose parts of k differ:
    k / 64 MMAs and at most 16 parts added up, each step off by at most two units in the last place (4 U) of the sum of
    magnitudes, in both."""
    o = ops()
    g = torch.Generator().manual_seed(n)
    a, w = torch.randn(n, k, generator=g).to(DEV), o.mx4_quantize((torch.randn(m, k, generator=g) * 0.02).to(DEV))
    whole = o.linear_mx4(a, w)
    size = o.mx4_values(o.mx4_quantize(a)).double().abs() @ o.mx4_values(w).double().abs().T
    for rows in (slice(0, 1), slice(5, 25), slice(n - 60, n)):
        alone = o.linear_mx4(a[rows].contiguous(), w)
        off = (alone.double() - whole[rows].double()).abs()
        assert (off <= 2 * 4 * U32 * (k / 64 + 16) * size[rows]).all()


@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 16), (8, 2, 128)])
def test_attention_is_its_operators(nh, nkv, hd):
    """q|k|v and o in 4 bits, bit for bit.  The rows and the weights of q, k and v are 4-bit numbers, so a part whose
    weights are the same numbers in bfloat16 has the same q, k and v; with an identity for o it gives attention's result
    itself, and the 4-bit product of that with o is what the part in 4 bits must give."""
    from janas_b200.cache import Cache
    from janas_b200.config import PartSpec
    from janas_b200.parts import LayerCache
    from test_parts_gpu import build, context
    o = ops()
    hidden, n = nh * hd, 75
    x = numbers(n, hidden, 5).to(DEV, BF16)
    qkv = {f"a.{t}_proj.weight": numbers(heads * hd, hidden, 6 + i).to(DEV, BF16)
           for i, (t, heads) in enumerate((("q", nh), ("k", nkv), ("v", nkv)))}
    wo = torch.randn(hidden, hidden, generator=torch.Generator().manual_seed(9)).to(DEV, BF16)
    norms = {f"a.{t}_norm.weight": torch.ones(hd, device=DEV, dtype=BF16) for t in "qk"}
    pos = PartSpec("rope_neox", {"rotary_dim": hd, "theta": 1e4, "max_positions": 128})
    spec = PartSpec("gqa_attention", {"hidden_size": hidden, "num_heads": nh, "num_kv_heads": nkv, "head_dim": hd,
                                      "qk_norm_eps": 1e-5, "window": 0, "position": pos})

    def runs(last, pack):
        part = build("mixer", spec, BF16)
        part.load("a", {**qkv, **norms, "a.o_proj.weight": last})
        if pack:
            assert part.pack() == 2
        part.prepare(128)
        cache = Cache([part.kv_spec()], [None], 128, 1, BF16, torch.device(DEV))
        s, g = cache.new_sequence(), cache.groups[0]
        out, at = [], 0
        for cnt in (60, 1, 1, 13):
            cache.reserve([s], [cnt])
            lc = LayerCache(k=g.k[0], v=g.v[0], block_table=torch.from_numpy(cache.block_table(g, [s])).to(DEV))
            out.append(part.forward(context([at], [cnt], BF16), x[at:at + cnt].contiguous(), lc).sum(0))
            cache.advance([s], [cnt])
            at += cnt
        return out

    plain, packed = runs(torch.eye(hidden, device=DEV, dtype=BF16), False), runs(wo, True)
    qo = o.mx4_quantize(wo)
    for a, got in zip(plain, packed):
        assert torch.equal(got, o.linear_mx4(a.to(BF16), qo)) and torch.equal(a, a.to(BF16).float())


def test_one_by_one_captured_and_not():
    """Prompts that run alone: captured decode steps give the tokens that eager ones do."""
    import janas_b200
    from helpers import model_dir
    from janas_b200 import lib
    from tiny import TINY, tokens
    rng = np.random.default_rng(7)
    prompts = [tokens(rng, n, TINY["D"]["vocab_size"]) for n in (3, 17, 80)]
    llm = janas_b200.open(model_dir("D"), janas_b200.LLMParams(n_ctx=256, max_batch=4, max_tokens=1024, weights="mx4"))
    captured = [llm.generate(p, 20)[0] for p in prompts]
    assert llm.engine.info()["graph_captures"] > 0
    lib.call("llm.set", llm=llm.engine._h.value, use_graphs=False)
    assert [llm.generate(p, 20)[0] for p in prompts] == captured
    llm.close()
