"""Microscaled 4-bit floats: rows and matrices brought to them and back, their products, the
norms around a sublayer, and all of them together, against plain forms in 64 bits.

The tolerances count roundings: a float32 is off by at most 2^-24 of its value, a bfloat16 by 2^-8; each test says
how many."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
DTYPES = [F32, BF16]
U32 = torch.finfo(F32).eps / 2
UBF = torch.finfo(BF16).eps / 2


def ops():
    from janas_b200.csrc import ops as o
    return o


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def plain_blocks(x):
    """(numbers, exponents, values) of x [n, k] in blocks of 32, by looking for the nearest of the eight magnitudes."""
    x = x.double().numpy()
    n, k = x.shape
    kb = -(-k // 32)
    p = np.zeros((n, kb * 32))
    p[:, :k] = x
    p = p.reshape(n, kb, 32)
    top = np.abs(p).max(-1)
    bad = ~np.isfinite(top)
    _, e = np.frexp(np.where(bad, 1.0, top))
    s = np.where(top > 0, np.maximum(e - 1 - 2, -127), -127)
    v = np.abs(np.where(bad[..., None], 0.0, p)) / np.ldexp(1.0, s)[..., None]
    q = np.zeros_like(v)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        q = np.where((v > mid) | ((v == mid) & (i % 2 == 1)), GRID[i + 1], q)     # a tie: the even index
    q = np.copysign(q, p)
    out = q * np.ldexp(1.0, s)[..., None]
    out[bad] = np.nan
    return q, s, torch.from_numpy(out.reshape(n, kb * 32)[:, :k].copy())


def special_rows(k, dtype):
    """Rows with every border between two numbers, zeros, the smallest and largest floats."""
    x = rnd(16, k, scale=1.0, seed=5)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, -0.25, -0.75, -1.25, -5.0, -7.5, 4.0])
    for r in range(6):
        m = min(k, 16)
        x[r, :m] = ties[:m] * 2.0 ** (3 * r - 8)
        x[r, m:] *= 2.0 ** (3 * r - 10)
    x[6] = 0.0
    x[7] = 1e-38                    # below: the exponent stops at -127
    x[8] = 2.0 ** -130
    x[9] = 3.3e38
    x[10] *= 1e30
    x[11, : max(1, k - 1)] = 0.0    # one value alone in the last block
    x[12] = -0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (1, 32), (3, 31), (5, 33), (130, 256), (129, 257), (8, 2560), (33, 1000), (7, 9728),
                                 (1000, 72), (2, 40000)])
def test_quantize(dtype, n, k):
    """Codes, scales and values bit by bit: every step of the definition is exact."""
    o = ops()
    x = torch.cat([rnd(n, k, dtype=dtype, scale=3.0), special_rows(k, dtype)])
    q = o.mx4_quantize(x.to(DEV))
    num, s, want = plain_blocks(x)
    rows, kb = x.shape[0], -(-k // 32)
    assert q.shape == (rows, k)
    codes = q.codes.cpu().numpy()
    assert codes.shape == (rows, kb * 16)
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(rows, kb, 32)
    got = np.where(nib & 8, -1.0, 1.0) * GRID[nib & 7]
    assert np.array_equal(got, num)
    sc = q.scales.cpu().numpy()
    for r in range(0, rows, max(1, rows // 40)):
        for b in range(kb):
            at = 512 * (b % 8 // 4) + 16 * (r % 32) + 4 * (r // 32 % 4) + b % 4
            assert sc[r // 128, b // 8, at] == s[r, b] + 127
    for odt in DTYPES:
        assert torch.equal(o.mx4_values(q, odt).cpu().double(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_not_finite(dtype):
    """A NaN or an infinity makes its block NaN, and no other."""
    o = ops()
    x = rnd(6, 100, dtype=dtype)
    x[0, 0], x[1, 40], x[2, 99], x[3, 64] = math.nan, math.inf, -math.inf, math.nan
    _, _, want = plain_blocks(x)
    got = o.mx4_values(o.mx4_quantize(x.to(DEV))).cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and got.isnan().sum() == 32 + 32 + 4 + 32
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_quantize_addresses(dtype, offset):
    """Rows whose first value lies at any address."""
    o = ops()
    flat = rnd(64 * 5 + 16, dtype=dtype).to(DEV)
    x = flat[offset:offset + 320].view(5, 64)
    assert torch.equal(o.mx4_values(o.mx4_quantize(x)).cpu().double(), plain_blocks(x.cpu())[2])


@pytest.mark.parametrize("S,n,ff,unit", [(1, 1, 1, (1.0, 0.0, 0.0)), (1, 9, 100, (1.0, 0.0, 0.0)), (3, 5, 333, (1.702, 7.0, 1.0)),
                                         (1, 130, 9728, (1.0, 0.0, 0.0)), (2, 33, 256, (1.0, 2.0, 0.0))])
def test_gated_unit(S, n, ff, unit):
    """The unit's values lie within a step of their block of the plain ones: the unit in float32 may fall on the other
    side of a border, or of a power of two."""
    o = ops()
    z = rnd(S, n, 2 * ff, seed=2)
    got = o.mx4_values(o.mx4_gated_unit(z.to(DEV), *unit)).cpu().double()
    t = z.double().sum(0)
    g, u = t[:, :ff], t[:, ff:]
    alpha, limit, shift = unit
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    act = g * torch.sigmoid(alpha * g) * (u + shift)
    _, s, want = plain_blocks(act)
    # float32: the sums (S roundings), the exponential and its argument, the divide and two products
    near = (S + 12) * U32 * (z.double().abs().sum(0).max() ** 2 + 1)
    step = torch.from_numpy(np.ldexp(1.0, s)).repeat_interleave(32, 1)[:, :ff]
    # what differs lies at a border: the ends of the error's interval differ as well
    lo, hi = plain_blocks(act - near)[2], plain_blocks(act + near)[2]
    assert ((lo != hi) | (got == want)).all()
    assert ((got - want).abs() <= 4.0 * step).all()
    assert (got != want).double().mean() <= 1e-3 + 33.0 / (n * ff)


def product_case(n, m, k, seed=0):
    o = ops()
    a, w = rnd(n, k, seed=seed), rnd(m, k, scale=0.02, seed=seed + 1)
    a[:, :: max(1, k // 5)] *= 8.0
    return o, a, w, plain_blocks(a)[2], plain_blocks(w)[2]


# a product's float32 sum: the products of 4-bit numbers and their scales are exact; a sum of k / 32 blocks in any order,
# rounded or cut off at each of at most k steps, is off by at most k U of the sum of magnitudes (twice that, cut off)
def product_bound(av, wv, k):
    return 2 * k * U32 * (av.abs() @ wv.abs().T) + 1e-30


SHAPES = [(1, 1, 1), (1, 16, 32), (3, 5, 31), (1, 6144, 2560), (8, 300, 2560), (16, 129, 257), (17, 128, 256), (33, 1000, 1037),
          (64, 512, 100), (65, 127, 4096), (77, 1003, 1037), (128, 256, 9728), (129, 385, 320), (200, 640, 2560),
          (300, 1024, 96), (513, 300, 1000), (1030, 257, 513)]


@pytest.mark.parametrize("n,m,k", SHAPES)
def test_linear(n, m, k):
    o, a, w, av, wv = product_case(n, m, k)
    want, tol = av @ wv.T, product_bound(av, wv, k)
    qw = o.mx4_quantize(w.to(DEV))
    got = o.linear_mx4(a.to(DEV), qw)
    assert got.shape == (n, m) and got.dtype == F32
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), (off / tol).max()
    # rows given in 4 bits, and once more: the same bits
    again = o.linear_mx4(o.mx4_quantize(a.to(DEV)), qw)
    assert torch.equal(again, got)
    half = o.linear_mx4(a.to(DEV), qw, BF16)
    assert half.dtype == BF16 and torch.equal(half, got.to(BF16))
    assert o.gemm_tc_error() == 0


@pytest.mark.parametrize("n", [0, 1, 5, 200])
def test_linear_of_bfloat16_rows(n):
    o = ops()
    a, w = rnd(n, 96, dtype=BF16), rnd(70, 96)
    got = o.linear_mx4(a.to(DEV), o.mx4_quantize(w.to(DEV)))
    av, wv = plain_blocks(a)[2], plain_blocks(w)[2]
    assert got.shape == (n, 70)
    assert ((got.cpu().double() - av @ wv.T).abs() <= product_bound(av, wv, 96)).all()


@pytest.mark.parametrize("n", [2, 40, 200])
def test_linear_not_finite(n):
    """A NaN or an infinity in a row, or in a feature, reaches all of that row or feature and nothing else."""
    o = ops()
    a, w = rnd(n, 300), rnd(200, 300)
    a[1, 7], w[150, 299], w[3, 40] = math.inf, math.nan, -math.inf
    got = o.linear_mx4(a.to(DEV), o.mx4_quantize(w.to(DEV))).cpu()
    want = torch.zeros(n, 200, dtype=torch.bool)
    want[1], want[:, 150], want[:, 3] = True, True, True
    assert torch.equal(got.isnan(), want) and got[~want].isfinite().all()


@pytest.mark.parametrize("n,m,k", [(8, 256, 512), (150, 256, 512)])
def test_linear_wide_scales(n, m, k):
    """Blocks whose powers of two lie far apart: each meets its own scale."""
    o = ops()
    e = torch.randint(-30, 30, (n, k // 32), generator=torch.Generator().manual_seed(3))
    f = torch.randint(-30, 30, (m, k // 32), generator=torch.Generator().manual_seed(4))
    a = rnd(n, k) * torch.exp2(e.float()).repeat_interleave(32, 1)
    w = rnd(m, k, seed=1) * torch.exp2(f.float()).repeat_interleave(32, 1)
    av, wv = plain_blocks(a)[2], plain_blocks(w)[2]
    got = o.linear_mx4(a.to(DEV), o.mx4_quantize(w.to(DEV))).cpu().double()
    assert ((got - av @ wv.T).abs() <= product_bound(av, wv, k)).all()


def plain_norm(t, w, b, eps, rms):
    t = t.double()
    if not rms:
        t = t - t.mean(-1, keepdim=True)
    r = t / ((t * t).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return r if b is None else r + b.double()


def norm_error(t, et, w, b, eps, rms):
    """How far a float32 norm of rows that are off by et [n] may be from the one of the rows t, per row.

    With c roundings in a sum of the row's terms (dm / 32 one after the other and a tree): the mean is off by et and
    c U max |t|; the deviation d by both and one rounding; 1 / sqrt(var + eps) by the relative error of d over the
    deviation's root mean square and by c + 8 roundings."""
    c = t.shape[1] / 32 + 16
    top = t.abs().amax(-1)
    d = t if rms else t - t.mean(-1, keepdim=True)
    sigma = (d.pow(2).mean(-1) + eps).sqrt()
    R = d.abs().amax(-1) / sigma
    ed = et + U32 * top + (0 if rms else et + c * U32 * top)
    return float(w.abs().max()) * (ed / sigma * (1 + R) + (c + 8) * U32 * R) + 2 * U32 * (float(b.abs().max()) if b is not None else 0)


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("n,dm,S", [(1, 1, 1), (1, 32, 2), (3, 100, 1), (8, 2560, 14), (33, 1037, 3), (5, 8192, 1), (4, 9001, 2),
                                    (200, 256, 1), (300, 2560, 1), (700, 516, 2), (2, 32768, 1), (1100, 64, 1), (4000, 516, 2), (1000, 2560, 1), (10000, 64, 1), (1500, 4100, 1)])
def test_norm_residual_norm(n, dm, S, gate, rms):
    o = ops()
    x, y = rnd(n, dm, scale=3.0), rnd(S, n, dm, seed=1)
    x[:, dm // 2] = 60.0
    yb, pw, pb, nw, nb, sc = (rnd(dm, seed=i, scale=0.1) + (1.0 if i in (3, 5) else 0.0) for i in range(2, 8))
    g, gb = rnd(2, n, dm + 7, seed=9), rnd(dm, seed=10)
    u = y.double().sum(0) + yb.double()
    if gate:
        u = u * torch.sigmoid(g.double().sum(0)[:, 5:5 + dm] + gb.double())
    wx = x.double() + sc.double() * plain_norm(u, pw, pb, 1e-5, rms)
    wh = plain_norm(wx, nw, nb, 1e-6, rms)
    # the sums' roundings, and a sigmoid whose argument is off by three of its own
    eu = (S + 2) * U32 * (y.double().abs().sum(0) + yb.double().abs()).amax(-1)
    eu = eu + (4 * U32 * (g.double().abs().sum(0).amax() + 1) + 8 * U32) * u.abs().amax(-1)
    ex = norm_error(u, eu, pw, pb, 1e-5, rms) * float(sc.abs().max())
    ex = ex + 4 * U32 * ((wx - x.double()).abs().amax(-1) + wx.abs().amax(-1))
    eh = norm_error(wx, ex, nw, nb, 1e-6, rms) + 2 * U32 * wh.abs().amax(-1)
    D = lambda t: None if t is None else t.to(DEV)   # noqa: E731
    for out in (F32, BF16, "mx4"):
        xd = D(x.clone())
        h = o.norm_residual_norm(xd, D(y), D(pw), D(nw), 1e-5, rms, D(yb), D(g) if gate else None, 5 if gate else 0,
                                 D(gb) if gate else None, D(sc), D(pb), D(nb), out, 1e-6)
        assert ((xd.cpu().double() - wx).abs() <= ex[:, None]).all()
        if out == "mx4":
            got = o.mx4_values(h).cpu().double()
            _, s, want = plain_blocks(wh)
            step = torch.from_numpy(np.ldexp(1.0, s)).repeat_interleave(32, 1)[:, :dm]
            # six is the largest number and stands for up to eight: two steps; a block that falls on the other side of a
            # power of two is off by one of these at most
            assert ((got - wh).abs() <= 2 * step * (1 + 1e-6) + eh[:, None]).all()
            assert (got != want).double().mean() <= 1e-3 + 33.0 / (n * dm)
        else:
            far = (h.cpu().double() - wh).abs()
            lim = eh[:, None] + (UBF * (wh.abs() + eh[:, None]) if out == BF16 else 0.0)
            assert (far <= lim).all(), (far / lim).max()


def test_norms_parts_left_out():
    """No norm of the result, no scale, a number for a scale, no next norm; x alone is then written."""
    o = ops()
    x, y, w = rnd(9, 300), rnd(9, 300, seed=1), 1 + rnd(300, scale=0.1)
    xd = x.to(DEV).clone()
    assert o.norm_residual_norm(xd, y.to(DEV), None, None, 1e-5, scale=0.5) is None
    assert torch.equal(xd.cpu(), x + 0.5 * y)
    xd = x.to(DEV).clone()
    h = o.norm_residual_norm(xd, y.to(DEV), None, w.to(DEV), 1e-5, out=F32)
    assert torch.equal(xd.cpu(), x + y)
    want = plain_norm(x + y, w, None, 1e-5, True)
    assert ((h.cpu().double() - want).abs() <= 64 * U32 * want.abs().max()).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_norms_not_finite(bad):
    """A value that is not finite makes its own row NaN, in 4 bits too, and no other."""
    o = ops()
    x, y, w = rnd(40, 512), rnd(40, 512, seed=1), torch.ones(512)
    y[7, 100] = bad
    for out in (F32, BF16, "mx4"):
        h = o.norm_residual_norm(x.to(DEV).clone(), y.to(DEV), w.to(DEV), w.to(DEV), 1e-5, out=out)
        h = (o.mx4_values(h) if out == "mx4" else h).cpu().float()
        assert h[7].isnan().any() and h[:7].isfinite().all() and h[8:].isfinite().all()
        if out == "mx4":
            assert h[7].isnan().all()


@pytest.mark.parametrize("n", [1, 8, 40, 300])
def test_feed_forward_in_4_bits(n):
    """Norms, gate-up, the gated unit and down as they follow one another: bit for bit what the steps give one by one
    with every 4-bit matrix written out and read back."""
    o = ops()
    dm, ff = 320, 712
    x, y, w1, w2, sc = rnd(n, dm), rnd(n, dm, seed=1), 1 + rnd(dm, scale=0.1), 1 + rnd(dm, scale=0.1, seed=2), rnd(dm, seed=3)
    gu, down = o.mx4_quantize(rnd(2 * ff, dm, scale=0.05).to(DEV)), o.mx4_quantize(rnd(dm, ff, scale=0.05, seed=4).to(DEV))
    xd, xe = x.to(DEV).clone(), x.to(DEV).clone()
    h = o.norm_residual_norm(xd, y.to(DEV), w1.to(DEV), w2.to(DEV), 1e-5, scale=sc.to(DEV), out="mx4")
    z = o.linear_mx4(h, gu)
    act = o.mx4_gated_unit(z)
    got = o.linear_mx4(act, down)
    # one by one, from floats
    hf = o.norm_residual_norm(xe, y.to(DEV), w1.to(DEV), w2.to(DEV), 1e-5, scale=sc.to(DEV), out=F32)
    assert torch.equal(xd, xe)
    assert torch.equal(o.mx4_values(h), o.mx4_values(o.mx4_quantize(hf)))
    assert torch.equal(z, o.linear_mx4(hf, gu))
    av = o.mx4_values(act).cpu().double()
    dv = o.mx4_values(down).cpu().double()
    assert ((got.cpu().double() - av @ dv.T).abs() <= product_bound(av, dv, ff)).all()
    unit = o.swiglu(z, F32)
    assert torch.equal(o.mx4_values(o.mx4_quantize(unit)), o.mx4_values(act))


@pytest.mark.parametrize("n", [4, 200])
def test_captured(n):
    """The chain in a CUDA graph, replayed with other rows, on a stream of its own."""
    o = ops()
    dm, ff = 256, 512
    w1 = torch.ones(dm, device=DEV)
    gu, down = o.mx4_quantize(rnd(2 * ff, dm).to(DEV)), o.mx4_quantize(rnd(dm, ff, seed=4).to(DEV))
    x, y = rnd(n, dm).to(DEV), rnd(n, dm, seed=1).to(DEV)

    def chain():
        h = o.norm_residual_norm(x, y, w1, w1, 1e-5, out="mx4")
        return o.linear_mx4(o.mx4_gated_unit(o.linear_mx4(h, gu)), down)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for seed in (11, 12):
        x0, y0 = rnd(n, dm, seed=seed).to(DEV), rnd(n, dm, seed=seed + 50).to(DEV)
        x.copy_(x0), y.copy_(y0)
        graph.replay()
        torch.cuda.synchronize()
        replayed, xr = got.clone(), x.clone()
        x.copy_(x0)
        want = chain()
        assert torch.equal(replayed, want) and torch.equal(xr, x)


def test_refusals():
    o = ops()
    E = o.KernelError
    x = rnd(4, 64).to(DEV)
    q = o.mx4_quantize(x)
    for bad in (x.cpu(), x.half(), x.t(), x[0], x.to(torch.int32), torch.empty((3, 0), device=DEV)):
        with pytest.raises(E):
            o.mx4_quantize(bad)
    for a, w, dt in ((rnd(2, 63).to(DEV), q, F32), (x.cpu(), q, F32), (x, x, F32), (x, q, torch.float16),
                     (o.mx4_quantize(rnd(2, 65).to(DEV)), q, F32), (x.t(), q, F32)):
        with pytest.raises(E):
            o.linear_mx4(a, w, dt)
    with pytest.raises(E):
        o.mx4_values(q, torch.float16)
    with pytest.raises(E):
        o.mx4_gated_unit(rnd(3, 7).to(DEV))
    with pytest.raises(E):
        o.Mx4(q.codes, q.scales, 5, 64)
    with pytest.raises(E):
        o.Mx4(q.codes.view(-1)[1:].new_empty(4, 32)[:, :].t().contiguous().t(), q.scales, 4, 64)
    w = torch.ones(64, device=DEV)
    good = dict(x=x, y=x.clone(), post_weight=w, next_weight=w, eps=1e-5)
    for change in (dict(x=x.cpu()), dict(y=x[:3]), dict(y=x.bfloat16()), dict(post_weight=w[:63]), dict(next_weight=w.bfloat16()),
                   dict(y_gate=x[:, :60].contiguous()), dict(y_gate=x, gate_col0=1), dict(y_gate=x, gate_col0=-1),
                   dict(gate_bias=w), dict(scale=w[:3]), dict(out=torch.float16), dict(post_weight=None, post_bias=w),
                   dict(next_weight=None, next_bias=w), dict(y=x.new_empty((0, 4, 64)))):
        with pytest.raises(E):
            o.norm_residual_norm(**{**good, **change})
    wide = torch.zeros((1, o.lib().jb_norm_residual_norm_most() + 1), device=DEV)
    with pytest.raises(E):
        o.norm_residual_norm(wide, wide.clone(), None, None, 1e-5)
    # nothing of a refused call was launched
    assert torch.equal(o.mx4_values(q), o.mx4_values(o.mx4_quantize(rnd(4, 64).to(DEV))))


def test_no_rows():
    o = ops()
    w = o.mx4_quantize(rnd(70, 96).to(DEV))
    e = torch.empty((0, 96), device=DEV)
    assert o.mx4_values(o.mx4_quantize(e)).shape == (0, 96)
    assert o.linear_mx4(e, w).shape == (0, 70)
    assert o.linear_mx4(rnd(3, 96).to(DEV), o.mx4_quantize(e)).shape == (3, 0)
    one = torch.ones(96, device=DEV)
    assert o.norm_residual_norm(e, e.clone(), one, one, 1e-5, out="mx4").shape == (0, 96)
    assert o.mx4_gated_unit(torch.empty((0, 96), device=DEV)).shape == (0, 48)


# the last: 237 tiles on 74 pairs leave 15, four pairs for each; sharing 12 chunks of k among four saves nine, too few
@pytest.mark.parametrize("n,m,k,launches", [(300, 700, 9728, 2), (2048, 2560, 4096, 2), (140, 257, 40000, 2),
                                            (600, 20000, 3000, 1)])
def test_linear_shared_tiles(n, m, k, launches):
    """Products whose last tiles are shared out along k: the same sums, once more the same bits, and rows that do not
    depend on how many there are beyond the rounding of the parts' sums."""
    o, a, w, av, wv = product_case(n, m, k)
    assert o.lib().jb_linear_mx4_launches(n, m, k, 0) == launches
    qa, qw = o.mx4_quantize(a.to(DEV)), o.mx4_quantize(w.to(DEV))
    got = o.linear_mx4(qa, qw)
    some = torch.randperm(n, generator=torch.Generator().manual_seed(1))[:40]
    want, tol = av[some] @ wv.T, product_bound(av[some], wv, k)
    assert ((got.cpu().double()[some] - want).abs() <= tol).all()
    assert torch.equal(got, o.linear_mx4(qa, qw)) and torch.equal(got.to(BF16), o.linear_mx4(qa, qw, BF16))
    assert o.gemm_tc_error() == 0


@pytest.mark.parametrize("n,dm,rms", [(1000, 2560, True), (10000, 64, False), (4000, 516, True)])
def test_norms_rows_by_themselves(n, dm, rms):
    """A row's bits do not depend on how many rows there are."""
    o = ops()
    x, y, g = rnd(n, dm).to(DEV), rnd(n, dm, seed=1).to(DEV), rnd(n, dm, seed=2).to(DEV)
    w = (1 + rnd(dm, scale=0.1)).to(DEV)
    xs = x.clone()
    h = o.norm_residual_norm(xs, y, w, w, 1e-5, rms, y_gate=g)
    for rows in (slice(0, 3), slice(n - 7, n)):
        few = x[rows].clone()
        hf = o.norm_residual_norm(few, y[rows].clone(), w, w, 1e-5, rms, y_gate=g[rows].clone())
        assert torch.equal(few, xs[rows]) and torch.equal(hf, h[rows])
    assert o.gemm_tc_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,m,k", [(1, 300, 30000), (5, 300, 30000), (16, 140, 26624), (20, 260, 30000), (32, 128, 30464), (3, 70, 29999)])
def test_linear_of_few_long_rows(dtype, n, m, k):
    """Rows packed in the product's kernel through several rounds of its stages."""
    o, a, w, _, wv = product_case(n, m, k)
    a = a.to(dtype)
    av = plain_blocks(a)[2]
    got = o.linear_mx4(a.to(DEV), o.mx4_quantize(w.to(DEV)))
    assert ((got.cpu().double() - av @ wv.T).abs() <= product_bound(av, wv, k)).all()
    assert torch.equal(got, o.linear_mx4(o.mx4_quantize(a.to(DEV)), o.mx4_quantize(w.to(DEV))))
    assert o.gemm_tc_error() == 0


@pytest.mark.parametrize("n", [5, 60, 300])
def test_weights_given_as_codes(n):
    """Codes and scales that the caller has written, right ahead of the product, in tensors of their own and in place."""
    o = ops()
    a, w = rnd(n, 544).to(DEV), o.mx4_quantize(rnd(400, 544, seed=1).to(DEV))
    want = o.linear_mx4(a, w)
    other = o.linear_mx4(a, o.mx4_quantize(rnd(400, 544, seed=2).to(DEV)))
    codes, scales = torch.zeros_like(w.codes), torch.zeros_like(w.scales)
    given = o.Mx4(codes, scales, 400, 544)
    qa = o.mx4_quantize(a)
    for _ in range(20):
        codes.copy_(w.codes), scales.copy_(w.scales)
        assert torch.equal(o.linear_mx4(qa, given), want)
        codes.zero_()
        assert not o.linear_mx4(qa, given).any()
    v = o.mx4_quantize(rnd(400, 544, seed=2).to(DEV))
    assert v.settled and torch.equal(o.linear_mx4(qa, v), other)
    v.codes.copy_(w.codes), v.scales.copy_(w.scales)
    assert not v.settled and torch.equal(o.linear_mx4(qa, v), want)


def test_norms_refuse_other_shapes_of_sums():
    o = ops()
    x, w = rnd(4, 64).to(DEV), torch.ones(64, device=DEV)
    for y in (x.view(1, 1, 4, 64), x.view(2, 2, 64), x[:, :63], x.view(-1), [1.0], x.cpu(), x.double()):
        with pytest.raises(o.KernelError):
            o.norm_residual_norm(x, y, w, w, 1e-5)
    with pytest.raises(o.KernelError):
        o.norm_residual_norm(x.bfloat16(), x, w, w, 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
# (a warp's items: an eighth of a tile's rows by a part's chunks.  128 x 260 x 768: 24 tiles of 16 rows, two parts of at most
# 2 chunks, 4 items; 127 x 130 x 3,001: 16 tiles, eight parts of at most 2; 128 x 3,000 x 2,560: 192 tiles of 16 rows, one
# part of 10, 20 items, over 12, and 96 of 32 rows, two parts of 5, 20 items too; 100 x 6,000 x 700: 329 tiles of 16 rows, over
# two an SM, and 188 of 32 rows, one part of 3, 12 items)
@pytest.mark.parametrize("n,m,k,launches", [(33, 300, 512, 1), (40, 1003, 1000, 1), (64, 140, 2048, 1), (70, 200, 1024, 1),
                                            (97, 500, 264, 1), (128, 260, 768, 1), (128, 260, 512, 1), (127, 130, 3001, 1), (128, 3000, 2560, 2),
                                            (100, 6000, 700, 1)])
def test_linear_of_some_rows(dtype, n, m, k, launches):
    """33 to 128 rows of floats: packed in the product's kernel where its CTAs have little to pack, ahead of it otherwise."""
    o, a, w, _, wv = product_case(n, m, k)
    assert o.lib().jb_linear_mx4_launches(n, m, k, 1) == launches
    a = a.to(dtype)
    av = plain_blocks(a)[2]
    qw = o.mx4_quantize(w.to(DEV))
    got = o.linear_mx4(a.to(DEV), qw)
    assert ((got.cpu().double() - av @ wv.T).abs() <= product_bound(av, wv, k)).all()
    half = o.linear_mx4(a.to(DEV), qw, BF16)
    assert torch.equal(half, got.to(BF16))
    assert o.gemm_tc_error() == 0
