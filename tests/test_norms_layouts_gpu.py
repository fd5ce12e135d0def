"""The norms around a sublayer on rows that lie elsewhere in memory: a row's bits are the same wherever whole 16-byte loads
fit, and elsewhere it is as near to 64 bits."""
import pytest
import torch

from test_mx4_gpu import U32, norm_error, plain_norm, rnd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def moved(t, off):
    """A copy that starts ``off`` floats behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 8, device=DEV)
    out = flat[off:off + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 == 4 * (off % 4)
    return out


@pytest.mark.parametrize("dm", [64, 516, 2560])
@pytest.mark.parametrize("rms", [True, False])
def test_rows_of_a_batch_that_lie_elsewhere(dm, rms):
    from janas_b200.csrc import ops
    n = 40
    x, y, g = rnd(n, dm, scale=3.0), rnd(n, dm, seed=1), rnd(n, dm, seed=2)
    w = 1 + rnd(dm, scale=0.1)
    wide = torch.cat([rnd(n, 3, seed=3), g], 1)           # the gate from a column that 16 bytes do not divide
    W = w.to(DEV)
    whole = x.to(DEV).clone()
    h = ops.norm_residual_norm(whole, y.to(DEV), W, W, 1e-5, rms, y_gate=g.to(DEV))
    u = y.double() * torch.sigmoid(g.double())
    wx = x.double() + plain_norm(u, w, None, 1e-5, rms)
    wh = plain_norm(wx, w, None, 1e-5, rms)
    # the gate's product and its sigmoid: the argument's rounding, the exponential's two, the reciprocal's and the product's
    ex = norm_error(u, 8 * U32 * u.abs().amax(-1), w, None, 1e-5, rms)
    ex = ex + 4 * U32 * ((wx - x.double()).abs().amax(-1) + wx.abs().amax(-1))
    eh = norm_error(wx, ex, w, None, 1e-5, rms) + 2 * U32 * wh.abs().amax(-1)
    rows = slice(7, 30)
    for off, at in ((0, 0), (4, 0), (1, 0), (2, 0), (3, 0), (0, 3)):
        xr = moved(x[rows], off)
        gate = moved(wide[rows], 0) if at else moved(g[rows], off)
        hr = ops.norm_residual_norm(xr, moved(y[rows], off), W, W, 1e-5, rms, y_gate=gate, gate_col0=at)
        if off % 4 == 0 and not at:
            assert torch.equal(xr, whole[rows]) and torch.equal(hr, h[rows])
        assert ((xr.cpu().double() - wx[rows]).abs() <= ex[rows, None]).all()
        assert ((hr.cpu().double() - wh[rows]).abs() <= eh[rows, None]).all()
