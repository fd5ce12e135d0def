"""Results at addresses that the kernels' widest stores do not fit: the C entries refuse them before a launch.  The
addresses stand for device memory that nothing reads."""
import pytest

from janas_b200.csrc import ops

EINVAL = -1
GOOD = 1 << 20


@pytest.mark.parametrize("off", [1, 2, 4, 8])
@pytest.mark.parametrize("dm", [64, 63])
def test_norms_refuse_codes_anywhere(off, dm):
    L = ops.lib()
    assert L.jb_norm_residual_norm(GOOD, GOOD, 1, dm, None, None, 0, 0, 0, 0, None, GOOD, None, 1e-5, None, 1.0, GOOD, None,
                                   1e-5, 1, GOOD + off, GOOD, 4, 1, dm, None) == EINVAL


@pytest.mark.parametrize("off", [1, 2, 4, 8])
@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("dt", [0, 1])
def test_products_refuse_results_anywhere(off, n, dt):
    """A result of a product that is joined from parts of k is stored four values at a time."""
    L = ops.lib()
    m, k = 256, 2560
    assert L.jb_linear_mx4(GOOD, GOOD, GOOD, GOOD, GOOD + off, dt, n, m, k, GOOD, 0, None) == EINVAL
    assert L.jb_linear_mx4_rows(GOOD, 1, GOOD, GOOD, GOOD + off, dt, n, m, k, GOOD, 0, None) == EINVAL
