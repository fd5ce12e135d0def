"""Products in 4 bits whose CTAs form clusters: a CTA that waits for tensor memory has no time limit, and one of its
cluster that has its columns keeps them meanwhile.  So as many of them as fit an SM's shared memory, of any products side by
side, must find columns there.  What the library says of its launches is checked by arithmetic; no GPU."""
import ctypes

import pytest

from janas_b200.csrc import ops

SMEM, OWN, MOST, COLS = 228 * 1024, 1024, 227 * 1024, 512     # of an SM, of each CTA beside its own, most of a CTA; columns


def cta(n, m, k, rows):
    out = (ctypes.c_int * 3)()
    assert ops.lib().jb_linear_mx4_cta(n, m, k, rows, ctypes.addressof(out)) == 0
    return tuple(out)


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("n", [1, 16, 17, 32, 33, 64, 65, 77, 128])
def test_columns_are_no_scarcer_than_shared_memory(n, rows):
    seen = set()
    for m in (1, 128, 130, 300, 640, 1280, 2560, 6144, 19456):
        for k in (1, 256, 257, 512, 513, 768, 1024, 1536, 2048, 2560, 3001, 4096, 9728, 30000):
            clustered, smem, cols = cta(n, m, k, rows)
            assert cols in (64, 128, 256) and 0 < smem <= MOST
            if clustered > 1:
                # columns for each CTA's share of the shared memory: then the sum over any CTAs that fit is at most COLS
                assert cols * SMEM <= COLS * (smem + OWN), (m, k, clustered, smem, cols)
                seen.add((smem, cols))
    assert seen


def test_a_pair_has_the_sm_to_itself():
    clustered, smem, cols = cta(129, 2560, 2560, 0)
    assert clustered == 2 and cols == COLS
    least = min(cta(n, m, k, 0)[1] for n in (1, 32, 64, 128) for m in (128, 1280) for k in (512, 2560))
    assert smem + least + 2 * OWN > SMEM


def test_sizes_that_are_refused():
    out = (ctypes.c_int * 3)()
    for n, m, k in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (0x7fffffff, 1, 1), (1, 0x7fffffff, 1), (1, 1, 0x7fffffff)):
        assert ops.lib().jb_linear_mx4_cta(n, m, k, 0, ctypes.addressof(out)) == -1
