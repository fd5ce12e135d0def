"""Products and matrices in 4 bits at the ends of 32-bit counts, and values that are no matrix in 4 bits: refused, by the C
entries and by the Python ones, before anything is allocated or launched."""
import pytest

from janas_b200.csrc import ops

LAST = 0x7fffffff
EINVAL = -1


class NoMemory:
    """Stands for a tensor whose device would have to give memory."""

    def new_empty(self, *args, **kwargs):
        raise AssertionError("allocated")


def test_c_entries_refuse_the_last_sizes():
    """Padding a size to whole blocks, chunks or tiles (up to 256) must not pass 2^31 - 1."""
    L = ops.lib()
    assert L.jb_mx4_code_bytes(1, LAST) == 0 and L.jb_mx4_scale_bytes(1, LAST) == 0
    assert L.jb_mx4_code_bytes(LAST, 1) == 0 and L.jb_mx4_scale_bytes(LAST, 1) == 0
    for n, m, k in ((LAST, 1, 32), (1, LAST, 32), (1, 1, LAST)):
        assert L.jb_linear_mx4_scratch(n, m, k, 1) == 0 and L.jb_linear_mx4_launches(n, m, k, 1) == 0
    for n, k in ((0, LAST), (LAST, 32)):
        assert L.jb_mx4_quantize(None, 0, None, None, n, k, 0, None) == EINVAL
        assert L.jb_mx4_values(None, None, None, 0, n, k, None) == EINVAL
    for n, m, k in ((0, LAST, 32), (LAST, 0, 32), (0, 0, LAST)):
        assert L.jb_linear_mx4(None, None, None, None, None, 0, n, m, k, None, 0, None) == EINVAL
        assert L.jb_linear_mx4_rows(None, 0, None, None, None, 0, n, m, k, None, 0, None) == EINVAL


def test_the_largest_sizes_that_are_taken():
    L = ops.lib()
    most = ops._MOST
    assert L.jb_mx4_code_bytes(1, most) == most // 32 * 16 and L.jb_mx4_scale_bytes(1, most) == most // 256 * 1024
    assert L.jb_mx4_code_bytes(most, 1) == most * 16 and L.jb_mx4_scale_bytes(most, 1) == most // 128 * 1024


@pytest.mark.parametrize("rows,k", [(2 ** 31, 32), (2 ** 32 + 1, 32), (1, 2 ** 31), (1, 2 ** 32 + 32), (LAST, 32), (1, LAST)])
def test_matrices_of_more_rows_or_values(rows, k):
    with pytest.raises(ops.KernelError):
        ops.Mx4._new(rows, k, NoMemory(), False)


def test_values_of_something_else():
    for q in (None, 3, NoMemory()):
        with pytest.raises(ops.KernelError):
            ops.mx4_values(q)


@pytest.mark.gpu
def test_rows_past_32_bits():
    """More rows than the kernels count: 2^31 of one value."""
    import torch
    dev = "cuda:0"
    many = torch.empty((2 ** 31, 1), dtype=torch.bfloat16, device=dev)
    w = ops.mx4_quantize(torch.ones((2, 1), device=dev))
    before = torch.cuda.memory_allocated()
    for call in (lambda: ops.mx4_quantize(many), lambda: ops.linear_mx4(many, w)):
        with pytest.raises(ops.KernelError):
            call()
    assert torch.cuda.memory_allocated() == before
    del many
    x = torch.empty((2 ** 31, 1), device=dev)
    with pytest.raises(ops.KernelError):
        ops.norm_residual_norm(x, x, None, None, 1e-5)
