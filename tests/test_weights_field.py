"""Where a caller of the C interface says that weights go to 4 bits: a field behind those of jb_llm_params, whose reserved
word stays unread and whose defaults are written into no more than its own bytes.  Structs are laid out here by hand."""
import ctypes

import pytest

OK, EINVAL, EOPEN = 0, -1, -3
P = ctypes.c_void_p
PLAIN = [("size", ctypes.c_uint32), ("n_ctx", ctypes.c_uint32), ("max_batch", ctypes.c_uint32), ("dtype", ctypes.c_int32),
           ("device", ctypes.c_int32), ("reserved", ctypes.c_uint32), ("max_tokens", ctypes.c_uint64)]


class Plain(ctypes.Structure):
    _fields_ = PLAIN


class WithWeights(ctypes.Structure):
    _fields_ = PLAIN + [("weights", ctypes.c_int32), ("reserved2", ctypes.c_uint32)]


@pytest.fixture(scope="module")
def L():
    from janas_b200.csrc import build
    lib = ctypes.CDLL(build.library_path())
    lib.jb_llm_last_error.restype = ctypes.c_char_p
    lib.jb_llm_open.argtypes = [ctypes.c_char_p, P, ctypes.POINTER(P)]
    lib.jb_llm_open_random.argtypes = [ctypes.c_char_p, ctypes.c_uint64, P, ctypes.POINTER(P)]
    return lib


def opened(L, p, folder):
    return L.jb_llm_open(str(folder).encode(), ctypes.byref(p), ctypes.byref(P()))


def test_the_reserved_word_is_not_read(L, tmp_path):
    """What a caller left there is neither a choice of weights nor refused: it is the folder that is missing."""
    for dtype in (0, 1):
        for word in (0, 1, 2, 0xffffffff):
            old = Plain(ctypes.sizeof(Plain), 128, 2, dtype, 0, word, 0)
            assert opened(L, old, tmp_path / "nothing") == EOPEN, L.jb_llm_last_error()
            new = WithWeights(ctypes.sizeof(WithWeights), 128, 2, dtype, 0, word, 0, 0, word)
            assert opened(L, new, tmp_path / "nothing") == EOPEN, L.jb_llm_last_error()


def test_weights_are_read_where_the_struct_has_them(L, tmp_path):
    p = WithWeights()
    L.jb_llm_weight_params_default(ctypes.byref(p))
    assert (p.n_ctx, p.max_batch, p.dtype, p.device, p.max_tokens) == (16384, 64, 0, 0, 0)
    assert p.size == ctypes.sizeof(WithWeights) and p.weights == 0
    p.weights = 1
    assert opened(L, p, tmp_path / "nothing") == EOPEN
    p.weights = 2
    assert opened(L, p, tmp_path / "nothing") == EINVAL and b"weights" in L.jb_llm_last_error()
    p.weights, p.dtype = 1, 1
    assert opened(L, p, tmp_path / "nothing") == EINVAL and b"BF16" in L.jb_llm_last_error()
    p.size = ctypes.sizeof(Plain)         # the field lies behind this struct's end
    assert opened(L, p, tmp_path / "nothing") == EOPEN


def test_defaults_end_with_the_struct(L):
    p = WithWeights(weights=7, reserved2=9)
    L.jb_llm_params_default(ctypes.byref(p))
    assert p.size == ctypes.sizeof(Plain) and (p.weights, p.reserved2) == (7, 9)


def test_the_packages_struct_is_the_headers():
    from janas_b200 import lib
    assert [(n, ctypes.sizeof(t)) for n, t in lib.Params._fields_] == [(n, ctypes.sizeof(t)) for n, t in WithWeights._fields_]
