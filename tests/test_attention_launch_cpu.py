"""The host side of csrc/mha.hip without a GPU: sizes that a launch cannot hold are refused before anything is started."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


class MhaArgs(ctypes.Structure):  # csrc/mha.h
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv", "delta", "part", "lens")]
                + [(n, ctypes.c_long * 3) for n in ("qs", "ks", "vs", "os", "dos", "dqs", "dks", "dvs")]
                + [(n, ctypes.c_int) for n in ("B", "Tq", "Tk", "H", "Hkv", "G", "D", "causal")]
                + [("scale", ctypes.c_float), ("gmul", ctypes.c_uint), ("gshift", ctypes.c_uint)]
                + [(n, ctypes.c_int) for n in ("splits", "split_tiles", "dq_splits", "dq_split_tiles", "kv_splits")])


def _lib():
    from masters_thesis_amd.ops import build
    from masters_thesis_amd.ops._lib import lib

    lib()
    so = ctypes.CDLL(str(build.ext_path()))
    so.mta_mha_plan.restype = ctypes.c_long
    so.mta_mha.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    so.mta_mha_plan.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    so.mta_rope.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_long, ctypes.c_int, ctypes.c_long, ctypes.c_int, ctypes.c_int,
                            ctypes.c_double, ctypes.c_int, ctypes.c_void_p]
    return so


@pytest.mark.skipif(torch.cuda.is_available(), reason="host checks: a launch would run")
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("b,tq,tk,causal", [(2 ** 24, 1, 1, 0), (2 ** 24 + 5, 3, 9, 1), (2 ** 20, 2 ** 11 + 1, 4, 0), (2 ** 30, 1, 1, 0)])
def test_more_threads_than_a_launch_holds(dtype, backward, b, tq, tk, causal):
    """256 threads to at most 128 rows of a sequence; a launch holds 2^32 - 1."""
    so = _lib()
    A = MhaArgs(B=b, Tq=tq, Tk=tk, H=1, Hkv=1, G=1, D=8, causal=causal, scale=1.0)
    assert so.mta_mha_plan(dtype, backward, ctypes.byref(A)) == 0
    assert so.mta_mha(dtype, backward, ctypes.byref(A), None) == 2


@pytest.mark.skipif(torch.cuda.is_available(), reason="host checks: a launch would run")
def test_rope_of_more_pairs_than_a_launch_holds():
    so = _lib()
    for dtype in (0, 2):
        assert so.mta_rope(dtype, None, 2 ** 31, 7, 4, 1, 4, 10000.0, 0, None) == 2
