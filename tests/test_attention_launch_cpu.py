"""The host side of csrc/mha.hip without a GPU: sizes that a launch cannot hold are refused before anything is started, and tensors that
share memory are found."""
import ctypes
import random

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

    if not build.ext_path().exists():
        build.build()
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


class Box(ctypes.Structure):  # csrc/mha.h MhaBox
    _fields_ = [("at", ctypes.c_long), ("strides", ctypes.c_long * 4), ("sizes", ctypes.c_long * 4)]


def _places(at, strides, sizes):
    x = torch.tensor([at])
    for s, n in zip(strides, sizes):
        x = (x[:, None] + s * torch.arange(n)).view(-1)
    return set(x.tolist())


def test_tensors_with_an_element_in_common():
    """Every answer against the sets of places: views of packed buffers, of other orders and sizes, nested or not."""
    so = _lib()
    g = random.Random(0)
    seen = {True: 0, False: 0}
    for trial in range(3000):
        b, t, h, d = g.randint(1, 3), g.randint(1, 5), g.randint(1, 7), g.choice([1, 2, 4])
        heads = h + g.randint(0, 6)
        orders = [(t * heads * d, heads * d, d, 1), (heads * t * d, d, t * d, 1), (heads * d, b * heads * d, d, 1)]
        one = g.randrange(3)
        boxes = []
        for _ in range(2):
            order = orders[one if g.random() < 0.8 else g.randrange(3)]
            n = (g.randint(0 if trial % 50 == 0 else 1, b), g.randint(1, t), g.randint(1, h), d)
            boxes.append((g.randint(0, heads * d), order, n))
        if trial % 7 == 0:  # strides that do not lie within each other
            boxes[0] = (g.randint(0, 20), tuple(g.randint(0, 9) for _ in range(4)), boxes[0][2])
        common = bool(_places(*boxes[0]) & _places(*boxes[1]))
        made = [Box(at, (ctypes.c_long * 4)(*s), (ctypes.c_long * 4)(*n)) for at, s, n in boxes]
        assert so.mta_mha_meet(ctypes.byref(made[0]), ctypes.byref(made[1])) == common, boxes
        seen[common] += 1
    assert min(seen.values()) > 500


def test_packed_gradients_of_long_calls():
    """q, k and v beside each other do not meet, a head later they do; at sizes whose places are not listed."""
    so = _lib()

    def box(at, n, t=1 << 20, b=1 << 12, heads=48, d=128):
        return Box(at * d, (ctypes.c_long * 4)(t * heads * d, heads * d, d, 1), (ctypes.c_long * 4)(b, t, n, d))

    q, k, v = box(0, 32), box(32, 8), box(40, 8)
    for x, y, common in ((q, k, 0), (k, v, 0), (q, v, 0), (q, box(31, 8), 1), (k, box(39, 8), 1), (q, box(48, 8), 1), (q, box(48 * 5 + 32, 8), 0)):
        assert so.mta_mha_meet(ctypes.byref(x), ctypes.byref(y)) == common
