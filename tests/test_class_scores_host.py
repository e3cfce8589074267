"""Argument checks of the class-score operators (csrc/ddt_classes.cpp), built unchanged against the CPU model of the host side: what is
refused, with which code, and that nothing is launched then; which layout and strides the kernels are handed for what is accepted."""
import ctypes as C
import os

import pytest

from ddt import _lib
from tests.mock_hip.build_lock import build_if_stale

HERE = os.path.dirname(os.path.abspath(__file__))
MOCK = os.path.join(HERE, "mock_hip")
CSRC = os.path.join(os.path.dirname(HERE), "distributed-decisiontrees_amd", "csrc")
EINVAL, EUNSUPPORTED = -1, -5


@pytest.fixture(scope="module")
def lib():
    out = os.path.join(MOCK, "libddt_classes_mock.so")
    srcs = [os.path.join(CSRC, "ddt_classes.cpp"), os.path.join(MOCK, "mock_classes.cpp")]
    deps = srcs + [os.path.join(MOCK, f) for f in ("mock_engine.cpp", "mock_runtime.cpp", "hip/hip_runtime.h", "rccl/rccl.h")] + \
        [os.path.join(CSRC, f) for f in ("ddt_classes.h", "ddt_engine_priv.h", "ddt_internal.h")] + \
        [os.path.join(os.path.dirname(HERE), "include", "ddt.h")]
    build_if_stale(out, deps, ["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-pthread", "-w", "-I" + MOCK, "-I" + CSRC, *srcs])
    L = _lib.bind_class_scores(C.CDLL(out))
    L.mock_note.restype, L.mock_error.restype, L.mock_error.argtypes = C.c_ulonglong, C.c_char_p, [C.c_void_p]
    return L


@pytest.fixture()
def engine(lib):
    h = C.c_void_p()
    assert lib.ddt_create(C.byref(h), 0) == 0
    yield h
    lib.ddt_destroy(h)


BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(BUF) + 63) // 64 * 64


def scores(n, K, rs, cs, data=P, dtype=0):
    return _lib.Scores(data, n, rs, cs, K, dtype)


def teacher(k=4, stride=4, T=1.0, ids=P, values=P, lse=None):
    return _lib.Teacher(ids, values, stride, lse, k, T)


def adjust(lib, e, i, a, o):
    return lib.ddt_adjust_scores_device(e, C.byref(i), C.byref(a), C.byref(o), None)


def top(lib, e, s, k=3, T=1.0, ids=P, values=P, lse=P):
    return lib.ddt_top_scores_device(e, C.byref(s), k, T, ids, values, lse, None)


BAD = {"overlapping rows": (5, 10, 9, 1), "overlapping classes": (5, 10, 1, 4), "no unit stride": (5, 10, 20, 2), "no class": (5, 0, 1, 1),
       "too many classes": (1, (1 << 20) + 1, 1 << 21, 1), "huge stride": (5, 10, 1 << 60, 1), "broadcast rows": (5, 10, 0, 1),
       "broadcast classes": (5, 10, 1, 0), "huge rows": (1 << 60, 1, 1, 1)}


@pytest.mark.parametrize("name", BAD)
def test_matrices_that_are_refused(lib, engine, name):
    s, before = scores(*BAD[name]), lib.mock_launches()
    assert top(lib, engine, s) == EINVAL and lib.mock_error(engine)
    assert adjust(lib, engine, s, _lib.Adjust(), s) == EINVAL
    assert lib.ddt_distill_device(engine, C.byref(s), C.byref(teacher()), P, None) == EINVAL
    assert lib.mock_launches() == before


def test_null_and_misaligned_arguments(lib, engine):
    before, ok = lib.mock_launches(), scores(5, 10, 10, 1)
    for bad in (scores(5, 10, 10, 1, None), scores(5, 10, 10, 1, P + 2), scores(5, 10, 10, 1, P + 1, 2), scores(5, 10, 10, 1, P, 3)):
        assert top(lib, engine, bad) == EINVAL
        assert adjust(lib, engine, ok, _lib.Adjust(), bad) == EINVAL
        assert lib.ddt_distill_grad_device(engine, C.byref(ok), C.byref(teacher()), None, 0, P, C.byref(bad), None) == EINVAL
    assert lib.ddt_top_scores_device(None, C.byref(ok), 3, 1.0, P, P, P, None) == EINVAL
    assert lib.ddt_top_scores_device(engine, None, 3, 1.0, P, P, P, None) == EINVAL
    assert lib.ddt_adjust_scores_device(engine, C.byref(ok), None, C.byref(ok), None) == EINVAL
    assert lib.ddt_adjust_scores_device(engine, C.byref(ok), C.byref(_lib.Adjust()), None, None) == EINVAL
    assert lib.ddt_distill_device(engine, C.byref(ok), None, P, None) == EINVAL
    assert lib.ddt_distill_grad_device(engine, C.byref(ok), C.byref(teacher()), None, 0, P, None, None) == EINVAL
    assert top(lib, engine, ok, ids=None) == EINVAL and top(lib, engine, ok, values=None) == EINVAL
    assert lib.ddt_distill_device(engine, C.byref(ok), C.byref(teacher()), None, None) == EINVAL
    assert lib.mock_launches() == before
    assert top(lib, engine, ok, lse=None) == 0 and lib.mock_launches() == before + 1   # the log-sum-exp may stay out


@pytest.mark.parametrize("k,T", [(0, 1.0), (257, 1.0), (3, 0.0), (3, -1.0), (3, float("nan")), (3, float("inf")), (3, 1e-4), (3, 1e4)])
def test_k_and_temperature(lib, engine, k, T):
    before, s = lib.mock_launches(), scores(5, 1000, 1000, 1)
    assert top(lib, engine, s, k, T) == EINVAL
    assert lib.ddt_distill_device(engine, C.byref(s), C.byref(teacher(k, 300, T)), P, None) == EINVAL
    assert lib.mock_launches() == before


def test_teacher(lib, engine):
    before, s = lib.mock_launches(), scores(5, 10, 10, 1)
    for t in (teacher(4, 3), teacher(ids=None), teacher(values=None)):
        assert lib.ddt_distill_device(engine, C.byref(s), C.byref(t), P, None) == EINVAL
    assert lib.ddt_distill_device(engine, C.byref(scores(5, 10, 1, 5)), C.byref(teacher()), P, None) == EINVAL      # class-major student
    assert lib.mock_launches() == before


def test_adjustments(lib, engine):
    before, s = lib.mock_launches(), scores(5, 70, 70, 1)
    A = _lib.Adjust
    for a in (A(allowed=P, allowed_row_stride=2), A(history_len=3), A(history=P, history_len=3), A(bias=P, bias_row_stride=1 << 60)):
        assert adjust(lib, engine, s, a, s) == EINVAL
    for o in (scores(5, 71, 71, 1, P + 8192), scores(4, 70, 70, 1, P + 8192), scores(5, 70, 70, 1, P + 8192, 1), scores(5, 70, 1, 5, P + 8192),
              scores(5, 70, 70, 1, P + 4), scores(5, 70, 71, 1, P)):
        assert adjust(lib, engine, s, A(), o) == EINVAL, (o.data - P, o.row_stride)
    assert lib.mock_launches() == before
    assert adjust(lib, engine, s, A(allowed=P, allowed_row_stride=3), s) == 0                                       # in place
    assert adjust(lib, engine, s, A(), scores(5, 70, 80, 1, P + 4 * 70 * 5)) == 0 and lib.mock_note(2) == 80          # right behind it
    assert adjust(lib, engine, s, A(history=P, history_first=P, history_len=0), s) == 0 and lib.mock_note(3) == 0    # an empty history is none


def test_layouts(lib, engine):
    def layout(s):
        assert top(lib, engine, s) == 0
        return lib.mock_note(0), lib.mock_note(1)

    assert layout(scores(5, 10, 10, 1)) == (0, 10) and layout(scores(5, 10, 16, 1)) == (0, 16)
    assert layout(scores(5, 10, 1, 5)) == (1, 5) and layout(scores(5, 10, 1, 8)) == (1, 8)
    assert layout(scores(1, 10, 77, 1)) == (0, 10)                                  # one row: its stride means nothing
    assert layout(scores(1, 10, 77, 8)) == (1, 8)                                   # one row out of a class-major matrix
    assert layout(scores(5, 1, 1, 77)) == (0, 1) and layout(scores(5, 1, 3, 77)) == (0, 3)
    s, o = scores(1, 10, 1, 1), scores(1, 10, 1, 4, P + 8192)                        # one row may change its layout with the result
    assert adjust(lib, engine, s, _lib.Adjust(), o) in (0, EINVAL)
    assert top(lib, engine, scores(5, 2048, 1, 5)) == 0
    assert top(lib, engine, scores(5, 2049, 1, 5)) == EUNSUPPORTED and top(lib, engine, scores(5, 2049, 2049, 1)) == 0


def test_no_rows_is_no_work(lib, engine):
    before, s = lib.mock_launches(), scores(0, 10, 10, 1, None)
    assert top(lib, engine, s, ids=None, values=None, lse=None) == 0 and adjust(lib, engine, s, _lib.Adjust(), s) == 0
    t = teacher(ids=None, values=None)
    assert lib.ddt_distill_device(engine, C.byref(s), C.byref(t), None, None) == 0
    assert lib.ddt_distill_grad_device(engine, C.byref(s), C.byref(t), None, 0, None, C.byref(s), None) == 0
    assert lib.mock_launches() == before


def test_gradient_buffers(lib, engine):
    s, t = scores(5, 10, 10, 1), teacher()

    def grad(g, loss=P + 32768, stride=0):
        return lib.ddt_distill_grad_device(engine, C.byref(s), C.byref(t), P, stride, loss, C.byref(g), None)

    assert grad(s) == 0 and grad(scores(5, 10, 12, 1, P + 4096), None, 1) == 0 and (lib.mock_note(2), lib.mock_note(3)) == (12, 1)
    assert grad(scores(5, 10, 1, 5, P + 4096)) == EINVAL and grad(scores(5, 10, 10, 1, P + 4)) == EINVAL
    assert grad(scores(5, 10, 10, 1, P + 4096, 1)) == EINVAL
