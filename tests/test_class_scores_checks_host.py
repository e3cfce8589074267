"""Argument checks of the class-score operators beyond tests/test_class_scores_host.py: single rows whose result has the other layout, strides
that no memory has, results at the ends of the matrix they are computed from."""
import ctypes as C

import pytest

from ddt import _lib
from tests.test_class_scores_host import EINVAL, P, adjust, engine, lib, scores, teacher, top  # noqa: F401


def note(lib):  # noqa: F811
    return tuple(lib.mock_note(i) for i in range(3))


def test_a_single_row_takes_the_layout_of_its_result(lib, engine):  # noqa: F811
    A, to = _lib.Adjust, P + 8192
    for i, o, want in ((scores(1, 10, 1, 1), scores(1, 10, 1, 4, to), (1, 1, 4)),       # contiguous -> every fourth element
                       (scores(1, 10, 1, 4), scores(1, 10, 1, 1, to), (1, 4, 1)),       # and back
                       (scores(1, 10, 77, 1), scores(1, 10, 3, 1, to), (0, 10, 10)),
                       (scores(1, 10, 1, 4), scores(1, 10, 1, 7, to), (1, 4, 7)),
                       (scores(5, 1, 1, 77), scores(5, 1, 3, 1, to), (0, 1, 3)),        # one class: rows three apart
                       (scores(5, 1, 3, 1), scores(5, 1, 1, 1, to), (0, 3, 1))):
        assert adjust(lib, engine, i, A(), o) == 0 and note(lib) == want, (want, note(lib))
    assert lib.mock_error(engine) == b""                                                # and nothing was said on the way
    before = lib.mock_launches()
    for o in (scores(1, 10, 1, 0, to), scores(1, 10, 1, 4, P + 16), scores(1, 11, 1, 4, to), scores(1, 10, 1, 4, to, 1)):
        assert adjust(lib, engine, scores(1, 10, 1, 1), A(), o) == EINVAL and lib.mock_error(engine)
    assert lib.mock_launches() == before


@pytest.mark.parametrize("stride", [2 ** 49, 2 ** 60, 2 ** 64 - 1])
def test_strides_that_no_memory_has(lib, engine, stride):  # noqa: F811
    s, before, A = scores(5, 10, 10, 1), lib.mock_launches(), _lib.Adjust
    t = teacher(stride=stride)
    assert lib.ddt_distill_device(engine, C.byref(s), C.byref(t), P, None) == EINVAL
    assert lib.ddt_distill_grad_device(engine, C.byref(s), C.byref(t), None, 0, P, C.byref(s), None) == EINVAL
    assert lib.ddt_distill_grad_device(engine, C.byref(s), C.byref(teacher()), P, stride, P, C.byref(s), None) == EINVAL
    for a in (A(bias=P, bias_row_stride=stride), A(bias=P, bias_class_stride=stride), A(allowed=P, allowed_row_stride=stride),
              A(history=P, history_first=P, history_len=stride)):
        assert adjust(lib, engine, s, a, s) == EINVAL
    for bad in (scores(5, 10, stride, 1), scores(5, 10, 1, stride), scores(stride, 10, 10, 1)):
        assert top(lib, engine, bad) == EINVAL
    assert lib.mock_launches() == before
    assert lib.ddt_distill_grad_device(engine, C.byref(scores(1, 10, 10, 1)), C.byref(t), None, stride, P, C.byref(scores(1, 10, 10, 1)), None) == 0


def test_results_at_the_ends_of_the_scores(lib, engine):  # noqa: F811
    """In place, right in front of the matrix and right behind it; not across it."""
    size = (4 * 12 + 10) * 4                                                           # five rows of 10, 12 apart
    s, A = scores(5, 10, 12, 1, P + 4096), _lib.Adjust
    for at, stride, want in ((0, 12, 0), (size, 12, 0), (-size, 12, 0), (size, 10, 0), (-200, 10, 0), (size - 4, 12, EINVAL), (4 - size, 12, EINVAL),
                             (0, 13, EINVAL), (0, 10, EINVAL), (40, 12, EINVAL)):
        o = scores(5, 10, stride, 1, P + 4096 + at)
        assert adjust(lib, engine, s, A(), o) == want, (at, stride)
        assert lib.ddt_distill_grad_device(engine, C.byref(s), C.byref(teacher()), None, 0, P, C.byref(o), None) == want, (at, stride)
