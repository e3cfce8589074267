"""Argument checks of the class-score operators beyond tests/test_class_scores_host.py: single rows whose result has the other layout, strides
no memory has, results that lie across what a call reads."""
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
