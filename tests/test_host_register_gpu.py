"""ddt_host_register on the device: what Engine.host_register answers is what the feeder then does, and bad ranges are refused."""
import mmap

import numpy as np
import pytest

import ddt
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def test_registered_or_staged(capsys):
    T, D, F, n = 40, 8, 32, 100_003
    m, x = O.gen_model(T, D, F, dist=1), O.gen_tuples(5, n, F, dist=1)
    e = ddt.Engine(0)
    e.load_model(ddt.make_params(T, D, F), m.wlines, m.flines)
    e.set_option("feeder_rows", 16_384)
    want, out = e.score(x), np.full(n, np.nan, np.float32)
    pinned = [e.host_register(x), e.host_register(out)]
    assert pinned[0] == pinned[1] == e.host_pinned(x) == e.host_pinned(out[3:])
    with capsys.disabled():
        print(f"[host buffers: {'pinned' if pinned[0] else 'staged'}]", end=" ")
    assert np.array_equal(e.score(x, out=out).view(np.uint32), want.view(np.uint32))
    e.host_unregister(x)
    e.host_unregister(out)
    assert not e.host_pinned(x) and not e.host_pinned(out)
    e.close()


def test_a_hole_is_no_range():
    e, page = ddt.Engine(0), mmap.PAGESIZE
    a = np.zeros(64, np.float32)
    for ptr, size in ((16, 64), (a.ctypes.data, 2 ** 63), (a.ctypes.data, 2 ** 64 - page)):
        assert e._L.ddt_host_register(e._h, ptr, size) == -1
    e.close()
