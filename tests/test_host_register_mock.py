"""ddt_host_register against the CPU model of the HIP runtime, whose hipHostRegister answers what a test sets: which failures leave the range
to be staged, which are reported, and what ddt_host_pinned says of each."""
import ctypes as C
import mmap

import numpy as np
import pytest

import ddt
from oracle import oracle as O
from tests.test_engine_mock import _bits, _engine, _load, mock  # noqa: F401

EINVAL, EHIP = -1, -3
OK, INVALID_VALUE, NO_MEMORY, REGISTERED, NOT_SUPPORTED = 0, 1, 2, 712, 801


@pytest.fixture()
def lib(mock):  # noqa: F811
    mock.mock_reset(0, 0, 8)
    yield mock
    mock.mock_pin_result(OK)


def register(lib, e, a):
    return lib.ddt_host_register(e, a.ctypes.data, a.nbytes)


@pytest.mark.parametrize("answer", [OK, INVALID_VALUE, NOT_SUPPORTED])
def test_register_score_unregister(lib, answer):
    T, D, F, n = 40, 8, 32, 2003
    m, x = O.gen_model(T, D, F, 1), O.gen_tuples(0, n, F, 1)
    e = _engine(lib)
    _load(lib, e, m, ddt.make_params(T, D, F), "q16_d8_c8_u4_gl_s2")
    assert lib.ddt_set_option(e, b"feeder_rows", 600) == 0
    out = np.full(n, np.nan, np.float32)
    lib.mock_pin_result(answer)
    assert register(lib, e, x) == 0 and register(lib, e, out) == 0
    assert register(lib, e, x) == EINVAL and b"already" in lib.ddt_last_error(e)       # twice, pinned or not
    pinned = int(answer == OK)
    for a in (x, out, x[5:9], out[7:]):
        assert lib.ddt_host_pinned(e, a.ctypes.data, a.nbytes) == pinned
    for size in (x.nbytes + 1, 2 ** 64 - 1, 2 ** 63):                                  # reaches past the range
        assert lib.ddt_host_pinned(e, x.ctypes.data + 4, size) == 0
    assert lib.ddt_score(e, x.ctypes.data, n, out.ctypes.data) == 0, lib.ddt_last_error(e)
    assert np.array_equal(_bits(out), _bits(O.score(m, x)))
    for a in (x, out):
        assert lib.ddt_host_unregister(e, a.ctypes.data) == 0 and lib.ddt_host_pinned(e, a.ctypes.data, a.nbytes) == 0
        assert lib.ddt_host_unregister(e, a.ctypes.data) == EINVAL
    assert register(lib, e, x) == 0                                                    # and once more
    lib.ddt_destroy(e)


@pytest.mark.parametrize("answer", [NO_MEMORY, REGISTERED, 999])
def test_failures_that_are_not_the_drivers_habit(lib, answer):
    e, x = _engine(lib), np.zeros(4096, np.float32)
    lib.mock_pin_result(answer)
    assert register(lib, e, x) == EHIP and b"hipHostRegister" in lib.ddt_last_error(e)
    assert lib.ddt_host_pinned(e, x.ctypes.data, x.nbytes) == 0 and lib.ddt_host_unregister(e, x.ctypes.data) == EINVAL
    lib.mock_pin_result(OK)
    assert register(lib, e, x) == 0 and lib.ddt_host_pinned(e, x.ctypes.data, x.nbytes) == 1
    lib.ddt_destroy(e)


@pytest.mark.parametrize("answer", [OK, INVALID_VALUE])
def test_ranges_that_are_no_memory(lib, answer):
    """A hole behind the array, a pointer into nowhere, a length that wraps: refused, whatever the driver would have said."""
    e, page = _engine(lib), mmap.PAGESIZE
    lib.mock_pin_result(answer)
    libc = C.CDLL(None, use_errno=True)
    libc.mmap.restype, libc.mmap.argtypes = C.c_void_p, [C.c_void_p, C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_long]
    libc.munmap.argtypes = [C.c_void_p, C.c_size_t]
    base = libc.mmap(None, 8 * page, mmap.PROT_READ | mmap.PROT_WRITE, mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS, -1, 0)
    assert libc.munmap(base + 4 * page, 4 * page) == 0
    for ptr, size in ((base, 4 * page + 1), (base + 4 * page, 16), (base + 100, 5 * page), (16, 16), (base, 2 ** 64 - 1), (base, 2 ** 63)):
        assert lib.ddt_host_register(e, ptr, size) == EINVAL, (ptr - base, size)
        assert lib.ddt_host_pinned(e, ptr, size) == 0 and lib.ddt_host_unregister(e, ptr) == EINVAL
    assert lib.ddt_host_register(e, base + 100, 4 * page - 100) == 0 and lib.ddt_host_unregister(e, base + 100) == 0
    assert lib.ddt_host_register(e, None, 16) == EINVAL and lib.ddt_host_register(e, base, 0) == EINVAL
    assert lib.ddt_host_register(None, base, 16) == EINVAL and lib.ddt_host_pinned(None, base, 16) == EINVAL
    libc.munmap(base, 4 * page)
    lib.ddt_destroy(e)
