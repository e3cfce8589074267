"""Every launch rule of the class-score operators on both of its sides, against the 64-bit forms and tolerances of
tests/test_class_scores_gpu.py: sizes just past each threshold, with rows that do not end on a whole pack.  Together the two files launch each
of the library's 244 kernels of these operators (a profiler's count)."""
import math

import numpy as np
import pytest

import ddt
from tests.test_class_scores_gpu import (HARD, TYPES, U, adjust_inputs, check_adjust, check_distill, check_top, close, distill64, matrix, rng,
                                        teacher_of)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


# tiles of 512 packs (2^17 packs and more), of several rows or a part of one; of 1024 packs (more than 6000 entries of history a row); fewer
# rows than waves, more rows than waves; class-major: several tiles of classes and of rows
@pytest.mark.parametrize("layout", ["rows", "rows_gap", "classes_gap"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,history", [(300, 5003, 200), (300, 5003, 0), (5000, 301, 20), (5000, 301, 0), (27_000, 33, 3), (2, 8193, 20_000),
                                         (1, 8193, 6001), (1, 8193, 6000), (2, 101, 20_000), (40, 1003, 20_000), (1100, 17, 5)])
def test_adjust(engine, n, K, history, dtype, layout):
    kw = adjust_inputs(n, K, 5, history, ["rows", "shared", "none"][K % 3], ["shared", "rows", "columns"][n % 3])
    check_adjust(engine, matrix(n, K, dtype, layout), kw)


# one thread per row with 1 .. 8 of the classes; 16 lanes per row with 1 .. 8 packs and where their limit of work is passed; a wave per row
# with 1 .. 8 packs; blocks of 256, 512 and 1024 threads
@pytest.mark.parametrize("layout", ["rows", "classes", "rows_gap", "classes_gap"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,k", [(517, 11, k) for k in range(1, 9)] + [(300, 32, 5), (300, 33, 5), (65536, 33, 4), (65535, 33, 4), (65536, 65, 4), (4096, 64, 16),
                                   (4097, 100, 7), (4097, 130, 3), (4095, 130, 3), (4100, 260, 3), (4100, 500, 12), (4100, 500, 13), (4100, 513, 3),
                                   (4100, 60, 16), (4100, 60, 17), (30, 257, 64), (30, 400, 65), (9, 1030, 33), (5, 2048, 128)])
def test_top_of_short_rows(engine, n, K, k, dtype, layout):
    check_top(engine, matrix(n, K, dtype, layout), k, [1.0, 2.0, 0.5][(n + k) % 3])


@pytest.mark.parametrize("layout", ["rows", "rows_gap"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,k", [(257, 16384, 32), (257, 16384, 33), (256, 16411, 128), (257, 16411, 50), (257, 16411, 65), (300, 50257, 64), (257, 70001, 256)])
def test_top_of_long_rows(engine, n, K, k, dtype, layout):
    check_top(engine, matrix(n, K, dtype, layout), k, 2.0)


def test_top_of_groups_of_chunks(engine):
    """More than 16 chunks of 512 threads' packs: a group holds several."""
    check_top(engine, matrix(257, 140_003, "fp32"), 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,k", [(16390, 64), (20003, 256)])
@pytest.mark.parametrize("kind", HARD)
def test_top_of_many_long_rows_that_tie_or_hold_nothing(engine, kind, K, k, dtype):
    n = 258
    x = matrix(n, K, dtype)
    c = torch.arange(K, device="cuda", dtype=torch.float32)
    if kind == "constant":
        x.fill_(-2.5)
    elif kind in ("ascending", "descending"):
        x.copy_(((c / K * 8 - 4) * (1 if kind == "ascending" else -1))[:, None].expand(K, n))
    elif kind == "two values":
        x.copy_(((c * 7919) % 3 == 0).float()[:, None].expand(K, n))
    elif kind == "lowest":
        x[torch.rand(K, n, device="cuda") < 0.5] = torch.finfo(TYPES[dtype]).min
        x[:, 1] = torch.finfo(TYPES[dtype]).min
    elif kind == "one allowed":
        x.fill_(-math.inf)
        x[K // 2] = -3.0
    elif kind == "nothing allowed":
        x[:, 1] = -math.inf
    elif kind == "few allowed":
        keep = x[::K // 3].clone()
        x.fill_(-math.inf)
        x[::K // 3] = keep
    elif kind == "nan":
        x[K // 3, 0] = math.nan
        x[:, 1] = math.nan
    elif kind == "inf":
        x[K // 3, 0] = math.inf
        x[0, 1] = math.inf
        x[K - 1, 1] = math.inf
    elif kind == "zeros":
        x.copy_(torch.where(c % 2 == 0, 0.0, -0.0)[:, None].expand(K, n))
    elif kind == "one thread":
        x.copy_(torch.where((c // 8) % 512 == 5, 9.0 + c / K, -1.0)[:, None].expand(K, n))
    check_top(engine, x, k, 0.5)


def check_apart(engine, x, ids, vals, lse, T, w):
    """check_distill where loss alone and loss with gradient run different kernels, whose sums take the row's packs in different orders: each
    is held to the 64-bit loss, not to the other"""
    want, grad, size = distill64(x.double().cpu().numpy(), ids, vals, lse, T, w.astype(np.float64))
    args = [None if a is None else torch.from_numpy(a).cuda() for a in (ids, vals, lse)]
    loss, g = engine.distill_grad_device(x, *args, row_weight=torch.from_numpy(w).cuda(), temperature=T)
    fi = torch.finfo(x.dtype)
    for got in (engine.distill_device(x, *args, temperature=T), loss):
        close(got.double().cpu(), want, 200 * U + U * np.abs(want))
    close(g.double().cpu(), grad, size + (fi.eps / 2) * (np.abs(grad) + size) + fi.smallest_normal * fi.eps / 2 + 2.0 ** -126)


# a thread per row with 1 .. 5 entries in registers and more of them; 16 lanes per row with 1 .. 16 packs; a wave with 1 .. 8; a block of 256
# with 4 packs a thread, reading twice, with 16 packs; of 512 and of 1024, reading twice
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,k", [(517, 11, k) for k in range(1, 8)] + [(300, 32, 6), (4096, 33, 2), (4095, 33, 2), (4100, 100, 5), (4100, 400, 5), (4100, 1030, 5),
                                   (4096, 1500, 64), (4096, 1030, 65), (513, 2049, 9), (513, 4095, 30), (513, 4100, 7), (512, 4100, 7), (513, 8195, 8), (513, 11_999, 3),
                                   (513, 12_001, 64)])
def test_distill(engine, n, K, k, dtype, rest):
    T = [1.0, 2.0, 0.5][(n + K + k) % 3]
    x = matrix(n, K, dtype, "rows_gap" if k % 2 else "rows").t()
    ids, vals, lse = teacher_of(n, K, k, T)
    (check_apart if n == 513 else check_distill)(engine, x, ids, vals, lse if rest else None, T, (0.5 + rng(n, K).random(n)).astype(np.float32))


@pytest.mark.parametrize("n,K,dtype", [(513, 16_001, "fp32"), (513, 16_387, "fp32"), (513, 65_537, "fp32"), (512, 65_537, "fp32"), (513, 23_999, "bf16"), (513, 24_003, "fp16"),
                                       (513, 32_001, "bf16"), (513, 32_001, "fp16"), (513, 32_771, "bf16"), (513, 131_075, "bf16")])
def test_distill_of_long_rows(engine, n, K, dtype):
    x = matrix(n, K, dtype, "rows_gap").t()
    ids, vals, lse = teacher_of(n, K, 60, 2.0)
    check_apart(engine, x, ids, vals, lse, 2.0, (0.5 + rng(n, K).random(n)).astype(np.float32))
    loss, want = engine.distill_grad_device(x, *(torch.from_numpy(a).cuda() for a in (ids, vals, lse)), temperature=2.0)
    again, got = engine.distill_grad_device(x, *(torch.from_numpy(a).cuda() for a in (ids, vals, lse)), temperature=2.0, grad=x)
    assert got is x and torch.equal(again, loss) and torch.equal(got, want)
