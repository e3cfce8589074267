"""Distillation of rows whose student has no probability left for the classes that the teacher does not list (all of them at -inf): the
loss is infinite where the teacher's rest is not 0, and the rest is nothing where every class is listed.

Tolerances as for every loss and gradient of the class-score operators: 200 u + u |loss|; w / T (terms) (204 u + 3 u |log p| / ln 2) and one
rounding to the type (u = 2^-24)."""
import math

import numpy as np
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(7, 10, 3), (7, 20, 7), (7, 32, 40), (4100, 60, 5), (4100, 60, 64), (7, 90, 128), (12, 500, 9), (600, 5003, 4), (600, 14000, 4),
          (600, 40001, 4), (12, 50257, 256)]


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


def rows(n, K, k, dtype, seed=0):
    g = np.random.default_rng([7, n, K, k, seed])
    x = torch.from_numpy((g.standard_normal((n, K)) * 2.5).astype(np.float32)).to(dtype).cuda()
    kk = min(k, K // 2)                                        # some class is never listed
    ids = np.full((n, k), -1, np.int32)
    for r in range(n):
        ids[r, :kk] = g.permutation(K)[:kk]
    values = (g.standard_normal((n, k)) * 2 + 5).astype(np.float32)
    full = np.log(np.exp(values[:, :kk].astype(np.float64)).sum(1))
    return x, ids, values, kk, full


def only(x, ids, r):
    """row r keeps its listed classes, the others go to -inf"""
    keep = torch.zeros(x.shape[1], dtype=torch.bool, device="cuda")
    keep[torch.from_numpy(ids[r][ids[r] >= 0]).long().cuda()] = True
    x[r, ~keep] = -math.inf


def check_row(x, ids, values, lse, loss, grad, r, infinite):
    """loss and gradient of row r (T = 1) against 64 bits: the student's softmax stands on the listed classes alone"""
    on = ids[r] >= 0
    z = x[r].double().cpu().numpy()
    p = np.exp(z - z.max())
    p /= p.sum()
    log_q = values[r][on].astype(np.float64) - float(lse[r])
    q = np.exp(log_q)
    want = np.inf if infinite else (q * (log_q - np.log(p[ids[r][on]]))).sum()
    got = loss[r].item()
    assert got == want if infinite else abs(got - want) <= 200 * U + U * abs(want), (r, got, want)
    g = p * q.sum()
    np.subtract.at(g, ids[r][on], q)
    fi = torch.finfo(x.dtype)
    with np.errstate(divide="ignore"):
        size = p * q.sum() * (204 + 3 * np.abs(np.where(p > 0, np.log(p), 0)) * 1.45) * U
    tol = size + fi.eps / 2 * (np.abs(g) + size) + fi.smallest_normal * fi.eps / 2 + 2.0 ** -126
    off = np.abs(grad[r].double().cpu().numpy() - g)
    assert (off <= tol).all(), (r, np.argwhere(off > tol)[:3], off.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,K,k", SHAPES)
def test_no_probability_left_for_the_rest(engine, n, K, k, dtype):
    x, ids, values, kk, full = rows(n, K, k, dtype)
    lse = (full + 0.4).astype(np.float32)                       # a rest of 0.33
    dev = lambda a: torch.from_numpy(a).cuda()
    plain = engine.distill_grad_device(x, dev(ids), dev(values), dev(lse))
    for r in range(3):
        only(x, ids, r)
    lse[1] = np.float32(full[1])                                # row 1: nothing left but the rounding of lse
    lse[2] = np.float32(full[2] - 0.1)                          # row 2: more than all (an lse of other numbers): no rest
    ids[3] = -1
    only(x, ids, 3)                                             # row 3: no entry, and no softmax that could matter
    loss, grad = engine.distill_grad_device(x, dev(ids), dev(values), dev(lse))
    alone = engine.distill_device(x, dev(ids), dev(values), dev(lse))
    assert torch.equal(alone.isinf(), loss.isinf()) and not loss.isnan().any() and not grad.isnan().any()
    for r, infinite in ((0, True), (1, False), (2, False)):
        check_row(x, ids, values, lse, loss, grad, r, infinite)
        assert not grad[r][x[r] == -math.inf].any()
        assert infinite or abs(alone[r].item() - loss[r].item()) <= 400 * U
    assert loss[3] == 0 and not grad[3].any()
    assert torch.equal(loss[4:], plain[0][4:]) and torch.equal(grad[4:], plain[1][4:])
    without = engine.distill_device(x, dev(ids), dev(values))   # normalised over the list: nothing is outside it
    assert without.isfinite().all()


@pytest.mark.parametrize("n,K,k", [(5, 1, 1), (5, 10, 10), (5, 32, 40), (4100, 60, 64), (5, 60, 200), (5, 200, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_class_is_listed(engine, n, K, k, dtype):
    """No class is left for a rest, whatever lse says: it is left out, and some class twice in the list makes no difference to that."""
    g = np.random.default_rng([9, n, K, k])
    x = torch.from_numpy((g.standard_normal((n, K)) * 2).astype(np.float32)).to(dtype).cuda()
    ids = np.stack([np.resize(g.permutation(K), k) for _ in range(n)]).astype(np.int32)
    values = (g.standard_normal((n, k)) * 2 + 5).astype(np.float32)
    lse = (np.log(np.exp(values.astype(np.float64)).sum(1)) + 0.4).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).cuda()
    loss, grad = engine.distill_grad_device(x, dev(ids), dev(values), dev(lse))
    for r in range(min(n, 5)):
        check_row(x, ids, values, lse, loss, grad, r, False)
    assert loss.isfinite().all()


@pytest.mark.parametrize("K", [10, 60, 500])
def test_lists_that_repeat_a_class_but_leave_another_out(engine, K):
    """As many entries as classes, and still a class outside them: the rest is counted by the classes listed, not by entries."""
    n, k = 4, min(K, 256)
    g = np.random.default_rng(K)
    ids = np.stack([g.permutation(K)[:k] for _ in range(n)]).astype(np.int32)
    ids[:, -1] = ids[:, 0]
    values = g.standard_normal((n, k)).astype(np.float32)
    lse = (np.log(np.exp(values.astype(np.float64)).sum(1)) + 0.4).astype(np.float32)
    x = torch.from_numpy(g.standard_normal((n, K)).astype(np.float32)).cuda()
    for r in range(n):
        only(x, ids, r)
    dev = lambda a: torch.from_numpy(a).cuda()
    loss, grad = engine.distill_grad_device(x, dev(ids), dev(values), dev(lse))
    for r in range(n):
        check_row(x, ids, values, lse, loss, grad, r, True)
