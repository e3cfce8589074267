"""Sums of exponentials over long rows of near-equal scores: one score ahead, all others alike, which rounds a running fp32 sum to the same
side again and again.

Tolerances (u = 2^-24): an exponential is off by 1 ulp (2 u) and by its argument's three roundings (3 u |a| ln 2 with |a| <= 20 where it
counts: 42 u); a group of up to 32 of them is added in four chains (10 u); groups are added in 64 bits; threads, waves and the block
merge in 12 additions and three exponentials whose arguments are 0 for rows like these (18 u), and the sum's logarithm carries all that
over: below 100 u.  The result is rounded once (u |result|)."""
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


def one_ahead(n, K, dtype, seed, below=8.0):
    """[n, K]: class 0 at 0, the others at one negative score, another in each row"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (-below * torch.rand((n, 1), generator=g, device="cuda")).to(dtype).expand(n, K).contiguous()
    x[:, 0] = 0
    return x


def log_sum(x, T=1.0):
    return torch.cat([torch.logsumexp(p.double() / T, 1) for p in x.split(max(1, (1 << 26) // x.shape[1]))])


def close(got, want, u=100):
    off = (got.double() - want).abs() / (U * (u + want.abs()))
    assert off.max() <= 1, off.max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,K,k", [(65536, 1000, 3), (65537, 2000, 8), (65600, 2048, 1), (66000, 61, 3)])
def test_class_major_rows_of_near_equal_scores(engine, n, K, k, dtype):
    x = one_ahead(n, K, dtype, K)
    ids, values, lse = engine.top_device(x.t().contiguous(), k, 1.0)
    close(lse, log_sum(x))
    assert torch.equal(ids, torch.arange(k, device="cuda", dtype=torch.int32).expand(n, k)) and torch.equal(values, x[:, :k].float())


@pytest.mark.parametrize("n,K", [(70, 2048), (300, 16384), (3, 1 << 20), (257, 1 << 20), (70000, 64)])
def test_row_major_rows_of_near_equal_scores(engine, n, K):
    x = one_ahead(n, K, torch.float32, K + n)
    ids, _, lse = engine.top_device(x.t(), 5, 1.0)
    close(lse, log_sum(x))
    assert torch.equal(ids, torch.arange(5, device="cuda", dtype=torch.int32).expand(n, 5))


@pytest.mark.parametrize("n,K", [(513, 1 << 20), (3, 1 << 20), (600, 50257)])
def test_losses_over_long_rows_of_near_equal_scores(engine, n, K):
    x = one_ahead(n, K, torch.float32, K)
    ids, values = torch.ones((n, 1), dtype=torch.int32, device="cuda"), torch.ones((n, 1), device="cuda")
    want = log_sum(x) - x[:, 1].double()                     # one class listed, no rest: the loss is -log p
    close(engine.distill_device(x, ids, values), want)
    loss, grad = engine.distill_grad_device(x, ids, values)
    close(loss, want)
    p = torch.exp(x[:, 2].double() - log_sum(x))
    off = (grad[:, 2].double() - p).abs() / (p * U)
    assert off.max() <= 200 + 3 * 14 * 1.45 + 5, off.max().item()


@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
def test_losses_over_long_rows_of_scores_far_from_zero(engine, T):
    """Scores near 2^21, where only their differences are exact: the largest score is taken off before the scaling."""
    n, K = 513, 600_001
    step = 0.25 * (1 + torch.arange(n, device="cuda") % 16)[:, None]
    x = (2.0 ** 21 + 8 - step).expand(n, K).contiguous()
    x[:, 0] = 2.0 ** 21 + 8
    ids, values = torch.ones((n, 1), dtype=torch.int32, device="cuda"), torch.ones((n, 1), device="cuda")
    far = step[:, 0].double() / T
    want = torch.log1p((K - 1) * torch.exp(-far)) + far
    close(engine.distill_device(x, ids, values, temperature=T), want)
    loss, grad = engine.distill_grad_device(x, ids, values, temperature=T)
    close(loss, want)
    assert torch.equal(grad[:, 2], grad[:, -1])
