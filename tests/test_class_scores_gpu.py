"""Class-score operators (Engine.adjust_device, top_device, distill*) against plain 64-bit implementations.

Tolerances (u = 2^-24, half a step of fp32 relative to the value; half a step of the scores' type: torch.finfo(type).eps / 2):
  adjust   at most six fp32 roundings of numbers no larger than |x| max(rep, 1 / rep) + freq N + pres + |bias|, one of the result's type
  lse      an exponential is off by 1 ulp and by the rounding of its argument a (three roundings, 3 u |a| ln 2; the sum weighs it with
           2^a, and sum 2^a |a| / sum 2^a <= log2 of the number of classes < 20): below 45 u; a thread adds at most 8 x 128 of them in
           groups of 8 (136 roundings), 10 merges with two roundings and two exponentials each: below 200 u for the sum, so for its
           logarithm; the result is rounded once more
  loss     everything of a row's own is 64 bit; the student's sum outside the listed classes is off by at most 200 u, moving log p by
           that much at most, against sum q <= 1: 200 u, and the result is rounded once
  gradient w / T (p_c Q + the rest's share of c) (200 u + 3 u |a| + 4 u) and one rounding to the type (values under its smallest
           normal: half its smallest step)"""
import math
import zlib

import numpy as np
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


def rng(*seed):
    return np.random.default_rng([zlib.crc32(s.encode()) if isinstance(s, str) else s for s in (7, *seed)])


def matrix(n, K, dtype, layout="rows", seed=0, scale=2.5):
    """[K, n] on the device.  layout: rows / classes (contiguous), rows_gap / classes_gap (a strided view that starts at an odd element)"""
    x = torch.from_numpy((rng(n, K, seed).standard_normal((n, K)) * scale).astype(np.float32)).to(TYPES[dtype])
    x = x.t() if layout.startswith("rows") else x.t().contiguous()
    major, minor = (n, K) if layout.startswith("rows") else (K, n)
    pitch, start = (minor + 5, 3) if layout.endswith("gap") else (minor, 0)
    buf = torch.full((start + major * pitch + 8,), 77.0, dtype=TYPES[dtype], device="cuda")
    view = buf[start:start + major * pitch].view(major, pitch)[:, :minor]
    view = view.t() if layout.startswith("rows") else view
    view.copy_(x.cuda())
    return view


def half_step(t):
    return torch.finfo(t).eps / 2


def rows64(x):
    """[n, K] in 64 bits on the host"""
    return x.t().double().cpu().numpy()


def close(got, want, tol):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(tol, np.shape(want))
    assert got.shape == want.shape
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3], tol[bad][:3])


# ---- adjust ---------------------------------------------------------------------------------------------------------------------
def adjust_inputs(n, K, seed, history=0, mask="none", bias="none"):
    g, kw = rng(n, K, seed, mask, bias), {}
    if history:
        lens = g.integers(0, history + 1, n)
        lens[0] = history
        if n > 2:
            lens[1] = 0
        first = np.concatenate([[0], np.cumsum(lens)])
        h = (g.random(first[-1]) ** 3 * K).astype(np.int32)
        h[g.random(h.size) < 0.03] = -1
        h[g.random(h.size) < 0.03] = K                      # no class of this matrix
        kw.update(history=h, history_first=first.astype(np.int64), history_prompt=(lens * g.random(n) * 1.2).astype(np.int32),
                  repetition=(0.7 + g.random(n)).astype(np.float32), frequency=g.random(n).astype(np.float32),
                  presence=g.random(n).astype(np.float32))
    if mask != "none":
        words = (K + 31) // 32
        m = g.integers(0, 2 ** 32, (n, words), dtype=np.uint64) | g.integers(0, 2 ** 32, (n, words), dtype=np.uint64)
        m[n // 2] = 0                                       # a row that allows nothing
        m = m.astype(np.uint32).view(np.int32)
        kw["allowed"] = m if mask == "rows" else m[0]
    if bias == "shared":
        kw["bias"] = g.standard_normal(K).astype(np.float32)
    elif bias == "rows":
        kw["bias"] = g.standard_normal((K, n)).astype(np.float32)
    elif bias == "columns":                                 # [K, n] as a view of [n, K]
        kw["bias"] = g.standard_normal((n, K)).astype(np.float32).T
    return kw


def adjust64(x, kw):
    n, K = x.shape
    x, size = x.copy(), np.abs(x)
    if "history" in kw:
        for r in range(n):
            lo, hi = kw["history_first"][r], kw["history_first"][r + 1]
            prompt = min(int(kw["history_prompt"][r]), hi - lo) if kw.get("history_prompt") is not None else 0
            ids = kw["history"][lo:hi].astype(np.int64)
            ok = (ids >= 0) & (ids < K)
            every = np.bincount(ids[ok], minlength=K)
            late = np.bincount(ids[prompt:][ok[prompt:]], minlength=K)
            rep, fr, pr = (float(kw[k][r]) if kw.get(k) is not None else d for k, d in (("repetition", 1), ("frequency", 0), ("presence", 0)))
            with np.errstate(invalid="ignore", divide="ignore"):
                x[r] = np.where(every > 0, np.where(x[r] > 0, x[r] / rep, x[r] * rep), x[r])
            x[r] -= fr * late
            x[r] -= pr * (late > 0)
            size[r] = size[r] * max(rep, 1 / rep) + fr * late + pr
    if "bias" in kw:
        b = kw["bias"].astype(np.float64)
        b = b.T if b.ndim == 2 else b
        x, size = x + b, size + np.abs(b)
    if "allowed" in kw:
        c = np.arange(K)
        on = (kw["allowed"].view(np.uint32)[..., c // 32] >> (c % 32).astype(np.uint32)) & 1
        x = np.where(np.broadcast_to(on, x.shape) != 0, x, -np.inf)
    return x, size


def on_device(kw):
    out = {}
    for k, v in kw.items():
        if k == "bias" and v.ndim == 2 and not v.flags.c_contiguous:
            out[k] = torch.from_numpy(np.ascontiguousarray(v.T)).cuda().t()
        else:
            out[k] = torch.from_numpy(np.ascontiguousarray(v)).cuda()
    return out


def check_adjust(engine, x, kw, **more):
    want, size = adjust64(rows64(x), kw)
    got = engine.adjust_device(x, **on_device(kw), **more)
    assert got.dtype == x.dtype and tuple(got.shape) == tuple(x.shape)
    with np.errstate(invalid="ignore"):
        close(rows64(got), want, 6 * U * size * 1.01 + half_step(x.dtype) * (np.abs(want) + 6 * U * size) + 2.0 ** -25 * (x.dtype == torch.float16))
    return got


ADJUST = [(1, 1, 5), (1, 33, 40), (2, 31, 0), (3, 64, 7), (5, 1000, 300), (300, 10, 6), (65, 257, 20), (7, 4099, 3000), (3, 8193, 9000),
          (2, 50257, 5000), (1, 131072, 1), (2000, 3, 0), (129, 300, 0)]


@pytest.mark.parametrize("layout", ["rows", "classes", "rows_gap", "classes_gap"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,history", ADJUST)
def test_adjust(engine, n, K, history, dtype, layout):
    i = ADJUST.index((n, K, history))
    mask, bias = ["none", "shared", "rows"][i % 3], ["shared", "rows", "columns", "none"][(i + len(layout)) % 4]
    kw = adjust_inputs(n, K, 1, history, mask, bias)
    check_adjust(engine, matrix(n, K, dtype, layout), kw)


@pytest.mark.parametrize("layout", ["rows", "classes_gap"])
@pytest.mark.parametrize("dtype", TYPES)
def test_adjust_in_place_writes_the_matrix_and_nothing_else(engine, dtype, layout):
    n, K = 9, 1003
    x = matrix(n, K, dtype, layout)
    whole = torch.as_strided(x, (x.untyped_storage().size() // x.element_size(),), (1,), 0)
    before = whole.clone()
    kw = adjust_inputs(n, K, 2, 50, "rows", "shared")
    want, _ = adjust64(rows64(x), kw)
    got = engine.adjust_device(x, **on_device(kw), out=x)
    assert got is x
    fresh = torch.empty_like(before).copy_(before)
    y = torch.as_strided(fresh, x.shape, x.stride(), x.storage_offset())
    assert torch.equal(engine.adjust_device(y, **on_device(kw)), x)                            # the same bits as into another buffer
    y.copy_(x)
    assert torch.equal(fresh.view(torch.uint8), whole.view(torch.uint8))                       # the gaps are as they were
    assert np.isneginf(rows64(x)).any() and np.array_equal(np.isneginf(rows64(x)), np.isneginf(want))


@pytest.mark.parametrize("layout", ["rows", "classes"])
def test_adjust_special_scores(engine, layout):
    x = matrix(4, 40, "fp32", layout)
    lowest = torch.finfo(torch.float32).min
    x[:5, 0] = torch.tensor([math.nan, math.inf, -math.inf, lowest, -lowest], device="cuda")
    x[:, 1] = math.nan
    x[:, 2] = lowest
    allowed = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    allowed[0, 0] = ~1                                                                          # NaN in a masked place
    allowed[1] = 0
    y = rows64(engine.adjust_device(x, allowed=allowed))
    assert np.isneginf(y[0, 0]) and y[0, 1] == np.inf and np.isneginf(y[0, 2]) and y[0, 3] == lowest and np.isneginf(y[1]).all()
    assert (y[2] == lowest).all() and np.array_equal(y[3], rows64(x)[3])


def test_adjust_takes_penalties_apart(engine):
    """Without a prompt part every entry counts; absent penalties are neutral; the prompt alone only feels the repetition penalty."""
    x = matrix(3, 50, "fp32")
    kw = adjust_inputs(3, 50, 3, 20)
    for drop in ({"history_prompt"}, {"repetition"}, {"frequency"}, {"presence"}, {"history_prompt", "repetition", "presence"}):
        check_adjust(engine, x, {k: v for k, v in kw.items() if k not in drop})
    all_prompt = dict(kw, history_prompt=np.full(3, 10 ** 6, np.int32))
    check_adjust(engine, x, all_prompt)


def test_adjust_survives_bad_histories(engine):
    """Offsets and class numbers come from the device: they are clamped, nothing outside the arrays is read or written."""
    n, K = 6, 100
    x = matrix(n, K, "fp32")
    h = np.array([3, 3, 2 ** 31 - 1, -2 ** 31, 99, 100], np.int32)
    first = np.array([0, -5, 2 ** 40, 3, 1, 6, -2 ** 62], np.int64)
    kw = dict(history=h, history_first=first, frequency=np.ones(n, np.float32), history_prompt=np.array([-3, 0, 2 ** 31 - 1, 0, 0, -2 ** 31], np.int32))
    got = rows64(engine.adjust_device(x, **on_device(kw)))
    for r in range(n):
        lo = min(max(int(first[r]), 0), 6)
        hi = max(min(max(int(first[r + 1]), 0), 6), lo)
        prompt = min(max(int(kw["history_prompt"][r]), 0), hi - lo)
        want = rows64(x)[r]
        for c in h[lo + prompt:hi]:
            if 0 <= c < K:
                want[c] -= 1
        close(got[r], want, 4 * U * (np.abs(want) + 4))


# ---- top -------------------------------------------------------------------------------------------------------------------------
def top64(x, k, T):
    n, K = x.shape
    order = np.argsort(np.where(np.isnan(x), np.inf, -x), axis=1, kind="stable")[:, :k]
    vals = np.take_along_axis(x, order, 1)
    gone = np.isnan(vals) | np.isneginf(vals)
    ids, vals = np.where(gone, -1, order), np.where(gone, -np.inf, vals)
    if K < k:
        ids = np.concatenate([ids, np.full((n, k - K), -1)], 1)
        vals = np.concatenate([vals, np.full((n, k - K), -np.inf)], 1)
    m = np.max(np.where(np.isnan(x), -np.inf, x), 1, keepdims=True)
    base = np.where(np.isfinite(m), m, 0)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        lse = np.log(np.exp((x - base) / T).sum(1)) + base[:, 0] / T
    lse = np.where(m[:, 0] == np.inf, np.inf, lse)
    return ids, vals, np.where(np.abs(lse) > np.finfo(np.float32).max, np.copysign(np.inf, lse), lse)   # beyond fp32: it rounds to infinity


def check_top(engine, x, k, T=1.0):
    ids, vals, lse = engine.top_device(x, k, T)
    wi, wv, wl = top64(rows64(x), k, T)
    assert ids.dtype == torch.int32 and values_equal(vals, wv)
    assert np.array_equal(ids.cpu().numpy(), wi), np.argwhere(ids.cpu().numpy() != wi)[:4]
    with np.errstate(invalid="ignore"):
        close(lse.double().cpu(), wl, 200 * U + U * np.abs(wl))


def values_equal(a, b):
    return np.array_equal(a.double().cpu().numpy(), b)


TOP = [(1, 1, 1), (3, 2, 2), (300, 10, 3), (1000, 32, 8), (257, 32, 9), (70, 33, 1), (5, 200, 256), (17, 513, 64), (33, 1000, 20), (4, 1025, 200),
       (2, 2047, 256), (3, 2048, 5), (3, 2049, 50), (4, 5000, 256), (2, 16384, 7), (2, 16385, 256), (3, 50257, 50), (1, 131071, 64),
       (1, 1 << 20, 33), (300, 7, 9), (270, 16, 16), (513, 17, 31), (300, 32, 40), (4100, 40, 5), (4096, 130, 16), (4099, 500, 9), (5000, 300, 3),
       (66000, 33, 8), (65537, 64, 2)]


@pytest.mark.parametrize("layout", ["rows", "rows_gap", "classes", "classes_gap"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,k", TOP)
def test_top(engine, n, K, k, dtype, layout):
    x = matrix(n, K, dtype, layout)
    if layout.startswith("classes") and K > 2048:
        if n > 1:
            with pytest.raises(ddt.DDTError, match="class-major"):
                engine.top_device(x, k)
        return
    check_top(engine, x, k, [1.0, 2.0, 0.5][(n + K) % 3])


HARD = ["constant", "ascending", "descending", "two values", "lowest", "one allowed", "nothing allowed", "few allowed", "nan", "inf", "zeros",
        "one thread"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 4096])
@pytest.mark.parametrize("K,k", [(7, 4), (32, 8), (12, 10), (31, 32), (100, 6), (300, 40), (2048, 256), (5000, 64), (40001, 256), (140000, 3)])
@pytest.mark.parametrize("kind", HARD)
def test_top_of_rows_that_tie_or_hold_nothing(engine, kind, K, k, dtype, n):
    if n > 3 and K > 300:
        return                                              # (many rows take other kernels for few classes only)
    x = matrix(n, K, dtype, "classes" if K <= 2048 and K % 2 == 0 else "rows")
    c = torch.arange(K, device="cuda", dtype=torch.float32)
    low = torch.finfo(TYPES[dtype]).min
    if kind == "constant":
        x.fill_(1.5)
    elif kind == "ascending":
        x.copy_((c / K * 8 - 4)[:, None].expand(K, n))
    elif kind == "descending":
        x.copy_((4 - c / K * 8)[:, None].expand(K, n))
    elif kind == "two values":
        x.copy_(((c * 7919) % 3 == 0).float()[:, None].expand(K, n))
    elif kind == "lowest":                              # a mask of the type's lowest value, one row of nothing else
        x[torch.rand(K, n, device="cuda") < 0.5] = low
        x[:, 1] = low
    elif kind == "one allowed":
        x.fill_(-math.inf)
        x[K // 2] = -3.0
    elif kind == "nothing allowed":
        x[:, 1] = -math.inf
    elif kind == "few allowed":
        keep = x[::max(1, K // 3)].clone()
        x.fill_(-math.inf)
        x[::max(1, K // 3)] = keep
    elif kind == "nan":
        x[K // 3, 0] = math.nan
        x[:, 1] = math.nan
    elif kind == "inf":
        x[K // 3, 0] = math.inf
        x[0, 1] = math.inf
        x[K - 1, 1] = math.inf
    elif kind == "zeros":                               # -0 and +0 are one score
        x.copy_(torch.where(c % 2 == 0, 0.0, -0.0)[:, None].expand(K, n))
    elif kind == "one thread":                          # the best stand in the columns that one thread reads
        x.copy_(torch.where((c // 8) % 256 == 5, 9.0 + c / K, -1.0)[:, None].expand(K, n))
    for T in (1.0, 2.0, 0.25):
        check_top(engine, x, k, T)


@pytest.mark.parametrize("K", [10, 300, 5000, 60000])
def test_sums_of_far_scores(engine, K):
    """Scores whose multiples leave the range that fp32 counts whole steps in, or fp32 itself: 10^4 to the lowest and largest number."""
    x = matrix(8, K, "fp32")
    for r, far in enumerate([1e4, -1e4, 3e6, 1e9, -1e20, 1e37, 3e38, -3e38]):
        x[:, r] = far + x[:, r] * (1.0 if abs(far) < 1e5 else 0.0)
        x[K // 2, r] = far
    check_top(engine, x, 5, 2.0)
    check_top(engine, x, 5, 0.5)


def test_top_rows_at_offsets_past_32_bits(engine):
    """A row that starts more than 2^32 elements behind the first."""
    K, stride = 3001, (1 << 32) + 5
    buf = torch.empty(stride + K, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (2, K), (stride, 1))
    x.copy_(matrix(2, K, "bf16").t())
    check_top(engine, x.t(), 20)
    got = engine.adjust_device(x.t(), bias=torch.ones(K, device="cuda"))
    assert torch.equal(got, (x.t().float() + 1).to(torch.bfloat16))


# ---- distill ---------------------------------------------------------------------------------------------------------------------
def teacher_of(n, K, k, T, seed=0, ragged=True):
    g = rng(n, K, k, seed, "teacher")
    kk = min(k, K)
    ids = np.stack([g.permutation(K)[:kk] if K < 5000 else g.choice(K, kk, replace=False) for _ in range(n)]).astype(np.int32)
    if k > kk:
        ids = np.concatenate([ids, np.full((n, k - kk), -1, np.int32)], 1)
    vals = np.sort(g.standard_normal((n, k)) * 2 + 5)[:, ::-1].astype(np.float32).copy()
    if ragged:
        ids[g.random((n, k)) < 0.1] = -1
        if n > 2:
            ids[1] = -1
            ids[2, 0] = K if K < 2 ** 31 - 1 else -7
    lse = (np.log(np.where(ids >= 0, np.exp(vals.astype(np.float64) / T), 0).sum(1) + 0.3 + g.random(n))).astype(np.float32)
    return ids, vals, lse


def distill64(x, ids, vals, lse, T, w):
    """-> loss, gradient, and what the gradient's terms amount to (its tolerance)"""
    n, K = x.shape
    loss, grad, size = np.zeros(n), np.zeros((n, K)), np.zeros((n, K))
    for r in range(n):
        ok = (ids[r] >= 0) & (ids[r] < K)
        if not ok.any():
            continue
        i, t = ids[r][ok].astype(np.int64), vals[r][ok].astype(np.float64) / T
        z = x[r] / T
        with np.errstate(invalid="ignore", divide="ignore"):
            if not (z.max() < np.inf) or z.max() == -np.inf:
                loss[r], grad[r] = np.nan, np.nan
                continue
            log_p = z - z.max() - np.log(np.exp(z - z.max()).sum())
            p = np.exp(log_p)
            if lse is None:
                log_q = t - t.max() - np.log(np.exp(t - t.max()).sum())
            else:
                log_q = t - float(lse[r])
            q = np.exp(log_q)
            out = np.ones(K, bool)
            out[i] = False
            p_r = p[out].sum()
            q_r = max(0.0, 1 - q.sum()) if lse is not None and p_r > 0 else 0.0
            loss[r] = np.where(q > 0, q * (log_q - log_p[i]), 0).sum() + (q_r * (np.log(q_r) - np.log(p_r)) if q_r > 0 else 0)
            Q = 1.0 if lse is None else q.sum() + q_r
            share = np.where(out, p * (q_r / p_r), 0.0) if q_r > 0 else np.zeros(K)
            grad[r] = p * Q - share
            np.subtract.at(grad[r], i, q)
            size[r] = (p * Q + share) * (204 + 3 * np.abs(np.where(np.isfinite(log_p), log_p, 0)) * 1.45)
        grad[r] *= w[r] / T
        size[r] *= w[r] / T * U
    return loss, grad, size


def check_distill(engine, x, ids, vals, lse, T, w=None, grad_out=None):
    """x [n, K] on the device"""
    n, K = x.shape
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()
    w64 = np.ones(n) if w is None else w.astype(np.float64)
    want, grad, size = distill64(x.double().cpu().numpy(), ids, vals, lse, T, w64)
    args = (dev(ids), dev(vals), dev(lse))
    loss = engine.distill_device(x, *args, temperature=T)
    tol = np.where(np.isfinite(want), 200 * U + U * np.abs(want), 0)
    close(loss.double().cpu(), want, tol)
    both, g = engine.distill_grad_device(x, *args, row_weight=dev(w), temperature=T, grad=grad_out)
    assert torch.equal(both, loss) or np.isnan(want).any()
    close(both.double().cpu(), want, tol)
    fi = torch.finfo(x.dtype)
    with np.errstate(invalid="ignore"):
        close(g.double().cpu(), grad, size + (fi.eps / 2) * (np.abs(grad) + size) + fi.smallest_normal * fi.eps / 2 + 2.0 ** -126)
    return loss, g


DISTILL = [(1, 1, 1), (3, 2, 2), (700, 10, 4), (257, 32, 40), (5, 33, 33), (6, 200, 256), (64, 1000, 16), (5000, 40, 3), (4097, 130, 64), (4100, 300, 65), (4096, 515, 20), (3, 2048, 65), (4, 2049, 50), (3, 5003, 256),
           (3, 16385, 64), (3, 50257, 256), (1, 131072, 1), (1, 1 << 20, 100)]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K,k", DISTILL)
def test_distill(engine, n, K, k, dtype, rest):
    T = [1.0, 2.0, 0.5, 4.0][(n + K + k) % 4]
    x = matrix(n, K, dtype, "rows_gap" if k % 2 else "rows").t()
    ids, vals, lse = teacher_of(n, K, k, T)
    w = (0.5 + rng(n, K).random(n)).astype(np.float32) if k % 3 else None
    check_distill(engine, x, ids, vals, lse if rest else None, T, w)


@pytest.mark.parametrize("n,K", [(4, 10), (4, 500), (4, 3000), (4, 20000), (4100, 60), (600, 3000)])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_lists_with_repeats_and_every_class(engine, n, K, rest):
    """The same class in several entries; lists of all the classes (no rest left to speak of)."""
    T = 2.0
    x = matrix(n, K, "fp32").t()
    k = min(K, 256)
    ids, vals, lse = teacher_of(n, K, k, T, ragged=False)
    ids[0, k // 2:] = ids[0, : k - k // 2]
    ids[1] = ids[1, 0]
    ids[2, -1] = ids[2, 0]
    check_distill(engine, x, ids, vals, lse if rest else None, T, np.resize(np.array([1, 2, 0, 0.5], np.float32), n))


@pytest.mark.parametrize("n,K", [(9, 10), (9, 500), (9, 3000), (9, 20000), (4100, 60), (4100, 500), (600, 3000), (600, 10000)])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_students_with_masked_classes(engine, n, K, rest):
    """-inf outside the list, everywhere outside it, in the list (the loss is infinite), in the whole row, and NaN, +inf, lowest values."""
    T, k = 1.0, 3
    x = matrix(n, K, "fp32").t().contiguous()
    ids, vals, lse = teacher_of(n, K, k, T, ragged=False)
    lse[1] = np.float32(np.log(np.exp(vals[1].astype(np.float64)).sum()))
    others = np.setdiff1d(np.arange(K), ids[1])
    x[0, int(np.setdiff1d(np.arange(K), ids[0])[0])] = -math.inf
    x[1, torch.from_numpy(others).cuda()] = -math.inf
    x[2, int(ids[2, 1])] = -math.inf
    x[3] = -math.inf
    x[4, K // 2] = math.nan
    x[5, K // 3] = math.inf
    x[6] = torch.finfo(torch.float32).min
    ids[7] = -1
    x[7] = math.nan                                           # a padded row: whatever stands there, loss 0 and gradient 0
    loss, grad = check_distill(engine, x, ids, vals, lse if rest else None, T)
    assert loss[2] == math.inf and loss[7] == 0 and not grad[7].any() and loss[3].isnan() and grad[3].isnan().all()


@pytest.mark.parametrize("n,K,k", [(12, 10, 3), (12, 20, 7), (4100, 60, 5), (12, 500, 9), (600, 5003, 4), (600, 40001, 4), (12, 50257, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_rows_without_a_softmax(engine, n, K, k, dtype):
    """NaN, wherever the row has no softmax of its student's or its teacher's -- also where all listed probabilities are 0; ordinary rows
    next to them stay as they are"""
    x = matrix(n, K, dtype, seed=5).t().contiguous()
    ids, vals, lse = teacher_of(n, K, k, 2.0, ragged=False)
    outside = [int(np.setdiff1d(np.arange(k + 1), ids[r])[0]) for r in range(n)]
    dev = lambda a: torch.from_numpy(a).cuda()
    plain, plain_grad = engine.distill_grad_device(x, dev(ids), dev(vals), dev(lse), temperature=2.0)
    want, grad, size = distill64(x.double().cpu().numpy(), ids, vals, lse, 2.0, np.ones(n))
    close(plain.double().cpu(), want, 200 * U + U * np.abs(want))
    fi = torch.finfo(x.dtype)
    close(plain_grad.double().cpu(), grad, size + (fi.eps / 2) * (np.abs(grad) + size) + fi.smallest_normal * fi.eps / 2 + 2.0 ** -126)
    vals[:4] = -np.inf                                # rows 0 .. 3: every listed probability is 0, the rest's is 1
    x[0, outside[0]], x[1, outside[1]], x[2] = float("nan"), float("inf"), float("-inf")
    vals[4, k - 1], vals[5, 0], lse[6] = np.nan, np.inf, np.nan
    x[7, int(ids[7, 0])] = float("nan")
    for given, bad, zero_rest in ((dev(lse), [0, 1, 2, 4, 5, 6, 7], [3]), (None, [0, 1, 2, 3, 4, 5, 7], [])):
        loss, grad = engine.distill_grad_device(x, dev(ids), dev(vals), given, temperature=2.0)
        assert torch.equal(engine.distill_device(x, dev(ids), dev(vals), given, temperature=2.0).isnan(), loss.isnan())
        assert loss.isnan().nonzero().flatten().tolist() == bad
        assert grad[bad].isnan().all() and not grad.isnan()[[r for r in range(n) if r not in bad]].any()
        if given is not None:
            assert torch.equal(loss[8:], plain[8:]) and torch.equal(grad[8:], plain_grad[8:])
        for r in zero_rest:                           # loss = -log p_R
            z = x[r].double().cpu().numpy() / 2.0
            e = np.exp(z - z.max())
            log_p = np.log(np.delete(e, ids[r]).sum() / e.sum())
            close(loss[r].item(), -log_p, 200 * U + U * abs(log_p))


@pytest.mark.parametrize("n,K", [(5, 10), (5, 500), (5, 5000), (5, 50257), (4100, 100), (4100, 1000), (600, 9000), (600, 33000), (520, 150001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_gradient_in_place(engine, n, K, dtype):
    T, k = 2.0, 8
    x = matrix(n, K, dtype, "rows_gap").t()
    ids, vals, lse = (torch.from_numpy(a).cuda() for a in teacher_of(n, K, k, T))
    loss, want = engine.distill_grad_device(x, ids, vals, lse, temperature=T)
    whole = torch.as_strided(x, (x.untyped_storage().size() // x.element_size(),), (1,), 0)
    expect = whole.clone()
    torch.as_strided(expect, x.shape, x.stride(), x.storage_offset()).copy_(want)
    again, got = engine.distill_grad_device(x, ids, vals, lse, temperature=T, grad=x)
    assert got is x and torch.equal(again, loss) and torch.equal(whole, expect)        # and the gaps between the rows are as they were


def test_distill_runs_are_alike(engine):
    x = matrix(40, 30011, "bf16").t()
    ids, vals, lse = (torch.from_numpy(a).cuda() for a in teacher_of(40, 30011, 100, 1.0))
    ids[:, 50:60] = ids[:, :10]
    one = engine.distill_grad_device(x, ids, vals, lse)
    for _ in range(3):
        two = engine.distill_grad_device(x, ids, vals, lse)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("K", [7, 90, 2500])
def test_distill_autograd(engine, K, rest):
    """The gradient that autograd takes back, against the formula's and against differences of the 64-bit loss."""
    n, k, T = 4, 5, 2.0
    x = matrix(n, K, "fp32").t().contiguous().requires_grad_()
    ids, vals, lse = teacher_of(n, K, k, T)
    args = [torch.from_numpy(a).cuda() for a in (ids, vals)] + [torch.from_numpy(lse).cuda() if rest else None]
    w = torch.tensor([1.0, 0.0, 2.0, -1.0], device="cuda")
    loss = engine.distill(x, *args, temperature=T)
    (g,) = torch.autograd.grad((loss * w).sum(), x)
    x64, l64 = x.detach().double().cpu().numpy(), lse if rest else None
    want, grad, size = distill64(x64, ids, vals, l64, T, w.cpu().numpy().astype(np.float64))
    close(loss.detach().double().cpu(), want, 200 * U + U * np.abs(want))
    close(g.double().cpu(), grad, np.abs(size) + U * np.abs(grad) + 2.0 ** -126)
    h = 1e-4
    for r, c in [(0, 0), (2, K // 2), (3, K - 1), (0, int(max(ids[0, 0], 0)))]:
        up, down = x64.copy(), x64.copy()
        up[r, c] += h
        down[r, c] -= h
        d = (distill64(up, ids, vals, l64, T, np.ones(n))[0][r] - distill64(down, ids, vals, l64, T, np.ones(n))[0][r]) / (2 * h)
        # differences: h^2 / 6 of a third derivative below 1 / T^3, and 64-bit roundings over h
        assert abs(d * float(w[r]) - float(g[r, c])) <= abs(float(w[r])) * (h * h + 1e-10) + float(abs(size[r, c])) + U * abs(float(g[r, c])) + 1e-9
    mean = engine.distill(x, *args, temperature=T).mean()                               # an upstream gradient of stride 0
    (gm,) = torch.autograd.grad(mean, x)
    _, want_m, size_m = distill64(x64, ids, vals, l64, T, np.full(n, 1 / n))
    close(gm.double().cpu(), want_m, size_m + U * np.abs(want_m) + 2.0 ** -126)


# ---- together --------------------------------------------------------------------------------------------------------------------
def forest(engine, K=10, T=100, F=28):
    w, f = ddt.synth_model(T, 6, F, 0)
    engine.load_model_multiclass(ddt.make_params(T, 6, F, clusters=1), w, f, K, True)
    return F


def test_from_tuples_to_a_students_gradient():
    """classify -> adjust (base scores, a mask) -> top -> distill, as one run, against the class sums the engine gives and 64-bit steps."""
    e = ddt.Engine(0)
    F, n, K, k, T = forest(e), 3001, 10, 4, 2.0
    d = e.synth_tuples_device(0, n, F, 0)
    base = torch.from_numpy(rng("base").standard_normal(K).astype(np.float32)).cuda()
    allowed = torch.tensor([0b1111011111], dtype=torch.int32, device="cuda")
    _, sums = e.classify_device(d)
    ids, vals, lse = e.top_classes_device(d, k, T, bias=base, allowed=allowed)
    adjusted = e.adjust_device(sums, bias=base, allowed=allowed)
    want, size = adjust64(rows64(sums), {"bias": base.cpu().numpy(), "allowed": allowed.cpu().numpy()})
    close(rows64(adjusted), want, 2 * U * size)
    wi, wv, wl = top64(rows64(adjusted), k, T)
    assert np.array_equal(ids.cpu().numpy(), wi) and values_equal(vals, wv) and not (wi == 5).any()
    close(lse.double().cpu(), wl, 200 * U + U * np.abs(wl))
    student = matrix(n, K, "fp32").t().contiguous().requires_grad_()
    loss = e.distill(student, ids, vals, lse, T)
    loss.mean().backward()
    w64, grad, gs = distill64(student.detach().double().cpu().numpy(), ids.cpu().numpy(), vals.cpu().numpy(), lse.cpu().numpy(), T, np.full(n, 1 / n))
    close(loss.detach().double().cpu(), w64, 200 * U + U * np.abs(w64))
    close(student.grad.double().cpu(), grad, gs + U * np.abs(grad) + 2.0 ** -126)
    label = e.top_classes_device(d, 1)[0][:, 0]                                          # k = 1 without adjustments: the engine's own label
    assert torch.equal(label, e.classify_device(d)[0]) and torch.equal(label, e.argmax_device(sums))
    e.close()


@pytest.mark.parametrize("n,K", [(33, 10), (33, 700), (33, 6000), (3, 700_000), (4200, 90)])
def test_captured_and_replayed(engine, n, K):
    """The three operators in one graph, replayed on new data with eager work of the same kind in between."""
    k, T = 4, 2.0
    x, y = matrix(n, K, "fp32", seed=1), matrix(n, K, "bf16", seed=2)
    kw = on_device(adjust_inputs(n, K, 4, 30, "rows", "shared"))
    w = torch.ones(n, device="cuda")

    def step(a, b):
        adjusted = engine.adjust_device(a, **kw)
        ids, vals, lse = engine.top_device(adjusted, k, T)
        return (adjusted, ids, vals, lse, *engine.distill_grad_device(b.t(), ids, vals, lse, w, T))

    step(x, y)
    torch.cuda.synchronize()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step(x, y)
    x2, y2 = x.clone(), y.clone()
    with torch.cuda.graph(g2):                                                           # a second graph of the same calls, replayed beside the first
        held2 = step(x2, y2)
    other = torch.cuda.Stream()
    for i in range(4):
        x.copy_(matrix(n, K, "fp32", seed=10 + i))
        y.copy_(matrix(n, K, "bf16", seed=20 + i))
        x2.copy_(matrix(n, K, "fp32", seed=30 + i))
        y2.copy_(matrix(n, K, "bf16", seed=40 + i))
        for t in (*held, *held2):
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(other):
            g2.replay()
        torch.cuda.synchronize()
        for got, want in zip((*held, *held2), (*step(x, y), *step(x2, y2))):
            assert torch.equal(got, want), i


def test_two_threads_on_streams_of_their_own(engine):
    """Nothing of a call outlives it in the engine: two threads that call it at once, each on its own stream, get what they get alone."""
    import threading

    xs = [matrix(200, 3000 + 77 * i, "fp32", seed=60 + i) for i in range(2)]
    want = [(*engine.top_device(x, 20), *engine.distill_grad_device(x.t(), *engine.top_device(x, 20))) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(30):
            top = engine.top_device(xs[i], 20, stream=s)
            got = (*top, *engine.distill_grad_device(xs[i].t(), *top, stream=s))
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_other_streams(engine):
    """Calls on a stream that is not current: ordered behind that stream's work, results allocated on it."""
    n, K, k = 64, 20000, 30
    s = torch.cuda.Stream()
    want = None
    for i in range(3):
        with torch.cuda.stream(s):
            x = matrix(n, K, "fp32", seed=50)
            a = x + 1.0
            torch.cuda._sleep(2_000_000)
            a.mul_(2.0)
        b = engine.adjust_device(a, bias=None, out=None, stream=s)
        ids, vals, lse = engine.top_device(b, k, stream=s)
        loss, grad = engine.distill_grad_device(b.t(), ids, vals, lse, stream=s)
        s.synchronize()
        got = (b, ids, vals, lse, loss, grad)
        if want is None:
            torch.cuda.synchronize()
            want = [t.clone() for t in got]
            assert torch.equal(b, (x + 1.0) * 2.0)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_no_rows(engine):
    x = torch.empty((12, 0), device="cuda")
    assert engine.adjust_device(x).shape == (12, 0)
    ids, vals, lse = engine.top_device(x, 3)
    assert ids.shape == (0, 3) and lse.shape == (0,)
    loss, grad = engine.distill_grad_device(x.t(), ids, vals, lse)
    assert loss.shape == (0,) and grad.shape == (0, 12)


def test_refusals(engine):
    x = matrix(4, 40, "fp32")
    f, i = torch.float32, torch.int32
    cuda = lambda *s, t=f: torch.zeros(s, dtype=t, device="cuda")
    ids, vals, lse = engine.top_device(x, 3)
    for call in (lambda: engine.adjust_device(x.cpu()), lambda: engine.adjust_device(x.double()), lambda: engine.adjust_device(x[0]),
                 lambda: engine.adjust_device(x, bias=cuda(41)), lambda: engine.adjust_device(x, bias=cuda(40, t=torch.float64)),
                 lambda: engine.adjust_device(x, bias=cuda(40).cpu()), lambda: engine.adjust_device(x, allowed=cuda(1, t=i)),
                 lambda: engine.adjust_device(x, allowed=cuda(4, 4, t=i)[:, ::2]), lambda: engine.adjust_device(x, history=cuda(5, t=i)),
                 lambda: engine.adjust_device(x, history=cuda(5, t=i), history_first=cuda(4, t=torch.int64)),
                 lambda: engine.adjust_device(x, presence=cuda(4)),
                 lambda: engine.adjust_device(x, history=cuda(5, t=i), history_first=cuda(5, t=torch.int64), frequency=cuda(8)[::2]),
                 lambda: engine.top_device(x, 3, ids=cuda(4, 2, t=i)), lambda: engine.distill_device(x.t(), ids.long(), vals),
                 lambda: engine.distill_device(x.t(), ids[:3], vals[:3]), lambda: engine.distill_device(x.t(), ids, vals, lse[:3]),
                 lambda: engine.distill_device(x.t(), ids.t().contiguous().t(), vals),
                 lambda: engine.distill_grad_device(x.t(), ids, vals, lse, row_weight=cuda(3))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: engine.top_device(x, 0), lambda: engine.top_device(x, 257), lambda: engine.top_device(x, 3, temperature=0.0),
                 lambda: engine.distill_device(x.t().contiguous().t().contiguous().t(), ids, vals), lambda: engine.adjust_device(x, out=cuda(40, 4)),
                 lambda: engine.top_device(x[:, ::2].t()[:, ::2].t(), 3), lambda: engine.distill_grad_device(x.t(), ids, vals, grad=torch.empty_like(x).t().half())):
        with pytest.raises(ddt.DDTError):
            call()


def test_streams_of_another_device_are_refused(engine):
    class Other:
        device_index, cuda_stream = engine.device + 1, 0

    x = matrix(3, 10, "fp32")
    ids, vals, lse = engine.top_device(x, 2)
    for call in (lambda: engine.adjust_device(x, out=torch.empty_like(x), stream=Other),
                 lambda: engine.top_device(x, 2, ids=ids, values=vals, lse=lse, stream=Other),
                 lambda: engine.distill_device(x.t(), ids, vals, loss=lse, stream=Other),
                 lambda: engine.distill_grad_device(x.t(), ids, vals, loss=lse, grad=torch.empty(3, 10, device="cuda"), stream=Other)):
        with pytest.raises(ValueError, match="stream"):
            call()


def test_teachers_of_one_entry_lie_in_any_order(engine):
    """one entry per row: the distance of a row's entries says nothing"""
    x = matrix(6, 10, "fp32").t()
    ids, vals, _ = teacher_of(6, 10, 1, 1.0, ragged=False)
    ids, vals = torch.from_numpy(ids).cuda(), torch.from_numpy(vals).cuda()
    want = engine.distill_device(x, ids, vals)
    assert torch.equal(engine.distill_device(x, ids.t().contiguous().t(), vals), want)
    wide = torch.stack([vals, vals], 1)[:, 0]         # rows two apart, the ids' one apart
    with pytest.raises(ValueError, match="equally far"):
        engine.distill_device(x, ids, wide)
