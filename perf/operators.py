"""Cases of the class-score operators: adjusting scores (penalties, biases, masks), the top scores of each row, and the
distillation loss of a student against a teacher's top scores.

`run` computes them in plain torch (own = False) or with the engine's calls (own = True); `exact` computes them in 64 bits,
row block by row block, straight from the definitions:

adjust   x = score; class in the row's history: x = x / rep if x > 0 else x * rep; x -= freq * times behind the prompt part;
         x -= pres if it stands behind the prompt part; x += bias; class not allowed: -inf
top      the k best classes of a row by (score descending, class ascending), never -inf (id -1, value -inf fill up), and
         lse = log sum exp(score / T)
distill  loss = KL(q || p) with p = softmax(student / T) and q the teacher's probabilities of its listed classes -- normalised
         over them, or, with the teacher's log-sum-exp over all its classes, with everything else as one more outcome
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
DEVICE = "cuda"


def listed():
    return [
        # one request of a decode loop: everything on, and latency is what counts
        {"name": "adjust_one_row", "op": "adjust", "rows": 1, "classes": 32000, "dtype": "bf16", "class_major": False,
         "history": 300, "bias": True, "mask": "rows"},
        # a full batch of a decode loop, ragged histories, every row with a grammar of its own
        {"name": "adjust_batch", "op": "adjust", "rows": 64, "classes": 128000, "dtype": "bf16", "class_major": False,
         "history": 8192, "bias": True, "mask": "rows"},
        # few rows with very long histories and an odd number of classes (rows then start at any address)
        {"name": "adjust_long_history", "op": "adjust", "rows": 32, "classes": 50257, "dtype": "fp32", "class_major": False,
         "history": 100000, "bias": False, "mask": "none"},
        # the class sums of a boosted 10-class ensemble get their base scores, one mask for the whole batch
        {"name": "adjust_class_sums", "op": "adjust", "rows": 4000000, "classes": 10, "dtype": "fp32", "class_major": True,
         "history": 0, "bias": True, "mask": "shared"},
        # one row's candidates for sampling
        {"name": "top_one_row", "op": "top", "rows": 1, "classes": 50257, "dtype": "fp16", "class_major": False, "k": 50,
         "temperature": 1.0},
        # a teacher's top logits over a batch of positions; two-byte scores tie all the time
        {"name": "top_batch", "op": "top", "rows": 512, "classes": 128000, "dtype": "bf16", "class_major": False, "k": 64,
         "temperature": 2.0},
        # a classifier head of a thousand classes
        {"name": "top_thousand", "op": "top", "rows": 16384, "classes": 1000, "dtype": "fp32", "class_major": False, "k": 20,
         "temperature": 1.0},
        # label, runners-up and their probabilities from the class sums of a 10-class ensemble
        {"name": "top_class_sums", "op": "top", "rows": 4000000, "classes": 10, "dtype": "fp32", "class_major": True, "k": 3,
         "temperature": 1.0},
        # a small training batch of a student network
        {"name": "distill_small", "op": "distill", "rows": 64, "classes": 1000, "dtype": "fp32", "k": 16, "rest": False,
         "temperature": 2.0, "train": True},
        # evaluation of a student: the loss alone
        {"name": "distill_eval", "op": "distill", "rows": 2048, "classes": 50257, "dtype": "fp16", "k": 50, "rest": True,
         "temperature": 1.0, "train": False},
        # a large training batch over a large set of classes
        {"name": "distill_train", "op": "distill", "rows": 8192, "classes": 128000, "dtype": "bf16", "k": 64, "rest": True,
         "temperature": 2.0, "train": True},
        # a network learns a 10-class ensemble from the rows the ensemble has scored
        {"name": "distill_class_sums", "op": "distill", "rows": 1000000, "classes": 10, "dtype": "fp32", "k": 4, "rest": False,
         "temperature": 2.0, "train": True},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["adjust", "top", "distill"])
    limit = {"adjust": 40_000_000, "top": 60_000_000, "distill": 300_000_000}[op]   # scores
    if op != "distill" and rng.random() < 0.3:                                      # class sums: [classes][rows]
        classes = spread(2, 200)
        case = {"op": op, "classes": classes, "rows": spread(1, min(4_000_000, limit // classes)), "dtype": "fp32",
                "class_major": True}
    else:
        classes = spread(2, 128_000)
        case = {"op": op, "classes": classes, "rows": spread(1, min(1_000_000, max(1, limit // classes))),
                "dtype": rng.choice(["fp32", "fp16", "bf16"])}
        if op != "distill":
            case["class_major"] = False
    if op == "adjust":
        most = min(100_000, 4_000_000 // case["rows"])
        case.update(history=spread(1, most) if most >= 1 and rng.random() < 0.7 else 0, bias=rng.random() < 0.5,
                    mask=rng.choice(["none", "shared", "rows"]))
    else:
        case.update(k=min(spread(1, 256), case["classes"]), temperature=rng.choice([0.5, 1.0, 2.0, 4.0]))
    if op == "distill":
        case.update(rest=rng.random() < 0.5, train=rng.random() < 0.7)
    return case


def _scores(case, gen):
    n, K = case["rows"], case["classes"]
    shape = (K, n) if case.get("class_major") else (n, K)
    x = torch.empty(shape, dtype=DTYPES[case["dtype"]], device=DEVICE)
    for part in x.split(max(1, (1 << 27) // shape[1])):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE) * 2.5)
    return x if case.get("class_major") else x.t()      # [classes, rows] either way


def _engine():
    """The engine a user's program has open (the operators need its device, not a loaded model)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    package = os.path.join(root, "distributed-decisiontrees_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ddt

    return ddt.Engine(0)


def _mask_words(case, gen):
    """Bits of the allowed classes, about one class in eight left out; the one mask of a batch leaves some class of it."""
    words = (case["classes"] + 31) // 32
    rows = case["rows"] if case["mask"] == "rows" else 1
    a, b, c = (torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device=DEVICE).to(torch.int32) for _ in range(3))
    m = a | b | c
    m[:, 0] |= 1
    return m if case["mask"] == "rows" else m[0]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    n, K = case["rows"], case["classes"]
    state = {"case": case}
    if case["op"] == "distill":
        student = _scores(case, gen).t()
        k = case["k"]
        ids = torch.empty((n, k), dtype=torch.int32, device=DEVICE)
        values = torch.empty((n, k), dtype=torch.float32, device=DEVICE)
        lse = torch.empty(n, dtype=torch.float32, device=DEVICE)
        step = max(1, (1 << 27) // K)
        for r in range(0, n, step):                      # the teacher: near the student, and surer of itself
            x = student[r:r + step]
            t = x.float() * 1.25 + torch.randn(x.shape, generator=gen, device=DEVICE)
            v, i = torch.topk(t, k, dim=1)
            values[r:r + step], ids[r:r + step] = v, i.to(torch.int32)
            lse[r:r + step] = torch.logsumexp(t / case["temperature"], dim=1)
        ids[torch.rand((n, 1), generator=gen, device=DEVICE).expand(n, k) < 0.02] = -1      # padded rows of the batch
        ragged = torch.randint(1, k + 1, (n, 1), generator=gen, device=DEVICE)              # nucleus cut: fewer than k classes
        if k > 1:
            cut = torch.rand((n, 1), generator=gen, device=DEVICE) < 0.25
            ids[cut & (torch.arange(k, device=DEVICE) >= ragged)] = -1
        state.update(student=student, ids=ids, values=values, lse=lse if case["rest"] else None)
        if case["train"]:
            state["weight"] = torch.rand(n, generator=gen, device=DEVICE) + 0.5             # loss scale x weight of the row
    else:
        state["scores"] = _scores(case, gen)
        if case["op"] == "top" and not case["class_major"]:                                 # classes that a mask took out
            for part in state["scores"].t().split(max(1, (1 << 27) // K)):
                part.masked_fill_(torch.rand(part.shape, generator=gen, device=DEVICE) < 0.1, -math.inf)
    if case["op"] == "adjust":
        state["bias"] = torch.randn(K, generator=gen, device=DEVICE) if case["bias"] else None
        state["allowed"] = _mask_words(case, gen) if case["mask"] != "none" else None
        if case["history"]:
            H = case["history"]
            lens = torch.randint(0, H + 1, (n,), generator=gen, device=DEVICE)
            lens[0] = H
            first = torch.zeros(n + 1, dtype=torch.int64, device=DEVICE)
            first[1:] = torch.cumsum(lens, 0)
            total = int(first[-1])
            u = torch.rand(total, generator=gen, device=DEVICE)
            state["history"] = (u * u * u * K).to(torch.int32).clamp_(max=K - 1)            # few classes come often
            state["history_first"] = first
            state["history_prompt"] = (lens * torch.rand(n, generator=gen, device=DEVICE)).to(torch.int32)
            state["repetition"] = 1.0 + 0.5 * torch.rand(n, generator=gen, device=DEVICE)
            state["frequency"] = 0.5 * torch.rand(n, generator=gen, device=DEVICE)
            state["presence"] = torch.rand(n, generator=gen, device=DEVICE)
    if own:
        state["engine"] = _engine()
    return state


# ---- the plain forms: 32 bits, rounded once at the end -------------------------------------------------------------
def _row_of(first, total):
    """Row of every history entry."""
    return torch.searchsorted(first, torch.arange(total, device=first.device), right=True) - 1


def _adjust(state):
    scores = state["scores"]
    x = scores.t().float()                                                       # [rows, classes]
    n, K = x.shape
    if "history" in state:
        history, first = state["history"].long(), state["history_first"]
        row = _row_of(first, history.numel())
        behind = torch.arange(history.numel(), device=x.device) - first[row] >= state["history_prompt"][row]
        flat = row * K + history
        seen = torch.zeros(n * K, dtype=torch.int32, device=x.device)
        seen.index_add_(0, flat, torch.ones_like(flat, dtype=torch.int32))
        said = torch.zeros(n * K, dtype=torch.int32, device=x.device)
        said.index_add_(0, flat, behind.int())
        seen, said = seen.view(n, K) > 0, said.view(n, K)
        rep = state["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - state["frequency"][:, None] * said.float()
        x = torch.where(said > 0, x - state["presence"][:, None], x)
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        bit = torch.arange(32, dtype=torch.int32, device=x.device)
        on = ((state["allowed"][..., None] >> bit) & 1).flatten(-2)[..., :K]
        x = torch.where(on != 0, x, -math.inf)
    return x.to(scores.dtype).t()


def _log_sum_exp(x):
    """In 64 bits behind the exponentials: long sums, and logarithms whose differences count."""
    top = x.amax(1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    return torch.log(torch.exp(x - top).sum(1, dtype=torch.float64)) + top[:, 0]


def _top(state):
    case, k = state["case"], state["case"]["k"]
    x = state["scores"].t().float()
    n, K = x.shape
    bits = (x + 0.0).contiguous().view(torch.int32)                              # -0 and +0 are one score
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()                          # whole numbers in the order of the scores
    key = (order << 32) | (K - 1 - torch.arange(K, device=x.device))             # equal scores: the lower class first
    ids = K - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    values = torch.gather(x, 1, ids)
    ids = torch.where(values == -math.inf, -1, ids)
    return ids.to(torch.int32), values, _log_sum_exp(x / case["temperature"]).float()


def _distill(state):
    case = state["case"]
    student, T = state["student"], case["temperature"]
    z = student.float() / T
    n, K = z.shape
    there = (state["ids"] >= 0) & (state["ids"] < K)
    ids = torch.where(there, state["ids"], 0).long()
    some = there.any(1)
    # the rows' own numbers in 64 bits: 1 - sum of q, and a loss near zero, are differences of near numbers
    t = torch.where(there, state["values"].double() / T, -math.inf)
    lse_t = torch.logsumexp(t, 1) if state["lse"] is None else state["lse"].double()
    log_q = t - torch.where(some, lse_t, 0.0)[:, None]
    q = torch.exp(log_q)
    listed_class = torch.zeros((n, K + 1), dtype=torch.bool, device=z.device)
    listed_class.scatter_(1, torch.where(there, ids, K), True)
    outside = ~listed_class[:, :K]
    lse, lse_r = _log_sum_exp(z), _log_sum_exp(torch.where(outside, z, -math.inf))
    p_r = torch.exp(lse_r - lse)
    log_p = torch.gather(student, 1, ids).double() / T - lse[:, None]
    # sum q log(q / p) = sum (q log(q / p) - q + p) + the student's share outside: every summand counts up from zero
    loss = torch.where(there, q * torch.where(q > 0, log_q - log_p, 0.0) - q + torch.exp(log_p), 0.0).sum(1)
    mass = q.sum(1)
    if case["rest"]:
        q_r = torch.where(p_r > 0, (1.0 - mass).clamp(min=0.0), 0.0)
        loss = loss + torch.where(q_r > 0, q_r * (torch.log(q_r) - (lse_r - lse)), 0.0) - q_r + p_r
        mass = mass + q_r
        loss = loss + (mass - 1.0)
    else:
        loss = loss + p_r
    loss = torch.where(some, loss, 0.0).float()
    if not case["train"]:
        return loss
    grad = torch.exp(z - lse.float()[:, None]) * mass.float()[:, None]
    if case["rest"]:
        share = torch.where(q_r > 0, q_r, 0.0).float()
        grad = grad - torch.where(outside, torch.exp(z - lse_r.float()[:, None]) * share[:, None], 0.0)
    grad.scatter_add_(1, ids, torch.where(there, -q, 0.0).float())
    grad = torch.where(some[:, None], grad * (state["weight"] / T)[:, None], 0.0)
    return loss, grad.to(student.dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"adjust": _adjust, "top": _top, "distill": _distill}[case["op"]](state)
    engine = state["engine"]
    if case["op"] == "adjust":
        return engine.adjust_device(state["scores"], bias=state["bias"], allowed=state["allowed"],
                                    **{name: state[name] for name in ("history", "history_first", "history_prompt", "repetition",
                                                                      "frequency", "presence") if name in state})
    if case["op"] == "top":
        return engine.top_device(state["scores"], case["k"], temperature=case["temperature"])
    teacher = (state["student"], state["ids"], state["values"], state["lse"])
    if case["train"]:
        return engine.distill_grad_device(*teacher, row_weight=state["weight"], temperature=case["temperature"])
    return engine.distill_device(*teacher, temperature=case["temperature"])


def work(case):
    n, K, size = case["rows"], case["classes"], BYTES[case["dtype"]]
    matrix = n * K * size
    if case["op"] == "adjust":
        masks = (K + 31) // 32 * 4 * {"none": 0, "shared": 1, "rows": n}[case["mask"]]
        extra = (n * (case["history"] // 2) * 4 + 24 * n) if case["history"] else 0      # lengths are uniform up to the longest
        return {"bytes": 2 * matrix + masks + extra + (4 * K if case["bias"] else 0), "flops": 6 * n * K}
    if case["op"] == "top":
        return {"bytes": matrix + n * (8 * case["k"] + 4), "flops": 4 * n * K}
    teacher = n * (8 * case["k"] + 4) + (4 * n if case["rest"] else 0)
    if not case["train"]:
        return {"bytes": matrix + teacher, "flops": 5 * n * K}
    return {"bytes": 2 * matrix + teacher + 4 * n, "flops": 10 * n * K}


# ---- 64 bits, from the definitions --------------------------------------------------------------------------------
def _blocks(n, K):
    step = max(1, 100_000_000 // max(1, K))
    return [(r, min(n, r + step)) for r in range(0, n, step)]


def _exact_adjust(case, state):
    scores = state["scores"].t()
    out = torch.empty(scores.shape, dtype=torch.float64, device=DEVICE)
    for a, b in _blocks(*scores.shape):
        x = scores[a:b].double()
        if case["history"]:
            lo, hi = int(state["history_first"][a]), int(state["history_first"][b])
            bounds = state["history_first"][a:b + 1] - lo
            entry = torch.arange(hi - lo, device=DEVICE)
            row = torch.bucketize(entry, bounds, right=True) - 1
            cls = state["history"][lo:hi].long()
            late = entry - bounds[row] >= state["history_prompt"][a:b].long()[row]
            n_all = torch.zeros_like(x).index_put_((row, cls), torch.ones_like(row, dtype=torch.float64), accumulate=True)
            n_late = torch.zeros_like(x).index_put_((row, cls), late.double(), accumulate=True)
            rep = state["repetition"][a:b].double()[:, None]
            factor = torch.where(x > 0, 1 / rep, rep)
            x = torch.where(n_all > 0, x * factor, x)
            x -= state["frequency"][a:b].double()[:, None] * n_late
            x -= state["presence"][a:b].double()[:, None] * (n_late > 0)
        if case["bias"]:
            x += state["bias"].double()
        if case["mask"] != "none":
            word = state["allowed"] if case["mask"] == "shared" else state["allowed"][a:b]
            c = torch.arange(x.shape[1], device=DEVICE)
            x[((word.long()[..., c // 32] >> (c % 32)) & 1 == 0).expand_as(x)] = -math.inf
        out[a:b] = x
    return out.t()


def _exact_top(case, state):
    scores, k = state["scores"].t(), case["k"]
    n, K = scores.shape
    ids = torch.empty((n, k), dtype=torch.int32, device=DEVICE)
    values = torch.empty((n, k), dtype=torch.float64, device=DEVICE)
    lse = torch.empty(n, dtype=torch.float64, device=DEVICE)
    for a, b in _blocks(n, K):
        x = scores[a:b].double()
        v, i = torch.sort(x, dim=1, descending=True, stable=True)                # stable: equal scores keep the order of the classes
        values[a:b] = v[:, :k]
        ids[a:b] = torch.where(torch.isinf(v[:, :k]), -1, i[:, :k])
        lse[a:b] = torch.logsumexp(x / case["temperature"], dim=1)
    return ids, values, lse


def _exact_distill(case, state):
    student, T, k = state["student"], case["temperature"], case["k"]
    n, K = student.shape
    losses = torch.zeros(n, dtype=torch.float64, device=DEVICE)
    grads = torch.zeros((n, K), dtype=torch.float64, device=DEVICE) if case["train"] else None
    for a, b in _blocks(n, K):
        log_p = torch.log_softmax(student[a:b].double() / T, dim=1)
        ids = state["ids"][a:b].long()
        gone = ids < 0
        t = (state["values"][a:b].double() / T).masked_fill(gone, -math.inf)
        norm = state["lse"][a:b].double() if case["rest"] else torch.logsumexp(t, dim=1)
        q = torch.exp(t - norm[:, None]).masked_fill(gone, 0.0)
        target = torch.zeros((b - a, K), dtype=torch.float64, device=DEVICE)
        inside = torch.zeros((b - a, K), dtype=torch.float64, device=DEVICE)
        for j in range(k):                                                       # entry by entry
            col = ids[:, j:j + 1].clamp(min=0)
            target.scatter_add_(1, col, q[:, j:j + 1])
            inside.scatter_add_(1, col, (~gone[:, j:j + 1]).double())
        inside = inside > 0
        loss = torch.xlogy(q, q).sum(1) - torch.where(target > 0, target * log_p, 0.0).sum(1)
        total = q.sum(1)
        if case["rest"]:
            log_r = torch.logsumexp(log_p.masked_fill(inside, -math.inf), dim=1)
            q_r = torch.where(torch.isinf(log_r), 0.0, (1 - total).clamp(min=0))
            loss += torch.where(q_r > 0, torch.xlogy(q_r, q_r) - q_r * log_r, 0.0)
            total = total + q_r
            if case["train"]:
                inner = torch.exp(log_p - log_r[:, None]).masked_fill(inside, 0.0)
                target += torch.where(q_r > 0, q_r, 0.0)[:, None] * torch.where(torch.isinf(log_r)[:, None], 0.0, inner)
        keep = ~gone.all(1)
        losses[a:b] = torch.where(keep, loss, 0.0)
        if case["train"]:
            g = (torch.exp(log_p) * total[:, None] - target) * (state["weight"][a:b].double() / T)[:, None]
            grads[a:b] = torch.where(keep[:, None], g, 0.0)
    return (losses, grads) if case["train"] else losses


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    return {"adjust": _exact_adjust, "top": _exact_top, "distill": _exact_distill}[case["op"]](case, state)
