"""More rows than a launch has blocks (2^20) times rows per block: the blocks go round again.  The rows repeat with a period, so the results
of the second round have to be those of the first, bit for bit (and those of the first are held to 64 bits elsewhere)."""
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BLOCKS = 1 << 20
PERIOD = 37


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()
    torch.cuda.empty_cache()


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


def rows(n, *shape, dtype=torch.float32, seed=0):
    """[n, *shape], row r = that of r % PERIOD"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    one = (torch.randn((PERIOD, *shape), generator=g, device="cuda") * 2).to(dtype)
    return one.expand(n // PERIOD, PERIOD, *shape).reshape(n, *shape)


def round_up(n):
    return (n + 3 * PERIOD) // PERIOD * PERIOD


def same_rounds(n, per_block, *results):
    """Rows of the second round, and those in front of it, against the first rows."""
    assert n > BLOCKS * per_block
    for t in results:
        first = t[:PERIOD]
        begin = (BLOCKS * per_block // PERIOD - 1) * PERIOD
        tail = t[begin:].view(-1, PERIOD, *t.shape[1:])
        assert len(tail) >= 2 and torch.equal(tail, first.expand_as(tail))
        assert not torch.equal(first, first[:1].expand_as(first))       # (the rows do differ)


@pytest.mark.parametrize("class_major", [False, True])
def test_top_with_a_thread_per_row(engine, class_major):
    n = round_up(BLOCKS * 256)
    x = rows(n, 2, dtype=torch.bfloat16)
    same_rounds(n, 256, *engine.top_device(x.t().contiguous() if class_major else x.t(), 1))


def test_top_of_all_classes_with_a_thread_per_row(engine):
    n = round_up(BLOCKS * 256)
    same_rounds(n, 256, *engine.top_device(rows(n, 2, dtype=torch.float16).t(), 9))


@pytest.mark.parametrize("k,per_block", [(9, 16), (17, 4)])              # 16 lanes per row, a wave per row
def test_top_of_short_rows(engine, k, per_block):
    n = round_up(BLOCKS * per_block)
    same_rounds(n, per_block, *engine.top_device(rows(n, 33, dtype=torch.bfloat16).t(), k))


@pytest.mark.parametrize("k", [9, 17])
def test_top_of_short_class_major_rows(engine, k):
    n = round_up(BLOCKS * 16)
    same_rounds(n, 16, *engine.top_device(rows(n, 33, dtype=torch.bfloat16).t().contiguous(), k))


def test_top_with_a_block_per_row(engine):
    n = round_up(BLOCKS)
    same_rounds(n, 1, *engine.top_device(rows(n, 2051, dtype=torch.bfloat16).t(), 40))


def teacher(n, K, k):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    ids = torch.randint(-1, K, (PERIOD, k), generator=g, device="cuda").to(torch.int32)
    return ids.expand(n // PERIOD, PERIOD, k).reshape(n, k), rows(n, k, seed=4), rows(n, seed=5) + 4.0


@pytest.mark.parametrize("K,k,per_block,dtype", [(3, 1, 256, torch.bfloat16), (33, 2, 16, torch.bfloat16), (33, 65, 4, torch.bfloat16), (2051, 5, 1, torch.float32),
                                                 (8195, 5, 1, torch.bfloat16)])
def test_distill(engine, K, k, per_block, dtype):
    n = round_up(BLOCKS * per_block)
    x, t = rows(n, K, dtype=dtype), teacher(n, K, k)
    same_rounds(n, per_block, engine.distill_device(x, *t))
    loss, grad = engine.distill_grad_device(x, *t, grad=x)
    same_rounds(n, per_block, loss, grad)


def histories(n, per_row, K):
    """every row the same number of entries"""
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    h = torch.randint(0, K, (PERIOD, per_row), generator=g, device="cuda").to(torch.int32)
    return dict(history=h.expand(n // PERIOD, PERIOD, per_row).reshape(-1), history_first=torch.arange(n + 1, device="cuda") * per_row,
                frequency=rows(n, seed=7), repetition=rows(n, seed=8).abs() + 0.5)


@pytest.mark.parametrize("history", [0, 3])
def test_adjust_of_rows(engine, history):
    K = 2048                                                            # a tile: 512 packs, a row of fp32
    n = round_up(BLOCKS)
    x, bias = rows(n, K), torch.randn(K, device="cuda")
    engine.adjust_device(x.t(), bias=bias, out=x.t(), **(histories(n, history, K) if history else {}))
    same_rounds(n, 1, x)


def test_adjust_of_rows_with_long_histories(engine):
    K, tiles = 1 << 20, 128                                             # a tile: 1024 packs, 128 of them a bf16 row
    n = round_up(BLOCKS // tiles)
    x = rows(n, K, dtype=torch.bfloat16)
    engine.adjust_device(x.t(), out=x.t(), **histories(n, 6007, K))
    tail = x[(BLOCKS // tiles // PERIOD - 1) * PERIOD:].view(-1, PERIOD, K)
    assert n * tiles > BLOCKS and len(tail) >= 2 and all(torch.equal(t, x[:PERIOD]) for t in tail)


@pytest.mark.parametrize("history", [0, 2])
def test_adjust_of_class_major_rows(engine, history):
    per_block = 64 if history else 1024                                 # rows of a tile, with one class
    n = round_up(BLOCKS * per_block)
    x = rows(n, 1).t().contiguous()
    kw = histories(n, history, 1) if history else dict(bias=torch.ones(1, device="cuda"))
    engine.adjust_device(x, out=x, **kw)
    same_rounds(n, per_block, x.view(n, 1))
