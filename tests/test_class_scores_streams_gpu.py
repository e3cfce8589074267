"""Tensors that a class-score call uses on a stream of its own: a caller who lets them go right after the call must not get their memory
back before that stream is done with them."""
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

N, K, WIDTH = 300, 8192, 4                  # tensors of more than 1 MiB lie in blocks of their own size


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


def f32(*shape):
    return torch.ones(shape, device="cuda")


def i32(*shape):
    return torch.ones(shape, dtype=torch.int32, device="cuda")


def calls(e):
    """name -> (tensors of the call, the call on a stream)"""
    words, many = (K + 31) // 32, 1_000_003
    teacher = lambda: dict(ids=i32(N, 256), values=f32(N, 256), lse=f32(N))
    return {
        "adjust": (lambda: dict(class_scores=f32(N, K).t(), bias=f32(K), allowed=-i32(N, words), history=i32(many),
                                history_first=torch.full((N + 1,), many, device="cuda") * torch.arange(N + 1, device="cuda").clamp(max=1),
                                history_prompt=i32(N), repetition=f32(N), frequency=f32(N), presence=f32(N), out=f32(N, K).t()), e.adjust_device),
        "top": (lambda: dict(class_scores=f32(N, K).t(), ids=i32(N, 256), values=f32(N, 256), lse=f32(N)),
                lambda stream, **kw: e.top_device(k=256, stream=stream, **kw)),
        "distill": (lambda: dict(student=f32(N, K), loss=f32(N), **teacher()), e.distill_device),
        "gradient": (lambda: dict(student=f32(N, K), row_weight=f32(N), loss=f32(N), grad=f32(N, K), **teacher()), e.distill_grad_device),
    }


@pytest.mark.parametrize("name", ["adjust", "top", "distill", "gradient"])
def test_memory_of_a_call_is_not_given_out_again_while_its_stream_works(engine, name):
    make, call = calls(engine)[name]
    tensors = make()
    sizes = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in tensors.values()}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)                        # about a tenth of a second: the call stands behind it
    result = call(stream=s, **tensors)
    del tensors, result
    again = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes.values()]
    assert not s.query()
    assert not {t.data_ptr() for t in again} & set(sizes)
    s.synchronize()


def test_tuples_and_adjustments_of_top_classes(engine):
    e = ddt.Engine(0)
    F, classes = 28, 10
    w, f = ddt.synth_model(100, 6, F, 0)
    e.load_model_multiclass(ddt.make_params(100, 6, F, clusters=1), w, f, classes, True)
    d = e.synth_tuples_device(0, 300_000, F, 0)
    bias = torch.randn((classes, 300_000), device="cuda")
    want = [t.clone() for t in e.top_classes_device(d, 3, bias=bias)]
    torch.cuda.synchronize()
    sizes = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (d, bias)}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
    got = e.top_classes_device(d, 3, stream=s, bias=bias)
    del d, bias
    again = [torch.empty(n, dtype=torch.uint8, device="cuda").fill_(255) for n in sizes.values()]
    assert not s.query() and not {t.data_ptr() for t in again} & set(sizes)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    e.close()


def test_the_current_stream_handed_in(engine):
    """The current stream by name is the same call as without one."""
    x = torch.randn((5, 300), device="cuda")
    for a, b in zip(engine.top_device(x.t(), 4), engine.top_device(x.t(), 4, stream=torch.cuda.current_stream())):
        assert torch.equal(a, b)
