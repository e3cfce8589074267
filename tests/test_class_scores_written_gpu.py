"""Tensors that the class-score calls write into: autograd has to learn of it, or the call is refused."""
import pytest

import ddt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    e = ddt.Engine(0)
    yield e
    e.close()


def inputs(engine, n=6, K=40, k=3):
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    student = torch.randn((n, K), generator=g, device="cuda")
    return student, engine.top_device(torch.randn((n, K), generator=g, device="cuda").t(), k)


@pytest.mark.parametrize("how", ["adjust", "gradient"])
def test_a_student_that_is_overwritten_between_loss_and_backward(engine, how):
    student, teacher = inputs(engine)
    student.requires_grad_()
    loss = engine.distill(student, *teacher)
    before = student.detach().clone()
    with torch.no_grad():
        if how == "adjust":
            engine.adjust_device(student.t(), bias=torch.ones(40, device="cuda"), out=student.t())
        else:
            engine.distill_grad_device(student, *teacher, grad=student)
    assert not torch.equal(student.detach(), before)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.sum().backward()


def test_a_teacher_that_is_overwritten_between_loss_and_backward(engine):
    student, teacher = inputs(engine)
    student.requires_grad_()
    for i in range(3):
        loss = engine.distill(student, *teacher)
        ids, values, lse = (t if j == i else None for j, t in enumerate(teacher))
        engine.top_device(student.detach().t(), 3, ids=ids, values=values, lse=lse)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.sum().backward()


def test_results_that_autograd_would_have_to_see(engine):
    student, teacher = inputs(engine)
    leaf = student.clone().requires_grad_()
    inner = leaf * 1.0
    loss, part = torch.zeros(6, device="cuda", requires_grad=True), torch.zeros((6, 3), device="cuda", requires_grad=True)
    for x in (leaf, inner):
        for call in (lambda: engine.adjust_device(x.t(), out=x.t()), lambda: engine.adjust_device(student.t(), out=x.t()),
                     lambda: engine.distill_grad_device(x, *teacher, grad=x), lambda: engine.distill_device(student, *teacher, loss=loss),
                     lambda: engine.distill_grad_device(student, *teacher, loss=loss), lambda: engine.top_device(student.t(), 3, values=part),
                     lambda: engine.top_device(student.t(), 3, lse=loss)):
            before = x.detach().clone()
            with pytest.raises(ValueError, match="requires grad"):
                call()
            assert torch.equal(x.detach(), before)
            with torch.no_grad():
                call()                                                   # nothing is being recorded: allowed
            with torch.no_grad():
                x.copy_(before)
    assert not engine.adjust_device(leaf.t()).requires_grad              # not in place: the result carries no gradient


def test_versions_count_every_call_that_writes(engine):
    student, teacher = inputs(engine)
    ids, values, lse = (t.clone() for t in teacher)
    loss, grad = torch.empty(6, device="cuda"), torch.empty_like(student)
    for call, written in ((lambda: engine.adjust_device(student.t(), out=grad.t()), [grad]),
                          (lambda: engine.top_device(student.t(), 3, ids=ids, values=values, lse=lse), [ids, values, lse]),
                          (lambda: engine.distill_device(student, *teacher, loss=loss), [loss]),
                          (lambda: engine.distill_grad_device(student, *teacher, loss=loss, grad=grad), [loss, grad])):
        everything = [student, *teacher, ids, values, lse, loss, grad]
        before = [t._version for t in everything]
        call()
        for t, v in zip(everything, before):
            assert t._version == v + any(t is w for w in written)


def test_results_inside_inference_mode(engine):
    with torch.inference_mode():
        student, teacher = inputs(engine)
        out = torch.empty_like(student)
        engine.adjust_device(student.t(), bias=torch.ones(40, device="cuda"), out=out.t())
        assert torch.equal(out, student + 1)
        assert not engine.distill(student, *teacher).requires_grad
