"""Gradients that reach the rotation's backward in other forms than plain memory, and inputs that need none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


class Wrapped(torch.Tensor):
    """A wrapper: the numbers are in `inner`, the tensor itself has no memory."""

    @staticmethod
    def __new__(cls, inner):
        x = torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype, device=inner.device)
        x.inner = inner
        return x

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        plain = lambda t: t.inner if isinstance(t, Wrapped) else t  # noqa: E731
        return func(*[plain(a) for a in args], **{n: plain(a) for n, a in (kwargs or {}).items()})


class GradientAs(torch.autograd.Function):
    """The identity, whose gradient comes in another form."""

    @staticmethod
    def forward(ctx, x, form):
        ctx.form = form
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        return ctx.form(g), None


def problem(ca, dtype=torch.float32):
    g = torch.Generator().manual_seed(5)
    q, k, gq, gk = (torch.randn(2, h, 7, 32, generator=g).to(dtype).cuda() for h in (4, 2, 4, 2))
    positions = torch.randint(0, 900, (2, 7), generator=g, dtype=torch.int32).cuda()
    return q.requires_grad_(), k.requires_grad_(), gq, gk, positions, ca.ChillRotary.of(32)


FORMS = {"plain": lambda x: x, "negated": lambda x: torch._neg_view(-x), "wrapped": Wrapped, "zero": lambda x: torch._efficientzerotensor(x.shape, device=x.device)}


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("of_q", FORMS)
@pytest.mark.parametrize("of_k", [*FORMS, None])
def test_forms_of_gradients(ca, monkeypatch, of_q, of_k, fast):
    from chill_attention import _eager

    q, k, gq, gk, positions, rotary = problem(ca)
    with torch.no_grad():
        inverse = rotary._replace(inv_freq=-rotary.inv_freq)
        zero = lambda form, x: torch.zeros_like(x) if form == "zero" else x  # noqa: E731
        want = ca.chill_rotate(zero(of_q, gq), zero(of_k, gk), positions, inverse)
    monkeypatch.setattr(_eager, "ENABLED", fast)
    a, b = ca.chill_rotate(q, k, positions, rotary)
    a = GradientAs.apply(a, FORMS[of_q])
    if of_k is None:
        (dq,) = torch.autograd.grad((a * gq).sum(), q)
    else:
        dq, dk = torch.autograd.grad((a * gq).sum() + (GradientAs.apply(b, FORMS[of_k]) * gk).sum(), (q, k))
        assert torch.equal(dk, want[1])
    assert torch.equal(dq, want[0])


@pytest.mark.parametrize("form", ["negated", "wrapped"])
def test_the_gradients_gradient_in_such_a_form(ca, form):
    q, k, gq, gk, positions, rotary = problem(ca)
    gq, gk = gq.requires_grad_(), gk.requires_grad_()
    out = ca.chill_rotate(q, k, positions, rotary)
    grads = torch.autograd.grad(out, (q, k), (gq, gk), create_graph=True)
    w = torch.randn_like(gq).detach()
    (d,) = torch.autograd.grad((GradientAs.apply(grads[0], FORMS[form]) * w).sum(), gq)  # turned forth again
    assert torch.equal(d, ca.chill_rotate(w, None, positions, rotary)[0])


def test_a_negated_gradient_is_differentiated(ca):
    q, k, gq, gk, positions, rotary = problem(ca)
    held = (-gq).requires_grad_()
    (dq,) = torch.autograd.grad(ca.chill_rotate(q, None, positions, rotary)[0], q, torch._neg_view(held), create_graph=True)
    w = torch.randn_like(gq)
    (d,) = torch.autograd.grad(dq, held, w)
    assert torch.equal(d, -ca.chill_rotate(w, None, positions, rotary)[0])


def test_batched_gradients(ca):
    """Rows of a Jacobian at once."""
    q, k, gq, gk, positions, rotary = problem(ca)
    out = ca.chill_rotate(q, k, positions, rotary)
    several = torch.stack([gq, 2 * gq, -gq]), torch.stack([gk, gk * 0, gk + 1])
    dq, dk = torch.autograd.grad(out, (q, k), several, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        one = torch.autograd.grad(out, (q, k), (several[0][i], several[1][i]), retain_graph=True)
        assert torch.equal(dq[i], one[0]) and torch.equal(dk[i], one[1])


def test_saved_tensors_may_be_packed(ca):
    q, k, gq, gk, positions, rotary = problem(ca, torch.bfloat16)
    rotary = rotary._replace(axes=torch.zeros(16, dtype=torch.int32, device="cuda"))
    want = torch.autograd.grad(ca.chill_rotate(q, k, positions, rotary), (q, k), (gq, gk))
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: (packed.append(1), x.cpu())[1], lambda x: x.cuda()):
        out = ca.chill_rotate(q, k, positions, rotary)
    got = torch.autograd.grad(out, (q, k), (gq, gk))
    assert len(packed) == 3 and all(torch.equal(x, y) for x, y in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        out = ca.chill_rotate(q, k, positions.expand(2, 7), rotary)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(out, (q, k), (gq, gk)), want))


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("needs_q", [True, False])
def test_only_what_needs_a_gradient_gets_one(ca, monkeypatch, needs_q, fast):
    """The turned form of a constant is a constant: nothing behind it works out a gradient for it, and the backward turns the other one alone."""
    from chill_attention import _decode_abi, _eager

    monkeypatch.setattr(_eager, "ENABLED", fast)
    q, k, gq, gk, positions, rotary = problem(ca)
    (k if needs_q else q).requires_grad_(False)
    out = ca.chill_rotate(q, k, positions, rotary)
    assert [x.requires_grad for x in out] == [needs_q, not needs_q]
    asked = []
    needed = out[0 if needs_q else 1]
    needed.register_hook(lambda g: asked.append(g.shape))
    (out[0].sum() * out[1].sum()).backward()
    leaf, constant = (q, k) if needs_q else (k, q)
    assert constant.grad is None and asked == [leaf.shape]
    (want,) = torch.autograd.grad(ca.chill_rotate(leaf, None, positions, rotary)[0], leaf, torch.ones_like(leaf) * out[1 if needs_q else 0].sum().detach())
    assert torch.equal(leaf.grad, want)
    for y in out:  # and once more, both ways of asking
        if y.requires_grad:
            (again,) = torch.autograd.grad(ca.chill_rotate(q, k, positions, rotary)[0 if needs_q else 1], leaf, gq if needs_q else gk)
            with torch.no_grad():
                assert torch.equal(again, ca.chill_rotate(gq if needs_q else gk, None, positions, rotary._replace(inv_freq=-rotary.inv_freq))[0])


@pytest.mark.parametrize("needs_q", [True, False])
def test_a_compiled_call_with_a_constant(ca, needs_q):
    torch._dynamo.reset()
    q, k, gq, gk, positions, rotary = problem(ca)
    leaf, constant = (q, k) if needs_q else (k, q)
    constant.requires_grad_(False)
    loss = lambda q, k: (lambda out: (out[0].sum() * out[1].sum(), out))(ca.chill_rotate(q, k, positions, rotary))  # noqa: E731
    got, out = torch.compile(loss, fullgraph=True, backend="aot_eager")(q, k)
    assert [x.requires_grad for x in out] == [needs_q, not needs_q]
    want, _ = loss(q, k)
    assert torch.allclose(torch.autograd.grad(got, leaf)[0], torch.autograd.grad(want, leaf)[0], rtol=1e-6, atol=1e-6)
