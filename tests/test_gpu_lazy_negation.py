"""Tensors whose sign is still to be applied (torch's negative bit, as of z.conj().imag) count with their sign in every call that reads memory itself."""
import pytest
import torch

from cache_helpers import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


def lazy(x):
    """x, held as the negative of what lies in memory."""
    y = torch._neg_view(-x)
    assert y.is_neg() and torch.equal(y, x) and y.stride() == x.stride()
    return y


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_the_imaginary_part_of_a_conjugate(ca):
    """What a user meets it in."""
    z = torch.complex(*torch.randn(2, 2, 3, 5, 64, device="cuda").unbind())
    x = z.conj().imag
    assert x.is_neg()
    positions, rotary = torch.arange(5, dtype=torch.int32, device="cuda").expand(2, 5), ca.ChillRotary.of(64)
    assert torch.equal(ca.chill_rotate(x, None, positions, rotary)[0], ca.chill_rotate(-z.imag, None, positions, rotary)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation(ca, dtype):
    q, k, v = (torch.randn(2, h, 5, 64, device="cuda").to(dtype) for h in (4, 2, 2))
    rotary, positions = ca.ChillRotary.of(64), ints([[1, 2, 3, 4, 5], [9, 8, 7, 6, 5]])
    want = ca.chill_rotate(q, k, positions, rotary)
    for a, b in ((lazy(q), k), (q, lazy(k)), (lazy(q), lazy(k))):
        for x, y in zip(ca.chill_rotate(a, b, positions, rotary), want):
            assert torch.equal(x, y)
    for x, y in zip(ca.chill_rotate(q, k, lazy(positions), rotary._replace(inv_freq=lazy(rotary.inv_freq))), want):
        assert torch.equal(x, y)
    caches = [torch.zeros(3, 2, 16, 64, device="cuda", dtype=dtype) for _ in range(4)]
    step = ca.ChillStep(ints([0, 0]), ints([5, 5]), ints([[0, 1, 2, 3, 4], [16, 17, 18, 19, 20]]), positions, None)
    want = ca.chill_rotate_append(q, k, v, *caches[:2], step, rotary)
    got = ca.chill_rotate_append(lazy(q), lazy(k), lazy(v), *caches[2:], step, rotary)
    assert torch.equal(got, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_selection(ca):
    logits, scores = torch.randn(6, 500, device="cuda"), -torch.rand(2, 3, device="cuda")
    want = ca.chill_beam_select(logits, scores)
    for a, b in ((lazy(logits), scores), (logits, lazy(scores))):
        for x, y in zip(ca.chill_beam_select(a, b), want):
            assert torch.equal(x, y)


def test_pages(ca):
    def state():
        pages, shared = ca.ChillPages.empty(3, 64, 20, 4), torch.zeros(20, dtype=torch.int32, device="cuda")
        lens = ints([9, 14, 3])
        ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, 14, 4)
        return pages, shared, lens

    (pages, shared, lens), (other, counts, _) = state(), state()
    k, v = (torch.randn(20, 2, 4, 8, device="cuda") for _ in range(2))
    k2, v2 = k.clone(), v.clone()
    one = ca.chill_pages_fork(pages, shared, lens, ints([0, 0, 1]), 4)
    two = ca.chill_pages_fork(other, counts, lazy(lens), lazy(ints([0, 0, 1])), 4)
    ca.chill_cache_copy(k, v, one[1])
    ca.chill_cache_copy(k2, v2, ca.ChillCopies(*map(lazy, two[1])))
    ca.chill_pages_trim(pages, ints([5, 5, 0]), 4, shared=shared)
    ca.chill_pages_trim(other, lazy(ints([5, 5, 0])), 4, shared=counts)
    moved = ca.chill_pages_compact(pages, 4, shared=shared), ca.chill_pages_compact(other, 4, shared=counts)
    for x, y in zip((one[0], *one[1], *moved[0], *pages, shared, k, v), (two[0], *two[1], *moved[1], *other, counts, k2, v2)):
        assert torch.equal(x, y)


def test_paged_cache(ca):
    p = Problem(torch.float32, 4, 2, 64, [9, 30], [2, 2], 2, 16)
    k_cache, v_cache = (t.nan_to_num(0.0).cuda() for t in (p.k_cache, p.v_cache))
    q, step, table, mask = p.q.cuda(), p.step(), p.table.cuda(), ca.CausalChillMask()
    want = ca.chill_attention_cached(q, k_cache, v_cache, table, step, mask)
    for args in ((lazy(q), k_cache, v_cache), (q, lazy(k_cache), v_cache), (q, k_cache, lazy(v_cache))):
        assert torch.equal(ca.chill_attention_cached(*args, table, step, mask), want)
    k, v = (torch.randn(2, 2, 2, 64, device="cuda") for _ in range(2))
    k2, v2 = k_cache.clone(), v_cache.clone()
    ca.chill_cache_append(k_cache, v_cache, k, v, step.slots)
    ca.chill_cache_append(k2, v2, lazy(k), lazy(v), step.slots)
    assert torch.equal(k_cache, k2) and torch.equal(v_cache, v2)


@pytest.mark.parametrize("fast", [True, False])
def test_what_is_changed_in_place_is_refused(ca, monkeypatch, fast):
    """Torch cannot apply a pending sign to what an operator changes, where it also returns something: no call takes it, and nothing is written."""
    from chill_attention import _eager

    monkeypatch.setattr(_eager, "ENABLED", fast)
    x, caches = torch.randn(1, 2, 3, 8, device="cuda"), [torch.randn(5, 2, 4, 8, device="cuda") for _ in range(2)]
    step = ca.ChillStep(ints([0]), ints([3]), ints([[0, 1, 2]]), ints([[0, 1, 2]]), None)
    pages, shared, lens = ca.ChillPages.empty(1, 16, 5, 4), torch.zeros(5, dtype=torch.int32, device="cuda"), ints([3])
    ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, 3, 4)
    copies = ca.ChillCopies(*(ints([n]) for n in (0, 1, 4, 1)))
    before = [t.clone() for t in (*caches, *pages, shared)]
    for n in range(2):
        pair = [lazy(c) if i == n else c for i, c in enumerate(caches)]
        calls = [lambda: ca.chill_rotate_append(x, x, x, *pair, step, ca.ChillRotary.of(8)), lambda: ca.chill_cache_append(*pair, x, x, step.slots),
                 lambda: ca.chill_cache_commit(*pair, pages.table, step, ints([[0]]), ints([1])), lambda: ca.chill_cache_copy(*pair, copies)]
        for call in calls:
            with pytest.raises(AssertionError, match="_cache is changed in place"):
                call()
    for name in pages._fields:
        some = pages._replace(**{name: lazy(getattr(pages, name))})
        calls = [lambda: ca.chill_pages_reserve(some, lens, lens, 3, 4), lambda: ca.chill_pages_fork(some, shared, lens, ints([0]), 4)]
        if name != "missing":  # the others do not touch it
            calls += [lambda: ca.chill_pages_trim(some, lens, 4), lambda: ca.chill_pages_trim(some, lens, 4, shared=shared), lambda: ca.chill_pages_compact(some, 4)]
        for call in calls:
            with pytest.raises(AssertionError, match=f"{name} is changed in place"):
                call()
    for call in (lambda: ca.chill_pages_fork(pages, lazy(shared), lens, ints([0]), 4), lambda: ca.chill_pages_trim(pages, lens, 4, shared=lazy(shared)),
                 lambda: ca.chill_pages_compact(pages, 4, shared=lazy(shared)), lambda: ca.chill_pages_reserve(pages, lens, lens, 3, 4, stored=lazy(lens))):
        with pytest.raises(AssertionError, match="(shared|stored) is changed in place"):
            call()
    for t, was in zip((*caches, *pages, shared), before):
        assert torch.equal(t, was)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", range(5))
def test_attention_and_its_gradients(ca, dtype, which):
    """q, k, v, the gradient of O and that of the LSE."""
    g = torch.Generator().manual_seed(which)
    q, k, v, do = (torch.randn(1, h, 70, 64, generator=g).to(dtype).cuda() for h in (4, 2, 2, 4))
    dlse = torch.randn(1, 4, 70, generator=g).cuda()
    mask = ca.CausalChillMask()

    def step(q, k, v, do, dlse):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ca.chill_attention(*leaves, mask, return_lse=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (do, dlse)))

    was = ca.is_deterministic()
    ca.set_deterministic(True)
    try:
        args = [q, k, v, do, dlse]
        want = step(*args)
        args[which] = lazy(args[which])
        for x, y in zip(step(*args), want):
            assert torch.equal(x, y)
        with torch.no_grad():
            assert torch.equal(ca.chill_attention(*args[:3], mask, lens=lazy(ints([33]))), ca.chill_attention(q, k, v, mask, lens=ints([33])))
    finally:
        ca.set_deterministic(was)


@pytest.mark.parametrize("which", range(4))
def test_attention_of_host_tensors(ca, which):
    from chill_attention.host import attention_fwd_bwd_host

    was = ca.is_deterministic()
    ca.set_deterministic(True)
    try:
        args = [torch.randn(1, h, 64, 64).bfloat16() for h in (4, 2, 2, 4)]
        want = attention_fwd_bwd_host(*args, ca.CausalChillMask())
        args[which] = lazy(args[which])
        for x, y in zip(attention_fwd_bwd_host(*args, ca.CausalChillMask()), want):
            assert torch.equal(x, y)
        with pytest.raises(AssertionError):
            attention_fwd_bwd_host(*args, ca.CausalChillMask(), out=tuple(torch._neg_view(x) for x in want))
    finally:
        ca.set_deterministic(was)
