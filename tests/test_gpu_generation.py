"""Rotation, cache, attention, selection and forking together; captured and compiled calls, streams, sizes beyond 32 bits, refusals."""
import math

import pytest
import torch

from oracle import decode_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------- a model, two ways
class Tiny:
    """Two layers of attention over rotated queries and keys between an embedding and its transpose; 64 bits on the CPU."""

    def __init__(self, vocab, H, Hkv, D, layers, seed):
        g = torch.Generator().manual_seed(seed)
        width = H * D
        n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64) / math.sqrt(s[0])  # noqa: E731
        self.H, self.Hkv, self.D, self.layers = H, Hkv, D, layers
        self.embed = torch.randn(vocab, width, generator=g, dtype=torch.float64)
        self.q, self.k, self.v = ([n(width, h * D) for _ in range(layers)] for h in (H, Hkv, Hkv))
        self.out = n(width, vocab) * 4
        self.inv_freq = (100.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float()

    def logits(self, tokens):
        """Of the last token of one sequence, from the whole of it."""
        x, L = self.embed[tokens], len(tokens)
        at = torch.arange(L)[None]
        for i in range(self.layers):
            q, k, v = ((x @ w[i]).view(1, L, -1, self.D).transpose(1, 2) for w in (self.q, self.k, self.v))
            q, k = orc.rotate(q, at, self.inv_freq), orc.rotate(k, at, self.inv_freq)
            k, v = (t.repeat_interleave(self.H // self.Hkv, 1) for t in (k, v))
            s = (q @ k.transpose(2, 3) / math.sqrt(self.D)).masked_fill(torch.ones(L, L).triu(1).bool(), -math.inf)
            x = x + (s.softmax(-1) @ v).transpose(1, 2).reshape(L, -1)
        return x[-1] @ self.out


def plain_beams(model, prompt, beams, steps, end):
    """Beam search by whole sequences: (scores, sequences), best first."""
    held = [(0.0, list(prompt), False)]
    for _ in range(steps):
        options = []
        for score, seq, done in held:
            if done:
                options.append((score, seq + [end], True))
                continue
            for token, p in enumerate(torch.log_softmax(model.logits(seq), 0).tolist()):
                options.append((score + p, seq + [token], token == end))
        held = sorted(options, key=lambda o: -o[0])[:beams]
    return held


@pytest.mark.parametrize("page,compacts", [(4, True), (16, False), (1, True)])
def test_beam_search_from_the_paged_cache(ca, page, compacts):
    """Against a search that works out every sequence from its beginning: the same beams; afterwards every page is free again."""
    vocab, H, Hkv, D, layers, beams, steps, end = 37, 4, 2, 16, 2, 3, 11, 5
    model = Tiny(vocab, H, Hkv, D, layers, 3)
    prompts = [[7, 9, 30, 2, 11, 18, 3], [1, 22]]
    groups, B, longest = len(prompts), len(prompts) * beams, 7
    weight = lambda w: w.float().cuda()  # noqa: E731
    embed, out = weight(model.embed), weight(model.out)
    rotary = ca.ChillRotary(model.inv_freq.cuda())
    num_pages = B * (-(-(longest + steps) // page) + 1)
    pages = ca.ChillPages.empty(B, longest + steps, num_pages, page)
    shared = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    k_cache, v_cache = (torch.full((layers, num_pages, Hkv, page, D), math.nan, device="cuda") for _ in range(2))
    lens, stored = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    mask = ca.CausalChillMask()

    def forward(tokens, new):
        nonlocal lens
        N = tokens.shape[1]
        step = ca.chill_pages_reserve(pages, lens, new, N, page, stored=stored)
        x = embed[tokens]
        for i in range(layers):
            q, k, v = ((x @ weight(w[i])).view(B, N, -1, D).transpose(1, 2) for w in (model.q, model.k, model.v))
            q = ca.chill_rotate_append(q, k, v, k_cache[i], v_cache[i], step, rotary)
            o = ca.chill_attention_cached(q, k_cache[i], v_cache[i], pages.table, step, mask)
            x = x + o.transpose(1, 2).reshape(B, N, -1)
        lens = lens + stored
        return x @ out

    # prompts in the first beam of each group
    tokens = torch.zeros(B, longest, dtype=torch.int64, device="cuda")
    new = torch.zeros(B, dtype=torch.int32, device="cuda")
    for g, p in enumerate(prompts):
        tokens[g * beams, :len(p)] = torch.tensor(p)
        new[g * beams] = len(p)
    logits = forward(tokens, new)[torch.arange(B), (new - 1).clamp(min=0).long()]
    scores = torch.full((groups, beams), -math.inf, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(groups, beams, dtype=torch.bool, device="cuda")
    history = torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    for t in range(steps):
        scores, parents, tokens = ca.chill_beam_select(logits, scores, finished=finished, end_token=end)
        rows = parents.view(-1)
        finished = finished.view(-1)[rows.long()].view(groups, beams) | (tokens == end)
        history = torch.cat([history[rows.long()], tokens.view(-1, 1)], 1)
        lens, copies = ca.chill_pages_fork(pages, shared, lens, rows, page)
        ca.chill_cache_copy(k_cache, v_cache, copies)
        if compacts and t % 3 == 2:
            ca.chill_cache_copy(k_cache, v_cache, ca.chill_pages_compact(pages, page, shared=shared))
        logits = forward(tokens.view(B, 1).long(), torch.ones_like(new))[:, 0]
    assert pages.missing.item() == 0
    for g, p in enumerate(prompts):
        want = plain_beams(model, p, beams, steps, end)
        gaps = [a[0] - b[0] for a, b in zip(want, want[1:])]
        assert min(gaps) > 1e-3  # so far apart that fp32 cannot exchange them
        for k, (score, seq, _) in enumerate(want):
            assert history[g * beams + k].tolist() == seq[len(p):]
            # logits of about 4 * 16 products each, 11 steps: 2e-5 covers (64 + 16) u of |x| up to 60 a step, ten times over
            assert abs(scores[g, k].item() - score) < 2e-3
    ca.chill_pages_trim(pages, torch.zeros_like(lens), page, shared=shared)
    assert pages.n_free.item() == num_pages and sorted(pages.free.tolist()) == list(range(num_pages)) and not shared.any() and not pages.held.any()


# --------------------------------------------------------------------------------------------------------- graphs
def beam_state(ca, seed, B=6, page=4, num_pages=80, layers=2):
    g = torch.Generator().manual_seed(seed)
    s = {"pages": ca.ChillPages.empty(B, 60, num_pages, page), "shared": torch.zeros(num_pages, dtype=torch.int32, device="cuda")}
    lens = torch.randint(1, 30, (B,), generator=g, dtype=torch.int32).cuda()
    ca.chill_pages_reserve(s["pages"], torch.zeros_like(lens), lens, 30, page)
    s["lens"] = lens
    s["k_cache"], s["v_cache"] = (torch.randn(layers, num_pages, 2, page, 16, generator=g).cuda() for _ in range(2))
    s["logits"] = torch.randn(B, 501, generator=g).cuda()
    s["scores"] = -torch.rand(2, B // 2, generator=g).cuda()
    s["q"], s["k"], s["v"] = (torch.randn(B, h, 1, 16, generator=g).cuda() for h in (4, 2, 2))
    s["rotary"] = ca.ChillRotary.of(16)
    s["one"] = torch.ones(B, dtype=torch.int32, device="cuda")
    s["stored"] = torch.empty(B, dtype=torch.int32, device="cuda")
    return s


def beam_step(ca, s, page=4):
    scores, parents, tokens = ca.chill_beam_select(s["logits"], s["scores"])
    lens, copies = ca.chill_pages_fork(s["pages"], s["shared"], s["lens"], parents.view(-1), page)
    ca.chill_cache_copy(s["k_cache"], s["v_cache"], copies)
    ca.chill_cache_copy(s["k_cache"], s["v_cache"], ca.chill_pages_compact(s["pages"], page, shared=s["shared"]))
    step = ca.chill_pages_reserve(s["pages"], lens, s["one"], 1, page, stored=s["stored"])
    q = ca.chill_rotate_append(s["q"], s["k"], s["v"], s["k_cache"][0], s["v_cache"][0], step, s["rotary"])
    q2, k2 = ca.chill_rotate(s["q"], s["k"], step.positions, s["rotary"])
    ca.chill_pages_trim(s["pages"], lens, page, shared=s["shared"])
    s["lens"].copy_(lens)
    return [scores, parents, tokens, lens, *copies, q, q2, k2]


def everything(s, out):
    return [*out, *s["pages"], s["shared"], s["lens"], s["k_cache"], s["v_cache"]]


def test_a_captured_step_is_replayed_with_other_contents(ca):
    a, b = beam_state(ca, 1), beam_state(ca, 1)
    fresh = beam_state(ca, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):  # nothing of it ran before
            out = beam_step(ca, a)
    torch.cuda.current_stream().wait_stream(stream)
    for turn in range(4):
        if turn == 2:  # other contents in the same tensors
            for s in (a, b):
                for name in ("logits", "scores", "q", "k", "v", "shared", "lens", "k_cache", "v_cache"):
                    s[name].copy_(fresh[name])
                for t, f in zip(s["pages"], fresh["pages"]):
                    t.copy_(f)
        graph.replay()
        want = beam_step(ca, b)
        torch.cuda.synchronize()
        for x, y in zip(everything(a, out), everything(b, want)):
            assert torch.equal(x, y)


def test_two_graphs_and_two_streams_do_not_share_anything(ca):
    """Two captured steps on streams of their own at once, with the same allocator pool: workspaces are each call's own."""
    states = [beam_state(ca, 3), beam_state(ca, 4)]
    copies = [beam_state(ca, 3), beam_state(ca, 4)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for s, stream in zip(states, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(beam_step(ca, s))
        graphs.append(graph)
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, out, c in zip(states, outs, copies):
        for _ in range(3):
            want = beam_step(ca, c)
        for x, y in zip(everything(s, out), everything(c, want)):
            assert torch.equal(x, y)


def test_another_stream_than_the_current_one_at_creation(ca):
    s, c = beam_state(ca, 5), beam_state(ca, 5)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)
        out = beam_step(ca, s)
    torch.cuda.current_stream().wait_stream(stream)
    want = beam_step(ca, c)
    for x, y in zip(everything(s, out), everything(c, want)):
        assert torch.equal(x, y)


def test_a_training_step_is_captured(ca):
    """Rotation, attention and their gradients in one graph, while nothing of an eager graph of the same leaves lives."""
    q, k, v = (torch.randn(2, h, 64, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2))
    rotary, positions = ca.ChillRotary.of(64), torch.arange(64, dtype=torch.int32, device="cuda").expand(2, 64)
    do = torch.randn(2, 4, 64, 64, device="cuda", dtype=torch.bfloat16)

    def step(leaves):
        a, b = ca.chill_rotate(*leaves[:2], positions, rotary)
        return torch.autograd.grad(ca.chill_attention(a, b, leaves[2], ca.CausalChillMask()), leaves, do)

    eager = step([t.clone().requires_grad_() for t in (q, k, v)])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(leaves)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(leaves)
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, eager):  # sums of dQ are not reproducible to the last bit: one step of bf16 around them
        assert torch.allclose(x, y, rtol=2.0 ** -7, atol=2.0 ** -7)


# ----------------------------------------------------------------------------------- dispatcher, compiled graphs, subclasses
def test_dispatcher_ops_give_the_same(ca, monkeypatch):
    from chill_attention import _eager

    a, b = beam_state(ca, 6), beam_state(ca, 6)
    out = beam_step(ca, a)
    monkeypatch.setattr(_eager, "ENABLED", False)
    want = beam_step(ca, b)
    for x, y in zip(everything(a, out), everything(b, want)):
        assert torch.equal(x, y)
    q, k = (torch.randn(2, 3, 5, 8, device="cuda").transpose(1, 2).requires_grad_() for _ in range(2))  # gradients through the ops
    positions, rotary = ints([[0, 5, 9], [1, 2, 3]]), ca.ChillRotary.of(6, axes=(0, 0, 0), interleaved=True)
    one = ca.chill_rotate(q, k, positions, rotary)
    grads = torch.autograd.grad(one, (q, k), (torch.ones_like(one[0]), one[1].detach()))
    lone = torch.autograd.grad(ca.chill_rotate(q, None, positions, rotary)[0].sum(), q)
    second = torch.autograd.grad(ca.chill_rotate(q, k, positions, rotary)[1].sum(), k)
    monkeypatch.setattr(_eager, "ENABLED", True)
    two = ca.chill_rotate(q, k, positions, rotary)
    for x, y in zip((*one, *grads), (*two, *torch.autograd.grad(two, (q, k), (torch.ones_like(two[0]), two[1].detach())))):
        assert torch.equal(x, y) and x.stride() == y.stride()
    assert torch.equal(lone[0], torch.autograd.grad(ca.chill_rotate(q, None, positions, rotary)[0].sum(), q)[0])
    assert torch.equal(second[0], torch.autograd.grad(ca.chill_rotate(q, k, positions, rotary)[1].sum(), k)[0])


def test_ops_pass_opcheck(ca):
    ops = torch.ops.chill_attention
    s = beam_state(ca, 7)
    step = ca.chill_pages_reserve(s["pages"], s["lens"], s["one"], 1, 4)
    q, k = s["q"].clone().requires_grad_(), s["k"].clone().requires_grad_()
    torch.library.opcheck(ops.rotate.default, (q, k, step.positions, s["rotary"].inv_freq, None, False, False))
    torch.library.opcheck(ops.rotate_append.default, (s["q"], s["k"], s["v"], s["k_cache"][0], s["v_cache"][0], step.slots, step.positions,
                                                      s["rotary"].inv_freq, None, False))
    torch.library.opcheck(ops.beam_select.default, (s["logits"], s["scores"], 3, None, 0))
    p = s["pages"]
    torch.library.opcheck(ops.pages_trim_shared.default, (p.table, p.held, p.free, p.n_free, s["shared"], s["lens"], 4))
    torch.library.opcheck(ops.pages_fork.default, (*p, s["shared"], s["lens"], torch.zeros_like(s["lens"]), 4))
    torch.library.opcheck(ops.pages_compact.default, (p.table, p.held, p.free, p.n_free, s["shared"], 4))
    copies = ca.ChillCopies(ints([0]), ints([70]), ints([3]), ints([1]))
    torch.library.opcheck(ops.cache_copy.default, (s["k_cache"], s["v_cache"], *copies))


@pytest.mark.parametrize("dynamic", [False, True])
def test_a_compiled_step(ca, dynamic):
    torch._dynamo.reset()
    a, b = beam_state(ca, 8), beam_state(ca, 8)
    beam_step(ca, beam_state(ca, 9))  # the native module is there
    compiled = torch.compile(lambda s: beam_step(ca, s), fullgraph=True, dynamic=dynamic, backend="aot_eager")
    for _ in range(2):
        out, want = compiled(a), beam_step(ca, b)
        for x, y in zip(everything(a, out), everything(b, want)):
            assert torch.equal(x, y)
    q = torch.randn(2, 3, 8, 64, device="cuda", requires_grad=True)
    positions, rotary = torch.arange(8, dtype=torch.int32, device="cuda").expand(2, 8), ca.ChillRotary.of(64)
    loss = lambda q: (ca.chill_rotate(q, None, positions, rotary)[0] ** 2).sum()  # noqa: E731
    (got,) = torch.autograd.grad(torch.compile(loss, fullgraph=True, dynamic=dynamic, backend="aot_eager")(q), q)
    (want,) = torch.autograd.grad(loss(q), q)
    assert torch.allclose(got, want, rtol=1e-6, atol=1e-6)


def test_versions_of_what_is_changed_in_place(ca):
    s = beam_state(ca, 10)
    versions = lambda: [t._version for t in (*s["pages"], s["shared"], s["k_cache"], s["v_cache"])]  # noqa: E731
    before = versions()
    beam_step(ca, s)
    assert all(x < y for x, y in zip(before, versions()))
    # a gradient that needs the cache's old contents says so
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (s["k_cache"] * w).sum()
    ca.chill_cache_copy(s["k_cache"], s["v_cache"], ca.ChillCopies(ints([0]), ints([1]), ints([1]), ints([1])))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        t = beam_state(ca, 10)
        beam_step(ca, t)


# ---------------------------------------------------------------------------------------------------- large sizes
def test_caches_and_logits_beyond_two_to_the_31_elements(ca):
    pages, page, Hkv, D = 33000, 64, 8, 128
    k_cache, v_cache = (torch.zeros(pages, Hkv, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k_cache.numel() > 2 ** 31
    rows = torch.randn(Hkv, page, D, device="cuda").bfloat16()
    k_cache[pages - 1] = rows
    v_cache[pages - 2] = rows
    ca.chill_cache_copy(k_cache, v_cache, ca.ChillCopies(ints([pages - 1, pages - 2]), ints([0, pages - 3]), ints([page, 5]), ints([2])))
    assert torch.equal(k_cache[0], rows) and torch.equal(v_cache[pages - 3, :, :5], rows[:, :5]) and not v_cache[pages - 3, :, 5:].any()
    q, k, v = (torch.randn(1, h, 2, D, device="cuda").bfloat16() for h in (16, Hkv, Hkv))
    step = ca.ChillStep(ints([0]), ints([2]), ints([[pages * page - 1, 3]]), ints([[7, 8]]), None)
    rotary = ca.ChillRotary.of(D)
    ca.chill_rotate_append(q, k, v, k_cache, v_cache, step, rotary)
    turned = ca.chill_rotate(k, None, step.positions, rotary)[0]
    assert torch.equal(k_cache[pages - 1, :, page - 1], turned[0, :, 0]) and torch.equal(k_cache[0, :, 3], turned[0, :, 1])
    assert torch.equal(v_cache[pages - 1, :, page - 1], v[0, :, 0])
    del k_cache, v_cache
    V, K = 1 << 20, 40
    logits = torch.zeros(54 * K, V, dtype=torch.bfloat16, device="cuda")
    assert logits.numel() > 2 ** 31
    logits[-1, V - 3] = 5.0
    out = ca.chill_beam_select(logits, torch.zeros(54, K, device="cuda"), 2)
    assert out.parents[-1].tolist() == [54 * K - 1, 53 * K] and out.tokens[-1].tolist() == [V - 3, 0]


# ------------------------------------------------------------------------------------------------------- refusals
def test_refusals(ca):
    x, at, rotary = torch.zeros(2, 4, 3, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ca.ChillRotary.of(64)

    def refused(call, match=None):
        with pytest.raises((AssertionError, RuntimeError), match=match):
            call()

    R = ca.chill_rotate
    refused(lambda: R(x, x[:1], at, rotary), "one batch")
    refused(lambda: R(x, x.half(), at, rotary))
    refused(lambda: R(x.double(), None, at, rotary))
    refused(lambda: R(x[0], None, at, rotary), "batch, heads")
    refused(lambda: R(x, None, at.long(), rotary), "int32")
    refused(lambda: R(x, None, at[:1], rotary), "positions must be")
    refused(lambda: R(x, None, at.cpu(), rotary), "int32")
    refused(lambda: R(x, None, at, ca.ChillRotary.of(66)), "more channels")
    refused(lambda: R(x, None, at, rotary._replace(inv_freq=rotary.inv_freq.double())), "float32")
    refused(lambda: R(x, None, at, rotary._replace(axes=at[0])), "axes")
    refused(lambda: R(x, None, at, rotary._replace(inv_freq=rotary.inv_freq.clone().requires_grad_())), "gradient")
    refused(lambda: R(x[:0], None, at[:0], rotary))
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        refused(lambda: R(forward_ad.make_dual(x, x), None, at, rotary), "tangent")
    cache = torch.zeros(8, 4, 16, 64, device="cuda")
    step = ca.ChillStep(at[:, 0].contiguous(), at[:, 0].contiguous(), at, at, None)
    A = lambda q=x, k=x, v=x, kc=cache, vc=cache.clone(), s=step, r=rotary: ca.chill_rotate_append(q, k, v, kc, vc, s, r)  # noqa: E731
    refused(lambda: A(k=x[:, :2], v=x[:, :2]), "kv heads")
    refused(lambda: A(q=x[:1]), "one batch")
    refused(lambda: A(q=x.clone().requires_grad_()), "no gradients")
    refused(lambda: A(kc=cache.half(), vc=cache.half()))
    refused(lambda: A(s=step._replace(slots=at[:, :2])), "slots")

    S, logits, scores = ca.chill_beam_select, torch.zeros(6, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    refused(lambda: S(logits[:5], scores), "row of logits for each")
    refused(lambda: S(logits, scores.double()), "float32")
    refused(lambda: S(logits.double(), scores), "logits must be")
    refused(lambda: S(logits.t().contiguous().t(), scores), "beside each other")
    refused(lambda: S(logits, scores, 65), "at most 64")
    refused(lambda: S(logits, scores, 0), "at most 64")
    refused(lambda: S(logits[:, :1], scores, 4), "fewer candidates")
    refused(lambda: S(logits, scores, finished=torch.zeros(2, 3, device="cuda")), "bool")
    refused(lambda: S(logits, scores, finished=torch.zeros(2, 3, dtype=torch.bool, device="cuda"), end_token=10), "end_token")
    refused(lambda: S(logits.clone().requires_grad_(), scores), "no gradients")
    refused(lambda: S(torch.zeros(130, 4, device="cuda"), torch.zeros(2, 65, device="cuda")), "at most 64")

    pages, lens = ca.ChillPages.empty(2, 100, 8, 16), torch.zeros(2, dtype=torch.int32, device="cuda")
    shared = torch.zeros(8, dtype=torch.int32, device="cuda")
    refused(lambda: ca.chill_pages_fork(pages, shared[:7], lens, lens, 16), "shared")
    refused(lambda: ca.chill_pages_fork(pages, shared, lens[:1], lens, 16), "lens")
    refused(lambda: ca.chill_pages_fork(pages, shared, lens, lens.long(), 16), "parents")
    refused(lambda: ca.chill_pages_trim(pages, lens, 16, shared=shared.float()), "shared")
    refused(lambda: ca.chill_pages_compact(pages, 16, shared=shared[:3]), "shared")
    refused(lambda: ca.chill_pages_compact(pages, 0))
    copies = ca.ChillCopies(lens, lens, lens, lens[:1])
    refused(lambda: ca.chill_cache_copy(cache, cache[:7], copies), "one shape")
    refused(lambda: ca.chill_cache_copy(cache, cache.clone(), copies._replace(rows=lens[:1])), "rows")
    refused(lambda: ca.chill_cache_copy(cache, cache.clone(), copies._replace(count=lens)), "count")
    refused(lambda: ca.chill_cache_copy(cache.clone().requires_grad_(), cache.clone(), copies), "no gradients")
    refused(lambda: ca.chill_cache_copy(cache[0, 0], cache[0, 0], copies), "one shape")
