"""Rotary positions, beam selection, shared pages and page copies on the GPU against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import decode_oracle as orc

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # and among the smallest numbers
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------------------ rotation
def check_turned(y, x, expected, pairs, interleaved, dtype):
    """cos and sin are off by at most 6 u (the angle in half turns, rounded to fp32: pi u / 2; sincospif: 2 u; the 64-bit angle: less than u / 2 at a hundred million turns), products
    and sum by 2 u more of |x1| + |x2|; then the result is rounded to its type.  Channels that stay are equal."""
    x = x.detach().cpu().double()
    y = y.detach().cpu()
    assert y.dtype == dtype and y.shape == expected.shape
    size = torch.zeros_like(x)
    for i in range(pairs):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        size[..., lo] = size[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    bound = 8 * U * size
    bound = bound + EPS[dtype] * (expected.abs() + bound) + TINY[dtype]
    assert ((y.double() - expected).abs() <= bound).all(), ((y.double() - expected).abs() / bound).max().item()
    assert torch.equal(y[..., 2 * pairs:].double(), x[..., 2 * pairs:])


def turn_of(ca, g, D, channels, axes, interleaved):
    which = None if axes == 1 else torch.randint(0, axes, (channels // 2,), generator=g).tolist()
    rotary = ca.ChillRotary.of(channels, axes=which, interleaved=interleaved)
    return rotary, which


def strided(shape, dtype, g, layout):
    B, H, L, D = shape
    if layout == "heads":  # [B, H, L, D], contiguous
        return torch.randn(shape, generator=g).to(dtype).cuda()
    if layout == "tokens":  # as a projection leaves it
        return torch.randn(B, L, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    if layout == "packed":  # part of a larger row, off by one element
        return torch.randn(B, L, H, D + 3, generator=g).to(dtype).cuda().transpose(1, 2)[..., 1:D + 1]
    return torch.randn(B, H, D, L, generator=g).to(dtype).cuda().transpose(2, 3)  # channels apart


ROTATIONS = [
    # dtype, B, H, Hkv, L, D, channels, axes, interleaved, layout
    (torch.float32, 1, 4, 2, 1, 64, 64, 1, False, "heads"),
    (torch.float32, 2, 3, 3, 37, 64, 64, 1, True, "tokens"),
    (torch.float32, 2, 2, 1, 19, 80, 50, 2, False, "heads"),
    (torch.float16, 3, 8, 2, 130, 128, 96, 3, True, "tokens"),
    (torch.float16, 1, 5, 5, 65, 32, 6, 3, False, "heads"),
    (torch.float16, 2, 2, 2, 9, 16, 2, 1, True, "packed"),
    (torch.bfloat16, 2, 16, 4, 257, 128, 128, 1, False, "tokens"),
    (torch.bfloat16, 1, 4, 1, 33, 256, 256, 3, True, "heads"),
    (torch.bfloat16, 2, 3, 1, 21, 64, 44, 2, False, "channels"),
    (torch.bfloat16, 5, 2, 2, 7, 128, 102, 1, True, "packed"),
    (torch.bfloat16, 1, 200, 3, 2, 64, 64, 1, False, "heads"),
]


@pytest.mark.parametrize("dtype,B,H,Hkv,L,D,channels,axes,interleaved,layout", ROTATIONS)
def test_rotate_and_its_gradient(ca, dtype, B, H, Hkv, L, D, channels, axes, interleaved, layout):
    g = torch.Generator().manual_seed(B * L + D)
    rotary, which = turn_of(ca, g, D, channels, axes, interleaved)
    q, k = (strided((B, h, L, D), dtype, g, layout).requires_grad_() for h in (H, Hkv))
    shape = (B, L) if axes == 1 else (axes, B, L)
    positions = torch.randint(0, 200000, shape, generator=g, dtype=torch.int32).cuda()
    gq, gk = (strided((B, h, L, D), dtype, g, "heads") for h in (H, Hkv))
    out = ca.chill_rotate(q, k, positions, rotary)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for x, y, gx, dx in ((q, out[0], gq, grads[0]), (k, out[1], gk, grads[1])):
        check_turned(y, x, orc.rotate(x, positions, rotary.inv_freq, which, interleaved), channels // 2, interleaved, dtype)
        check_turned(dx, gx, orc.rotate(gx, positions, rotary.inv_freq, which, interleaved, inverse=True), channels // 2, interleaved, dtype)
        if layout in ("heads", "tokens"):
            assert y.stride() == x.stride()
    alone = ca.chill_rotate(q.detach(), None, positions, rotary)
    assert alone[1] is None and torch.equal(alone[0], out[0])


def test_far_positions(ca):
    """Positions up to 2^31 - 1: the 64-bit angle is off by 2^-22 turns there at most, 1.5e-6 radians."""
    rotary = ca.ChillRotary.of(64)
    positions = ints([[0, 1, 10 ** 6, 2 ** 24 + 1, 2 ** 29 - 1, 2 ** 31 - 1, -5]])
    q = torch.randn(1, 2, 7, 64, device="cuda")
    y, _ = ca.chill_rotate(q, None, positions, rotary)
    expected = orc.rotate(q, positions, rotary.inv_freq)
    size = (q.double().cpu()[..., :32].abs() + q.double().cpu()[..., 32:].abs()).repeat(1, 1, 1, 2)
    assert ((y.cpu().double() - expected).abs() <= (2e-6 + 9 * U) * size).all()


def test_rotate_gradients_of_shared_and_missing_inputs(ca):
    g = torch.Generator().manual_seed(3)
    rotary = ca.ChillRotary.of(32)
    positions = torch.arange(11, dtype=torch.int32, device="cuda").expand(2, 11)  # one row for all
    base = torch.randn(1, 1, 11, 32, generator=g).cuda().requires_grad_()
    q = base.expand(2, 3, 11, 32)
    y, _ = ca.chill_rotate(q, None, positions, rotary)
    w = torch.randn(2, 3, 11, 32, generator=g).cuda()
    (y * w).sum().backward()
    expected = orc.rotate(w, positions, rotary.inv_freq, inverse=True).sum((0, 1), keepdim=True)
    assert torch.allclose(base.grad.cpu().double(), expected, rtol=0, atol=6 * 12 * U * w.abs().sum().item() / 32)
    # one of the results is not used; the sum's gradient is an expanded tensor
    q, k = (torch.randn(2, h, 11, 32, generator=g).cuda().requires_grad_() for h in (3, 1))
    out = ca.chill_rotate(q, k, positions, rotary)
    out[1].sum().backward()
    assert q.grad is None
    ones = torch.ones_like(k).detach()
    check_turned(k.grad, ones, orc.rotate(ones, positions, rotary.inv_freq, inverse=True), 16, False, torch.float32)
    # the gradient of the gradient: turned forth again
    q = torch.randn(1, 1, 11, 32, generator=g, dtype=torch.float32).cuda().requires_grad_()
    y, _ = ca.chill_rotate(q, None, positions[:1], rotary)
    v = torch.randn(1, 1, 11, 32, generator=g).cuda().requires_grad_()
    (dq,) = torch.autograd.grad(y, q, v, create_graph=True)
    (dv,) = torch.autograd.grad(dq, v, w[:1, :1])
    check_turned(dv, w[:1, :1], orc.rotate(w[:1, :1], positions[:1], rotary.inv_freq), 16, False, torch.float32)


def test_rotate_gradient_against_differences(ca):
    """The map is linear, so a difference over any distance is exact but for roundings: L(q + h v) - L(q) over h against the gradient times v."""
    g = torch.Generator().manual_seed(9)
    rotary, which = turn_of(ca, g, 64, 48, 2, True)
    positions = torch.randint(0, 3000, (2, 2, 13), generator=g, dtype=torch.int32).cuda()
    q, v, w = (torch.randn(2, 3, 13, 64, generator=g).cuda() for _ in range(3))
    q.requires_grad_()
    loss = lambda x: (ca.chill_rotate(x, None, positions, rotary)[0].double() * w.double()).sum()  # noqa: E731
    (dq,) = torch.autograd.grad(loss(q), q)
    with torch.no_grad():
        ahead = (loss(q + v) - loss(q)).item()
    along = (dq.double() * v.double()).sum().item()
    size = ((q.detach().abs() + v.abs() + 1) * (w.abs() + 1)).sum().item()
    assert abs(ahead - along) <= 40 * U * size


@pytest.mark.parametrize("dtype,H,Hkv,N,D,page,channels,axes,interleaved,layout", [
    (torch.bfloat16, 8, 2, 1, 128, 64, 128, 1, False, "tokens"),
    (torch.float16, 6, 2, 50, 64, 16, 48, 3, True, "tokens"),
    (torch.float32, 4, 4, 5, 64, 16, 64, 1, False, "heads"),
    (torch.bfloat16, 3, 1, 9, 80, 24, 50, 2, True, "packed"),
    (torch.float16, 2, 2, 3, 32, 5, 32, 1, False, "channels"),
])
@pytest.mark.parametrize("rows_first", [False, True])
def test_rotate_append(ca, dtype, H, Hkv, N, D, page, channels, axes, interleaved, layout, rows_first):
    g = torch.Generator().manual_seed(N + D)
    rotary, which = turn_of(ca, g, D, channels, axes, interleaved)
    lens, new = ints([0, 3 * page - 1, 7]), ints([N, max(N - 2, 0), 0])
    B = 3
    pages = ca.ChillPages.empty(B, 4 * page + N, 40, page)
    ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, 3 * page, page)
    step = ca.chill_pages_reserve(pages, lens, new, N, page)
    if rows_first:  # [num_pages, page, heads, channels] in memory
        k_cache, v_cache = (torch.randn(40, page, Hkv, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    else:
        k_cache, v_cache = (torch.randn(40, Hkv, page, D, generator=g).to(dtype).cuda() for _ in range(2))
    q, k, v = (strided((B, h, N, D), dtype, g, layout) for h in (H, Hkv, Hkv))
    positions = None if axes == 1 else torch.randint(0, 5000, (axes, B, N), generator=g, dtype=torch.int32).cuda()
    at = step.positions if positions is None else positions
    k_before, v_before = k_cache.clone(), v_cache.clone()
    out = ca.chill_rotate_append(q, k, v, k_cache, v_cache, step, rotary, positions)
    check_turned(out, q, orc.rotate(q, at, rotary.inv_freq, which, interleaved), channels // 2, interleaved, dtype)
    slots = step.slots.cpu()
    assert (slots[2] == -1).all() and (slots[0] >= 0).all()
    b, i = (slots >= 0).nonzero(as_tuple=True)
    where = slots[b, i].long()
    stored = k_cache[where // page, :, where % page].transpose(0, 1)[None]  # [1, heads, tokens, channels]
    turned = orc.rotate(k, at, rotary.inv_freq, which, interleaved)[b, :, i].transpose(0, 1)[None]
    check_turned(stored, k[b, :, i].transpose(0, 1)[None], turned, channels // 2, interleaved, dtype)
    assert torch.equal(v_cache[where // page, :, where % page], v[b, :, i])
    for cache, before in ((k_cache, k_before), (v_cache, v_before)):  # everything else is as it was
        cache[where // page, :, where % page] = before[where // page, :, where % page]
        assert torch.equal(cache, before)
    # the two calls one after the other give the same
    k2, v2 = k_before.clone(), v_before.clone()
    q2, turned_k = ca.chill_rotate(q, k, at, rotary)
    ca.chill_cache_append(k2, v2, turned_k, v, step.slots)
    ca.chill_rotate_append(q, k, v, k_cache, v_cache, step, rotary, positions)
    assert torch.equal(out, q2) and torch.equal(k_cache, k2) and torch.equal(v_cache, v2)


# ------------------------------------------------------------------------------------------------------------ selection
def score_bound(x, c):
    """x: a row of logits, c: scores, in 64 bits.  A term of the sum: difference to the maximum and its product with log2 e (2 u of d each way), exponential 2^-22, a thread's
    32 terms in two sums 17 u, rescaled up to 16 times at 2^-22 each; d counts by its weight, E[d] <= log V + spread, taken as 40.  The result is rounded to fp32."""
    return 17 * 2.0 ** -22 + 17 * U + 2 * 40 * U + U * c.abs()


def check_select(out, logits, scores, count, finished=None, end=0):
    want, rows, tokens = orc.select(logits.cpu(), scores.cpu(), count, None if finished is None else finished.cpu(), end)
    got = out.scores.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and (got[got.isinf()] == want[want.isinf()]).all()
    fine = want.isfinite()
    bound = score_bound(logits, want)
    assert ((got - want).abs()[fine] <= bound[fine]).all(), ((got - want).abs() / bound)[fine].max()
    same = (out.parents.cpu() == rows) & (out.tokens.cpu() == tokens)
    if not same.all():  # only where two candidates of different beams are nearer than the bound
        G, K = scores.shape
        for g, m in (~same).nonzero().tolist():
            near = [(want[g, m] - want[g, n]).abs() <= 2 * bound[g, m] for n in (m - 1, m + 1) if 0 <= n < count]
            assert any(near) or m == count - 1, (g, m)
            assert rows[g, m] != out.parents[g, m].item() or tokens[g, m] == out.tokens[g, m].item()
    return want, rows, tokens


SELECTIONS = [
    # dtype, groups, beams, count, vocab
    (torch.float32, 1, 1, 1, 1), (torch.float32, 3, 1, 1, 100), (torch.float32, 1, 4, 4, 32000), (torch.float32, 2, 32, 64, 5003),
    (torch.float32, 5, 3, 6, 257), (torch.float16, 2, 5, 10, 4099), (torch.float16, 7, 64, 64, 129), (torch.float16, 1, 2, 33, 20001),
    (torch.bfloat16, 40, 8, 16, 1000), (torch.bfloat16, 1, 6, 12, 50021), (torch.bfloat16, 2, 16, 32, 16384), (torch.bfloat16, 200, 4, 8, 1111),
    (torch.bfloat16, 1, 1, 64, 64), (torch.float32, 2, 64, 1, 7), (torch.float32, 1, 7, 49, 7),
]


@pytest.mark.parametrize("dtype,G,K,M,V", SELECTIONS)
@pytest.mark.parametrize("kind", ["plain", "banned", "ends"])
def test_select(ca, dtype, G, K, M, V, kind):
    g = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(G * K, V, generator=g) * 2.5).to(dtype).cuda()
    scores = (-30 * torch.rand(G, K, generator=g)).cuda()
    finished = None
    if kind == "banned":
        logits.masked_fill_((torch.rand(G * K, V, generator=g) < 0.3).cuda(), -math.inf)
        scores[:, K // 2 + 1:] = -math.inf
    if kind == "ends":
        finished = (torch.rand(G, K, generator=g) < 0.5).cuda()
        logits[finished.view(-1)] = math.nan  # not looked at
    out = ca.chill_beam_select(logits, scores, M, finished=finished, end_token=V // 2)
    assert out.scores.shape == out.parents.shape == out.tokens.shape == (G, M)
    assert out.scores.dtype == torch.float32 and out.parents.dtype == out.tokens.dtype == torch.int32
    check_select(out, logits, scores, M, finished, V // 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [4096, 4097, 999])
def test_select_ties(ca, dtype, V):
    """Equal logits, equal beams (at addresses of their own), sorted and constant rows: places decide."""
    g = torch.Generator().manual_seed(V)
    few = torch.randint(-3, 3, (6, V), generator=g).to(dtype)
    few[3] = few[1]
    few[5] = few[0]
    scores = torch.tensor([[0.0, -1.0, -0.5, -1.0, -2.0, 0.0]])
    for rows in (few, torch.zeros(6, V, dtype=dtype), few.sort(1).values, few.sort(1, descending=True).values):
        out = ca.chill_beam_select(rows.cuda(), scores.cuda(), 64)
        want, parents, tokens = orc.select(rows, scores, 64)
        assert torch.equal(out.parents.cpu().long(), parents) and torch.equal(out.tokens.cpu().long(), tokens)


def test_select_orders_within_a_beam_by_the_logits_themselves(ca):
    """Neighbouring fp32 logits whose scores round to one number: the larger logit comes first, whatever its place."""
    x = torch.full((1, 1000), -5.0)
    x[0, 100], x[0, 200], x[0, 300] = 1.0, 1.0 + 2 ** -23, 1.0 + 2 ** -22
    out = ca.chill_beam_select(x.cuda(), torch.tensor([[-300.0]]).cuda(), 3)
    assert out.tokens.tolist() == [[300, 200, 100]] and out.scores[0, 0] == out.scores[0, 2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_select_extremes(ca, dtype):
    low, V = torch.finfo(dtype).min, 777
    g = torch.Generator().manual_seed(1)
    x = torch.randn(8, V, generator=g).to(dtype)
    x[0] = low                      # nothing but the lowest value: all alike
    x[1, 5:] = low                  # a mask of the lowest value
    x[2] = -math.inf                # nothing at all
    x[3, 40] = math.nan
    x[4, 9], x[4, :3] = math.inf, -math.inf
    x[5, 1:] = -math.inf            # one token
    x[6] = torch.finfo(dtype).max
    for beams in ([0], [1], [2], [5], [6], [7], [0, 1, 2], [3, 7], [7, 4], [3, 4], [2, 5], list(range(8))):
        rows, scores = x[beams], torch.linspace(-3, -1, len(beams))[None]
        for M in (1, 4, 40):
            out = ca.chill_beam_select(rows.cuda(), scores.cuda(), M)
            want, parents, tokens = orc.select(rows, scores, M)
            assert torch.equal(out.parents.cpu().long(), parents), (beams, M)
            assert torch.equal(out.tokens.cpu().long(), tokens), (beams, M)
            check_select(out, rows, scores, M)
    for s in (math.nan, math.inf, -math.inf):
        scores = torch.tensor([[-1.0, s]])
        out = ca.chill_beam_select(x[[7, 7]].cuda(), scores.cuda(), 5)
        want, parents, tokens = orc.select(x[[7, 7]], scores, 5)
        assert torch.equal(out.parents.cpu().long(), parents) and torch.equal(out.tokens.cpu().long(), tokens)
        assert torch.equal(out.scores.cpu().isnan(), want.isnan())
        over = torch.tensor([[False, True]])
        out = ca.chill_beam_select(x[[7, 7]].cuda(), scores.cuda(), 5, finished=over.cuda(), end_token=3)
        want, parents, tokens = orc.select(x[[7, 7]], scores, 5, over, 3)
        assert torch.equal(out.parents.cpu().long(), parents) and torch.equal(out.tokens.cpu().long(), tokens)


@pytest.mark.parametrize("dtype,V,M", [(torch.float32, 40000, 64), (torch.bfloat16, 70001, 5), (torch.float16, 33000, 33)])
def test_select_of_rows_in_order(ca, dtype, V, M):
    """Ascending, descending and constant rows and steps: what is kept runs over again and again."""
    up = torch.arange(V, dtype=torch.float64) / V * 8 - 4
    rows = torch.stack([up, up.flip(0), torch.zeros(V, dtype=torch.float64), (up * 3).floor(), torch.where(torch.arange(V) % 7 == 0, up, -math.inf)]).to(dtype)
    for beams in ([0], [1], [2], [3], [4], [0, 1, 2, 3, 4]):
        scores = torch.zeros(1, len(beams))
        out = ca.chill_beam_select(rows[beams].cuda(), scores.cuda(), M)
        want, parents, tokens = orc.select(rows[beams], scores, M)
        if len(beams) == 1:
            assert torch.equal(out.tokens.cpu().long(), tokens)
        check_select(out, rows[beams], scores, M)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 140000), (torch.float32, 70001)])
def test_select_of_many_long_rows(ca, dtype, V):
    """More rows than the GPU has room for at once: a row is one segment, and that of several rounds."""
    g = torch.Generator(device="cuda").manual_seed(V)
    G, K, M = 11, 60, 7
    logits = (torch.randn(G * K, V, generator=g, device="cuda") * 2.5).to(dtype)
    logits[3 * K + 1] = logits[3 * K + 1].sort().values
    scores = -5 * torch.rand(G, K, generator=g, device="cuda")
    out = ca.chill_beam_select(logits, scores, M)
    for group in (0, 3, 10):
        part = ca.ChillBeams(out.scores[group:group + 1], out.parents[group:group + 1] - group * K, out.tokens[group:group + 1])
        check_select(part, logits[group * K:(group + 1) * K], scores[group:group + 1], M)


def test_select_of_strided_rows(ca):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(6, 1200, generator=g).cuda()
    for offset, V in ((0, 1000), (1, 1000), (3, 1001), (0, 1)):
        rows = wide[:, offset:offset + V]
        out = ca.chill_beam_select(rows, torch.zeros(2, 3, device="cuda"), 3)
        check_select(out, rows, torch.zeros(2, 3), 3)


# ------------------------------------------------------------------------------------------------------------ pages
def check_pages(pages, shared, table, held, stack, counts):
    assert pages.table.tolist() == table and pages.held.tolist() == held
    n = pages.n_free.item()
    assert n == len(stack) and pages.free.tolist()[:n] == stack
    if shared is not None:
        assert shared.tolist() == counts


def copies_of(copies):
    n = copies.count.item()
    assert copies.source[n:].tolist() == [-1] * (copies.source.numel() - n) == copies.target[n:].tolist() and not copies.rows[n:].any()
    return list(zip(copies.source[:n].tolist(), copies.target[:n].tolist(), copies.rows[:n].tolist()))


def state_of(pages, shared):
    return pages.table.tolist(), pages.held.tolist(), pages.free.tolist(), pages.n_free.item(), shared.tolist()


@pytest.mark.parametrize("B,ctx,page,num_pages,seed", [
    (1, 40, 16, 10, 0), (4, 700, 16, 260, 1), (6, 100, 5, 160, 2), (3, 30, 1, 100, 3), (40, 200, 8, 1200, 4), (70, 3000, 16, 14000, 5), (600, 20, 4, 4000, 6),
    (4, 60, 16, 17, 7), (12, 90, 8, 70, 8), (24, 5000, 1, 40000, 9), (9, 20000, 2, 60000, 10),
])
def test_fork_trim_and_compact(ca, B, ctx, page, num_pages, seed):
    """A run of forks with tokens in between, cuts and compactions; where there are few pages some rows get none."""
    g = torch.Generator().manual_seed(seed)
    pages = ca.ChillPages.empty(B, ctx + 40, num_pages, page)
    shared = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    stored = torch.empty_like(lens)
    first = torch.randint(0, ctx, (B,), generator=g, dtype=torch.int32).cuda()
    first[1:] = torch.where(torch.rand(B - 1, generator=g).cuda() < 0.5, first[1:], 0)  # some are empty to begin with
    ca.chill_pages_reserve(pages, lens, first, ctx, page, stored=stored)
    lens = stored.clone()
    for turn in range(7):
        parents = torch.randint(-1, B, (B,), generator=g, dtype=torch.int32)
        if turn % 3 == 1:
            parents = torch.where(torch.rand(B, generator=g) < 0.6, torch.arange(B, dtype=torch.int32), parents)
        if turn == 4:
            parents = torch.full((B,), int(parents[0]), dtype=torch.int32)  # all from one (or from none)
        before = state_of(pages, shared)
        table, held, stack, counts, missing, out, orders = orc.fork(*before[:4], before[4], lens.tolist(), parents.tolist(), page)
        lens, copies = ca.chill_pages_fork(pages, shared, lens, parents.cuda(), page)
        check_pages(pages, shared, table, held, stack, counts)
        assert lens.tolist() == out and pages.missing.item() == missing and copies_of(copies) == orders
        if turn % 2:  # cut back, inside shared pages too
            lens = (lens.float() * torch.rand(B, generator=g).cuda()).int()
            before = state_of(pages, shared)
            table, held, stack, counts = orc.trim_shared(*before, lens.tolist(), page)
            ca.chill_pages_trim(pages, lens, page, shared=shared)
            check_pages(pages, shared, table, held, stack, counts)
            before = state_of(pages, shared)
            table, stack, counts, moves = orc.compact(*before, num_pages)
            copies = ca.chill_pages_compact(pages, page, shared=shared)
            check_pages(pages, shared, table, held, stack, counts)
            assert copies_of(copies) == [(a, b, page) for a, b in moves]
            lens, copies = ca.chill_pages_fork(pages, shared, lens, torch.arange(B, dtype=torch.int32, device="cuda"), page)  # pages to write to
        more = torch.randint(0, 12, (B,), generator=g, dtype=torch.int32).cuda()
        more = torch.minimum(more, pages.table.shape[1] * page - lens)
        ca.chill_pages_reserve(pages, lens, more, 12, page, stored=stored)
        lens = lens + stored
        counts = {}
        for row, h in zip(pages.table.tolist(), pages.held.tolist()):
            for q in row[:h]:
                counts[q] = counts.get(q, 0) + 1
        on_stack = pages.free.tolist()[:pages.n_free.item()]
        assert not set(counts) & set(on_stack) and len(counts) + len(on_stack) == num_pages and len(set(on_stack)) == len(on_stack)
        assert shared.tolist() == [counts.get(q, 1) - 1 for q in range(num_pages)]


def test_compact_without_shares_and_at_the_ends(ca):
    for used in (0, 1, 5, 8):
        pages = ca.ChillPages.empty(1, 32, 8, 4)
        lens = ints([4 * used])
        ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, 32, 4)
        copies = ca.chill_pages_compact(pages, 4)
        assert copies.count.item() == 0 and pages.table.tolist()[0][:used] == list(range(used)) and pages.n_free.item() == 8 - used
    pages = ca.ChillPages.empty(2, 4, 1, 4)
    ca.chill_pages_reserve(pages, ints([0, 0]), ints([1, 0]), 1, 4)
    assert copies_of(ca.chill_pages_compact(pages, 4)) == []


def test_bad_pages_and_lengths_do_no_harm(ca):
    """Tables with entries that are no pages, lengths and counts that are nonsense: nothing outside is written (what was there stays), and what is whole works."""
    B, page, num_pages, width = 4, 4, 20, 6
    room = torch.full((B + 2, width + 3), 77, dtype=torch.int32, device="cuda")
    table = room[1:B + 1, :width]
    table.copy_(ints([[0, 1, 99, -7, -1, -1], [2, 3, -1, -1, -1, -1], [4, 4, 4, -1, -1, -1], [5, 6, 7, 8, 9, 10]]))
    held, free = ints([4, 900, 3, -3]), torch.full((num_pages + 8,), 55, dtype=torch.int32, device="cuda")
    free[4:4 + num_pages] = torch.arange(num_pages, dtype=torch.int32, device="cuda")
    counts = torch.full((num_pages + 8,), 66, dtype=torch.int32, device="cuda")
    counts[4:4 + num_pages] = 0
    pages = ca.ChillPages(table, held, free[4:4 + num_pages], ints([500]), ints([0]))
    for parents in ([1, 0, -9, 2 ** 31 - 1], [3, 3, 3, 3], [0, 1, 2, 3], [-1, -1, -1, -1]):
        lens, copies = ca.chill_pages_fork(pages, counts[4:4 + num_pages], ints([15, 2 ** 31 - 1, -4, 10]), ints(parents), page)
        ca.chill_pages_trim(pages, ints([3, -5, 2 ** 31 - 1, 0]), page, shared=counts[4:4 + num_pages])
        ca.chill_pages_compact(pages, page, shared=counts[4:4 + num_pages])
        torch.cuda.synchronize()
        assert (room[0] == 77).all() and (room[-1] == 77).all() and (room[:, width:] == 77).all()
        assert (free[:4] == 55).all() and (free[-4:] == 55).all() and (counts[:4] == 66).all() and (counts[-4:] == 66).all()
        assert 0 <= pages.n_free.item() <= num_pages and ((pages.held >= 0) & (pages.held <= width)).all() and (lens >= 0).all()


# ------------------------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("dtype,layers,Hkv,page,D,rows_first", [
    (torch.bfloat16, 0, 8, 16, 128, False), (torch.float16, 3, 2, 16, 64, True), (torch.float32, 2, 1, 5, 20, False), (torch.bfloat16, 1, 3, 7, 33, False),
    (torch.float16, 0, 1, 256, 256, True), (torch.float32, 1, 2, 1, 4, False),
])
def test_cache_copy(ca, dtype, layers, Hkv, page, D, rows_first):
    g = torch.Generator().manual_seed(D)
    num_pages = 50
    shape = (max(layers, 1), num_pages, page, Hkv, D) if rows_first else (max(layers, 1), num_pages, Hkv, page, D)
    k_cache, v_cache = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
    if rows_first:
        k_cache, v_cache = k_cache.transpose(2, 3), v_cache.transpose(2, 3)
    if not layers:
        k_cache, v_cache = k_cache[0], v_cache[0]
    order = torch.randperm(num_pages, generator=g)[:24].tolist()
    source, target = order[:12], order[12:]
    rows = torch.randint(-1, page + 2, (12,), generator=g).tolist()
    source[3], target[5] = -1, num_pages  # no pages
    for count in (0, 1, 9, 12, 500, -4):
        expected = [k_cache.clone(), v_cache.clone()]
        for a, b, n in list(zip(source, target, rows))[:max(count, 0)]:
            if a >= 0 and b < num_pages:
                for x in expected:
                    x[..., b, :, :max(n, 0), :] = x[..., a, :, :max(n, 0), :]
        ca.chill_cache_copy(k_cache, v_cache, ca.ChillCopies(ints(source), ints(target), ints(rows), ints([count])))
        assert torch.equal(k_cache, expected[0]) and torch.equal(v_cache, expected[1]), count


def test_cache_copy_of_one_tensor(ca):
    cache = torch.randn(9, 2, 8, 64, device="cuda")
    expected = cache.clone()
    expected[7, :, :5] = expected[2, :, :5]
    ca.chill_cache_copy(cache, cache, ca.ChillCopies(ints([2]), ints([7]), ints([5]), ints([1])))
    assert torch.equal(cache, expected)


@pytest.mark.parametrize("dtype,V", [(torch.float32, 5000), (torch.bfloat16, 40001)])
def test_select_of_one_row_for_all_beams(ca, dtype, V):
    """Rows no elements apart, and rows that overlap: equal beams are ties, the lowest first."""
    row = torch.randn(V + 40, generator=torch.Generator().manual_seed(V)).to(dtype)
    for step in (0, 1, 8):
        rows = row.cuda().as_strided((6, V), (step, 1))
        scores = torch.tensor([[-1.0, 0.0, 0.0], [0.0, 0.0, -0.5]])
        out = ca.chill_beam_select(rows, scores.cuda(), 7)
        want, parents, tokens = orc.select(rows.cpu(), scores, 7)
        assert torch.equal(out.parents.cpu().long(), parents) and torch.equal(out.tokens.cpu().long(), tokens)
        check_select(out, rows, scores, 7)


@pytest.mark.parametrize("mark", [-1e9, torch.finfo(torch.float32).min])
def test_select_with_marks_for_missing_beams(ca, mark):
    """The first step with a low score instead of -inf for the beams that are not there yet."""
    g = torch.Generator().manual_seed(4)
    logits = (torch.randn(8, 3001, generator=g) * 2).bfloat16()
    scores = torch.full((2, 4), mark)
    scores[:, 0] = 0
    out = ca.chill_beam_select(logits.cuda(), scores.cuda(), 8)
    check_select(out, logits, scores, 8)
    assert (out.parents.cpu() == torch.tensor([[0], [4]])).all()


@pytest.mark.parametrize("K,M,V", [(4, 64, 500), (4, 64, 20), (3, 17, 30000), (40, 64, 700), (40, 64, 3), (64, 5, 9000)])
@pytest.mark.parametrize("score", [-2.0 ** 50, -1e30, torch.finfo(torch.float32).min])
def test_select_where_scores_hide_the_logits(ca, K, M, V, score):
    """Scores so large that 64 bits round a beam's candidates to few numbers, or to one: the lowest beam, then the largest logit, then the lowest token comes first."""
    g = torch.Generator().manual_seed(V)
    row = torch.randint(-12, 12, (V,), generator=g) / 4.0
    rows = torch.stack([row[torch.randperm(V, generator=g)] for _ in range(K)])  # one row in several orders, for one sum
    scores = torch.full((1, K), score)
    scores[0, K // 2] *= 0.5
    beam, token = torch.arange(K)[:, None].expand(K, V).flatten(), torch.arange(V).repeat(K)
    value = scores[0].double()[:, None] + (rows.double() - torch.logsumexp(row.double(), 0))
    order = sorted(range(K * V), key=lambda n: (-value.flatten()[n].item(), beam[n].item(), -rows.flatten()[n].item(), n)) if K * V <= 4000 else None
    if order is None:  # stable sorts, the last key first
        order = torch.arange(K * V)
        for key in (-rows.flatten(), beam, -value.flatten()):
            order = order[key[order].sort(stable=True).indices]
    order = torch.as_tensor(order)[:M]
    out = ca.chill_beam_select(rows.cuda(), scores.cuda(), M)
    assert out.parents[0].tolist() == beam[order].tolist() and out.tokens[0].tolist() == token[order].tolist()
    assert torch.equal(out.scores[0].cpu(), value.flatten()[order].float())


def test_select_of_the_largest_vocabulary(ca):
    V = 2 ** 26
    x = torch.zeros(2, V, dtype=torch.bfloat16, device="cuda")
    places = [(0, V - 1, 30.0), (1, 0, 29.0), (1, V - 1, 28.0), (0, V // 2, 27.0)]
    for beam, token, value in places:
        x[beam, token] = value
    out = ca.chill_beam_select(x, torch.zeros(1, 2, device="cuda"), 4)
    lse = [math.log((V - 2) + sum(math.exp(v) for b, _, v in places if b == beam)) for beam in range(2)]
    want = sorted(((v - lse[b], b, t) for b, t, v in places), reverse=True)
    assert list(zip(out.parents[0].tolist(), out.tokens[0].tolist())) == [(b, t) for _, b, t in want]
    # half a step of fp32, of the results; a batch's 32 terms of at most 1 are added up in fp32 (2^-19 of their sum, below 2^-26 of the whole)
    assert all(abs(got - w[0]) <= 2.0 ** -24 * abs(w[0]) + 2.0 ** -18 for got, w in zip(out.scores[0].tolist(), want))


def test_fork_of_the_largest_batch(ca):
    """8192 requests, every other one twice, in a cluster; shared memory beyond the default limit."""
    B, page = 8192, 4
    pages, shared = ca.ChillPages.empty(B, 24, 5 * B, page), torch.zeros(5 * B, dtype=torch.int32, device="cuda")
    lens = torch.arange(B, dtype=torch.int32, device="cuda") % 14 + 1
    ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, 14, page)
    before = state_of(pages, shared)
    parents = torch.arange(B, dtype=torch.int32, device="cuda") // 2 * 2
    table, held, stack, counts, missing, out, orders = orc.fork(*before, lens.tolist(), parents.tolist(), page)
    lens, copies = ca.chill_pages_fork(pages, shared, lens, parents, page)
    check_pages(pages, shared, table, held, stack, counts)
    assert lens.tolist() == out and copies_of(copies) == orders and missing == pages.missing.item() == 0
