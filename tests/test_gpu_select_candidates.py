"""The candidates that a selection returns, each by its own value: what is returned at a place has that place's score, is nobody else's, and within a beam the order is exact."""
import math

import pytest
import torch

from test_gpu_decode import SELECTIONS, U, score_bound


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


def values_of(logits, scores, finished, end):
    """[groups, beams, vocab] in 64 bits; finite rows, or rows of nothing but -inf."""
    G, K = scores.shape
    x = logits.detach().cpu().double().view(G, K, -1)
    lse = torch.logsumexp(x, 2, keepdim=True)
    c = torch.where(x == -math.inf, -math.inf, scores.cpu().double()[..., None] + (x - lse))
    c[scores.cpu() == -math.inf] = -math.inf
    if finished is not None:
        over = finished.cpu()
        c[over] = -math.inf
        c[..., end][over] = scores.cpu().double()[over]
    return c


def check_candidates(out, logits, scores, count, finished=None, end=0):
    """The kernel's value of a candidate is off by the bound at most (its last part, U |c|, is the rounding of what is written), so the m-th of its order is worth the m-th largest
    value but for twice that."""
    G, K = scores.shape
    V = logits.shape[1]
    c = values_of(logits, scores, finished, end)
    parents, tokens, got = out.parents.cpu().long(), out.tokens.cpu().long(), out.scores.cpu().double()
    beams = parents - torch.arange(G)[:, None] * K
    assert ((beams >= 0) & (beams < K) & (tokens >= 0) & (tokens < V)).all()
    places = beams * V + tokens
    assert all(len(set(row.tolist())) == count for row in places)
    own, want = c.view(G, -1).gather(1, places), c.view(G, -1).topk(count, dim=1).values
    assert torch.equal(own == -math.inf, want == -math.inf) and torch.equal(got == -math.inf, want == -math.inf)
    fine = want.isfinite()
    bound = score_bound(logits, want)
    apart = bound - U * want.abs()
    assert ((own - want).abs()[fine] <= 2 * apart[fine] + 2.0 ** -50 * want.abs()[fine]).all()
    assert ((got - own).abs()[fine] <= bound[fine]).all()
    x = logits.detach().cpu().double().view(G, K, V)
    for g in range(G):
        for k in range(K):
            mine = tokens[g][fine[g] & (beams[g] == k)]
            if finished is not None and finished[g, k]:
                assert mine.tolist() in ([], [end])
            else:
                assert torch.equal(mine, x[g, k].sort(descending=True, stable=True).indices[:mine.numel()])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,G,K,M,V", SELECTIONS + [(torch.float32, 3, 64, 1, 1000), (torch.bfloat16, 6, 8, 1, 30000), (torch.float16, 1, 3, 1, 9)])
@pytest.mark.parametrize("kind", ["plain", "banned", "ends"])
def test_each_candidate(ca, dtype, G, K, M, V, kind):
    g = torch.Generator().manual_seed(V + 3 * K)
    logits = (torch.randn(G * K, V, generator=g) * 2.5).to(dtype).cuda()
    scores = (-30 * torch.rand(G, K, generator=g)).cuda()
    finished = None
    if kind == "banned":
        logits.masked_fill_((torch.rand(G * K, V, generator=g) < 0.3).cuda(), -math.inf)
        scores[:, K // 2 + 1:] = -math.inf
    if kind == "ends":
        finished = (torch.rand(G, K, generator=g) < 0.5).cuda()
    out = ca.chill_beam_select(logits, scores, M, finished=finished, end_token=V // 2)
    check_candidates(out, logits, scores, M, finished, V // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_close_beams(ca, shift):
    """Beams whose scores and rows are nearly alike, so that candidates of different beams lie side by side."""
    g = torch.Generator().manual_seed(8)
    row = torch.randn(1, 20011, generator=g) * 2
    logits = (row + 1e-3 * torch.randn(12, 20011, generator=g)).bfloat16()
    wide = torch.zeros(12, 20011 + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, shift:shift + 20011] = logits.cuda()
    scores = -1 - 1e-3 * torch.rand(2, 6, generator=g)
    check_candidates(ca.chill_beam_select(wide[:, shift:shift + 20011], scores.cuda(), 40), logits, scores, 40)


def test_the_check_finds_mistakes():
    """Wrong tokens, wrong beams, exchanged and repeated candidates, at any place, the last one too."""
    g = torch.Generator().manual_seed(2)
    logits, scores = torch.randn(4, 50, generator=g), torch.tensor([[-1.0, -1.5], [-0.5, -0.25]])
    from oracle import decode_oracle as orc
    from types import SimpleNamespace

    for count in (1, 5):
        want, rows, tokens = orc.select(logits, scores, count)
        good = dict(scores=want.float(), parents=rows.int(), tokens=tokens.int())
        check_candidates(SimpleNamespace(**good), logits, scores, count)
        for m in {0, count - 1}:
            for name, change in (("tokens", lambda x: (x + 1) % 50), ("parents", lambda x: x ^ 1), ("scores", lambda x: x + 1e-4)):
                bad = {n: t.clone() for n, t in good.items()}
                bad[name][1, m] = change(bad[name][1, m])
                with pytest.raises(AssertionError):
                    check_candidates(SimpleNamespace(**bad), logits, scores, count)
        if count > 1:
            bad = {n: t.clone() for n, t in good.items()}
            for t in bad.values():
                t[0, -1] = t[0, -2]
            with pytest.raises(AssertionError):
                check_candidates(SimpleNamespace(**bad), logits, scores, count)
