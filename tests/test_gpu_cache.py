"""Paged cache on the GPU: pages, storing, attention of new tokens, accepted paths; against the 64-bit oracle."""
import pytest
import torch

from cache_helpers import Problem, check_attention, masks
from helpers import ensure_built
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    ensure_built()
    from chill_attention import _cache_abi

    lib = _cache_abi.load_library()
    yield lib
    assert lib.chill_cache_read_device_status() == 0


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def strided(t, layout):
    """The same values with other strides."""
    t = t.cuda()
    if layout == "transposed":  # [.., head, row, channel] kept as [.., row, head, channel]
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "padded":      # rows 16-byte aligned, with gaps of NaN
        wide = torch.full((*t.shape[:3], t.shape[3] + 16), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., :t.shape[3]] = t
        return wide[..., :t.shape[3]]
    if layout == "odd":         # channels two apart, base not aligned
        wide = torch.full((*t.shape[:3], 2 * t.shape[3] + 1), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., 1::2] = t
        return wide[..., 1::2]
    return t


def attend(p, mask, layout="plain", flags=0):
    from chill_attention import cache

    scale = p.q.shape[3] ** -0.5
    q, k, v = (strided(t, layout) for t in (p.q, p.k_cache, p.v_cache))
    return cache._attention(q, k, v, p.table.cuda(), p.step(), mask, scale, True, flags), scale


def kernel_of(p, flags=0):
    """Which kernel serves the contiguous call."""
    import ctypes

    from chill_attention import _cabi, _cache_abi

    B, H, N, D = p.q.shape
    a = _cache_abi.CachedArgs()
    a.mask = _cabi.mask_desc(_cabi.MASK_CAUSAL, ())
    a.B, a.H, a.H_kv, a.N, a.D, a.dtype = B, H, p.k_cache.shape[1], N, D, _cabi._DTYPES[p.dtype]
    a.page_size, a.num_pages, a.table_width, a.sm_scale, a.flags = p.page, p.k_cache.shape[0], p.table.shape[1], 1.0, flags
    a.q = a.k_cache = a.v_cache = a.o = a.table = a.lens = a.new_lens = 4096
    for name, t in (("q_strides", p.q), ("o_strides", p.q), ("k_cache_strides", p.k_cache), ("v_cache_strides", p.v_cache)):
        setattr(a, name, (ctypes.c_int64 * 4)(*t.stride()))
    return _cache_abi.load_library().chill_cached_kernel(ctypes.byref(a))


def run_and_check(p, mask, layout="plain", flags=0):
    (o, lse), scale = attend(p, mask, layout, flags)
    assert o.shape == p.q.shape and o.is_contiguous()
    from chill_attention import _cache_abi

    tensor_cores = layout not in ("odd",) and kernel_of(p, flags) != _cache_abi.CACHED_CUDA_CORES
    check_attention(o, lse, p, mask, scale, tensor_cores)
    return o, lse


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
RAGGED = [300, 0, 1, 64, 63, 129, 17, 200]


# Keys the tables have room for: up to 512 every CTA takes whole (request, kv head) units; beyond that the work is cut into shares.
ROOMS = {"whole": 0, "shares": 600}


@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("kind", ["one", "chain", "tree"])
@pytest.mark.parametrize("mask", list(masks()))
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_masks_and_ragged_lengths(dtype, mask, kind, room):
    N = 1 if kind == "one" else 9
    new = [N, N, 0, max(N - 2, 1), N, 1, N, 0]
    p = Problem(dtype, 6, 2, 64, RAGGED, new, N, 16, tree=kind == "tree", seed=len(mask) + N, room=ROOMS[room])
    run_and_check(p, masks()[mask])


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_head_dims_and_groups(dtype, room, group, D):
    p = Problem(dtype, 2 * group, 2, D, [70, 3, 128, 0], [5, 2, 5, 5], 5, 32, tree=group != 3, seed=D + group, room=ROOMS[room])
    run_and_check(p, masks()["causal"])


@pytest.mark.parametrize("layout", ["transposed", "padded", "odd"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_strides(dtype, layout):
    for N, D in ((3, 64), (40, 128)):
        p = Problem(dtype, 8, 2, D, [90, 31, 64], [N, N - 1, N], N, 16, tree=True, seed=D, room=600 if N == 3 else 0)
        run_and_check(p, masks()["window"], layout)
        if D == 128:
            run_and_check(Problem(dtype, 8, 2, D, [90, 31, 64], [N, N - 1, N], N, 16, tree=True, seed=D, room=600), masks()["window"], layout)


@pytest.mark.parametrize("page", [1, 5, 8, 16, 48, 64, 100, 128, 512])
def test_page_sizes(page):
    for N, dtype in ((2, torch.bfloat16), (33, torch.float16)):
        for room in ROOMS.values():
            p = Problem(dtype, 4, 2, 64, [257, 40, 0, 99], [N, 1, N, N], N, page, tree=True, seed=page, room=room)
            run_and_check(p, masks()["causal"])


@pytest.mark.parametrize("N", [15, 16, 17, 31, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_row_tiles(kind, N):
    for D, dtype, room in ((64, torch.bfloat16, 600), (128, torch.float16, 600), (256, torch.bfloat16, 600), (128, torch.bfloat16, 0)):
        p = Problem(dtype, 4, 1, D, [150, 10, 64], [N, N - 3, 1], N, 64, tree=kind == "tree", seed=N, room=room)
        run_and_check(p, masks()["window_ahead" if N % 2 else "causal"])


@pytest.mark.parametrize("N", [9, 16, 17, 31, 33, 70])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_row_tiles_on_the_cuda_cores(kind, N):
    """Tiles of 16 and of 32 rows, every head dim, pages that are no multiple of anything."""
    for D, dtype, page, room in ((16, torch.float32, 16, 600), (32, torch.float32, 48, 0), (64, torch.bfloat16, 5, 600),
                                 (64, torch.float32, 7, 600), (128, torch.float32, 64, 600), (256, torch.float32, 5, 600), (256, torch.float16, 3, 0)):
        p = Problem(dtype, 4, 4, D, [150, 10, 64], [N, N - 3, 1], N, page, tree=kind == "tree", seed=N, room=room)
        run_and_check(p, masks()["window_ahead" if N % 2 else "causal"])


@pytest.mark.parametrize("N", [6, 12, 20])
def test_many_whole_units_on_the_cuda_cores(N):
    """Short tables and more units than the SMs have few of: tiles of 8, 16 and 32 rows, each by one CTA."""
    lens = [(37 * b) % 90 for b in range(80)]
    new = [N - b % 3 for b in range(80)]
    run_and_check(Problem(torch.float32, 8, 8, 32, lens, new, N, 16, tree=True, seed=N), masks()["causal"])


@pytest.mark.parametrize("G", [5, 7, 48, 100, 128, 130])
def test_groups_that_do_not_divide_a_tile(G):
    """Tiles of rows hold whole tokens: 125, 126, 96, 100 and 128 of 128 rows; a token with more goes elsewhere."""
    from chill_attention import _cache_abi

    p = Problem(torch.bfloat16, 2 * G, 2, 64, [150, 70], [9, 6], 9, 16, tree=True, seed=G, room=600)
    assert kernel_of(p) == (_cache_abi.CACHED_ROWS if G == 130 else _cache_abi.CACHED_TILES)
    run_and_check(p, masks()["causal"])


@pytest.mark.parametrize("G", [1, 2])
@pytest.mark.parametrize("D", [32, 128, 256])
def test_many_rows_of_few_heads(D, G):
    p = Problem(torch.bfloat16, 2 * G, 2, D, [100, 0, 400], [130, 70, 129], 130, 32, tree=G == 2, seed=G, room=600)
    run_and_check(p, masks()["chunkwise"])


def test_which_kernel_serves_a_call():
    from chill_attention import _cabi, _cache_abi

    def ask(dtype=torch.bfloat16, H=4, Hkv=2, D=64, N=1, page=16, flags=0):
        return kernel_of(Problem(dtype, H, Hkv, D, [10], [N], N, page), flags)

    for D in (16, 32, 64, 128):
        assert ask(D=D) == ask(D=D, N=16) == _cache_abi.CACHED_ROWS and ask(D=D, N=17) == _cache_abi.CACHED_TILES  # 32 rows at most
    assert ask(D=256, N=8) == _cache_abi.CACHED_ROWS and ask(D=256, N=9) == _cache_abi.CACHED_TILES              # 16
    assert ask(dtype=torch.float32) == ask(page=12) == ask(page=1) == ask(flags=_cabi.FLAG_FORCE_GENERIC) == _cache_abi.CACHED_CUDA_CORES
    assert ask(page=8) == ask(page=24) == _cache_abi.CACHED_ROWS


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_one_long_request_is_split(dtype):
    for N in (1, 6, 70):
        p = Problem(dtype, 4, 1, 64, [5000], [N], N, 64, tree=N == 6, seed=N)
        run_and_check(p, masks()["causal"])


def test_sharp_scores_over_many_parts():
    """Scores of tens: parts whose maxima differ by hundreds of powers of two."""
    p = Problem(torch.float16, 8, 2, 128, [3000, 2000], [4, 4], 4, 32, tree=True, seed=4, sharp=16.0)
    run_and_check(p, masks()["causal"])


@pytest.mark.parametrize("room", list(ROOMS))
def test_many_short_requests(room):
    """More (request, tile of rows) pairs than every CTA sums up by itself."""
    B = 1100
    p = Problem(torch.bfloat16, 2, 1, 64, [(7 * b) % 40 for b in range(B)], [(b % 3) for b in range(B)], 2, 16, seed=1, room=ROOMS[room])
    run_and_check(p, masks()["causal"])


@pytest.mark.parametrize("dtype,N,D", [(torch.bfloat16, 1, 64), (torch.float16, 5, 64), (torch.float32, 1, 16)], ids=str)
def test_small_shares_for_whoever_is_done_first(dtype, N, D):
    """Enough keys (24 tiles of 64 for each CTA) that the last sixth of them is handed out as the CTAs get done."""
    lens = [57000, 120, 61000, 40000, 58000, 90]
    heads = 6 if dtype == torch.float32 else 4
    p = Problem(dtype, heads, heads, D, lens, [N] * 6, N, 64, tree=N > 1, seed=D, room=62000)
    o, lse = run_and_check(p, masks()["causal"])
    (again, _), _ = attend(p, masks()["causal"])
    assert torch.equal(o, again)  # whoever had them
    short = Problem(dtype, 4, 4, D, [300, 20], [N] * 2, N, 64, seed=D, room=400000)  # room for as many, few there
    run_and_check(short, masks()["causal"])


@pytest.mark.parametrize("name", ["full", "causal"])
def test_a_batch_with_mixed_steps(name):
    """Prompts, single tokens and idle requests in one call: tiles of rows that hold no token."""
    p = Problem(torch.float16, 8, 2, 128, [0, 700, 30, 0, 256], [150, 1, 0, 3, 64], 150, 16, seed=8)
    run_and_check(p, masks()[name])


@pytest.mark.parametrize("N", [2, 40])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_keys_without_a_page_are_not_there(dtype, N):
    holes = [(0, 0, -1), (0, 3, 10 ** 6), (1, 0, -1), (1, 1, -7), (1, 2, -1), (1, 3, 2 ** 30), (1, 4, -1), (2, 2, -2 ** 31)]
    for room in ROOMS.values():
        p = Problem(dtype, 4, 2, 64, [130, 30, 80], [N, N, N], N, 16, tree=True, seed=9, holes=holes, room=room)
        o, lse = run_and_check(p, masks()["causal"])
    q = Problem(dtype, 4, 2, 64, [130, 30], [N, N], N, 16, seed=9, holes=[(b, j, -1) for b in (0, 1) for j in range((130 if b == 0 else 30) // 16 + 1 + N // 16)])
    o, lse = run_and_check(q, masks()["causal"])
    if N == 2:
        assert torch.isneginf(lse).all() and (o == 0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")], ids=str)
@pytest.mark.parametrize("kind,N", [("tree", 9), ("tree", 70), ("chain", 9), ("chain", 70)])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_what_hidden_keys_hold_does_not_matter(dtype, kind, N, value):
    """Keys and values that are not finite reach the rows that see them and no others."""
    mask = masks()["causal" if kind == "tree" else "window"]
    p = Problem(dtype, 4, 2, 64, [150, 64, 3000], [N, N - 1, N], N, 16, tree=kind == "tree", seed=N)
    clean = p.k_cache.clone(), p.v_cache.clone()
    poisoned = [[1, 4], [0], [2]] if kind == "tree" else [[-30, 1], [-36], [-35, -1]]  # new tokens; below zero: cached ones before them
    sees = torch.zeros(3, N, dtype=torch.bool)
    for b, keys in enumerate(poisoned):
        c = p.lens[b]
        for n, j in enumerate(keys):
            page, row = int(p.table[b, (c + j) // 16]), (c + j) % 16
            p.v_cache[page, :, row, 3] = value
            if n == 0:
                p.k_cache[page, 1, row] = value
            for i in range(p.new[b]):
                sees[b, i] |= j in p.sets[b][i] if kind == "tree" else i - 37 <= j <= i
    assert sees.any() and not sees.all()
    (o, lse), scale = attend(p, mask)
    o_cpu = o.cpu()
    for b in range(3):
        for i in range(p.new[b]):
            if sees[b, i]:
                assert not torch.isfinite(o_cpu[b, :, i, 3]).any()
    p.k_cache, p.v_cache = clean
    check_attention(o, lse, p, mask, scale, dtype != torch.float32, rows=~sees)


def test_lengths_beyond_the_table_and_below_zero():
    p = Problem(torch.bfloat16, 4, 2, 64, [60, 50, 20], [8, 8, 8], 8, 16, seed=2)
    from chill_attention import ChillStep, chill_attention_cached

    s = p.step()
    step = ChillStep(ints([10 ** 9, -5, 20]), ints([10 ** 9, -3, 2 ** 31 - 1]), s.slots, s.positions, None)
    o, lse = chill_attention_cached(p.q.cuda(), p.k_cache.nan_to_num(0.5).cuda(), p.v_cache.nan_to_num(0.5).cuda(), p.table.cuda(), step, masks()["causal"],
                                    return_lse=True)
    assert torch.isfinite(o).all() and (o[1] == 0).all() and (lse[1] == 0).all()
    want, _ = chill_attention_cached(p.q.cuda(), p.k_cache.nan_to_num(0.5).cuda(), p.v_cache.nan_to_num(0.5).cuda(), p.table.cuda(), s, masks()["causal"],
                                     return_lse=True)
    assert torch.equal(o[2], want[2])


def test_same_result_every_time():
    p = Problem(torch.bfloat16, 8, 2, 128, [2500, 900, 100], [6, 6, 2], 6, 64, tree=True, seed=3)
    (a, la), _ = attend(p, masks()["causal"])
    for _ in range(3):
        (b, lb), _ = attend(p, masks()["causal"])
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_custom_mask():
    import os

    import chill_attention as ca

    here = os.path.dirname(os.path.abspath(__file__))

    class DilatedCausalMask(ca.ChillMask):
        cuda_functor_header = os.path.join(here, "custom_masks", "dilated_causal_mask.h")
        cuda_functor = "DilatedCausalMask"

    dilation = 3
    mask = DilatedCausalMask((dilation,))
    p = Problem(torch.float16, 4, 2, 64, [100, 33], [4, 4], 4, 16, seed=5)
    (o, lse), scale = attend(p, mask)
    real = orc.builtin_mask_dense
    orc.builtin_mask_dense = lambda name, args, q, k: (q[:, None] >= k[None]) & ((q[:, None] - k[None]) % dilation == 0)
    try:
        check_attention(o, lse, p, mask, scale, True)
    finally:
        orc.builtin_mask_dense = real


# ------------------------------------------------------------------------------------------------------- pages
def check_pages(pages, table, held, stack, missing=None):
    assert pages.table.tolist() == table and pages.held.tolist() == held
    assert pages.n_free.item() == len(stack) and pages.free[:len(stack)].tolist() == stack
    if missing is not None:
        assert pages.missing.item() == missing


@pytest.mark.parametrize("B,N,page", [(1, 1, 16), (3, 5, 1), (8, 1, 16), (70, 33, 7), (600, 4, 16), (1500, 1, 64), (2, 3000, 16)])
def test_reserve_and_trim_follow_the_oracle(B, N, page):
    import chill_attention as ca

    g = torch.Generator().manual_seed(B + N)
    draw = lambda hi: torch.randint(0, hi + 1, (B,), generator=g).tolist()  # noqa: E731
    num = B * (-(-(60 + N) // page)) * 2 // 3 + 3  # not always enough
    pages = ca.ChillPages.empty(B, 60 + N, num, page)
    table, held, stack = pages.table.tolist(), pages.held.tolist(), pages.free.tolist()
    lens = [0] * B
    for turn in range(4):
        new = draw(N)
        parents = [[int(x) for x in torch.randint(-2, i + 2, (1,), generator=g)] [0] for _ in range(B) for i in range(N)] if turn == 2 and N < 100 else None
        parents = [parents[b * N:(b + 1) * N] for b in range(B)] if parents else None
        step = ca.chill_pages_reserve(pages, ints(lens), ints(new), N, page, ints(parents) if parents else None)
        table, held, n, missing, slots, positions, sets = orc.reserve(table, held, stack, len(stack), lens, new, N, page, parents)
        stack = stack[:n]
        check_pages(pages, table, held, stack, missing)
        assert step.slots.tolist() == slots and step.positions.tolist() == positions
        if parents is None:
            assert step.ancestors is None
        else:
            bits = step.ancestors.cpu()
            for b in range(B):
                for i in range(N):
                    assert {j for j in range(N) if (int(bits[b, i, j // 32]) >> (j % 32)) & 1} == sets[b][i]
        lens = [min(c + n, len(table[0]) * page) if turn != 1 else 0 if b % 3 == 0 else c for b, (c, n) in enumerate(zip(lens, new))]
        lens = [min(c, h * page) for c, h in zip(lens, held)]
        ca.chill_pages_trim(pages, ints(lens), page)
        table, held, stack = orc.trim(table, held, stack, len(stack), lens, page)
        check_pages(pages, table, held, stack)
    ca.chill_pages_trim(pages, ints([0] * B), page)
    assert pages.n_free.item() == num and sorted(pages.free.tolist()) == list(range(num)) and (pages.table == -1).all()


def test_reserve_survives_nonsense():
    import chill_attention as ca

    pages = ca.ChillPages.empty(4, 64, 6, 16)
    step = ca.chill_pages_reserve(pages, ints([-9, 2 ** 31 - 1, 10, 0]), ints([-1, 2 ** 31 - 1, 3, 7]), 8, 16)
    assert pages.held.tolist() == [0, 4, 1, 1] and pages.n_free.item() == 0 and pages.missing.item() == 0
    assert step.slots[0].tolist() == [-1] * 8 and step.slots[1].tolist() == [-1] * 8 and (step.slots[2, :3] >= 0).all()
    pages.held.fill_(100)
    pages.n_free.fill_(1000)
    ca.chill_pages_trim(pages, ints([0, 0, 0, 0]), 16)  # a stack that is full already takes nothing more
    assert pages.n_free.item() == 6 and (pages.table == -1).all()


# -------------------------------------------------------------------------------------------- storing and keeping
@pytest.mark.parametrize("layout", ["plain", "transposed", "padded", "odd"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_append(dtype, layout):
    import chill_attention as ca

    for D, N, page in ((64, 7, 16), (16, 1, 5), (256, 70, 64)):
        p = Problem(dtype, 3, 3, D, [10, 0, 77], [N, 0, N - 1], N, page, seed=D)
        k, v = torch.randn(3, 3, N, D).to(dtype), torch.randn(3, 3, N, D).to(dtype)
        want_k, want_v = p.k_cache.clone(), p.v_cache.clone()
        for b in range(3):
            for i, s in enumerate(p.slots[b]):
                if s >= 0:
                    want_k[s // page, :, s % page], want_v[s // page, :, s % page] = k[b, :, i], v[b, :, i]
        slots = p.step().slots
        slots[1, 0] = p.k_cache.shape[0] * page  # outside the cache
        kc, vc = strided(p.k_cache, layout), strided(p.v_cache, layout)
        ca.chill_cache_append(kc, vc, strided(k, layout), strided(v, layout), slots)
        assert torch.equal(kc.cpu().nan_to_num(7), want_k.nan_to_num(7))
        assert torch.equal(vc.cpu().nan_to_num(7), want_v.nan_to_num(7))


@pytest.mark.parametrize("layout", ["plain", "transposed", "odd"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_commit(dtype, layout):
    import chill_attention as ca

    N, page, lens = 40, 16, [10, 0, 77, 15, 30]
    paths = [[0, 3, 4, 9, 20, 21, 22, 30, 31, 35, 38, 39], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [39] + [0] * 11,
             [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 50], [5, 3, -1, 90, 4, 39, 39, 7, 8, 9, 10, 11]]
    accepted, new = [12, 11, 1, 99, 8], [40, 40, 40, 12, 40]
    for D in (64, 256):
        p = Problem(dtype, 2, 2, D, lens, new, N, page, tree=True, seed=D)
        want_k, want_v = p.k_cache.clone(), p.v_cache.clone()
        for b, c in enumerate(lens):
            for j in range(min(accepted[b], 12, new[b])):
                f = paths[b][j]
                if j < f < new[b]:
                    for w, have in ((want_k, p.k_cache), (want_v, p.v_cache)):
                        w[p.table[b, (c + j) // page], :, (c + j) % page] = have[p.table[b, (c + f) // page], :, (c + f) % page]
        kc, vc = strided(p.k_cache, layout), strided(p.v_cache, layout)
        out = ca.chill_cache_commit(kc, vc, p.table.cuda(), p.step(), ints(paths), ints(accepted))
        assert out.tolist() == [22, 11, 78, 27, 38]
        assert torch.equal(kc.cpu().nan_to_num(7), want_k.nan_to_num(7)) and torch.equal(vc.cpu().nan_to_num(7), want_v.nan_to_num(7))


# ------------------------------------------------------------------------------------------------ the operators together
def run_session(mask, dtype, total, chunks, page, H, Hkv, D, seed=0):
    """A batch of two, fed in chunks through the cache; returns the rows of q, k, v, o as whole sequences."""
    import chill_attention as ca

    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(2, h, total, D, device="cuda", generator=g).to(dtype) for h in (H, Hkv, Hkv))
    pages = ca.ChillPages.empty(2, total, 2 * (-(-total // page)), page)
    kc, vc = (torch.full((2 * (-(-total // page)), Hkv, page, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    lens, parts = ints([0, 0]), []
    at = 0
    for n in chunks:
        new = ints([n, n])
        step = ca.chill_pages_reserve(pages, lens, new, n, page)
        ca.chill_cache_append(kc, vc, k[:, :, at:at + n], v[:, :, at:at + n], step.slots)
        parts.append(ca.chill_attention_cached(q[:, :, at:at + n], kc, vc, pages.table, step, mask, return_lse=True))
        lens = lens + new
        at += n
    assert at == total and pages.missing.item() == 0
    return q, k, v, torch.cat([o for o, _ in parts], 2), torch.cat([s for _, s in parts], 2)


@pytest.mark.parametrize("name", ["causal", "window", "prefix_lm", "chunkwise"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "fp16", "bf16"])
def test_a_sequence_through_the_cache_is_the_sequence_at_once(dtype, name):
    """Chunks of any size and single tokens give what chill_attention gives for the whole sequence (a chunk of a chunkwise mask has to
    come at once, a prefix too)."""
    import chill_attention as ca
    from helpers import O_ATOL

    mask = masks()[name]
    chunks = [24, 48, 24, 72, 24] if name == "chunkwise" else [60, 1, 1, 70, 3, 1, 55, 1]
    q, k, v, o, lse = run_session(mask, dtype, 192, chunks, 16, 4, 2, 64)
    want, want_lse = ca.chill_attention(q, k, v, mask=mask, return_lse=True)
    # both are within the operator's bar of the exact result
    assert (o.float() - want.float()).abs().max().item() <= 2 * O_ATOL[dtype]
    assert (lse - want_lse).abs().max().item() <= 1e-3 * 8


def test_speculative_steps():
    """Trees of drafts, an accepted path kept, the next tree: the cache then holds what feeding the accepted tokens one by one gives, and
    every node's attention is that of its own path as a sequence."""
    import chill_attention as ca

    D, page, N, B = 64, 16, 12, 2
    g = torch.Generator().manual_seed(3)
    pages = ca.ChillPages.empty(B, 200, 40, page)
    kc, vc = (torch.full((40, 2, page, D), float("nan"), device="cuda") for _ in range(2))
    lens = ints([0, 0])
    kept_k, kept_v = [[] for _ in range(B)], [[] for _ in range(B)]
    for turn in range(6):
        parents = [[int(torch.randint(max(-1, i - 3), i, (1,), generator=g)) for i in range(N)] for _ in range(B)]
        new = [N, N - turn]
        q, k, v = torch.randn(B, 4, N, D, generator=g), torch.randn(B, 2, N, D, generator=g), torch.randn(B, 2, N, D, generator=g)
        step = ca.chill_pages_reserve(pages, lens, ints(new), N, page, ints(parents))
        ca.chill_cache_append(kc, vc, k.cuda(), v.cuda(), step.slots)
        o = ca.chill_attention_cached(q.cuda(), kc, vc, pages.table, step, ca.CausalChillMask())
        path, accepted = [], []
        for b in range(B):
            chain = []  # the longest way down to the last real node
            node = new[b] - 1
            while node >= 0:
                chain.append(node)
                node = parents[b][node]
            chain = chain[::-1]
            if chain:  # attention of the path's last node, from the kept tokens and its own path alone
                ks = torch.stack(kept_k[b] + [k[b, :, i] for i in chain], 1).double()
                vs = torch.stack(kept_v[b] + [v[b, :, i] for i in chain], 1).double()
                for h in range(4):
                    w = torch.softmax(ks[h // 2] @ q[b, h, chain[-1]].double() * D ** -0.5, 0)
                    assert ((w @ vs[h // 2]) - o[b, h, chain[-1]].cpu().double()).abs().max() < 1e-5
            take = min(len(chain), turn + 1)
            path.append((chain + [0] * N)[:N])
            accepted.append(take)
            kept_k[b] += [k[b, :, i] for i in chain[:take]]
            kept_v[b] += [v[b, :, i] for i in chain[:take]]
        lens = ca.chill_cache_commit(kc, vc, pages.table, step, ints(path), ints(accepted))
        assert lens.tolist() == [len(x) for x in kept_k]
        ca.chill_pages_trim(pages, lens, page)
        assert pages.held.tolist() == [-(-len(x) // page) for x in kept_k]
    for b in range(B):
        for t, (x, y) in enumerate(zip(kept_k[b], kept_v[b])):
            where = int(pages.table[b, t // page])
            assert torch.equal(kc[where, :, t % page].cpu(), x) and torch.equal(vc[where, :, t % page].cpu(), y)


def test_a_captured_step_is_replayed_with_other_lengths():
    """One graph of all operators; lengths, tokens and pages change between replays, two graphs are alive at once."""
    import chill_attention as ca

    D, page, N, B = 64, 16, 4, 3
    mask = ca.CausalChillMask()

    class Session:
        def __init__(self):
            self.pages = ca.ChillPages.empty(B, 400, 80, page)
            self.kc, self.vc = (torch.full((80, 2, page, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            self.lens, self.new = ints([0] * B), ints([N] * B)
            self.q, self.k, self.v = (torch.zeros(B, h, N, D, dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2))

        def pass_(self):
            step = ca.chill_pages_reserve(self.pages, self.lens, self.new, N, page)
            ca.chill_cache_append(self.kc, self.vc, self.k, self.v, step.slots)
            o = ca.chill_attention_cached(self.q, self.kc, self.vc, self.pages.table, step, mask)
            self.lens.add_(self.new)
            return o

        def reset(self):
            ca.chill_pages_trim(self.pages, ints([0] * B), page)
            self.lens.zero_()
            self.kc.fill_(float("nan"))
            self.vc.fill_(float("nan"))

    eager, one, two = Session(), Session(), Session()
    graphs = []
    for s in (one, two):
        s.pass_()  # warm-up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = s.pass_()
        s.reset()
        graphs.append((s, graph, o))
    for turn in range(20):
        data = [torch.randn_like(t) for t in (eager.q, eager.k, eager.v)]
        new = ints([turn % (N + 1), N, (3 * turn) % (N + 1)])
        for s in (eager, one, two):
            for t, d in zip((s.q, s.k, s.v), data):
                t.copy_(d)
            s.new.copy_(new)
        want = eager.pass_()
        for s, graph, o in graphs:
            graph.replay()
        for s, graph, o in graphs:
            assert torch.equal(o, want) and torch.equal(s.lens, eager.lens) and torch.equal(s.pages.table, eager.pages.table)


def test_a_call_can_be_captured_before_any_ran():
    import os
    import subprocess
    import sys

    from helpers import ROOT

    code = """
import sys; sys.path[:0] = [%r, %r, %r]
import torch, chill_attention as ca
from cache_helpers import Problem
for N, dtype in ((1, torch.bfloat16), (40, torch.float16), (1, torch.float32)):
    p = Problem(dtype, 4, 2, 64, [900, 20], [N, N], N, 16, seed=N)
    args = [p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step(), ca.CausalChillMask()]
    pages, lens = ca.ChillPages.empty(2, 100, 20, 16), torch.zeros(2, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ca.chill_attention_cached(*args)
        step = ca.chill_pages_reserve(pages, lens, args[4].new_lens, N, 16)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, ca.chill_attention_cached(*args)) and (step.slots >= 0).all()
print("captured")
""" % (os.path.join(ROOT, "chill-attention_b200"), ROOT, os.path.join(ROOT, "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_a_compiled_step():
    import chill_attention as ca

    p = Problem(torch.bfloat16, 8, 2, 64, [250, 90], [6, 5], 6, 16, tree=True, seed=3, room=600)
    mask = masks()["window"]
    q, table, parents = p.q.cuda(), p.table.cuda(), ints(p.parents)
    k, v = torch.randn(2, 2, 6, 64, device="cuda", dtype=torch.bfloat16), torch.randn(2, 2, 6, 64, device="cuda", dtype=torch.bfloat16)
    path, accepted = ints([[0, 2, 5], [1, 3, 4]]), ints([2, 3])

    def step(pages, kc, vc, lens, new):
        s = ca.chill_pages_reserve(pages, lens, new, 6, 16, parents)
        ca.chill_cache_append(kc, vc, k, v, s.slots)
        o, lse = ca.chill_attention_cached(q, kc, vc, pages.table, s, mask, return_lse=True)
        lens = ca.chill_cache_commit(kc, vc, pages.table, s, path, accepted)
        ca.chill_pages_trim(pages, lens, 16)
        return o, lse, lens

    def state():
        pages = ca.ChillPages(table.clone(), ints(p.held), ints(p.spare_pages + [-1] * (p.k_cache.shape[0] - len(p.spare_pages))), ints([len(p.spare_pages)]), ints([0]))
        return pages, p.k_cache.nan_to_num(0.25).cuda(), p.v_cache.nan_to_num(0.25).cuda(), ints(p.lens), ints(p.new)

    a, b = state(), state()
    want = step(*a)
    got = torch.compile(step, fullgraph=True)(*b)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert all(torch.equal(x, y) for x, y in zip([*a[0], a[1], a[2]], [*b[0], b[1], b[2]]))


def test_caches_with_more_than_two_to_the_31_elements():
    """Pages whose offsets do not fit 32 bits, in elements and in bytes."""
    import chill_attention as ca

    page, Hkv, D, B, N = 64, 8, 64, 2, 3
    pages = 2 ** 31 // (page * Hkv * D) + 40
    kc, vc = (torch.empty(pages, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    high = list(range(pages - 8, pages))
    for tree in (False, True):
        p = Problem(torch.float16, 16, Hkv, D, [100, 130], [N, N], N, page, tree=tree, seed=1, room=600)
        where = {int(x): high[i] for i, x in enumerate(sorted(set(p.table[p.table >= 0].tolist())))}
        for a, b in where.items():
            kc[b], vc[b] = p.k_cache[a].cuda(), p.v_cache[a].cuda()
        table = torch.tensor([[where.get(x, -1) for x in row] for row in p.table.tolist()], dtype=torch.int32, device="cuda")
        for flags in (0, 1):
            from chill_attention import cache

            o, lse = cache._attention(p.q.cuda(), kc, vc, table, p.step(), masks()["causal"], D ** -0.5, True, flags)
            check_attention(o, lse, p, masks()["causal"], D ** -0.5, flags == 0)
        step = p.step()
        slots = ints([[where[s // page] * page + s % page for s in row] for row in p.slots])
        k, v = (torch.randn(B, Hkv, N, D, device="cuda").half() for _ in range(2))
        ca.chill_cache_append(kc, vc, k, v, slots)
        out = ca.chill_cache_commit(kc, vc, table, step, ints([[1, 2], [2, 2]]), ints([2, 1]))
        assert out.tolist() == [102, 131]
        for b, path in ((0, [1, 2, 2]), (1, [2, 1, 2])):
            for i, f in enumerate(path):
                s = int(slots[b, i])
                assert torch.equal(kc[s // page, :, s % page], k[b, :, f]) and torch.equal(vc[s // page, :, s % page], v[b, :, f])


def test_another_stream():
    import chill_attention as ca

    p = Problem(torch.bfloat16, 8, 2, 128, [2500, 900], [6, 6], 6, 64, tree=True, seed=3)
    args = [p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step(), ca.CausalChillMask()]
    want = ca.chill_attention_cached(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for turn in range(4):
        for s in streams:  # calls that can overlap: each has a workspace of its own
            with torch.cuda.stream(s):
                outs.append(ca.chill_attention_cached(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_dispatcher_ops_give_the_same():
    from chill_attention import cache

    p = Problem(torch.float16, 8, 2, 64, [250, 90], [6, 5], 6, 16, tree=True, seed=3)
    mask = masks()["window"]
    (o, lse), scale = attend(p, mask)
    s = p.step()
    o2, lse2 = torch.ops.chill_attention.cached_forward(p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), s.lens, s.new_lens, s.positions,
                                                        s.ancestors, mask.name, list(mask.constargs), scale, 0)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    import chill_attention as ca

    a, b = (ca.ChillPages.empty(2, 300, 50, 16) for _ in range(2))
    want = ca.chill_pages_reserve(a, s.lens, s.new_lens, 6, 16, ints(p.parents))
    got = torch.ops.chill_attention.pages_reserve(*b, s.lens, s.new_lens, 6, 16, ints(p.parents))
    assert all(torch.equal(x, y) for x, y in zip(want[2:], got)) and all(torch.equal(x, y) for x, y in zip(a, b))
    torch.library.opcheck(torch.ops.chill_attention.cache_append.default,
                          (p.k_cache.cuda(), p.v_cache.cuda(), torch.randn(2, 2, 6, 64).half().cuda(), torch.randn(2, 2, 6, 64).half().cuda(), s.slots),
                          test_utils=("test_schema", "test_faketensor"))
    assert cache._MASKS[mask.name][1] >= 0


def test_refusals():
    import chill_attention as ca

    p = Problem(torch.bfloat16, 4, 2, 64, [40, 20], [3, 3], 3, 16, tree=True, seed=1)
    q, kc, vc, table, step, mask = p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step(), ca.CausalChillMask()
    call = ca.chill_attention_cached
    bad = [
        (q.half(), kc, vc, table, step), (q[:, :3], kc, vc, table, step), (q, kc, vc[1:], table, step), (q, kc.float(), vc, table, step),
        (q, kc, vc, table.long(), step), (q, kc, vc, table[:1], step), (q[..., :48], kc[..., :48], vc[..., :48], table, step), (q[:0], kc, vc, table[:0], step),
        (q, kc, vc, table, step._replace(lens=step.lens.long())), (q, kc, vc, table, step._replace(new_lens=step.new_lens[:1])),
        (q, kc, vc, table, step._replace(positions=step.positions[:, :2])), (q, kc, vc, table, step._replace(ancestors=step.ancestors[..., :0])),
        (q, kc, vc, table, step._replace(lens=step.lens.cpu())), (q.cpu(), kc, vc, table, step),
        (q.clone().requires_grad_(True), kc, vc, table, step),
    ]
    for args in bad:
        with pytest.raises(AssertionError):
            call(*args, mask)
    with torch.no_grad():
        call(q.clone().requires_grad_(True), kc, vc, table, step, mask)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="invalid argument"):
            call(q, kc, vc, table, step, mask, sm_scale=scale)
    k = torch.randn(2, 2, 3, 64, device="cuda", dtype=torch.bfloat16)
    for args in [(kc, vc, k.float(), k, step.slots), (kc, vc, k[:, :1], k[:, :1], step.slots), (kc, vc, k, k, step.slots.long()),
                 (kc, vc, k, k, step.slots[:, :2]), (kc, vc, k.clone().requires_grad_(True), k, step.slots)]:
        with pytest.raises(AssertionError):
            ca.chill_cache_append(*args)
    path, accepted = ints([[0, 1], [0, 2]]), ints([1, 2])
    for args in [(kc, vc, table, step, path[:1], accepted), (kc, vc, table, step, path, accepted.long()), (kc, vc, table, step, path[:, :0], accepted)]:
        with pytest.raises(AssertionError):
            ca.chill_cache_commit(*args)
    pages = ca.ChillPages.empty(2, 100, 8, 16)
    for args in [(pages, step.lens.long(), step.new_lens, 3, 16), (pages, step.lens, step.new_lens[:1], 3, 16), (pages, step.lens, step.new_lens, 0, 16),
                 (pages, step.lens, step.new_lens, 3, 0), (pages, step.lens, step.new_lens, 3, 16, ints([[0, 1], [0, 1]])),
                 (pages._replace(held=pages.held[:1]), step.lens, step.new_lens, 3, 16)]:
        with pytest.raises(AssertionError):
            ca.chill_pages_reserve(*args)
    with pytest.raises(AssertionError):
        ca.chill_pages_trim(pages, step.lens[:1], 16)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")], ids=str)
@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("dtype,N,D,page", [(torch.bfloat16, 9, 64, 16), (torch.float16, 9, 128, 16), (torch.bfloat16, 70, 64, 16), (torch.float16, 70, 128, 16),
                                            (torch.bfloat16, 20, 256, 16), (torch.float32, 1, 64, 16), (torch.float32, 9, 64, 16), (torch.bfloat16, 9, 64, 5)], ids=str)
def test_a_score_that_is_not_finite_shows(dtype, N, D, page, room, value):
    """One key, seen by every row and not finite in K alone, at each of the 64 places of a tile: scores of NaN or +inf leave nothing finite in a
    row of O, one of -inf is a weight of 0, and the rows of the other kv head know nothing of it."""
    p = Problem(dtype, 4, 2, D, [200] * 64, [N] * 64, N, page, seed=N, room=ROOMS[room])
    for b in range(64):
        where, row = int(p.table[b, (64 + b) // page]), (64 + b) % page
        p.k_cache[where, 1, row, b % D] = value
    (o, lse), scale = attend(p, masks()["causal"])
    o_ref = p.oracle(masks()["causal"], scale)[0]
    finite = torch.isfinite(o_ref).all(-1)  # [batch, head, token]
    assert finite[:, :2].all() and (value == float("-inf") or not finite[:, 2:].all())
    gone = ~finite.cuda()
    assert not torch.isfinite(o[gone]).any() and not torch.isfinite(lse[gone]).any()
    clean = Clean(p, finite)
    check_attention(*(torch.where(finite.cuda().view(*finite.shape, *[1] * (x.ndim - 3)), x, 0) for x in (o, lse)), clean, masks()["causal"], scale, dtype != torch.float32)


class Clean:
    """A problem whose rows outside of `finite` [batch, head, token] are zeros on both sides; scores of -inf have no part in the bound."""

    def __init__(self, problem, finite):
        self.q, self.new, self.N, self.dtype, self.v_cache = problem.q, problem.new, problem.N, problem.dtype, problem.v_cache
        self.problem, self.finite = problem, finite

    def oracle(self, mask, scale):
        o, lse, size, _, keys = self.problem.oracle(mask, scale)
        k = self.problem.k_cache
        self.problem.k_cache = torch.where(torch.isfinite(k), k, 0)
        most = self.problem.oracle(mask, scale)[3]
        self.problem.k_cache = k
        return tuple(torch.where(self.finite.view(*self.finite.shape, *[1] * (x.ndim - 3)), x, 0) for x in (o, lse, size, most, keys))


@pytest.mark.parametrize("dtype,N,D", [(torch.bfloat16, 9, 64), (torch.bfloat16, 70, 64), (torch.float16, 70, 128), (torch.float32, 9, 64)], ids=str)
def test_scores_of_minus_infinity_everywhere(dtype, N, D):
    """Every key of a kv head is -inf in a channel in which the rows are positive: nothing is left for these rows, as where nothing is seen."""
    p = Problem(dtype, 4, 2, D, [200, 130], [N, N], N, 16, seed=N)
    p.k_cache[:, 1, :, 3] = float("-inf")
    p.q[:, 2:, :, 3] = p.q[:, 2:, :, 3].abs() + 0.25
    (o, lse), _ = attend(p, masks()["causal"])
    assert (o[:, 2:] == 0).all() and torch.isneginf(lse[:, 2:]).all()
    assert torch.isfinite(o[:, :2]).all() and torch.isfinite(lse[:, :2]).all()


def test_a_repair_may_take_longer_than_a_wait(_lib):
    """A key that is not finite, behind 400,000 others: its rows are worked out again key by key for seconds, which the other warps of the CTA
    have to sit out.  The other request, whose turn comes after it in the same CTA, is served as if nothing had been."""
    import chill_attention as ca

    H, N, D, page, lens = 64, 256, 64, 64, [400000, 3000]
    blocks = [-(-(c + N) // page) for c in lens]
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.randn(sum(blocks), 1, page, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    table = torch.full((2, max(blocks)), -1, dtype=torch.int32, device="cuda")
    table[0], table[1, :blocks[1]] = torch.arange(blocks[0]), torch.arange(blocks[0], sum(blocks))
    q = torch.randn(2, H, N, D, device="cuda", dtype=torch.bfloat16, generator=g)
    positions = ints(lens)[:, None] + torch.arange(N, device="cuda", dtype=torch.int32)
    step = ca.ChillStep(ints(lens), ints([N, N]), positions, positions, None)
    want, want_lse = ca.chill_attention_cached(q, kc, vc, table, step, ca.CausalChillMask(), return_lse=True)
    kc[399990 // page, 0, 399990 % page] = float("nan")
    o, lse = ca.chill_attention_cached(q, kc, vc, table, step, ca.CausalChillMask(), return_lse=True)
    assert torch.equal(o[1], want[1]) and torch.equal(lse[1], want_lse[1])
    assert torch.isnan(o[0]).all() and torch.isnan(lse[0]).all()
    assert _lib.chill_cache_read_device_status() == 0


def test_a_session_that_runs_short_of_pages():
    """Request 1 gets too few pages, request 0 leaves, request 1 goes on with what it was short of: its rows are those of a session that never
    ran short, and nothing of request 0 is among its keys."""
    import chill_attention as ca
    from helpers import O_ATOL

    page, D, total = 16, 64, 40
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(2, h, total, D, device="cuda", generator=g) for h in (4, 2, 2))
    want = ca.chill_attention(q, k, v, mask=ca.CausalChillMask())
    pages = ca.ChillPages.empty(2, 64, 4, page)
    kc, vc = (torch.full((4, 2, page, D), 50.0, device="cuda") for _ in range(2))
    lens, done = ints([0, 0]), [0, 0]
    stored, got = [], ints([-9, -9])
    for turn, new in enumerate([(20, 10), (12, 30), (0, 8)]):
        N = max(new)
        row = lambda t: torch.stack([torch.nn.functional.pad(t[b, :, done[b]:done[b] + new[b]], (0, 0, 0, N - t[b, :, done[b]:done[b] + new[b]].shape[1])) for b in range(2)])  # noqa: E731
        step = ca.chill_pages_reserve(pages, lens, ints(new), N, page, stored=got)
        stored.append(got.tolist())
        assert stored[-1] == (step.slots >= 0).sum(1).tolist()
        ca.chill_cache_append(kc, vc, row(k), row(v), step.slots)
        o = ca.chill_attention_cached(row(q), kc, vc, pages.table, step, ca.CausalChillMask())
        for b, n in enumerate(stored[-1]):
            if n > 0:  # both are within the operator's bar of the exact result
                assert (o[b, :, :n] - want[b, :, done[b]:done[b] + n]).abs().max() <= 2 * O_ATOL[torch.float32]
            done[b] += n
        lens = lens + got
        assert lens.tolist() == done
        if turn == 1:
            assert pages.missing.item() == 1
            lens, done = lens * ints([0, 1]), [0, done[1]]
            ca.chill_pages_trim(pages, lens, page)
    assert stored == [[20, 10], [12, 22], [0, 8]] and done == [0, total]


@pytest.mark.parametrize("B,N,page", [(3, 5, 1), (70, 33, 7), (300, 40, 16)])
def test_stored_counts_the_slots(B, N, page):
    import chill_attention as ca

    g = torch.Generator().manual_seed(B)
    draw = lambda hi: torch.randint(0, hi + 1, (B,), generator=g).tolist()  # noqa: E731
    for num in (1, B * (20 + N) // page // 2 + 1, B * (-(-(20 + N) // page))):
        pages = ca.ChillPages.empty(B, 10 + N, num, page)  # some tables are full too
        for parents in (None, torch.full((B, N), -1, dtype=torch.int32, device="cuda")):
            stored = torch.full((B,), -9, dtype=torch.int32, device="cuda")
            step = ca.chill_pages_reserve(pages, ints(draw(20)), ints(draw(N)), N, page, parents, stored)
            assert stored.tolist() == (step.slots >= 0).sum(1).tolist()


def test_commit_ends_before_the_first_token_without_a_page():
    import chill_attention as ca

    page, D = 16, 64
    pages = ca.ChillPages.empty(3, 64, 3, page)
    kc, vc = (torch.full((3, 1, page, D), 9.0, device="cuda") for _ in range(2))
    stored = ints([0, 0, 0])
    ca.chill_pages_reserve(pages, ints([0, 0, 0]), ints([10, 14, 14]), 14, page, stored=stored)
    assert stored.tolist() == [10, 14, 14]
    step = ca.chill_pages_reserve(pages, ints([10, 14, 14]), ints([4, 6, 6]), 6, page, ints([[-1] * 6] * 3), stored)
    assert stored.tolist() == [4, 2, 2] and pages.missing.item() == 2
    k = torch.arange(18, device="cuda", dtype=torch.float32).view(3, 1, 6, 1).expand(3, 1, 6, D)
    ca.chill_cache_append(kc, vc, k, -k, step.slots)
    lens = ca.chill_cache_commit(kc, vc, pages.table, step, ints([[1, 3, 5], [0, 1, 2], [1, 4, 5]]), ints([2, 3, 3]))
    assert lens.tolist() == [12, 16, 15]
    rows = lambda b, t: kc[int(pages.table[b, t // page]), 0, t % page, 0].item()  # noqa: E731
    assert [rows(0, 10), rows(0, 11)] == [1, 3] and [rows(1, 14), rows(1, 15)] == [6, 7] and rows(2, 14) == 13


@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("D,N", [(32, 2), (64, 2), (64, 13), (128, 2), (128, 13), (256, 2)])
def test_many_pieces_one_after_the_other(D, N, room):
    """Every CTA of the kernel for few rows joins its warps' states where the Q of the piece after the next one goes."""
    from chill_attention import _cache_abi

    B = 1000
    p = Problem(torch.bfloat16, 2, 1, D, [(11 * b) % 70 for b in range(B)], [N - b % 2 for b in range(B)], N, 16, tree=N > 2, seed=D, room=ROOMS[room])
    assert kernel_of(p) == _cache_abi.CACHED_ROWS
    o, lse = run_and_check(p, masks()["causal"])
    for _ in range(3):
        (again, lse_again), _ = attend(p, masks()["causal"])
        assert torch.equal(o, again) and torch.equal(lse, lse_again)


def test_sizes_beyond_32_bits_are_refused():
    """Not cut to their low bits: one page of memory that stands for 2^32 + 1 of them, and so on."""
    import chill_attention as ca

    p = Problem(torch.bfloat16, 4, 2, 64, [40, 20], [3, 3], 3, 16, tree=True, seed=1)
    q, kc, vc, table, step = p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step()
    pages, lens, far = ca.ChillPages.empty(2, 100, 8, 16), ints([0, 0]), 2 ** 32 + 1
    many = kc[:1].expand(far, -1, -1, -1)
    path = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for call in (lambda: ca.chill_attention_cached(q, many, many, table, step, ca.CausalChillMask()),
                 lambda: ca.chill_cache_append(many, many, kc[:2, :, :3], kc[:2, :, :3], step.slots),
                 lambda: ca.chill_cache_commit(many, many, table, step, ints([[0], [0]]), ints([1, 1])),
                 lambda: ca.chill_cache_commit(kc, vc, table, step, path.expand(2, far), ints([1, 1])),
                 lambda: ca.chill_attention_cached(q[:, :, :1].expand(-1, -1, far, -1), kc, vc, table, step, ca.CausalChillMask()),
                 lambda: ca.chill_pages_reserve(pages, lens, lens, far, 16), lambda: ca.chill_pages_reserve(pages, lens, lens, 1, far),
                 lambda: ca.chill_pages_trim(pages, lens, far), lambda: ca.chill_pages_trim(pages._replace(free=path[0].expand(far)), lens, 16),
                 lambda: ca.chill_pages_trim(pages._replace(table=path.expand(2, far)), lens, 16)):
        with pytest.raises(AssertionError):
            call()


def test_autograd_notices_what_is_changed_in_place():
    import chill_attention as ca

    kc, vc = (torch.zeros(4, 1, 16, 64, device="cuda") for _ in range(2))
    w = torch.ones(64, device="cuda", requires_grad=True)
    new = torch.randn(1, 1, 3, 64, device="cuda")
    pages, lens = ca.ChillPages.empty(1, 64, 4, 16), ints([0])

    def versions():
        return [t._version for t in (*pages, kc, vc)]

    before = versions()
    step = ca.chill_pages_reserve(pages, lens, ints([3]), 3, 16, ints([[-1, 0, 0]]))
    reserved = versions()
    assert all(a > b for a, b in zip(reserved[:5], before[:5])) and reserved[5:] == before[5:]
    y = (kc * w).sum()  # saves kc
    ca.chill_cache_append(kc, vc, new, new, step.slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    appended = versions()
    assert appended[:5] == reserved[:5] and all(a > b for a, b in zip(appended[5:], reserved[5:]))
    lens = ca.chill_cache_commit(kc, vc, pages.table, step, ints([[0, 2]]), ints([2]))
    committed = versions()
    assert all(a > b for a, b in zip(committed[5:], appended[5:]))
    ca.chill_pages_trim(pages, lens, 16)
    assert all(a > b for a, b in zip(versions()[:4], committed[:4]))
    with torch.inference_mode():  # tensors without a version
        kc, vc = torch.zeros_like(kc), torch.zeros_like(vc)
    ca.chill_cache_append(kc, vc, new, new, step.slots)
    assert torch.equal(kc[int(pages.table[0, 0]), 0, :3], new[0, 0])


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    """Forward-mode derivatives are not dropped without a word, not under no_grad either."""
    import chill_attention as ca
    from torch.autograd import forward_ad

    p = Problem(torch.float32, 4, 2, 64, [40, 20], [3, 3], 3, 16, tree=True, seed=1)
    q, kc, vc, table, step = p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step()
    k, path, accepted = torch.randn(2, 2, 3, 64, device="cuda"), ints([[0, 1], [0, 2]]), ints([1, 2])
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))  # noqa: E731
        for call in (lambda: ca.chill_attention_cached(dual(q), kc, vc, table, step, ca.CausalChillMask()),
                     lambda: ca.chill_attention_cached(q, kc, dual(vc), table, step, ca.CausalChillMask()),
                     lambda: ca.chill_cache_append(kc, vc, dual(k), k, step.slots), lambda: ca.chill_cache_append(dual(kc), vc, k, k, step.slots),
                     lambda: ca.chill_cache_commit(kc, dual(vc), table, step, path, accepted)):
            with pytest.raises(AssertionError, match="tangents"):
                call()
        ca.chill_attention_cached(q, kc, vc, table, step, ca.CausalChillMask())


def test_a_tensor_that_watches_its_operators():
    """A subclass sees the dispatcher op whichever argument it is."""
    import chill_attention as ca

    class Watching(torch.Tensor):
        seen = []

        @staticmethod
        def __new__(cls, held):
            t = torch.Tensor._make_subclass(cls, held)
            t.held = held
            return t

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            cls.seen.append(str(func))
            return func(*(a.held if isinstance(a, cls) else a for a in args), **(kwargs or {}))

    p = Problem(torch.bfloat16, 4, 2, 64, [40, 20], [3, 3], 3, 16, tree=True, seed=1)
    q, kc, vc, table, step = p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step()
    want = ca.chill_attention_cached(q, kc, vc, table, step, ca.CausalChillMask())
    for changed in ((Watching(q), step), (q, step._replace(positions=Watching(step.positions))), (q, step._replace(ancestors=Watching(step.ancestors)))):
        Watching.seen.clear()
        o = ca.chill_attention_cached(changed[0], kc, vc, table, changed[1], ca.CausalChillMask())
        assert any("cached_forward" in name for name in Watching.seen) and torch.equal(o, want)
    for lens, parents in ((Watching(ints([0, 0])), ints(p.parents)), (ints([0, 0]), Watching(ints(p.parents)))):
        Watching.seen.clear()
        got = ca.chill_pages_reserve(ca.ChillPages.empty(2, 100, 8, 16), lens, step.new_lens, 3, 16, parents)
        assert any("pages_reserve" in name for name in Watching.seen) and (got.slots >= 0).all()


@pytest.mark.parametrize("name,status", [("libchill_cache_b200.so", "chill_cache_read_device_status"), ("libchill_b200.so", "chill_read_device_status")])
def test_the_status_word_after_a_reset_of_the_device(name, status):
    """A process that resets its device (its own context alone) finds the word again."""
    import glob
    import os
    import subprocess
    import sys

    from chill_attention import _cabi

    runtime = glob.glob(os.path.join(os.path.dirname(os.path.dirname(torch.__file__)), "nvidia", "cuda_runtime", "lib", "libcudart.so.*"))
    if not runtime:
        pytest.skip("no shared CUDA runtime")
    code = f"""
import ctypes
read = getattr(ctypes.CDLL({os.path.join(_cabi.LIB_DIR, name)!r}), {status!r})
runtime = ctypes.CDLL({runtime[0]!r})
print(read(), runtime.cudaDeviceReset(), read(), read())
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.stdout.split() == ["0"] * 4, r.stdout + r.stderr[-2000:]


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_commit_of_one_tensor_for_keys_and_values(layout):
    """Each row moves once, also along a path whose rows are sources after they were targets."""
    import chill_attention as ca

    N, D, lens = 40, 256, [10, 0, 77]
    paths, accepted = [list(range(1, 21)), list(range(0, 40, 2)), list(range(20, 40))], [20, 20, 20]
    p = Problem(torch.bfloat16, 2, 2, D, lens, [N] * 3, N, 16, tree=True, seed=1)
    want = p.k_cache.clone()
    for b, c in enumerate(lens):
        for j, f in enumerate(paths[b]):
            want[p.table[b, (c + j) // 16], :, (c + j) % 16] = p.k_cache[p.table[b, (c + f) // 16], :, (c + f) % 16]
    for _ in range(5):
        cache = strided(p.k_cache, layout).clone() if layout == "plain" else strided(p.k_cache, layout)
        assert ca.chill_cache_commit(cache, cache, p.table.cuda(), p.step(), ints(paths), ints(accepted)).tolist() == [30, 20, 97]
        assert torch.equal(cache.cpu().nan_to_num(7), want.nan_to_num(7))


def test_nothing_of_a_call_comes_after_it():
    """A table with room for small shares and few keys there: the kernel that clears their counter is waited for, so what takes the
    workspace's memory next keeps its bytes."""
    import ctypes

    from chill_attention import _cabi, _cache_abi

    p = Problem(torch.bfloat16, 4, 4, 64, [300, 20], [2] * 2, 2, 64, tree=True, seed=5, room=400000)
    a = _cache_abi.CachedArgs()
    a.mask = _cabi.mask_desc(_cabi.MASK_CAUSAL, ())
    a.B, a.H, a.H_kv, a.N, a.D, a.dtype, a.page_size, a.num_pages, a.table_width, a.sm_scale = 2, 4, 4, 2, 64, 2, 64, p.k_cache.shape[0], p.table.shape[1], 1.0
    for name, t in (("q_strides", p.q), ("k_cache_strides", p.k_cache), ("v_cache_strides", p.v_cache)):
        setattr(a, name, (ctypes.c_int64 * 4)(*t.stride()))
    size = _cache_abi.load_library().chill_cached_workspace_bytes(ctypes.byref(a))
    assert size > 0
    args = p.q.cuda(), p.k_cache.cuda(), p.v_cache.cuda(), p.table.cuda(), p.step(), masks()["causal"]
    import chill_attention as ca

    want = ca.chill_attention_cached(*args)
    for _ in range(50):
        o = ca.chill_attention_cached(*args)
        behind = torch.full((size,), 7, dtype=torch.uint8, device="cuda")
        assert (behind == 7).all() and torch.equal(o, want)
        del behind


def test_stored_through_the_dispatcher_and_its_refusals():
    import chill_attention as ca

    lens, new, parents = ints([0, 5]), ints([20, 30]), ints([[-1] * 30] * 2)

    def reserve(pages, stored):
        return ca.chill_pages_reserve(pages, lens, new, 30, 16, parents, stored).slots

    results = []
    for call in (reserve, torch.compile(reserve, fullgraph=True), lambda pages, stored: torch.ops.chill_attention.pages_reserve_stored(
            *pages, lens, new, 30, 16, parents, stored)[0]):
        pages, stored = ca.ChillPages.empty(2, 100, 3, 16), ints([-9, -9])
        version = stored._version
        slots = call(pages, stored)
        assert stored.tolist() == (slots >= 0).sum(1).tolist() == [20, 11] and stored._version > version
        results.append((slots, *pages))
    assert all(torch.equal(x, y) for other in results[1:] for x, y in zip(results[0], other))
    pages = ca.ChillPages.empty(2, 100, 3, 16)
    for bad in (ints([0]), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32), ints([0, 0, 0, 0])[::2]):
        with pytest.raises(AssertionError):
            reserve(pages, bad)
    for taken in (lens, new, pages.held):
        with pytest.raises(RuntimeError, match="invalid argument"):
            reserve(pages, taken)
    assert pages.n_free.item() == 3


@pytest.mark.parametrize("dtype,N,G,page", [(torch.bfloat16, 2, 4, 16), (torch.float16, 9, 2, 16), (torch.bfloat16, 70, 2, 16), (torch.float32, 1, 1, 16),
                                            (torch.float32, 9, 1, 16), (torch.float16, 3, 2, 5)], ids=str)
@pytest.mark.parametrize("length", [200, 1500, 30000])
def test_a_query_that_is_not_finite_shows(dtype, N, G, page, length):
    """Rows that have nothing but NaN for scores, over whole units, a few parts and many of them; the other rows are as without these."""
    p = Problem(dtype, 2 * G, 2, 64, [length, 40], [N, N], N, page, tree=N > 3, seed=N)
    (want, want_lse), scale = attend(p, masks()["causal"])
    was = p.q[0, 1, N - 1, 5].clone()
    p.q[0, 1, N - 1, 5] = float("nan")
    (o, lse), _ = attend(p, masks()["causal"])
    assert torch.isnan(o[0, 1, N - 1]).all() and torch.isnan(lse[0, 1, N - 1])
    p.q[0, 1, N - 1, 5] = was
    o[0, 1, N - 1], lse[0, 1, N - 1] = want[0, 1, N - 1], want_lse[0, 1, N - 1]
    check_attention(o, lse, p, masks()["causal"], scale, dtype != torch.float32)


@pytest.mark.parametrize("room", list(ROOMS))
@pytest.mark.parametrize("dtype,N,G,page", [(torch.float32, 1, 1, 16), (torch.float32, 2, 2, 16), (torch.float32, 9, 1, 16), (torch.float16, 2, 1, 5),
                                            (torch.bfloat16, 2, 4, 16), (torch.bfloat16, 70, 2, 16)], ids=str)
def test_a_value_that_is_not_finite_shows_whatever_its_weight(dtype, N, G, page, room):
    """A visible key far below the others (its weight is 0 in 32 bits) or at -inf: 0 times what it holds is NaN, in that channel alone."""
    for k in (-1000.0, float("-inf")):
        p = Problem(dtype, 2 * G, 2, 64, [200, 40], [N, N], N, page, tree=N > 2, seed=N, room=ROOMS[room])
        p.q[..., 0] = p.q[..., 0].abs() + 1.0
        where, row = int(p.table[0, 70 // page]), 70 % page
        p.k_cache[where, 0, row] = 0
        p.k_cache[where, 0, row, 0] = k
        p.v_cache[where, 0, row, 3] = float("nan")
        (o, lse), _ = attend(p, masks()["causal"])
        assert torch.isnan(o[0, :G, :, 3]).all() and torch.isfinite(lse).all()
        o[0, :G, :, 3] = 0
        assert torch.isfinite(o).all()


@pytest.mark.parametrize("dynamic", [None, True])
def test_a_compiled_step_with_other_sizes(dynamic):
    """Graphs of one traced step for batches and steps of other sizes."""
    import chill_attention as ca

    mask = masks()["window"]

    def step(pages, kc, vc, lens, new, q, k, v, parents, path, accepted):
        s = ca.chill_pages_reserve(pages, lens, new, q.shape[2], 16, parents)
        ca.chill_cache_append(kc, vc, k, v, s.slots)
        o, lse = ca.chill_attention_cached(q, kc, vc, pages.table, s, mask, return_lse=True)
        lens = ca.chill_cache_commit(kc, vc, pages.table, s, path, accepted)
        ca.chill_pages_trim(pages, lens, 16)
        return o, lse, lens

    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, dynamic=dynamic)
    for lens, N in (([250, 90], 6), ([30, 200], 9), ([77, 5, 300], 4), ([1] * 5, 33)):
        B = len(lens)
        p = Problem(torch.bfloat16, 8, 2, 64, lens, [N] * B, N, 16, tree=True, seed=N, room=600)
        k, v = (torch.randn(B, 2, N, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))

        def state():
            free = ints(p.spare_pages + [-1] * (p.k_cache.shape[0] - len(p.spare_pages)))
            pages = ca.ChillPages(p.table.cuda(), ints(p.held), free, ints([len(p.spare_pages)]), ints([0]))
            return pages, p.k_cache.nan_to_num(0.25).cuda(), p.v_cache.nan_to_num(0.25).cuda(), ints(p.lens), ints(p.new)

        a, b = state(), state()
        args = p.q.cuda(), k, v, ints(p.parents), ints([[0, 2, 3]] * B), ints([2] * B)
        want, got = step(*a, *args), compiled(*b, *args)
        assert all(torch.equal(x, y) for x, y in zip([*want, *a[0], a[1], a[2]], [*got, *b[0], b[1], b[2]]))
    torch._dynamo.reset()
