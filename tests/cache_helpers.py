"""Problems of the paged-cache tests: inputs, the 64-bit result and how far a kernel may be from it."""
import torch

from oracle import cache_oracle as orc

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def masks():
    import chill_attention as ca

    return {"full": ca.FullChillMask(), "causal": ca.CausalChillMask(), "window": ca.SlidingWindowChillMask(37, 0),
            "window_ahead": ca.SlidingWindowChillMask(50, 3), "chunkwise": ca.ChunkwiseChillMask(24, 2), "prefix_lm": ca.PrefixLMChillMask(30)}


class Problem:
    """CPU tensors of one call; .cuda() gives the arguments of the public functions."""

    def __init__(self, dtype, H, Hkv, D, lens, new, N, page, tree=False, seed=0, holes=(), spare=2, sharp=1.0, room=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.page, self.N, self.chain = dtype, page, N, not tree
        B = len(lens)
        self.lens, self.new = list(lens), list(new)
        blocks = [-(-(c + min(max(n, 0), N)) // page) for c, n in zip(lens, new)]
        pages, width = sum(blocks) + spare, max(max(blocks), 1) + 1
        width = max(width, -(-room // page))  # room: keys the table has room for
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(blocks):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        whole = self.table.tolist()
        for b, block, value in holes:
            self.table[b, block] = value
        self.held, self.spare_pages = blocks, order[at:]
        self.q = (torch.randn(B, H, N, D, generator=g) * sharp).to(dtype)
        self.k_cache, self.v_cache = (torch.full((pages, Hkv, page, D), float("nan"), dtype=dtype) for _ in range(2))
        for b, (c, n) in enumerate(zip(lens, new)):  # rows that are in use; everything else stays NaN
            for t in range(c + min(max(n, 0), N)):
                p = int(self.table[b, t // page])
                if 0 <= p < pages:
                    self.k_cache[p, :, t % page] = torch.randn(Hkv, D, generator=g).to(dtype)
                    self.v_cache[p, :, t % page] = torch.randn(Hkv, D, generator=g).to(dtype)
        self.parents = [[int(torch.randint(max(-1, i - 4), i, (1,), generator=g)) for i in range(N)] for _ in range(B)] if tree else None
        _, _, _, _, self.slots, self.positions, self.sets = orc.reserve(whole, blocks, [], 0, self.lens, self.new, N, page, self.parents)

    def step(self, device="cuda"):
        from chill_attention import ChillStep

        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        bits = None
        if not self.chain:
            words = (self.N + 31) // 32
            bits = torch.zeros(len(self.lens), self.N, words, dtype=torch.int64)
            for b, family in enumerate(self.sets):
                for i, s in enumerate(family):
                    for j in s:
                        bits[b, i, j // 32] |= 1 << (j % 32)
            bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).to(device)
        return ChillStep(ints(self.lens), ints(self.new), ints(self.slots), ints(self.positions), bits)

    def oracle(self, mask, scale):
        return orc.attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.new, self.positions, self.sets, mask, scale, self.chain)


def check_attention(o, lse, problem, mask, scale, tensor_cores, rows=None):
    """O and LSE against 64 bits.  With u = 2^-24, D channels, T keys, z = max_t sum_d scale |q_d k_td| of a row and A = sum_t p_t |v_t|:
    a score (natural units) is off by at most d = (D + 8) u z (fp32 products and sums of exact inputs, scale, subtraction of the
    maximum) and a weight by e^d - 1 + 2^-21 (two ulp of exp2 for the weight, two for a rescaling); sums over the keys add T u.
    Numerator and denominator both: 2 (d + 2^-21 + (T + 8) u) A, for d << 1.  Kernels that feed 16-bit weights to the tensor cores round each
    once, half a step eps, and where fp16 has no more exponents than 2^-24, 2^-25 of the largest weight absolutely: eps A + T 2^-25
    max|v| (the largest weight is 1 up to a factor of 2^8 from a lazily updated maximum, which only helps).  Then the result is rounded
    to its type.  LSE: (d + 2^-21 + (T + 8) u) / ln 2 and half a step of fp32."""
    o_ref, lse_ref, size, most, keys = problem.oracle(mask, scale)
    u, D = 2.0 ** -24, problem.q.shape[3]
    rel = (D + 8) * u * most + 2.0 ** -21 + (keys + 8) * u
    assert rel.max() < 0.01
    bound = 2 * rel[..., None] * size
    if tensor_cores:
        v = problem.v_cache[torch.isfinite(problem.v_cache)].abs().max().item() if torch.isfinite(problem.v_cache).any() else 0.0
        bound = bound + EPS[problem.dtype] * size + (keys[..., None] * 2.0 ** -25 * v if problem.dtype == torch.float16 else 0.0)
    tiny = 2.0 ** -25 if problem.dtype == torch.float16 else 1e-37  # half of the smallest value there is
    bound = bound + EPS[problem.dtype] * (o_ref.abs() + bound) + tiny
    o, lse = o.detach().cpu().double(), lse.detach().cpu().double()
    assert o.shape == o_ref.shape
    if rows is not None:  # [batch, token]: these alone
        o, lse = (torch.where(rows.view(len(rows), 1, -1, *[1] * (x.ndim - 3)), x, y) for x, y in ((o, o_ref), (lse, lse_ref)))
    assert torch.isfinite(o).all()
    excess = ((o - o_ref).abs() / bound).max().item()
    assert excess <= 1.0, f"O is {excess:.2f} times the bound off"
    assert torch.equal(torch.isneginf(lse), torch.isneginf(lse_ref))
    fin = torch.isfinite(lse_ref)
    lse_bound = rel / 0.6931 + u * lse_ref.abs()
    assert ((lse - lse_ref).abs()[fin] <= lse_bound[fin]).all(), f"LSE off by {((lse - lse_ref).abs() - lse_bound)[fin].max().item()}"
    for b, n in enumerate(problem.new):
        assert (o[b, :, min(max(n, 0), problem.N):] == 0).all() and (lse[b, :, min(max(n, 0), problem.N):] == 0).all()
