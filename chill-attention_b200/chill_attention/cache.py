"""Serving from a paged cache: pages and slots for new tokens, storing their keys and values, attention of the new tokens (one
for each request, a chunk of a prompt, or a tree of drafted tokens) over the cache, and keeping the accepted path of a tree.

    pages = ChillPages.empty(batch, max_len, num_pages, page_size)        # integer tensors, on the GPU
    k_cache = torch.empty(num_pages, kv_heads, page_size, head_dim, dtype=..., device="cuda")   # v_cache alike
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")           # tokens in the cache
    stored = torch.empty_like(lens)
    while ...:                                                            # one step, for every layer its own caches
        step = chill_pages_reserve(pages, lens, new_lens, max_new, page_size, parents, stored)
        # project; rotate q and k to step.positions
        chill_cache_append(k_cache, v_cache, k, v, step.slots)            # k, v: [batch, kv_heads, max_new, head_dim]
        o = chill_attention_cached(q, k_cache, v_cache, pages.table, step, mask)
        # a tree: choose the path to keep, then
        lens = chill_cache_commit(k_cache, v_cache, pages.table, step, path, accepted)
        # a chain: lens = lens + stored   (new_lens, unless pages ran out: what got no page comes again in a later step)
    chill_pages_trim(pages, lens, page_size)                              # lens[b] = 0: request b is done

Nothing here synchronises or copies to the host, lengths are read on the GPU, and every call can be captured into a CUDA graph and
replayed with other lengths in the same tensors; torch.compile traces the calls as dispatcher ops (a mask class after its first eager
call).  Work is enqueued on the current stream of the tensors' device; calls that use the
same pages on different streams are ordered by the caller.  There are no gradients: tensors that require them are refused.  The
reference has no counterpart; a mask means here what it means to ``chill_attention``, for tokens at the positions of the step.
"""
from __future__ import annotations

import ctypes as C
import typing

import torch
from torch.autograd import forward_ad

from . import _cabi, _cache_abi, _decode_abi, _eager, chill
from .mask import ChillMask

_HEAD_DIMS = chill._HEAD_DIMS
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
#: entry points a native CacheLibrary object is made of, in its order
_ENTRY_POINTS = ("chill_cached_fwd", "chill_cached_workspace_bytes", "chill_pages_reserve_stored", "chill_pages_trim", "chill_cache_append",
                 "chill_cache_commit")
#: library -> its native call object; mask class name -> (call object, functor id, class)
_NATIVE: dict = {}
_MASKS: dict[str, tuple] = {}


class ChillPages(typing.NamedTuple):
    """Which pages a batch of requests holds and which are free; int32 tensors on the GPU, changed in place.

    table: [batch, blocks], page of every block of page_size tokens (-1: none); held: [batch], blocks with a page;
    free: [num_pages], a stack, n_free: [1], its height; missing: [1], pages that the last reservation or fork wanted and did not get."""

    table: torch.Tensor
    held: torch.Tensor
    free: torch.Tensor
    n_free: torch.Tensor
    missing: torch.Tensor

    @classmethod
    def empty(cls, batch: int, max_len: int, num_pages: int, page_size: int, device="cuda") -> "ChillPages":
        """No request holds a page; a request can grow to max_len tokens (rounded up to whole pages)."""
        assert batch >= 1 and max_len >= 1 and num_pages >= 1 and page_size >= 1
        ints = {"dtype": torch.int32, "device": device}
        return cls(torch.full((batch, -(-max_len // page_size)), -1, **ints), torch.zeros(batch, **ints),
                   torch.arange(num_pages - 1, -1, -1, **ints), torch.full((1,), num_pages, **ints), torch.zeros(1, **ints))


class ChillCopies(typing.NamedTuple):
    """Pages to be copied, int32 tensors on the GPU: the first rows[i] rows of page source[i] go to page target[i], for i < count ([1])."""

    source: torch.Tensor
    target: torch.Tensor
    rows: torch.Tensor
    count: torch.Tensor


class ChillStep(typing.NamedTuple):
    """The new tokens of a step, int32 tensors on the GPU: lens [batch] tokens in the cache before, new_lens [batch] new ones,
    slots [batch, max_new] page * page_size + row of each (-1: none), positions [batch, max_new], and for trees ancestors
    [batch, max_new, (max_new + 31) // 32]: bit j of row i says that token j is token i or above it."""

    lens: torch.Tensor
    new_lens: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    ancestors: typing.Optional[torch.Tensor]


def _native(lib=None):
    """The native call object of a library (None: the one of the built-in masks)."""
    native = _NATIVE.get(lib)
    if native is None:
        found = lib or _cache_abi.load_library()
        functions = [getattr(found, name) for name in _ENTRY_POINTS] + [_cabi.load_library().chill_status_string, found.chill_cache_last_cuda_error]
        native = _NATIVE[lib] = _eager.extension().CacheLibrary([C.cast(f, C.c_void_p).value for f in functions])
    return native


_is_compiling = torch.compiler.is_compiling
_dispatch_depth, _function_depth, _functorch_top = _eager._dispatch_depth, _eager._function_depth, _eager._functorch_top


def _direct() -> bool:
    """Whether a call can go to the native module: the eager path is on (CHILL_ATTENTION_EAGER_FAST), nothing watches the dispatcher.
    (The module itself turns away tensors that are watched, or not on a GPU.)"""
    return not _is_compiling() and _eager.ENABLED and _eager._PROBES_OK and _dispatch_depth() == 0 and _function_depth() == 0 and _functorch_top() is None


# --------------------------------------------------------------------------------------------- argument checks, with messages
def _check_ints(like, **named):
    for name, (t, shape) in named.items():
        assert isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.is_contiguous(), f"{name} must be a contiguous int32 tensor"
        assert tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}"
        assert t.device == like.device, f"{name} must be on {like.device}"


def _check_sizes(**named):
    for name, t in named.items():
        for size in t.shape:
            assert size < 2 ** 31, f"the sizes of {name} must fit 32 bits"


def _check_changed(**named):
    """Tensors that a call changes in place: torch cannot apply a pending sign there for an operator that also returns something."""
    if not _is_compiling():
        for name, t in named.items():
            assert not t.is_neg(), f"{name} is changed in place and has a sign that is still to be applied: resolve_neg() makes a tensor of its own"


def _check_table(table):
    _check_sizes(table=table)
    assert table.is_cuda, "the paged cache runs on CUDA tensors only"
    assert table.dtype == torch.int32 and table.ndim == 2 and table.numel() > 0, "table must be an int32 tensor [batch, blocks]"
    assert table.stride(1) == 1 and (table.shape[0] == 1 or table.stride(0) >= table.shape[1]), "the rows of table must be contiguous"


def _check_pages(pages, lens, page_size):
    _check_table(pages.table)
    B = pages.table.shape[0]
    assert 1 <= page_size < 2 ** 31 and pages.free.ndim == 1 and pages.free.numel() >= 1
    _check_sizes(free=pages.free)
    _check_ints(pages.table, held=(pages.held, (B,)), free=(pages.free, pages.free.shape), n_free=(pages.n_free, (1,)), lens=(lens, (B,)))
    _check_changed(table=pages.table, held=pages.held, free=pages.free, n_free=pages.n_free)


def _check_caches(k_cache, v_cache):
    _check_sizes(k_cache=k_cache)
    assert k_cache.is_cuda and k_cache.device == v_cache.device, "the caches must be CUDA tensors on one device"
    assert k_cache.ndim == 4 and k_cache.shape == v_cache.shape and k_cache.numel() > 0, \
        "k_cache and v_cache must have one shape [num_pages, kv_heads, page_size, head_dim]"
    assert k_cache.dtype == v_cache.dtype and k_cache.dtype in _DTYPES


def _check_grad(*tensors):
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), \
        "the paged cache has no gradients: call it under torch.no_grad() or with detached tensors"
    if not _is_compiling():
        assert all(forward_ad.unpack_dual(t).tangent is None for t in tensors), "the paged cache has no gradients: the tensors carry tangents"


def _check_rows(k_cache, v_cache, k, v, slots):
    _check_caches(k_cache, v_cache)
    _check_sizes(k=k)
    assert k.ndim == 4 and k.shape == v.shape and k.numel() > 0, "k and v must have one shape [batch, kv_heads, max_new, head_dim]"
    assert k.shape[1] == k_cache.shape[1] and k.shape[3] == k_cache.shape[3], "kv heads and head dim must be those of the caches"
    assert k.dtype == v.dtype == k_cache.dtype and k.device == v.device == k_cache.device
    _check_ints(k_cache, slots=(slots, (k.shape[0], k.shape[2])))
    _check_changed(k_cache=k_cache, v_cache=v_cache)
    _check_grad(k_cache, v_cache, k, v)


def _check_commit(k_cache, v_cache, table, lens, new_lens, path, accepted):
    _check_caches(k_cache, v_cache)
    _check_table(table)
    assert table.device == k_cache.device
    B = table.shape[0]
    _check_sizes(path=path)
    assert path.ndim == 2 and path.shape[1] >= 1, "path must be [batch, longest path]"
    _check_ints(k_cache, lens=(lens, (B,)), new_lens=(new_lens, (B,)), path=(path, (B, path.shape[1])), accepted=(accepted, (B,)))
    _check_changed(k_cache=k_cache, v_cache=v_cache)
    _check_grad(k_cache, v_cache)


def _check_attention(q, k_cache, v_cache, table, lens, new_lens, positions, ancestors):
    _check_caches(k_cache, v_cache)
    _check_table(table)
    _check_sizes(q=q)
    assert q.ndim == 4 and q.numel() > 0, "q must be [batch, heads, max_new, head_dim]"
    B, H, N, D = q.shape
    assert D in _HEAD_DIMS, f"head dim must be one of {sorted(_HEAD_DIMS)}"
    assert k_cache.shape[3] == D and H % k_cache.shape[1] == 0 and table.shape[0] == B
    assert q.dtype == k_cache.dtype and q.device == k_cache.device == table.device
    _check_ints(q, lens=(lens, (B,)), new_lens=(new_lens, (B,)), positions=(positions, (B, N)))
    if ancestors is not None:
        _check_ints(q, ancestors=(ancestors, (B, N, (N + 31) // 32)))
    _check_grad(q, k_cache, v_cache)


# ------------------------------------------------------------------------- dispatcher ops: torch.compile, modes, subclasses
def _reserve(pages, lens, new_lens, max_new, page_size, parents, stored):
    _check_pages(pages, lens, page_size)
    _check_reserve(pages, new_lens, max_new, parents, stored)
    slots, positions, ancestors = _eager.extension().pages_reserve(_native(), *pages, lens, new_lens, max_new, page_size, parents, stored)
    return slots, positions, ancestors if ancestors is not None else slots.new_empty(0)


@torch.library.custom_op("chill_attention::pages_reserve", mutates_args=("table", "held", "free", "n_free", "missing"), device_types=("cuda",))
def _reserve_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, missing: torch.Tensor, lens: torch.Tensor,
                new_lens: torch.Tensor, max_new: int, page_size: int,
                parents: typing.Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _reserve(ChillPages(table, held, free, n_free, missing), lens, new_lens, max_new, page_size, parents, None)


@torch.library.custom_op("chill_attention::pages_reserve_stored", mutates_args=("table", "held", "free", "n_free", "missing", "stored"),
                         device_types=("cuda",))
def _reserve_stored_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, missing: torch.Tensor, lens: torch.Tensor,
                       new_lens: torch.Tensor, max_new: int, page_size: int, parents: typing.Optional[torch.Tensor],
                       stored: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _reserve(ChillPages(table, held, free, n_free, missing), lens, new_lens, max_new, page_size, parents, stored)


@_reserve_stored_op.register_fake
@_reserve_op.register_fake
def _(table, held, free, n_free, missing, lens, new_lens, max_new, page_size, parents, stored=None):
    B = table.shape[0]
    shape = (B, max_new, (max_new + 31) // 32) if parents is not None else (0,)
    return table.new_empty(B, max_new), table.new_empty(B, max_new), table.new_empty(shape)


@torch.library.custom_op("chill_attention::pages_trim", mutates_args=("table", "held", "free", "n_free"), device_types=("cuda",))
def _trim_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, lens: torch.Tensor, page_size: int) -> None:
    _check_pages(ChillPages(table, held, free, n_free, n_free), lens, page_size)
    _eager.extension().pages_trim(_native(), table, held, free, n_free, lens, page_size)


@_trim_op.register_fake
def _(table, held, free, n_free, lens, page_size):
    return None


@torch.library.custom_op("chill_attention::cache_append", mutates_args=("k_cache", "v_cache"), device_types=("cuda",))
def _append_op(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    _check_rows(k_cache, v_cache, k, v, slots)
    _eager.extension().cache_append(_native(), k_cache, v_cache, k, v, slots)


@_append_op.register_fake
def _(k_cache, v_cache, k, v, slots):
    return None


@torch.library.custom_op("chill_attention::cache_commit", mutates_args=("k_cache", "v_cache"), device_types=("cuda",))
def _commit_op(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, max_new: int,
               path: torch.Tensor, accepted: torch.Tensor) -> torch.Tensor:
    _check_commit(k_cache, v_cache, table, lens, new_lens, path, accepted)
    return _eager.extension().cache_commit(_native(), k_cache, v_cache, table, lens, new_lens, max_new, path, accepted)


@_commit_op.register_fake
def _(k_cache, v_cache, table, lens, new_lens, max_new, path, accepted):
    return torch.empty_like(lens)


@torch.library.custom_op("chill_attention::cached_forward", mutates_args=(), device_types=("cuda",))
def _attention_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor,
                  positions: torch.Tensor, ancestors: typing.Optional[torch.Tensor], mask_name: str,
                  mask_args: typing.List[typing.Union[int, float, bool]], sm_scale: float, flags: int) -> tuple[torch.Tensor, torch.Tensor]:
    _check_attention(q, k_cache, v_cache, table, lens, new_lens, positions, ancestors)
    native, functor_id, _ = _MASKS[mask_name]
    return _eager.extension().cached_attention(native, functor_id, q, k_cache, v_cache, table, lens, new_lens, positions, ancestors,
                                               tuple(mask_args), sm_scale, True, flags)


@_attention_op.register_fake
def _(q, k_cache, v_cache, table, lens, new_lens, positions, ancestors, mask_name, mask_args, sm_scale, flags):
    return torch.empty_like(q, memory_format=torch.contiguous_format), q.new_empty(q.shape[:3], dtype=torch.float32)


# The operators of pages that several requests share (libchill_decode_b200.so)
def _decode():
    from . import rotary

    return rotary._NATIVE or rotary._native()


def _places(pages):
    return pages.table, pages.held, pages.free, pages.n_free


def _check_fork(pages, shared, lens, parents, page_size):
    _check_pages(pages, lens, page_size)
    B = pages.table.shape[0]
    assert B <= _decode_abi.FORK_MAX, f"a fork takes at most {_decode_abi.FORK_MAX} requests"
    _check_ints(pages.table, missing=(pages.missing, (1,)), shared=(shared, pages.free.shape), parents=(parents, (B,)))
    _check_changed(missing=pages.missing, shared=shared)


def _check_compact(pages, page_size, shared):
    _check_pages(pages, pages.held, page_size)
    if shared is not None:
        _check_ints(pages.table, shared=(shared, pages.free.shape))
        _check_changed(shared=shared)


def _check_copy(k_cache, v_cache, copies):
    _check_sizes(k_cache=k_cache)
    assert k_cache.is_cuda and k_cache.device == v_cache.device, "the caches must be CUDA tensors on one device"
    assert k_cache.ndim in (4, 5) and k_cache.shape == v_cache.shape and k_cache.numel() > 0, \
        "k_cache and v_cache must have one shape [num_pages, kv_heads, page_size, head_dim], or [layers, ...]"
    assert k_cache.dtype == v_cache.dtype and k_cache.dtype in _DTYPES
    source, target, rows, count = copies
    assert isinstance(source, torch.Tensor) and source.ndim == 1 and source.numel() > 0
    _check_sizes(source=source)
    _check_ints(k_cache, source=(source, source.shape), target=(target, source.shape), rows=(rows, source.shape), count=(count, (1,)))
    _check_changed(k_cache=k_cache, v_cache=v_cache)
    _check_grad(k_cache, v_cache)


@torch.library.custom_op("chill_attention::pages_trim_shared", mutates_args=("table", "held", "free", "n_free", "shared"), device_types=("cuda",))
def _trim_shared_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, shared: torch.Tensor, lens: torch.Tensor,
                    page_size: int) -> None:
    _check_pages(ChillPages(table, held, free, n_free, n_free), lens, page_size)
    _check_ints(table, shared=(shared, free.shape))
    _eager.extension().pages_trim_shared(_decode(), table, held, free, n_free, shared, lens, page_size)


@_trim_shared_op.register_fake
def _(table, held, free, n_free, shared, lens, page_size):
    return None


@torch.library.custom_op("chill_attention::pages_fork", mutates_args=("table", "held", "free", "n_free", "missing", "shared"), device_types=("cuda",))
def _fork_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, missing: torch.Tensor, shared: torch.Tensor, lens: torch.Tensor,
             parents: torch.Tensor, page_size: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_fork(ChillPages(table, held, free, n_free, missing), shared, lens, parents, page_size)
    return _eager.extension().pages_fork(_decode(), table, held, free, n_free, missing, shared, lens, parents, page_size)


@_fork_op.register_fake
def _(table, held, free, n_free, missing, shared, lens, parents, page_size):
    B = table.shape[0]
    return (*(table.new_empty(B) for _ in range(4)), table.new_empty(1))


@torch.library.custom_op("chill_attention::pages_compact", mutates_args=("table", "free", "n_free", "shared"), device_types=("cuda",))
def _compact_op(table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, shared: typing.Optional[torch.Tensor],
                page_size: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_compact(ChillPages(table, held, free, n_free, n_free), page_size, shared)
    return _eager.extension().pages_compact(_decode(), table, held, free, n_free, shared, page_size)


@_compact_op.register_fake
def _(table, held, free, n_free, shared, page_size):
    n = max(free.shape[0] // 2, 1)
    return (*(table.new_empty(n) for _ in range(3)), table.new_empty(1))


@torch.library.custom_op("chill_attention::cache_copy", mutates_args=("k_cache", "v_cache"), device_types=("cuda",))
def _copy_op(k_cache: torch.Tensor, v_cache: torch.Tensor, source: torch.Tensor, target: torch.Tensor, rows: torch.Tensor, count: torch.Tensor) -> None:
    _check_copy(k_cache, v_cache, (source, target, rows, count))
    _eager.extension().cache_copy(_decode(), k_cache, v_cache, source, target, rows, count)


@_copy_op.register_fake
def _(k_cache, v_cache, source, target, rows, count):
    return None


# ------------------------------------------------------------------------------------------------------------ public calls
def _check_reserve(pages, new_lens, max_new, parents, stored):
    B = pages.table.shape[0]
    assert 1 <= max_new < 2 ** 31
    _check_ints(pages.table, missing=(pages.missing, (1,)), new_lens=(new_lens, (B,)))
    _check_changed(missing=pages.missing)
    if parents is not None:
        _check_ints(pages.table, parents=(parents, (B, max_new)))
    if stored is not None:
        _check_ints(pages.table, stored=(stored, (B,)))
        _check_changed(stored=stored)


def chill_pages_reserve(pages: ChillPages, lens: torch.Tensor, new_lens: torch.Tensor, max_new: int, page_size: int,
                        parents: torch.Tensor | None = None, stored: torch.Tensor | None = None) -> ChillStep:
    """Pages for ``new_lens[b]`` tokens behind the ``lens[b]`` that request b has, and where they go.

    Args:
        pages: changed in place.  Pages are taken from the top of the stack, requests in order; a request keeps what it holds
            already.  Where the stack runs out, or a table is full, the tokens left without a page get slot -1 (they are not
            stored, and nobody sees them) and ``pages.missing`` says how many pages the stack was short of.  Only the others may
            be counted in lens afterwards (see stored): a page that a later step finds for a token that was never stored holds what
            its former owner left there.
        lens, new_lens: int32 [batch]; new_lens is clamped to [0, max_new].
        max_new: second dimension of the step's tensors.
        page_size: rows of a page of the caches.
        parents: int32 [batch, max_new] for trees of drafted tokens: number of each token's parent among the new ones, smaller than its
            own; anything else (-1) makes it a child of the last cached token.  Without it the new tokens are a chain.
        stored: int32 [batch], written where given (a tensor of its own): how many of a request's new tokens got a slot, the first so many.

    Returns: the step's ChillStep; positions are lens[b] + depth (chain: lens[b] + number).
    """
    if _direct():
        native = _NATIVE.get(None) or _native()
        out = _eager._extension.pages_reserve(native, *pages, lens, new_lens, max_new, page_size, parents, stored)
        if out is not None:
            return ChillStep(lens, new_lens, *out)
    _check_pages(pages, lens, page_size)
    _check_reserve(pages, new_lens, max_new, parents, stored)
    if stored is None:
        slots, positions, ancestors = _reserve_op(*pages, lens, new_lens, max_new, page_size, parents)
    else:
        slots, positions, ancestors = _reserve_stored_op(*pages, lens, new_lens, max_new, page_size, parents, stored)
    return ChillStep(lens, new_lens, slots, positions, ancestors if parents is not None else None)


def chill_pages_trim(pages: ChillPages, lens: torch.Tensor, page_size: int, shared: torch.Tensor | None = None) -> None:
    """Gives the pages behind ``lens[b]`` tokens of every request back (``lens[b] = 0``: all of them), in place.

    The exact inverse of a reservation: what it gives back is what the same reservation takes again, in the same order.

    ``shared``, int32 [num_pages], changed in place: how many requests beyond one hold a page (``chill_pages_fork``).  Given that, a page goes back when the last of its
    holders lets go of it.  Without it pages must have one holder each.  A request that is cut back inside a page that others hold, and grows again, would write into it:
    ``chill_pages_fork`` with its own number as parent gives it a page of its own first."""
    if shared is not None:
        if _direct() and _eager.extension().pages_trim_shared(_decode(), *_places(pages), shared, lens, page_size):
            return
        _check_pages(pages, lens, page_size)
        _check_ints(pages.table, shared=(shared, pages.free.shape))
        _check_changed(shared=shared)
        _trim_shared_op(*_places(pages), shared, lens, page_size)
        return
    if _direct() and _eager.extension().pages_trim(_NATIVE.get(None) or _native(), pages.table, pages.held, pages.free, pages.n_free, lens, page_size):
        return
    _check_pages(pages, lens, page_size)
    _trim_op(pages.table, pages.held, pages.free, pages.n_free, lens, page_size)


def chill_pages_fork(pages: ChillPages, shared: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, page_size: int) -> tuple[torch.Tensor, ChillCopies]:
    """Request b goes on from where request ``parents[b]`` is: it takes over that one's ``lens[parents[b]]`` tokens, all requests at once and in place.

    Whole pages are shared between the children of a request.  A page that is only begun is written to next, so it has one holder: the first child keeps it (if no other
    request holds it), every other one gets a page from the stack, into which ``chill_cache_copy`` has to copy what is written.  Pages that nobody holds any more, those
    of requests without children and those behind the tokens among them, go back to the stack, in the order of the requests and blocks that held them first, the first on top.

    Args:
        pages: changed in place.
        shared: int32 [num_pages], changed in place: how many requests beyond one hold a page; zeros to begin with (``chill_pages_reserve`` hands out pages with one holder).
        lens: int32 [batch], tokens of each request.
        parents: int32 [batch]; itself to stay as it is, anything outside [0, batch): the request is empty afterwards.

    Returns: (tokens of each request now, int32 [batch]; the copies to be made in every layer's caches before anything else is written there).  Where the stack runs
    out of pages (``pages.missing`` says of how many) a request keeps whole pages only, and its tokens say so.  At most 8192 requests.
    """
    if _direct():
        out = _eager.extension().pages_fork(_decode(), *pages, shared, lens, parents, page_size)
        if out is not None:
            return out[0], ChillCopies(*out[1:])
    _check_fork(pages, shared, lens, parents, page_size)
    out = _fork_op(*pages, shared, lens, parents, page_size)
    return out[0], ChillCopies(*out[1:])


def chill_pages_compact(pages: ChillPages, page_size: int, shared: torch.Tensor | None = None) -> ChillCopies:
    """Moves the pages in use to the bottom of the pool, in place: with U of them, the highest one goes to the lowest free page below U, and so on; afterwards pages
    0 ... U - 1 are in use and the stack has the lowest free page on top.

    Every page that is not on the stack counts as used, whether a table names it or not; tables and ``shared`` follow.

    Returns: the copies to be made in every layer's caches (whole pages; sources and targets have none in common) before anything else is read or written there.
    """
    if _direct():
        out = _eager.extension().pages_compact(_decode(), *_places(pages), shared, page_size)
        if out is not None:
            return ChillCopies(*out)
    _check_compact(pages, page_size, shared)
    return ChillCopies(*_compact_op(*_places(pages), shared, page_size))


def chill_cache_copy(k_cache: torch.Tensor, v_cache: torch.Tensor, copies: ChillCopies) -> None:
    """Copies pages, in place: the first ``rows[i]`` rows of page ``source[i]`` to page ``target[i]``, for i < count.

    Args:
        k_cache, v_cache: [num_pages, kv_heads, page_size, head_dim], or those of all layers [layers, num_pages, ...]; any strides.  They may be the same tensor, but not
            overlap otherwise.
        copies: of ``chill_pages_fork`` or ``chill_pages_compact``, or the caller's own; orders with a page outside the cache are left out, a target must not be source or
            target of another order.
    """
    if _direct() and _eager.extension().cache_copy(_decode(), k_cache, v_cache, *copies):
        return
    _check_copy(k_cache, v_cache, copies)
    _copy_op(k_cache, v_cache, *copies)


def chill_cache_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Stores the rows of ``k`` and ``v`` ([batch, kv_heads, max_new, head_dim], any strides) at ``slots`` of the caches
    ([num_pages, kv_heads, page_size, head_dim], any strides), in place.  Tokens whose slot is outside the cache (-1) are left out; rows that
    no slot names stay as they are, one that two tokens name holds either's."""
    if _direct() and _eager.extension().cache_append(_NATIVE.get(None) or _native(), k_cache, v_cache, k, v, slots):
        return
    _check_rows(k_cache, v_cache, k, v, slots)
    _append_op(k_cache, v_cache, k, v, slots)


def chill_cache_commit(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, step: ChillStep, path: torch.Tensor,
                       accepted: torch.Tensor) -> torch.Tensor:
    """Keeps the accepted path of every request's tree: its keys and values become the next rows behind the cached ones, in place.

    Args:
        path: int32 [batch, longest path], numbers of the accepted tokens from the root on (increasing).
        accepted: int32 [batch], how many of them; clamped to [0, min(longest path, new_lens[b])].

    Returns: int32 [batch], the new lengths ``lens + accepted``, without the accepted tokens from the first one without a page on.  k_cache and
    v_cache may be the same tensor, but not overlap otherwise.  Pages stay reserved; ``chill_pages_trim`` gives spare ones back.
    """
    N = step.slots.shape[1]
    if _direct():
        out = _eager.extension().cache_commit(_NATIVE.get(None) or _native(), k_cache, v_cache, table, step.lens, step.new_lens, N, path, accepted)
        if out is not None:
            return out
    _check_commit(k_cache, v_cache, table, step.lens, step.new_lens, path, accepted)
    return _commit_op(k_cache, v_cache, table, step.lens, step.new_lens, N, path, accepted)


def _mask_functor(mask: ChillMask):
    """Finds the native call object and the functor id that serve this mask class (builds the custom library if needed)."""
    functor, header = getattr(mask, "cuda_functor", None), getattr(mask, "cuda_functor_header", None)
    if header is not None:
        from .custom import build_custom_cache_library

        if not functor:
            raise ValueError(f"{mask.name}: cuda_functor_header is set but cuda_functor (struct name) is not")
        found = _native(_cache_abi.load_library(build_custom_cache_library(header, functor))), _cabi.MASK_CUSTOM
    elif functor in _cabi.BUILTIN_FUNCTOR_IDS:
        found = _native(), _cabi.BUILTIN_FUNCTOR_IDS[functor]
    else:
        raise NotImplementedError(f"{mask.name} has no CUDA functor: set `cuda_functor` to a built-in functor name or provide "
                                  "`cuda_functor_header` + `cuda_functor` (see chill_attention/custom.py)")
    _MASKS[mask.name] = *found, type(mask)


def _check_same_name(mask: ChillMask):
    """The dispatcher op knows a mask by its class name: another class of that name has to mean the same functor."""
    known = _MASKS[mask.name][2]
    same = all(getattr(mask, a, None) == getattr(known, a, None) for a in ("cuda_functor", "cuda_functor_header"))
    if not same:
        raise ValueError(f"two mask classes are named {mask.name} and have different CUDA functors: give one of them another name")


def chill_attention_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, step: ChillStep, mask: ChillMask,
                           sm_scale: float | None = None, return_lse: bool = False):
    """Exact softmax attention of the step's new tokens over the cached and the new keys that ``mask`` allows.

    Token i of request b stands at position ``step.positions[b, i]`` in a tree and at ``step.lens[b] + i`` in a chain (whatever
    ``step.positions`` holds; ``chill_pages_reserve`` puts the same there), and sees cached key t (position t) iff the mask allows the pair, and
    new key j iff the mask allows their positions and, in a tree, j is an ancestor of i or i itself.  In a chain a mask that looks ahead (full,
    chunkwise) lets a token see the new ones behind it.  Keys without a page are not there.

    Args:
        q: [batch, heads, max_new, head_dim], fp16 / bf16 / fp32, any strides; heads a multiple of the caches' kv heads.
        k_cache, v_cache: [num_pages, kv_heads, page_size, head_dim], any strides; the new tokens' rows are stored already.
        table: ``pages.table``.
        mask: a ChillMask instance; its functor sees lens[b] + new_lens[b] as the sequence length.
        sm_scale: softmax scale, positive, default head_dim ** -0.5.
        return_lse: also return the log-sum-exp of every row in log2 units, shape [batch, heads, max_new].

    Returns: O, or (O, LSE).  A token that sees nothing: O = 0, LSE = -inf; rows at or behind new_lens[b]: zeros, LSE 0.

    Scores, sums and O are kept in fp32.  16-bit caches on the tensor cores: the softmax weights go into the second product rounded once to
    the caches' type (as in ``chill_attention``), with up to 16 rows (tokens times the heads that share a kv head) as two such numbers; so a
    token's last bits depend on how many stand beside it.  A key that is not finite shows in the rows that see it and in no others; these are
    worked out key by key, which over long tables takes seconds.
    """
    return _attention(q, k_cache, v_cache, table, step, mask, sm_scale, return_lse, 0)


def _attention(q, k_cache, v_cache, table, step, mask, sm_scale, return_lse, flags):
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5
    if mask.name not in _MASKS:
        _mask_functor(mask)
    elif _MASKS[mask.name][2] is not type(mask):
        _check_same_name(mask)
    lens, new_lens, _, positions, ancestors = step
    if _direct():
        native, functor_id, _ = _MASKS[mask.name]
        out = _eager._extension.cached_attention(native, functor_id, q, k_cache, v_cache, table, lens, new_lens, positions, ancestors,
                                                 mask.constargs, sm_scale, return_lse, flags)
        if out is not None:
            return out
    _check_attention(q, k_cache, v_cache, table, lens, new_lens, positions, ancestors)
    o, lse = _attention_op(q, k_cache, v_cache, table, lens, new_lens, positions, ancestors, mask.name, mask.constargs, sm_scale, flags)
    return (o, lse) if return_lse else o
