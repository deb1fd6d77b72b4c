"""Rotary positions: queries and keys turned by the angles of their positions, for training (``chill_rotate``, differentiable) and for serving from
a paged cache (``chill_rotate_append``: one launch that also stores keys and values).

    rotary = ChillRotary.of(head_dim)                                      # the frequencies, on the GPU
    q, k = chill_rotate(q, k, positions, rotary)                           # then chill_attention(q, k, v, mask)
    q = chill_rotate_append(q, k, v, k_cache, v_cache, step, rotary)       # then chill_attention_cached(q, ..., step, mask)

Pair i of a row at positions p is turned by the angle a = p[axes[i]] * inv_freq[i]:  y1 = x1 cos a - x2 sin a,  y2 = x2 cos a + x1 sin a.  Angles are
worked out in 64 bits (far positions lose nothing), the rest in fp32; results are rounded once.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as C
import typing

import torch
from torch.autograd import forward_ad

from . import _cabi, _decode_abi, _eager, cache

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
#: entry points the native DecodeLibrary object is made of, in its order
_ENTRY_POINTS = ("chill_rotate", "chill_rotate_append", "chill_beam_select", "chill_select_workspace_bytes", "chill_pages_fork", "chill_pages_trim_shared",
                 "chill_pages_compact", "chill_share_workspace_bytes", "chill_cache_copy")
_NATIVE = None


def _native():
    """The native call object of libchill_decode_b200.so."""
    global _NATIVE
    if _NATIVE is None:
        found = _decode_abi.load_library()
        functions = [getattr(found, name) for name in _ENTRY_POINTS] + [_cabi.load_library().chill_status_string, found.chill_decode_last_cuda_error]
        _NATIVE = _eager.extension().DecodeLibrary([C.cast(f, C.c_void_p).value for f in functions])
    return _NATIVE


class ChillRotary(typing.NamedTuple):
    """What turns: inv_freq, float32 [pairs] on the GPU, radians a position; axes, int32 [pairs], row of the positions that turns a pair (None: there is one
    row); interleaved: pair i is channels (2 i, 2 i + 1), otherwise (i, i + pairs).  Channels from 2 * pairs on stay as they are."""

    inv_freq: torch.Tensor
    axes: typing.Optional[torch.Tensor] = None
    interleaved: bool = False

    @classmethod
    def of(cls, channels: int, base: float = 10000.0, axes: typing.Sequence[int] | None = None, interleaved: bool = False, device="cuda") -> "ChillRotary":
        """inv_freq[i] = base ** (-2 i / channels) for ``channels // 2`` pairs, rounded to fp32 from 64 bits.

        Args:
            channels: how many of a head's channels turn, an even number.
            axes: for several axes (time, height, width, ...), the axis of each pair; e.g. (0,) * 16 + (1,) * 24 + (2,) * 24.
        """
        assert channels >= 2 and channels % 2 == 0, "an even number of channels turns"
        assert axes is None or (len(axes) == channels // 2 and min(axes) >= 0), "axes names the axis of every pair"
        inv_freq = (base ** (-torch.arange(0, channels, 2, dtype=torch.float64) / channels)).float().to(device)
        return cls(inv_freq, None if axes is None else torch.tensor(tuple(axes), dtype=torch.int32, device=device), interleaved)


# --------------------------------------------------------------------------------------------- argument checks, with messages
def _check_where(x, positions, rotary):
    inv_freq, axes, _ = rotary
    B, _, L, D = x.shape
    assert B * L * D < 2 ** 31, "batch * tokens * channels must stay below 2^31"
    assert isinstance(inv_freq, torch.Tensor) and inv_freq.dtype == torch.float32 and inv_freq.ndim == 1 and inv_freq.is_contiguous(), \
        "rotary.inv_freq must be a contiguous float32 tensor [pairs]"
    assert inv_freq.device == x.device and 1 <= inv_freq.shape[0] and 2 * inv_freq.shape[0] <= D, "rotary has more channels than a head, or is elsewhere"
    assert not (torch.is_grad_enabled() and inv_freq.requires_grad), "there is no gradient for rotary.inv_freq"
    if axes is not None:
        cache._check_ints(x, axes=(axes, inv_freq.shape))
    assert isinstance(positions, torch.Tensor) and positions.dtype == torch.int32 and positions.device == x.device, f"positions must be int32 on {x.device}"
    assert positions.ndim in (2, 3) and tuple(positions.shape[-2:]) == (B, L) and positions.shape[0] >= 1, \
        f"positions must be [{B}, {L}] or [axes, {B}, {L}], not {tuple(positions.shape)}"
    assert positions.ndim == 2 or positions.shape[0] == 1 or axes is not None, "several rows of positions, and no rotary.axes that says which pair turns by which"


def _check_rotate(q, k, positions, rotary):
    for name, x in (("q", q), ("k", k)):
        if x is not None:
            assert x.is_cuda, "rotary positions run on CUDA tensors only"
            assert x.ndim == 4 and x.numel() > 0, f"{name} must be [batch, heads, tokens, channels]"
            assert x.dtype in _DTYPES and x.dtype == q.dtype and x.device == q.device
            assert x.shape[0] == q.shape[0] and x.shape[2:] == q.shape[2:], "q and k must have one batch, tokens and channels"
            cache._check_sizes(**{name: x})
    _check_where(q, positions, rotary)


def _check_append(q, k, v, k_cache, v_cache, slots, positions, rotary):
    cache._check_rows(k_cache, v_cache, k, v, slots)
    assert q.ndim == 4 and q.numel() > 0 and q.dtype == k.dtype and q.device == k.device and q.is_cuda
    assert q.shape[0] == k.shape[0] and q.shape[2:] == k.shape[2:], "q and k must have one batch, tokens and channels"
    _check_where(q, positions, rotary)
    cache._check_grad(q, rotary.inv_freq)


# ------------------------------------------------------------------------- dispatcher ops: torch.compile, modes, subclasses
@torch.library.custom_op("chill_attention::rotate", mutates_args=(), device_types=("cuda",))
def _rotate_op(q: torch.Tensor, k: typing.Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, axes: typing.Optional[torch.Tensor],
               interleaved: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _check_rotate(q, k, positions, ChillRotary(inv_freq, axes, interleaved))
    q_out, k_out = _eager.extension().rotate(_native(), q, k, positions, inv_freq, axes, interleaved, inverse)
    return q_out, k_out if k is not None else q.new_empty(0)


@_rotate_op.register_fake
def _(q, k, positions, inv_freq, axes, interleaved, inverse):
    return torch.empty_like(q), torch.empty_like(k) if k is not None else q.new_empty(0)


def _rotate_setup(ctx, inputs, output):
    q, k, positions, inv_freq, axes, ctx.interleaved, ctx.inverse = inputs
    ctx.has_k = k is not None
    # a constant turned is a constant: nothing behind it works out a gradient
    ctx.mark_non_differentiable(*(y for x, y in zip((q, k), output) if x is None or not x.requires_grad))
    ctx.save_for_backward(positions, inv_freq, axes)
    ctx.set_materialize_grads(False)


def _rotate_backward(ctx, gq, gk):
    turned = lambda x, y: _rotate_op(x, y, *ctx.saved_tensors, ctx.interleaved, not ctx.inverse)  # noqa: E731
    dq = dk = None
    gk = gk if ctx.has_k else None
    if gq is not None:
        dq, dk = turned(gq, gk)
        dk = dk if gk is not None else None
    elif gk is not None:
        dk, _ = turned(gk, None)
    return dq, dk, None, None, None, None, None


_rotate_op.register_autograd(_rotate_backward, setup_context=_rotate_setup)


@torch.library.custom_op("chill_attention::rotate_append", mutates_args=("k_cache", "v_cache"), device_types=("cuda",))
def _append_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
               inv_freq: torch.Tensor, axes: typing.Optional[torch.Tensor], interleaved: bool) -> torch.Tensor:
    _check_append(q, k, v, k_cache, v_cache, slots, positions, ChillRotary(inv_freq, axes, interleaved))
    return _eager.extension().rotate_append(_native(), q, k, v, k_cache, v_cache, slots, positions, inv_freq, axes, interleaved)


@_append_op.register_fake
def _(q, k, v, k_cache, v_cache, slots, positions, inv_freq, axes, interleaved):
    return torch.empty_like(q)


# ------------------------------------------------------------------------------------------------------------ public calls
def chill_rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: ChillRotary):
    """q and k turned to ``positions``, as new tensors; differentiable in q and k (the gradient is turned back).

    Args:
        q: [batch, heads, tokens, channels], fp16 / bf16 / fp32, any strides.
        k: the same with kv_heads, or None: q alone is turned.
        positions: int32 [batch, tokens], or for several axes (``rotary.axes``) [axes, batch, tokens]; any strides (``.expand`` for one row of positions).
            A pair whose axis is beyond the rows takes the last one: with one row every axis has it.
        rotary: frequencies, axes and pairing.

    Returns: (q, k) turned, with the strides of the inputs where these are dense; k is None where it was.
    """
    if cache._direct():
        out = _eager.extension().rotate(_NATIVE or _native(), q, k, positions, *rotary, False)
        if out is not None:
            return out
    _check_rotate(q, k, positions, rotary)
    if not torch.compiler.is_compiling():
        assert all(x is None or forward_ad.unpack_dual(x).tangent is None for x in (q, k)), "there is no forward-mode derivative: q or k carries a tangent"
    q_out, k_out = _rotate_op(q, k, positions, *rotary, False)
    return q_out, k_out if k is not None else None


def chill_rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, step: cache.ChillStep,
                        rotary: ChillRotary, positions: torch.Tensor | None = None) -> torch.Tensor:
    """The new tokens of a step: k is turned and stored in the cache together with v, in place, and q is returned turned.  What
    ``chill_rotate`` and ``chill_cache_append`` do one after the other, in one launch and without k in between.

    Args:
        q: [batch, heads, max_new, head_dim]; k, v: [batch, kv_heads, max_new, head_dim]; any strides.
        k_cache, v_cache: [num_pages, kv_heads, page_size, head_dim], any strides; the rows of ``step.slots`` are written (-1: none).
        step: of ``chill_pages_reserve``.
        positions: default ``step.positions``; for several axes int32 [axes, batch, max_new].  With one row of positions every axis has these
            (a pair whose axis is beyond the rows takes the last one).

    There are no gradients: tensors that require them are refused.
    """
    if positions is None:
        positions = step.positions
    if cache._direct():
        out = _eager.extension().rotate_append(_NATIVE or _native(), q, k, v, k_cache, v_cache, step.slots, positions, *rotary)
        if out is not None:
            return out
    _check_append(q, k, v, k_cache, v_cache, step.slots, positions, rotary)
    return _append_op(q, k, v, k_cache, v_cache, step.slots, positions, *rotary)
