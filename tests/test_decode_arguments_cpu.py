"""Arguments of include/chill_decode.h that contradict one another or are too large, and shapes that say nothing of what is meant: refused without a GPU."""
import ctypes

import pytest
import torch

from helpers import ensure_built
from test_decode_cpu import made


@pytest.fixture(scope="module")
def lib():
    ensure_built()
    from chill_attention import _decode_abi

    return _decode_abi.load_library()


def test_a_result_without_its_input(lib):
    """q or k may be missing, but not while there is a place for the result: nobody would write it."""
    from chill_attention import _decode_abi as abi

    def call(**changes):
        sizes = dict(B=2, H=4, H_kv=2, L=8, D=64, dtype=2, pairs=32, n_axes=1)
        return lib.chill_rotate(made(abi.RotateArgs, ["inv_freq", "positions", "q", "k", "q_out", "k_out"], **{**sizes, **changes}), None)

    assert call(q=None) == call(k=None) == call(q_out=None) == call(k_out=None) == -1
    assert call(q=None, q_out=None, H_kv=0) == call(k=None, k_out=None, H=0) == -1


def test_rows_of_positions_and_axes():
    from chill_attention import ChillRotary, rotary

    x, at = torch.zeros(2, 4, 3, 16), torch.zeros(3, 2, 3, dtype=torch.int32)
    plain, three = ChillRotary.of(16, device="cpu"), ChillRotary.of(16, axes=(0, 1, 2, 2, 1, 0, 0, 0), device="cpu")
    with pytest.raises(AssertionError, match="rotary.axes"):
        rotary._check_where(x, at, plain)
    for positions, which in ((at, three), (at[:2], three), (at[:1], three), (at[0], three), (at[:1], plain), (at[0], plain)):
        rotary._check_where(x, positions, which)


def test_pools_of_so_many_pages_that_their_numbers_leave_32_bits(lib):
    """A cluster's shares of 2^31 - 1 pages end beyond what an int holds."""
    from chill_attention import _decode_abi as abi

    every = ("table", "held", "free_pages", "n_free", "shared", "lens", "missing", "parents", "source", "target", "rows", "count", "workspace")

    def args(num_pages, **changes):
        return made(abi.ShareArgs, every, **{**dict(B=4, page_size=1, num_pages=num_pages, table_width=20, table_stride=20, workspace_bytes=1 << 40, out_lens=8192), **changes})

    for n in (2 ** 31 - 1, 2 ** 31 - 8, 2 ** 30 + 1):
        assert lib.chill_share_workspace_bytes(args(n)) == 0
        assert all(call(args(n), None) == -4 for call in (lib.chill_pages_fork, lib.chill_pages_trim_shared, lib.chill_pages_compact))
    assert lib.chill_share_workspace_bytes(args(2 ** 30)) > 4 * 2 ** 30
    assert all(call(args(2 ** 30, workspace_bytes=100), None) == -1 for call in (lib.chill_pages_fork, lib.chill_pages_trim_shared, lib.chill_pages_compact))
