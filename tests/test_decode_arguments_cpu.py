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
