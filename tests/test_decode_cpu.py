"""Rotary positions, beam selection, shared pages and page copies without a GPU: C structs, refusals, the oracle's own consistency."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from helpers import ROOT, ensure_built
from oracle import decode_oracle as orc


@pytest.fixture(scope="module")
def lib():
    ensure_built()
    from chill_attention import _decode_abi

    return _decode_abi.load_library()


def test_struct_sizes_match_header():
    from chill_attention import _decode_abi as abi

    assert ctypes.sizeof(abi.RotateArgs) == 40 + 24 + 24 + 16 + 64 + 16 + 64 + 8 + 32 + 16 + 64 + 8 + 8
    assert ctypes.sizeof(abi.SelectArgs) == 16 + 8 * 11
    assert ctypes.sizeof(abi.ShareArgs) == 16 + 16 + 8 * 13 + 8
    assert ctypes.sizeof(abi.CopyArgs) == 24 + 16 + 80 + 32 + 8


def test_header_and_exports(lib, tmp_path):
    """Everything include/chill_decode.h declares is exported, the header is plain C99, and its structs have the binding's sizes."""
    from chill_attention import _decode_abi as abi

    text = open(os.path.join(ROOT, "include", "chill_decode.h")).read()
    names = set(re.findall(r"\b(chill_[a-z_0-9]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(abi.EXPORTS) and all(hasattr(lib, n) for n in names)
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    src = tmp_path / "use.c"
    src.write_text('#include "chill_decode.h"\n#include <stdio.h>\nint main(void) {\n'
                   '  printf("%zu %zu %zu %zu", sizeof(chill_rotate_args), sizeof(chill_select_args), sizeof(chill_share_args), sizeof(chill_copy_args));\n'
                   "  return chill_beam_select(0, 0) == CHILL_E_INVALID && chill_decode_abi_version() == CHILL_DECODE_ABI_VERSION ? 0 : 1; }\n")
    exe, lib_dir = tmp_path / "use", os.path.dirname(abi.DEFAULT_LIB)
    r = subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-L", lib_dir,
                        "-l:libchill_decode_b200.so", f"-Wl,-rpath,{lib_dir}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0
    assert [int(n) for n in out.stdout.split()] == [ctypes.sizeof(t) for t in (abi.RotateArgs, abi.SelectArgs, abi.ShareArgs, abi.CopyArgs)]


def made(cls, pointers, **values):
    a = cls()
    for name in pointers:
        setattr(a, name, 4096)
    for name, value in values.items():
        if isinstance(value, tuple):
            value = (ctypes.c_int64 * len(value))(*value)
        setattr(a, name, value)
    return ctypes.byref(a)


def test_rotation_refusals(lib):
    from chill_attention import _decode_abi as abi

    def call(append=False, **changes):
        pointers = ["inv_freq", "positions", "q", "k", "q_out", "k_out"] + (["v", "k_cache", "v_cache", "slots"] if append else [])
        sizes = dict(B=2, H=4, H_kv=2, L=8, D=64, dtype=2, pairs=32, n_axes=1, num_pages=10, page_size=16)
        args = made(abi.RotateArgs, pointers, **{**sizes, **changes})
        return (lib.chill_rotate_append if append else lib.chill_rotate)(args, None)

    assert lib.chill_rotate(None, None) == lib.chill_rotate_append(None, None) == -1
    for append in (False, True):
        for name in ("B", "H", "H_kv", "L", "D", "pairs", "n_axes"):
            assert call(append, **{name: 0}) == call(append, **{name: -2}) == -1, name
        assert call(append, pairs=33) == -1 and call(append, dtype=5) == -2 and call(append, interleaved=2) == -1 and call(append, inverse=-1) == -1
        assert call(append, B=2 ** 15, L=2 ** 15, D=64) == -4 and call(append, B=2 ** 30, L=2 ** 30) == -4
        for name in ("inv_freq", "positions", "q_out"):
            assert call(append, **{name: None}) == -1, name
    assert call(k_out=None) == -1 and call(q=None, k=None) == -1
    for name in ("q", "k", "v", "k_cache", "v_cache", "slots"):
        assert call(True, **{name: None}) == -1, name
    assert call(True, inverse=1) == -1 and call(True, num_pages=0) == -1 and call(True, page_size=0) == -1
    assert call(True, num_pages=2 ** 28, page_size=16) == -4


def test_selection_refusals(lib):
    from chill_attention import _decode_abi as abi

    def call(**changes):
        return lib.chill_beam_select(made(abi.SelectArgs, ("logits", "scores", "out_scores", "out_rows", "out_tokens", "workspace"),
                                          **{**dict(G=2, K=4, M=4, dtype=0, V=100, row_stride=100, workspace_bytes=1 << 20), **changes}), None)

    assert lib.chill_beam_select(None, None) == -1
    for name in ("G", "K", "M", "V"):
        assert call(**{name: 0}) == call(**{name: -1}) == -1
    assert call(dtype=3) == -2
    assert call(K=65) == call(M=65) == call(V=2 ** 30 + 1) == call(G=20000) == -4
    assert call(K=1, V=3) == -1  # fewer candidates than are asked for
    for name in ("logits", "scores", "out_scores", "out_rows", "out_tokens", "workspace"):
        assert call(**{name: None}) == -1
    assert call(workspace=4104) == call(workspace_bytes=100) == -1
    assert call(finished=4096, end_token=100) == call(finished=4096, end_token=-1) == -1


def test_the_largest_vocabulary(lib):
    """A token has 26 bits beside its beam and its logit."""
    from chill_attention import _decode_abi as abi

    def call(V):
        return lib.chill_beam_select(made(abi.SelectArgs, ("logits", "scores", "out_scores", "out_rows", "out_tokens"), G=1, K=1, M=1, dtype=0, V=V, row_stride=V), None)

    assert call(2 ** 26 + 1) == call(2 ** 31) == -4
    assert call(2 ** 26) == -1  # what is missing is the workspace


def test_page_refusals(lib):
    from chill_attention import _decode_abi as abi

    every = ("table", "held", "free_pages", "n_free", "shared", "lens", "missing", "parents", "source", "target", "rows", "count", "workspace")

    def args(**changes):
        sizes = dict(B=4, page_size=16, num_pages=100, table_width=20, table_stride=20, workspace_bytes=1 << 20, out_lens=8192)
        return made(abi.ShareArgs, every, **{**sizes, **changes})

    calls = (lib.chill_pages_fork, lib.chill_pages_trim_shared, lib.chill_pages_compact)
    for call in calls:
        assert call(None, None) == -1
        for name in ("B", "page_size", "num_pages", "table_width"):
            assert call(args(**{name: 0}), None) == call(args(**{name: -1}), None) == -1
        for name in ("table", "held", "free_pages", "n_free", "workspace"):
            assert call(args(**{name: None}), None) == -1
        assert call(args(table_stride=19), None) == -1 and call(args(workspace_bytes=100), None) == -1 and call(args(workspace=4100), None) == -1
        assert call(args(B=65536), None) == call(args(num_pages=2 ** 27), None) == call(args(table_width=2 ** 26), None) == -4
        assert call(args(B=60000, table_width=2 ** 20, table_stride=2 ** 20, workspace_bytes=1 << 50), None) == -4
    for name in ("shared", "lens", "missing", "parents", "out_lens", "source", "target", "rows", "count"):
        assert lib.chill_pages_fork(args(**{name: None}), None) == -1, name
    assert lib.chill_pages_fork(args(B=8193, workspace_bytes=1 << 30), None) == -4
    assert lib.chill_pages_fork(args(out_lens=4096), None) == -1  # lens itself
    assert lib.chill_pages_trim_shared(args(shared=None), None) == lib.chill_pages_trim_shared(args(lens=None), None) == -1
    assert lib.chill_pages_compact(args(source=None), None) == lib.chill_pages_compact(args(count=None), None) == -1
    sizes = [lib.chill_share_workspace_bytes(args(**c)) for c in ({}, {"B": 8}, {"num_pages": 10 ** 6}, {"B": 0})]
    assert sizes[0] >= 4 * (4 * 20 + 2 * 4 + 100) and sizes[1] > 0 and sizes[2] > 4 * 10 ** 6 and sizes[3] == 0
    assert lib.chill_share_workspace_bytes(None) == 0

    def copy(**changes):
        return lib.chill_cache_copy(made(abi.CopyArgs, ("k_cache", "source", "target", "rows", "count"),
                                         **{**dict(layers=1, num_pages=10, H_kv=2, page_size=16, D=64, dtype=1, orders=5, v_cache=8192), **changes}), None)

    assert lib.chill_cache_copy(None, None) == -1
    for name in ("layers", "num_pages", "H_kv", "page_size", "D", "orders"):
        assert copy(**{name: 0}) == -1
    for name in ("k_cache", "v_cache", "source", "target", "rows", "count"):
        assert copy(**{name: None}) == -1
    assert copy(dtype=9) == -2 and copy(num_pages=2 ** 28) == -4 and copy(page_size=2 ** 20, D=2 ** 12) == -4
    assert copy(v_cache=4096, k_cache_strides=(1, 2, 3, 4, 5)) == -1  # one tensor in two layouts


def test_public_calls_refuse_what_is_not_on_a_gpu(lib):
    import chill_attention as ca

    x, at = torch.zeros(2, 4, 3, 64), torch.zeros(2, 3, dtype=torch.int32)
    rotary = ca.ChillRotary.of(64, device="cpu")
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_rotate(x, x, at, rotary)
    step = ca.ChillStep(at[:, 0], at[:, 0], at, at, None)
    cache = torch.zeros(8, 4, 16, 64)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_rotate_append(x, x, x, cache, cache, step, rotary)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_beam_select(torch.zeros(4, 10), torch.zeros(2, 2))
    pages, lens, shared = ca.ChillPages.empty(2, 100, 8, 16, device="cpu"), torch.zeros(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    for call in (lambda: ca.chill_pages_fork(pages, shared, lens, lens, 16), lambda: ca.chill_pages_trim(pages, lens, 16, shared=shared),
                 lambda: ca.chill_pages_compact(pages, 16), lambda: ca.chill_cache_copy(cache, cache, ca.ChillCopies(lens, lens, lens, lens[:1]))):
        with pytest.raises(AssertionError, match="CUDA"):
            call()


def test_rotary_handle():
    import chill_attention as ca

    r = ca.ChillRotary.of(8, base=100.0, axes=(0, 1, 1, 2), interleaved=True, device="cpu")
    assert r.inv_freq.dtype == torch.float32 and r.axes.tolist() == [0, 1, 1, 2] and r.interleaved
    assert torch.equal(r.inv_freq, torch.tensor([100.0 ** -(2 * i / 8) for i in range(4)], dtype=torch.float64).float())
    for bad in (dict(channels=7), dict(channels=0), dict(channels=4, axes=(0,)), dict(channels=4, axes=(0, -1))):
        with pytest.raises(AssertionError):
            ca.ChillRotary.of(device="cpu", **bad)


def test_oracle_rotation_turns_and_turns_back():
    x = torch.randn(2, 3, 5, 16, dtype=torch.float64)
    at = torch.randint(0, 1000, (2, 2, 5))
    inv = torch.tensor([1.0, 0.3, 0.01])
    for interleaved in (False, True):
        y = orc.rotate(x, at, inv, [0, 1, 1], interleaved)
        assert torch.equal(y[..., 6:], x[..., 6:]) and torch.allclose(y[..., :6].norm(dim=-1), x[..., :6].norm(dim=-1))
        assert torch.allclose(orc.rotate(y, at, inv, [0, 1, 1], interleaved, inverse=True), x)


def test_oracle_fork_and_trim_keep_every_page_once():
    """Two requests become three beams and end: the stack has every page again."""
    free = list(range(9, -1, -1))
    table, held, n_free, _, _, _, _ = __import__("oracle.cache_oracle", fromlist=["reserve"]).reserve([[-1] * 4 for _ in range(3)], [0] * 3, free, 10, [0] * 3, [10, 5, 0], 16, 4)
    shared = [0] * 10
    table, held, stack, shared, missing, lens, copies = orc.fork(table, held, free, n_free, shared, [10, 5, 0], [0, 0, 0], 4)
    assert lens == [10, 10, 10] and missing == 0 and len(copies) == 2 and sorted(shared) == [0] * 8 + [2, 2]
    assert copies[0][0] == copies[1][0] == table[0][2] and {c[2] for c in copies} == {2}
    table, held, stack, shared = orc.trim_shared(table, held, stack + [0] * (10 - len(stack)), len(stack), shared, [0, 0, 0], 4)
    assert sorted(stack) == list(range(10)) and shared == [0] * 10 and held == [0, 0, 0]


def test_oracle_select():
    x = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]], dtype=torch.float64))
    values, rows, tokens = orc.select(x, torch.tensor([[0.0, -1.0]]), 4)
    assert rows.tolist() == [[0, 1, 0, 0]] and tokens.tolist() == [[0, 2, 1, 2]]
    assert torch.allclose(values, torch.log(torch.tensor([[0.5, 0.8 / 2.718281828459045, 0.25, 0.25]], dtype=torch.float64)))
