"""Paged cache without a GPU: C structs, refusals of the C ABI and of the public functions, the oracle's own consistency."""
import ctypes

import pytest
import torch

from helpers import ensure_built
from oracle import cache_oracle as orc


@pytest.fixture(scope="module")
def lib():
    ensure_built()
    from chill_attention import _cache_abi

    return _cache_abi.load_library()


def cached_args(**changes):
    from chill_attention import _cabi, _cache_abi

    a = _cache_abi.CachedArgs()
    a.mask = _cabi.mask_desc(_cabi.MASK_CAUSAL, ())
    a.B, a.H, a.H_kv, a.N, a.D, a.dtype = 2, 8, 2, 4, 64, 2
    a.page_size, a.num_pages, a.table_width, a.sm_scale = 16, 100, 20, 0.125
    a.q = a.k_cache = a.v_cache = a.o = a.table = a.lens = a.new_lens = a.workspace = 4096
    row = 64
    for name, st in (("q_strides", (8 * 4 * row, 4 * row, row, 1)), ("o_strides", (8 * 4 * row, 4 * row, row, 1)),
                     ("k_cache_strides", (2 * 16 * row, 16 * row, row, 1)), ("v_cache_strides", (2 * 16 * row, 16 * row, row, 1))):
        setattr(a, name, (ctypes.c_int64 * 4)(*st))
    a.table_stride = 20
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def test_struct_sizes_match_header():
    from chill_attention import _cache_abi

    assert ctypes.sizeof(_cache_abi.PagesArgs) == 24 + 8 * 2 + 8 * 10
    assert ctypes.sizeof(_cache_abi.CacheRowsArgs) == 40 + 16 + 64 + 16 + 64 + 8 + 16 + 8 * 5
    assert ctypes.sizeof(_cache_abi.CachedArgs) == 136 + 48 + 40 + 128 + 24 + 16 + 48


def test_attention_refusals(lib):
    call = lambda **c: lib.chill_cached_fwd(ctypes.byref(cached_args(**c)), None)  # noqa: E731
    assert lib.chill_cached_fwd(None, None) == -1
    for name in ("B", "H", "H_kv", "N", "D", "page_size", "num_pages", "table_width"):
        assert call(**{name: 0}) == -1, name
        assert call(**{name: -3}) == -1, name
    for name in ("q", "k_cache", "v_cache", "o", "table", "lens", "new_lens", "workspace"):
        assert call(**{name: None}) == -1, name
    assert call(H=9) == -1                                      # not a multiple of the kv heads
    assert call(dtype=7) == -2 and call(D=272) == -2 and call(D=20) == -2
    assert call(sm_scale=0.0) == -1 and call(sm_scale=-1.0) == -1 and call(sm_scale=float("nan")) == -1 and call(sm_scale=float("inf")) == -1
    assert call(num_pages=2 ** 27, page_size=16) == -4          # slots pass 31 bits
    assert call(table_width=2 ** 26, page_size=16, num_pages=2) == -4
    assert call(B=70000) == -4 and call(H=70000) == -4
    assert call(workspace_bytes=0) == -1 and call(workspace=4096 + 8, workspace_bytes=1 << 40) == -1
    assert call(ancestors=4096, positions=None) == -1
    a = cached_args()
    a.mask.id = 17
    assert lib.chill_cached_fwd(ctypes.byref(a), None) == -2
    assert lib.chill_cached_workspace_bytes(ctypes.byref(cached_args())) > 0
    assert lib.chill_cached_workspace_bytes(ctypes.byref(cached_args(D=20))) == 0
    assert lib.chill_cached_kernel(ctypes.byref(cached_args(D=20))) == -2


def test_page_and_row_refusals(lib):
    from chill_attention import _cache_abi

    def pages(**changes):
        a = _cache_abi.PagesArgs()
        a.B, a.N, a.page_size, a.num_pages, a.table_width, a.table_stride = 4, 3, 16, 100, 20, 20
        for name in ("table", "held", "free_pages", "n_free", "missing", "lens", "new_lens", "slots", "positions"):
            setattr(a, name, 4096)
        for name, value in changes.items():
            setattr(a, name, value)
        return ctypes.byref(a)

    assert lib.chill_pages_reserve(None, None) == lib.chill_pages_trim(None, None) == -1
    for name in ("B", "page_size", "num_pages", "table_width"):
        assert lib.chill_pages_reserve(pages(**{name: 0}), None) == lib.chill_pages_trim(pages(**{name: -1}), None) == -1
    for name in ("table", "held", "free_pages", "n_free", "lens"):
        assert lib.chill_pages_reserve(pages(**{name: None}), None) == lib.chill_pages_trim(pages(**{name: None}), None) == -1
    for name in ("missing", "new_lens", "slots", "positions"):
        assert lib.chill_pages_reserve(pages(**{name: None}), None) == -1
    assert lib.chill_pages_reserve(pages(N=0), None) == -1
    assert lib.chill_pages_reserve(pages(parents=4096), None) == lib.chill_pages_reserve(pages(ancestors=4096), None) == -1
    assert lib.chill_pages_reserve(pages(table_stride=19), None) == -1
    assert lib.chill_pages_reserve(pages(B=65536), None) == lib.chill_pages_reserve(pages(num_pages=2 ** 27), None) == -4
    assert lib.chill_pages_trim(pages(table_width=2 ** 26), None) == -4

    for name in ("lens", "new_lens", "held", "table", "slots"):  # stored is an array of its own
        assert lib.chill_pages_reserve_stored(pages(**{name: 8192}), 8192, None) == -1
    # sums of pages over the requests are 32 bits wide: tables with more entries than that
    for B, width in ((65535, 2 ** 16), (8, 2 ** 28), (5, 2 ** 29)):
        big = pages(B=B, page_size=1, num_pages=2 ** 30, table_width=width, table_stride=width)
        assert lib.chill_pages_reserve(big, None) == lib.chill_pages_reserve_stored(big, None, None) == lib.chill_pages_trim(big, None) == -4

    def rows(**changes):
        a = _cache_abi.CacheRowsArgs()
        a.B, a.H_kv, a.N, a.D, a.dtype, a.page_size, a.num_pages, a.table_width, a.A = 4, 2, 3, 64, 2, 16, 100, 20, 2
        for name in ("k_cache", "v_cache", "k", "v", "slots", "table", "lens", "new_lens", "path", "accepted", "out_lens"):
            setattr(a, name, 4096)
        for name, value in changes.items():
            setattr(a, name, value)
        return ctypes.byref(a)

    for call in (lib.chill_cache_append, lib.chill_cache_commit):
        assert call(None, None) == -1
        for name in ("B", "H_kv", "N", "D", "page_size", "num_pages"):
            assert call(rows(**{name: 0}), None) == -1
        assert call(rows(dtype=5), None) == -2 and call(rows(num_pages=2 ** 27), None) == -4 and call(rows(k_cache=None), None) == -1
    for name in ("k", "v", "slots"):
        assert lib.chill_cache_append(rows(**{name: None}), None) == -1
    for name in ("table", "lens", "new_lens", "path", "accepted", "out_lens"):
        assert lib.chill_cache_commit(rows(**{name: None}), None) == -1
    assert lib.chill_cache_commit(rows(), None) == -1  # out_lens is lens: the CTAs of a request all read its length
    strides = (ctypes.c_int64 * 4)(2048, 1024, 64, 1)
    apart = dict(out_lens=8192, k_cache_strides=strides)  # one tensor for K and V, in two layouts
    assert lib.chill_cache_commit(rows(**apart), None) == -1
    assert lib.chill_cache_commit(rows(A=0), None) == -1 and lib.chill_cache_commit(rows(table_width=0), None) == -1


def test_cpu_tensors_are_refused(lib):
    import chill_attention as ca

    pages = ca.ChillPages.empty(2, 100, 8, 16, device="cpu")
    assert pages.table.shape == (2, 7) and pages.free.tolist() == list(range(7, -1, -1)) and pages.n_free.item() == 8
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_pages_reserve(pages, lens, lens, 1, 16)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_pages_trim(pages, lens, 16)
    cache = torch.zeros(8, 2, 16, 64)
    step = ca.ChillStep(lens, lens, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32), None)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_cache_append(cache, cache, torch.zeros(2, 2, 3, 64), torch.zeros(2, 2, 3, 64), step.slots)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_cache_commit(cache, cache, pages.table, step, step.slots, lens)
    with pytest.raises(AssertionError, match="CUDA"):
        ca.chill_attention_cached(torch.zeros(2, 4, 3, 64), cache, cache, pages.table, step, ca.CausalChillMask())


def test_two_mask_classes_of_one_name():
    from chill_attention import CausalChillMask, cache

    def make(functor, **more):
        return type("OneName", (CausalChillMask,), {"cuda_functor": functor, **more})()

    first = make("CausalMask")
    cache._MASKS["OneName"] = (None, 0, type(first))
    try:
        cache._check_same_name(make("CausalMask"))  # the same functor: whichever class
        for other in (make("FullMask"), make("CausalMask", cuda_functor_header="/tmp/x.h")):
            with pytest.raises(ValueError, match="two mask classes"):
                cache._attention(torch.zeros(1, 1, 1, 64), None, None, None, (None,) * 5, other, None, False, 0)
    finally:
        del cache._MASKS["OneName"]


@pytest.mark.parametrize("fullgraph", [False, True])
def test_two_mask_classes_of_one_name_under_compile(lib, fullgraph):
    """A graph finds its kernel by the class name, so the second class is refused while it is traced too."""
    from chill_attention import CausalChillMask, cache

    def make(functor, **more):
        return type("OneName", (CausalChillMask,), {"cuda_functor": functor, **more})()

    def run(mask):
        torch._dynamo.reset()
        call = lambda q: cache._attention(q, q, q, q, (q,) * 5, mask, None, False, 0)  # noqa: E731
        return torch.compile(call, backend="eager", fullgraph=fullgraph)(torch.zeros(1, 1, 1, 64))

    first = make("CausalMask")
    cache._MASKS["OneName"] = (cache._native(), 1, type(first))
    try:
        for other in (make("FullMask"), make("CausalMask", cuda_functor_header="/tmp/x.h")):
            with pytest.raises(Exception, match="two mask classes"):
                run(other)
        for same in (first, make("CausalMask")):  # goes on, to the next check
            with pytest.raises(Exception, match="CUDA tensors"):
                run(same)
    finally:
        del cache._MASKS["OneName"]
        torch._dynamo.reset()


def test_the_switch_of_the_eager_path(monkeypatch):
    """CHILL_ATTENTION_EAGER_FAST=0 sends these calls to the dispatcher ops too."""
    from chill_attention import _eager, cache

    monkeypatch.setattr(_eager, "ENABLED", True)
    assert cache._direct()
    monkeypatch.setattr(_eager, "ENABLED", False)
    assert not cache._direct()


def test_oracle_trim_undoes_reserve():
    table, held, free = [[5, -1, -1, -1], [-1] * 4, [7, 2, -1, -1]], [1, 0, 2], [9, 8, 6, 4, 3, 1, 0]
    lens, new = [10, 0, 20], [30, 16, 0]
    t, h, n, missing, slots, positions, _ = orc.reserve(table, held, free, len(free), lens, new, 32, 16)
    assert t == [[5, 0, 1, -1], [3, -1, -1, -1], [7, 2, -1, -1]] and h == [3, 1, 2] and n == 4 and missing == 0
    assert slots[0][:7] == [5 * 16 + 10 + i for i in range(6)] + [0] and positions[1][:3] == [0, 1, 2] and slots[2] == [-1] * 32
    t, h, stack = orc.trim(t, h, free, n, lens, 16)
    assert (t, h, stack) == (table, held, free)


def test_header_and_exports(lib, tmp_path):
    """Everything include/chill_cache.h declares is exported, and the header is plain C99."""
    import os
    import re
    import shutil
    import subprocess

    from chill_attention import _cache_abi
    from helpers import ROOT

    text = open(os.path.join(ROOT, "include", "chill_cache.h")).read()
    names = set(re.findall(r"\b(chill_[a-z_0-9]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(_cache_abi.EXPORTS) and all(hasattr(lib, n) for n in names)
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    src = tmp_path / "use.c"
    src.write_text('#include "chill_cache.h"\nint main(void) { chill_cached_args a = {0}; chill_pages_args b = {0}; chill_cache_rows_args c = {0};\n'
                   "  (void)b; (void)c; return chill_cached_fwd(&a, 0) == CHILL_E_INVALID && chill_cache_abi_version() == CHILL_CACHE_ABI_VERSION ? 0 : 1; }\n")
    exe, lib_dir = tmp_path / "use", os.path.dirname(_cache_abi.DEFAULT_LIB)
    r = subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-L", lib_dir,
                        "-l:libchill_cache_b200.so", f"-Wl,-rpath,{lib_dir}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(exe)]).returncode == 0
