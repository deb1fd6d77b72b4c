"""Forks and trims whose shared memory lies just around what a kernel gets without asking for more, as the first calls of a process: a larger call before them would
have raised the limit for them.  Run as a script this file is that process."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "chill-attention_b200"), ROOT, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)

pytestmark = pytest.mark.gpu

# what, requests, blocks of a table's row: each the first call of a kernel of its own (tables in shared memory or not), 49008 to 49152 bytes beside the 144 that it always has
EDGES = [("fork", 256, 704), ("fork", 256, 705), ("fork", 16, 1475), ("fork", 4896, 128), ("trim", 64, 1482), ("trim", 192, 740), ("trim", 65535, 16)]


def run(what, B, width):
    import chill_attention as ca
    from oracle import decode_oracle as orc
    from test_gpu_decode import check_pages, copies_of, state_of

    page, g = 4, torch.Generator().manual_seed(B)
    lens = torch.randint(0, 12, (B,), generator=g, dtype=torch.int32)
    lens[B // 2] = width * page  # one row is full
    num_pages = int(((lens + page - 1) // page).sum()) + B
    pages, shared = ca.ChillPages.empty(B, width * page, num_pages, page), torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    lens = lens.cuda()
    ca.chill_pages_reserve(pages, torch.zeros_like(lens), lens, int(lens.max()), page)
    before = state_of(pages, shared)
    if what == "trim":
        lens = lens // 2
        ca.chill_pages_trim(pages, lens, page, shared=shared)
        table, held, stack, counts = orc.trim_shared(*before, lens.tolist(), page)
        check_pages(pages, shared, table, held, stack, counts)
        return
    parents = torch.arange(B, dtype=torch.int32, device="cuda") // 2 * 2
    after, copies = ca.chill_pages_fork(pages, shared, lens, parents, page)
    table, held, stack, counts, missing, out, orders = orc.fork(*before, lens.tolist(), parents.tolist(), page)
    check_pages(pages, shared, table, held, stack, counts)
    assert after.tolist() == out and copies_of(copies) == orders and pages.missing.item() == missing


@pytest.mark.parametrize("what,B,width", EDGES)
def test_the_first_call_of_a_process(what, B, width):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), what, str(B), str(width)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


if __name__ == "__main__":
    run(sys.argv[1], int(sys.argv[2]), int(sys.argv[3]))
