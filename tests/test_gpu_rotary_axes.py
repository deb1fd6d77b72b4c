"""Rows of positions, the axes that name them, and frequencies."""
import pytest
import torch

from oracle import decode_oracle as orc
from test_gpu_decode import check_turned, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca():
    import chill_attention

    return chill_attention


def test_rows_of_positions_that_nothing_names_are_refused(ca):
    x, at, rotary = torch.randn(2, 4, 3, 64, device="cuda"), torch.zeros(3, 2, 3, dtype=torch.int32, device="cuda"), ca.ChillRotary.of(64)
    with pytest.raises(AssertionError, match="rotary.axes"):
        ca.chill_rotate(x, None, at, rotary)
    cache = torch.zeros(8, 4, 16, 64, device="cuda")
    step = ca.ChillStep(ints([0, 0]), ints([3, 3]), ints([[0, 1, 2], [16, 17, 18]]), at[0].contiguous(), None)
    with pytest.raises(AssertionError, match="rotary.axes"):
        ca.chill_rotate_append(x, x, x, cache, cache.clone(), step, rotary, at)
    assert not cache.any()
    assert torch.equal(ca.chill_rotate(x, None, at[:1], rotary)[0], ca.chill_rotate(x, None, at[0], rotary)[0])  # one row, said with its axis


@pytest.mark.parametrize("rows", [1, 2])
def test_axes_beyond_the_rows_take_the_last_one(ca, rows):
    g = torch.Generator().manual_seed(1)
    which = [0, 1, 2, 2, 1, 0, 5, 1]
    rotary = ca.ChillRotary.of(16, axes=which)
    x = torch.randn(2, 3, 9, 24, generator=g).cuda()
    positions = torch.randint(0, 400, (rows, 2, 9), generator=g, dtype=torch.int32).cuda()
    y, _ = ca.chill_rotate(x, None, positions, rotary)
    check_turned(y, x, orc.rotate(x, positions, rotary.inv_freq, which), 8, False, torch.float32)
    if rows == 1:  # a step's own positions: every axis has these
        assert torch.equal(y, ca.chill_rotate(x, None, positions[0], rotary)[0])


def test_frequencies_that_ask_for_gradients(ca):
    """Refused while gradients are recorded, taken where they are not, whichever way a call goes."""
    from chill_attention import _eager

    x, at = torch.randn(1, 2, 3, 8, device="cuda"), ints([[4, 5, 6]])
    rotary = ca.ChillRotary.of(8)
    held = rotary._replace(inv_freq=rotary.inv_freq.clone().requires_grad_())
    want = ca.chill_rotate(x, None, at, rotary)[0]
    for fast in (True, False):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(_eager, "ENABLED", fast)
            with pytest.raises(AssertionError, match="gradient"):
                ca.chill_rotate(x, None, at, held)
            with torch.no_grad():
                assert torch.equal(ca.chill_rotate(x, None, at, held)[0], want)
