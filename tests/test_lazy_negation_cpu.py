"""Attention over a sharded sequence hands its kernels tensors whose memory holds the numbers themselves, without a sign that is still to be applied."""
import pytest
import torch
import torch.distributed as dist

from test_dist_cpu import _oracle_local_backward, _oracle_local_forward


@pytest.fixture
def alone():
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    yield
    dist.destroy_process_group()


@pytest.mark.parametrize("which", range(4))
def test_sharded_attention(alone, which):
    import chill_attention as ca
    from chill_attention.dist import HaloBuffer, sequence_sharded_attention

    def stored(call):
        def checked(mask, *args, **kwargs):
            assert not any(isinstance(t, torch.Tensor) and t.is_neg() for t in (*args, *kwargs.values()))
            return call(mask, *args, **kwargs)
        return checked

    g = torch.Generator().manual_seed(4)
    tensors = [torch.randn(1, h, 24, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4)]  # q, k, v, gradient
    mask = ca.SlidingWindowChillMask(6, 0)

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = sequence_sharded_attention(*leaves, mask, 24, local_forward=stored(_oracle_local_forward), local_backward=stored(_oracle_local_backward))
        return o, *torch.autograd.grad(o, leaves, do)

    want = step(*tensors)
    negated = list(tensors)
    negated[which] = torch._neg_view(-tensors[which])
    for x, y in zip(step(*negated), want):
        assert torch.equal(x, y)
    buffers = [HaloBuffer.like(t, 6, 0) for t in tensors[1:3]]
    with pytest.raises(ValueError, match="halo_buffers"):
        sequence_sharded_attention(tensors[0], torch._neg_view(buffers[0].local), buffers[1].local, mask, 24, halo_buffers=buffers)
