"""GPU: the adapters' calls on a stream that is not the current one."""
import pytest
import torch

from _lora import Problem, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["stream", "handle", "default"])
def test_buffers_come_from_the_streams_own_pool(ks, cuda, monkeypatch, form):
    """What plan and backward allocate belongs to the stream that their kernels run on: a block of the current stream's pool may have been
    freed there while kernels of the current stream, which the other does not wait for, still use it."""
    side = torch.cuda.Stream()
    handle = 0 if form == "default" else side.cuda_stream
    stream = side if form == "stream" else handle
    p = Problem(300, 3, 16, 128, 256, seed=1)
    made = []
    empty = torch.empty

    def watched(*size, **how):
        made.append(torch.cuda.current_stream().cuda_stream)
        return empty(*size, **how)

    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):     # neither the default stream nor the call's
        out, d_x, d_a, d_b = torch.empty_like(p.base), torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b)
        h = torch.empty(300, 16, device=cuda)
        torch.cuda.synchronize()
        monkeypatch.setattr(torch, "empty", watched)
        ids, offsets = ks.lora.plan(p.ids, p.adapters, stream=stream)
        ks.lora.apply(out, p.base, p.x, p.a, p.b, p.scales, ids, offsets, h=h, stream=stream)
        ks.lora.backward(d_x, d_a, d_b, p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales, ids, offsets, stream=stream)
        monkeypatch.undo()
        here = torch.cuda.current_stream().cuda_stream
    assert len(made) == 3 and set(made) == {handle} and here != handle
    torch.cuda.synchronize()
    want, bound, hd, _ = p.forward()
    check("out", out, want, bound)
    grads, bounds = p.backward(hd.float())
    for what, x, y, b in zip(("d_x", "d_a", "d_b"), (d_x, d_a, d_b), grads, bounds):
        check(what, x, y, b * 1.01)   # (the forward pass's own h instead of the 64-bit one)


def test_a_block_that_the_current_stream_still_reads_is_not_taken(ks, cuda):
    """A tensor is freed while a long run of the current stream's kernels has yet to read it; the call on another stream leaves it alone."""
    p = Problem(2048, 3, 16, 128, 256, seed=1)
    ids, offsets = ks.lora.plan(p.ids, p.adapters)
    h = torch.zeros(2048, 16, device=cuda)
    d_x, d_a, d_b = torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b)
    size = ks.lora.backward_workspace(2048, 3, 16, 128, 256)
    side = torch.cuda.Stream()
    total = torch.zeros(1, device=cuda)
    big = torch.randn(8192, 8192, device=cuda)
    torch.cuda.synchronize()
    block = torch.full((size // 4,), 1.0, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        big = big @ big * 1e-2                       # milliseconds
    total += block.sum()
    del block
    ks.lora.backward(d_x, d_a, d_b, p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales, ids, offsets, stream=side)
    torch.cuda.synchronize()
    assert float(total) == size // 4
