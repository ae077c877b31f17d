"""GPU: gradients of the routed layer's steps written over what they are made from: the same bits as beside it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (60, 7), (64, 8), (256, 8), (257, 32), (1024, 32)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gate(ks, cuda, dtype, experts, top_k, renormalize):
    tokens = 1000
    g = torch.Generator(device=cuda).manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g, device=cuda).to(dtype)
    w, idx = torch.topk(torch.softmax(logits.float(), 1), top_k, dim=1)
    idx, d_w = idx.to(torch.int32), torch.randn(tokens, top_k, generator=g, device=cuda)
    call = lambda out, l: ks.moe.gate_softmax_topk_backward(out, d_w, w, idx, l, tokens, experts, top_k, renormalize=renormalize)  # noqa: E731
    beside = call(torch.empty_like(logits), logits)
    for _ in range(5):
        over = logits.clone()
        call(over, over)
        assert torch.equal(over, beside)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,top_k,hidden", [(5, 3, 33), (300, 8, 1024)])
def test_weighted_sum(ks, cuda, dtype, tokens, top_k, hidden):
    g = torch.Generator(device=cuda).manual_seed(tokens)
    ids = torch.randperm(tokens * top_k, generator=g, device=cuda).to(torch.int32)
    ids[::7] = -1
    permuted, d_out = (torch.randn(r, hidden, generator=g, device=cuda).to(dtype) for r in (tokens * top_k, tokens))
    w = torch.rand(tokens, top_k, generator=g, device=cuda)
    beside = ks.moe.unpermute_backward(torch.empty_like(permuted), torch.empty_like(w), d_out, permuted, ids, w, tokens, top_k, hidden)
    over = permuted.clone()
    d_w = torch.empty_like(w)
    ks.moe.unpermute_backward(over, d_w, d_out, over, ids, w, tokens, top_k, hidden)
    assert torch.equal(over, beside[0]) and torch.equal(d_w, beside[1])
