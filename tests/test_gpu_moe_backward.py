"""GPU: gradients of the routed layer's steps, against 64 bits.

Bounds: u = eps(T)/2 for the one rounding of an output; a fp32 sum of n terms is off by at most n * 2^-24 times the sum
of the magnitudes, whatever its order; expf by two units in the last place, 2^-22."""
import pytest
import torch

from _lora import check, half_step

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
ULP = 2.0 ** -24


def _routing(ks, tokens, experts, top_k, dropped, cuda, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    idx = torch.rand(tokens, experts, generator=g, device=cuda).topk(top_k, 1).indices.to(torch.int32)
    idx = torch.where(torch.rand(tokens, top_k, generator=g, device=cuda) < dropped, -1, idx).contiguous()
    ids = torch.empty(tokens * top_k, dtype=torch.int32, device=cuda)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=cuda)
    ks.moe.compute_permutation(ids, offsets, idx, tokens, experts, top_k)
    return g, ids, offsets


ROWS = [
    (1, 1, 1, 1, 0.0, F32), (1, 8, 8, 7168, 0.0, BF), (3, 4, 2, 5, 0.3, HF), (48, 64, 8, 7168, 0.0, BF),
    (100, 16, 3, 1000, 0.2, F32), (333, 8, 2, 4096, 0.0, HF), (17, 4, 4, 8, 1.0, BF), (600, 256, 8, 264, 0.9, BF),
    (5000, 16, 2, 72, 0.1, HF), (1100, 32, 6, 516, 0.125, F32), (9, 40, 33, 130, 0.1, BF), (40_000, 4, 1, 16, 0.3, BF),
    (2, 8, 8, 28_672, 0.0, F32),
]


@pytest.mark.parametrize("tokens,experts,top_k,hidden,dropped,dtype", ROWS)
def test_unpermute_backward(ks, cuda, tokens, experts, top_k, hidden, dropped, dtype):
    g, ids, _ = _routing(ks, tokens, experts, top_k, dropped, cuda)
    pairs = tokens * top_k
    d_out = torch.randn(tokens, hidden, generator=g, device=cuda).to(dtype)
    permuted = torch.randn(pairs, hidden, generator=g, device=cuda).to(dtype)
    permuted[ids < 0] = float("nan")   # not to be read
    w = torch.rand(tokens, top_k, generator=g, device=cuda)
    d_p, d_w = ks.moe.unpermute_backward(torch.full_like(permuted, 9.0), torch.full_like(w, 9.0), d_out, permuted, ids, w, tokens, top_k,
                                         hidden)
    want_p, want_w, mag = torch.zeros(pairs, hidden, dtype=torch.float64, device=cuda), *(
        torch.zeros(pairs, dtype=torch.float64, device=cuda) for _ in range(2))
    rows = (ids >= 0).nonzero()[:, 0]
    pair = ids[rows].long()
    d = d_out[pair // top_k].double()
    want_p[rows] = w.flatten()[pair].double()[:, None] * d
    want_w[pair] = (d * permuted[rows].double()).sum(1)
    mag[pair] = (d * permuted[rows].double()).abs().sum(1)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    check("d_permuted", d_p, want_p, want_p.abs() * (half_step(dtype) + 2 * ULP) + tiny)
    check("d_weights", d_w.flatten(), want_w, hidden * ULP * mag)
    # over its input
    over = permuted.clone()
    again = ks.moe.unpermute_backward(over, torch.empty_like(w), d_out, over, ids, w, tokens, top_k, hidden)
    assert torch.equal(again[0], d_p) and torch.equal(again[1], d_w)


@pytest.mark.parametrize("tokens,experts,top_k,hidden,dropped,dtype", ROWS)
def test_permute_backward(ks, cuda, tokens, experts, top_k, hidden, dropped, dtype):
    g, ids, _ = _routing(ks, tokens, experts, top_k, dropped, cuda, seed=1)
    d_p = torch.randn(tokens * top_k, hidden, generator=g, device=cuda).to(dtype)
    d_p[ids < 0] = float("nan")   # not to be read
    got = ks.moe.permute_backward(torch.full((tokens, hidden), 9.0, dtype=dtype, device=cuda), d_p, ids, tokens, top_k, hidden)
    want, mag = torch.zeros(2, tokens, hidden, dtype=torch.float64, device=cuda)
    rows = (ids >= 0).nonzero()[:, 0]
    token = ids[rows].long() // top_k
    want.index_add_(0, token, d_p[rows].double())
    mag.index_add_(0, token, d_p[rows].double().abs())
    check("d_input", got, want, half_step(dtype) * (want.abs() + top_k * ULP * mag) + top_k * ULP * mag)


# above 4096 pairs: slots in several groups, rows of several segments, whole and single elements
MANY = [(200, 64, 33, 264, 0.1, BF), (150, 64, 40, 131, 0.1, HF), (700, 16, 9, 1032, 0.0, F32), (520, 32, 12, 130, 0.2, BF),
        (513, 64, 8, 7168, 0.125, BF), (1400, 8, 3, 8200, 0.1, HF), (4200, 8, 1, 4104, 0.0, F32), (2100, 16, 2, 24, 0.9, F32),
        (600, 8, 8, 1024, 1.0, BF)]


@pytest.mark.parametrize("tokens,experts,top_k,hidden,dropped,dtype", MANY)
def test_permute_backward_many_pairs(ks, cuda, tokens, experts, top_k, hidden, dropped, dtype):
    test_permute_backward(ks, cuda, tokens, experts, top_k, hidden, dropped, dtype)


@pytest.mark.parametrize("tokens", [50, 3000])
def test_unaligned_rows(ks, cuda, tokens):
    """Buffers that begin off a 16-byte boundary."""
    g, ids, _ = _routing(ks, tokens, 8, 2, 0.1, cuda)
    flat = torch.randn(2 * tokens * 64 + 1, generator=g, device=cuda).to(BF)
    d_p = flat[1:].view(2 * tokens, 64)
    a = ks.moe.permute_backward(torch.empty(tokens, 64, dtype=BF, device=cuda), d_p, ids, tokens, 2, 64)
    b = ks.moe.permute_backward(torch.empty(tokens, 64, dtype=BF, device=cuda), d_p.clone(), ids, tokens, 2, 64)
    assert torch.equal(a, b)
    w = torch.rand(tokens, 2, generator=g, device=cuda)
    d_out = torch.randn(tokens, 64, generator=g, device=cuda).to(BF)
    a = ks.moe.unpermute_backward(torch.empty(2 * tokens, 64, dtype=BF, device=cuda), torch.empty_like(w), d_out, d_p, ids, w, tokens, 2, 64)
    b = ks.moe.unpermute_backward(torch.empty(2 * tokens, 64, dtype=BF, device=cuda), torch.empty_like(w), d_out, d_p.clone(), ids, w, tokens,
                                  2, 64)
    # the sums run over other pieces: 64 products in fp32 either way
    assert torch.equal(a[0], b[0]) and (a[1] - b[1]).abs().max() <= 64 * 2 * ULP * 64 * 16


GATES = [(1, 1, 1, F32), (5, 8, 8, BF), (512, 64, 8, F32), (33, 60, 4, HF), (100, 100, 7, F32), (257, 256, 8, BF), (40, 1000, 32, BF),
         (64, 160, 6, HF), (3, 1024, 1, F32), (1000, 16, 2, BF), (31, 8, 3, F32)]


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k,dtype", GATES)
def test_gate_backward(ks, cuda, tokens, experts, top_k, dtype, renormalize):
    g = torch.Generator(device=cuda).manual_seed(tokens)
    logits = (torch.randn(tokens, experts, generator=g, device=cuda) * 3).to(dtype)
    w, idx = torch.empty(tokens, top_k, device=cuda), torch.empty(tokens, top_k, dtype=torch.int32, device=cuda)
    ks.moe.gate_softmax_topk(w, idx, logits, tokens, experts, top_k, renormalize=renormalize)
    dw = torch.randn(tokens, top_k, generator=g, device=cuda)
    got = ks.moe.gate_softmax_topk_backward(torch.full_like(logits, 9.0), dw, w, idx, None if renormalize else logits, tokens, experts, top_k,
                                            renormalize=renormalize)
    # autograd in 64 bits, through the chosen experts
    leaf = logits.double().requires_grad_()
    p = torch.softmax(leaf, 1).gather(1, idx.long())
    wd = p / p.sum(1, keepdim=True) if renormalize else p
    want, = torch.autograd.grad((wd * dw.double()).sum(), leaf)
    # the weights that the gate gave are off by (experts + 8) units of 2^-23 at most, and so is the softmax here; then top_k products
    c = (experts + top_k + 16) * 2 * ULP
    scale = (wd.detach() * dw.double().abs()).sum(1, keepdim=True)
    chosen = torch.zeros_like(want).scatter_add(1, idx.long(), wd.detach() * (dw.double().abs() + scale))
    mag = chosen if renormalize else torch.softmax(leaf.detach(), 1) * scale + chosen
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    # autograd's own rounding: at an expert that was not chosen it has p (s - s') for two sums s, s' of the same top_k terms, each of
    # them off by (experts + top_k + 16) * 2^-53 of their magnitudes' sum, where the formula has 0
    oracle = (experts + top_k + 16) * 2 * 2.0 ** -53 * scale
    check("d_logits", got, want, half_step(dtype) * (want.abs() + c * mag) + c * mag + tiny + oracle)
    if not renormalize:
        over = logits.clone()
        ks.moe.gate_softmax_topk_backward(over, dw, w, idx, over, tokens, experts, top_k, renormalize=False)
        assert torch.equal(over, got)


@pytest.mark.parametrize("experts", [8, 100])
def test_gate_backward_slots_out_of_range_and_twice(ks, cuda, experts):
    idx = torch.tensor([[-1, 3, 3], [experts, 0, 2 ** 31 - 1]], dtype=torch.int32, device=cuda)
    w = torch.tensor([[0.5, 0.25, 0.125], [0.5, 0.25, 0.125]], device=cuda)
    dw = torch.tensor([[float("nan"), 2.0, 4.0], [float("inf"), 8.0, float("nan")]], device=cuda)
    got = ks.moe.gate_softmax_topk_backward(torch.empty(2, experts, device=cuda), dw, w, idx, None, 2, experts, 3)
    want = torch.zeros(2, experts, device=cuda)
    want[0, 3] = 0.25 * (2 - 1.0) + 0.125 * (4 - 1.0)    # s = 0.5 + 0.5
    want[1, 0] = 0.25 * (8 - 2.0)
    assert torch.equal(got, want)


def test_rows_behind_two_to_the_31_elements(ks, cuda):
    tokens, top_k, hidden = 150_000, 2, 8192
    g, ids, _ = _routing(ks, tokens, 4, top_k, 0.0, cuda)
    d_p = torch.empty(tokens * top_k, hidden, dtype=BF, device=cuda)
    d_p.copy_((torch.arange(tokens * top_k, device=cuda) % 64)[:, None])
    got = ks.moe.permute_backward(torch.empty(tokens, hidden, dtype=BF, device=cuda), d_p, ids, tokens, top_k, hidden)
    inv = torch.empty(tokens * top_k, dtype=torch.long, device=cuda)
    inv[ids.long()] = torch.arange(tokens * top_k, device=cuda)
    sums = (inv.view(tokens, 2) % 64).sum(1).to(BF)      # whole numbers below 128: exact
    assert torch.equal(got[:, 0], sums) and torch.equal(got[:, -1], sums)
    w = torch.ones(tokens, top_k, device=cuda)
    _, d_w = ks.moe.unpermute_backward(d_p, torch.empty_like(w), got, d_p, ids, w, tokens, top_k, hidden)
    want = sums.float()[:, None] * (inv.view(tokens, 2) % 64) * hidden       # up to 2^27, multiples of 2^13: exact
    assert torch.equal(d_w, want)
    assert torch.equal(d_p[:, -1].view(-1)[inv.view(tokens, 2)[:, 0]], sums)


def test_no_tokens(ks, cuda):
    e = torch.empty(0, 64, dtype=BF, device=cuda)
    w = torch.empty(0, 2, device=cuda)
    i = torch.empty(0, dtype=torch.int32, device=cuda)
    ks.moe.permute_backward(e, e, i, 0, 2, 64)
    ks.moe.unpermute_backward(e, w, e, e, i, w, 0, 2, 64)
    ks.moe.gate_softmax_topk_backward(torch.empty(0, 8, device=cuda), w, w, i, None, 0, 8, 2)


@pytest.mark.parametrize("tokens", [60, 3000])
def test_layer_and_its_gradient(ks, cuda, tokens):
    """The steps as a routed layer uses them, 16-bit experts: its gradient against autograd in 64 bits on the same rounded steps'
    formula, and once more captured and replayed."""
    experts, top_k, hidden, inner = 8, 2, 128, 96
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(tokens, hidden, generator=g, device=cuda).to(BF)
    router = torch.randn(hidden, experts, generator=g, device=cuda).to(BF) * 0.1
    weight = (torch.randn(experts, hidden, inner, generator=g, device=cuda) * hidden ** -0.5).to(BF)
    weight_t = weight.transpose(1, 2).contiguous()
    d_y = torch.randn(tokens, inner, generator=g, device=cuda).to(BF)
    logits = x @ router
    pairs = tokens * top_k
    f32 = dict(device=cuda)
    w, idx = torch.empty(tokens, top_k, **f32), torch.empty(tokens, top_k, dtype=torch.int32, device=cuda)
    ids, offsets = torch.empty(pairs, dtype=torch.int32, device=cuda), torch.empty(experts + 1, dtype=torch.int32, device=cuda)
    xp, yp = torch.empty(pairs, hidden, dtype=BF, device=cuda), torch.empty(pairs, inner, dtype=BF, device=cuda)
    d_yp, d_w, d_xp = torch.empty_like(yp), torch.empty_like(w), torch.empty_like(xp)
    d_x, d_logits, y = torch.empty_like(x), torch.empty_like(logits), torch.empty_like(d_y)

    def step():
        ks.moe.gate_softmax_topk(w, idx, logits, tokens, experts, top_k)
        ks.moe.compute_permutation(ids, offsets, idx, tokens, experts, top_k)
        ks.moe.permute(xp, x, ids, tokens, top_k, hidden)
        ks.moe.grouped_gemm(yp, xp, weight, offsets, experts, pairs, inner, hidden)
        ks.moe.unpermute(y, yp, ids, w, tokens, top_k, inner)
        ks.moe.unpermute_backward(d_yp, d_w, d_y, yp, ids, w, tokens, top_k, inner)
        ks.moe.grouped_gemm(d_xp, d_yp, weight_t, offsets, experts, pairs, hidden, inner)
        ks.moe.permute_backward(d_x, d_xp, ids, tokens, top_k, hidden)
        ks.moe.gate_softmax_topk_backward(d_logits, d_w, w, idx, None, tokens, experts, top_k)

    step()
    xd, ld = x.double().requires_grad_(), logits.double().requires_grad_()
    p = torch.softmax(ld, 1).gather(1, idx.long())
    p = p / p.sum(1, keepdim=True)
    out = torch.einsum("th,tkhi->tki", xd, weight.double()[idx.long()])
    yd = (p[..., None] * out).sum(1)
    want_x, want_l = torch.autograd.grad((yd * d_y.double()).sum(), (xd, ld))
    # three roundings to bf16 on the way of d_x, one of them of the result; two on the way of d_logits: relative to the tensors'
    # sizes, independent roundings of at most u each add up to less than 3u of the norm
    u = half_step(BF)
    for got, want in ((d_x, want_x), (d_logits, want_l)):
        assert (got.double() - want).norm() <= 3 * u * want.norm()
    eager = d_x.clone(), d_logits.clone(), d_w.clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for t in (d_x, d_logits, d_w, d_yp, d_xp):
        t.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, (d_x, d_logits, d_w)))
