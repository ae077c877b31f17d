"""GPU: how finely the adapters' kernels hold an inner vector between its two products.

The inner vectors A x and s B^T d_out are sums in fp32 and h is given in fp32, so outputs that depend on their last bits have to come
out. The tests build inner numbers of which all but the last bits cancel."""
import pytest
import torch

from _lora import STEP, Problem, chain, check, half_step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _pieces(count, seed):
    """Numbers v of 22 bits as three bf16 numbers, the nearest first: (v, first, first + second, third), all exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = (torch.randint(2 ** 21, 2 ** 22, (count,), generator=g, device="cuda").float() * 2.0 ** -20)
    v = v * (torch.randint(0, 2, (count,), generator=g, device="cuda") * 2 - 1)
    first = v.bfloat16().float()
    second = (v - first).bfloat16().float()
    return v, first, second, v - first - second


def _expect(what, got, last, first):
    """``got`` is ``last`` but for its own rounding and one fp32 step of the cancelled numbers in each of the two sums that make them, and in
    theirs (instructions of 16 products may truncate)."""
    bound = 4 * STEP * first.abs() + half_step(BF) * last.abs()
    shows = int((last.abs() > bound).sum())
    assert shows, "the last bits would not show"
    bad = (got.float() - last).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}"


@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("tokens", [5, 40, 700])
def test_outputs_see_all_bits_of_the_inner_vector(ks, cuda, tokens, rank):
    k, n = 64, 72
    v, first, second, last = _pieces(tokens, tokens + rank)
    three = torch.zeros(tokens, k, device=cuda)
    three[:, 16], three[:, 17], three[:, 18] = first, second, last
    order, offsets = ks.lora.plan(torch.zeros(tokens, dtype=torch.int32, device=cuda), 1)
    one = torch.ones(1, device=cuda)
    # h_0 = v, h_(last rank) = first + second; out = h_0 - h_(last rank)
    a, b = torch.zeros(1, rank, k, device=cuda), torch.zeros(1, n, rank, device=cuda)
    a[0, 0, 16:19], a[0, -1, 16:18] = 1, 1
    b[0, :, 0], b[0, :, -1] = 1, -1
    base = torch.zeros(tokens, n, dtype=BF, device=cuda)
    out = ks.lora.apply(torch.empty_like(base), base, three.to(BF), a.to(BF), b.to(BF), one, order, offsets)
    _expect("out", out, last[:, None].expand(-1, n), first[:, None])
    # the same with the roles of the factors changed: g_0 = v, g_(last rank) = first + second; d_x = g_0 - g_(last rank)
    d_out = torch.zeros(tokens, n, device=cuda)
    d_out[:, 16:19] = three[:, 16:19]
    a, b = torch.zeros(1, rank, k, device=cuda), torch.zeros(1, n, rank, device=cuda)
    b[0, 16:19, 0], b[0, 16:18, -1] = 1, 1
    a[0, 0], a[0, -1] = 1, -1
    base = torch.zeros(tokens, k, dtype=BF, device=cuda)
    d_x, _, _ = ks.lora.backward(torch.empty_like(base), torch.empty_like(a, dtype=BF), torch.empty_like(b, dtype=BF), base, d_out.to(BF), three.to(BF),
                                 torch.zeros(tokens, rank, device=cuda), a.to(BF), b.to(BF), one, order, offsets)
    _expect("d_x", d_x, last[:, None].expand(-1, k), first[:, None])


@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("adapters", [3, 200])
def test_factors_gradients_see_all_bits_of_the_inner_vectors(ks, cuda, adapters, rank):
    """Two rows of an adapter whose numbers cancel but for the last bits."""
    k, n = 264, 320
    v, first, second, last = _pieces(adapters, adapters + rank)
    tokens = 2 * adapters
    order, offsets = ks.lora.plan(torch.arange(tokens, dtype=torch.int32, device=cuda) // 2, adapters)
    one = torch.ones(adapters, device=cuda)
    signs = torch.tensor([1.0, -1.0], device=cuda).repeat(adapters)[:, None]
    a, b = torch.zeros(adapters, rank, k, dtype=BF, device=cuda), torch.zeros(adapters, n, rank, dtype=BF, device=cuda)
    b[:, :3] = 1                                                    # g = the sum of d_out's first three
    base = torch.zeros(tokens, k, dtype=BF, device=cuda)

    def call(d_out, x, h):
        return ks.lora.backward(torch.empty_like(base), torch.empty_like(a), torch.empty_like(b), base, d_out.to(BF), x.to(BF), h, a, b, one,
                                order, offsets)

    d_out = torch.zeros(tokens, n, device=cuda)
    d_out[::2, 0], d_out[::2, 1], d_out[::2, 2] = first, second, last
    d_out[1::2, 0], d_out[1::2, 1] = first, second
    _, d_a, _ = call(d_out, signs.expand(-1, k), torch.zeros(tokens, rank, device=cuda))
    _expect("d_a", d_a, last[:, None, None].expand(-1, rank, k), first[:, None, None])
    h = torch.empty(tokens, rank, device=cuda)
    h[::2], h[1::2] = v[:, None], (first + second)[:, None]
    _, _, d_b = call(signs.expand(-1, n), base, h)
    _expect("d_b", d_b, last[:, None, None].expand(-1, n, rank), first[:, None, None])


def _falling(rank, size, device):
    """Factors 1 .. size over the ranks, powers of two."""
    return torch.exp2(torch.round(torch.linspace(0, size, rank, device=device)))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [8, 24, 64, 128])
@pytest.mark.parametrize("tokens", [3, 40, 700])
def test_outputs_of_ranks_far_below_the_largest(ks, cuda, tokens, rank, dtype):
    """The numbers of an inner vector fall to 2^-18 of the largest (which f16 factors can express), and every output depends on one of them."""
    p = Problem(tokens, 2, rank, 64, 128, dtype, seed=rank)
    fall = _falling(rank, -18, cuda)
    owner = torch.arange(128, device=cuda) % rank
    mask = owner[:, None] == torch.arange(rank, device=cuda)
    ids, offsets = ks.lora.plan(p.ids, p.adapters)
    p.a = (p.a.float() * fall[:, None]).to(dtype)
    p.b = torch.where(mask, p.b.float() / fall * 2.0 ** -8, 0).to(dtype)
    p.base = torch.zeros_like(p.base)
    want, bound, _, _ = p.forward()
    out = ks.lora.apply(torch.empty_like(p.base), p.base, p.x, p.a, p.b, p.scales, ids, offsets)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    check("out", out, want, bound + tiny)
    # the roles of the factors changed: g falls, and every column of d_x depends on one of its numbers
    p = Problem(tokens, 2, rank, 128, 64, dtype, seed=rank)
    p.b = (p.b.float() * fall).to(dtype)
    p.a = torch.where(mask.t(), p.a.float() / fall[:, None] * 2.0 ** -4, 0).to(dtype).contiguous()
    p.d_x_base = torch.zeros_like(p.d_x_base)
    h = torch.zeros(tokens, rank, device=cuda)
    want, bounds = p.backward(h)
    got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales,
                           ids, offsets)
    check("d_x", got[0], want[0], bounds[0])
    check("d_a", got[1], want[1], bounds[1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [8, 64, 128])
@pytest.mark.parametrize("fall", [-14, -20, -30, -45, -90])
@pytest.mark.parametrize("tokens", [70, 1500])
def test_gradients_of_ranks_far_below_the_largest(ks, cuda, tokens, fall, rank, dtype):
    """h falls over the ranks, and each of d_b's elements is held to its own sum."""
    p = Problem(tokens, 2, rank, 72, 264, dtype, seed=tokens)
    ids, offsets = ks.lora.plan(p.ids, p.adapters)
    g = torch.Generator(device=cuda).manual_seed(rank)
    h = torch.randn(tokens, rank, generator=g, device=cuda) * _falling(rank, fall, cuda) * 2.0 ** 12
    want, bounds = p.backward(h)
    got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales,
                           ids, offsets)
    for what, x, y, b in zip(("d_x", "d_a", "d_b"), got, want, bounds):
        check(what, x, y, b)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [16, 96])
@pytest.mark.parametrize("size", [12, 24, 34, 60, 100])
@pytest.mark.parametrize("tokens", [70, 1500])
def test_gradients_beside_a_row_far_above_the_others(ks, cuda, tokens, size, rank, dtype):
    """A row whose h is huge and whose d_out is zero, and one whose g is large and whose x is zero, change nothing."""
    p = Problem(tokens, 2, rank, 264, 136, dtype, seed=tokens + 1)
    ids, offsets = ks.lora.plan(p.ids, p.adapters)
    g = torch.Generator(device=cuda).manual_seed(rank)
    h = torch.randn(tokens, rank, generator=g, device=cuda)
    h[tokens // 2] *= 2.0 ** size
    p.d_out[tokens // 2] = 0
    top = 13 if dtype is HF else size
    p.d_out[tokens // 3] *= 2.0 ** top
    p.d_out[[i for i in range(tokens) if i != tokens // 3]] *= 2.0 ** (top - size if dtype is HF and size <= 24 else 0)
    p.x[tokens // 3] = 0
    p.b = (p.b.float() * 2.0 ** -6).to(dtype)
    h[tokens // 3] = 0
    want, bounds = p.backward(h)
    got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales,
                           ids, offsets)
    for what, x, y, b in zip(("d_a", "d_b"), got[1:], want[1:], bounds[1:]):
        check(what, x, y, b)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [8, 12, 64, 128])
@pytest.mark.parametrize("where", ["x", "d_out", "h"])
@pytest.mark.parametrize("tokens", [70, 1500])
def test_gradients_of_numbers_that_are_not_finite(ks, cuda, tokens, where, rank, dtype):
    """An infinity in a row makes infinities of the sums' own signs in the factors' gradients, and NaN only where fp32 has it."""
    p = Problem(tokens, 3, rank, 136, 264, dtype, seed=rank)
    p.ids[:6] = torch.tensor([0, 0, 1, 1, 2, 2], dtype=torch.int32, device=cuda)
    ids, offsets = ks.lora.plan(p.ids, p.adapters)
    g = torch.Generator(device=cuda).manual_seed(rank)
    h = torch.randn(tokens, rank, generator=g, device=cuda)
    inf = float("inf")
    if where == "x":
        p.x[0, 5], p.x[2, 7], p.x[3, 7], p.x[4, 0] = inf, inf, -inf, float("nan")
    elif where == "d_out":
        p.d_out[0, 5], p.d_out[2, 7], p.d_out[3, 7], p.d_out[4, 0] = inf, inf, -inf, float("nan")
    else:
        h[0, 1], h[2, 3], h[3, 3], h[4, 0] = inf, inf, -inf, float("nan")
    want, bounds = p.backward(h)
    got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales,
                           ids, offsets)
    for what, x, y, b in zip(("d_a", "d_b"), got[1:], want[1:], bounds[1:]):
        fine = torch.isfinite(y)
        assert torch.equal(torch.isnan(x), torch.isnan(y)), what
        inf = torch.isinf(y)
        assert torch.equal(x[inf].double(), y[inf]), what
        check(what, x[fine], y[fine], b[fine])
