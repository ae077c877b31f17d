"""GPU: low-rank adapters of many requests and their gradient, against 64 bits."""
import pytest
import torch

from _lora import Problem, check, half_step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# tokens, adapters, rank, K, N, dtype, without, active
SHAPES = [
    (1, 1, 8, 64, 64, BF, 0.0, 1),
    (1, 8, 16, 4096, 4096, BF, 0.0, 8),
    (2, 3, 16, 4096, 520, HF, 0.0, 3),
    (5, 2, 5, 33, 17, BF, 0.0, 2),               # nothing is a multiple of anything
    (7, 3, 1, 1, 1, HF, 0.3, 3),
    (48, 64, 16, 1024, 2048, HF, 0.1, 64),       # nearly an adapter a row
    (33, 5, 64, 2048, 1032, BF, 0.2, 2),         # adapters without rows
    (40, 1, 128, 512, 11008, BF, 0.0, 1),
    (9, 2, 24, 264, 136, HF, 0.0, 2),
    (130, 4, 16, 136, 264, BF, 0.1, 4),
    (300, 5, 64, 512, 1024, HF, 0.2, 5),
    (257, 3, 128, 200, 72, BF, 0.0, 3),
    (777, 24, 64, 2048, 1544, BF, 0.2, 24),
    (1000, 1, 8, 1024, 512, HF, 0.0, 1),
    (513, 2, 20, 100, 60, BF, 0.5, 2),           # widths of 4 elements only
    (600, 3, 256, 256, 128, HF, 0.0, 3),         # a rank beyond 128
    (2050, 7, 96, 768, 640, BF, 0.1, 6),
    (500, 3, 32, 264, 520, HF, 0.1, 3),
    (512, 200, 16, 128, 72, BF, 0.2, 150),
    (513, 200, 16, 128, 72, BF, 0.2, 150),
]


def _plan(ks, p):
    return ks.lora.plan(p.ids, p.adapters)


@pytest.mark.parametrize("tokens,adapters,rank,k,n,dtype,without,active", SHAPES)
def test_apply(ks, cuda, tokens, adapters, rank, k, n, dtype, without, active):
    p = Problem(tokens, adapters, rank, k, n, dtype, without, active, seed=tokens)
    ids, offsets = _plan(ks, p)
    want, bound, h_want, h_bound = p.forward()
    h = torch.full((tokens, rank), float("nan"), device=cuda)
    out = ks.lora.apply(torch.full_like(p.base, float("nan")), p.base, p.x, p.a, p.b, p.scales, ids, offsets, h=h)
    check("out", out, want, bound)
    has = p.ids >= 0
    check("h", h[has], h_want[has], h_bound[has])
    assert torch.isnan(h[~has]).all(), "rows without an adapter keep what h held"
    assert torch.equal(out[~has], p.base[~has])
    # the same in place, without h, and a second time: the same bits
    again = p.base.clone()
    ks.lora.apply(again, again, p.x, p.a, p.b, p.scales, ids, offsets)
    assert torch.equal(again, out)


@pytest.mark.parametrize("tokens,adapters,rank,k,n,dtype,without,active", [s for s in SHAPES if s[0] != 2])
def test_backward(ks, cuda, tokens, adapters, rank, k, n, dtype, without, active):
    p = Problem(tokens, adapters, rank, k, n, dtype, without, active, seed=tokens + 1)
    ids, offsets = _plan(ks, p)
    h = p.forward()[2].float()
    h[p.ids < 0] = float("nan")   # not to be read
    want, bounds = p.backward(h)

    def call(d_x):
        return ks.lora.backward(d_x, torch.full_like(p.a, float("nan")), torch.full_like(p.b, float("nan")), p.d_x_base, p.d_out, p.x, h,
                                p.a, p.b, p.scales, ids, offsets)

    got = call(torch.full_like(p.d_x_base, float("nan")))
    for what, x, y, b in zip(("d_x", "d_a", "d_b"), got, want, bounds):
        check(what, x, y, b)
    again = call(torch.empty_like(p.d_x_base))
    assert all(torch.equal(x, y) for x, y in zip(got, again)), "the same call gives the same bits"
    in_place = p.d_x_base.clone()
    ks.lora.backward(in_place, torch.empty_like(p.a), torch.empty_like(p.b), in_place, p.d_out, p.x, h, p.a, p.b, p.scales, ids,
                     offsets)
    assert torch.equal(in_place, got[0])


@pytest.mark.parametrize("tokens,adapters", [(0, 3), (1, 1), (5, 1023), (4096, 7), (200_001, 33)])
def test_plan(ks, cuda, tokens, adapters):
    g = torch.Generator(device=cuda).manual_seed(tokens)
    ids = torch.randint(-2, adapters + 3, (tokens,), generator=g, device=cuda, dtype=torch.int32)
    order, offsets = ks.lora.plan(ids, adapters)
    group = torch.where((ids < 0) | (ids >= adapters), adapters, ids.long())
    assert torch.equal(order.long(), torch.sort(group, stable=True).indices)
    counts = torch.bincount(group, minlength=adapters + 1)
    assert offsets.tolist() == [0] + counts.cumsum(0).tolist()


def test_no_rows(ks, cuda):
    p = Problem(0, 2, 8, 64, 32)
    ids, offsets = _plan(ks, p)
    assert ks.lora.apply(p.base, p.base, p.x, p.a, p.b, p.scales, ids, offsets).shape == (0, 32)
    d_a, d_b = torch.full_like(p.a, float("nan")), torch.full_like(p.b, float("nan"))
    ks.lora.backward(p.d_x_base, d_a, d_b, p.d_x_base, p.d_out, p.x, torch.empty(0, 8, device=cuda), p.a, p.b, p.scales, ids, offsets)
    assert not d_a.any() and not d_b.any()


@pytest.mark.parametrize("tokens", [3, 20, 700])
def test_no_adapter_at_all(ks, cuda, tokens):
    p = Problem(tokens, 4, 16, 256, 512, without=2.0)
    ids, offsets = _plan(ks, p)
    out = ks.lora.apply(torch.empty_like(p.base), p.base, p.x, p.a, p.b, p.scales, ids, offsets)
    assert torch.equal(out, p.base)
    h = torch.full((tokens, 16), float("nan"), device=cuda)
    got = ks.lora.backward(torch.empty_like(p.x), torch.full_like(p.a, float("nan")), torch.full_like(p.b, float("nan")),
                           p.d_x_base, p.d_out, p.x, h, p.a, p.b, p.scales, ids, offsets)
    assert torch.equal(got[0], p.d_x_base) and not got[1].any() and not got[2].any()


@pytest.mark.parametrize("tokens", [6, 150, 1500])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_columns_of_wider_tensors(ks, cuda, tokens, dtype):
    """x, base, out and the gradients as column ranges of wider tensors; what lies beside them stays."""
    k, n, r = 256, 192, 16
    p = Problem(tokens, 3, r, k, n, dtype, without=0.1)
    ids, offsets = _plan(ks, p)
    want, bound, h, _ = p.forward()
    wide_x = torch.full((tokens, k + 40), float("nan"), dtype=dtype, device=cuda)
    wide_x[:, 8:8 + k] = p.x
    fused = torch.full((tokens, 3 * n), 7.0, dtype=dtype, device=cuda)
    fused[:, n:2 * n] = p.base
    part = fused[:, n:2 * n]
    ks.lora.apply(part, part, wide_x[:, 8:8 + k], p.a, p.b, p.scales, ids, offsets)
    check("out", part, want, bound)
    assert (fused[:, :n] == 7).all() and (fused[:, 2 * n:] == 7).all()
    # odd distances and offsets: the kernels for any alignment
    odd = torch.full((tokens, n + 3), 7.0, dtype=dtype, device=cuda)
    odd[:, 1:1 + n] = p.base
    ks.lora.apply(odd[:, 1:1 + n], odd[:, 1:1 + n], wide_x[:, 8:8 + k], p.a, p.b, p.scales, ids, offsets)
    check("out", odd[:, 1:1 + n], want, bound)
    assert (odd[:, 0] == 7).all() and (odd[:, 1 + n:] == 7).all()
    wide_dout = torch.full((tokens, 2 * n), float("nan"), dtype=dtype, device=cuda)
    wide_dout[:, n:] = p.d_out
    wide_dx = torch.full((tokens, 2 * k), 7.0, dtype=dtype, device=cuda)
    hf = h.float()
    want, bounds = p.backward(hf)
    got = ks.lora.backward(wide_dx[:, k:], torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, wide_dout[:, n:],
                           wide_x[:, 8:8 + k], hf, p.a, p.b, p.scales, ids, offsets)
    for what, x, y, b in zip(("d_x", "d_a", "d_b"), got, want, bounds):
        check(what, x, y, b)
    assert (wide_dx[:, :k] == 7).all()


@pytest.mark.parametrize("tokens", [20, 400])
def test_rows_of_others_do_not_matter(ks, cuda, tokens):
    """Infinities and NaN in rows without an adapter, or of another adapter, stay where they are."""
    p = Problem(tokens, 3, 16, 512, 256, without=0.3, seed=5)
    sick = p.ids == 1
    none = p.ids < 0
    clean = ~(sick | none)
    p.x[sick] = float("inf")
    p.x[none] = float("nan")
    p.base[none] = float("nan")
    p.d_out[none] = float("nan")
    p.d_out[sick] = float("inf")
    ids, offsets = _plan(ks, p)
    want, bound, h, _ = p.forward()
    hf = h.float()
    out = ks.lora.apply(torch.empty_like(p.base), p.base, p.x, p.a, p.b, p.scales, ids, offsets)
    check("out", out[clean], want[clean], bound[clean])
    assert torch.isnan(out[none]).all() and not torch.isfinite(out[sick]).any()
    want, bounds = p.backward(hf)
    d_x, d_a, d_b = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, hf,
                                     p.a, p.b, p.scales, ids, offsets)
    check("d_x", d_x[clean], want[0][clean], bounds[0][clean])
    assert torch.equal(d_x[none], p.d_x_base[none])
    for a in (0, 2):
        check("d_a", d_a[a], want[1][a], bounds[1][a])
        check("d_b", d_b[a], want[2][a], bounds[2][a])


@pytest.mark.parametrize("tokens", [12, 900])
def test_places_left_out_keep_their_rows(ks, cuda, tokens):
    """Ids out of range in the plan are left out, rows that no place names stay as they were."""
    p = Problem(tokens, 2, 16, 256, 128, seed=3)
    ids, offsets = _plan(ks, p)
    named = torch.ones(tokens, dtype=torch.bool, device=cuda)
    named[ids[::5].long()] = False
    ids[::5] = torch.tensor([-1, tokens, 2 ** 31 - 1], dtype=torch.int32, device=cuda).repeat(tokens)[:ids[::5].numel()]
    want, bound, h, _ = p.forward()
    out = torch.full_like(p.base, 9.0)
    ks.lora.apply(out, p.base, p.x, p.a, p.b, p.scales, ids, offsets)
    check("out", out[named], want[named], bound[named])
    assert (out[~named] == 9).all()
    p.ids = torch.where(named, p.ids, -1)
    hf = h.float()
    want, bounds = p.backward(hf)
    d_x, d_a, d_b = ks.lora.backward(torch.full_like(p.x, 9.0), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x,
                                     hf, p.a, p.b, p.scales, ids, offsets)
    check("d_x", d_x[named], want[0][named], bounds[0][named])
    assert (d_x[~named] == 9).all()
    check("d_a", d_a, want[1], bounds[1])
    check("d_b", d_b, want[2], bounds[2])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens", [8, 300])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 11])
def test_inner_vector_beyond_f16(ks, cuda, tokens, dtype, size):
    """A x far below and above what f16 holds (h up to 2^22, g likewise) with factors that bring it back."""
    p = Problem(tokens, 2, 16, 256, 128, dtype, seed=9)
    small = 1 / size
    p.x = (p.x.float() * size).to(dtype)
    p.a = (p.a.float() * size).to(dtype)
    p.b = (p.b.float() * small).to(dtype)
    p.scales = p.scales * small
    ids, offsets = _plan(ks, p)
    want, bound, h, _ = p.forward()
    tiny = torch.finfo(dtype).smallest_normal
    out = ks.lora.apply(torch.empty_like(p.base), p.base, p.x, p.a, p.b, p.scales, ids, offsets)
    check("out", out, want, bound + tiny)
    p.scales = p.scales * size ** 2
    if size > 1:   # (so that the factors' gradients fit)
        p.d_out = (p.d_out.float() * 2.0 ** -9).to(dtype)
    hf = h.float()
    want, bounds = p.backward(hf)
    fits = [w.abs().max() < torch.finfo(dtype).max for w in want]
    got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, hf, p.a, p.b,
                           p.scales, ids, offsets)
    for what, x, y, b, ok in zip(("d_x", "d_a", "d_b"), got, want, bounds, fits):
        if ok:
            check(what, x, y, b)


def test_gradient_against_differences(ks, cuda):
    """<d_out, out(x + e v) - out(x - e v)> / 2e against the gradients, in directions of all three arguments."""
    p = Problem(40, 2, 8, 64, 48, HF, seed=2)
    ids, offsets = _plan(ks, p)
    h = torch.empty(40, 8, device=cuda)
    ks.lora.apply(torch.empty_like(p.base), p.base, p.x, p.a, p.b, p.scales, ids, offsets, h=h)
    zero = torch.zeros_like(p.x)
    d_x, d_a, d_b = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), zero, p.d_out, p.x, h, p.a, p.b,
                                     p.scales, ids, offsets)
    g = torch.Generator(device=cuda).manual_seed(0)
    for name, grad in (("x", d_x), ("a", d_a), ("b", d_b)):
        at = getattr(p, name)
        v = torch.randn(at.shape, generator=g, device=cuda, dtype=torch.float64)
        def value(e):
            setattr(p, name, at.double() + e * v)
            out = p.forward()[0]
            setattr(p, name, at)
            return float((p.d_out.double() * out).sum())
        slope = (value(1e-3) - value(-1e-3)) / 2e-3     # exact: the output is linear in each argument
        mine = float((grad.double() * v).sum())
        # each gradient is off by half a step (and as much again for what its sum brings): added up over random directions
        allow = float((2 * half_step(HF) * grad.double().abs() * v.abs()).sum()) + 1e-6 * abs(slope)
        assert abs(mine - slope) <= allow, (name, mine, slope, allow)


def test_far_rows(ks, cuda):
    """Rows that begin behind 2^31 elements."""
    tokens, n = 140_000, 16384
    p = Problem(8, 2, 8, 64, 64)
    big = torch.zeros(tokens, n, dtype=BF, device=cuda)
    x = torch.zeros(tokens, 64, dtype=BF, device=cuda)
    at = torch.tensor([0, 1, 70_000, 131_071, 131_072, 131_073, 139_998, 139_999], device=cuda)
    x[at] = p.x
    part = big[:, n - 64:]
    part[at] = p.base
    ids = torch.full((tokens,), -1, dtype=torch.int32, device=cuda)
    ids[at] = p.ids
    order, offsets = ks.lora.plan(ids, 2)
    ks.lora.apply(part, part, x, p.a, p.b, p.scales, order, offsets)
    want, bound, _, _ = p.forward()
    check("out", part[at], want, bound)
    assert int((big != 0).any(1).sum()) == 8


@pytest.mark.parametrize("tokens", [1, 24, 600])
def test_captured_beside_an_eager_call(ks, cuda, tokens):
    """A graph of both directions replays on new contents, with eager calls on another stream meanwhile."""
    p, q = (Problem(tokens, 3, 16, 256, 512, seed=s) for s in (1, 2))
    h = torch.empty(tokens, 16, device=cuda)
    out, d_x, d_a, d_b = torch.empty_like(p.base), torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b)
    live = {name: getattr(p, name).clone() for name in ("ids", "x", "base", "a", "b", "scales", "d_out", "d_x_base")}
    order, offsets = torch.empty(tokens, dtype=torch.int32, device=cuda), torch.empty(5, dtype=torch.int32, device=cuda)

    def step(v, out, h, d_x, d_a, d_b, order, offsets):
        ks.lora.plan(v["ids"], 3, order, offsets)
        ks.lora.apply(out, v["base"], v["x"], v["a"], v["b"], v["scales"], order, offsets, h=h)
        ks.lora.backward(d_x, d_a, d_b, v["d_x_base"], v["d_out"], v["x"], h, v["a"], v["b"], v["scales"], order, offsets)

    step(live, out, h, d_x, d_a, d_b, order, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(live, out, h, d_x, d_a, d_b, order, offsets)
    for name, t in live.items():
        t.copy_(getattr(q, name))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager = [torch.empty_like(t) for t in (out, h, d_x, d_a, d_b, order, offsets)]
    graph.replay()
    with torch.cuda.stream(side):
        step({name: getattr(p, name) for name in live}, *eager)
    torch.cuda.synchronize()
    for prob, got in ((q, (out, d_x, d_a, d_b)), (p, (eager[0], *eager[2:5]))):
        want, bound, hd, _ = prob.forward()
        check("out", got[0], want, bound)
        grads, bounds = prob.backward(hd.float())
        for what, x, y, b in zip(("d_x", "d_a", "d_b"), got[1:], grads, bounds):
            check(what, x, y, b * 1.01)   # (the forward pass's own h instead of the 64-bit one)


def test_experts_adapters_on_a_routed_layers_rows(ks, cuda):
    """sorted_ids = None: rows already in group order, dropped pairs' rows at the end keep their base."""
    rows, experts, k, n = 260, 6, 128, 192
    p = Problem(rows, experts, 8, k, n, without=0.2, seed=4)
    order, offsets = ks.lora.plan(p.ids, experts)
    o = order.long()
    out = ks.lora.apply(torch.empty_like(p.base), p.base[o].contiguous(), p.x[o].contiguous(), p.a, p.b, p.scales, None, offsets[:-1].contiguous())
    want, bound, _, _ = p.forward()
    check("out", out, want[o], bound[o])


@pytest.mark.parametrize("rank", [16, 64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_sequences_beside_rows_that_are_not_numbers(ks, cuda, rank, dtype):
    """Runs of rows of one adapter, of odd lengths, with NaN and infinities in the rows between and behind them, as columns of wider
    tensors; with the rows' numbers and without, to the bit."""
    lengths = [(0, 200), (1, 64), (2, 63), (4, 129), (5, 70)]       # adapters 3 and 5: no row, rows that no longer count
    ids = torch.cat([torch.full((n,), a) for a, n in lengths])
    p = Problem(ids.numel(), 5, rank, 328, 520, dtype, seed=7)
    p.ids = torch.where(ids < 5, ids, -1).to(torch.int32).to(cuda)
    none = p.ids < 0
    _, _, h, _ = p.forward()
    hf = h.float()
    want, bounds = p.backward(hf)
    x, d_out, d_x = (torch.full((p.tokens, w + 64), float("nan"), dtype=dtype, device=cuda) for w in (p.k, p.n, p.k))
    x[:, 8:8 + p.k], d_out[:, 16:16 + p.n] = p.x, p.d_out
    x[none], d_out[none] = float("nan"), float("inf")
    hf[none] = float("nan")
    ids, offsets = _plan(ks, p)
    results = []
    for order in (ids, None):
        d_a, d_b = torch.full_like(p.a, 9.0), torch.full_like(p.b, 9.0)
        ks.lora.backward(d_x[:, 24:24 + p.k], d_a, d_b, p.d_x_base, d_out[:, 16:16 + p.n], x[:, 8:8 + p.k], hf, p.a, p.b, p.scales, order, offsets)
        results.append((d_x[:, 24:24 + p.k].clone(), d_a, d_b))
    for what, got, w, b in zip(("d_x", "d_a", "d_b"), results[0], want, bounds):
        check(what, got, w, b)
    assert torch.equal(results[0][0][none], p.d_x_base[none])
    assert not results[0][1][3].any() and not results[0][2][3].any()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("tokens,adapters,active", [(4096, 2, 1), (5000, 8, 3), (3000, 6, 6)])
def test_backward_of_long_batches(ks, cuda, tokens, adapters, active):
    """Slabs whose rows several CTAs share, some adapters without rows; every run gives the same bits."""
    p = Problem(tokens, adapters, 16, 1024, 768, seed=9, active=active)
    ids, offsets = _plan(ks, p)
    _, _, h, _ = p.forward()
    hf = h.float()
    want, bounds = p.backward(hf)
    first = None
    for _ in range(3):
        got = ks.lora.backward(torch.empty_like(p.x), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, hf, p.a, p.b,
                               p.scales, ids, offsets)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    for what, x, y, b in zip(("d_x", "d_a", "d_b"), first, want, bounds):
        check(what, x, y, b)
