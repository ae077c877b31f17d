"""GPU: the adapters' calls with part of a table of offsets (a rank's own experts, say): it begins behind the first place."""
import pytest
import torch

from _lora import Problem, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,rank,k,n", [(100, 16, 64, 128), (900, 16, 64, 128), (100, 5, 64, 128), (900, 16, 60, 128), (900, 16, 64, 124),
                                             (700, 136, 64, 128)])
@pytest.mark.parametrize("numbered", [True, False])
def test_places_in_front_of_the_first_offset_are_left_out(ks, cuda, tokens, rank, k, n, numbered):
    """The same by every kernel: rows there keep what they held, and the factors' gradients do not see them."""
    p = Problem(tokens, 6, rank, k, n, without=0.1, seed=rank)
    if not numbered:     # rows in the adapters' order
        p.ids = torch.sort(torch.where(p.ids < 0, 6, p.ids)).values.to(torch.int32)
    ids, offsets = ks.lora.plan(p.ids, 6)
    before = p.ids < 2
    before &= p.ids >= 0
    p.ids = torch.where((p.ids >= 2) & (p.ids < 6), p.ids - 2, -1)
    assert before.sum() > 10
    part = offsets[2:7].contiguous()
    p.adapters, p.a, p.b, p.scales = 4, p.a[2:].contiguous(), p.b[2:].contiguous(), p.scales[2:].contiguous()
    order = ids if numbered else None
    want, bound, h_want, h_bound = p.forward()
    h = torch.full((tokens, rank), 9.0, device=cuda)
    out = ks.lora.apply(torch.full_like(p.base, 9.0), p.base, p.x, p.a, p.b, p.scales, order, part, h=h)
    check("out", out[~before], want[~before], bound[~before])
    assert (out[before] == 9).all() and (h[p.ids < 0] == 9).all()
    check("h", h[p.ids >= 0], h_want[p.ids >= 0], h_bound[p.ids >= 0])
    hf = h_want.float()
    want, bounds = p.backward(hf)
    d_x, d_a, d_b = ks.lora.backward(torch.full_like(p.x, 9.0), torch.empty_like(p.a), torch.empty_like(p.b), p.d_x_base, p.d_out, p.x, hf, p.a,
                                     p.b, p.scales, order, part)
    check("d_x", d_x[~before], want[0][~before], bounds[0][~before])
    assert (d_x[before] == 9).all()
    check("d_a", d_a, want[1], bounds[1])
    check("d_b", d_b, want[2], bounds[2])
