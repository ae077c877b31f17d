"""Inputs, 64-bit references and error bounds for the adapters' tests.

Bounds. u = eps(T)/2 is the one rounding of an output. A sum of n products in fp32, in a chain or by tensor-core
instructions of 16 products that may truncate, is off by at most (n/16 + 32) * 2^-23 times the sum of the magnitudes. The inner
vector enters the second product as two 16-bit numbers, off by at most 2^-18 of it in bf16, 2^-24 in f16 (2^-17 is
taken for both, with the row's scaling to a power of two exact)."""
import torch

STEP = 2.0 ** -23


def chain(n):
    return (n / 16 + 32) * STEP


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Problem:
    def __init__(self, tokens, adapters, rank, k, n, dtype=torch.bfloat16, without=0.0, active=None, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)

        self.tokens, self.adapters, self.rank, self.k, self.n, self.dtype = tokens, adapters, rank, k, n, dtype
        ids = torch.randint(0, active or adapters, (tokens,), generator=g, device=device)
        none = torch.rand(tokens, generator=g, device=device) < without
        self.ids = torch.where(none, -1, ids).to(torch.int32)
        self.x = normal(tokens, k)
        self.base = normal(tokens, n)
        self.a = normal(adapters, rank, k, std=k ** -0.5)
        self.b = normal(adapters, n, rank, std=0.1)
        self.scales = torch.rand(adapters, generator=g, device=device) + 0.5
        self.d_out = normal(tokens, n, std=0.05)
        self.d_x_base = normal(tokens, k, std=0.05)

    def rows(self, a):
        return (self.ids == a).nonzero()[:, 0]

    def forward(self):
        """(out, bound, h, h bound) in 64 bits; h is zero for rows without an adapter."""
        out, mag = self.base.double(), torch.zeros(self.tokens, self.n, dtype=torch.float64, device=self.x.device)
        h = torch.zeros(self.tokens, self.rank, dtype=torch.float64, device=self.x.device)
        hmag = torch.zeros_like(h)
        for a in range(self.adapters):
            r = self.rows(a)
            x, fa, fb, s = self.x[r].double(), self.a[a].double(), self.b[a].double(), float(self.scales[a])
            h[r], hmag[r] = x @ fa.t(), x.abs() @ fa.t().abs()
            out[r] += s * (h[r] @ fb.t())
            mag[r] = s * (hmag[r] @ fb.t().abs())
        c = chain(self.k) + chain(self.rank) + 2.0 ** -17
        bound = half_step(self.dtype) * (out.abs() + c * mag) + c * mag + 2 * STEP * self.base.abs().double()
        return out, bound, h, chain(self.k) * hmag

    def backward(self, h):
        """((d_x, d_a, d_b), bounds) in 64 bits for the fp32 ``h`` that the call is given."""
        u = half_step(self.dtype)
        d_x, xmag = self.d_x_base.double(), torch.zeros(self.tokens, self.k, dtype=torch.float64, device=self.x.device)
        d_a, d_b = torch.zeros_like(self.a, dtype=torch.float64), torch.zeros_like(self.b, dtype=torch.float64)
        a_mag, b_mag = torch.zeros_like(d_a), torch.zeros_like(d_b)
        for a in range(self.adapters):
            r = self.rows(a)
            x, fa, fb, s = self.x[r].double(), self.a[a].double(), self.b[a].double(), float(self.scales[a])
            dout, hr = self.d_out[r].double(), h[r].double()
            g, gmag = s * (dout @ fb), s * (dout.abs() @ fb.abs())
            d_x[r] += g @ fa
            xmag[r] = gmag @ fa.abs()
            d_a[a], a_mag[a] = g.t() @ x, gmag.t() @ x.abs()
            d_b[a], b_mag[a] = s * (dout.t() @ hr), s * (dout.abs().t() @ hr.abs())
        cx = chain(self.n) + chain(self.rank) + 2.0 ** -17
        ca = chain(self.n) + chain(self.tokens) + 2.0 ** -17
        cb = chain(self.tokens) + 2.0 ** -17
        tiny = torch.finfo(self.dtype).smallest_normal * torch.finfo(self.dtype).eps   # half a subnormal step and some
        bounds = (u * (d_x.abs() + cx * xmag) + cx * xmag + 2 * STEP * self.d_x_base.abs().double() + tiny,
                  u * (d_a.abs() + ca * a_mag) + ca * a_mag + tiny, u * (d_b.abs() + cb * b_mag) + cb * b_mag + tiny)
        return (d_x, d_a, d_b), bounds


def check(what, got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements off by more than their bound; first {i}: "
                             f"{float(got[i])} where {float(want[i])} +- {float(bound[i])} is expected")
