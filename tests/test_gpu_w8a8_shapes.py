"""Every shape of the int8 products' work-groups (w8a8_rule.CALLS; each test asserts that its call takes the shape that it is
for) with 16- and 32-bit outputs, rows of outputs apart and at odd starts, and the largest row strides.

Products are exact (one integer sum, three roundings, done here the same).  SwiGLU of exact g and u: 6 E of |h| with E = 2^-24
(exp 2 E, 1 + exp, the division and the product E each, and 1 E of slack), the stored type's half step, half of the smallest f16
step 2^-25, and 2^-120 of |u| where exp overflows."""
import pytest
import torch

from w8a8_rule import CALLS, IDS, shape

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def codes(seed, rows, n, into=None):
    """int8 rows of a whole number of 16 bytes (or the given view), and scales."""
    g = torch.Generator().manual_seed(seed)
    q = torch.empty(rows, (n + 15) // 16 * 16, dtype=torch.int8, device=DEV)[:, :n] if into is None else into
    q.copy_(torch.randint(-128, 128, (rows, n), generator=g).to(torch.int8))
    return q, (torch.rand(rows, generator=g) + 0.5).to(DEV)


def product(q, s, w, ws):
    return (q.double() @ w.double().T).float() * s[:, None] * ws


class Case:
    def __init__(self, call, store=None, seed=1):
        self.name, self.T, self.K, self.N, self.gated = call
        assert shape(self.T, self.K, self.N, self.gated) == self.name
        # columns of `store`, or rows of their own
        at = lambda i, rows: None if store is None else store[:rows, 65536 * i:65536 * i + self.K]   # noqa: E731
        self.q, s = codes(seed, self.T, self.K, at(0, self.T))
        self.s = s / (5000.0 * self.K ** 0.5)           # products of about 1 in the mean
        self.w, self.ws = codes(seed + 1, self.N, self.K, at(1, self.N))
        self.want = product(self.q, self.s, self.w, self.ws)
        if self.gated:
            self.u, self.us = codes(seed + 2, self.N, self.K, at(2, self.N))
            g, u = self.want.double(), product(self.q, self.s, self.u, self.us).double()
            self.want = g * torch.sigmoid(g) * u
            self.tol = 6 * E * self.want.abs() + u.abs() * 2.0 ** -120

    def run(self, xm, out):
        if self.gated:
            return xm.w8a8_swiglu(self.q, self.s, self.w, self.ws, self.u, self.us, out=out)
        return xm.w8a8_gemm(self.q, self.s, self.w, self.ws, out=out)

    def check(self, y):
        if not self.gated:
            assert torch.equal(y, self.want.to(y.dtype))
            return
        half = 0 if y.dtype == torch.float32 else torch.finfo(y.dtype).eps / 2 * self.want.abs() * (1 + 1e-6) + 2.0 ** -25
        assert ((y.double() - self.want).abs() <= self.tol + half).all()


@pytest.mark.parametrize("call", CALLS, ids=IDS)
def test_types_and_layouts(xm, call):
    """Rows of outputs next to each other, 16 bytes apart and by an odd number of values, from an even and an odd start; what is
    between, before and behind them stays."""
    c = Case(call)
    for t in TYPES:
        for ld, off in ((c.N, 0), ((c.N + 15) // 8 * 8, 0), ((c.N + 15) // 8 * 8, 2), (c.N + 1 + c.N % 2, 1)):
            store = torch.full(((c.T + 1) * ld + off,), 7.0, dtype=t, device=DEV)
            y = store[off:].view(c.T + 1, ld)
            c.run(xm, y[:c.T, :c.N])
            c.check(y[:c.T, :c.N])
            assert (y[c.T] == 7).all() and (y[:, c.N:] == 7).all() and (store[:off] == 7).all()


@pytest.mark.parametrize("call", [c for c in CALLS if c[0] in ("128x128", "128x256", "256x256")],
                         ids=lambda c: f"{'gated ' if c[4] else ''}{c[0]}")
def test_the_largest_strides(xm, call):
    """Rows of x and of the weights 8 MiB apart: a work-group's 256 rows reach 2^31 - 2^23 bytes past their first, the whole 2^35."""
    free = torch.cuda.mem_get_info()[0]
    rows, ld = max(call[1], call[3]), 1 << 23
    if free < rows * ld + (8 << 30):
        pytest.skip(f"{rows * ld >> 30} GiB of {free >> 30} free")
    store = torch.empty(rows, ld, dtype=torch.int8, device=DEV)
    try:
        c = Case(call, store, seed=5)
        assert c.q.stride(0) == c.w.stride(0) == ld
        c.check(c.run(xm, torch.empty(c.T, c.N, dtype=torch.bfloat16, device=DEV)))
    finally:
        c = None
        del store
        torch.cuda.empty_cache()
