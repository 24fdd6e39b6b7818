"""A row's norm and int8 row do not depend on how many rows a call has, wherever 16-byte accesses take the rows; up to 4096
values they are the same in norms, joins and joins of parts too.  Elsewhere the squares may be summed in another order.

Random rows would hardly tell: another order moves the 64-bit sum by some 2^-53 of it, and r = 1 / sqrt(mean + eps), rounded to
24 bits, moves with it once in 10^8 rows.  So the rows here end in four values that bring r next to the middle between two
neighbouring fp32 numbers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6
E = 2.0 ** -24


def border_rows(seed, n_rows, n):
    """fp32 rows whose exact 1 / sqrt(sum / n + eps) is within some 2^-53 of the middle of two fp32 numbers."""
    assert np.finfo(np.longdouble).nmant >= 63
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n_rows, n)).astype(np.float32)
    x[:, -4:] = 0
    ss = (x.astype(np.longdouble) ** 2).sum(1)
    inv_n, eps = np.longdouble(1.0 / n), np.longdouble(np.float32(EPS))
    r = (1 / np.sqrt((ss + 0.7) * inv_n + eps)).astype(np.float32)
    mid = (r.astype(np.longdouble) + np.nextafter(r, np.float32(0)).astype(np.longdouble)) / 2
    rest = (1 / mid ** 2 - eps) / inv_n - ss
    assert (rest > 0).all()
    for i in range(-4, 0):
        v = np.sqrt(np.maximum(rest, 0)).astype(np.float32)
        v = np.where(v.astype(np.longdouble) ** 2 > rest, np.nextafter(v, np.float32(0)), v)
        x[:, i] = v
        rest = rest - v.astype(np.longdouble) ** 2
    return torch.from_numpy(x).to(DEV)


def results(xm, x, k=2):
    """The norm of x by every entry point, as {entry: (rows, codes, scales)}."""
    T, n = x.shape
    zero, parts, weights = torch.zeros_like(x), torch.zeros(T * k, n, device=DEV), torch.ones(T, k, device=DEV)
    plain = xm.block_join_cfg(next_eps=EPS)              # out = x, next = its norm
    normed = xm.block_join_cfg(norm=True, norm_eps=EPS)  # out = 0 + the norm of x
    return {"norm": xm.block_norm(x, None, EPS, quant=True),
            "join": xm.block_join(zero, x, plain, next_type=torch.float32, quant=True)[1:],
            "combine": xm.moe_combine_join(parts, weights, x, plain, next_type=torch.float32, quant=True)[1:],
            "joined norm": xm.block_join(x, zero, normed)[:1]}


def same(got, want, what):
    for v, w in zip(got, want):
        assert torch.equal(v, w[:len(v)]), (what, (v != w[:len(v)]).reshape(len(v), -1).any(1).sum().item())


def near(got, want):
    """Rows of r and of its neighbour: 2 E of the value, and the two products' roundings on each side, 4 E; a code moves by one
    at most, a scale as the largest value and its own rounding."""
    (y, *codes), (z, *wanted) = got, want
    z = z[:len(y)]
    assert ((y - z).abs() <= 6.01 * E * z.abs()).all()
    if codes:
        assert ((codes[0].int() - wanted[0][:len(y)].int()).abs() <= 1).all()
        assert ((codes[1] - wanted[1][:len(y)]).abs() <= 8.01 * E * codes[1]).all()


@pytest.mark.parametrize("n", [512, 1536, 2560, 4096, 5120, 6144, 7168, 8192, 8200, 16384, 1001, 3007, 4095, 8201, 5121, 6001, 8191])
def test_a_row_is_the_same_in_every_batch(xm, n):
    x = border_rows(n, 1040, n)
    every = results(xm, x)
    for T in (512, 511, 7, 1):
        for name, got in results(xm, x[:T]).items():
            if n % 8 and 4096 < n <= 8192:
                near(got, every[name])
            else:
                same(got, every[name], (name, T))
    for name, got in every.items():
        if n % 8 == 0 and n <= 4096:
            same(got, every["norm"], name)
        else:
            near(got, every["norm"])
