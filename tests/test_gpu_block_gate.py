"""The join of an MoE layer's parts beside the layer's own combine (native_moe_combine_multi): the sums of a gated shared row.

The combine's gate is 1 / (1 + expf(-z)) in fp32: expf within 2 E (one step), the sum and the division E each, 4 E of the gate; the
join's is rounded once, E.  Each product with the shared row rounds once, 2 E, and each sum of the row onto the parts', E of it.
(E = 2^-24.)  expf overflows past z = -88, where the gate is under 2^-126."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24


@pytest.mark.parametrize("T,n,k", [(1, 64, 1), (7, 2048, 8), (300, 1000, 3), (64, 5120, 4)])
def test_gated_shared_rows(xm, T, n, k):
    g = torch.Generator().manual_seed(T)
    parts, shared = torch.randn(T * k, n, generator=g).to(DEV), torch.randn(T, n, generator=g).to(DEV)
    weights, z = torch.rand(T, k, generator=g).to(DEV), (4 * torch.randn(T, generator=g)).to(DEV)
    z[T // 2], z[-1] = 100.0, -100.0
    want = torch.empty(T, n, device=DEV)
    xm.native_moe_combine_multi(parts, weights, shared, want, n, k, T, shared_gate=z)
    got = xm.moe_combine_join(parts, weights, torch.zeros(T, n, device=DEV), xm.block_join_cfg(), shared=shared, shared_gate=z)[0]
    row = shared.double().abs() * torch.sigmoid(z.double())[:, None]
    bound = 7.01 * E * row + shared.double().abs() * 2.0 ** -126 + 2.01 * E * want.double().abs()
    assert ((got.double() - want.double()).abs() <= bound).all()
    # without the gate: the same bits
    xm.native_moe_combine_multi(parts, weights, shared, want, n, k, T)
    assert torch.equal(xm.moe_combine_join(parts, weights, torch.zeros(T, n, device=DEV), xm.block_join_cfg(), shared=shared)[0], want)
