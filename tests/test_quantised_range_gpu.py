"""Attention over a cache in 8 and 4 bits of values at both ends of the range that is promised."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import quantised

    return quantised


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nodes, d, n", [(1, 64, 1500), (3, 128, 900), (40, 64, 1500), (1, 256, 200)])
def test_values_of_any_promised_size(ops, dtype, bits, nodes, d, n):
    """Values times a power of two give outputs times it: codes are the same, scales, products and sums exactly as much larger.  Scores rise
    by 24 along the keys, so that exponentials grow to 2^30 before their reference follows.  Left: one rounding of the output's type, and
    of f32 sums 2^-22 of the largest value, where a part too small for bf16 moves a rounding."""
    print(dtype, bits, nodes, d, n, flush=True)
    gen = torch.Generator().manual_seed(40)
    b, hq, hkv, page = 2, 4, 2, 16
    per = -(-(n + nodes) // page)
    table = torch.randperm(b * per, generator=gen).int().view(b, per).cuda()
    along = torch.randn(d, generator=gen).sign()
    rise = 24.0 * torch.arange(n + nodes) / n  # of the scores, in natural units
    k = (rise[None, None, :, None] / d ** 0.5 * along + 0.1 * torch.randn((b, hkv, n + nodes, d), generator=gen)).to(dtype).cuda()
    v = torch.randn((b, hkv, n + nodes, d), generator=gen).to(dtype).cuda()
    q = (along + 0.1 * torch.randn((b, hq, nodes, d), generator=gen)).to(dtype).cuda()
    lengths = torch.tensor([n, n // 3], dtype=torch.int32, device="cuda")
    results = {}
    for exponent in (0, 70, -70):
        cache = ops.QuantisedCache.empty(b * per, hkv, page, d, bits)
        ops.store(cache, k, (v.double() * 2.0 ** exponent).to(dtype), table=table)
        o, lse = ops.tree_attention(q, cache, lengths, table=table)
        results[exponent] = o.cpu().double() * 2.0 ** -exponent, lse.cpu()
    want, lse = results[0]
    assert bool(want.isfinite().all()) and bool((want != 0).any())
    unit = 2.0 ** -7 if dtype is BF16 else 2.0 ** -23
    for exponent in (70, -70):
        got, other = results[exponent]
        assert torch.equal(lse, other)
        off = (got - want).abs()
        assert bool((off <= unit * want.abs() + 2.0 ** -22 * float(v.abs().max())).all()), (exponent, float(off.max()))
