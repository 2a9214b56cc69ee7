"""Eviction where the new cache's pages are not all given."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import attention

    return attention


def cache(seed, dtype, b, hkv, n, d):
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((b, hkv, n, d), generator=gen).to(dtype).cuda() for _ in range(2))
    return k, v, torch.rand((b, hkv, n), generator=gen).cuda()


@pytest.mark.parametrize("dtype,d,n,keep", [(BF16, 64, 100, 40), (F32, 128, 700, 300), (BF16, 128, 900, 900)], ids=str)  # one launch, two, nothing leaves
@pytest.mark.parametrize("missing", [-1, 10 ** 6, -2 ** 31])
def test_a_page_that_is_not_given_is_not_written(ops, dtype, d, n, keep, missing):
    """What would go to a page outside the new cache goes nowhere; page 0, another sequence's, keeps what it holds."""
    b, hkv, page = 2, 2, 16
    k, v, weights = cache(n, dtype, b, hkv, n, d)
    per = -(-keep // page)
    table = torch.arange(2 * per, dtype=torch.int32).view(2, per) + 1
    table[0, 1], table[1, per - 1], table[1, 0] = missing, missing, missing
    held = [torch.full((2 * per + 1, hkv, page, d), -7.0, dtype=dtype, device="cuda") for _ in range(2)]
    out = (*held, torch.empty((b, hkv, keep), device="cuda"), torch.empty((b, hkv, keep), dtype=torch.int32, device="cuda"), torch.empty(b, dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([n, n - 3], dtype=torch.int32, device="cuda")
    ops.evict(k, v, weights, lengths, keep, 10, table_out=table.cuda(), out=out)
    positions = out[3].cpu()
    for x, new in zip((k.cpu(), v.cpu()), (held[0].cpu(), held[1].cpu())):
        assert bool((new[0] == -7.0).all())
        for s in range(b):
            stay = min(keep, int(lengths[s]))
            for index in range(per):
                at = slice(index * page, min((index + 1) * page, stay))
                if 0 <= int(table[s, index]) < 2 * per + 1:
                    for h in range(hkv):
                        assert torch.equal(new[table[s, index], h, :at.stop - at.start], x[s, h, positions[s, h, at].long()])
        # pages that nobody was given
        unused = set(range(2 * per + 1)) - {int(p) for p in table.flatten()}
        assert all(bool((new[p] == -7.0).all()) for p in unused)


def test_lengths_and_weights_are_not_cut_in_place(ops):
    k, v, weights = cache(3, BF16, 2, 2, 90, 64)
    lengths = torch.full((2,), 90, dtype=torch.int32, device="cuda")
    new = ops.evict(k, v, weights, lengths, 30, 5)
    wide = torch.empty((2, 2, 90), dtype=torch.int32, device="cuda")
    for out in ((*new[:4], lengths), (*new[:2], weights, wide, new[4])):
        with pytest.raises(RuntimeError, match="evict.*share memory"):
            ops.evict(k, v, weights, lengths, 30, 5, out=out)
    positions = new[3].clone()
    again = ops.evict(*new[:3], new[4], 10, 2, positions=positions)
    with pytest.raises(RuntimeError, match="evict.*share memory"):
        ops.evict(*new[:3], new[4], 10, 2, positions=positions, out=(*again[:3], positions.view(-1)[:40].view(2, 2, 10), again[4]))
    assert lengths.tolist() == [90, 90]
