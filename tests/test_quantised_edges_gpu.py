"""A cache in 8 and 4 bits where its table is a view of a wider one."""
import pytest
import torch

from quantised_oracle import decode, encode

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import quantised

    return quantised


def views(gen, b, most):
    """Tables of b sequences that are cut out of [b, most], every entry of which is a page of its own."""
    wide = torch.randperm(b * most, generator=gen).int().view(b, most).cuda()
    return wide, {"front": wide[:, :3], "middle": wide[:, 2:5], "end": wide[:, most - 2:], "one": wide[:, 4:5], "all": wide}


@pytest.mark.parametrize("bits, dtype, d", [(4, BF16, 128), (8, BF16, 40), (4, F32, 64), (8, F32, 256)])
@pytest.mark.parametrize("which", ["front", "middle", "end", "one", "all"])
def test_slots_past_a_table_that_is_a_view(ops, bits, dtype, d, which):
    """Tokens past the pages that a view lists are not written, and read as zeros: neither the entries beside the view nor the next
    sequence's are the sequence's own."""
    print(bits, dtype, d, which, flush=True)
    gen = torch.Generator().manual_seed(21)
    b, hkv, page, most = 3, 2, 16, 7
    _, tables = views(gen, b, most)
    table = tables[which]
    room = page * table.shape[1]
    cache, plain = (ops.QuantisedCache(*(x.fill_(77) for x in other._tensors), d, bits) for other in (ops.QuantisedCache.empty(b * most, hkv, page, d, bits) for _ in range(2)))
    n = page * most + 40
    k, v = (torch.randn((b, hkv, n, d), generator=gen).to(dtype).cuda() for _ in range(2))
    first = torch.tensor([0, -5, room - 3], dtype=torch.int32, device="cuda")
    ops.store(cache, k, v, first=first, table=table)
    ops.store(plain, k, v, first=first, table=table.clone(memory_format=torch.contiguous_format))
    for got, want in zip(cache._tensors, plain._tensors):
        assert torch.equal(got, want)
    beside = sorted(set(range(b * most)) - set(table.flatten().tolist()))
    assert all(bool((x[beside] == 77).all()) for x in cache._tensors)
    whole = torch.zeros_like(first)
    got = ops.load(cache, n, first=whole, table=table, dtype=dtype)
    for x, y in zip(got, (k, v)):
        kept = decode(*encode(y.cpu(), bits), d, bits)
        x = x.cpu().double()
        assert not x[:, :, room:].any()
        assert torch.equal(x[0, :, :room], kept[0, :, :room])
        assert torch.equal(x[1, :, :room], kept[1, :, 5:5 + room])
        assert torch.equal(x[2, :, room - 3:room], kept[2, :, :3])


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_over_a_table_that_is_a_view(ops, bits):
    gen = torch.Generator().manual_seed(22)
    b, hq, hkv, page, most, d = 3, 8, 2, 16, 40, 64
    cache = ops.QuantisedCache.empty(b * most, hkv, page, d, bits)
    wide, _ = views(gen, b, most)
    k, v = (torch.randn((b, hkv, page * most, d), generator=gen).to(BF16).cuda() for _ in range(2))
    ops.store(cache, k, v, table=wide)
    for nodes in (1, 30):
        q = torch.randn((b, hq, nodes, d), generator=gen).to(BF16).cuda()
        lengths = torch.tensor([10 ** 6, 100, 0], dtype=torch.int32, device="cuda")
        for table in (wide[:, :9], wide[:, 11:30], wide[:, 38:]):
            got = ops.tree_attention(q, cache, lengths, table=table)
            want = ops.tree_attention(q, cache, lengths, table=table.contiguous())
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
