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


def test_new_weights_past_what_stays_are_zero(ops):
    """A sequence shorter than the budget: what the next token's weights are added to in the slots behind it."""
    b, hkv, d, n, keep = 3, 2, 64, 50, 40
    k, v, weights = cache(5, BF16, b, hkv, n, d)
    lengths = torch.tensor([50, 17, 0], dtype=torch.int32, device="cuda")
    for size in (b * hkv * keep, b * hkv * (keep + 8)):
        spoil = [torch.full((2 ** 17,), math.nan, device="cuda") for _ in range(64)]
        del spoil  # (its memory is what the next tensors get)
        _, _, new, _, held = ops.evict(k, v, weights, lengths, keep, 5, room=size // (b * hkv) - keep)
        assert new.shape[2] == size // (b * hkv) and held.tolist() == [40, 17, 0]
        for s, stay in enumerate(held.tolist()):
            assert bool((new[s, :, stay:] == 0).all()) and bool((new[s, :, :stay] > 0).all())


def test_a_full_cache_is_cut_and_served_on(ops):
    """Evicted with room for drafted tokens, which are appended, checked as a tree, taken over in part, and followed by others."""
    from attend_oracle import Attention, within

    b, hq, hkv, d, n, keep, recent, nodes = 2, 4, 2, 64, 150, 40, 8, 3
    gen = torch.Generator().manual_seed(6)
    k, v, weights = cache(6, BF16, b, hkv, n, d)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    start = lengths.clone()  # positions go on where the text does
    k, v, weights, positions, lengths = ops.evict(k, v, weights, lengths, keep, recent, room=2 * nodes)
    assert k.shape == (b, hkv, keep + 2 * nodes, d) and positions.shape == weights.shape == (b, hkv, keep + 2 * nodes)
    tree = torch.tensor([0b001, 0b011, 0b101], device="cuda")  # nodes 1 and 2 follow node 0
    depth = torch.tensor([0, 1, 1])
    taken = 2
    for step in range(2):
        held = int(lengths[0])
        new = [torch.randn((b, hkv, nodes, d), generator=gen).to(BF16).cuda() for _ in range(2)]
        q = torch.randn((b, hq, nodes, d), generator=gen).to(BF16).cuda()
        k[:, :, held:held + nodes], v[:, :, held:held + nodes] = new
        before = weights.clone()
        o, _ = ops.tree_attention(q, k, v, lengths, visible=tree, slopes=slopes, start=start, positions=positions, weights=weights, counted=(1 << taken) - 1)
        at = torch.cat([positions[:, :, :held].cpu(), (start.cpu()[:, None] + depth)[:, None].expand(b, hkv, nodes)], 2)
        distance = ((start.cpu()[:, None] + depth)[:, None, :, None] - at.repeat_interleave(hq // hkv, 1)[:, :, None]).abs().double()
        hidden = torch.cat([torch.zeros((nodes, held), dtype=torch.bool), (tree.cpu()[:, None] >> torch.arange(nodes) & 1) == 0], 1)[None].expand(b, -1, -1)
        want = Attention(q, k[:, :, :held + nodes], v[:, :, :held + nodes], slopes=slopes, hidden=hidden, distance=distance)
        within(o, want.o, want.o_bound, f"o of step {step}")
        want.p[:, :, taken:] = 0
        ref, bound = want.weights()
        within(weights[:, :, :held + nodes], before[:, :, :held + nodes].cpu().double() + ref, bound + 2.0 ** -23 * before.max().item(), f"weights of step {step}")
        weights[:, :, held + taken:] = 0
        positions[:, :, held:held + taken] = start[:, None, None] + torch.arange(taken, device="cuda", dtype=torch.int32)
        lengths, start = lengths + taken, start + taken


def test_room_is_checked(ops):
    k, v, weights = cache(7, F32, 1, 1, 20, 64)
    lengths = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="room"):
        ops.evict(k, v, weights, lengths, 5, 1, room=-1)
    with pytest.raises(ValueError, match="room"):
        ops.evict(k, v, weights, lengths, 5, 1, room=3, out=ops.evict(k, v, weights, lengths, 5, 1))
