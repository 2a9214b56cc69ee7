"""Trees of drafted tokens over a cache in pages, and eviction from it, against float64 and plain selection on the CPU."""
import math

import pytest
import torch

from attend_oracle import Attention, within

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import attention

    return attention


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=F32, device="cuda")


def signed(word):
    return word - (1 << 64) if word >> 63 else word


def tree_words(gen, nodes):
    words = []
    for t in range(nodes):
        parent = int(torch.randint(0, t, (1,), generator=gen)) if t else None
        words.append((words[parent] if t else 0) | 1 << t)
    return words


class Cache:
    """A cache in pages, in an order of their own, filled with `rest` where no sequence has a slot."""

    def __init__(self, seed, dtype, b, hkv, d, page, slots, heads_last=False, rest=math.nan):
        gen = self.gen = torch.Generator().manual_seed(seed)
        per = max(1, -(-slots // page))
        self.page, self.slots, self.per, self.rest = page, slots, per, rest
        order = torch.randperm(b * per + 2, generator=gen)[:b * per].view(b, per)
        shape = (b * per + 2, page, hkv, d) if heads_last else (b * per + 2, hkv, page, d)
        k, v = (torch.full(shape, rest, dtype=dtype).cuda() for _ in range(2))
        self.k, self.v = (x.transpose(1, 2) if heads_last else x for x in (k, v))
        self.table = order.int().cuda()
        self.dense = [torch.randn((b, hkv, slots, d), generator=gen).to(dtype) for _ in range(2)]

    def fill(self, lengths):
        """The first lengths[s] slots of every sequence."""
        for s, n in enumerate(lengths):
            for x, dense in ((self.k, self.dense[0]), (self.v, self.dense[1])):
                for slot0 in range(0, n, self.page):
                    slot1 = min(n, slot0 + self.page)
                    x[self.table[s, slot0 // self.page], :, :slot1 - slot0] = dense[s, :, slot0:slot1].cuda()


# type, b, hq, hkv, nodes, longest, d, page, cap, bias, accumulate, heads last
TREES = [
    (BF16, 1, 1, 1, 1, 0, 64, 16, 0.0, False, False, False),
    (F32, 1, 1, 1, 1, 1, 8, 1, 0.0, False, True, False),
    (BF16, 3, 8, 2, 1, 700, 128, 64, 0.0, False, True, True),
    (BF16, 2, 4, 4, 1, 90, 64, 7, 0.0, True, True, False),
    (BF16, 2, 8, 2, 5, 333, 128, 16, 30.0, False, False, True),
    (BF16, 2, 8, 2, 48, 1500, 128, 33, 50.0, True, True, False),
    (BF16, 1, 6, 1, 64, 2500, 64, 256, 0.0, False, True, False),
    (BF16, 1, 4, 2, 9, 500, 256, 64, 0.0, True, False, False),
    (BF16, 1, 40, 1, 1, 300, 80, 16, 0.0, False, True, True),
    (F32, 2, 4, 2, 1, 300, 64, 20, 0.0, True, True, False),
    (F32, 1, 8, 2, 12, 400, 128, 64, 10.0, False, True, True),
    (F32, 1, 2, 1, 33, 129, 256, 64, 0.0, False, False, False),
    (F32, 2, 3, 3, 64, 65, 40, 16, 0.0, True, True, False),
]


def names(case):
    return "-".join(str(x).replace("torch.", "") for x in case)


# Work that is dealt out over many sequences, tables of more pages and biases of more keys than a workgroup looks up at once.
DEALT = [
    (BF16, 70, 4, 2, 1, 300, 64, 16, 0.0, False, True, True),
    (F32, 130, 2, 1, 3, 40, 64, 5, 0.0, True, False, False),
    (BF16, 2, 2, 1, 5, 1500, 128, 1, 0.0, True, True, True),
    (BF16, 1, 2, 2, 2, 9000, 64, 2, 0.0, False, False, False),
    (F32, 2, 4, 1, 40, 2500, 64, 1, 20.0, True, True, True),
    (BF16, 2, 8, 1, 64, 1700, 128, 7, 0.0, False, False, True),
    (BF16, 1, 6, 2, 33, 1300, 256, 64, 30.0, True, True, False),
    (F32, 1, 3, 1, 50, 700, 256, 16, 0.0, False, False, True),
    (F32, 5, 3, 1, 11, 700, 256, 16, 0.0, False, True, True),
    (F32, 3, 6, 2, 4, 1500, 64, 16, 0.0, True, True, True),
    (F32, 70, 6, 6, 5, 400, 64, 16, 0.0, False, True, True),
    (BF16, 70, 2, 1, 2, 2300, 64, 64, 0.0, False, True, True),
    (BF16, 3, 8, 2, 8, 1100, 128, 64, 0.0, True, True, False),
]


@pytest.mark.parametrize("case", DEALT, ids=names)
def test_trees_of_many_keys(ops, case):
    test_trees(ops, case)


@pytest.mark.parametrize("case", TREES, ids=names)
def test_trees(ops, case):
    dtype, b, hq, hkv, nodes, longest, d, page, cap, bias, accumulate, heads_last = case
    print(names(case), flush=True)
    cache = Cache(nodes + longest, dtype, b, hkv, d, page, longest + nodes, heads_last)
    lengths = [longest] + [int(torch.randint(0, longest + 1, (1,), generator=cache.gen)) for _ in range(b - 1)]
    cache.fill([n + nodes for n in lengths])
    words = [tree_words(cache.gen, nodes) for _ in range(b)]
    q = (torch.randn((b, hq, nodes, d), generator=cache.gen) * 1.5).to(dtype).cuda()
    slots = cache.per * page
    weights = torch.rand((b, hkv, slots + 3), generator=cache.gen).cuda()
    options = {"cap": cap, "slopes": slopes_of(hq) if bias else None}
    kept = {"weights": weights, "weights_out": torch.full_like(weights, -1.0)} if accumulate else {}
    o, lse = ops.tree_attention(q, cache.k, cache.v, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table=cache.table,
                                visible=torch.tensor([[signed(w) for w in row] for row in words], device="cuda"), **options, **kept)
    for s, n in enumerate(lengths):
        total = n + nodes
        sees = torch.tensor([[bool(w >> u & 1) for u in range(nodes)] for w in words[s]])
        hidden = torch.cat([torch.zeros((nodes, n), dtype=torch.bool), ~sees], 1)[None]
        depth = sees.sum(1) - 1
        position = torch.cat([torch.arange(n), n + depth])
        distance = (n + depth[:, None] - position[None]).abs().double().expand(1, hq, nodes, total)
        want = Attention(q[s:s + 1], cache.dense[0][s:s + 1, :, :total], cache.dense[1][s:s + 1, :, :total], hidden=hidden, distance=distance, **options)
        within(o[s:s + 1], want.o, want.o_bound, f"o of sequence {s}")
        within(lse[s:s + 1], want.lse, want.lse_bound, f"lse of sequence {s}")
        if accumulate:
            step, bound = want.weights()
            before = weights[s:s + 1].cpu().double()
            expected = before.clone()
            expected[:, :, :total] += step
            full = torch.full_like(expected, 2.0 ** -23 * float(expected.max()))
            full[:, :, :total] += bound
            within(kept["weights_out"][s:s + 1, :, :slots], expected[:, :, :slots], full[:, :, :slots], f"weights of sequence {s}")
    if accumulate:
        assert bool((kept["weights_out"][:, :, slots:] == -1.0).all())


def test_a_chain_is_causal_and_counted_nodes_count(ops):
    dtype, b, hq, hkv, nodes, d = BF16, 2, 4, 2, 6, 64
    cache = Cache(7, dtype, b, hkv, d, 32, 100 + nodes)
    cache.fill([100 + nodes] * b)
    lengths = torch.full((b,), 100, dtype=torch.int32, device="cuda")
    q = torch.randn((b, hq, nodes, d), generator=cache.gen).to(dtype).cuda()
    weights = torch.zeros((b, hkv, 106), device="cuda")
    o, lse = ops.tree_attention(q, cache.k, cache.v, lengths, table=cache.table, weights=weights, counted=0b100001, max_length=106)
    want = Attention(q, cache.dense[0], cache.dense[1], causal=True)
    within(o, want.o, want.o_bound, "o")
    want.p[:, :, 1:5] = 0.0
    within(weights, *want.weights(), "weights")
    # one word for all sequences
    words = torch.tensor([(2 << t) - 1 for t in range(nodes)], device="cuda")
    assert torch.equal(o, ops.tree_attention(q, cache.k, cache.v, lengths, table=cache.table, visible=words, max_length=106)[0])


def test_positions_of_a_cut_cache(ops):
    dtype, b, hq, hkv, d, n = F32, 2, 4, 2, 64, 77
    cache = Cache(8, dtype, b, hkv, d, 16, n + 1)
    cache.fill([n + 1] * b)
    positions = torch.randint(0, 900, (b, hkv, n + 1), generator=cache.gen, dtype=torch.int32).sort(-1).values
    q = torch.randn((b, hq, 1, d), generator=cache.gen).cuda()
    start = torch.tensor([900, 950], dtype=torch.int32, device="cuda")
    slopes = slopes_of(hq)
    o, lse = ops.tree_attention(q, cache.k, cache.v, torch.full((b,), n, dtype=torch.int32, device="cuda"), table=cache.table, slopes=slopes, start=start,
                                positions=positions.cuda(), max_length=n + 1)
    of = positions.repeat_interleave(hq // hkv, 1).clone()
    of[:, :, n] = start.cpu()[:, None]
    distance = (start.cpu().view(b, 1, 1, 1) - of[:, :, None, :]).abs().double()
    want = Attention(q, cache.dense[0], cache.dense[1], slopes=slopes, distance=distance, hidden=torch.zeros((b, 1, n + 1), dtype=torch.bool))
    within(o, want.o, want.o_bound, "o")


def test_nodes_that_see_nothing(ops):
    cache = Cache(9, BF16, 1, 1, 64, 16, 3)
    cache.fill([3])
    q = torch.randn((1, 2, 3, 64), generator=cache.gen).to(BF16).cuda()
    o, lse = ops.tree_attention(q, cache.k, cache.v, torch.zeros(1, dtype=torch.int32, device="cuda"), table=cache.table,
                                visible=torch.tensor([[1, 0, 5]], device="cuda"))
    assert torch.equal(o[:, :, 1], torch.zeros_like(o[:, :, 1])) and bool((lse[:, :, 1] == -math.inf).all())
    assert torch.equal(o[0, 0, 0].cpu(), cache.dense[1][0, 0, 0])


def test_a_cache_without_a_table_and_slices(ops):
    """The longest part of each sequence's own page; a length past it is cut."""
    gen = torch.Generator().manual_seed(10)
    b, hq, hkv, n, d = 3, 4, 4, 200, 64
    k, v = (torch.randn((b, hkv, n, d), generator=gen).to(BF16).cuda() for _ in range(2))
    q = torch.randn((b, hq, 1, d), generator=gen).to(BF16).cuda()
    lengths = torch.tensor([199, 5000, 50], dtype=torch.int32, device="cuda")
    o, lse = ops.tree_attention(q, k, v, lengths)
    hidden = torch.arange(n)[None, None, :] >= torch.tensor([200, 200, 51])[:, None, None]
    want = Attention(q, k, v, hidden=hidden)
    within(o, want.o, want.o_bound, "o")


def test_one_token_of_a_long_cache_in_a_graph(ops):
    gen = torch.Generator().manual_seed(12)
    k, v = (torch.randn((1, 2, 5000, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    q = torch.randn((1, 8, 1, 64), generator=gen).to(BF16).cuda()
    lengths = torch.tensor([4000], dtype=torch.int32, device="cuda")
    weights = torch.rand((1, 2, 5000), generator=gen).cuda()
    out = torch.empty_like(weights)
    ops.tree_attention(q, k, v, lengths, weights=weights, weights_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = ops.tree_attention(q, k, v, lengths, weights=weights, weights_out=out)
    for n in (4000, 77, 4999):
        lengths.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(out)
        eager, eager_lse = ops.tree_attention(q, k, v, lengths, weights=weights, weights_out=again)
        assert torch.equal(o, eager) and torch.equal(lse, eager_lse) and torch.equal(out, again)
        want = Attention(q, k[:, :, :n + 1], v[:, :, :n + 1])
        within(o, want.o, want.o_bound, f"o at {n}")


# ---------------------------------------------------------------- eviction
def chosen_slots(weights, n, keep, recent):
    if n <= keep:
        return list(range(n))
    rank = [-math.inf if math.isnan(w) else w for w in weights[:n - recent]]
    old = sorted(range(n - recent), key=lambda j: -rank[j])[:keep - recent]
    return sorted(old) + list(range(n - recent, n))


# type, b, hkv, longest, keep, recent, d, page, page of the new cache, kind of weights
EVICTIONS = [
    (BF16, 1, 1, 2, 1, 0, 64, 16, 1, "spread"),
    (BF16, 3, 2, 700, 200, 50, 128, 64, 16, "spread"),
    (F32, 2, 3, 501, 101, 101, 40, 7, 33, "spread"),
    (BF16, 2, 2, 2300, 1100, 0, 64, 256, 64, "equal"),
    (F32, 2, 1, 1500, 333, 17, 8, 16, 16, "few"),
    (BF16, 1, 2, 4097, 2048, 100, 256, 64, 64, "negative"),
    (BF16, 2, 2, 300, 100, 10, 80, 16, 16, "odd"),
    (F32, 1, 2, 90, 90, 5, 64, 16, 100, "spread"),
    (F32, 2, 2, 60, 90, 5, 64, 16, 100, "spread"),
    (BF16, 1, 1, 40000, 777, 3, 64, 512, 16, "spread"),
]


@pytest.mark.parametrize("case", EVICTIONS, ids=names)
def test_evictions(ops, case):
    dtype, b, hkv, longest, keep, recent, d, page, page_out, kind = case
    print(names(case), flush=True)
    cache = Cache(longest + keep, dtype, b, hkv, d, page, longest, heads_last=True, rest=0.0)
    gen = cache.gen
    lengths = [longest] + [int(torch.randint(0, longest + 1, (1,), generator=gen)) for _ in range(b - 1)]
    cache.fill(lengths)
    weights = torch.rand((b, hkv, longest + 5), generator=gen) ** 8
    if kind == "equal":
        weights[:] = 0.25
    elif kind == "few":
        weights = torch.randint(0, 3, weights.shape, generator=gen).float()
    elif kind == "negative":
        weights = torch.randn(weights.shape, generator=gen)
    elif kind == "odd":
        weights[:, :, ::7], weights[:, :, 1::7], weights[:, :, 2::7], weights[:, :, 3::7] = math.nan, math.inf, -0.0, 0.0
    positions = torch.randint(0, 10 ** 6, (b, hkv, longest), generator=gen, dtype=torch.int32)
    per_out = -(-keep // page_out)
    k_out, v_out = (torch.full((b * per_out, hkv, page_out, d), -3.0, dtype=dtype, device="cuda") for _ in range(2))
    table_out = torch.randperm(b * per_out, generator=gen).view(b, per_out).int().cuda()
    out = (k_out, v_out, torch.full((b, hkv, keep), -3.0, device="cuda"), torch.full((b, hkv, keep), -3, dtype=torch.int32, device="cuda"),
           torch.full((b,), -3, dtype=torch.int32, device="cuda"))
    got = ops.evict(cache.k, cache.v, weights.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, recent, table=cache.table,
                    positions=positions.cuda(), table_out=table_out, out=out, max_length=longest)
    assert got is out
    assert out[4].tolist() == [min(n, keep) for n in lengths]
    for s, n in enumerate(lengths):
        for h in range(hkv):
            slots = chosen_slots(weights[s, h].tolist(), n, keep, recent)
            at = torch.tensor(slots, dtype=torch.long)
            assert out[3][s, h, :len(slots)].tolist() == positions[s, h, at].tolist()
            assert torch.equal(out[2][s, h, :len(slots)].cpu().view(torch.int32), weights[s, h, at].view(torch.int32))
            for x, dense in ((k_out, cache.dense[0]), (v_out, cache.dense[1])):
                rows = x[table_out[s].long(), h].reshape(per_out * page_out, d).cpu()
                assert torch.equal(rows[:len(slots)], dense[s, h, at])
                assert bool((rows[len(slots):] == -3.0).all())
            assert bool((out[2][s, h, len(slots):] == -3.0).all()) and bool((out[3][s, h, len(slots):] == -3).all())


@pytest.mark.parametrize("case", [(F32, 1, 1, 20011, 3000, 17, 64, 64, 100, "few"), (BF16, 1, 2, 40000, 35001, 0, 64, 256, 256, "odd")], ids=names)
def test_evictions_of_long_caches(ops, case):
    test_evictions(ops, case)


def test_offsets_that_pass_32_bits(ops):
    """Pages beyond 4 GiB of K and of V: read by a token, cut, and read again; keys of a prompt whose heads lie as far apart."""
    pages, page, d, n, nodes, keep = 300000, 64, 128, 700, 3, 200
    gen = torch.Generator().manual_seed(41)
    k, v = (torch.empty((pages, 1, page, d), dtype=BF16, device="cuda") for _ in range(2))
    dense = [torch.randn((1, 1, 704, d), generator=gen).to(BF16) for _ in range(2)]
    table = torch.arange(pages - 1, pages - 12, -1, dtype=torch.int32, device="cuda")[None]
    for x, of in zip((k, v), dense):
        x[table[0].long(), 0] = of.view(11, page, d).cuda()
    q = torch.randn((1, 4, nodes, d), generator=gen).to(BF16).cuda()
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    hidden = torch.cat([torch.zeros((nodes, n), dtype=torch.bool), torch.ones((nodes, nodes), dtype=torch.bool).triu(1)], 1)[None]
    want = Attention(q, dense[0][:, :, :n + nodes], dense[1][:, :, :n + nodes], hidden=hidden)
    o, lse = ops.tree_attention(q, k, v, lengths, table=table)
    within(o, want.o, want.o_bound, "o")
    weights = torch.rand((1, 1, n), generator=gen)
    k2, v2, *_ = ops.evict(k, v, weights.cuda(), lengths, keep, 10, table=table, max_length=n)
    at = torch.tensor(chosen_slots(weights[0, 0].tolist(), n, keep, 10), dtype=torch.long)
    assert torch.equal(k2[0, 0].cpu(), dense[0][0, 0, at]) and torch.equal(v2[0, 0].cpu(), dense[1][0, 0, at])
    del v
    far = k.view(-1).as_strided((1, 2, 90, d), (0, 2 ** 31 + 64, d, 1))
    for h in range(2):
        far[0, h] = dense[h][0, 0, :90].cuda()
    q = torch.randn((1, 2, 90, d), generator=gen).to(BF16).cuda()
    want = Attention(q, far, far, causal=True)
    o, _ = ops.attention(q, far, far, causal=True)
    within(o, want.o, want.o_bound, "o of far heads")


def test_evicted_caches_serve_on(ops):
    """New tensors, one page a sequence; then a token against the cut cache is attention over what stayed."""
    gen = torch.Generator().manual_seed(33)
    b, hq, hkv, n, d, keep = 2, 4, 2, 150, 64, 40
    k, v = (torch.randn((b, hkv, n, d), generator=gen).to(BF16).cuda() for _ in range(2))
    weights = torch.rand((b, hkv, n), generator=gen).cuda()
    k2, v2, weights2, positions, lengths = ops.evict(k, v, weights, torch.full((b,), n, dtype=torch.int32, device="cuda"), keep, 8)
    at = positions.long()[..., None].expand(b, hkv, keep, d)
    assert torch.equal(k2, k.gather(2, at)) and torch.equal(v2, v.gather(2, at)) and torch.equal(weights2, weights.gather(2, positions.long()))
    assert lengths.tolist() == [keep] * b
    q = torch.randn((b, hq, 1, d), generator=gen).to(BF16).cuda()
    o, _ = ops.tree_attention(q, k2, v2, lengths - 1)
    want = Attention(q, k2, v2)
    within(o, want.o, want.o_bound, "o")


def test_refusals(ops):
    gen = torch.Generator().manual_seed(44)
    k, v = (torch.randn((4, 2, 16, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    q = torch.randn((2, 4, 3, 64), generator=gen).to(BF16).cuda()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([5, 20], dtype=torch.int32, device="cuda")
    weights = torch.zeros((2, 2, 32), device="cuda")
    ops.tree_attention(q, k, v, lengths, table=table, weights=weights)
    for bad in (lambda: ops.tree_attention(q, k.float(), v, lengths, table=table), lambda: ops.tree_attention(q, k, v, lengths.long(), table=table),
                lambda: ops.tree_attention(q, k, v, lengths, table=table.long()), lambda: ops.tree_attention(q, k, v, lengths.cpu(), table=table)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.tree_attention(q, k, v, lengths[:1], table=table), lambda: ops.tree_attention(q, k, v, lengths, table=table[:1]),
                lambda: ops.tree_attention(q, k, v, lengths, table=table, visible=torch.zeros((2, 4), dtype=torch.int64, device="cuda")),
                lambda: ops.tree_attention(q, k, v, lengths, table=table, weights_out=weights)):
        with pytest.raises(ValueError):
            bad()
    many = torch.zeros((2, 4, 65, 64), dtype=BF16, device="cuda")
    for bad in (lambda: ops.tree_attention(many, k, v, lengths, table=table), lambda: ops.tree_attention(q, k, v, lengths, table=table, cap=-2.0),
                lambda: ops.tree_attention(q, k, v, lengths, table=table, max_length=2),
                lambda: ops.tree_attention(q, k, v, lengths, table=table, weights=torch.zeros((2, 2, 31), device="cuda")),
                lambda: ops.tree_attention(torch.zeros((5, 4, 1, 64), dtype=BF16, device="cuda"), k, v, torch.zeros(5, dtype=torch.int32, device="cuda"))):
        with pytest.raises(RuntimeError, match="tree_attention"):
            bad()
    for keep, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises((RuntimeError, ValueError)):
            ops.evict(k, v, weights, lengths, keep, recent, table=table)
    with pytest.raises(RuntimeError, match="evict"):  # room for 16 of 20 entries
        out = (k[:2].clone(), v[:2].clone(), torch.zeros((2, 2, 20), device="cuda"), torch.zeros((2, 2, 20), dtype=torch.int32, device="cuda"), lengths.clone())
        ops.evict(k, v, weights, lengths, 20, 2, table=table, out=out, table_out=torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"))
