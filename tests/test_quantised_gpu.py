"""A cache in 8 and 4 bits in pages: writing, reading back and attention over it, against float64 on the CPU."""
import math

import pytest
import torch

from attend_oracle import Attention, within
from quantised_oracle import decode, encode, packed

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import quantised

    return quantised


def names(case):
    return "-".join(str(x).replace("torch.", "") for x in case)


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


def rough(gen, *shape):
    """Values of many magnitudes: rows of one, tiny and huge ones, zeros, halves between codes."""
    x = torch.randn(shape, generator=gen)
    kind = torch.randint(0, 8, shape[:-1], generator=gen)[..., None]
    x = torch.where(kind == 1, x * 1e-38, x)
    x = torch.where(kind == 2, x * 3e37, x)
    x = torch.where(kind == 3, torch.zeros_like(x), x)
    x = torch.where(kind == 4, (x * 8).round() / 4, x)
    x = torch.where(kind == 5, torch.exp(x * 8), x)
    x = torch.where((kind == 6) & (torch.rand(shape, generator=gen) < 0.9), -torch.zeros_like(x), x)
    return x


class Pages:
    """A cache in pages in an order of their own, all bytes 255 (no numbers) to begin with."""

    def __init__(self, ops, gen, bits, b, hkv, d, page, slots, heads_last=False, rest=255):
        self.per = max(1, -(-slots // page))
        self.page, self.b, self.bits, self.d = page, b, bits, d
        columns = -(-d // 32) * 32
        order = torch.randperm(b * self.per + 2, generator=gen)[:b * self.per].view(b, self.per)
        pages = b * self.per + 2

        def memory(width):
            if heads_last:  # (a row's bytes with room after them, heads beside each other)
                return torch.full((pages, page, hkv, width + 16), rest, dtype=torch.uint8, device="cuda").transpose(1, 2)[..., :width]
            return torch.full((pages, hkv, page, width), rest, dtype=torch.uint8, device="cuda")

        self.cache = ops.QuantisedCache(memory(columns * bits // 8), memory(columns // 32), memory(columns * bits // 8), memory(columns // 32), d, bits)
        self.table = order.int().cuda()

    def slot(self, s, n):
        return self.table[s, n // self.page].long(), n % self.page

    def fill(self, gen, lengths, dtype):
        """Codes of random rows in the first lengths[s] slots; their values [b, hkv, most, d] in dtype (exact)."""
        dense = []
        for codes, scales in ((self.cache.k, self.cache.k_scales), (self.cache.v, self.cache.v_scales)):
            values = torch.randn((self.b, codes.shape[1], max(lengths), self.d), generator=gen)
            values[..., 1] *= 5
            code, scale = encode(values, self.bits)
            kept = decode(code, scale, self.d, self.bits).to(dtype)
            rows = packed(code, self.bits).cuda()
            scale = scale.cuda()
            for s, n in enumerate(lengths):
                at = torch.arange(n, device="cuda")
                page, slot = self.slot(s, at)
                codes[page, :, slot] = rows[s, :, :n].transpose(0, 1)
                scales[page, :, slot] = scale[s, :, :n].transpose(0, 1)
            dense.append(kept)
        return dense


# type, bits, b, hkv, n, d, page, heads last
MOVES = [
    (BF16, 4, 1, 1, 1, 8, 1, False),
    (BF16, 4, 2, 3, 50, 128, 16, False),
    (BF16, 8, 2, 3, 50, 128, 16, True),
    (BF16, 4, 3, 2, 33, 72, 7, True),
    (BF16, 8, 3, 2, 33, 40, 64, False),
    (BF16, 4, 2, 1, 9, 256, 5, True),
    (BF16, 8, 1, 5, 130, 192, 32, False),
    (F32, 4, 2, 3, 70, 64, 16, False),
    (F32, 8, 2, 2, 21, 136, 8, True),
    (F32, 4, 1, 4, 5, 256, 256, False),
    (F32, 8, 4, 1, 1, 32, 3, False),
]


@pytest.mark.parametrize("case", MOVES, ids=names)
def test_store_and_load(ops, case):
    dtype, bits, b, hkv, n, d, page, heads_last = case
    print(names(case), flush=True)
    gen = torch.Generator().manual_seed(n + d)
    slots = n + 11
    at = Pages(ops, gen, bits, b, hkv, d, page, slots, heads_last)
    first = torch.randint(0, 11, (b,), generator=gen)
    counts = torch.randint(0, n + 1, (b,), generator=gen)
    counts[0] = n
    k, v = (rough(gen, b, n, hkv, d).to(dtype).transpose(1, 2) if heads_last else rough(gen, b, hkv, n, d).to(dtype) for _ in range(2))
    want = [x.clone().cpu() for x in (at.cache.k, at.cache.k_scales, at.cache.v, at.cache.v_scales)]
    kept = []
    for x, codes, scales in ((k, want[0], want[1]), (v, want[2], want[3])):
        code, scale = encode(x, bits)
        value = decode(code, scale, d, bits)
        for s in range(b):
            for t in range(int(counts[s])):
                page_at, slot = (int(y) for y in at.slot(s, int(first[s]) + t))
                codes[page_at, :, slot] = packed(code, bits)[s, :, t]
                scales[page_at, :, slot] = scale[s, :, t]
            value[s, :, int(counts[s]):] = 0
        kept.append(value)
    where = {"first": first.int().cuda(), "counts": counts.int().cuda(), "table": at.table}
    ops.store(at.cache, k.cuda(), v.cuda(), **where)
    for got, expected, name in zip((at.cache.k, at.cache.k_scales, at.cache.v, at.cache.v_scales), want, ("k", "k scales", "v", "v scales")):
        assert torch.equal(got.cpu(), expected), name
    for out_dtype in (BF16, F32):
        results = ops.load(at.cache, n, dtype=out_dtype, **where)
        out = [torch.full((b, n, hkv, d), 9.0, dtype=out_dtype, device="cuda").transpose(1, 2) for _ in range(2)]
        ops.load(at.cache, n, out=out, **where)
        for got, again, expected in zip(results, out, kept):
            assert got.dtype == out_dtype and torch.equal(got.cpu().double(), expected) and torch.equal(got, again)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_every_number_of_a_type(ops, bits, dtype):
    """All bf16 bit patterns (f32: as many of its own), a block to each so that the scale is its own, or 32 to a block."""
    patterns = (torch.arange(65536) << 16) + (0 if dtype is BF16 else torch.arange(65536) * 40503 % 65536)
    x = torch.where(patterns >= 2 ** 31, patterns - 2 ** 32, patterns).int().view(F32)
    alone = torch.zeros((1, 1, 65536, 32))
    alone[0, 0, torch.arange(65536), torch.arange(65536) % 32] = x
    order = torch.randperm(65536, generator=torch.Generator().manual_seed(1))
    for values in (alone, x[order].view(1, 1, 2048, 32), x.view(1, 1, 2048, 32)):
        values = values.to(dtype)
        n = values.shape[2]
        cache = ops.QuantisedCache.empty(1, 1, n, 32, bits)
        ops.store(cache, values.cuda(), values.cuda())
        code, scale = encode(values, bits)
        assert torch.equal(cache.k.cpu(), packed(code, bits)) and torch.equal(cache.v_scales.cpu(), scale)
        got = ops.load(cache, n, dtype=dtype)[0].cpu().double()
        want = decode(code, scale, 32, bits)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_what_is_not_there_is_not_written(ops):
    """Slots before 0 and past the pages, pages that the cache does not have; they read as zeros, and as page 0."""
    gen = torch.Generator().manual_seed(3)
    cache = ops.QuantisedCache.empty(4, 2, 8, 64, 4)
    table = torch.tensor([[1, 9], [2, -1]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn((2, 2, 20, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    first = torch.tensor([-3, 4], dtype=torch.int32, device="cuda")
    ops.store(cache, k, v, first=first, table=table)
    assert not cache.k[0].any() and not cache.k[3].any() and not cache.k_scales[0].any()
    assert cache.k[1].any() and not cache.k[2, :, :4].any() and cache.k[2, :, 4:].any()
    got, _ = ops.load(cache, 20, first=first, table=table, dtype=F32)
    kept = decode(*encode(k.cpu(), 4), 64, 4)
    want = torch.zeros((2, 2, 20, 64), dtype=torch.float64)
    want[0, :, 3:11], want[1, :, :4] = kept[0, :, 3:11], kept[1, :, :4]  # (page 0 holds zeros)
    assert torch.equal(got.cpu().double(), want)
    # without pages and without tokens
    empty = ops.QuantisedCache.empty(0, 2, 8, 64, 4)
    none = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    ops.store(empty, k, v, table=none)
    assert not ops.load(empty, 20, table=none)[0].any()
    assert ops.load(cache, 0, table=table)[0].shape == (2, 2, 0, 64)
    ops.store(cache, k[:, :, :0], v[:, :, :0], table=table)


# type, bits, b, hq, hkv, nodes, longest, d, page, cap, bias, heads last
TREES = [
    (BF16, 4, 1, 1, 1, 1, 0, 64, 16, 0.0, False, False),
    (F32, 4, 1, 1, 1, 1, 1, 8, 1, 0.0, False, False),
    (BF16, 4, 3, 8, 2, 1, 700, 128, 64, 0.0, False, True),
    (BF16, 8, 3, 8, 2, 1, 700, 128, 64, 0.0, True, False),
    (BF16, 4, 2, 4, 4, 1, 90, 64, 7, 0.0, True, False),
    (BF16, 4, 2, 8, 2, 5, 333, 128, 16, 30.0, False, True),
    (BF16, 4, 2, 8, 2, 48, 1500, 128, 33, 50.0, True, False),
    (BF16, 8, 2, 8, 2, 48, 1500, 128, 33, 50.0, False, True),
    (BF16, 4, 1, 6, 1, 64, 2500, 64, 256, 0.0, False, False),
    (BF16, 8, 1, 4, 2, 9, 500, 256, 64, 0.0, True, True),
    (BF16, 4, 1, 4, 2, 1, 900, 256, 64, 0.0, True, False),
    (BF16, 4, 1, 40, 1, 1, 300, 80, 16, 0.0, False, True),
    (BF16, 8, 1, 4, 4, 1, 1000, 96, 16, 0.0, False, False),
    (BF16, 4, 2, 3, 1, 3, 200, 192, 16, 0.0, False, True),
    (F32, 4, 2, 4, 2, 1, 300, 64, 20, 0.0, True, False),
    (F32, 8, 1, 8, 2, 12, 400, 128, 64, 10.0, False, True),
    (F32, 4, 1, 2, 1, 33, 129, 256, 64, 0.0, False, False),
    (F32, 8, 2, 3, 3, 64, 65, 40, 16, 0.0, True, False),
    (F32, 4, 1, 8, 8, 1, 2000, 128, 64, 0.0, False, False),
    (F32, 4, 1, 8, 1, 16, 1000, 64, 64, 20.0, True, True),
    # work dealt out over many sequences, tables of more pages and biases of more keys than a workgroup looks up at once
    (BF16, 4, 70, 4, 2, 1, 300, 64, 16, 0.0, False, True),
    (F32, 4, 130, 2, 1, 3, 40, 64, 5, 0.0, True, False),
    (BF16, 4, 2, 2, 1, 5, 1500, 128, 1, 0.0, True, True),
    (BF16, 8, 1, 2, 2, 2, 9000, 64, 2, 0.0, False, False),
    (BF16, 4, 1, 2, 2, 1, 9000, 128, 8, 0.0, False, False),
    (BF16, 4, 2, 8, 1, 64, 1700, 128, 7, 0.0, False, True),
    (BF16, 4, 70, 2, 1, 2, 2300, 64, 64, 0.0, False, False),
    (BF16, 4, 3, 8, 2, 8, 1100, 128, 64, 0.0, True, False),
    (F32, 8, 5, 3, 1, 11, 700, 256, 16, 0.0, False, True),
    (BF16, 8, 2, 16, 2, 4, 5000, 128, 256, 0.0, False, False),
    # rows of a key head where the kernels change, pages of a tile and of several, head sizes between those of the kernels
    (BF16, 4, 2, 16, 1, 1, 700, 64, 64, 0.0, False, False),
    (BF16, 4, 2, 17, 1, 1, 700, 64, 128, 0.0, False, False),
    (BF16, 8, 1, 8, 1, 8, 600, 128, 32, 20.0, False, False),
    (BF16, 4, 1, 13, 1, 5, 600, 128, 64, 0.0, True, True),
    (F32, 4, 1, 16, 1, 1, 1500, 128, 64, 0.0, True, False),
    (F32, 8, 1, 3, 1, 6, 1500, 128, 32, 0.0, False, False),
    (BF16, 8, 1, 2, 2, 1, 1200, 136, 64, 0.0, False, True),
    (BF16, 4, 1, 2, 2, 1, 1200, 160, 64, 0.0, False, False),
    (BF16, 4, 1, 2, 1, 20, 300, 200, 64, 0.0, False, False),
    (F32, 4, 1, 2, 2, 1, 1200, 224, 16, 0.0, False, False),
    (F32, 8, 1, 2, 1, 1, 700, 256, 64, 0.0, False, True),
    (BF16, 8, 2, 4, 2, 1, 500, 32, 32, 0.0, False, False),
    (BF16, 4, 2, 4, 2, 1, 500, 32, 64, 0.0, False, True),
    (BF16, 8, 2, 4, 2, 1, 500, 48, 7, 0.0, False, False),
    (BF16, 4, 1, 8, 1, 1, 20000, 128, 64, 0.0, False, False),
    (F32, 8, 1, 4, 1, 2, 9000, 64, 16, 0.0, False, False),
]


@pytest.mark.parametrize("case", TREES, ids=names)
def test_trees(ops, case):
    dtype, bits, b, hq, hkv, nodes, longest, d, page, cap, bias, heads_last = case
    print(names(case), flush=True)
    gen = torch.Generator().manual_seed(nodes + longest)
    at = Pages(ops, gen, bits, b, hkv, d, page, longest + nodes, heads_last)
    lengths = [longest] + [int(torch.randint(0, longest + 1, (1,), generator=gen)) for _ in range(b - 1)]
    k, v = at.fill(gen, [n + nodes for n in lengths], dtype)
    words = [tree_words(gen, nodes) for _ in range(b)]
    q = (torch.randn((b, nodes, hq, d), generator=gen) * 1.5).to(dtype).cuda().transpose(1, 2)
    options = {"cap": cap, "slopes": slopes_of(hq) if bias else None}
    o, lse = ops.tree_attention(q, at.cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table=at.table,
                                visible=torch.tensor([[signed(w) for w in row] for row in words], device="cuda"), **options)
    for s, n in enumerate(lengths):
        total = n + nodes
        sees = torch.tensor([[bool(w >> u & 1) for u in range(nodes)] for w in words[s]])
        hidden = torch.cat([torch.zeros((nodes, n), dtype=torch.bool), ~sees], 1)[None]
        depth = sees.sum(1) - 1
        position = torch.cat([torch.arange(n), n + depth])
        distance = (n + depth[:, None] - position[None]).abs().double().expand(1, hq, nodes, total)
        want = Attention(q[s:s + 1], k[s:s + 1, :, :total], v[s:s + 1, :, :total], hidden=hidden, distance=distance, **options)
        within(o[s:s + 1], want.o, want.o_bound, f"o of sequence {s}")
        within(lse[s:s + 1], want.lse, want.lse_bound, f"lse of sequence {s}")


@pytest.mark.parametrize("dtype, nodes", [(BF16, 1), (BF16, 40), (F32, 1)])
@pytest.mark.parametrize("bits", [4, 8])
def test_against_the_cache_read_back(ops, bits, dtype, nodes):
    """The same attention over what load gives: rounding of the same products in another order."""
    from i_amd import attention

    gen = torch.Generator().manual_seed(bits)
    b, hq, hkv, n, d = 2, 8, 2, 500, 128
    at = Pages(ops, gen, bits, b, hkv, d, 16, n + nodes)
    k, v = at.fill(gen, [n + nodes] * b, dtype)
    q = torch.randn((b, hq, nodes, d), generator=gen).to(dtype).cuda()
    lengths = torch.tensor([n, 123], dtype=torch.int32, device="cuda")
    o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table)
    k, v = ops.load(at.cache, n + nodes, table=at.table, dtype=dtype)
    o2, lse2 = attention.tree_attention(q, k, v, lengths)
    # (weights and outputs are rounded on either side: two roundings of the type each)
    unit = 2.0 ** -8 if dtype is BF16 else 2.0 ** -20
    assert float((o.float() - o2.float()).abs().max()) <= 4 * unit * float(v.float().abs().max())
    assert float((lse - lse2).abs().max()) <= 2.0 ** -16


def test_slots_that_nobody_sees_may_hold_anything(ops):
    """No numbers past the end, and in a slot of a node that no node sees; a seen one that is no number shows."""
    gen = torch.Generator().manual_seed(5)
    for bits, dtype, hq in ((4, BF16, 4), (8, BF16, 64), (4, F32, 2)):
        at = Pages(ops, gen, bits, 1, 1, 64, 16, 43)
        k, v = at.fill(gen, [43], dtype)
        page, slot = at.slot(0, 41)
        for scales in (at.cache.k_scales, at.cache.v_scales):
            scales[page, :, slot] = 255
        q = torch.randn((1, hq, 3, 64), generator=gen).to(dtype).cuda()
        words = torch.tensor([[1, 0, 5]], device="cuda")  # (node 1 sees nothing, and nobody sees it)
        lengths = torch.tensor([40], dtype=torch.int32, device="cuda")
        o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table, visible=words)
        hidden = torch.zeros((1, 3, 43), dtype=torch.bool)
        hidden[0, :, 41], hidden[0, 0, 42], hidden[0, 1, 40:] = True, True, True
        want = Attention(q, k, v, hidden=hidden)
        within(o, want.o, want.o_bound, "o")
        # the whole tree sees nothing of a cache without keys
        o, lse = ops.tree_attention(q, at.cache, torch.zeros_like(lengths), table=at.table, visible=torch.zeros_like(words))
        assert not o.any() and bool((lse == -math.inf).all())
        page, slot = at.slot(0, 7)
        at.cache.v_scales[page, :, slot] = 255
        o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table, visible=words)
        assert bool(o.isnan().all()) and bool(lse.isfinite().all())
        at.cache.k_scales[page, :, slot] = 255
        o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table, visible=words)
        assert bool(o.isnan().all()) and bool(lse.isnan().all())


def test_without_a_table_and_lengths_past_the_end(ops):
    gen = torch.Generator().manual_seed(10)
    b, hq, hkv, n, d = 3, 4, 4, 200, 64
    k, v = (torch.randn((b, hkv, n, d), generator=gen).to(BF16).cuda() for _ in range(2))
    cache = ops.QuantisedCache.empty(b, hkv, n, d, 8)
    ops.store(cache, k, v)
    k, v = ops.load(cache, n)
    q = torch.randn((b, hq, 1, d), generator=gen).to(BF16).cuda()
    o, lse = ops.tree_attention(q, cache, torch.tensor([199, 5000, -50], dtype=torch.int32, device="cuda"))
    hidden = torch.arange(n)[None, None, :] >= torch.tensor([200, 200, 1])[:, None, None]
    want = Attention(q, k, v, hidden=hidden)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")


def test_positions_of_a_cut_cache(ops):
    b, hq, hkv, d, n = 2, 4, 2, 64, 77
    gen = torch.Generator().manual_seed(8)
    at = Pages(ops, gen, 4, b, hkv, d, 16, n + 1)
    k, v = at.fill(gen, [n + 1] * b, F32)
    positions = torch.randint(0, 900, (b, hkv, n + 1), generator=gen, dtype=torch.int32).sort(-1).values
    q = torch.randn((b, hq, 1, d), generator=gen).cuda()
    start = torch.tensor([900, 950], dtype=torch.int32, device="cuda")
    slopes = slopes_of(hq)
    o, _ = ops.tree_attention(q, at.cache, torch.full((b,), n, dtype=torch.int32, device="cuda"), table=at.table, slopes=slopes, start=start,
                              positions=positions.cuda(), max_length=n + 1)
    of = positions.repeat_interleave(hq // hkv, 1).clone()
    of[:, :, n] = start.cpu()[:, None]
    distance = (start.cpu().view(b, 1, 1, 1) - of[:, :, None, :]).abs().double()
    want = Attention(q, k, v, slopes=slopes, distance=distance, hidden=torch.zeros((b, 1, n + 1), dtype=torch.bool))
    within(o, want.o, want.o_bound, "o")


def test_a_step_in_a_graph(ops):
    """Rotation, writing and attention of one token, captured together and replayed with eager work between."""
    from i_amd import rotary

    gen = torch.Generator().manual_seed(12)
    b, hq, hkv, d, page, per = 3, 8, 2, 64, 16, 20
    f = rotary.frequencies(d // 2)
    weight = (1 + 0.1 * torch.randn(d, generator=gen)).to(BF16).cuda()
    caches = [ops.QuantisedCache.empty(b * per, hkv, page, d, 4) for _ in range(2)]
    table = torch.randperm(b * per, generator=gen).int().view(b, per).cuda()
    x = torch.empty((b, 1, hq + 2 * hkv, d), dtype=BF16, device="cuda")
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step(cache):
        q, k, v = (part.transpose(1, 2) for part in x.split([hq, hkv, hkv], 2))
        q, k = rotary.rotate(q, k, lengths[:, None], f, q_weight=weight, k_weight=weight)
        ops.store(cache, k, v, first=lengths, table=table)
        return ops.tree_attention(q, cache, lengths, table=table)

    step(caches[0])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kept = step(caches[0])
    for n in (0, 1, 2, 100, 319, 5):
        x.copy_(torch.randn(x.shape, generator=gen))
        lengths.copy_(torch.tensor([n, n // 2, n // 3]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1])
        for got, expected in zip(kept, want):
            assert torch.equal(got, expected), n
        for name in ("k", "k_scales", "v", "v_scales"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), n


def test_refusals(ops):
    cache = ops.QuantisedCache.empty(2, 2, 16, 64, 4)
    k = torch.zeros((2, 2, 4, 64), dtype=BF16, device="cuda")
    q = torch.zeros((2, 4, 1, 64), dtype=BF16, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.store(cache, k[..., :32], k[..., :32]), lambda: ops.store(cache, k, k[:, :, :2]), lambda: ops.store(cache, k[:, :1], k[:, :1]),
                 lambda: ops.store(cache, k, k, first=lengths[:1]), lambda: ops.store(cache, k, k, table=table[:1]), lambda: ops.load(cache, -1),
                 lambda: ops.load(cache, 4, counts=lengths[:1], table=table), lambda: ops.store(cache, k, k, table=table[:, :0]),
                 lambda: ops.tree_attention(q[..., :32], cache, lengths),
                 lambda: ops.tree_attention(q, cache, lengths[:1]), lambda: ops.tree_attention(q, cache, lengths, slopes=torch.zeros(3, device="cuda")),
                 lambda: ops.load(cache, 4, out=(k, k[:, :, :2])), lambda: ops.load(cache, 1, out=(k[:, :, :1].expand(2, 2, 1, 64), k[:1, :, :1].expand(2, 2, 1, 64))),
                 lambda: ops.QuantisedCache(cache.k, cache.k_scales[:1], cache.v, cache.v_scales, 64, 4),
                 lambda: ops.QuantisedCache(cache.k[:1].expand(2, 2, 16, 32), cache.k_scales, cache.v, cache.v_scales, 64, 4),
                 lambda: ops.QuantisedCache.empty(2, 2, 16, 60, 4)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.store(cache, k.half(), k.half()), lambda: ops.store(cache, k, k.float()), lambda: ops.load(cache, 4, dtype=torch.float16),
                 lambda: ops.tree_attention(q, cache, lengths.long()), lambda: ops.store(cache, k, k, table=table.long()),
                 lambda: ops.QuantisedCache(cache.k.char(), cache.k_scales, cache.v, cache.v_scales, 64, 4)):
        with pytest.raises(TypeError):
            call()
    # nodes that do not fit the pages, no page for a sequence, strides of codes that are not multiples of 16
    for call in (lambda: ops.tree_attention(torch.zeros((2, 4, 17, 64), dtype=BF16, device="cuda"), cache, lengths),
                 lambda: ops.tree_attention(q.repeat(2, 1, 1, 1), cache, torch.zeros(4, dtype=torch.int32, device="cuda")),
                 lambda: ops.tree_attention(q[:, :3], cache, lengths),
                 lambda: ops.store(ops.QuantisedCache(*(torch.zeros((2, 2, 16, w + 1), dtype=torch.uint8, device="cuda")[..., :w] for w in (32, 2, 32, 2)), 64, 4), k, k)):
        with pytest.raises(RuntimeError):
            call()


def test_long_cache_of_few_heads_again_and_again(ops):
    """Many runs a head and their join; the same call gives the same bits."""
    gen = torch.Generator().manual_seed(14)
    for dtype, bits, d, nodes in ((BF16, 4, 64, 1), (BF16, 8, 256, 5), (F32, 4, 128, 1), (F32, 8, 256, 20)):
        at = Pages(ops, gen, bits, 1, 1, d, 64, 6000 + nodes)
        k, v = at.fill(gen, [6000 + nodes], dtype)
        q = torch.randn((1, 2, nodes, d), generator=gen).to(dtype).cuda()
        lengths = torch.tensor([6000], dtype=torch.int32, device="cuda")
        o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table)
        hidden = torch.ones((nodes, nodes), dtype=torch.bool).triu(1)
        want = Attention(q, k, v, hidden=torch.cat([torch.zeros((nodes, 6000), dtype=torch.bool), hidden], 1)[None])
        within(o, want.o, want.o_bound, "o")
        within(lse, want.lse, want.lse_bound, "lse")
        # one word a node for all sequences, outputs given, in another layout
        words = torch.tensor([(2 << t) - 1 for t in range(nodes)], device="cuda")
        out = torch.empty((1, nodes, 2, d), dtype=dtype, device="cuda").transpose(1, 2)
        again = ops.tree_attention(q, at.cache, lengths, table=at.table, visible=words, out=out, lse=torch.empty_like(lse))
        assert again[0] is out and torch.equal(out, o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype, bits, d", [(BF16, 4, 64), (F32, 8, 104)])
def test_many_rows_of_one_head_in_many_runs(ops, dtype, bits, d):
    """More rows than a workgroup a row joins, in more runs than are joined at once."""
    gen = torch.Generator().manual_seed(20)
    hq, nodes, length = 64, 40, 3000
    at = Pages(ops, gen, bits, 1, 1, d, 64, length + nodes)
    k, v = at.fill(gen, [length + nodes], dtype)
    q = torch.randn((1, hq, nodes, d), generator=gen).to(dtype).cuda()
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    words = torch.tensor([(2 << t) - 1 for t in range(nodes)], device="cuda")
    o, lse = ops.tree_attention(q, at.cache, lengths, table=at.table, visible=words)
    hidden = torch.cat([torch.zeros((nodes, length), dtype=torch.bool), torch.ones((nodes, nodes), dtype=torch.bool).triu(1)], 1)[None]
    want = Attention(q, k, v, hidden=hidden)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")


def test_pages_that_there_are_not_and_pages_twice(ops):
    """An entry outside the cache is page 0; sequences may share pages."""
    gen = torch.Generator().manual_seed(15)
    b, hq, hkv, d, page = 2, 4, 2, 64, 16
    cache = ops.QuantisedCache.empty(5, hkv, page, d, 4)
    k, v = (torch.randn((5, hkv, page, d), generator=gen).to(BF16).cuda() for _ in range(2))
    ops.store(cache, k, v)
    k, v = ops.load(cache, page)
    q = torch.randn((b, hq, 1, d), generator=gen).to(BF16).cuda()
    table = torch.tensor([[3, 2 ** 31 - 1, 1], [3, -7, 4]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([47, 40], dtype=torch.int32, device="cuda")
    o, lse = ops.tree_attention(q, cache, lengths, table=table)
    listed = torch.tensor([[3, 0, 1], [3, 0, 4]])
    dense = [x.cpu()[listed].transpose(1, 2).reshape(b, hkv, 48, d) for x in (k, v)]
    want = Attention(q, *dense, hidden=torch.arange(48)[None, None, :] > torch.tensor([47, 40])[:, None, None])
    within(o, want.o, want.o_bound, "o")
    got = ops.load(cache, 48, table=table)
    assert torch.equal(got[0].cpu(), dense[0]) and torch.equal(got[1].cpu(), dense[1])


def test_pages_that_are_far_apart(ops):
    """Offsets past 32 bits in codes and scales, of pages and of heads."""
    gen = torch.Generator().manual_seed(16)
    memory = torch.zeros(11 * 2 ** 30, dtype=torch.uint8, device="cuda")
    for bits in (4, 8):
        row = 64 * bits // 8
        for apart in ("pages", "heads"):
            far, near = 5 * 2 ** 29, 2 ** 20
            strides = (far, near) if apart == "pages" else (near, far)
            place = lambda at, width, step: memory[at:].as_strided((4, 2, 64, width), (*strides, step, 1))  # noqa: E731
            far_cache = ops.QuantisedCache(place(0, row, row), place(2 ** 16, 2, 2), place(2 ** 17, row, row), place(2 ** 18, 2, 2), 64, bits)
            near_cache = ops.QuantisedCache.empty(4, 2, 64, 64, bits)
            k, v = (torch.randn((1, 2, 250, 64), generator=gen).to(BF16).cuda() for _ in range(2))
            table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device="cuda")
            q = torch.randn((1, 4, 1, 64), generator=gen).to(BF16).cuda()
            many = torch.randn((1, 4, 12, 64), generator=gen).to(BF16).cuda()
            lengths = torch.tensor([230], dtype=torch.int32, device="cuda")
            results = []
            for cache in (far_cache, near_cache):
                ops.store(cache, k, v, table=table)
                results.append((*ops.load(cache, 250, table=table), *ops.tree_attention(q, cache, lengths, table=table), *ops.tree_attention(many, cache, lengths, table=table)))
            for one, two in zip(*results):
                assert torch.equal(one, two)


def test_copies_of_a_cache_have_memory_of_their_own(ops):
    """A copied and a pickled cache are written to without touching the first."""
    import copy
    import pickle

    gen = torch.Generator().manual_seed(18)
    cache = ops.QuantisedCache.empty(2, 2, 16, 64, 8)
    k, v = (torch.randn((2, 2, 16, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    ops.store(cache, k, v)
    kept = [x.clone() for x in ops.load(cache, 16)]
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert other.k.data_ptr() != cache.k.data_ptr()
        for x, y in zip(ops.load(other, 16), kept):
            assert torch.equal(x, y)
        ops.store(other, v, k)
        for x, y, z in zip(ops.load(cache, 16), kept, ops.load(other, 16)):
            assert torch.equal(x, y) and not torch.equal(x, z)


def test_more_rows_than_a_launch_is_wide(ops):
    """2^28 rows of 16 threads, all but four a sequence without a slot: the last workgroups have theirs written."""
    gen = torch.Generator().manual_seed(19)
    b, n = 256, 2 ** 20
    k, v = (torch.randn((1, 1, 1, 128), generator=gen).to(BF16).cuda() for _ in range(2))
    cache = ops.QuantisedCache.empty(b, 1, 4, 128, 4)
    first = torch.full((b,), 4 - n, dtype=torch.int32, device="cuda")
    ops.store(cache, k.expand(b, 1, n, 128), v.expand(b, 1, n, 128), first=first)
    near = ops.QuantisedCache.empty(1, 1, 1, 128, 4)
    ops.store(near, k, v)
    for x, y in zip(ops.load(cache, 4), ops.load(near, 1)):
        assert y.any() and torch.equal(x, y.expand_as(x))


def test_another_stream(ops):
    gen = torch.Generator().manual_seed(17)
    at = [Pages(ops, gen, 4, 2, 2, 64, 16, 3001) for _ in range(2)]
    for pages in at:
        pages.fill(gen, [3001, 3001], BF16)
    q = torch.randn((2, 8, 1, 64), generator=gen).to(BF16).cuda()
    lengths = torch.tensor([3000, 1700], dtype=torch.int32, device="cuda")
    want = [ops.tree_attention(q, pages.cache, lengths, table=pages.table) for pages in at]
    torch.cuda.synchronize()
    got = []
    for pages, stream in zip(at, [torch.cuda.Stream() for _ in at]):
        with torch.cuda.stream(stream):
            for _ in range(4):
                results = ops.tree_attention(q, pages.cache, lengths, table=pages.table)
            got.append(results)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("bits, dtype", [(4, BF16), (8, BF16), (4, F32)])
def test_a_prompt_and_its_tokens(ops, bits, dtype):
    """Rotation, cache and attention as a model uses them: a prompt written, then tokens one by one and a tree, against attention over
    everything with the keys and values that the cache holds."""
    from i_amd import rotary

    gen = torch.Generator().manual_seed(bits)
    b, hq, hkv, n, steps, d, page = 2, 8, 2, 150, 5, 64, 16
    x = torch.randn((b, n + steps, hq + 2 * hkv, d), generator=gen).to(dtype).cuda()
    f = rotary.frequencies(d // 2)
    weight = (1 + 0.1 * torch.randn(d, generator=gen)).to(dtype).cuda()
    q, k, v = (part.transpose(1, 2) for part in x.split([hq, hkv, hkv], 2))
    q, k = rotary.rotate(q, k, torch.arange(n + steps, dtype=torch.int32, device="cuda"), f, q_weight=weight, k_weight=weight)
    per = -(-(n + steps) // page)
    cache = ops.QuantisedCache.empty(b * per, hkv, page, d, bits)
    table = torch.randperm(b * per, generator=gen).int().view(b, per).cuda()
    counts = torch.tensor([n, n - 37], dtype=torch.int32, device="cuda")  # (a padded batch)
    ops.store(cache, k[:, :, :n], v[:, :, :n], counts=counts, table=table)
    kept = [decode(*encode(y.cpu(), bits), d, bits).to(dtype) for y in (k, v)]
    lengths, outputs = counts.clone(), []
    at = torch.arange(steps, device="cuda") + counts[:, None]
    for t in range(steps):
        pick = at[:, None, t, None, None].expand(-1, hkv, 1, d)
        ops.store(cache, k.gather(2, pick), v.gather(2, pick), first=lengths, table=table)
        outputs.append(ops.tree_attention(q.gather(2, at[:, None, t, None, None].expand(-1, hq, 1, d)), cache, lengths, table=table)[0])
        lengths += 1
    tree, _ = ops.tree_attention(q.gather(2, at[:, None, :, None].expand(-1, hq, steps, d)), cache, counts, table=table)
    for s in range(b):
        first = int(counts[s])
        want = Attention(q[s:s + 1, :, first:first + steps], kept[0][s:s + 1, :, :first + steps], kept[1][s:s + 1, :, :first + steps], causal=True)
        within(torch.cat(outputs, 2)[s:s + 1], want.o, want.o_bound, "tokens")
        within(tree[s:s + 1], want.o, want.o_bound, "tree")
