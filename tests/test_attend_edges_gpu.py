"""Attention with masks where a call holds more than it uses: unseen keys in between, queries that see nothing, bounds at the ends of their type."""
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


def tensors(seed, dtype, b, hq, hkv, nq, nk, d):
    gen = torch.Generator().manual_seed(seed)

    def make(h, n, spread):
        return (torch.randn((b, n, h, d), generator=gen) * spread).to(dtype).cuda().transpose(1, 2)

    return make(hq, nq, 1.5), make(hkv, nk, 1.0), make(hkv, nk, 1.0), make(hq, nq, 1.0)


def everything(ops, want, q, k, v, grad, **options):
    """Forward, gradients and key weights against the oracle; returns o, lse and dq."""
    o, lse = ops.attention(q, k, v, **options)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")
    return o, lse


def gradients(ops, want, grads, q, k, v, grad, o, lse, **options):
    """`grads`: what the oracle says of the gradients."""
    got = ops.attention_backward(grad, q, k, v, o, lse, **options)
    for x, ref, bound, name in zip(got, *grads, ("dq", "dk", "dv")):
        within(x, ref, bound, name)
    weights, bound = want.weights()
    within(ops.key_weights(q, k, lse, **options), weights, bound, "weights")
    return got


def intervals(b, n, *spans):
    """first and last of n queries: those of a span see it, the others nothing; each sequence's spans a little further on."""
    first, last = torch.zeros((b, n), dtype=torch.int32), torch.zeros((b, n), dtype=torch.int32)
    for s in range(b):
        for lo, hi in spans:
            lo, hi = min(lo + s, n), min(hi + 2 * s, n)
            first[s, lo:hi], last[s, lo:hi] = lo, hi
    return {"first": first.cuda(), "last": last.cuda()}


# heads of the three ways that queries are dealt out, by their number of 128-query tiles: below 64, 64 .. 256, more
HEADS = [(1, 4, 2), (2, 40, 10), (3, 64, 16)]
SHAPES = [(BF16, 64), (BF16, 80), (BF16, 128), (BF16, 256), (F32, 64), (F32, 128), (F32, 256)]


# ---------------------------------------------------------------- keys that nobody sees, between keys that are seen
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dtype,d", SHAPES, ids=str)
def test_a_gap_between_documents_may_hold_anything(ops, heads, dtype, d):
    b, hq, hkv = heads
    n = 200
    print(dtype, d, heads, flush=True)
    q, k, v, grad = tensors(d + hq, dtype, b, hq, hkv, n, n, d)
    options = intervals(b, n, (0, 40), (64, 130), (141, 194))
    want = Attention(q, k, v, **options)
    grads = want.gradients(grad)
    dead = (want.hidden[:, 0].all(1))[:, None, :, None].cuda()
    k = torch.where(dead, math.nan, k)
    v = torch.where(dead, math.inf, v)
    o, lse = everything(ops, want, q, k, v, grad, **options)
    gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_gaps_of_one_key(ops, dtype, causal):
    """Neighbouring queries whose intervals leave single keys out, with a cap and a bias."""
    b, hq, hkv, nq, nk, d = 1, 8, 2, 50, 173, 64
    q, k, v, grad = tensors(3, dtype, b, hq, hkv, nq, nk, d)
    first = (torch.arange(nq, dtype=torch.int32) * 3 + nk - 3 * nq).expand(b, nq).contiguous().cuda()
    options = dict(first=first, last=first + 2, causal=causal, cap=9.0, slopes=torch.linspace(0.1, 0.9, hq, device="cuda"))
    want = Attention(q, k, v, **options)
    grads = want.gradients(grad)
    dead = (want.hidden[:, 0].all(1))[:, None, :, None].cuda()
    assert int(dead.sum()) >= nk - 2 * nq
    for poison in (math.nan, -math.inf):
        k, v = torch.where(dead, poison, k), torch.where(dead, poison, v)
        o, lse = everything(ops, want, q, k, v, grad, **options)
        gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


@pytest.mark.parametrize("dtype,hq,hkv,nodes,length,d", [(BF16, 4, 2, 5, 90, 64), (BF16, 8, 2, 5, 1500, 128), (BF16, 8, 2, 48, 300, 128), (BF16, 8, 1, 20, 900, 256),
                                                        (F32, 4, 2, 5, 90, 64), (F32, 4, 2, 7, 700, 128), (F32, 2, 1, 40, 130, 64), (F32, 2, 1, 9, 200, 256)])
def test_a_slot_that_no_node_sees_may_hold_anything(ops, dtype, hq, hkv, nodes, length, d):
    """Drafted tokens given up: their slots are in no node's word, the last one's too."""
    q, k, v, _ = tensors(nodes + d, dtype, 2, hq, hkv, nodes, length + nodes, d)
    k, v = k.contiguous(), v.contiguous()
    gone = {1, 3, nodes - 1}
    words = [sum(1 << u for u in range(t + 1) if u not in gone) for t in range(nodes)]
    sees = torch.tensor([[bool(w >> u & 1) for u in range(nodes)] for w in words])
    hidden = torch.cat([torch.zeros((nodes, length), dtype=torch.bool), ~sees], 1)[None].expand(2, -1, -1)
    want = Attention(q, k, v, hidden=hidden)
    for u in gone:
        k[:, :, length + u], v[:, :, length + u] = math.nan, math.inf
    weights = torch.zeros((2, hkv, length + nodes), device="cuda")
    o, lse = ops.tree_attention(q, k, v, torch.full((2,), length, dtype=torch.int32, device="cuda"), visible=torch.tensor(words, device="cuda"), weights=weights)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")
    within(weights, *want.weights(), "weights")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("hq", [2, 80])
def test_a_gap_after_any_query(ops, dtype, hq):
    """Two intervals with a gap, the first `split` queries in the one or the other of them, on either side of every tile's edge."""
    b, hkv, nq, nk, d = 2, 2, 130, 90, 64
    for split in (1, 7, 14, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129):
        q, k, v, grad = tensors(split, dtype, b, hq, hkv, nq, nk, d)
        first, last = (torch.zeros((b, nq), dtype=torch.int32) for _ in range(2))
        for s, (one, other) in enumerate((((3, 37), (41, 80)), ((41, 80), (3, 37)))):
            first[s, :split], last[s, :split] = one
            first[s, split:], last[s, split:] = other
        options = {"first": first.cuda(), "last": last.cuda()}
        want = Attention(q, k, v, **options)
        grads = want.gradients(grad)
        for x in (k, v):
            x[:, :, :3], x[:, :, 37:41], x[:, :, 80:] = math.nan, math.inf, math.nan
        o, lse = everything(ops, want, q, k, v, grad, **options)
        gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_gaps_between_intervals_in_any_order(ops, dtype, heads):
    """Short intervals anywhere, some queries that see nothing between them: most keys are seen by nobody, or by few."""
    b, hq, hkv = heads
    nq, nk, d = 150, 700, 64
    gen = torch.Generator().manual_seed(hq)
    for empty in (0.0, 0.3, 0.9):
        q, k, v, grad = tensors(hq, dtype, b, hq, hkv, nq, nk, d)
        first = torch.randint(0, nk, (b, nq), generator=gen, dtype=torch.int32)
        last = first + torch.randint(1, 9, (b, nq), generator=gen, dtype=torch.int32)
        last = torch.where(torch.rand((b, nq), generator=gen) < empty, first, last)
        options = {"first": first.cuda(), "last": last.cuda()}
        want = Attention(q, k, v, **options)
        grads = want.gradients(grad)
        dead = want.hidden[:, 0].all(1)[:, None, :, None].cuda()
        k, v = torch.where(dead, math.nan, k), torch.where(dead, math.inf, v)
        o, lse = everything(ops, want, q, k, v, grad, **options)
        gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


# ---------------------------------------------------------------- bounds at the ends of their type
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_bounds_at_the_ends_of_their_type(ops, dtype, heads, causal):
    """A query whose last is the lowest int32 (or whose first is the highest) sees nothing, whatever its other bound is."""
    b, hq, hkv = heads
    nq, nk, d = 150, 130, 64
    q, k, v, grad = tensors(7 + hq, dtype, b, hq, hkv, nq, nk, d)
    gen = torch.Generator().manual_seed(hq)
    first = torch.randint(-3, 60, (b, nq), generator=gen, dtype=torch.int32)
    last = first + torch.randint(1, 90, (b, nq), generator=gen, dtype=torch.int32)
    low, high = -2 ** 31, 2 ** 31 - 1
    last[:, 3::7], last[:, 4::11], first[:, 5::13], last[:, 5::26] = low, low + 40, high, low
    first[:, 6::17], last[:, 6::17] = low, high  # everything
    options = {"first": first.cuda(), "last": last.cuda(), "causal": causal}
    want = Attention(q, k, v, **options)
    grads = want.gradients(grad)
    o, lse = everything(ops, want, q, k, v, grad, **options)
    gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


# ---------------------------------------------------------------- queries that see nothing
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dtype,d", SHAPES, ids=str)
def test_a_query_that_sees_nothing_may_hold_anything(ops, heads, dtype, d):
    """Padded queries: no number in q, in the gradient of o, or in both; they take part in no gradient and in no weight."""
    b, hq, hkv = heads
    n = 170
    print(dtype, d, heads, flush=True)
    q, k, v, grad = tensors(d + hq + 1, dtype, b, hq, hkv, n, n, d)
    options = dict(intervals(b, n, (0, 40), (64, 130), (141, 160)), cap=12.0)
    want = Attention(q, k, v, **options)
    grads = want.gradients(grad)
    blind = want.hidden[:, 0].all(2)[:, None, :, None].cuda()
    q, grad = torch.where(blind, math.nan, q), torch.where(blind, math.inf, grad)
    o, lse = everything(ops, want, q, k, v, grad, **options)
    got = gradients(ops, want, grads, q, k, v, grad, o, lse, **options)
    assert bool((got[0][blind.expand_as(got[0])] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("hq", [4, 80])
def test_causal_queries_ahead_of_the_keys_may_hold_anything(ops, dtype, hq):
    """More queries than keys: the first ones see nothing, without a bound that is given."""
    b, hkv, nq, nk, d = 2, 2, 210, 133, 64
    q, k, v, grad = tensors(hq, dtype, b, hq, hkv, nq, nk, d)
    options = {"causal": True, "slopes": torch.linspace(0.05, 0.4, hq, device="cuda")}
    want = Attention(q, k, v, **options)
    grads = want.gradients(grad)
    q[:, :, :nq - nk], grad[:, :, :nq - nk] = math.inf, math.nan
    o, lse = everything(ops, want, q, k, v, grad, **options)
    gradients(ops, want, grads, q, k, v, grad, o, lse, **options)


# ---------------------------------------------------------------- more key tiles and queries than are planned at once
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("nq,nk", [(20, 40000), (20000, 50)])
@pytest.mark.parametrize("causal", [False, True])
def test_long_sides(ops, dtype, nq, nk, causal):
    b, hq, hkv, d = 2, 2, 1, 64
    q, k, v, grad = tensors(nq, dtype, b, hq, hkv, nq, nk, d)
    gen = torch.Generator().manual_seed(nk)
    first = torch.randint(0, nk, (b, nq), generator=gen, dtype=torch.int32)
    for options in ({}, {"first": first.cuda(), "last": (first + nk // 3).cuda()}):
        options = dict(options, causal=causal)
        want = Attention(q, k, v, **options)
        o, lse = everything(ops, want, q, k, v, grad, **options)
        gradients(ops, want, want.gradients(grad), q, k, v, grad, o, lse, **options)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_a_long_window(ops, dtype):
    """Both sides long, a window: parts of it are what the same window gives on a part of the tokens."""
    n, width, hq, hkv, d = 33500, 40, 2, 1, 64
    q, k, v, grad = tensors(n, dtype, 1, hq, hkv, n, n, d)
    options = {"causal": True, "first": ops.window_bounds(1, n, n, width, "cuda")}
    o, lse = ops.attention(q, k, v, **options)
    got = ops.attention_backward(grad, q, k, v, o, lse, **options)
    weights = ops.key_weights(q, k, lse, **options)
    for at in (0, 16384 - 100, 32768 - 100, n - 240):
        lo, hi = max(at - width, 0), min(at + 240, n)
        here, inside = slice(lo, hi), slice(at - lo, at - lo + 200)
        part = [x[:, :, here] for x in (q, k, v)]
        want = Attention(*part, causal=True, first=ops.window_bounds(1, hi - lo, hi - lo, width, "cuda"))
        refs, bounds = want.gradients(grad[:, :, here])
        whole = slice(at, at + 200)
        within(o[:, :, whole], want.o[:, :, inside], want.o_bound[:, :, inside], f"o at {at}")
        for x, ref, bound, name in zip(got, refs, bounds, ("dq", "dk", "dv")):
            within(x[:, :, whole], ref[:, :, inside], bound[:, :, inside], f"{name} at {at}")
        within(weights[:, :, whole], *(x[:, :, inside] for x in want.weights()), f"weights at {at}")


# ---------------------------------------------------------------- which nodes' weights count
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("length", [37, 3000])
@pytest.mark.parametrize("nodes", [1, 5, 64])
def test_no_node_counts(ops, dtype, length, nodes):
    """No drafted token was taken over: the weights stay as they are, in a new tensor or in their own, for short caches and long ones."""
    print(dtype, length, nodes, flush=True)
    q, k, v, _ = tensors(nodes + length, dtype, 2, 4, 2, nodes, length + nodes, 64)
    k, v = k.contiguous(), v.contiguous()
    weights = torch.rand((2, 2, length + nodes), device="cuda")
    lengths = torch.full((2,), length, dtype=torch.int32, device="cuda")
    before, out = weights.clone(), torch.full_like(weights, math.nan)
    o, _ = ops.tree_attention(q, k, v, lengths, weights=weights, weights_out=out, counted=0)
    assert torch.equal(out, before) and torch.equal(weights, before)
    ops.tree_attention(q, k, v, lengths, weights=weights, counted=0)
    assert torch.equal(weights, before)
    want = Attention(q, k, v, causal=True)
    within(o, want.o, want.o_bound, "o")


def test_all_64_nodes_count(ops):
    """A mask of all nodes, as (1 << accepted) - 1 makes it, whatever their number; one past them is refused."""
    nodes, length = 64, 90
    q, k, v, _ = tensors(5, BF16, 1, 4, 2, nodes, length + nodes, 64)
    k, v = k.contiguous(), v.contiguous()
    lengths = torch.full((1,), length, dtype=torch.int32, device="cuda")
    want, bound = Attention(q, k, v, causal=True).weights()
    for counted in ((1 << 64) - 1, -1):
        weights = torch.zeros((1, 2, length + nodes), device="cuda")
        ops.tree_attention(q, k, v, lengths, weights=weights, counted=counted)
        within(weights, want, bound, "weights")
    for counted in (1 << 64, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="counted"):
            ops.tree_attention(q, k, v, lengths, weights=weights, counted=counted)


# ---------------------------------------------------------------- caps far below the scores
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("scale,cap", [(1.0, 1e-7), (1e6, 1.0), (-3.0, 1e-12), (1e-3, 1e-20), (0.125, 1e-30)])
def test_caps_far_below_the_scores(ops, dtype, scale, cap):
    """Scores at plus or minus the cap, and 0 where q or k are: tanh's polynomial has no finite coefficients there."""
    b, hq, hkv, n, d = 1, 4, 2, 70, 64
    q, k, v, grad = tensors(2, dtype, b, hq, hkv, n, n, d)
    q[:, :, 5], k[:, :, 7], k[:, :, 20:30] = 0.0, 0.0, 0.0
    options = {"scale": scale, "cap": cap, "causal": True}
    want = Attention(q, k, v, **options)
    o, lse = ops.attention(q, k, v, **options)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")
    within(ops.key_weights(q, k, lse, **options), *want.weights(), "weights")
    assert all(bool(x.isfinite().all()) for x in ops.attention_backward(grad, q, k, v, o, lse, **options))
    lengths = torch.full((1,), n - 1, dtype=torch.int32, device="cuda")
    o, _ = ops.tree_attention(q[:, :, 5:6].contiguous(), k.contiguous(), v.contiguous(), lengths, scale=scale, cap=cap)
    want = Attention(q[:, :, 5:6], k, v, scale=scale, cap=cap)
    within(o, want.o, want.o_bound, "o of a token")
