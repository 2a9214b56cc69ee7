"""Norms and rotary positions of queries and keys, forward and backward, against float64 on the CPU."""
import pytest
import torch

from attend_oracle import within
from rotary_oracle import Rotation, turned

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import rotary

    return rotary


def names(case):
    return "-".join(str(x).replace("torch.", "") for x in case)


# type, b, hq, hkv, n, d, pairs, axes, interleaved, norms (q, k; weights in f32: "w"), layout, far
CASES = [
    (BF16, 1, 1, 1, 1, 8, 4, 1, False, "qk", "dense", 0),
    (BF16, 2, 8, 2, 33, 128, 64, 1, False, "qk", "joint", 1000000),
    (BF16, 2, 4, 4, 70, 64, 32, 1, True, "qk", "joint", 7),
    (BF16, 3, 5, 1, 17, 80, 40, 3, False, "q", "dense", 1000),
    (BF16, 1, 3, 3, 129, 72, 36, 3, True, "", "joint", 0),
    (BF16, 2, 6, 2, 40, 256, 128, 1, False, "qkw", "joint", 5),
    (BF16, 1, 2, 1, 5, 256, 13, 2, True, "k", "dense", 5),
    (BF16, 2, 3, 1, 19, 128, 13, 2, False, "qk", "joint", 100),
    (BF16, 2, 3, 1, 19, 96, 24, 1, False, "qk", "joint", 100),
    (BF16, 2, 3, 1, 19, 200, 100, 1, False, "qkw", "joint", 100),
    (BF16, 2, 3, 0, 19, 64, 32, 1, False, "q", "joint", 100),
    (BF16, 2, 3, 1, 21, 128, 0, 0, False, "qk", "joint", 0),
    (BF16, 1, 40, 8, 1000, 128, 64, 1, False, "qk", "joint", 0),
    (F32, 3, 3, 3, 257, 64, 24, 2, False, "qk", "joint", 0),
    (F32, 1, 2, 2, 31, 128, 64, 1, True, "qk", "dense", 2000000000),
    (F32, 2, 4, 1, 9, 56, 7, 2, False, "qk", "joint", 10),
    (F32, 1, 4, 2, 65, 256, 127, 3, True, "q", "joint", 10),
    (F32, 1, 4, 2, 65, 248, 124, 3, False, "qk", "joint", 10),
    (F32, 4, 1, 1, 3, 16, 8, 1, False, "", "dense", 1000000),
    (F32, 1, 1, 1, 64, 32, 1, 1, False, "k", "dense", 3),
    # pairs that are a multiple of 4: whole rows, rows with columns that do not turn, and one more lane than a row has
    (BF16, 2, 6, 2, 37, 40, 20, 2, False, "qk", "joint", 50),
    (BF16, 2, 2, 2, 20, 72, 36, 1, False, "qkw", "dense", 50),
    (F32, 2, 2, 1, 20, 104, 52, 1, False, "qk", "joint", 50),
    (BF16, 1, 2, 1, 9, 128, 52, 3, False, "qk", "joint", 50),
    (BF16, 1, 2, 1, 9, 120, 44, 1, False, "qk", "joint", 50),
    (F32, 1, 3, 2, 33, 64, 12, 1, False, "qk", "dense", 9),
    (BF16, 1, 3, 2, 33, 64, 4, 1, False, "", "dense", 9),
    (BF16, 1, 3, 1, 33, 248, 124, 1, False, "q", "joint", 9),
    (F32, 1, 3, 1, 5, 8, 2, 1, False, "q", "joint", 9),
    (BF16, 1, 3, 1, 5, 16, 6, 1, False, "q", "joint", 9),
]


def operands(case, seed=0):
    dtype, b, hq, hkv, n, d, pairs, axes, interleaved, norms, layout, far = case
    gen = torch.Generator().manual_seed(seed)
    if layout == "joint":
        joint = (torch.randn((b, n, hq + 2 * hkv + 1, d), generator=gen) * 2).to(dtype).cuda()
        q, k = joint[:, :, :hq].transpose(1, 2), joint[:, :, hq:hq + hkv].transpose(1, 2)
    else:
        q, k = ((torch.randn((b, h, n, d), generator=gen) * 2).to(dtype).cuda() for h in (hq, hkv))
    options = {}
    if pairs:
        first = torch.randint(0, far + 1, (max(axes, 1), b, 1), generator=gen)
        positions = (first + torch.randint(0, 50, (max(axes, 1), b, n), generator=gen)).int()
        options = {"positions": positions.cuda() if axes > 1 else positions[0].cuda(), "frequencies": (10000.0 ** (-torch.arange(pairs) / pairs)).float().cuda(),
                   "interleaved": interleaved}
        if axes > 1:
            options["axes"] = torch.randint(0, axes, (pairs,), generator=gen).int().cuda()
    weights = {}
    for name in "qk":
        if name in norms and (name == "q" or hkv):
            weights[f"{name}_weight"] = (1 + 0.3 * torch.randn(d, generator=gen)).to(F32 if "w" in norms else dtype).cuda()
    grads = [torch.randn(x.shape, generator=gen).to(dtype).cuda() for x in (q, k)]
    return q, k if hkv else None, options, weights, grads


def sides(q, k, options, weights):
    for name, x in (("q", q), ("k", k)):
        if x is not None:
            yield name, x, Rotation(x, weight=weights.get(f"{name}_weight"), **options)


@pytest.mark.parametrize("case", CASES, ids=names)
def test_forward(ops, case):
    print(names(case), flush=True)
    q, k, options, weights, _ = operands(case)
    results = ops.rotate(q, k, **options, **weights)
    for (name, x, want), got in zip(sides(q, k, options, weights), results):
        within(got, want.y, want.y_bound, name)
    # again over the operands themselves: the same bits
    before = [None if x is None else x.clone() for x in results]
    ops.rotate(q, k, **options, **weights, out=(q, k))
    for got, want in zip((q, k), before):
        assert got is None or torch.equal(got, want)


@pytest.mark.parametrize("case", CASES, ids=names)
def test_gradient(ops, case):
    print(names(case), flush=True)
    q, k, options, weights, (grad_q, grad_k) = operands(case, 1)
    grad_k = None if k is None else grad_k
    dq, dk, dqw, dkw = ops.rotate_backward(grad_q, grad_k, q, k, **options, **weights)
    got = {"q": (dq, dqw), "k": (dk, dkw)}
    for name, x, want in sides(q, k, options, weights):
        weight = weights.get(f"{name}_weight")
        dx, bound, dw, dw_bound = want.gradients(grad_q if name == "q" else grad_k, None if weight is None else weight.dtype)
        within(got[name][0], dx, bound, f"d{name}")
        if weight is None:
            assert got[name][1] is None
        else:
            within(got[name][1], dw, dw_bound, f"d{name}_weight")
    # the same call gives the same bits, over the gradients given too
    again = ops.rotate_backward(grad_q, grad_k, q, k, **options, **weights, grads=(grad_q, grad_k))
    for one, two in zip(again, (dq, dk, dqw, dkw)):
        assert (one is None) == (two is None) and (one is None or torch.equal(one, two))


def test_gradient_against_differences(ops):
    """f32: the derivative along a direction, by central differences of the definition in 64 bits."""
    case = (F32, 2, 3, 2, 5, 64, 24, 2, False, "qk", "dense", 30)
    q, k, options, weights, (grad_q, grad_k) = operands(case, 3)
    grads = ops.rotate_backward(grad_q, grad_k, q, k, **options, **weights)
    gen = torch.Generator().manual_seed(9)
    steps = [torch.randn(x.shape, generator=gen).double() for x in (q, k, weights["q_weight"], weights["k_weight"])]
    values = [x.cpu().double() for x in (q, k, weights["q_weight"], weights["k_weight"])]

    def loss(h):
        q, k, qw, kw = (x + h * step for x, step in zip(values, steps))
        total = 0.0
        for x, w, g in ((q, qw, grad_q), (k, kw, grad_k)):
            turning = Rotation(x.float(), **options).turning
            n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
            total += (turned(n, *turning) * g.cpu().double()).sum()
        return total

    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = sum((g.cpu().double() * step).sum() for g, step in zip(grads, steps))
    # the differences' own error is (1e-5)^2 of a third derivative; f32 gradients of ~2000 terms: 1e-5 of their size
    size = sum((g.cpu().double() * step).abs().sum() for g, step in zip(grads, steps))
    assert abs(got - slope) < 1e-5 * size


def test_autograd(ops):
    case = (BF16, 2, 4, 2, 33, 64, 32, 1, False, "qk", "joint", 100)
    q, k, options, weights, (grad_q, grad_k) = operands(case, 4)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, weights["q_weight"], weights["k_weight"])]
    y, z = ops.rotated(leaves[0], leaves[1], options["positions"], options["frequencies"], q_weight=leaves[2], k_weight=leaves[3])
    # a gradient that arrives expanded and one that arrives transposed
    (y.float() * grad_q.float()).sum().backward(retain_graph=True)
    want = ops.rotate_backward(grad_q, torch.zeros_like(grad_k), q, k, **options, **weights)
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[2].grad, want[2])
    assert not leaves[1].grad.any() and not leaves[3].grad.any()
    for leaf in leaves:
        leaf.grad = None
    (y.sum() + z.sum()).backward()
    ones = ops.rotate_backward(torch.ones_like(grad_q), torch.ones_like(grad_k), q, k, **options, **weights)
    for leaf, one in zip(leaves, ones):
        assert torch.equal(leaf.grad, one)
    # no gradient of the gradient, and constants may not change in between
    y, z = ops.rotated(leaves[0], leaves[1], options["positions"], options["frequencies"], q_weight=leaves[2], k_weight=leaves[3])
    first = torch.autograd.grad(y.float().square().sum(), leaves[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="gradient of its gradient"):
        first.float().sum().backward()
    y, z = ops.rotated(leaves[0], leaves[1], options["positions"], options["frequencies"], q_weight=leaves[2], k_weight=leaves[3])
    options["positions"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


def test_what_is_not_turned_is_not_touched(ops):
    """Infinities and NaN stay in their row, and without a norm in their pair."""
    x = torch.randn((1, 2, 4, 64), dtype=BF16, device="cuda")
    x[0, 0, 1, 40], x[0, 1, 2, 63], x[0, 1, 3, 1] = float("inf"), float("nan"), float("inf")
    f = ops.frequencies(20)
    at = torch.arange(1, 5, dtype=torch.int32, device="cuda")
    for interleaved in (False, True):
        y, _ = ops.rotate(x, None, at, f, interleaved=interleaved)
        clean = torch.where(x.isfinite(), x, torch.zeros_like(x))
        z, _ = ops.rotate(clean, None, at, f, interleaved=interleaved)
        odd = ~y.isfinite()
        assert torch.equal(torch.where(odd, 0, y), torch.where(odd, 0, z))
        pair = 0 if interleaved else 21
        assert set(map(tuple, odd.nonzero().tolist())) == {(0, 0, 1, 40), (0, 1, 2, 63), (0, 1, 3, 1), (0, 1, 3, pair)}
    y, _ = ops.rotate(x, None, at, f, q_weight=torch.ones(64, dtype=BF16, device="cuda"))
    assert y[0, 0, 0].isfinite().all() and y[0, 0, 2:].isfinite().all() and y[0, 1, :2].isfinite().all()


def test_shared_positions(ops):
    q = torch.randn((3, 2, 7, 64), dtype=F32, device="cuda")
    f, at = ops.frequencies(32), torch.arange(7, dtype=torch.int32, device="cuda") * 3
    one, _ = ops.rotate(q, None, at, f)
    two, _ = ops.rotate(q, None, at.expand(3, 7), f)
    three, _ = ops.rotate(q, None, at.repeat(3, 1), f)
    assert torch.equal(one, two) and torch.equal(one, three)
    axes = ops.sections(10, 22)
    assert axes.tolist() == [0] * 10 + [1] * 22
    grid = torch.stack([at, at + 5])
    one, _ = ops.rotate(q, None, grid, f, axes=axes)
    two, _ = ops.rotate(q, None, grid[:, None].repeat(1, 3, 1), f, axes=axes)
    assert torch.equal(one, two)
    # an axis that there is not counts as the nearest
    wild = torch.where(axes == 1, 9, -4).int()
    three, _ = ops.rotate(q, None, grid, f, axes=wild)
    assert torch.equal(one, three)


def test_nothing_to_do(ops):
    f, at = ops.frequencies(32), torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    w = torch.ones(64, device="cuda")
    for b, n in ((2, 0), (0, 3)):
        q = torch.zeros((b, 4, n, 64), device="cuda")
        at = torch.zeros((b, n), dtype=torch.int32, device="cuda")
        y, _ = ops.rotate(q, None, at, f, q_weight=w)
        assert y.shape == q.shape
        dq, _, dw, _ = ops.rotate_backward(q, None, q, None, at, f, q_weight=w)
        assert dq.shape == q.shape and not dw.any() and dw.isfinite().all()


def test_captured(ops):
    """Forward and backward in a graph, replayed with eager calls between."""
    case = (BF16, 2, 8, 2, 100, 128, 64, 1, False, "qk", "dense", 1000)
    q, k, options, weights, (grad_q, grad_k) = operands(case, 5)

    def calls():
        return (*ops.rotate(q, k, **options, **weights), *ops.rotate_backward(grad_q, grad_k, q, k, **options, **weights))

    calls()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            kept = calls()
    torch.cuda.synchronize()
    for n in range(3):
        q.copy_(torch.randn_like(q))
        grad_k.copy_(torch.randn_like(grad_k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(kept, calls()):
            assert torch.equal(got, want), n


def test_without_keys_and_without_heads(ops):
    """Queries alone under autograd; a side without heads has no rows, and a weight's gradient of zeros."""
    q = torch.randn((2, 3, 5, 64), dtype=F32, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    f, at = ops.frequencies(32), torch.arange(5, dtype=torch.int32, device="cuda")
    y, none = ops.rotated(q, None, at, f, q_weight=w)
    assert none is None
    y.square().sum().backward()
    want = ops.rotate_backward(2 * y.detach(), None, q.detach(), None, at, f, q_weight=w.detach())
    assert torch.equal(q.grad, want[0]) and torch.equal(w.grad, want[2]) and want[1] is None and want[3] is None
    nobody = torch.zeros((2, 0, 5, 64), device="cuda")
    k = q.detach()
    z, y2 = ops.rotate(nobody, k, at, f, q_weight=w.detach(), k_weight=w.detach())
    assert z.shape == nobody.shape and torch.equal(y2, y.detach())
    _, dk, dqw, dkw = ops.rotate_backward(nobody, k, nobody, k, at, f, q_weight=w.detach(), k_weight=w.detach())
    assert not dqw.any() and dqw.isfinite().all() and dkw.any() and dk.any()


def test_positions_far_and_negative(ops):
    """The whole range of positions: angles as exact as near ones."""
    far = torch.tensor([[0, -1, 2 ** 31 - 1, -2 ** 31, 123456789, -987654321]], dtype=torch.int32)
    x = torch.randn((1, 2, 6, 64), generator=torch.Generator().manual_seed(2))
    f = ops.frequencies(32, 1e6)
    y, _ = ops.rotate(x.cuda(), None, far.cuda(), f)
    want = Rotation(x, far, f)
    within(y, want.y, want.y_bound, "y")


def test_another_stream_and_two_calls_at_once(ops):
    """Calls on two streams at the same time, on operands of their own."""
    case = (BF16, 2, 16, 4, 300, 128, 64, 1, False, "qk", "joint", 1000)
    sets = [operands(case, seed) for seed in (11, 12)]
    want = [(*ops.rotate(q, k, **o, **w), *ops.rotate_backward(*g, q, k, **o, **w)) for q, k, o, w, g in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for stream, (q, k, o, w, g) in zip(streams, sets):
        with torch.cuda.stream(stream):
            for _ in range(3):
                results = (*ops.rotate(q, k, **o, **w), *ops.rotate_backward(*g, q, k, **o, **w))
            got.append(results)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_rows_that_are_far_apart(ops):
    """Offsets past 32 bits: heads more than 2^32 bytes apart."""
    memory = torch.zeros((2 ** 32 + 2 ** 20) // 2, dtype=BF16, device="cuda")
    x = memory.as_strided((1, 2, 4, 64), (0, 2 ** 31, 64, 1))
    x.copy_(torch.randn((1, 2, 4, 64)))
    f, at = ops.frequencies(32), torch.arange(4, dtype=torch.int32, device="cuda")
    near = x.contiguous()
    y, _ = ops.rotate(near, None, at, f)
    ops.rotate(x, None, at, f, out=(x, None))
    assert torch.equal(x, y)


def test_more_rows_than_a_launch_is_wide(ops):
    """2^28 rows of one head, whose workgroups take more than one tile of them each."""
    b, n = 256, 2 ** 20
    f, at = ops.frequencies(4), torch.arange(n, dtype=torch.int32, device="cuda")
    one = torch.randn((1, 1, n, 8), device="cuda").to(BF16)
    q = one.expand(b, 1, n, 8).contiguous()
    ops.rotate(q, None, at, f, out=(q, None))
    y, _ = ops.rotate(one, None, at, f)
    for s in (0, 1, 100, 254, 255):
        assert torch.equal(q[s], y[0])


def test_refusals(ops):
    q = torch.zeros((2, 4, 8, 64), dtype=BF16, device="cuda")
    k, w = q[:, :2].contiguous(), torch.ones(64, dtype=BF16, device="cuda")
    f, at = ops.frequencies(32), torch.zeros((2, 8), dtype=torch.int32, device="cuda")
    axes = ops.sections(16, 16)
    for call in (lambda: ops.rotate(q, k, at), lambda: ops.rotate(q, k, None, f), lambda: ops.rotate(q, k, at[:1], f), lambda: ops.rotate(q, k[:, :, :4], at, f),
                 lambda: ops.rotate(q, k, at, f, axes=axes[:8]), lambda: ops.rotate(q, k, at[None], f), lambda: ops.rotate(q, k, q_weight=w[:32]),
                 lambda: ops.rotate(q, None, k_weight=w), lambda: ops.rotate(q[0], None), lambda: ops.rotate(q, k, out=(q, k[:1])),
                 lambda: ops.rotate(q, k, torch.zeros((2, 16), dtype=torch.int32, device="cuda")[:, ::2], f), lambda: ops.rotate(q, k, axes=axes),
                 lambda: ops.rotate(q, k, out=(q[:1].expand(2, 4, 8, 64), k)), lambda: ops.rotate(q.transpose(2, 3), None)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.rotate(q, k.float()), lambda: ops.rotate(q, k, at.long(), f), lambda: ops.rotate(q, k, at, f.double()), lambda: ops.rotate(q, k, q_weight=w.half()),
                 lambda: ops.rotate(q, k, q_weight=w, k_weight=w.float()), lambda: ops.rotate(q.half(), None), lambda: ops.rotate(q, k, at.cpu(), f)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ops.rotate(q, k, at, ops.frequencies(33)), lambda: ops.rotate(q[..., :60], None), lambda: ops.rotate(q[..., 4:60], None),
                 lambda: ops.rotate(q, None, eps=-1.0), lambda: ops.rotate(q, None, out=(q.transpose(1, 2).contiguous().as_strided((2, 4, 8, 64), (2048, 68, 256, 1)), None))):
        with pytest.raises(RuntimeError):
            call()
