"""Attention with masks, caps and biases, its gradient and the weights of keys, against float64 on the CPU."""
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


def tensors(seed, dtype, b, hq, hkv, nq, nk, d, rows_first=False):
    gen = torch.Generator().manual_seed(seed)

    def make(h, n, spread):
        x = (torch.randn((b, n, h, d), generator=gen) * spread).to(dtype).cuda()
        return x.transpose(1, 2) if rows_first else x.transpose(1, 2).contiguous()

    return make(hq, nq, 1.5), make(hkv, nk, 1.0), make(hkv, nk, 1.0), make(hq, nq, 1.0)


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=F32, device="cuda")


def bounds_of(ops, kind, b, nq, nk, seed=0):
    gen = torch.Generator().manual_seed(seed + 17)
    if kind in ("none", "causal"):
        return {"causal": kind == "causal"}
    if kind == "documents":
        ids = (torch.rand((b, nk), generator=gen) < 0.06).int().cumsum(1).cuda()
        first, last = ops.document_bounds(ids)
        return {"causal": True, "first": first[:, nk - nq:].contiguous()}
    if kind == "whole_documents":
        ids = (torch.rand((b, nk), generator=gen) < 0.03).int().cumsum(1).cuda()
        first, last = ops.document_bounds(ids)
        return {"first": first[:, nk - nq:].contiguous(), "last": last[:, nk - nq:].contiguous()}
    if kind == "prefix":
        prefix = torch.randint(0, nk + 1, (b,), generator=gen).cuda()
        return {"last": ops.prefix_bounds(prefix, nk)[:, nk - nq:].contiguous()}
    if kind == "window":
        return {"causal": True, "first": ops.window_bounds(b, nq, nk, 19, "cuda")}
    # any interval at all: empty ones, ones outside the keys
    first = torch.randint(-5, nk + 5, (b, nq), generator=gen, dtype=torch.int32).cuda()
    width = torch.randint(-3, nk // 2 + 2, (b, nq), generator=gen, dtype=torch.int32).cuda()
    return {"first": first, "last": first + width}


# type, b, hq, hkv, nq, nk, d, mask, cap, bias, rows first
CASES = [
    (BF16, 1, 1, 1, 1, 1, 64, "causal", 0.0, False, False),
    (F32, 1, 1, 1, 1, 1, 8, "none", 0.0, False, False),
    (BF16, 2, 4, 2, 130, 130, 128, "causal", 0.0, False, True),
    (BF16, 1, 3, 1, 257, 257, 128, "causal", 30.0, True, True),
    (F32, 1, 2, 2, 130, 130, 64, "causal", 0.0, False, False),
    (F32, 2, 4, 2, 97, 97, 128, "documents", 20.0, True, True),
    (BF16, 2, 2, 2, 333, 333, 80, "documents", 0.0, True, True),
    (BF16, 1, 2, 1, 300, 300, 96, "whole_documents", 0.0, False, False),
    (BF16, 2, 2, 2, 200, 200, 64, "prefix", 0.0, False, True),
    (BF16, 1, 6, 2, 191, 191, 256, "causal", 50.0, False, True),
    (F32, 1, 2, 1, 65, 65, 256, "window", 0.0, True, False),
    (F32, 1, 2, 1, 70, 70, 200, "prefix", 0.0, False, False),
    (F32, 1, 3, 3, 150, 150, 88, "window", 0.0, False, True),
    (BF16, 1, 2, 2, 129, 129, 40, "window", 0.0, True, False),
    (BF16, 2, 2, 1, 100, 177, 64, "causal", 0.0, False, False),
    (BF16, 1, 2, 1, 177, 100, 64, "causal", 0.0, True, False),   # the first queries see nothing
    (F32, 1, 2, 1, 90, 33, 64, "causal", 0.0, False, False),
    (BF16, 2, 2, 1, 150, 210, 128, "any", 0.0, False, True),
    (F32, 2, 2, 1, 150, 140, 64, "any", 10.0, True, False),
    (BF16, 1, 16, 1, 40, 40, 104, "none", 0.0, False, False),
    (F32, 1, 1, 1, 1, 200, 64, "none", 0.0, True, False),
    (BF16, 1, 8, 2, 2, 513, 128, "causal", 0.0, False, True),
    (BF16, 3, 1, 1, 513, 3, 64, "none", 0.0, False, False),
]


def names(case):
    return "-".join(str(x).replace("torch.", "") for x in case)


@pytest.mark.parametrize("case", CASES, ids=names)
def test_forward_gradient_and_weights(ops, case):
    dtype, b, hq, hkv, nq, nk, d, mask, cap, bias, rows_first = case
    print(names(case), flush=True)
    q, k, v, grad = tensors(nq + nk + d, dtype, b, hq, hkv, nq, nk, d, rows_first)
    options = dict(bounds_of(ops, mask, b, nq, nk, d), cap=cap, slopes=slopes_of(hq) if bias else None)
    want = Attention(q, k, v, **options)
    o, lse = ops.attention(q, k, v, **options)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")
    got = ops.attention_backward(grad, q, k, v, o, lse, **options)
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(got, gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)
    weights, bound = want.weights()
    within(ops.key_weights(q, k, lse, **options), weights, bound, "weights")


# Queries are dealt out in three ways, by the number of their 128-query tiles: few above, 64 .. 256 and more than 256 here.
DEALT = [(dtype, b, hq, hq // 4, nq, nk, d, mask, cap, bias, True)
         for dtype in (BF16, F32)
         for d, mask, cap, bias in ((64, "causal", 0.0, False), (80, "documents", 20.0, False), (128, "any", 0.0, True), (256, "prefix", 30.0, False))
         for b, hq, nq, nk in ((2, 40, 130, 203), (3, 44, 200, 200))]


@pytest.mark.parametrize("case", DEALT, ids=names)
def test_many_queries(ops, case):
    test_forward_gradient_and_weights(ops, case)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sums_do_not_change_from_run_to_run(ops, dtype):
    q, k, v, grad = tensors(5, dtype, 1, 8, 1, 300, 300, 64)
    options = {"causal": True, "cap": 20.0}
    o, lse = ops.attention(q, k, v, **options)
    first = ops.attention_backward(grad, q, k, v, o, lse, **options)
    weights = ops.key_weights(q, k, lse, **options)
    for _ in range(3):
        again = ops.attention_backward(grad, q, k, v, o, lse, **options)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert torch.equal(weights, ops.key_weights(q, k, lse, **options))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_scales(ops, scale, cap):
    q, k, v, grad = tensors(11, F32, 1, 2, 2, 70, 70, 64)
    options = {"causal": True, "scale": scale, "cap": cap}
    want = Attention(q, k, v, **options)
    o, lse = ops.attention(q, k, v, **options)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(ops.attention_backward(grad, q, k, v, o, lse, **options), gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_that_grow_along_the_keys(ops, dtype):
    """The running maximum moves in every tile, and scores reach far past what exp holds without it."""
    q, k, v, grad = tensors(3, dtype, 1, 1, 1, 64, 400, 64)
    q, k = q.abs(), (k.abs() * torch.linspace(0.1, 40.0, 400, device="cuda")[:, None]).to(dtype)
    want = Attention(q, k, v, scale=0.3)
    o, lse = ops.attention(q, k, v, scale=0.3)
    within(o, want.o, want.o_bound, "o")
    within(lse, want.lse, want.lse_bound, "lse")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_keys_that_nobody_sees_may_hold_anything(ops, dtype, poison):
    b, n, length, d = 2, 200, 130, 64
    q, k, v, grad = tensors(9, dtype, b, 2, 1, n, n, d)
    last = torch.full((b, n), length, dtype=torch.int32, device="cuda")
    want = Attention(q, k, v, last=last)
    k[:, :, length:], v[:, :, length:] = poison, poison
    o, lse = ops.attention(q, k, v, last=last)
    within(o, want.o, want.o_bound, "o")
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(ops.attention_backward(grad, q, k, v, o, lse, last=last), gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)
    weights, bound = want.weights()
    within(ops.key_weights(q, k, lse, last=last), weights, bound, "weights")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq", [20, 80])  # (more queries than above: see DEALT)
def test_unseen_keys_beside_many_queries(ops, dtype, hq):
    b, n, length, d = 2, 200, 130, 128
    q, k, v, grad = tensors(10, dtype, b, hq, hq // 4, n, n, d)
    last = torch.full((b, n), length, dtype=torch.int32, device="cuda")
    last[:, 7::9] = 0  # rows that see nothing
    want = Attention(q, k, v, last=last)
    k[:, :, length:], v[:, :, length:] = math.nan, math.inf
    o, lse = ops.attention(q, k, v, last=last)
    within(o, want.o, want.o_bound, "o")
    assert bool((o[:, :, 7::9] == 0).all()) and bool((lse[:, :, 7::9] == -math.inf).all())
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(ops.attention_backward(grad, q, k, v, o, lse, last=last), gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)


def test_keys_of_the_lowest_value(ops):
    """A mask written into the operands as the type's lowest value instead of as bounds."""
    q, k, v, _ = tensors(13, F32, 1, 1, 1, 40, 90, 64)
    q, k = q.abs() + 0.1, k * 0.5
    k[:, :, 50:] = torch.finfo(F32).min
    o, lse = ops.attention(q, k, v, scale=1e-3)
    want = Attention(q, k[:, :, :50], v[:, :, :50], scale=1e-3)
    within(o, want.o, want.o_bound, "o")


def test_a_gradient_by_differences(ops):
    """The f32 gradient against central differences of the f32 forward pass."""
    q, k, v, grad = tensors(21, F32, 1, 2, 1, 24, 24, 16)
    options = {"causal": True, "cap": 4.0, "slopes": slopes_of(2)}
    o, lse = ops.attention(q, k, v, **options)
    got = ops.attention_backward(grad, q, k, v, o, lse, **options)
    gen = torch.Generator().manual_seed(4)
    step = 2.0 ** -6
    for which in range(3):
        for _ in range(4):
            way = torch.randn(got[which].shape, generator=gen).cuda()
            sides = []
            for sign in (step, -step):
                operands = [q, k, v]
                operands[which] = operands[which] + sign * way
                sides.append((ops.attention(*operands, **options)[0].double() * grad.double()).sum())
            slope = (sides[0] - sides[1]) / (2 * step)
            # third-order term of the difference (the loss is smooth on the scale of 1) and f32 rounding over the step
            scale = (got[which].double().abs() * way.double().abs()).sum()
            assert abs((got[which].double() * way.double()).sum() - slope) < 2e-2 * scale


def test_autograd(ops):
    q, k, v, grad = tensors(8, F32, 1, 4, 2, 50, 50, 32)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    options = {"causal": True, "cap": 6.0}
    o = ops.differentiable(q, k, v, **options)
    o.backward(grad)
    want = Attention(q, k, v, **options)
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip((q, k, v), gradients, bounds, ("dq", "dk", "dv")):
        within(x.grad, ref, bound, name)
    # a gradient of one value for all (expanded, stride 0)
    q.grad = k.grad = v.grad = None
    ops.differentiable(q, k, v, **options).sum().backward()
    gradients, bounds = want.gradients(torch.ones_like(grad))
    within(q.grad, gradients[0], bounds[0], "dq")


def test_broadcast_operands(ops):
    """Keys of one sequence for all sequences, by a stride of zero."""
    q, k, v, grad = tensors(31, BF16, 3, 2, 2, 70, 90, 64)
    k, v = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    want = Attention(q, k, v)
    o, lse = ops.attention(q, k, v)
    within(o, want.o, want.o_bound, "o")
    grads = tuple(torch.empty(x.shape, dtype=BF16, device="cuda") for x in (q, k, v))
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(ops.attention_backward(grad, q, k, v, o, lse, grads=grads), gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)


def test_weights_are_added(ops):
    q, k, _, _ = tensors(41, BF16, 2, 4, 2, 60, 60, 64)
    _, lse = ops.attention(q, k, k, causal=True)
    step = ops.key_weights(q, k, lse, causal=True)
    before = torch.rand_like(step)
    assert torch.allclose(ops.key_weights(q, k, lse, causal=True, weights=before), before + step, rtol=1e-6, atol=0)
    kept = before.clone()
    assert ops.key_weights(q, k, lse, causal=True, weights=kept, out=kept) is kept
    assert torch.allclose(kept, before + step, rtol=1e-6, atol=0)


def test_another_stream_and_given_outputs(ops):
    q, k, v, grad = tensors(51, BF16, 1, 2, 2, 260, 260, 64)
    want = Attention(q, k, v, causal=True)
    o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:3], math.nan, dtype=F32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ops.attention(q, k, v, causal=True, out=o, lse=lse)[0] is o
        got = ops.attention_backward(grad, q, k, v, o, lse, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    within(o, want.o, want.o_bound, "o")
    gradients, bounds = want.gradients(grad)
    for x, ref, bound, name in zip(got, gradients, bounds, ("dq", "dk", "dv")):
        within(x, ref, bound, name)


def test_a_graph_of_the_calls(ops):
    q, k, v, grad = tensors(61, BF16, 1, 4, 1, 150, 150, 64)
    options = {"causal": True, "cap": 20.0}
    o, lse = ops.attention(q, k, v, **options)
    grads = ops.attention_backward(grad, q, k, v, o, lse, **options)
    weights = ops.key_weights(q, k, lse, **options)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, lse2 = ops.attention(q, k, v, **options)
        grads2 = ops.attention_backward(grad, q, k, v, o2, lse2, **options)
        weights2 = ops.key_weights(q, k, lse2, **options)
    for _ in range(3):
        for x in (o2, lse2, weights2, *grads2):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, lse2) and torch.equal(weights, weights2)
        assert all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_no_keys_and_no_queries(ops):
    q, k, v, grad = tensors(71, BF16, 2, 2, 1, 5, 0, 64)
    o, lse = ops.attention(q, k, v)
    assert torch.equal(o, torch.zeros_like(o)) and bool((lse == -math.inf).all())
    dq, dk, dv = ops.attention_backward(grad, q, k, v, o, lse)
    assert torch.equal(dq, torch.zeros_like(dq)) and dk.shape[2] == 0
    q, k, v, grad = tensors(72, BF16, 2, 2, 1, 0, 5, 64)
    o, lse = ops.attention(q, k, v)
    assert o.numel() == 0
    dq, dk, dv = ops.attention_backward(grad, q, k, v, o, lse)
    assert torch.equal(dk, torch.zeros_like(dk)) and torch.equal(dv, torch.zeros_like(dv))
    assert torch.equal(ops.key_weights(q, k, lse), torch.zeros((2, 1, 5), device="cuda"))


def test_refusals(ops):
    q, k, v, grad = tensors(81, BF16, 1, 4, 2, 20, 20, 64)
    o, lse = ops.attention(q, k, v)
    for bad in (lambda: ops.attention(q.float(), k, v), lambda: ops.attention(q.cpu(), k, v), lambda: ops.attention(q.half(), k, v),
                lambda: ops.attention(q, k, v, first=torch.zeros((1, 20), dtype=torch.int64, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.attention(q[0], k, v), lambda: ops.attention(q, k[..., :32], v), lambda: ops.attention(q, k, v[:, :1]),
                lambda: ops.attention(q, k, v, slopes=slopes_of(3)), lambda: ops.attention(q, k, v, out=q[:, :1].expand_as(q)),
                lambda: ops.attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.attention(q, k, v, cap=-1.0), lambda: ops.attention(q, k, v, cap=math.inf), lambda: ops.attention(q, k, v, scale=math.nan),
                lambda: ops.attention(q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous()),
                lambda: ops.attention(q[:, :3], k, v), lambda: ops.attention(q[..., 4:44], k[..., 4:44], v[..., 4:44])):
        with pytest.raises(RuntimeError, match="attention"):
            bad()
    with pytest.raises(RuntimeError, match="attention_backward"):
        ops.attention_backward(grad, q, k, v, o, lse, cap=-1.0)
