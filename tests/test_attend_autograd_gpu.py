"""attention as an autograd function: what it refuses, and bounds that change between its two passes."""
import pytest
import torch

from attend_oracle import Attention, within

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import attention

    return attention


def tensors(dtype, b=1, hq=4, hkv=2, n=60, d=32):
    gen = torch.Generator().manual_seed(n)
    q, k, v, grad = ((torch.randn((b, h, n, d), generator=gen) * spread).to(dtype).cuda() for h, spread in ((hq, 1.5), (hkv, 1.0), (hkv, 1.0), (hq, 1.0)))
    return *(x.requires_grad_() for x in (q, k, v)), grad


def test_a_gradient_of_a_gradient_is_refused(ops):
    """There is no second-order gradient: a penalty on the gradient is an error, not a penalty without attention's part."""
    q, k, v, grad = tensors(F32)
    o = ops.differentiable(q, k, v, causal=True)
    gq, = torch.autograd.grad(o, q, grad, create_graph=True)
    assert gq.requires_grad
    with pytest.raises(RuntimeError, match="no gradient of its gradient"):
        gq.square().sum().backward()
    # with parameters outside, whose graph goes on
    w = torch.ones((), device="cuda", requires_grad=True)
    gk, = torch.autograd.grad(ops.differentiable(q * w, k, v, causal=True), w, grad, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its gradient"):
        gk.backward()


@pytest.mark.parametrize("which", ["first", "last", "slopes"])
def test_bounds_that_change_before_the_gradient_are_an_error(ops, which):
    q, k, v, grad = tensors(F32)
    constants = {"first": ops.window_bounds(1, 60, 60, 9, "cuda"), "last": torch.full((1, 60), 50, dtype=torch.int32, device="cuda"),
                 "slopes": torch.full((4,), 0.25, device="cuda")}
    o = ops.differentiable(q, k, v, causal=True, **constants)
    constants[which].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(grad)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_all_options_through_autograd(ops, dtype):
    q, k, v, grad = tensors(dtype, b=2, n=75)
    options = dict(causal=True, first=ops.window_bounds(2, 75, 75, 20, "cuda"), last=torch.full((2, 75), 70, dtype=torch.int32, device="cuda"),
                   slopes=torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda"), cap=15.0, scale=0.2)
    want = Attention(q, k, v, **options)
    ops.differentiable(q, k, v, **options).backward(grad)
    for x, ref, bound, name in zip((q, k, v), *want.gradients(grad), ("dq", "dk", "dv")):
        within(x.grad, ref, bound, name)
