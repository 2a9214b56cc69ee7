"""How far gradients in bf16 are from 64 bits, next to what rounding the exact ones to bf16 costs.

Both are norms over a whole tensor.  dq and dk take dS in 16 bits and sums in 32, so that next to their own rounding (2^-9) only
delta = do.o counts, whose o is rounded too.  That error is p times as large in every dS, a part 1 / sqrt(keys that share the weight) of a
row's gradient: it has to be kept out of rows of few keys, whose delta is summed from p and do.v instead.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from i_amd import attention

    return attention


def exact(q, k, v, grad, hidden, scale, cap, slopes):
    q, k, v, grad = (x.cpu().double() for x in (q, k, v, grad))
    b, hq, n, _ = q.shape
    group = hq // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s, bend = q @ kk.transpose(2, 3) * scale, 1.0
    if cap:
        t = torch.tanh(s / cap)
        s, bend = cap * t, 1 - t * t
    if slopes is not None:
        s = s - slopes.cpu().double().view(1, hq, 1, 1) * (torch.arange(n)[:, None] - torch.arange(n)).abs()
    p = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
    ds = p * (grad @ vv.transpose(2, 3) - (grad * (p @ vv)).sum(-1, keepdim=True)) * bend * scale
    shared = lambda x: x.view(b, k.shape[1], group, *x.shape[2:]).sum(2)  # noqa: E731
    return ds @ kk, shared(ds.transpose(2, 3) @ q), shared(p.transpose(2, 3) @ grad)


def off(x, want):
    return float((x.cpu().double() - want).norm() / want.norm())


# b, hq, hkv, n, d, kind of mask, cap, bias
CASES = [(8, 16, 4, 2, 64, "none", 0.0, False), (8, 16, 4, 3, 128, "causal", 0.0, False), (4, 16, 4, 5, 64, "none", 0.0, True), (6, 80, 10, 12, 96, "causal", 0.0, False),
         (4, 8, 8, 16, 128, "causal", 2.0, True), (4, 8, 8, 16, 256, "none", 30.0, False), (2, 16, 4, 600, 128, "documents 2", 0.0, False),
         (2, 16, 4, 600, 64, "documents 9", 30.0, False), (1, 64, 16, 600, 64, "documents 16", 0.0, True), (2, 16, 4, 500, 128, "window 2", 0.0, False), (1, 80, 80, 500, 64, "window 7", 0.0, True)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients_of_rows_of_few_keys(ops, case):
    b, hq, hkv, n, d, mask, cap, bias = case
    gen = torch.Generator().manual_seed(n + d)
    q, k, v, grad = ((torch.randn((b, n, h, d), generator=gen) * spread).to(BF16).cuda().transpose(1, 2) for h, spread in ((hq, 1.5), (hkv, 1.0), (hkv, 1.0), (hq, 1.0)))
    i = torch.arange(n)
    hidden, options = torch.zeros((n, n), dtype=torch.bool), {"cap": cap, "slopes": torch.linspace(0.02, 0.3, hq, device="cuda") if bias else None}
    if mask != "none":
        options["causal"] = True
        hidden |= i[None] > i[:, None]
    if mask.startswith("documents"):
        ids = i // int(mask.split()[1])
        options["first"] = ops.document_bounds(ids.expand(b, n).cuda())[0]
        hidden |= ids[None] != ids[:, None]
    elif mask.startswith("window"):
        width = int(mask.split()[1])
        options["first"] = ops.window_bounds(b, n, n, width, "cuda")
        hidden |= i[None] <= i[:, None] - width
    o, lse = ops.attention(q, k, v, **options)
    got = ops.attention_backward(grad, q, k, v, o, lse, **options)
    want = exact(q, k, v, grad, hidden, d ** -0.5, cap, options["slopes"])
    for x, ref, name, most in zip(got, want, ("dq", "dk", "dv"), (1.1, 1.1, 1.5)):
        # (dv takes P in bf16, an error as large as its rounding: the square root of 2)
        assert off(x, ref) <= most * off(ref.to(BF16), ref), f"{name}: {off(x, ref) / off(ref.to(BF16), ref):.2f} times what rounding costs"
