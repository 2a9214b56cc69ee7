"""Norms and rotary positions: calls after other calls."""
import pytest
import torch

from attend_oracle import within
from rotary_oracle import Rotation

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from i_amd import rotary

    return rotary


# pairs and whether they are neighbours, of 128 columns: halves, neighbours, quads, and pairs in no such order
LAYOUTS = [(64, False), (13, False), (13, True), (20, False), (64, True), (0, False)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("order", [1, -1])
def test_gradients_of_one_size_and_several_layouts(ops, dtype, order):
    """Gradients of the same operands whose pairs lie in another way, one after another in either order."""
    gen = torch.Generator().manual_seed(30)
    # (a size of its own for each order and type, so that neither finds what the other left)
    b, hq, hkv, n, d = 2, 6, 3, 3000 + 8 * order, 128
    q, k, grad_q, grad_k = (torch.randn((b, h, n, d), generator=gen).to(dtype).cuda() for h in (hq, hkv, hq, hkv))
    weights = {f"{side}_weight": (1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).cuda() for side in "qk"}
    at = torch.randint(0, 5000, (b, n), generator=gen).int().cuda()
    for pairs, interleaved in LAYOUTS[::order]:
        print(pairs, interleaved, flush=True)
        turning = {"positions": at, "frequencies": ops.frequencies(pairs)} if pairs else {}
        got = ops.rotate_backward(grad_q, grad_k, q, k, interleaved=interleaved, **turning, **weights)
        for x, grad, weight, dx, dw in ((q, grad_q, weights["q_weight"], got[0], got[2]), (k, grad_k, weights["k_weight"], got[1], got[3])):
            want = Rotation(x, weight=weight, interleaved=interleaved, **turning).gradients(grad, dtype)
            within(dx, want[0], want[1], "dx")
            within(dw, want[2], want[3], "dw")


@pytest.mark.parametrize("pairs, interleaved", [(64, False), (64, True), (52, False), (61, False)])
def test_cosines_and_sines_themselves(ops, pairs, interleaved):
    """Pairs (1, 0) in f32 turn into the cosine and sine of their angle, and back into cosine and negative sine.  The angle's remainder is
    rounded to f32, off by at most 2^-26 of a turn, 2 pi 2^-26 of a cosine or sine (two roundings in 64 bits before it add less than 2^-33 at
    these positions); the functions are off by at most two steps of values below 1, 2 2^-24."""
    gen = torch.Generator().manual_seed(31)
    b, n, d = 2, 1000, 128
    at = torch.randint(-10 ** 6, 10 ** 6, (b, n), generator=gen).int()
    f = ops.frequencies(pairs, 100.0)
    j = torch.arange(pairs)
    a, c = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    x = torch.zeros((b, 1, n, d))
    x[..., a] = 1.0
    angle = at.double()[:, None, :, None] * f.cpu().double()
    off = 2 * torch.pi * 2.0 ** -26 + 2.0 ** -23 + 2.0 ** -33
    y, _ = ops.rotate(x.cuda(), None, at.cuda(), f, interleaved=interleaved)
    z = ops.rotate_backward(x.cuda(), None, x.cuda(), None, at.cuda(), f, interleaved=interleaved)[0]
    for got, sine in ((y.cpu().double(), torch.sin(angle)), (z.cpu().double(), -torch.sin(angle))):
        assert float((got[..., a] - torch.cos(angle)).abs().max()) <= off
        assert float((got[..., c] - sine).abs().max()) <= off
