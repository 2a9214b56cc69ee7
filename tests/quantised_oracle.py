"""A cache in 8 or 4 bits from its definition, on the CPU: the number of every code, and the nearest of them."""
import math

import torch

TOP = 1.75 * 2.0 ** 127


def numbers(bits):
    """The number of every code, float64 (8 bits: codes 127 and 255 are no numbers)."""
    fraction_bits, bias = (1, 1) if bits == 4 else (3, 7)
    half, result = 1 << (bits - 1), []
    for code in range(half):
        exponent, fraction = code >> fraction_bits, (code % (1 << fraction_bits)) / (1 << fraction_bits)
        result.append(2.0 ** (exponent - bias) * (1 + fraction) if exponent else 2.0 ** (1 - bias) * fraction)
    if bits == 8:
        result[127] = math.nan
    return torch.tensor(result + [-x for x in result], dtype=torch.float64)


def power(exponent):
    return (exponent.long() + 1023 << 52).view(torch.float64)


def encode(values, bits):
    """Codes (one a column of the padded row) and scale bytes of rows of d columns."""
    x = torch.zeros((*values.shape[:-1], -(-values.shape[-1] // 32) * 32), dtype=torch.float64)
    x[..., :values.shape[-1]] = values.double()
    x = x.unflatten(-1, (-1, 32))
    of = numbers(bits)[:1 << (bits - 1)]
    of = of[of.isfinite()]
    beyond, least = (7.0, -125) if bits == 4 else (464.0, -117)
    top = x.abs().amax(-1)
    none = ~(top <= TOP)  # (NaN too)
    top = torch.where(none, 1.0, top)
    exponent = torch.full(top.shape, least)
    for e in range(least, 128):
        exponent = torch.where(top > beyond * power(exponent), torch.full_like(exponent, e), exponent)
    size = (x.abs() / power(exponent)[..., None]).nan_to_num(0.0, 0.0, 0.0)
    middle = (of[1:] + of[:-1]) / 2
    code = torch.bucketize(size, middle)  # (a size in the middle: the lower one)
    tie = code < len(middle)
    tie &= size == middle[code.clamp(max=len(middle) - 1)]
    code = torch.where(tie & (code % 2 == 1), code + 1, code)
    code = code + (1 << (bits - 1)) * torch.signbit(x)
    code = torch.where(none[..., None], 0, code).flatten(-2)
    return code.to(torch.uint8), torch.where(none, 255, exponent + 127).to(torch.uint8)


def packed(code, bits):
    return code if bits == 8 else code[..., 0::2] + 16 * code[..., 1::2]


def decode(code, scales, d, bits):
    """float64 values; NaN for a scale of 255."""
    scale = torch.where(scales == 255, math.nan, power(scales.long() - 127))
    return (numbers(bits)[code.long()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)[..., :d]
