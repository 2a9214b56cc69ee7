"""What goes into attention and where its keys are kept: the operators that are timed.

A case is a dict of plain values whose "path" names the operator:

  rotate   queries and keys of every head normalised and turned by their position (along one axis or several), one pass
  train    the same forward and backward, gradients of the norms' weights included
  store    keys and values written to a cache of 8 or 4 bits in pages, and what was written read back
  load     a stretch of such a cache read back
  attend   the nodes of a tree of drafted tokens (or one token) against such a cache

listed() holds calls of each kind of use, draw() gives others of the same ranges.  Positions, lengths and trees follow
from the case alone, values from the seed.

The cache: a row (slot, key head) of d columns, padded with zeros to a multiple of 32, is kept as blocks of 32 columns.  A block has
a scale 2^(byte - 127) and 32 codes: 4 bits, the numbers 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives (a sign, two bits of exponent, one of
fraction; column 2 j in the low half of byte j), or 8 bits (a sign, four bits of exponent, three of fraction, 448 at most).
The scale is the smallest power of two that leaves no element further than half of the largest step above the largest number:
the largest magnitude over the scale is at most 7 (4 bits) or 464 (8 bits).
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_BLOCK = 32
_EPS = 1e-6


# ---------------------------------------------------------------- the cases
def _rotate_case(path, dtype, b, hq, hkv, n, d, pairs, axes=1, interleaved=False, norm=True, far=0):
    """pairs: columns that turn, two by two; far: the position of a sequence's first token is up to this."""
    return {"path": path, "dtype": dtype, "b": b, "hq": hq, "hkv": hkv, "n": n, "d": d, "pairs": pairs, "axes": axes,
            "interleaved": interleaved, "norm": norm, "far": far}


def _cache_case(path, dtype, bits, b, hkv, n, longest, d, page):
    """n tokens a sequence, the last of them at slot longest - 1 of the longest one."""
    return {"path": path, "dtype": dtype, "bits": bits, "b": b, "hkv": hkv, "n": n, "longest": longest, "d": d, "page": page}


def _attend_case(dtype, bits, b, hq, hkv, nodes, longest, d, page, cap=0.0, bias=False):
    return {"path": "attend", "dtype": dtype, "bits": bits, "b": b, "hq": hq, "hkv": hkv, "nodes": nodes, "longest": longest, "d": d,
            "page": page, "cap": cap, "bias": bias}


def listed():
    return [
        # the queries and keys of a batch of prompts, views of what one product left
        dict(_rotate_case("rotate", "bf16", 4, 32, 8, 4096, 128, 64), name="prompt_rotate"),
        # the next token of every sequence, far into its text: latency
        dict(_rotate_case("rotate", "bf16", 32, 32, 8, 1, 128, 64, far=1000000), name="token_rotate"),
        # a clip of video: time, height and width turn shares of the columns of their own, no norms
        dict(_rotate_case("rotate", "bf16", 1, 16, 16, 6001, 72, 36, axes=3, interleaved=True, norm=False), name="video_rotate"),
        # a training step over packed documents
        dict(_rotate_case("train", "bf16", 2, 16, 4, 2048, 128, 64), name="train_rotate"),
        # a small f32 model of images, a part of the columns turned by row and column
        dict(_rotate_case("train", "f32", 3, 3, 3, 257, 64, 24, axes=2), name="train_images"),
        # prompts into the cache, and what it holds of them
        dict(_cache_case("store", "bf16", 4, 4, 8, 4096, 4096, 128, 64), name="store_prompts"),
        # one token of every sequence into the cache: latency
        dict(_cache_case("store", "bf16", 8, 32, 8, 1, 2000, 128, 16), name="store_tokens"),
        # a long cache read back, for a program that computes with it elsewhere
        dict(_cache_case("load", "bf16", 4, 8, 8, 8192, 8192, 128, 64), name="load_long"),
        # one new token of every sequence of a batch
        dict(_attend_case("bf16", 4, 32, 32, 8, 1, 8192, 128, 64), name="token_4bit"),
        # a tree of drafted tokens for every sequence, small pages, capped scores
        dict(_attend_case("bf16", 4, 8, 32, 8, 48, 4096, 128, 16, cap=50.0), name="draft_4bit"),
        # one token of two very long sequences, 8 bits: the work is split over the keys
        dict(_attend_case("bf16", 8, 2, 16, 2, 1, 65536, 128, 256), name="token_8bit"),
        # one token of one short sequence in f32: latency
        dict(_attend_case("f32", 4, 1, 8, 8, 1, 200, 64, 256, bias=True), name="single_4bit"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng, most):
    hkv = _spread(rng, 1, most)
    return hkv * rng.choice([1, 1, 2, 3, 4, 8]), hkv


def _head_size(rng):
    return rng.choice([64, 128, 64, 128, 8 * rng.randint(4, 16)])


def _drawn(rng):
    path = rng.choice(["rotate", "rotate", "train", "store", "load", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    d = _head_size(rng)
    if path in ("rotate", "train"):
        hq, hkv = _heads(rng, 16)
        pairs = rng.choice([d // 2, d // 2, d // 4, rng.randint(1, d // 2)])
        return _rotate_case(path, dtype, _spread(rng, 1, 32), hq, hkv, _spread(rng, 1, 8192), d, pairs, rng.choice([1, 1, 2, 3]),
                            rng.random() < 0.4, rng.random() < 0.7, rng.choice([0, 0, 1000, 1000000]))
    bits, page = rng.choice([4, 4, 8]), rng.choice([16, 64, 256, rng.randint(5, 100)])
    if path == "attend":
        hq, hkv = _heads(rng, 16)
        nodes = 1 if rng.random() < 0.5 else _spread(rng, 2, 64)
        return _attend_case(dtype, bits, _spread(rng, 1, 64), hq, hkv, nodes, _spread(rng, 1, 32768), d, page, rng.choice([0.0, 0.0, 30.0, 50.0]),
                            rng.random() < 0.3)
    longest = _spread(rng, 1, 16384)
    n = min(longest, 1 if rng.random() < 0.3 else _spread(rng, 1, 16384))
    return _cache_case(path, dtype, bits, _spread(rng, 1, 64), _spread(rng, 1, 16), n, longest, d, page)


def _affordable(case):
    """No more than the largest listed case: matrix work at the rate of its type, memory, and what the plain form holds."""
    w = work(case)
    if w["flops"] / (1.2e15 if case["dtype"] == "bf16" else 1.2e14) + w["bytes"] / 4e12 > 8.5e-5:
        return False
    if "hkv" in case and "longest" in case and case["b"] * case["hkv"] * case["longest"] * case["d"] > 2 ** 28:
        return False
    return case["path"] != "attend" or case["b"] * case["hq"] * case["nodes"] * case["longest"] <= 2 ** 26


def draw(rng):
    while True:
        case = _drawn(rng)
        if _affordable(case):
            return case


# ---------------------------------------------------------------- what follows from a case: positions, lengths, trees
def _layout(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _positions(case):
    """[axes, b, n]: one axis counts the tokens of a document, two are row and column of an image, three time, row and column."""
    rng, n, axes = _layout(case), case["n"], case["axes"]
    result = [[], [], []][:axes]
    for _ in range(case["b"]):
        first = rng.randint(0, case["far"])
        if axes == 1:
            row, at = [], first
            for _ in range(n):
                row.append(at)
                at = 0 if rng.random() < 0.002 else at + 1
            result[0].append(row)
            continue
        width = max(1, int(math.sqrt(n if axes == 2 else n ** (2 / 3))))
        if axes == 3:
            result[0].append([first + t // (width * width) for t in range(n)])
        result[-2].append([t // width % width if axes == 3 else first + t // width for t in range(n)])
        result[-1].append([t % width for t in range(n)])
    return result


def _axis_of(case):
    """The axis that a pair of columns turns by: shares in order, the first the smallest."""
    pairs, axes = case["pairs"], case["axes"]
    first = pairs // axes if axes < 3 else pairs // 4
    rest = pairs - first
    second = rest // (axes - 1) if axes > 1 else 0
    return [0] * (pairs if axes == 1 else first) + [1] * second + [2] * (rest - second if axes == 3 else 0)


def _lengths(case):
    """Slots before the nodes (attend), or after the tokens (store, load)."""
    rng, longest = _layout(case), case["longest"]
    least = max(1, longest // 8, case.get("n", 1) if case["path"] == "store" and case["n"] == 1 else 1)
    return [longest if s == 0 else _spread(rng, least, longest) for s in range(case["b"])]


def _first_and_counts(case):
    """Of every sequence the first slot that is written or read, and how many."""
    counts = [min(case["n"], length) for length in _lengths(case)]
    return [length - count for length, count in zip(_lengths(case), counts)], counts


def _trees(case):
    """Bit u of a node's word: the node sees node u (its ancestors and itself; a node comes after its parent)."""
    rng = _layout(case)
    words = []
    for _ in range(case["b"]):
        seen = []
        for t in range(case["nodes"]):
            seen.append((seen[rng.randrange(t)] if t else 0) | (1 << t))
        words.append([w - (1 << 64) if w >> 63 else w for w in seen])
    return words


def _pages(case, slots):
    """Pages per sequence, and for every sequence its pages in an order that is not theirs in memory."""
    rng = _layout(case)
    per = -(-slots // case["page"])
    order = list(range(case["b"] * per))
    rng.shuffle(order)
    return per, [order[s * per:(s + 1) * per] for s in range(case["b"])]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)

    state = {"case": case}
    b, hkv, d = case["b"], case["hkv"], case["d"]
    if case["path"] in ("rotate", "train"):
        hq, n, pairs = case["hq"], case["n"], case["pairs"]
        # queries, keys and values as one product leaves them
        joint = normal(b, n, hq + 2 * hkv, d, scale=2.0)
        positions = torch.tensor(_positions(case), dtype=torch.int32, device=device)
        base = 1e4 if case["axes"] > 1 else 1e6
        state.update(q=joint[:, :, :hq].transpose(1, 2), k=joint[:, :, hq:hq + hkv].transpose(1, 2),
                     positions=positions if case["axes"] > 1 else positions[0],
                     axes=torch.tensor(_axis_of(case), dtype=torch.int32, device=device) if case["axes"] > 1 else None,
                     frequencies=(base ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)).float())
        for name in ("q_weight", "k_weight"):
            state[name] = (1.0 + 0.3 * torch.randn(d, generator=gen, device=device)).to(dtype) if case["norm"] else None
        if case["path"] == "train":
            state.update(grad_q=normal(b, hq, n, d), grad_k=normal(b, hkv, n, d))
        return state

    page, bits = case["page"], case["bits"]
    slots = case["longest"] + case.get("nodes", 0)
    per, table = _pages(case, slots)
    state.update(per=per, table=torch.tensor(table, dtype=torch.int32, device=device))
    cache = {}
    for name in ("k", "v"):
        if case["path"] == "store":
            shape = (b * per, hkv, page)
            codes = torch.zeros((*shape, _columns(d) * bits // 8), dtype=torch.uint8, device=device)
            scales = torch.zeros((*shape, _columns(d) // _BLOCK), dtype=torch.uint8, device=device)
            # (a channel that is larger than the others, as keys have them)
            state[name] = normal(b, case["n"], hkv, d).transpose(1, 2)
            state[name][..., 3] *= 6
        else:
            values = torch.randn((b * per, hkv, page, d), generator=gen, device=device)
            values[..., 3] *= 3
            codes, scales = _encode(values, bits)
            del values
        cache[name], cache[f"{name}_scales"] = codes, scales
    state["cache"] = cache
    if own:
        from i_amd.quantised import QuantisedCache

        state["handle"] = QuantisedCache(**cache, d=d, bits=bits)
    if case["path"] == "attend":
        hq = case["hq"]
        state.update(q=normal(b, hq, case["nodes"], d, scale=1.5), scale=d ** -0.5, slopes=_slopes(hq, device) if case["bias"] else None,
                     lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=device),
                     visible=torch.tensor(_trees(case), dtype=torch.int64, device=device))
        return state
    state["first"], state["counts"] = (torch.tensor(x, dtype=torch.int32, device=device) for x in _first_and_counts(case))
    return state


def _columns(d):
    return -(-d // _BLOCK) * _BLOCK


def _slopes(heads, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=device)


# ---------------------------------------------------------------- one pass
def run(state):
    path = state["case"]["path"]
    return (_OWN if own else _PLAIN)[path](state)


def _turning(state):
    return {"positions": state["positions"], "frequencies": state["frequencies"], "axes": state["axes"], "interleaved": state["case"]["interleaved"],
            "q_weight": state["q_weight"], "k_weight": state["k_weight"], "eps": _EPS}


def _own_rotate(state):
    from i_amd.rotary import rotate

    return rotate(state["q"], state["k"], **_turning(state))


def _own_train(state):
    from i_amd.rotary import rotate, rotate_backward

    turning = _turning(state)
    outputs = rotate(state["q"], state["k"], **turning)
    grads = rotate_backward(state["grad_q"], state["grad_k"], state["q"], state["k"], **turning)
    return outputs + tuple(g for g in grads if g is not None)


def _own_store(state):
    from i_amd.quantised import store

    store(state["handle"], state["k"], state["v"], first=state["first"], counts=state["counts"], table=state["table"])
    return _own_load(state)


def _own_load(state):
    from i_amd.quantised import load

    case = state["case"]
    return load(state["handle"], case["n"], first=state["first"], counts=state["counts"], table=state["table"], dtype=_TYPES[case["dtype"]])


def _own_attend(state):
    from i_amd.quantised import tree_attention

    return tree_attention(state["q"], state["handle"], state["lengths"], table=state["table"], visible=state["visible"], scale=state["scale"],
                          cap=state["case"]["cap"], slopes=state["slopes"])


_OWN = {"rotate": _own_rotate, "train": _own_train, "store": _own_store, "load": _own_load, "attend": _own_attend}


# ---------------------------------------------------------------- the plain form
def _turns(state):
    """Cosine and sine of every token's pairs, [b, 1, n, pairs].  (Angles in 64 bits: positions reach millions.)"""
    positions = state["positions"] if state["axes"] is not None else state["positions"][None]
    of_pair = positions[state["axes"].long()] if state["axes"] is not None else positions.expand(state["case"]["pairs"], -1, -1)
    angle = of_pair.permute(1, 2, 0).double() * state["frequencies"].double()
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _pairs_of(x, case):
    """The two columns of every pair, and the columns that do not turn."""
    pairs = case["pairs"]
    if case["interleaved"]:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], x[..., 2 * pairs:]
    return x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]


def _turned(x, cos, sin, case):
    first, second, rest = _pairs_of(x, case)
    first, second = first * cos - second * sin, second * cos + first * sin
    if case["interleaved"]:
        return torch.cat([torch.stack([first, second], -1).flatten(-2), rest], -1)
    return torch.cat([first, second, rest], -1)


def _plain_rotate(state):
    case = state["case"]
    cos, sin = _turns(state)
    outputs = []
    for name in ("q", "k"):
        x = state[name].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * state[f"{name}_weight"].float()
        outputs.append(_turned(x, cos, sin, case).to(state[name].dtype))
    return tuple(outputs)


def _plain_train(state):
    case = state["case"]
    cos, sin = _turns(state)
    grads, weights = [], []
    for name in ("q", "k"):
        g = _turned(state[f"grad_{name}"].float(), cos, -sin, case)
        if case["norm"]:
            x, weight = state[name].float(), state[f"{name}_weight"].float()
            inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
            x = x * inverse
            weights.append((g * x).sum((0, 1, 2), dtype=torch.float64).to(state[f"{name}_weight"].dtype))
            g = g * weight
            g = (g - x * (g * x).mean(-1, keepdim=True)) * inverse
        grads.append(g.to(state[name].dtype))
    return (*_plain_rotate(state), *grads, *weights)


def _power(exponent):
    """2^exponent in 32 bits, from its bits: exact on any device."""
    return (exponent.int() + 127 << 23).view(torch.float32)


def _encode(values, bits):
    """Codes and scales of rows of d columns."""
    shape, d = values.shape[:-1], values.shape[-1]
    x = torch.zeros((*shape, _columns(d)), dtype=torch.float32, device=values.device)
    x[..., :d] = values
    x = x.view(*shape, -1, _BLOCK)
    top = x.abs().amax(-1)
    fraction, exponent = torch.frexp(top)  # fraction 1/2 .. 1: half of what the rule compares with
    if bits == 4:
        byte = exponent - 1 - 2 + (fraction > 0.875) + 127
        least = 2
    else:
        byte = exponent - 1 - 8 + (fraction > 0.90625) + 127
        least = 10
    byte = torch.where(top > 0, byte.clamp(min=least), least)
    size = (x * _power(127 - byte)[..., None]).abs()
    # halves go to the even code
    if bits == 8:
        size = size.clamp(max=448)
        octave = (torch.frexp(size).exponent - 1).clamp(min=-6)
        steps = (size * _power(3 - octave)).round()  # 0 .. 8 in the lowest octave, 8 .. 16 in the others
        codes = (octave + 6) * 8 + steps.int()
    else:
        size = size.clamp(max=6)
        # steps of 1/2 below 2, of 1 below 4, of 2 above
        codes = torch.where(size < 2, (size * 2).round(), torch.where(size < 4, size.round() + 2, (size / 2).round() + 4)).int()
    codes = (codes + (1 << bits - 1) * torch.signbit(x)).to(torch.uint8)
    if bits == 4:
        codes = codes[..., 0::2] + 16 * codes[..., 1::2]
    return codes.flatten(-2), byte.to(torch.uint8)


def _decode(codes, scales, d, bits):
    """The values of rows, in 32 bits."""
    code = codes.int() if bits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    fraction, bias = (3, 7) if bits == 8 else (1, 1)
    size = code & (1 << bits - 1) - 1
    octave = (size >> fraction).clamp(min=1)
    steps = size - (octave - 1 << fraction)
    x = steps * _power(octave - bias - fraction)
    x = torch.where(code >> bits - 1 == 1, -x, x).view(*scales.shape, _BLOCK)
    return (x * _power(scales.int() - 127)[..., None]).flatten(-2)[..., :d]


def _slots_of(state):
    """Page, slot in it and validity of token t of sequence s, [b, n]."""
    case = state["case"]
    at = torch.arange(case["n"], device=state["table"].device)
    slot = state["first"][:, None] + at
    live = at < state["counts"][:, None]
    slot = torch.where(live, slot, 0).long()
    return torch.gather(state["table"].long(), 1, slot // case["page"]), slot % case["page"], live


def _plain_store(state):
    page, slot, live = _slots_of(state)
    cache, bits = state["cache"], state["case"]["bits"]
    page_at, slot_at = page[live], slot[live]
    for name in ("k", "v"):
        codes, scales = _encode(state[name].transpose(1, 2)[live].float(), bits)
        cache[name][page_at, :, slot_at] = codes
        cache[f"{name}_scales"][page_at, :, slot_at] = scales
    return _plain_load(state)


def _plain_load(state):
    case, cache = state["case"], state["cache"]
    page, slot, live = _slots_of(state)
    outputs = []
    for name in ("k", "v"):
        values = _decode(cache[name][page, :, slot], cache[f"{name}_scales"][page, :, slot], case["d"], case["bits"])
        values = torch.where(live[:, :, None, None], values, torch.zeros_like(values))
        outputs.append(values.transpose(1, 2).to(_TYPES[case["dtype"]]))
    return tuple(outputs)


def _plain_attend(state):
    case, cache = state["case"], state["cache"]
    hq, hkv, nodes, d, group = case["hq"], case["hkv"], case["nodes"], case["d"], case["hq"] // case["hkv"]
    slots = state["per"] * case["page"]
    at = torch.arange(slots, device=state["q"].device)
    bit = torch.arange(nodes, device=at.device)
    outputs, logs = [], []
    for s in range(case["b"]):
        pages = state["table"][s].long()
        k, v = (_decode(cache[name][pages], cache[f"{name}_scales"][pages], d, case["bits"]).transpose(0, 1).reshape(hkv, slots, d) for name in ("k", "v"))
        length = state["lengths"][s]
        node = at - length
        sees = (state["visible"][s][:, None] >> bit[None, :]) & 1
        depth = sees.sum(1) - 1
        of_tree = (node >= 0) & (node < nodes)
        node = node.clamp(0, nodes - 1)
        shown = (at < length)[None, :] | (of_tree[None, :] & (sees[:, node] == 1))
        scores = state["q"][s].float().reshape(hkv, group * nodes, d) @ k.transpose(1, 2) * state["scale"]
        if case["cap"]:
            scores = torch.tanh(scores / case["cap"]) * case["cap"]
        scores = scores.view(hkv, group, nodes, slots)
        if state["slopes"] is not None:
            where = torch.where(at < length, at, length + depth[node])
            scores = scores - state["slopes"].view(hkv, group, 1, 1) * ((length + depth)[:, None] - where[None, :]).abs().float()
        scores = scores.masked_fill(~shown, -math.inf).view(hkv, group * nodes, slots)
        top = scores.amax(-1, keepdim=True)
        e = torch.exp(scores - top)
        total = e.sum(-1, keepdim=True)
        outputs.append((e / total @ v).view(hq, nodes, d))
        logs.append((top + torch.log(total)).view(hq, nodes))
    return torch.stack(outputs).to(state["q"].dtype), torch.stack(logs)


_PLAIN = {"rotate": _plain_rotate, "train": _plain_train, "store": _plain_store, "load": _plain_load, "attend": _plain_attend}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["path"] in ("rotate", "train"):
        return _exact_rotate(state)
    if case["path"] == "attend":
        return _exact_attend(state)
    return _exact_cache(state)


def _exact_rotate(state):
    """A pair is a complex number that is multiplied by e^(i angle); gradients by automatic differentiation."""
    case = state["case"]
    pairs, b, n = case["pairs"], case["b"], case["n"]
    positions = state["positions"].view(case["axes"], b, n)
    angle = torch.empty((b, n, pairs), dtype=torch.float64, device=positions.device)
    for j, axis in enumerate(_axis_of(case)):
        angle[:, :, j] = positions[axis].double() * state["frequencies"][j].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    column = torch.arange(pairs, device=angle.device)
    first, second = (2 * column, 2 * column + 1) if case["interleaved"] else (column, column + pairs)
    train, outputs, grads, weights = case["path"] == "train", [], [], []
    for name in ("q", "k"):
        x = state[name].double().requires_grad_(train)
        y, leaves = x, [x]
        if case["norm"]:
            weight = state[f"{name}_weight"].double().requires_grad_(train)
            leaves.append(weight)
            y = y / (y.square().sum(-1, keepdim=True) / case["d"] + _EPS).sqrt() * weight
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)
        outputs.append(y.detach())
        if train:
            found = torch.autograd.grad(y, leaves, state[f"grad_{name}"].double())
            grads.append(found[0])
            weights += found[1:]
    return (*outputs, *grads, *weights)


def _exact_power(exponent):
    return (exponent.long() + 1023 << 52).view(torch.float64)


def _exact_numbers(bits, device):
    """The number of every code."""
    numbers = []
    for code in range(1 << bits):
        fraction_bits, bias = (1, 1) if bits == 4 else (3, 7)
        size = code & ((1 << (bits - 1)) - 1)
        exponent, fraction = size >> fraction_bits, (size & ((1 << fraction_bits) - 1)) / (1 << fraction_bits)
        number = 2.0 ** (exponent - bias) * (1 + fraction) if exponent else 2.0 ** (1 - bias) * fraction
        numbers.append(-number if code >> (bits - 1) else number)
    if bits == 8:
        numbers[127], numbers[255] = math.nan, math.nan
    return torch.tensor(numbers, dtype=torch.float64, device=device)


def _exact_values(codes, scales, d, bits):
    numbers = _exact_numbers(bits, codes.device)
    codes = codes.long()
    if bits == 4:
        codes = torch.stack([codes % 16, codes // 16], -1).flatten(-2)
    scale = _exact_power(scales.long() - 127)
    return (numbers[codes].unflatten(-1, (-1, _BLOCK)) * scale[..., None]).flatten(-2)[..., :d]


def _exact_kept(values, bits):
    """What rows of values become: for every element the nearest number, of two equally near ones the one whose code is even."""
    numbers = _exact_numbers(bits, values.device)
    count = 8 if bits == 4 else 127
    numbers = numbers[:count]
    most, beyond = (6.0, 7.0) if bits == 4 else (448.0, 464.0)
    d = values.shape[-1]
    result = torch.zeros_like(values)
    for c0 in range(0, d, _BLOCK):
        x = values[..., c0:c0 + _BLOCK]
        top = x.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0) / beyond)) - 1
        for _ in range(3):
            power = torch.where(top > beyond * _exact_power(power), power + 1, power)
        scale = _exact_power(power.clamp(min=-125 if bits == 4 else -117))
        size = (x.abs() / scale).clamp(max=most)
        above = torch.searchsorted(numbers, size.contiguous()).clamp(max=count - 1)
        below = (above - 1).clamp(min=0)
        up, down = numbers[above] - size, size - numbers[below]
        code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
        result[..., c0:c0 + _BLOCK] = torch.copysign(numbers[code] * scale, x)
    return result


def _exact_cache(state):
    case, cache = state["case"], state["cache"]
    first, counts, table = (state[name].tolist() for name in ("first", "counts", "table"))
    outputs = []
    for name in ("k", "v"):
        out = torch.zeros((case["b"], case["hkv"], case["n"], case["d"]), dtype=torch.float64, device=cache[name].device)
        for s, (at, count) in enumerate(zip(first, counts)):
            if case["path"] == "store":
                out[s, :, :count] = _exact_kept(state[name][s, :, :count].double(), case["bits"])
                continue
            slot = torch.arange(at, at + count, device=out.device)
            page = torch.tensor(table[s], device=out.device)[slot // case["page"]]
            codes, scales = (cache[n][page, :, slot % case["page"]].transpose(0, 1) for n in (name, f"{name}_scales"))
            out[s, :, :count] = _exact_values(codes, scales, case["d"], case["bits"])
        outputs.append(out)
    return tuple(outputs)


def _exact_attend(state):
    case, cache = state["case"], state["cache"]
    hq, nodes, d, page, group = case["hq"], case["nodes"], case["d"], case["page"], case["hq"] // case["hkv"]
    device = state["q"].device
    o = torch.zeros(state["q"].shape, dtype=torch.float64, device=device)
    lse = torch.zeros(o.shape[:3], dtype=torch.float64, device=device)
    table, lengths, words = state["table"].tolist(), state["lengths"].tolist(), state["visible"].tolist()
    for s in range(case["b"]):
        total = lengths[s] + nodes
        slot = torch.arange(total, device=device)
        pages = torch.tensor(table[s], device=device)[slot // page]
        hidden = torch.tensor([[not (w >> u) & 1 for u in range(nodes)] for w in words[s]], device=device)
        hidden = torch.cat([torch.zeros((nodes, lengths[s]), dtype=torch.bool, device=device), hidden], 1)
        depth = torch.tensor([bin(w & (2 ** 64 - 1)).count("1") - 1 for w in words[s]], device=device)
        position = torch.cat([slot[:lengths[s]], lengths[s] + depth])
        distance = (lengths[s] + depth[:, None] - position[None, :]).abs().double()
        for g in range(case["hkv"]):
            keys, values = (_exact_values(cache[name][pages, g, slot % page], cache[f"{name}_scales"][pages, g, slot % page], d, case["bits"]) for name in ("k", "v"))
            for h in range(g * group, (g + 1) * group):
                logits = torch.einsum("id,jd->ij", state["q"][s, h].double(), keys).mul(state["scale"])
                if case["cap"]:
                    logits = case["cap"] * torch.tanh(logits / case["cap"])
                if state["slopes"] is not None:
                    logits = logits - float(state["slopes"][h]) * distance
                logits = logits.masked_fill(hidden, -math.inf)
                o[s, h], lse[s, h] = logits.softmax(1) @ values, logits.logsumexp(1)
    return o, lse


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e, d, b, hkv = _BYTES[case["dtype"]], case["d"], case["b"], case["hkv"]
    if case["path"] in ("rotate", "train"):
        rows = b * (case["hq"] + hkv) * case["n"]
        held = 4 * b * case["n"] * case["axes"] + 4 * case["pairs"] + (2 * e * d if case["norm"] else 0)
        per = 6 * case["pairs"] + (4 * d if case["norm"] else 0)
        if case["path"] == "rotate":
            return {"bytes": 2 * e * d * rows + held, "flops": per * rows}
        # inputs (of the norms' gradients as well) and gradients in, outputs and gradients out
        return {"bytes": 4 * e * d * rows + held + (2 * e * d if case["norm"] else 0), "flops": 3 * per * rows}
    row = _columns(d) * case["bits"] // 8 + _columns(d) // _BLOCK
    if case["path"] == "attend":
        hq, nodes = case["hq"], case["nodes"]
        tokens = sum(_lengths(case)) + b * nodes
        seen = nodes * sum(_lengths(case)) + sum(bin(w & (2 ** 64 - 1)).count("1") for words in _trees(case) for w in words)
        return {"bytes": 2 * row * hkv * tokens + 2 * e * d * b * hq * nodes + 4 * b * hq * nodes, "flops": 4 * d * hq * seen}
    tokens, out = sum(_first_and_counts(case)[1]) * hkv, 2 * e * d * b * hkv * case["n"]
    if case["path"] == "load":
        return {"bytes": 2 * row * tokens + out, "flops": 0}
    return {"bytes": 2 * e * d * tokens + 2 * row * tokens + out, "flops": 0}
