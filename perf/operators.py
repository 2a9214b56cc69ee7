"""Attention with masks and what serves and trains with it: the operators that are timed.

A case is a dict of plain values whose "path" names the operator:

  attention  forward: causal, document, prefix and window masks, capped scores, a bias that grows with distance
  train      forward and backward of the same
  weights    the attention weight that every key of a prompt received, summed over its queries
  tree       the nodes of a tree of drafted tokens (or one token) against a cache in pages
  evict      the cache entries of least accumulated weight leave, the others move together

listed() holds calls of each kind of use, draw() gives others of the same ranges.  Masks, lengths and trees follow
from the case alone, values from the seed.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}


# ---------------------------------------------------------------- the cases
def _dense(path, dtype, b, hq, hkv, n, d, mask, cap=0.0, bias=False, rows_first=True):
    """Queries and keys of the same tokens; rows_first: stored [b, n, h, d], as a projection leaves them."""
    return {"path": path, "dtype": dtype, "b": b, "hq": hq, "hkv": hkv, "n": n, "d": d, "mask": mask, "cap": cap, "bias": bias,
            "rows_first": rows_first}


def _tree_case(dtype, b, hq, hkv, nodes, longest, d, page, cap=0.0, bias=False, accumulate=False):
    return {"path": "tree", "dtype": dtype, "b": b, "hq": hq, "hkv": hkv, "nodes": nodes, "longest": longest, "d": d, "page": page,
            "cap": cap, "bias": bias, "accumulate": accumulate}


def _evict_case(dtype, b, hkv, longest, keep, recent, d, page):
    return {"path": "evict", "dtype": dtype, "b": b, "hkv": hkv, "longest": longest, "keep": keep, "recent": recent, "d": d, "page": page}


def listed():
    return [
        # a batch of prompts through a layer whose scores are capped: the largest call
        dict(_dense("attention", "bf16", 4, 32, 8, 4096, 128, "causal", cap=50.0), name="prompt_capped"),
        # sequences of uneven length packed into one row, a head size no tile divides, a bias by distance
        dict(_dense("attention", "bf16", 1, 16, 16, 6001, 80, "documents", bias=True), name="packed_documents"),
        # one short prompt in f32 whose first part sees itself whole: launches and the way into the library count
        dict(_dense("attention", "f32", 1, 4, 4, 333, 64, "prefix", rows_first=False), name="prefix_small"),
        # a training step's attention over packed documents
        dict(_dense("train", "bf16", 2, 16, 4, 2048, 128, "documents", cap=30.0), name="train_documents"),
        # a small f32 model with a sliding window and a bias by distance
        dict(_dense("train", "f32", 1, 3, 3, 257, 64, "window", bias=True, rows_first=False), name="train_small"),
        # what each key of a prompt received, before the cache is cut
        dict(_dense("weights", "bf16", 2, 32, 8, 4096, 128, "causal"), name="weights_prompt"),
        # the same for one f32 prompt of odd length
        dict(_dense("weights", "f32", 1, 6, 2, 777, 64, "prefix", rows_first=False), name="weights_odd"),
        # one new token of every sequence, the weights of the cache kept up to date
        dict(_tree_case("bf16", 32, 32, 8, 1, 8192, 128, 64, accumulate=True), name="decode"),
        # a tree of drafted tokens for every sequence, small pages, capped scores
        dict(_tree_case("bf16", 8, 32, 8, 48, 4096, 128, 16, cap=50.0), name="draft_tree"),
        # one token of one short sequence: latency
        dict(_tree_case("f32", 1, 8, 8, 1, 200, 64, 256, bias=True), name="single_token"),
        # caches of a batch cut to a quarter
        dict(_evict_case("bf16", 16, 8, 8192, 2048, 256, 128, 64), name="evict_batch"),
        # one short cache, odd numbers
        dict(_evict_case("f32", 1, 4, 500, 101, 17, 64, 512), name="evict_small"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng, most):
    hkv = _spread(rng, 1, most)
    return hkv * rng.choice([1, 1, 2, 3, 4, 8]), hkv


def _head_size(rng):
    return rng.choice([64, 128, 64, 128, 8 * rng.randint(4, 16)])


def _drawn(rng):
    path = rng.choice(["attention", "attention", "train", "weights", "tree", "tree", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    if path == "tree":
        hq, hkv = _heads(rng, 16)
        nodes = 1 if rng.random() < 0.4 else _spread(rng, 2, 64)
        longest = _spread(rng, 1, 16384)
        return _tree_case(dtype, _spread(rng, 1, 64), hq, hkv, nodes, longest, _head_size(rng), rng.choice([16, 64, 256, rng.randint(5, 100)]),
                          cap, rng.random() < 0.3, rng.random() < 0.4)
    if path == "evict":
        longest = _spread(rng, 2, 32768)
        keep = max(1, int(longest * rng.uniform(0.1, 0.9)))
        return _evict_case(dtype, _spread(rng, 1, 32), _spread(rng, 1, 16), longest, keep, int(keep * rng.uniform(0.0, 0.5)), _head_size(rng),
                           rng.choice([16, 64, 256, rng.randint(5, 100)]))
    hq, hkv = _heads(rng, 16)
    n = _spread(rng, 1, 8192)
    mask = rng.choice(["none", "causal", "causal", "documents", "whole_documents", "prefix", "window"])
    return _dense(path, dtype, _spread(rng, 1, 8), hq, hkv, n, _head_size(rng), mask, cap, rng.random() < 0.3, rng.random() < 0.6)


def _affordable(case):
    """No more than the largest listed case: matrix work at the rate of its type, memory, and the plain form's passes over the pairs."""
    w = work(case)
    seconds = w["flops"] / (1.2e15 if case["dtype"] == "bf16" else 1.2e14) + w["bytes"] / 4e12
    if case["path"] in ("attention", "train", "weights") and case["b"] * case["hq"] * case["n"] ** 2 > 4 * 32 * 4096 ** 2:
        return False
    if case["path"] == "tree" and case["b"] * case["hq"] * case["nodes"] * case["longest"] > 4 * 32 * 4096 ** 2 // 4:
        return False
    if case["path"] in ("tree", "evict") and 2 * case["b"] * case["hkv"] * case["longest"] * case["d"] * _BYTES[case["dtype"]] > 2 ** 32:
        return False
    return seconds < 5e-4 and 3072 not in case.values()


def draw(rng):
    while True:
        case = _drawn(rng)
        if _affordable(case):
            return case


# ---------------------------------------------------------------- what follows from a case: bounds, lengths, trees
def _layout(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _bounds(case):
    """Per sequence the first and the one-past-last visible key of every query, without what "causal" adds; None: no bound."""
    rng, n, b = _layout(case), case["n"], case["b"]
    mask = case["mask"]
    if mask in ("none", "causal"):
        return None, None
    first, last = [], []
    for _ in range(b):
        if mask in ("documents", "whole_documents"):
            at = 0
            lo, hi = [], []
            while at < n:
                length = min(n - at, _spread(rng, max(1, n // 40), max(2, n // 3)))
                lo += [at] * length
                hi += [at + length] * length
                at += length
            first.append(lo)
            last.append(hi)
        elif mask == "prefix":
            prefix = rng.randint(0, n)
            last.append([max(i + 1, prefix) for i in range(n)])
        else:
            width = _spread(rng, max(1, n // 16), max(2, n // 2))
            first.append([max(0, i + 1 - width) for i in range(n)])
    return first or None, (last or None) if mask != "documents" else None


def _causal(case):
    return case["mask"] in ("causal", "documents", "window")


def _pairs(case):
    """Visible (query, key) pairs of one head, all sequences."""
    first, last = _bounds(case)
    n, total = case["n"], 0
    for s in range(case["b"]):
        for i in range(n):
            lo = first[s][i] if first else 0
            hi = last[s][i] if last else n
            if _causal(case):
                hi = min(hi, i + 1)
            total += max(0, hi - lo)
    return total


def _lengths(case):
    rng = _layout(case)
    return [case["longest"] if s == 0 else _spread(rng, max(1, case["longest"] // 8), case["longest"]) for s in range(case["b"])]


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
    if case["path"] in ("attention", "train", "weights"):
        b, hq, hkv, n, d = (case[k] for k in ("b", "hq", "hkv", "n", "d"))

        def heads(h, scale=1.0):
            return normal(b, n, h, d, scale=scale).transpose(1, 2) if case["rows_first"] else normal(b, h, n, d, scale=scale)

        first, last = _bounds(case)
        # (queries with some spread, so that a softmax prefers some keys to others)
        state.update(q=heads(hq, 1.5), k=heads(hkv), v=heads(hkv), scale=d ** -0.5,
                     first=None if first is None else torch.tensor(first, dtype=torch.int32, device=device),
                     last=None if last is None else torch.tensor(last, dtype=torch.int32, device=device),
                     slopes=_slopes(hq, device) if case["bias"] else None)
        if case["path"] == "train":
            state["do"] = heads(hq)
        if case["path"] == "weights":
            # the forward pass of the prompt left these
            state["lse"] = torch.cat([_plain_scores(state, s)[0].logsumexp(-1) for s in range(b)]).view(b, hq, n)
        return state

    b, hkv, d, page = case["b"], case["hkv"], case["d"], case["page"]
    slots = case["longest"] + case.get("nodes", 0)
    per, table = _pages(case, slots)
    state.update(k=normal(b * per, hkv, page, d), v=normal(b * per, hkv, page, d), per=per,
                 table=torch.tensor(table, dtype=torch.int32, device=device),
                 lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=device))
    if case["path"] == "tree":
        hq = case["hq"]
        state.update(q=normal(b, hq, case["nodes"], d, scale=1.5), scale=d ** -0.5, slopes=_slopes(hq, device) if case["bias"] else None,
                     visible=torch.tensor(_trees(case), dtype=torch.int64, device=device))
        if case["accumulate"]:
            state["weights"] = torch.rand((b, hkv, per * page), generator=gen, device=device) ** 4
            state["weights_out"] = torch.zeros_like(state["weights"])
        return state
    # a few keys hold most of the weight, as in attention
    state["weights"] = torch.rand((b, hkv, per * page), generator=gen, device=device) ** 8 * 30.0
    keep = case["keep"]
    per_out = -(-keep // page)
    zeros = lambda *shape, dtype: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
    # where a program keeps the shortened cache: dense pages, in order
    state["out"] = {"k": zeros(b * per_out, hkv, page, d, dtype=dtype), "v": zeros(b * per_out, hkv, page, d, dtype=dtype),
                    "weights": zeros(b, hkv, keep, dtype=torch.float32), "positions": zeros(b, hkv, keep, dtype=torch.int32),
                    "lengths": zeros(b, dtype=torch.int32)}
    state["table_out"] = torch.arange(b * per_out, dtype=torch.int32, device=device).view(b, per_out)
    return state


def _slopes(heads, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=device)


# ---------------------------------------------------------------- one pass
def run(state):
    path = state["case"]["path"]
    return (_OWN if own else _PLAIN)[path](state)


def _options(state):
    case = state["case"]
    return {"scale": state["scale"], "cap": case["cap"], "slopes": state["slopes"], "causal": _causal(case), "first": state["first"],
            "last": state["last"]}


def _own_attention(state):
    from i_amd.attention import attention

    return attention(state["q"], state["k"], state["v"], **_options(state))


def _own_train(state):
    from i_amd.attention import attention, attention_backward

    options = _options(state)
    o, lse = attention(state["q"], state["k"], state["v"], **options)
    return (o, lse) + attention_backward(state["do"], state["q"], state["k"], state["v"], o, lse, **options)


def _own_weights(state):
    from i_amd.attention import key_weights

    return key_weights(state["q"], state["k"], state["lse"], **_options(state))


def _own_tree(state):
    from i_amd.attention import tree_attention

    case = state["case"]
    kept = {"weights": state["weights"], "weights_out": state["weights_out"]} if case["accumulate"] else {}
    o, lse = tree_attention(state["q"], state["k"], state["v"], state["lengths"], table=state["table"], visible=state["visible"],
                            scale=state["scale"], cap=case["cap"], slopes=state["slopes"], **kept)
    return (o, lse, state["weights_out"]) if case["accumulate"] else (o, lse)


def _own_evict(state):
    from i_amd.attention import evict

    case = state["case"]
    kept = evict(state["k"], state["v"], state["weights"], state["lengths"], case["keep"], case["recent"], table=state["table"],
                 table_out=state["table_out"], out=tuple(state["out"].values()))
    return dict(zip(state["out"], kept))


_OWN = {"attention": _own_attention, "train": _own_train, "weights": _own_weights, "tree": _own_tree, "evict": _own_evict}


# ---------------------------------------------------------------- the plain form
def _plain_scores(state, s):
    """Scores of sequence s, [hkv, group * n, n], hidden ones at -inf; the capped scores over the cap; the mask."""
    case = state["case"]
    hkv, n, d, group = case["hkv"], case["n"], case["d"], case["hq"] // case["hkv"]
    q = state["q"][s].float().reshape(hkv, group * n, d)
    scores = q @ state["k"][s].float().transpose(1, 2) * state["scale"]
    bent = None
    if case["cap"]:
        bent = torch.tanh(scores / case["cap"])
        scores = bent * case["cap"]
    at = torch.arange(n, device=q.device)
    if state["slopes"] is not None:
        distance = (at[:, None] - at[None, :]).abs().float()
        scores = (scores.view(hkv, group, n, n) - state["slopes"].view(hkv, group, 1, 1) * distance).view(hkv, group * n, n)
    shown = torch.ones((n, n), dtype=torch.bool, device=q.device)
    if _causal(case):
        shown &= at[None, :] <= at[:, None]
    if state["first"] is not None:
        shown &= at[None, :] >= state["first"][s][:, None]
    if state["last"] is not None:
        shown &= at[None, :] < state["last"][s][:, None]
    scores = scores.view(hkv, group, n, n).masked_fill(~shown, -math.inf).view(hkv, group * n, n)
    return scores, bent


def _softmax(scores):
    """Probabilities and log of the sum; zeros where nothing is visible."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), (top + torch.log(total)).squeeze(-1)


def _plain_attention(state):
    case = state["case"]
    hq, n, d = case["hq"], case["n"], case["d"]
    outputs, logs = [], []
    for s in range(case["b"]):
        p, lse = _softmax(_plain_scores(state, s)[0])
        outputs.append((p @ state["v"][s].float()).view(hq, n, d))
        logs.append(lse.view(hq, n))
    return torch.stack(outputs).to(state["q"].dtype), torch.stack(logs)


def _plain_train(state):
    case = state["case"]
    hq, hkv, n, d, group = case["hq"], case["hkv"], case["n"], case["d"], case["hq"] // case["hkv"]
    results = [[], [], [], [], []]
    for s in range(case["b"]):
        scores, bent = _plain_scores(state, s)
        p, lse = _softmax(scores)
        q, k, v, do = (state[name][s].float() for name in ("q", "k", "v", "do"))
        q, do = q.reshape(hkv, group * n, d), do.reshape(hkv, group * n, d)
        o = p @ v
        ds = p * (do @ v.transpose(1, 2) - (do * o).sum(-1, keepdim=True))
        if bent is not None:
            ds = ds * (1.0 - bent * bent)
        ds = ds * state["scale"]
        for kept, value in zip(results, (o.view(hq, n, d), lse.view(hq, n), (ds @ k).view(hq, n, d), ds.transpose(1, 2) @ q, p.transpose(1, 2) @ do)):
            kept.append(value)
    o, lse, dq, dk, dv = (torch.stack(r) for r in results)
    dtype = state["q"].dtype
    return o.to(dtype), lse, dq.to(dtype), dk.to(dtype), dv.to(dtype)


def _plain_weights(state):
    case = state["case"]
    sums = []
    for s in range(case["b"]):
        scores, _ = _plain_scores(state, s)
        sums.append(torch.exp(scores - state["lse"][s].reshape(case["hkv"], -1, 1)).sum(1))
    return torch.stack(sums)


def _plain_tree(state):
    case = state["case"]
    hq, hkv, nodes, d, group = case["hq"], case["hkv"], case["nodes"], case["d"], case["hq"] // case["hkv"]
    slots = state["per"] * case["page"]
    at = torch.arange(slots, device=state["q"].device)
    bit = torch.arange(nodes, device=at.device)
    outputs, logs, weights = [], [], []
    for s in range(case["b"]):
        pages = state["table"][s].long()
        k = state["k"][pages].transpose(0, 1).reshape(hkv, slots, d).float()
        v = state["v"][pages].transpose(0, 1).reshape(hkv, slots, d).float()
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
        p, lse = _softmax(scores.masked_fill(~shown, -math.inf).view(hkv, group * nodes, slots))
        shown_at_all = (at < length + nodes)[None, :, None]
        outputs.append((p @ torch.where(shown_at_all, v, torch.zeros_like(v))).view(hq, nodes, d))
        logs.append(lse.view(hq, nodes))
        if case["accumulate"]:
            weights.append(state["weights"][s] + p.sum(1))
    o, lse = torch.stack(outputs).to(state["q"].dtype), torch.stack(logs)
    return (o, lse, torch.stack(weights)) if case["accumulate"] else (o, lse)


def _plain_evict(state):
    case, out = state["case"], state["out"]
    hkv, page, d, keep, recent = case["hkv"], case["page"], case["d"], case["keep"], case["recent"]
    slots, b = state["per"] * page, case["b"]
    at = torch.arange(slots, device=state["k"].device)
    length = state["lengths"].long()[:, None, None]
    # the recent ones first, then by weight; slots past the end last
    rank = torch.where(at >= length, -math.inf, torch.where(at >= length - recent, math.inf, state["weights"]))
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    held = length.clamp(max=keep)
    slot = torch.arange(keep, device=at.device)
    chosen = torch.sort(torch.where(slot < held, chosen, slots), dim=-1).values
    live = (slot < held).expand(b, hkv, keep)
    chosen = torch.where(live, chosen, 0)
    s, h = torch.arange(b, device=at.device)[:, None, None], torch.arange(hkv, device=at.device)[None, :, None]
    from_page, to_page = state["table"].long()[s, chosen // page], state["table_out"].long()[s, slot // page]
    result = {name: torch.zeros_like(t) for name, t in out.items()}
    zero = torch.zeros((), dtype=state["k"].dtype, device=at.device)
    for name in ("k", "v"):
        result[name][to_page, h, slot % page] = torch.where(live[..., None], state[name][from_page, h, chosen % page], zero)
    result["weights"] = torch.where(live, state["weights"].gather(-1, chosen), result["weights"])
    result["positions"] = torch.where(live, chosen, 0).int()
    result["lengths"] = held.view(b).int()
    return result


_PLAIN = {"attention": _plain_attention, "train": _plain_train, "weights": _plain_weights, "tree": _plain_tree, "evict": _plain_evict}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["path"] == "evict":
        return _exact_evict(state)
    if case["path"] == "tree":
        return _exact_tree(state)
    return _exact_dense(state)


def _attend(case, slopes, scale, q, keys, hidden, distance):
    """log-weights of one head: q [rows, d], keys [n, d]."""
    z = torch.einsum("id,jd->ij", q, keys).mul(scale)
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    if slopes is not None:
        z = z - float(slopes) * distance
    return z.masked_fill(hidden, -math.inf)


def _exact_dense(state):
    case = state["case"]
    b, hq, hkv, n, d = (case[k] for k in ("b", "hq", "hkv", "n", "d"))
    group = hq // hkv
    q, k, v = (state[name].double() for name in ("q", "k", "v"))
    i, j = torch.meshgrid(torch.arange(n, device=q.device), torch.arange(n, device=q.device), indexing="ij")
    distance = (i - j).abs().double() if case["bias"] else None
    train, o, lse = case["path"] == "train", torch.zeros_like(q), torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    weights = torch.zeros((b, hkv, n), dtype=torch.float64, device=q.device)
    if train:
        dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    for s in range(b):
        hidden = torch.zeros((n, n), dtype=torch.bool, device=q.device)
        if case["mask"] in ("causal", "documents", "window"):
            hidden |= j > i
        if state["first"] is not None:
            hidden |= j < state["first"][s].long()[:, None]
        if state["last"] is not None:
            hidden |= j >= state["last"][s].long()[:, None]
        for h in range(hq):
            operands = [q[s, h], k[s, h // group], v[s, h // group]]
            if train:
                operands = [t.clone().requires_grad_() for t in operands]
            slope = None if state["slopes"] is None else state["slopes"][h]
            logits = _attend(case, slope, state["scale"], operands[0], operands[1], hidden, distance)
            if case["path"] == "weights":
                weights[s, h // group] += (logits - state["lse"][s, h].double()[:, None]).exp().sum(0)
                continue
            with torch.no_grad():
                lse[s, h] = logits.logsumexp(1)
            out = logits.softmax(1) @ operands[2]
            o[s, h] = out.detach()
            if train:
                grads = torch.autograd.grad(out, operands, state["do"][s, h].double())
                dq[s, h] = grads[0]
                dk[s, h // group] += grads[1]
                dv[s, h // group] += grads[2]
    if case["path"] == "weights":
        return weights
    return (o, lse, dq, dk, dv) if train else (o, lse)


def _exact_tree(state):
    case = state["case"]
    hq, nodes, d, page, group = case["hq"], case["nodes"], case["d"], case["page"], case["hq"] // case["hkv"]
    device = state["q"].device
    o = torch.zeros(state["q"].shape, dtype=torch.float64, device=device)
    lse = torch.zeros(o.shape[:3], dtype=torch.float64, device=device)
    weights = state["weights"].double().clone() if case["accumulate"] else None
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
            keys, values = state["k"][pages, g, slot % page].double(), state["v"][pages, g, slot % page].double()
            for h in range(g * group, (g + 1) * group):
                slope = None if state["slopes"] is None else state["slopes"][h]
                logits = _attend(case, slope, state["scale"], state["q"][s, h].double(), keys, hidden, distance)
                p = logits.softmax(1)
                o[s, h], lse[s, h] = p @ values, logits.logsumexp(1)
                if weights is not None:
                    weights[s, g, :total] += p.sum(0)
    return (o, lse) if weights is None else (o, lse, weights)


def _exact_evict(state):
    case = state["case"]
    keep, recent, page = case["keep"], case["recent"], case["page"]
    result = {name: torch.zeros(t.shape, dtype=torch.float64, device=t.device) for name, t in state["out"].items()}
    lengths, table, table_out = (state[n].tolist() for n in ("lengths", "table", "table_out"))
    weights = state["weights"].cpu().numpy()
    for s, n in enumerate(lengths):
        result["lengths"][s] = min(n, keep)
        for h in range(case["hkv"]):
            w = weights[s, h]
            if n <= keep:
                chosen = list(range(n))
            else:
                old = (-w[:n - recent]).argsort(kind="stable")[:keep - recent]
                chosen = sorted(old.tolist()) + list(range(n - recent, n))
            at = torch.tensor(chosen, device=state["k"].device)
            slot = torch.arange(len(chosen), device=at.device)
            source = torch.tensor(table[s], device=at.device)[at // page]
            target = torch.tensor(table_out[s], device=at.device)[slot // page]
            for name in ("k", "v"):
                result[name][target, h, slot % page] = state[name][source, h, at % page].double()
            result["weights"][s, h, :len(chosen)] = state["weights"][s, h, at].double()
            result["positions"][s, h, :len(chosen)] = at.double()
    result["positions"], result["lengths"] = result["positions"].int(), result["lengths"].int()
    return result


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e, d, b, hkv = _BYTES[case["dtype"]], case["d"], case["b"], case["hkv"]
    if case["path"] == "tree":
        hq, nodes = case["hq"], case["nodes"]
        tokens = sum(_lengths(case)) + b * nodes
        seen = nodes * sum(_lengths(case)) + sum(bin(w & (2 ** 64 - 1)).count("1") for words in _trees(case) for w in words)
        held = 2 * 4 * hkv * tokens if case["accumulate"] else 0
        return {"bytes": 2 * e * d * hkv * tokens + 2 * e * d * b * hq * nodes + 4 * b * hq * nodes + held, "flops": 4 * d * hq * seen}
    if case["path"] == "evict":
        kept = sum(min(n, case["keep"]) for n in _lengths(case))
        return {"bytes": 4 * hkv * sum(_lengths(case)) + 4 * e * d * hkv * kept + 8 * hkv * kept, "flops": 0}
    hq, n = case["hq"], case["n"]
    queries, keys, pairs = e * d * b * hq * n, e * d * b * hkv * n, hq * _pairs(case)
    if case["path"] == "attention":
        return {"bytes": 2 * queries + 2 * keys + 4 * b * hq * n, "flops": 4 * d * pairs}
    if case["path"] == "weights":
        return {"bytes": queries + keys + 4 * b * hq * n + 4 * b * hkv * n, "flops": 2 * d * pairs}
    # forward two products of a pair's row, backward five
    return {"bytes": 4 * queries + 4 * keys + 4 * b * hq * n, "flops": 14 * d * pairs}
