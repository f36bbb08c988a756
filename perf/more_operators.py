"""Performance cases of several continuations of one sequence over the paged 8-bit
key/value cache: trees of drafted tokens, and sequences that share pages.

``tree`` is attention of drafted tokens that branch: each sees the tokens before all
drafts and its own ancestors.  ``step`` is what one layer and the cache's owner run to
verify drafts: positions and ancestors from the parents, rotation and append at
those positions, attention, the walk along the tokens that the model agrees with, and
the move of their keys and values behind the context.  ``keep`` is that move in all
layers' caches.  ``fork`` lets rows of a block table go on as other rows (beams,
samples of one prompt): full pages are shared, the pages that are appended to next are
each row's own, pages that nobody holds are free.  ``copy`` copies whole pages.

Sizes: Llama-3-8B (32 query and 8 key/value heads of 128, 32 layers), Qwen2-7B (28 and
4, 28 layers), the Qwen3-MoE layer (32 and 4), and generic heads of 64 and 256.  Where
``own`` is true, ``run`` calls ``kairyu_amd.attention``, ``kairyu_amd.drafts`` and
``kairyu_amd.pages``; otherwise it computes the same in elementary operations.
"""

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _tree_case(name, kind, seqs, nodes, length, heads, kv_heads, dim, *, page=64, ragged=True, pad=0, window=0,
               qk_norm=False, dtype="bf16"):
    """``seqs`` sequences of at most ``length`` tokens, the last ``nodes`` (at most) of each drafted."""
    return {"name": name, "kind": kind, "seqs": seqs, "nodes": nodes, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged, "pad": pad, "window": window,
            "qk_norm": qk_norm, "dtype": dtype}


def _keep_case(name, layers, seqs, nodes, length, kv_heads, dim, *, page=64):
    return {"name": name, "kind": "keep", "layers": layers, "seqs": seqs, "nodes": nodes, "length": length,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _fork_case(name, layers, requests, beams, length, kv_heads, dim, *, page=64, room=1, ended=0):
    """``requests`` of ``beams`` rows each; every ``ended``-th request is given back (0: none)."""
    return {"name": name, "kind": "fork", "layers": layers, "requests": requests, "beams": beams, "length": length,
            "kv_heads": kv_heads, "dim": dim, "page": page, "room": room, "ended": ended}


def _copy_case(name, layers, count, kv_heads, dim, *, page=64):
    return {"name": name, "kind": "copy", "layers": layers, "count": count, "kv_heads": kv_heads, "dim": dim, "page": page}


def listed():
    return [
        # one user's drafts, 900 tokens in: launch latency
        _tree_case("tree_1", "tree", 1, 12, 900, 32, 8, 128, ragged=False),
        # a busy server's batch of ragged trees and contexts
        _tree_case("tree_32", "tree", 32, 32, 6000, 32, 4, 128),
        # two long documents, wide trees: the token axis is all there is to split
        _tree_case("tree_long", "tree", 2, 48, 100003, 28, 4, 128, ragged=False, dtype="fp16"),
        # sliding window, narrow heads, small pages, padding rows
        _tree_case("tree_window", "tree", 24, 16, 5000, 16, 16, 64, page=16, window=1024, dtype="fp16", pad=5),
        # one user's verification of a layer: six small calls in a row
        _tree_case("step_1", "step", 1, 8, 700, 28, 4, 128, ragged=False),
        # a batch's, with head norms
        _tree_case("step_16", "step", 16, 24, 3000, 32, 8, 128, qk_norm=True),
        # one user's accepted tokens in all layers
        _keep_case("keep_1", 32, 1, 12, 900, 8, 128),
        # a batch's, in small pages that the moves cross
        _keep_case("keep_64", 28, 64, 32, 2000, 4, 128, page=16),
        # the beams of two requests after one step
        _fork_case("fork_8", 32, 2, 4, 1000, 8, 128),
        # a server's beams in all layers, some requests ended
        _fork_case("fork_128", 16, 32, 4, 1500, 8, 128, ended=8),
        # a few pages of one prefix
        _copy_case("copy_4", 32, 4, 8, 128),
        # many sequences' pages moved at once, the largest call
        _copy_case("copy_512", 16, 512, 8, 128),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _cost(case):
    w = work(case)
    return w["flops"] / 5e14 + w["bytes"] / 4e12


def draw(rng):
    kind = rng.choices(("tree", "step", "keep", "fork", "copy"), (4, 2, 2, 2, 1))[0]
    page = rng.choice((16, 32, 64, 128))
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (28, 4, 128), (32, 4, 128), (16, 16, 64), (8, 1, 256), (40, 8, 128)))
    if kind in ("tree", "step"):
        nodes = _log_int(rng, 1, 64)
        case = _tree_case("", kind, _log_int(rng, 1, 64), nodes, nodes + _log_int(rng, 1, 65536 if kind == "tree" else 4096),
                          heads, kv_heads, dim, page=page, ragged=rng.random() < 0.7, pad=rng.choice((0, 0, 3)),
                          window=rng.choice((0, 0, 0, 512)), qk_norm=rng.random() < 0.3,
                          dtype=rng.choice(("bf16", "bf16", "fp16")))
        shrink = "seqs"
    elif kind == "keep":
        nodes = _log_int(rng, 2, 64)
        case = _keep_case("", _log_int(rng, 1, 48), _log_int(rng, 1, 128), nodes, nodes + _log_int(rng, 1, 3000), kv_heads,
                          dim, page=page)
        shrink = "layers"
    elif kind == "fork":
        case = _fork_case("", _log_int(rng, 1, 32), _log_int(rng, 1, 48), rng.randint(1, 8), _log_int(rng, 1, 2500), kv_heads,
                          dim, page=page, room=rng.choice((1, 1, 9, 200)), ended=rng.choice((0, 0, 3)))
        shrink = "layers"
    else:
        case = _copy_case("", _log_int(rng, 1, 32), _log_int(rng, 1, 512), kv_heads, dim, page=page)
        shrink = "count"
    case.pop("name")
    most = max(_cost(c) for c in listed() if c["kind"] == kind)

    def large():
        if kind in ("tree", "step"):  # (the plain form's scores)
            return case["seqs"] * case["nodes"] * case["heads"] * case["length"] > 6e8
        return kind != "copy" and _pool_bytes(case) > 6e9

    while _cost(case) > most or large():
        if case[shrink] == 1:
            case["length"] = max(case.get("nodes", 1), case["length"] // 2)
        else:
            case[shrink] = max(1, case[shrink] * 2 // 3)
    return case


# ------------------------------------------------------- what the case alone fixes
def _rng(case):
    return random.Random(case["seqs"] * 1000003 + case["length"] * 101 + case["nodes"])


def _lengths(case):
    """(drafted tokens, tokens after them) of each sequence."""
    rng = _rng(case)
    new, total = [], []
    for i in range(case["seqs"]):
        if i == 0 or not case.get("ragged", True):  # the first has the full length
            n, t = case["nodes"], case["length"]
        else:
            n = rng.randint((case["nodes"] + 1) // 2, case["nodes"])
            t = n + rng.randint(0, case["length"] - case["nodes"])
        new.append(n)
        total.append(t)
    return new, total


def _kept_counts(case):
    """Tokens that each sequence of a ``keep`` case keeps: the pending one and a few of the drafted."""
    rng = _rng(case)
    return [min(n, 1 + rng.randint(0, 7)) for n in _lengths(case)[0]]


def _requests(case):
    """(tokens, parent beams or None where it has ended) of each request of a ``fork`` case."""
    rng = random.Random(case["requests"] * 1000003 + case["length"] * 101 + case["beams"])
    out = []
    for r in range(case["requests"]):
        tokens = case["length"] if r == 0 else rng.randint(max(1, case["length"] // 8), case["length"])
        parents = sorted(rng.randrange(case["beams"]) for _ in range(case["beams"]))
        out.append((tokens, None if case["ended"] and r % case["ended"] == case["ended"] - 1 else parents))
    return out


def _fork_pages(case):
    page, beams = case["page"], case["beams"]
    own_pages = -(-(case["room"] + page) // page)  # a row's last page, and those of its room
    return sum(t // page + beams * (1 + own_pages) for t, _ in _requests(case)) + 2


def _pool_bytes(case):
    if case["kind"] == "keep":
        pages = sum(-(-t // case["page"]) for t in _lengths(case)[1]) + 2
    else:
        pages = _fork_pages(case)
    return pages * case["layers"] * case["kv_heads"] * case["page"] * case["dim"] * 2


def work(case):
    kind, d, hk, page = case["kind"], case["dim"], case["kv_heads"], case["page"]
    token = hk * 2 * d  # bytes of one token's keys and values
    if kind == "copy":
        return {"bytes": 2 * case["count"] * case["layers"] * (page * token + 8 * hk), "flops": 0}
    if kind == "keep":
        moved = sum(max(c - 1, 0) for c in _kept_counts(case))  # (the pending token is in its place)
        return {"bytes": case["layers"] * (2 * moved * token + 16 * hk * case["seqs"]) + 4 * case["seqs"] * case["nodes"], "flops": 0}
    if kind == "fork":
        total, rows = 0, case["requests"] * case["beams"]
        wide = -(-(case["length"] + case["room"]) // page)
        for t, parents in _requests(case):
            if parents is not None:  # the first child keeps the last page, the others copy it
                total += 2 * (case["beams"] - len(set(parents))) * case["layers"] * ((t % page) * token + 8 * hk)
        return {"bytes": total + 8 * rows * wide + 4 * _fork_pages(case), "flops": 0}
    hq = case["heads"]
    rows, pairs, seen = 0, 0, 0
    for n, t in zip(*_lengths(case)):
        context = min(t - n, case["window"]) if case["window"] else t - n
        rows += n
        pairs += n * context + n * min(n, 5)
        seen += context + n
    total = {"bytes": rows * hq * d * 4 + seen * hk * (2 * d + 8 / page) + 12 * rows, "flops": 4 * pairs * hq * d}
    if kind == "step":
        total["bytes"] += rows * (hq * d * 4 + hk * d * 6 + 4 * d + 24)
        total["flops"] += rows * (hq + hk) * d * 3
    return total


# ------------------------------------------------------------------------- inputs
def _power(e):
    """2^e in fp32, from its bits."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _stack(case, pages, g, layers):
    """Caches of all layers: codes ``[layers, pages, kv heads, page, dim]`` without NaN, power-of-two scales."""
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    stack = {}
    for name in "kv":
        codes = torch.empty(shape, device="cuda", dtype=torch.uint8)
        # (signs and exponents alike often: -126 to 126 but for the sign bit)
        torch.randint(0, 127, shape, generator=g, device="cuda", dtype=torch.uint8, out=codes)
        codes[..., ::2] |= 0x80
        stack[name] = codes.view(E4M3)
        stack[name + "_scale"] = _power(torch.randint(-8, -5, shape[:3], generator=g, device="cuda"))
    return stack


def _parents(n, rng):
    """A tree of ``n`` nodes, the first its root, parents before children, at most 8 deep."""
    parents, depth = [-1], [0]
    for i in range(1, n):
        p = rng.randrange(max(0, i - 12), i)
        while depth[p] >= 7:
            p = parents[p]
        parents.append(p)
        depth.append(depth[p] + 1)
    return parents


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _table(held, pages, g, wide):
    """Block table of ``held[b]`` pages a sequence, in any order; -1 behind them."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    place = torch.full((len(held), wide), -1, dtype=torch.int64)
    start = 0
    for b, n in enumerate(held):
        place[b, :n] = torch.arange(start, start + n)
        start += n
    place = place.cuda()
    return torch.where(place >= 0, order[place.clamp(min=0)], place.to(torch.int32))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    kind, page, hk, d = case["kind"], case["page"], case["kv_heads"], case["dim"]
    if kind == "copy":
        pages = 2 * case["count"] + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        return {"case": case, "stack": _stack(case, pages, g, case["layers"]),
                "sources": order[: case["count"]].clone(), "targets": order[case["count"]: 2 * case["count"]].clone()}
    if kind == "fork":
        return _prepare_fork(case, g)
    new, total = _lengths(case)
    held = [-(-t // page) for t in total]
    pages, wide = sum(held) + 2, max(held)
    state = {"case": case, "table": _table(held, pages, g, wide), "cu": _ints([0] + new).cumsum(0).to(torch.int32),
             "lengths": _ints(total), "most": max(new), "most_tokens": max(total)}
    if kind == "keep":
        kept = torch.full((len(new), max(new)), -1, dtype=torch.int32)
        for b, (n, c) in enumerate(zip(new, _kept_counts(case))):
            kept[b, :c] = torch.tensor([0] + sorted(rng.sample(range(1, n), c - 1)), dtype=torch.int32)
        return state | {"stack": _stack(case, pages, g, case["layers"]), "kept": kept.cuda(), "counts": _ints(_kept_counts(case))}

    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # what earlier steps stored: codes near the top of e4m3's range, some channels larger than
    # others, and in slots past the end whatever was there, NaN among it
    channel = torch.exp(randn(hk, 1, d) * 0.5)
    cache = {}
    for name, span in (("k", 100.0), ("v", 90.0)):
        codes = torch.empty((pages, hk, page, d), device="cuda", dtype=E4M3)
        for at in range(0, pages, 512):
            part = codes[at: at + 512]
            part.copy_((randn(*part.shape) * (channel if name == "k" else 1.0) * span).clamp(-448, 448))
        cache[name] = codes
        cache[name + "_scale"] = _power(torch.randint(-8, -5, (pages, hk), generator=g, device="cuda"))
    last = torch.tensor(total, device="cuda") - 1
    tail = state["table"][torch.arange(len(new), device="cuda"), last // page].long()
    behind = torch.arange(page, device="cuda") > (last % page)[:, None]
    for name in "kv":
        codes = cache[name].view(torch.uint8)
        codes[tail] = torch.where(behind[:, None, :, None], torch.full_like(codes[tail], 0x7F), codes[tail])
    rows, hq = sum(new) + case["pad"], case["heads"]
    packed = randn(rows, (hq + 2 * hk) * d).to(dtype)
    packed[:, : hq * d] *= 2
    q, k, v = (x.unflatten(-1, (-1, d)) for x in packed.split((hq * d, hk * d, hk * d), dim=-1))
    trees = [_parents(n, rng) for n in new]
    parents = _ints([p for tree in trees for p in tree] + [-1] * case["pad"])
    state |= {"q": q, "k": k, "v": v, "cache": cache, "parents": parents}
    if kind == "tree":
        state["mask"], state["positions"] = _tree(state)
        return state
    # what the drafter proposed, and what the model says after each node: for most nodes with
    # children that one of them was right
    tokens = [rng.randrange(32000) for _ in range(rows)]
    targets = [rng.randrange(32000) for _ in range(rows)]
    row = 0
    for tree in trees:
        for i, p in enumerate(tree):
            if p >= 0 and rng.random() < 0.6:
                targets[row + p] = tokens[row + i]
        row += len(tree)
    freq = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.arange(max(total), dtype=torch.float64)[:, None] * freq
    return state | {"tokens": torch.tensor(tokens).cuda(), "targets": torch.tensor(targets).cuda(),
                    "cos_sin": torch.cat((angle.cos(), angle.sin()), dim=-1).float().cuda(),
                    "norms": [(randn(d) * 0.1 + 1).to(dtype) for _ in "qk"] if case["qk_norm"] else [None, None]}


def _prepare_fork(case, g):
    """Requests whose beams share the full pages of their context and hold their last page alone."""
    page, beams = case["page"], case["beams"]
    pages = _fork_pages(case)
    wide = -(-(case["length"] + case["room"]) // page) + 1
    table, lengths, parents, next_page = [], [], [], 0
    for r, (tokens, kids) in enumerate(_requests(case)):
        full = list(range(next_page, next_page + tokens // page))
        next_page += len(full)
        for b in range(beams):
            mine = [next_page] if tokens % page else []
            next_page += len(mine)
            table.append(full + mine + [-1] * (wide - len(full) - len(mine)))
            lengths.append(tokens)
            parents.append(-1 if kids is None else r * beams + kids[b])
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    place = torch.tensor(table).cuda()
    table = torch.where(place >= 0, order[place.clamp(min=0)], place.to(torch.int32))
    holders = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    holders.index_add_(0, torch.where(table >= 0, table, pages).flatten().long(), torch.ones_like(table).flatten())
    return {"case": case, "stack": _stack(case, pages, g, case["layers"]), "table": table, "lengths": _ints(lengths),
            "parents": _ints(parents), "holders": holders[:pages].clone()}


# -------------------------------------------------------------------- plain forms
def _rows(state):
    """(sequence, index there) of each row that has a sequence."""
    cu = state["cu"].long()
    at = torch.arange(state["q"].shape[0] - state["case"]["pad"], device="cuda")
    seq = torch.searchsorted(cu[1:], at, right=True)
    return seq, at - cu[seq]


def _ancestors(state):
    """``[S, most, most]``: whether node j is i itself or an ancestor; and the nodes' parents ``[S, most]``, -1 past the last."""
    most, cu, parents = state["most"], state["cu"].long(), state["parents"].long()
    node = torch.arange(most, device="cuda")
    here = node < (cu[1:] - cu[:-1])[:, None]
    parent = torch.where(here, parents[(cu[:-1, None] + node).clamp(max=parents.numel() - 1)], -1)
    up = ((parent[..., None] == node) | (node[:, None] == node)).float()  # a node and its parent
    for _ in range(most.bit_length()):  # twice as far each time
        up = torch.matmul(up, up).clamp(max=1)
    return up.bool() & here[..., None], parent


def _tree(state):
    """Ancestor bits ``[R, words]`` and positions ``[R]``: no bits and -1 for padding."""
    up, _ = _ancestors(state)
    seq, node = _rows(state)
    words = -(-state["most"] // 32)
    bits = torch.nn.functional.pad(up, (0, 32 * words - state["most"]))[seq, node].unflatten(-1, (words, 32)).long()
    mask = (bits << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 2**31, mask - 2**32, mask).to(torch.int32)
    first = state["lengths"].long() - (state["cu"][1:] - state["cu"][:-1])
    positions = (first[seq] + up[seq, node].sum(-1) - 1).to(torch.int32)
    pad = state["case"]["pad"]
    return torch.nn.functional.pad(mask, (0, 0, 0, pad)), torch.nn.functional.pad(positions, (0, pad), value=-1)


def _head_norm(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _scale_for(amax):
    """The smallest power of two that brings ``amax`` (at least 1e-12) within 448."""
    m, e = torch.frexp(amax.clamp(min=1e-12))
    return _power(e - 9 + (m > 0.875).int())


def _append(state, positions):
    """Rotates by ``positions`` and stores in the sequences' last slots."""
    case, cache, table = state["case"], state["cache"], state["table"].long()
    pages, hk, page, d = cache["k"].shape
    seq, node = _rows(state)
    rows = seq.numel()
    cu, lengths = state["cu"].long(), state["lengths"].long()
    pos = lengths[seq] - (cu[seq + 1] - cu[seq]) + node
    cos, sin = state["cos_sin"][positions[:rows].long()][:, None].chunk(2, -1)
    q, k, v = (state[n][:rows].float() for n in "qkv")
    if case["qk_norm"]:
        q, k = _head_norm(q, state["norms"][0]), _head_norm(k, state["norms"][1])
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    at, slot = table[seq, pos // page], pos % page
    first = torch.full((pages,), page, device="cuda").scatter_reduce(0, at, slot, "amin")[:, None]
    head = at[cu[:-1]]  # each sequence's first page, which may hold earlier tokens
    for name, x in (("k", k), ("v", v)):
        codes, scale = cache[name].view(torch.uint8), cache[name + "_scale"]
        need = _scale_for(torch.zeros((pages, hk), device="cuda").index_reduce(0, at, x.abs().amax(-1), "amax"))
        grown = torch.where(first == page, scale, torch.where(first > 0, torch.maximum(scale, need), need))
        old = codes[head]
        moved = old.view(E4M3).float() * (scale[head] / grown[head])[..., None, None]
        keep = torch.arange(page, device="cuda") < first[head]
        codes[head] = torch.where(keep[:, None, :, None], moved.clamp(-448, 448).to(E4M3).view(torch.uint8), old)
        scale.copy_(grown)
        value = (x / scale[at][..., None]).clamp(-448, 448).to(E4M3)
        codes[at[:, None], torch.arange(hk, device="cuda"), slot[:, None]] = value.view(torch.uint8)
    return torch.nn.functional.pad(q.to(state["q"].dtype), (0, 0, 0, 0, 0, case["pad"]))


def _attend(state, q, mask, positions):
    case, cache = state["case"], state["cache"]
    page, most = case["page"], state["most"]
    rows, hq, d = q.shape
    hk = case["kv_heads"]
    cu, lengths = state["cu"].long(), state["lengths"].long()
    at = state["table"][:, : -(-state["most_tokens"] // page)].long().clamp(min=0)

    def gathered(name):  # [sequences, kv heads, tokens, dim]
        x = cache[name].view(torch.uint8)[at].view(E4M3).float() * cache[name + "_scale"][at][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)

    token = torch.arange(at.shape[1] * page, device="cuda")
    here = token < lengths[:, None]
    first = lengths - (cu[1:] - cu[:-1])
    index = (cu[:-1, None] + torch.arange(most, device="cuda")).clamp(max=rows - 1)
    node = (token - first[:, None])[:, None].expand(-1, most, -1)  # [sequences, rows, tokens]
    word = mask[index].gather(2, (node >> 5).clamp(0, mask.shape[1] - 1))
    visible = (node < 0) | (((word >> (node & 31)) & 1) == 1)
    if case["window"]:
        visible &= (node >= 0) | (token > positions[index][..., None] - case["window"])
    visible &= here[:, None]
    k = gathered("k")
    qs = q.float()[index].unflatten(2, (hk, hq // hk)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # rows and heads of a group
    s = torch.matmul(qs, k.transpose(-1, -2)) * d**-0.5
    del k
    s = s.unflatten(2, (most, -1)).masked_fill_(~visible[:, None, :, None], -math.inf).flatten(2, 3)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = gathered("v").masked_fill_(~here[:, None, :, None], 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.unflatten(2, (most, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    seq, row = _rows(state)
    return torch.nn.functional.pad(o[seq, row].to(q.dtype), (0, 0, 0, 0, 0, case["pad"]))


def _accept(state):
    """Nodes kept ``[S, most]`` (-1 behind them), their number, and the token after the last of them."""
    most, cu, tokens, targets = state["most"], state["cu"].long(), state["tokens"], state["targets"]
    up, parent = _ancestors(state)
    node = torch.arange(most, device="cuda")
    index = (cu[:-1, None] + node).clamp(max=tokens.numel() - 1)
    token, target = tokens[index], targets[index]
    right = (parent >= 0) & (token == target.gather(1, parent.clamp(min=0)))
    # the lowest of the children that are right
    same = (parent[:, :, None] == parent[:, None]) & right[:, None] & (node < node[:, None])
    right = (right & ~same.any(-1)) | (node == 0)
    kept = (right[:, None] | ~up).all(-1) & up.any(-1)
    order = torch.where(kept, node, most).sort(-1).values
    counts = kept.sum(-1)
    last = order.gather(1, (counts - 1).clamp(min=0)[:, None]).clamp(max=most - 1)
    following = torch.where(counts > 0, target.gather(1, last)[:, 0], -1)
    return torch.where(order < most, order, -1).to(torch.int32), counts.to(torch.int32), following


def _keep(state, stack, kept, counts):
    """Token ``first + kept[i]`` of each sequence to slot ``first + i``; the new lengths."""
    page, table, cu, lengths = state["case"]["page"], state["table"].long(), state["cu"].long(), state["lengths"].long()
    n = cu[1:] - cu[:-1]
    first = lengths - n
    i = torch.arange(kept.shape[1], device="cuda")
    here = i < counts[:, None]
    seq = torch.arange(len(lengths), device="cuda")[:, None].expand_as(here)[here]
    source, target = (first[:, None] + kept)[here], (first[:, None] + i)[here]
    from_page, to_page = table[seq, source // page], table[seq, target // page]
    # pages that hold earlier tokens
    old = torch.where(first % page > 0, table.gather(1, (first // page).clamp(max=table.shape[1] - 1)[:, None])[:, 0], -1)
    old = old[old >= 0]
    before = torch.arange(page, device="cuda") < (first % page)[first % page > 0][:, None]
    for name in "kv":
        codes, scale = stack[name].view(torch.uint8), stack[name + "_scale"]
        part = torch.zeros_like(scale).index_reduce(1, to_page, scale[:, from_page], "amax")
        touched = part > 0
        part.index_reduce_(1, old, scale[:, old], "amax")
        grown = torch.where(touched, part, scale)
        moved = codes[:, from_page, :, source % page].view(E4M3).float()  # [tokens, layers, heads, dim]
        moved = moved * (scale[:, from_page] / grown[:, to_page]).transpose(0, 1)[..., None]
        whole = codes[:, old]
        again = (whole.view(E4M3).float() * (scale[:, old] / grown[:, old])[..., None, None]).to(E4M3).view(torch.uint8)
        codes[:, old] = torch.where(before[None, :, None, :, None], again, whole)
        codes[:, to_page, :, target % page] = moved.to(E4M3).view(torch.uint8)
        scale.copy_(grown)
    return (first + counts).to(torch.int32)


def _copy(state):
    at, to = state["sources"].long(), state["targets"].long()
    for name, x in state["stack"].items():
        raw = x.view(torch.uint8) if name in "kv" else x
        raw[:, to] = raw[:, at]


def _fork(state):
    case, stack, holders = state["case"], state["stack"], state["holders"]
    page, room, pages = case["page"], case["room"], holders.numel()
    table, parents = state["table"].long(), state["parents"].long()
    rows, wide = table.shape
    lives = parents >= 0
    of = parents.clamp(min=0)
    mine = torch.where(lives[:, None], table[of], -1)
    tokens = torch.where(lives, state["lengths"].long()[of], 0)
    slot = torch.arange(wide, device="cuda")
    begin = (tokens // page)[:, None]
    region = lives[:, None] & (slot >= begin) & (slot <= ((tokens + room - 1) // page)[:, None])
    row = torch.arange(rows, device="cuda")
    eldest = torch.full((rows,), rows, device="cuda").scatter_reduce(0, of, torch.where(lives, row, rows), "amin")
    alone = (mine >= 0) & (holders[mine.clamp(min=0)] == 1) & (eldest[of] == row)[:, None]
    need = region & ~alone
    free = holders == 0
    listed_free = torch.full((pages + 1,), -1, device="cuda")
    listed_free[torch.where(free, free.cumsum(0) - 1, pages)] = torch.arange(pages, device="cuda")
    listed_free[pages] = -1
    rank = (need.flatten().cumsum(0) - 1).view_as(need)
    enough = rank < free.sum()
    fresh = torch.where(need & enough, listed_free[torch.where(enough, rank, pages).clamp(min=0)], -1)
    result = torch.where(need, fresh, torch.where((slot < begin) | region, mine, -1))
    # the tokens of a last page that is not the row's own
    at = begin.clamp(max=wide - 1)
    copied = need.gather(1, at)[:, 0] & (tokens % page > 0) & (mine.gather(1, at)[:, 0] >= 0) & (fresh.gather(1, at)[:, 0] >= 0)
    copied &= tokens // page < wide
    source, target = mine.gather(1, at)[copied, 0], fresh.gather(1, at)[copied, 0]
    held = torch.arange(page, device="cuda") < (tokens % page)[copied, None]
    for name in "kv":
        codes, scale = stack[name].view(torch.uint8), stack[name + "_scale"]
        codes[:, target] = torch.where(held[None, :, None, :, None], codes[:, source], codes[:, target])
        scale[:, target] = scale[:, source]
    count = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    for x, step in ((table, -1), (result, 1)):
        count.index_add_(0, torch.where(x >= 0, x, pages).flatten(), torch.full((x.numel(),), step, dtype=torch.int32, device="cuda"))
    holders += count[:pages]
    missing = (need.sum() - free.sum()).clamp(min=0).to(torch.int32)[None]
    return result.to(torch.int32), tokens.to(torch.int32), missing


# ---------------------------------------------------------------------------- run
def _caches(state):
    """The layers' caches as the framework takes them: made once, kept by the program."""
    from kairyu_amd.attention import PagedKvCache
    from kairyu_amd.pages import KvCaches

    if "caches" not in state:
        stack = state["stack"]
        parts = [stack[n].unbind(0) for n in ("k", "v", "k_scale", "v_scale")]
        state["caches"] = KvCaches([PagedKvCache(*x) for x in zip(*parts)])
    return state["caches"]


def _run_own(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind in ("copy", "keep", "fork"):
        from kairyu_amd.drafts import keep_tokens
        from kairyu_amd.pages import copy_pages, fork_sequences

        caches = _caches(state)
        if kind == "copy":
            copy_pages(caches, state["sources"], state["targets"])
            return ()
        if kind == "keep":
            return (keep_tokens(caches, state["table"], state["cu"], state["lengths"], state["kept"], state["counts"]),)
        return fork_sequences(caches, state["holders"], state["table"], state["lengths"], state["parents"], case["room"])
    from kairyu_amd.attention import DraftTree, PagedKvCache, rotate_append, tree_attention
    from kairyu_amd.drafts import accept_drafts, draft_tree, keep_tokens

    pool = PagedKvCache(*(state["cache"][n] for n in ("k", "v", "k_scale", "v_scale")))
    where = (pool, state["table"], state["cu"], state["lengths"])
    if kind == "tree":
        return (tree_attention(state["q"], *where, DraftTree(state["mask"], state["positions"]), window=case["window"]),)
    tree = draft_tree(state["parents"], state["cu"], state["lengths"], state["most"])
    q = rotate_append(state["q"], state["k"], state["v"], *where, state["cos_sin"], positions=tree.positions,
                      q_norm=state["norms"][0], k_norm=state["norms"][1])
    o = tree_attention(q, *where, tree, window=case["window"])
    accepted = accept_drafts(state["tokens"], state["targets"], state["parents"], state["cu"], state["most"])
    lengths = keep_tokens(*where, *accepted[:2])
    return tree.mask, tree.positions, q, o, *accepted, lengths


def _run_plain(state):
    kind = state["case"]["kind"]
    if kind == "copy":
        _copy(state)
        return ()
    if kind == "keep":
        return (_keep(state, state["stack"], state["kept"], state["counts"]),)
    if kind == "fork":
        return _fork(state)
    if kind == "tree":
        return (_attend(state, state["q"], state["mask"], state["positions"]),)
    mask, positions = _tree(state)
    q = _append(state, positions)
    o = _attend(state, q, mask, positions)
    accepted = _accept(state)
    stack = {n: x[None] for n, x in state["cache"].items()}
    return mask, positions, q, o, *accepted, _keep(state, stack, *accepted[:2])


NAMES = {"copy": (), "keep": ("lengths",), "fork": ("table", "lengths", "missing"), "tree": ("o",),
         "step": ("mask", "positions", "q", "o", "kept", "counts", "following", "lengths")}


def run(state):
    kind = state["case"]["kind"]
    out = dict(zip(NAMES[kind], _run_own(state) if own else _run_plain(state)))
    if kind == "fork":  # the next step goes on with these
        state["table"], state["lengths"] = out["table"], out["lengths"]
        out["holders"] = state["holders"]
    if kind in ("copy", "keep", "fork"):
        out |= state["stack"]
    elif kind == "step":
        out |= state["cache"]
    return out


# ----------------------------------------------------------------- 64-bit definitions
def _to_e4m3(x):
    """The nearest e4m3 value of each fp64 value within 448, ties to the even one; NaN stays."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_keep(s, value, scale, kept, counts):
    """Moves in place: ``value`` and ``scale`` are ``[layers, pages, ...]`` in fp64 by name."""
    page, table = s["case"]["page"], s["table"].tolist()
    cu, lengths = s["cu"].tolist(), s["lengths"].tolist()
    for b, total in enumerate(lengths):
        first, c = total - (cu[b + 1] - cu[b]), int(counts[b])
        place = {}  # page -> [(slot, page and slot it comes from)], as the tokens lie afterwards
        for t in range(first - first % page, first):
            place.setdefault(table[b][t // page], []).append((t % page, table[b][t // page], t % page))
        for i in range(c):
            t, u = first + i, first + int(kept[b][i])
            place.setdefault(table[b][t // page], []).append((t % page, table[b][u // page], u % page))
        if not c:
            continue
        arrivals = {table[b][(first + i) // page] for i in range(c)}
        for name in "kv":
            new = {}
            for p in arrivals:
                held = place[p]
                top = torch.stack([scale[name][:, q] for _, q, _ in held]).amax(0)
                at = torch.tensor([x[0] for x in held], device="cuda")
                of = torch.tensor([x[1] for x in held], device="cuda")
                slot = torch.tensor([x[2] for x in held], device="cuda")
                moved = value[name][:, of, :, slot] * (scale[name][:, of].transpose(0, 1) / top)[..., None]
                new[p] = (at, _to_e4m3(moved), top)
            for p, (at, moved, top) in new.items():
                value[name][:, p].index_copy_(2, at, moved.permute(1, 2, 0, 3))
                scale[name][:, p] = top


def _exact_attend(s, q, value, scale, see):
    """``see(b, node)``: the drafted tokens that a node sees, and its position."""
    case = s["case"]
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    row = 0
    for b, (n, t) in enumerate(zip(*_lengths(case))):
        first = t - n
        seen = torch.zeros((n, t), dtype=torch.bool)
        for i in range(n):
            nodes, position = see(b, i)
            seen[i, max(0, position + 1 - case["window"]) if case["window"] else 0: first] = True
            seen[i, torch.tensor(nodes) + first] = True
        hidden = ~seen.cuda().repeat_interleave(hq // hk, 0)
        pages = s["table"][b, : -(-t // page)].long()
        for h in range(hk):
            k, v = ((value[x].view(torch.uint8)[pages, h].view(E4M3).double() if value[x].dtype is E4M3 else value[x][pages, h])
                    * scale[x][pages, h].double()[:, None, None] for x in "kv")
            k, v = k.reshape(-1, d)[:t], v.reshape(-1, d)[:t]
            part = q[row: row + n, h * (hq // hk): (h + 1) * (hq // hk)].double()
            z = (part.reshape(-1, d) @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            o[row: row + n, h * (hq // hk): (h + 1) * (hq // hk)] = (torch.softmax(z, 1) @ v).reshape(part.shape)
        row += n
    return o


def _chains(s):
    """Each node's ancestors with itself, by sequence."""
    parents, cu = s["parents"].tolist(), s["cu"].tolist()
    chains = []
    for b in range(len(cu) - 1):
        mine = []
        for p in parents[cu[b]: cu[b + 1]]:
            mine.append((mine[p] if p >= 0 else []) + [len(mine)])
        chains.append(mine)
    return chains


def exact(case, seed):
    w = work(case)
    if w["flops"] > 4e12 or w["bytes"] > 4e9:
        return None
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    if kind == "tree":
        chains = _chains(s)
        totals = list(zip(*_lengths(case)))

        def see(b, i):
            return chains[b][i], totals[b][1] - totals[b][0] + len(chains[b][i]) - 1

        return {"o": _exact_attend(s, s["q"], s["cache"], {n: s["cache"][n + "_scale"] for n in "kv"}, see)}
    if kind == "step":
        return _exact_step(s)
    value = {n: s["stack"][n].float().double() for n in "kv"}
    scale = {n: s["stack"][n + "_scale"].double() for n in "kv"}
    out = {}
    if kind == "copy":
        for at, to in zip(s["sources"].tolist(), s["targets"].tolist()):
            for x in (*value.values(), *scale.values()):
                x[:, to] = x[:, at]
    elif kind == "keep":
        _exact_keep(s, value, scale, s["kept"].tolist(), s["counts"].tolist())
    else:
        # the pages in a dictionary of holders, row by row
        table, lengths, parents = s["table"].tolist(), s["lengths"].tolist(), s["parents"].tolist()
        free = iter([p for p, n in enumerate(s["holders"].tolist()) if n == 0])
        heard = set()
        for p in parents:
            if p < 0:
                continue
            eldest = p not in heard
            heard.add(p)
            first, last = lengths[p] // page, (lengths[p] + case["room"] - 1) // page
            for slot in range(first, min(last + 1, len(table[p]))):
                old = table[p][slot]
                if old >= 0 and eldest and int(s["holders"][old]) == 1:
                    continue
                fresh = next(free)
                if slot == first and lengths[p] % page and old >= 0:
                    for n in "kv":
                        value[n][:, fresh, :, : lengths[p] % page] = value[n][:, old, :, : lengths[p] % page]
                        scale[n][:, fresh] = scale[n][:, old]
    return out | {**value, **{n + "_scale": x for n, x in scale.items()}}


def _exact_step(s):
    case = s["case"]
    d, page = case["dim"], case["page"]
    value = {n: s["cache"][n].float().double() for n in "kv"}
    scale = {n: s["cache"][n + "_scale"].double() for n in "kv"}
    vectors = {n: s[n].double() for n in "qkv"}
    if case["qk_norm"]:
        for n, weight in zip("qk", s["norms"]):
            x = vectors[n]
            vectors[n] = x / (x.pow(2).mean(2, keepdim=True) + 1e-6).sqrt() * weight.double()
    chains, table = _chains(s), s["cos_sin"].double()
    turned = {"q": torch.zeros_like(vectors["q"]), "k": vectors["k"].clone()}
    row, kept, counts = 0, [], []
    tokens, targets = s["tokens"].tolist(), s["targets"].tolist()
    for b, (n, t) in enumerate(zip(*_lengths(case))):
        first = t - n
        at = torch.tensor([first + len(c) - 1 for c in chains[b]], device="cuda")
        cos, sin = table[at, None, : d // 2], table[at, None, d // 2:]
        for name in "qk":
            x = vectors[name][row: row + n]
            turned[name][row: row + n] = torch.cat((x[..., : d // 2] * cos - x[..., d // 2:] * sin,
                                                    x[..., d // 2:] * cos + x[..., : d // 2] * sin), -1)
        for slot in range(first // page, (t - 1) // page + 1):
            low, high = max(first, slot * page), min(t, slot * page + page)  # tokens stored in this page
            p, before = int(s["table"][b, slot]), low - slot * page
            for name, x in (("k", turned["k"]), ("v", vectors["v"])):
                part = x[row + low - first: row + high - first].transpose(0, 1)
                fresh = torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)).clamp(min=1e-12) / 448)))
                if before:
                    fresh = torch.maximum(fresh, scale[name][p])
                    value[name][p, :, :before] = _to_e4m3(value[name][p, :, :before] * (scale[name][p] / fresh)[:, None, None])
                scale[name][p] = fresh
                value[name][p, :, before: high - slot * page] = _to_e4m3(part / fresh[:, None, None])
        walk = [0]
        while (right := [i for i, c in enumerate(chains[b]) if len(c) > 1 and c[-2] == walk[-1]
                         and tokens[row + i] == targets[row + walk[-1]]]):
            walk.append(right[0])
        kept.append(walk)
        counts.append(len(walk))
        row += n
    totals = list(zip(*_lengths(case)))

    def see(b, i):
        return chains[b][i], totals[b][1] - totals[b][0] + len(chains[b][i]) - 1

    o = _exact_attend(s, turned["q"].to(s["q"].dtype), value, scale, see)
    value, scale = {n: x[None] for n, x in value.items()}, {n: x[None] for n, x in scale.items()}
    _exact_keep(s, value, scale, kept, counts)
    return {"q": turned["q"], "o": o, **{n: x[0] for n, x in value.items()},
            **{n + "_scale": x[0] for n, x in scale.items()}}
