"""Definitions of drafted trees, kept tokens and forked sequences, row by row in Python
(none of the package's code); codes and scales in 64 bits as in ``oracle/attention.py``."""

from __future__ import annotations

import torch

from oracle.attention import to_e4m3


def spans(rows, cu):
    """(first row, rows) of each sequence."""

    cu = [min(max(int(c), 0), rows) for c in cu]
    return [(lo, max(hi - lo, 0)) for lo, hi in zip(cu, cu[1:])]


def chains(parents, row, n):
    """Each node's ancestors from the root on, itself last."""

    out = []
    for i in range(n):
        p = int(parents[row + i])
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def tree(parents, cu, lengths, most, window=0):
    """``(seen, positions)``: the set of new tokens that each row sees, and its position or -1."""

    rows = parents.shape[0]
    seen, positions = [set() for _ in range(rows)], [-1] * rows
    for (row, n), length in zip(spans(rows, cu), lengths.tolist()):
        first = max(length, 0) - n
        for i, chain in enumerate(chains(parents, row, min(n, most))):
            position = first + len(chain) - 1
            if first + i >= 0 and position >= 0:
                positions[row + i] = position
                seen[row + i] = {j for j in chain if not window or len(chain) - 1 - chain.index(j) < window}
    return seen, positions


def unpack(mask):
    """The set bits of each row."""

    return [{j for j in range(32 * mask.shape[1]) if int(mask[r, j // 32]) >> (j % 32) & 1} for r in range(mask.shape[0])]


def pack(seen, words):
    mask = torch.zeros((len(seen), words), dtype=torch.int64)
    for r, bits in enumerate(seen):
        for j in bits:
            if j < 32 * words:
                mask[r, j // 32] |= 1 << j % 32
    return torch.where(mask >= 2**31, mask - 2**32, mask).to(torch.int32)


def seen_by(seen, positions, window=0):
    """For ``oracle.attention.attend``: tokens before the new ones, and those in ``seen``."""

    def of(row, n, first, tokens):
        out = torch.zeros((n, tokens), dtype=torch.bool)
        for i in range(n):
            if int(positions[row + i]) < 0:
                continue
            begin = max(max(int(positions[row + i]), first) - window + 1, 0) if window else 0
            out[i, begin: max(min(first, tokens), 0)] = True
            for j in seen[row + i]:
                if 0 <= first + j < tokens:
                    out[i, first + j] = True
        return out

    return of


def walk(tokens, targets, parents, cu, most):
    """``[(kept, following)]`` of each sequence."""

    out = []
    for row, n in spans(tokens.shape[0], cu):
        n = min(n, most)
        kept = [0] if n else []
        while kept:
            right = [i for i in range(kept[-1] + 1, n)
                     if int(parents[row + i]) == kept[-1] and int(tokens[row + i]) == int(targets[row + kept[-1]])]
            if not right:
                break
            kept.append(right[0])
        out.append((kept, int(targets[row + kept[-1]]) if kept else -1))
    return out


def keep(cache, table, cu, lengths, kept, counts):
    """``(new cache, new lengths)``; a cache as in ``oracle.attention``."""

    new = {n: t.clone() for n, t in cache.items()}
    pages, _, page, _ = cache["k"].shape
    out = []
    for s, (row, n) in enumerate(spans(1 << 24, cu)):
        first = max(int(lengths[s]), 0) - n
        before = max(first, 0)

        def at(t):
            slot = t // page
            p = int(table[s, slot]) if slot < table.shape[1] else -1
            return (p, t % page) if 0 <= p < pages else None

        nodes = []
        for i, node in enumerate(kept[s, : max(int(counts[s]), 0)].tolist()):
            above = nodes[-1] if nodes else -1
            if first < 0 or node <= above or node >= min(n, 1024) or at(first + node) is None or at(first + i) is None:
                break
            nodes.append(node)
        out.append(before + len(nodes))
        if not nodes:
            continue
        holds = {}  # page -> {slot: (page, slot) that its token is in now}
        for i, node in enumerate(nodes):
            p, slot = at(first + i)
            holds.setdefault(p, {})[slot] = at(first + node)
        p = at(first)[0]
        for slot in range(first % page):
            holds[p][slot] = (p, slot)
        for p, tokens in holds.items():
            for name in "kv":
                scale = torch.stack([cache[name + "_scale"][q] for q, _ in tokens.values()]).amax(0)
                new[name + "_scale"][p] = scale
                for slot, (q, of) in tokens.items():
                    new[name][p, :, slot] = to_e4m3(cache[name][q, :, of] * (cache[name + "_scale"][q] / scale)[:, None])
    return new, out


def fork(holders, table, lengths, parents, room, page):
    """``(new table, new lengths, new holders, copies, missing)``; copies are (from, to, tokens)."""

    pages, width = holders.shape[0], table.shape[1]

    def entry(s, slot):
        p = int(table[s, slot])
        return p if 0 <= p < pages else -1

    free = [p for p in range(pages) if int(holders[p]) == 0]
    new, out, copies, heard, missing = [], [], [], set(), 0
    for s in parents.tolist():
        row = [-1] * width
        if not 0 <= s < table.shape[0]:
            new.append(row)
            out.append(0)
            continue
        length = max(int(lengths[s]), 0)
        out.append(length)
        for slot in range(width):
            lo, hi = slot * page, (slot + 1) * page
            if hi <= length or (room == 0 and lo < length):
                row[slot] = entry(s, slot)
            elif lo < length + room:
                old = entry(s, slot)
                if s not in heard and old >= 0 and int(holders[old]) == 1:
                    row[slot] = old
                elif free:
                    row[slot] = free.pop(0)
                    if lo < length and old >= 0:
                        copies.append((old, row[slot], length - lo))
                else:
                    missing += 1
        heard.add(s)
        new.append(row)
    held = holders.tolist()
    for s in range(table.shape[0]):
        for slot in range(width):
            if entry(s, slot) >= 0:
                held[entry(s, slot)] -= 1
    for row in new:
        for p in row:
            if p >= 0:
                held[p] += 1
    return new, out, held, copies, missing
