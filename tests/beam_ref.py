"""Plain references of beam search's selection (float64) and of the page pool's operators (whole numbers)."""

import math

import torch


def candidates(logits, scores, most):
    """The first `most` candidates of one request, best first: (score, beam, logit, token).  logits [beams, vocab] and
    scores [beams] in float64."""
    x, vocab = logits, logits.shape[1]
    bad = ~scores.isfinite() | x.isnan().any(1) | (x == math.inf).any(1) | (x == -math.inf).all(1)
    x = torch.where(bad[:, None], -math.inf, x)
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    total = torch.where(bad[:, None], -math.inf, scores[:, None] + (x - lse)).flatten()
    x = x.flatten()
    keep = torch.nonzero(total.float().isfinite())[:, 0]  # by beam and token
    for key in (-x, torch.div(torch.arange(x.numel()), vocab, rounding_mode="floor"), -total):  # least important first
        keep = keep[torch.sort(key[keep], stable=True).indices]
    keep = keep[:most].tolist()
    return [(float(total[i]), i // vocab, float(x[i]), i % vocab) for i in keep]


def beam_step(logits, scores, ends):
    """(tokens, parents, scores, ended tokens, ended parents, ended scores, the least distance between the scores of two
    beams' candidates whose order matters)."""
    out, gap = [[] for _ in range(6)], math.inf
    beams = scores.shape[1]
    for r in range(scores.shape[0]):
        ranked = candidates(logits[r].double(), scores[r].double(), beams * (len(ends) + 1) + 1)
        runs = [f for f in ranked if f[3] not in ends][:beams]
        over = [f for f in ranked[:beams] if f[3] in ends]
        seen = 0
        for a, b in zip(ranked, ranked[1:]):
            if a[1] != b[1] and a[0] != b[0]:
                gap = min(gap, a[0] - b[0])
            seen += a[3] not in ends
            if seen > beams:
                break
        for at, chosen in ((0, runs), (3, over)):
            pad = beams - len(chosen)
            out[at].append([f[3] for f in chosen] + [-1] * pad)
            out[at + 1].append([f[1] for f in chosen] + [-1] * pad)
            out[at + 2].append([f[0] for f in chosen] + [-math.inf] * pad)
    return [*out, gap]


def score_bound(score, vocab):
    """How far a score may be off: its own rounding; a term's exp (one step), its argument (m - x roundings of half a
    step each, at most ln vocab on average) and three additions of eight terms."""
    return 2.0 ** -24 * abs(score) + 2.0 ** -23 * (4 + math.log(vocab))


def pages_of(length, page, width):
    return min(-(-max(length, 0) // page), width)


def reorder(parents, table, lens, shares, free, count, page):
    """The rules of l20_reorder_block_tables on lists; (table, lens, shares, free, count, pairs, short)."""
    groups, beams = len(parents), len(parents[0]) if parents else 0
    width, pages, pool = len(table[0]) if table else 0, len(shares), len(free)
    table, shares, free = [list(r) for r in table], list(shares), list(free)
    new_table, new_lens, change, wanted = [list(r) for r in table], [], {}, []
    for g in range(groups):
        alive = [q if 0 <= q < beams else -1 for q in parents[g]]
        for i in range(beams):
            row, q = g * beams + i, alive[i]
            for v in table[row][:pages_of(lens[row], page, width)]:
                if 0 <= v < pages:
                    change[v] = change.get(v, 0) - 1
            length = max(lens[g * beams + q], 0) if q >= 0 else 0
            new_lens.append(length)
            if q < 0:
                continue
            source = table[g * beams + q]
            keeper = q if alive[q] == q else alive.index(q)
            own = length // page if length % page and keeper != i and length // page < width else -1
            for c in range(pages_of(length, page, width)):
                if c == own and 0 <= source[c] < pages:
                    wanted.append((row, c, source[c], length % page))
                    continue
                new_table[row][c] = source[c]
                if 0 <= source[c] < pages:
                    change[source[c]] = change.get(source[c], 0) + 1
    freed = []
    for v, d in change.items():
        if d:
            shares[v] += d
            if shares[v] == -1:
                shares[v] = 0
                freed.append(v)
    count = min(max(count, 0), pool)
    for v in sorted(freed):
        if count < pool:
            free[count] = v
            count += 1
    pairs, short = [], 0
    for row, c, source, tokens in wanted:
        got = -1
        if count:
            count -= 1
            got = free[count] if 0 <= free[count] < pages else -1
        new_table[row][c] = got
        if got >= 0:
            pairs.append((source, got, tokens))
        else:
            short += 1
    return new_table, new_lens, shares, free, count, pairs, short


def compact(limit, table, lens, shares, free, count, page, room):
    """The rules of l20_compact_pages on lists; (table, shares, free, count, pairs, left behind)."""
    width, pages, pool = len(table[0]) if table else 0, len(shares), len(free)
    table, shares, free = [list(r) for r in table], list(shares), list(free)
    count = min(max(count, 0), pool)
    high = sorted({v for r, n in zip(table, lens) for v in r[:pages_of(n, page, width)] if limit <= v < pages})
    low = sorted({v for v in free[:count] if 0 <= v < limit})
    moves = min(len(high), len(low), room)
    to = dict(zip(high[:moves], low[:moves]))
    for r, n in zip(table, lens):
        for c in range(pages_of(n, page, width)):
            r[c] = to.get(r[c], r[c])
    for a, b in to.items():
        shares[b], shares[a] = shares[a], 0
    rest = low[moves:][::-1]
    free[:len(rest)] = rest
    return table, shares, free, len(rest), [(a, b, page) for a, b in to.items()], len(high) - moves
