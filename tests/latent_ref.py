"""Float64 references of latent attention and the block-table builder, and the bounds their tests hold
kernels to.

A rounding is off by at most half a step: ``half(t)`` = eps / 2 relative (2^-8 bf16, 2^-11 fp16).  The attention
kernels round P once for the product with V and the result once; scores, sums and accumulators are fp32."""

import math

import torch

ROPE = 64


def half(dtype):
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, visible, scale, dtype):
    """q [R, dk], k [L, dk], v [L, dv] float64, visible [R, L] bool -> (out, lse, out bound, lse bound).

    The bound of an output element, |v| averaged with the row's weights as a:
      half |out|              its own rounding
      half a                  P's rounding, each weight off by at most half
      2 d a                   scores off by at most d: dk fp32 additions of products that are exact in fp32
                              (dk 2^-24 sum |q k| scale), and the exponent's own error (exp2 of a number of up to
                              |s| units rounded to fp32, 2^-23 |s|; numerator and denominator)
      L 2^-24 a               the fp32 sums over keys
      fp16: 2^-25 sum |v|     weights below 2^-14 of the largest are rounded to the subnormal grid
    """
    s = (q @ k.T) * scale
    s = s.masked_fill(~visible, -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    p = torch.where(visible, torch.exp(s - lse.clamp_min(-1e300)[:, None]), torch.zeros_like(s))
    out = p @ v
    a = p @ v.abs()
    spread = ((q.abs() @ k.abs().T) * scale).masked_fill(~visible, 0.0).amax(dim=-1) if k.shape[0] else q.new_zeros(q.shape[0])
    d = (k.shape[1] * 2.0 ** -24 + 2.0 ** -23) * spread + 2.0 ** -22
    h = half(dtype)
    bound = h * out.abs() + (h + 2 * d[:, None] + (k.shape[0] + 64) * 2.0 ** -24) * a
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (visible.double() @ v.abs()) + 2.0 ** -25
    lse_bound = d + 2.0 ** -22 * lse.abs().nan_to_num(0, 0, 0) + (k.shape[0] + 64) * 2.0 ** -24
    return out, lse, bound * 1.01, lse_bound


def assert_rows(got, got_lse, want, lse, bound, lse_bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} elements off, worst {float((err / bound.clamp_min(1e-30)).max()):.2f} bounds"
    if got_lse is not None:
        empty = torch.isinf(lse)
        assert torch.equal(torch.isinf(got_lse), empty) and bool((got_lse[empty] < 0).all()), what
        off = (got_lse.double() - lse).abs()[~empty]
        assert bool((off <= lse_bound[~empty]).all()), f"{what}: lse off by {float(off.max()):.2e}"


def rows_of_cache(cache, table, b, tokens, scale):
    """The first `tokens` rows of sequence b in float64, and which of them lie on pages inside the cache."""
    page = cache.shape[1]
    t = torch.arange(tokens, device=cache.device)
    col = t // page
    inside = col < table.shape[1]
    ids = table[b, col.clamp_max(table.shape[1] - 1)].long()
    inside &= (ids >= 0) & (ids < cache.shape[0])
    flat = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    rows = flat[ids.clamp(0, cache.shape[0] - 1), t % page]
    rows = rows.view(cache.dtype) if cache.element_size() == 1 else rows
    rows = rows.double() * scale
    return torch.where(inside[:, None], rows, torch.zeros_like(rows)), inside


def check_decode(got, got_lse, query, cache, table, lens, rank, q_len, softmax_scale, cache_scale, max_len=None):
    heads = query.shape[1]
    for b, length in enumerate(lens.tolist()):
        tokens = min(max(length, 0), table.shape[1] * cache.shape[1], max_len if max_len is not None else 1 << 60)
        rows, inside = rows_of_cache(cache, table, b, tokens, cache_scale)
        t = torch.arange(tokens, device=query.device)
        for i in range(q_len):
            r = b * q_len + i
            visible = (inside & (t <= length - q_len + i)).expand(heads, tokens)
            want = attend(query[r].double(), rows, rows[:, :rank], visible, softmax_scale, query.dtype)
            assert_rows(got[r], None if got_lse is None else got_lse[r], *want, f"sequence {b} row {i}")


def check_prompt(got, got_lse, query, key, key_rope, value, cu_q, cu_k, softmax_scale, causal=True):
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        n, m = q1 - q0, k1 - k0
        visible = torch.ones(n, m, dtype=torch.bool, device=query.device)
        if causal:
            visible = visible.tril(m - n)
        for h in range(query.shape[1]):
            k = torch.cat([key[k0:k1, h], key_rope[k0:k1]], dim=-1).double()
            want = attend(query[q0:q1, h].double(), k, value[k0:k1, h].double(), visible, softmax_scale, query.dtype)
            assert_rows(got[q0:q1, h], None if got_lse is None else got_lse[q0:q1, h], *want, f"sequence {b} head {h}")


def block_tables(cached, new, table, free, count, tokens, page):
    """The builder in plain Python: lists in, a dict of lists out."""
    table, stack = [list(row) for row in table], list(free[:count])
    width, pool = len(table[0]), len(free)
    cached = [max(c, 0) for c in cached]
    for b, n in enumerate(new):
        if n < 0:
            stack += table[b][:min(-(-cached[b] // page), width)]
    stack = stack[:pool]
    free = stack + list(free[len(stack):])
    cu, seq_lens, served, dry = [0], [], [], False
    for b, n in enumerate(new):
        c, n_tok = cached[b], max(n, 0)
        cu.append(cu[-1] + n_tok)
        held, total = -(-c // page), -(-(c + n_tok) // page)
        ok = n >= 0 and total <= width and cu[-1] <= tokens
        if ok and total > held:
            if dry or total - held > len(stack):
                ok, dry = False, True
            else:
                for k in range(held, total):
                    table[b][k] = stack.pop()
        served.append(ok)
        seq_lens.append(c + n_tok if ok else (0 if n < 0 else c))
    slots, positions = [-1] * tokens, [0] * tokens
    for b, n in enumerate(new):
        for k in range(max(n, 0)):
            t, pos = cu[b] + k, cached[b] + k
            if t < tokens:
                positions[t] = pos
                if served[b]:
                    slots[t] = table[b][pos // page] * page + pos % page
    return {"table": table, "free": free, "left": len(stack), "slots": slots, "positions": positions,
            "cu": [min(c, tokens) for c in cu], "seq_lens": seq_lens}
