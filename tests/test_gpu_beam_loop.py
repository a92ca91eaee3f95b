"""GPU: beam search over the paged cache -- block tables, cache producer, paged attention, selection, rows that follow
their parents, copies of pages, compaction -- against every hypothesis's own keys and values in float64."""

import math

import pytest
import torch

import beam_ref as R

pytestmark = pytest.mark.gpu
PAGE, BEAMS, VOCAB, HEADS, KV, DIM, LAYERS, END = 16, 4, 211, 6, 2, 64, 2, 3


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")


def attend(q, k, v):
    """q [HEADS, DIM], k and v [tokens, KV, DIM] in float64."""
    k, v = (x.repeat_interleave(HEADS // KV, dim=1).transpose(0, 1) for x in (k, v))
    p = torch.softmax((k @ q[:, :, None])[..., 0] * DIM ** -0.5, dim=-1)
    return (p[:, None, :] @ v)[:, 0]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_a_search(fp8):
    import l20_beam_search as bs
    import l20_block_tables as bt
    import l20_paged_split_kv as kv
    import l20_rope_kv as rope

    dtype, prompts, steps, pool = torch.bfloat16, [37, 16, 5], 24, 96
    groups, rows, width = len(prompts), len(prompts) * BEAMS, 6
    g = torch.Generator().manual_seed(12)
    rand = lambda *shape: torch.randn(*shape, generator=g).to(dtype).cuda()  # noqa: E731
    theta = torch.rand(200, DIM // 2, generator=g) * 6.28
    cs = torch.cat([theta.cos(), theta.sin()], -1).cuda()
    scale = 1 / 32.0 if fp8 else 1.0
    # a layer's query, key and value of a token; the head reads the layers' outputs
    table_of = [[rand(VOCAB, n, DIM) for n in (HEADS, KV, KV)] for _ in range(LAYERS)]
    head = torch.randn(LAYERS * HEADS * DIM, VOCAB, generator=g).cuda() / 4
    caches = [torch.full((pool, 2, PAGE, KV, DIM), float("nan")).to(torch.float8_e4m3fn if fp8 else dtype).cuda()
              for _ in range(LAYERS)]
    views = [v for c in caches for v in c.unbind(1)]
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    lens, shares = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(pool, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, generator=g).to(torch.int32).cuda()
    count = torch.tensor([pool], dtype=torch.int32, device="cuda")
    cu, grown = torch.zeros(rows + 1, dtype=torch.int32, device="cuda"), torch.zeros_like(lens)
    copies = bt.PageCopies.empty(rows, "cuda")
    scores = torch.full((groups, BEAMS), -math.inf)
    scores[:, 0] = 0.0
    scores = scores.cuda()
    texts = [torch.randint(0, VOCAB, (prompts[r // BEAMS],), generator=g).tolist() if r % BEAMS == 0 else [] for r in range(rows)]
    fed = [list(t) for t in texts]  # what a row appends to the cache in this step
    held = [[[torch.zeros(0, KV, DIM, dtype=torch.float64, device="cuda")] * 2 for _ in range(LAYERS)] for _ in range(rows)]

    def stored(x):
        return (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn).double() * scale if fp8 else x.double()

    def append():
        new = torch.tensor([len(f) for f in fed], dtype=torch.int32, device="cuda")
        tokens = torch.tensor([t for f in fed for t in f], device="cuda")
        n = len(tokens)
        slots, positions = (torch.zeros(n, dtype=torch.int64, device="cuda") for _ in range(2))
        bt.l20_build_block_tables(lens, new, table, free, count, slots, positions, cu, grown, PAGE)
        lens.copy_(grown)
        at, outs = cu.tolist(), []
        for layer in range(LAYERS):
            q, k, v = (t[tokens] for t in table_of[layer])
            kc, vc = caches[layer].unbind(1)
            rope.l20_rope_and_cache(q, k, v, positions, cs, True, kc, vc, slots, k_scale=scale, v_scale=scale)
            last = torch.tensor([max(at[r + 1] - 1, 0) for r in range(rows)], device="cuda")
            query = q[last].contiguous()
            if fp8:
                out = kv.l20_paged_split_kv_attention_fp8(query, kc, vc, table, lens, k_scale=scale, v_scale=scale,
                                                          max_seq_len=width * PAGE)
            else:
                out = kv.l20_paged_split_kv_attention(query, kc, vc, table, lens, max_seq_len=width * PAGE)
            for r in range(rows):
                held[r][layer] = [torch.cat([h, stored(x[at[r]:at[r + 1]])]) for h, x in zip(held[r][layer], (k, v))]
                if fed[r]:
                    want = attend(query[r].double(), *held[r][layer])
                    # the output's rounding, and fp32 sums of probabilities and products (a part in 2^12 of the values)
                    bound = 2.0 ** -8 * want.abs() + 2.0 ** -12 * held[r][layer][1].abs().max()
                    assert ((out[r].double() - want).abs() <= bound).all(), (r, layer, len(texts[r]))
            outs.append(out.flatten(1))
        assert lens.tolist() == [len(t) for t in texts]
        return torch.cat(outs, -1).float() @ head

    finished = []
    for step in range(steps):
        if not any(fed):
            break
        logits = append()
        if step == 9:  # a request is given up: its beams die, its pages go back
            scores[1] = -math.inf
        if step == 5:
            logits[:, END] += 12
        out = bs.l20_beam_search_step(logits, scores, end_tokens=[END])
        want = R.beam_step(logits.view(groups, BEAMS, VOCAB).cpu(), scores.cpu(), [END])
        assert want[6] > 1e-6
        assert (out.tokens.tolist(), out.parents.tolist()) == (want[0], want[1])
        assert (out.ended_tokens.tolist(), out.ended_parents.tolist()) == (want[3], want[4])
        scores = out.scores
        finished += [texts[b * BEAMS + q] for b in range(groups) for q in want[4][b] if q >= 0]
        bt.l20_reorder_block_tables(out.parents, table, lens, shares, free, count, PAGE, copies=copies)
        bt.l20_copy_pages(copies, views)
        assert int(copies.count[1]) == 0
        # each row goes on with its parent's text, keys and values
        source = [b * BEAMS + q if q >= 0 else -1 for b in range(groups) for q in want[1][b]]
        fed = [[t] if t >= 0 else [] for b in range(groups) for t in want[0][b]]
        texts = [texts[s] + f if s >= 0 else [] for s, f in zip(source, fed)]
        held = [[list(layer) for layer in held[s]] if s >= 0 else
                [[h[:0] for h in layer] for layer in held[r]] for r, s in enumerate(source)]
        if step == 14:  # the pool shrinks to what is held and a few pages to go on with
            limit = pool - int(count) + 12
            moves = bt.l20_compact_pages(limit, table, lens, shares, free, count, PAGE)
            bt.l20_copy_pages(moves, views)
            assert int(moves.count[0]) > 0 and int(moves.count[1]) == 0 and int(count) == 12
            for c in caches:  # nothing is read beyond the limit any more
                c[limit:] = torch.full((1,), float("nan")).to(c.dtype).cuda()
    assert any(finished) and step == steps - 1
    assert not any(texts[BEAMS:2 * BEAMS]) and all(texts[:BEAMS]) and all(texts[2 * BEAMS:])
    gone = torch.full((groups, BEAMS), -1, dtype=torch.int32, device="cuda")
    bt.l20_reorder_block_tables(gone, table, lens, shares, free, count, PAGE, copies=copies)
    assert sorted(free[:int(count)].tolist()) == list(range(limit)) and not shares.any() and not lens.any()
