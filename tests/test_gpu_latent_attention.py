"""GPU: latent attention over a paged cache and over expanded prompts against float64, with bounds derived in
latent_ref.attend."""

import math

import pytest
import torch

import latent_ref as R

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")
    import l20_latent_attention  # noqa: F401


def make_decode(lens, heads, q_len=1, rank=512, dtype=torch.bfloat16, fp8=False, page=16, seed=0, spare=3, poison=True):
    """A paged cache whose cells outside the sequences hold NaN (poison), pages in random order."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-max(n, 0) // page) for n in lens]
    pool, width = sum(held) + spare, max(held + [1]) + 2
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.randint(0, pool, (len(lens), width), generator=g, dtype=torch.int32)
    cache = torch.full((pool, page, rank + 64), float("nan") if poison else 0.0)
    at = 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
        for k in range(held[b]):
            rows = min(page, n - k * page)
            cache[table[b, k].long(), :rows] = torch.randn(rows, rank + 64, generator=g)
    scale = 1.0
    if fp8:
        scale = 1.0 / 32
        cache = (cache / scale).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        cache = cache.to(dtype)
    query = torch.randn(len(lens) * q_len, heads, rank + 64, generator=g).to(dtype)
    return {"query": query.cuda(), "cache": cache.cuda(), "table": table.cuda(), "rank": rank, "q_len": q_len,
            "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "cache_scale": scale}


def run_decode(c, lse=True, **kw):
    import l20_latent_attention as la

    rows, heads = c["query"].shape[:2]
    out_lse = torch.empty(rows, heads, dtype=torch.float32, device="cuda") if lse else None
    out = la.l20_paged_latent_attention(c["query"], c["cache"], c["table"], c["lens"], softmax_scale=SCALE,
                                        kv_rank=c["rank"], cache_scale=c["cache_scale"], q_len=c["q_len"], lse=out_lse, **kw)
    torch.cuda.synchronize()
    return out, out_lse


def check_decode(c, out, lse, **kw):
    R.check_decode(out, lse, c["query"], c["cache"], c["table"], c["lens"], c["rank"], c["q_len"], SCALE, c["cache_scale"], **kw)


EDGES = [1, 15, 16, 17, 63, 64, 65, 127, 300]
DECODE = [
    # lens, heads, q_len, rank, page
    (EDGES, 16, 1, 512, 16),
    (EDGES, 5, 1, 256, 32),
    ([700, 3], 28, 1, 512, 64),        # two blocks of 16 rows, the second ragged
    ([130, 1, 64], 64, 1, 512, 16),    # four
    ([100, 65], 128, 1, 512, 16),      # eight, two workgroups a run
    ([90, 33, 200], 7, 5, 256, 48),    # rows of several drafts in a block
    ([70, 5], 20, 4, 512, 16),
    ([2000], 16, 1, 512, 16),          # one sequence over many runs
    ([1, 2, 0, 3], 9, 3, 512, 16),     # fewer tokens than drafts, and none
]


@pytest.mark.parametrize("spec", DECODE, ids=[f"{len(s[0])}x{max(s[0])}_h{s[1]}_q{s[2]}_r{s[3]}_p{s[4]}" for s in DECODE])
@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                       (torch.float16, True)], ids=["bf16", "fp16", "bf16_e4m3", "fp16_e4m3"])
@pytest.mark.parametrize("rows", [16, 32, 64], ids=["rows16", "rows32", "rows64"])
def test_decode_against_float64(spec, dtype, fp8, rows):
    """The bound on the lengths says how much work there may be, and so how many rows a workgroup takes."""
    lens, heads, q_len, rank, page = spec
    c = make_decode(lens, heads, q_len, rank, dtype, fp8, page, seed=sum(lens) + heads)
    units = len(lens) * -(-heads * q_len // 16)
    tiles = {16: 0, 32: 5000, 64: 20000}[rows] // units
    check_decode(c, *run_decode(c, max_seq_len=max(c["table"].shape[1] * page, tiles * (64 if fp8 else 32))))


def test_decode_many_short_sequences_share_runs():
    """More sequences than runs: whole ones, and ones cut at a run's end, of every length about a tile."""
    lens = [(37 * i) % 200 for i in range(600)]
    c = make_decode(lens, 16, rank=256, seed=5)
    check_decode(c, *run_decode(c))
    check_decode(c, *run_decode(c, max_seq_len=1000))


@pytest.mark.parametrize("heads,q_len,batch", [(64, 1, 300), (16, 2, 270), (30, 3, 90)], ids=["64", "2x16", "3x30"])
@pytest.mark.parametrize("fp8", [True, False], ids=["e4m3", "model"])
def test_decode_many_short_sequences_whole(heads, q_len, batch, fp8):
    """Workgroups of 64 and 32 rows that take a sequence each."""
    lens = [(13 * i) % 90 for i in range(batch)]
    c = make_decode(lens, heads, q_len, fp8=fp8, seed=35)
    check_decode(c, *run_decode(c))


def test_decode_masks_what_the_table_does_not_hold():
    """Pages below 0 or beyond the cache, lengths beyond the table and beyond max_seq_len."""
    c = make_decode([200, 100, 90, 64], 16, seed=6, poison=False)
    c["table"][0, 3] = -1
    c["table"][0, 5] = c["cache"].shape[0]
    c["table"][1, 0] = 2 ** 31 - 1
    c["table"][2, :] = -7  # nothing of it is there
    c["lens"][3] = 100000
    out, lse = run_decode(c)
    check_decode(c, out, lse)
    assert bool((out[2] == 0).all()) and bool(torch.isneginf(lse[2]).all())
    out, lse = run_decode(c, max_seq_len=70)
    check_decode(c, out, lse, max_len=70)


def test_decode_strided_views():
    """Query, output and LSE as views, a cache inside a wider allocation, the block table a slice."""
    import l20_latent_attention as la

    c = make_decode([80, 33], 12, page=16, seed=7)
    wide = torch.zeros(2, 15, 640, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:14, 64:] = c["query"]
    pool = torch.full((c["cache"].shape[0], 2, 16, 576), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool[:, 1] = c["cache"]
    table = torch.full((4, c["table"].shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    table[1:3, :c["table"].shape[1]] = c["table"]
    out = torch.full((2, 13, 600), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((12, 2), 7.0, device="cuda").t()
    la.l20_paged_latent_attention(wide[:, 2:14, 64:], pool[:, 1], table[1:3, :c["table"].shape[1]], c["lens"],
                                  softmax_scale=SCALE, output=out[:, 1:, 40:552], lse=lse)
    torch.cuda.synchronize()
    check_decode(c, out[:, 1:, 40:552], lse)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 1:, :40] == 7).all()) and bool((out[:, 1:, 552:] == 7).all())


def test_decode_large_scores_and_sinks():
    """Scores of hundreds: one token takes nearly all weight, in the first and in a late tile."""
    c = make_decode([500, 500], 16, seed=8, poison=False)
    c["query"] *= 8
    c["cache"][c["table"][0, 0].long(), 0] *= 12
    c["cache"][c["table"][1, 25].long(), 3] *= 12
    check_decode(c, *run_decode(c))


def test_decode_nan_in_one_sequence_stays_there():
    c = make_decode([100, 100, 100], 16, seed=9, poison=False)
    clean, _ = run_decode(c)
    c["cache"][c["table"][1, 2].long(), 5] = float("nan")
    out, _ = run_decode(c)
    assert bool(torch.isnan(out[1]).all())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


@pytest.mark.parametrize("fp8", [True, False], ids=["e4m3", "model"])
@pytest.mark.parametrize("heads", [5, 16, 40])
@pytest.mark.parametrize("rank", [512, 256])
@pytest.mark.parametrize("bound", [None, 100000], ids=["few", "long"])
def test_decode_nan_of_a_draft_reaches_only_the_rows_that_see_it(fp8, heads, rank, bound):
    """The last, and the second last, token of two sequences hold NaN; the rows before them are as without."""
    q_len = 3
    c = make_decode([70, 2, 129, 900, 64], heads, q_len=q_len, rank=rank, fp8=fp8, seed=31, poison=False)
    clean, clean_lse = run_decode(c, max_seq_len=bound)
    kept = c["cache"].clone()
    for b, t in ((0, 69), (2, 127), (3, 899), (4, 63)):
        c["cache"][c["table"][b, t // 16].long(), t % 16] = float("nan")
    out, lse = run_decode(c, max_seq_len=bound)
    c["cache"] = kept
    seen = torch.zeros(5, q_len, dtype=torch.bool, device="cuda")
    seen[[0, 2, 2, 3, 4], [2, 1, 2, 2, 2]] = True
    seen = seen.flatten()
    assert bool(torch.isnan(out[seen]).all()) and bool(torch.isnan(lse[seen]).all())
    out[seen], lse[seen] = clean[seen], clean_lse[seen]
    check_decode(c, out, lse)


def test_decode_one_sequence_one_page_of_any_stride():
    """The stride of a dimension of size 1 says nothing."""
    c = make_decode([15], 1, seed=32, spare=0)
    want, want_lse = run_decode(c)
    check_decode(c, want, want_lse)
    c["query"] = c["query"].as_strided((1, 1, 576), (7, 5, 1))
    c["cache"] = c["cache"].as_strided((1, 16, 576), (1, 576, 1))
    out, lse = run_decode(c, output=torch.empty(512, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 512), (3, 1, 1)))
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_two_decode_calls_at_once():
    """Two streams, a workspace each: what they give alone."""
    import l20_latent_attention as la

    cases = [make_decode([3000, 1, 2000, 700], 16, seed=33), make_decode([900] * 6, 40, q_len=2, fp8=True, seed=34)]
    want = [run_decode(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs, spaces = [torch.empty_like(w[0]) for w in want], []
    for c in cases:
        spaces.append(la.allocate_l20_paged_latent_workspace(c["query"], c["cache"], c["table"].shape[1] * 16, q_len=c["q_len"]))
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, o, ws in zip(cases, streams, outs, spaces):
            with torch.cuda.stream(s):
                la.l20_paged_latent_attention(c["query"], c["cache"], c["table"], c["lens"], softmax_scale=SCALE,
                                              cache_scale=c["cache_scale"], q_len=c["q_len"], output=o, workspace=ws)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w[0])


def test_decode_workspace_is_reused_and_calls_repeat_bitwise():
    import l20_latent_attention as la

    big, small = make_decode([3000, 64, 1500], 28, q_len=2, seed=10), make_decode([40, 900], 28, q_len=2, seed=11)
    ws = la.allocate_l20_paged_latent_workspace(big["query"], big["cache"], 3100, q_len=2)
    ws.fill_(255)  # NaN bit patterns
    a = run_decode(big, workspace=ws, max_seq_len=3100)
    b = run_decode(small, workspace=ws, max_seq_len=1000)
    again = run_decode(big, workspace=ws, max_seq_len=3100)
    check_decode(big, *a)
    check_decode(small, *b)
    assert torch.equal(a[0], again[0]) and torch.equal(a[1], again[1])


def test_decode_cache_offsets_beyond_32_bits():
    """A page pool of more than 4 GB: the pages in use lie at its end."""
    c = make_decode([200], 16, seed=12)
    pages = (5 << 30) // (16 * 576 * 2)
    pool = torch.empty(pages, 16, 576, dtype=torch.bfloat16, device="cuda")
    n = c["cache"].shape[0]
    pool[pages - n:] = c["cache"]
    small = c["cache"]
    out, lse = run_decode(c)
    c["cache"], c["table"] = pool, c["table"] + (pages - n)
    big_out, big_lse = run_decode(c)
    assert torch.equal(out, big_out) and torch.equal(lse, big_lse)
    c["cache"], c["table"] = small, c["table"] - (pages - n)
    check_decode(c, out, lse)


def test_decode_on_another_stream_and_in_a_graph():
    import l20_latent_attention as la

    c = make_decode([700, 64, 1, 0, 300], 20, seed=13)
    want, want_lse = run_decode(c, max_seq_len=800)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = run_decode(c, max_seq_len=800)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    ws = la.allocate_l20_paged_latent_workspace(c["query"], c["cache"], 800)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    graph = torch.cuda.CUDAGraph()

    def step():
        la.l20_paged_latent_attention(c["query"], c["cache"], c["table"], c["lens"], softmax_scale=SCALE, max_seq_len=800,
                                      output=out, workspace=ws, lse=lse)

    step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    base = c["lens"].clone()
    for k in range(4):  # lengths change between replays; eager calls between them
        c["lens"].copy_((base - 11 * k).clamp_min(0))
        out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_lse = run_decode(c, max_seq_len=800)
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse)
        check_decode(c, out, lse)


# --------------------------------------------------------------------------- prompts
def make_prompt(lens, keys, heads, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    cu_q, cu_k = [0], [0]
    for n, k in zip(lens, keys):
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + k)
    up = torch.randn(cu_k[-1], heads, 256, generator=g).to(dtype).cuda()
    return {"query": torch.randn(cu_q[-1], heads, 192, generator=g).to(dtype).cuda(), "key": up[..., :128],
            "value": up[..., 128:], "key_rope": torch.randn(cu_k[-1], 64, generator=g).to(dtype).cuda(),
            "cu_q": torch.tensor(cu_q, dtype=torch.int32).cuda(), "cu_k": torch.tensor(cu_k, dtype=torch.int32).cuda(),
            "max_q": max(lens)}


def run_prompt(c, causal=True, **kw):
    import l20_latent_attention as la

    lse = torch.full(c["query"].shape[:2], 5.0, device="cuda")
    out = la.l20_latent_prompt_attention(c["query"], c["key"], c["key_rope"], c["value"], c["cu_q"], c["cu_k"], c["max_q"],
                                         causal=causal, lse=lse, **kw)
    torch.cuda.synchronize()
    return out, lse


PROMPT = [
    ([1, 130, 64, 17], [1, 130, 64, 17], 3),
    ([63, 65, 127, 129], [63, 65, 127, 129], 2),
    ([300], [300], 5),
    ([5, 130], [700, 333], 4),            # chunks behind cached tokens
    ([40, 1, 3], [10, 0, 200], 2),        # fewer keys than queries: rows that see nothing
    ([700], [700], 1),
    # (from here on the keys are split over runs)
    ([1, 300, 0, 129], [4000, 1900, 50, 1029], 3),
    ([1700, 1], [1600, 3000], 2),         # blocks of rows that see nothing
    ([260], [4000], 1),
    ([200, 100] + [3] * 9, [9000, 8000, 100, 50, 1, 64, 65, 128, 30, 0, 90], 8),  # runs of several blocks
]


@pytest.mark.parametrize("spec", PROMPT, ids=[f"q{'_'.join(map(str, s[0][:4]))}_k{'_'.join(map(str, s[1][:4]))}_h{s[2]}" for s in PROMPT])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_prompt_against_float64(spec, dtype, causal):
    lens, keys, heads = spec
    c = make_prompt(lens, keys, heads, dtype, seed=sum(lens) + heads)
    out, lse = run_prompt(c, causal)
    R.check_prompt(out, lse, c["query"], c["key"], c["key_rope"], c["value"], c["cu_q"], c["cu_k"], SCALE, causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_prompt_nan_of_a_later_key_reaches_only_the_rows_that_see_it(dtype):
    c = make_prompt([200, 90], [200, 210], 3, dtype, seed=25)
    clean, clean_lse = run_prompt(c)
    value, key = c["value"].clone(), c["key"].clone()
    c["value"][137, 1, 9] = float("inf")   # seen by rows 137 .. 199 of the first sequence
    c["key"][200 + 150, 2] = float("nan")  # by rows 30 .. 89 of the second
    c["value"][200 + 150, 2] = float("nan")
    out, lse = run_prompt(c)
    assert bool(torch.isinf(out[137:200, 1, 9]).all()) and bool(torch.isnan(out[230:, 2]).all())
    out[137:200, 1, 9] = clean[137:200, 1, 9]
    out[230:, 2], lse[230:, 2] = clean[230:, 2], clean_lse[230:, 2]
    R.check_prompt(out, lse, c["query"], key, c["key_rope"], value, c["cu_q"], c["cu_k"], SCALE)


def test_prompt_split_with_a_used_workspace_on_another_stream_and_in_a_graph():
    """Any contents of the workspace; replays with other lengths; NaN keys that some rows of a split block do not see."""
    import l20_latent_attention as la

    c = make_prompt([200, 90], [1800, 1490], 3, seed=26)
    ws = la.allocate_l20_latent_prompt_workspace(c["query"], c["key"], 2, c["max_q"])
    assert ws.numel() > 0
    ws.fill_(255)
    clean, clean_lse = run_prompt(c, workspace=ws)
    R.check_prompt(clean, clean_lse, c["query"], c["key"], c["key_rope"], c["value"], c["cu_q"], c["cu_k"], SCALE)
    whole, _ = run_prompt(c, workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))
    assert float((whole.float() - clean.float()).abs().max()) < 0.02
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, again_lse = run_prompt(c, workspace=ws)
    side.synchronize()
    assert torch.equal(again, clean) and torch.equal(again_lse, clean_lse)
    with pytest.raises(RuntimeError, match="workspace is too small"):
        run_prompt(c, workspace=ws[:1024])
    out, lse = torch.empty_like(clean), torch.empty_like(clean_lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        la.l20_latent_prompt_attention(c["query"], c["key"], c["key_rope"], c["value"], c["cu_q"], c["cu_k"], c["max_q"],
                                       output=out, lse=lse, workspace=ws)
    for k in range(4):
        c["cu_q"].copy_(torch.tensor([0, 200 - 30 * k, 290 - 40 * k], dtype=torch.int32))
        c["cu_k"].copy_(torch.tensor([0, 1800 - 400 * k, 3290 - 450 * k], dtype=torch.int32))
        out.fill_(3)
        lse.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_lse = run_prompt(c, output=torch.full_like(out, 3))
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse)
    c["cu_q"].copy_(torch.tensor([0, 200, 290], dtype=torch.int32))
    c["cu_k"].copy_(torch.tensor([0, 1800, 3290], dtype=torch.int32))
    c["key"][1600 + 137, 1] = float("nan")
    c["value"][1600 + 137, 1] = float("nan")
    got, got_lse = run_prompt(c, workspace=ws)
    assert bool(torch.isnan(got[137:200, 1]).all())
    keep = torch.ones(290, 3, dtype=torch.bool, device="cuda")
    keep[137:200, 1] = False
    assert float((got.float() - clean.float()).abs()[keep].max()) < 0.02
    assert float((got_lse - clean_lse).abs()[keep].max()) < 1e-4


def test_prompt_leaves_other_rows_alone():
    """Rows behind the last sequence, and rows beyond max_seqlen_q of theirs, keep what they held; NaN keys behind
    the last sequence and values of other sequences reach nobody."""
    c = make_prompt([50, 70, 30], [50, 70, 30], 4, seed=21)
    want, want_lse = run_prompt(c)
    c["cu_q"] = c["cu_q"][:3].contiguous()
    c["cu_k"] = c["cu_k"][:3].contiguous()
    c["key"][120:] = float("nan")
    c["value"][120:] = float("nan")
    c["key_rope"][120:] = float("nan")
    c["max_q"] = 60
    out = torch.full_like(want, 9.0)
    got, lse = run_prompt(c, output=out)
    assert torch.equal(got[:110], want[:110]) and torch.equal(lse[:110], want_lse[:110])
    assert bool((got[110:] == 9).all()) and bool((lse[110:] == 5).all())


def test_prompt_strided_views_and_large_scores():
    import l20_latent_attention as la

    c = make_prompt([90], [150], 4, seed=22)
    query = torch.randn(90, 9, 256, device="cuda").to(torch.bfloat16)
    query[:, 2:6, 64:] = c["query"] * 8
    out = torch.full((90, 6, 136), 3.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.zeros(150, 640, dtype=torch.bfloat16, device="cuda")
    rope[:, 512:576] = c["key_rope"]
    la.l20_latent_prompt_attention(query[:, 2:6, 64:], c["key"], rope[:, 512:576], c["value"], c["cu_q"], c["cu_k"], 90,
                                   output=out[:, 1:5, 4:132])
    torch.cuda.synchronize()
    R.check_prompt(out[:, 1:5, 4:132], None, query[:, 2:6, 64:], c["key"], c["key_rope"], c["value"], c["cu_q"], c["cu_k"], SCALE)
    assert bool((out[:, 0] == 3).all()) and bool((out[..., :4] == 3).all()) and bool((out[..., 132:] == 3).all())


def test_prompt_agrees_with_decode_of_its_last_token():
    """Expanded and absorbed forms of one model: o = W_v (sum p c) with q absorbed through W_k, in fp16."""
    import l20_latent_attention as la

    g = torch.Generator().manual_seed(23)
    n, heads, rank = 150, 4, 512
    latent = torch.randn(n, rank, generator=g).half()
    rope = torch.randn(n, 64, generator=g).half()
    w_k, w_v = (torch.randn(heads, 128, rank, generator=g) / 24 for _ in range(2))
    key = torch.einsum("tr,hdr->thd", latent.float(), w_k).half().cuda()
    value = torch.einsum("tr,hdr->thd", latent.float(), w_v).half().cuda()
    query = torch.randn(n, heads, 192, generator=g).half()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = la.l20_latent_prompt_attention(query.cuda(), key, rope.cuda(), value, cu, cu, n)
    absorbed = torch.cat([torch.einsum("hd,hdr->hr", query[-1, :, :128].float(), w_k), query[-1, :, 128:].float()], -1)
    pages = -(-n // 16)
    cache = torch.zeros(pages * 16, rank + 64, dtype=torch.float16)
    cache[:n] = torch.cat([latent, rope], -1)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    dec = la.l20_paged_latent_attention(absorbed.half().cuda()[None], cache.view(pages, 16, -1).cuda(), table, lens,
                                        softmax_scale=SCALE)
    dec = torch.einsum("hr,hdr->hd", dec[0].cpu().float(), w_v)
    # Both forms round keys, queries, weights and results to fp16 (2^-11 each); a score error of a few 2^-11 |s|
    # with |s| up to ~5 moves a weight by ~1%, far below one token's exchange.
    ref = out[-1].cpu().float()
    assert float((dec - ref).norm() / ref.norm()) < 2e-2


def test_refusals():
    import l20_latent_attention as la

    c = make_decode([64], 8, seed=30)
    ok = dict(softmax_scale=SCALE)
    args = (c["query"], c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="rank 256 or 512"):
        la.l20_paged_latent_attention(*args, kv_rank=384, **ok)
    with pytest.raises(RuntimeError, match="query"):
        la.l20_paged_latent_attention(c["query"].float(), *args[1:], **ok)
    with pytest.raises(RuntimeError, match="float8_e4m3fn or the model dtype"):
        la.l20_paged_latent_attention(c["query"].half(), *args[1:], **ok)
    with pytest.raises(RuntimeError, match="seq_lens must be contiguous int32"):
        la.l20_paged_latent_attention(*args[:3], c["lens"].long(), **ok)
    with pytest.raises(RuntimeError, match="block table"):
        la.l20_paged_latent_attention(*args[:2], c["table"].long(), c["lens"], **ok)
    with pytest.raises(RuntimeError, match="workspace is too small"):
        la.l20_paged_latent_attention(*args, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"), max_seq_len=1000, **ok)
    with pytest.raises(RuntimeError, match="same device"):
        la.l20_paged_latent_attention(*args[:3], c["lens"].cpu(), **ok)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        la.l20_paged_latent_attention(*args, softmax_scale=math.inf)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        shifted = torch.zeros(1, 8, 577, dtype=torch.bfloat16, device="cuda")[..., 1:]
        la.l20_paged_latent_attention(shifted, *args[1:], **ok)
    p = make_prompt([8], [8], 2, seed=31)
    with pytest.raises(RuntimeError, match="one dtype"):
        la.l20_latent_prompt_attention(p["query"], p["key"], p["key_rope"].half(), p["value"], p["cu_q"], p["cu_k"], 8)
    with pytest.raises(RuntimeError, match="key and value"):
        la.l20_latent_prompt_attention(p["query"], p["key"][:, :1], p["key_rope"], p["value"], p["cu_q"], p["cu_k"], 8)
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        la.l20_latent_prompt_attention(p["query"], p["key"], p["key_rope"], p["value"], p["cu_q"].long(), p["cu_k"], 8)


@pytest.mark.parametrize("lens,keys", [([70, 40, 3], [65, 130, 1]), ([260], [4001])], ids=["whole", "split"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_prompt_infinite_value_of_the_last_key(lens, keys, dtype, causal):
    """Where a sequence ends inside a tile: infinite dims for the rows that see the last key, all else as without."""
    c = make_prompt(lens, keys, 2, dtype, seed=27)
    clean, clean_lse = run_prompt(c, causal)
    value = c["value"].clone()
    hit = torch.zeros_like(clean)
    ends = list(zip(c["cu_q"].tolist(), c["cu_q"][1:].tolist(), c["cu_k"][1:].tolist()))
    for q0, q1, k1 in ends:
        c["value"][k1 - 1, 1, 9], c["value"][k1 - 1, 0, 127] = float("inf"), -float("inf")
        first = q1 - 1 if causal else q0  # (the last row alone sees the last key)
        hit[first:q1, 1, 9], hit[first:q1, 0, 127] = 1, -1
    out, lse = run_prompt(c, causal)
    assert torch.equal(out.isinf(), hit != 0) and bool((out.isinf() * out.sign() == hit).all())
    out[hit != 0] = clean[hit != 0]
    R.check_prompt(out, lse, c["query"], c["key"], c["key_rope"], value, c["cu_q"], c["cu_k"], SCALE, causal)


@pytest.mark.parametrize("lens,keys", [([200, 70], [200, 333]), ([260], [4000])], ids=["whole", "split"])
def test_prompt_value_that_all_rows_see_changes_its_dim_alone(lens, keys):
    """No row is computed again for a value that it sees: the other dims are the same bits (and take no longer)."""
    c = make_prompt(lens, keys, 2, seed=28)
    clean, clean_lse = run_prompt(c)
    for k0 in c["cu_k"].tolist()[:-1]:
        c["value"][k0, 1, 9], c["value"][k0, 0, 64] = float("inf"), float("nan")
    out, lse = run_prompt(c)
    assert bool(out[:, 1, 9].isinf().all()) and bool(out[:, 0, 64].isnan().all())
    out[:, 1, 9], out[:, 0, 64] = clean[:, 1, 9], clean[:, 0, 64]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("bound", [None, 100000], ids=["few", "long"])
def test_decode_value_that_all_drafts_see_changes_its_dim_alone(bound):
    """As above, by a token that its score of -inf gives a weight of 0."""
    q_len, dim = 3, 9
    c = make_decode([70, 2, 129, 900, 64], 16, q_len=q_len, seed=36, poison=False)
    c["query"][..., dim] = c["query"][..., dim].abs().clamp_min(0.125)
    for b, t in ((0, 3), (2, 100), (3, 890), (4, 0)):
        c["cache"][c["table"][b, t // 16].long(), t % 16, dim] = -30000.0  # weight 0, finite
    clean, clean_lse = run_decode(c, max_seq_len=bound)
    for b, t in ((0, 3), (2, 100), (3, 890), (4, 0)):
        c["cache"][c["table"][b, t // 16].long(), t % 16, dim] = -float("inf")
    out, lse = run_decode(c, max_seq_len=bound)
    hit = torch.ones(5, q_len, dtype=torch.bool, device="cuda")
    hit[1] = False
    hit = hit.flatten()
    assert bool(out[hit][..., dim].isnan().all()) and not bool(out[~hit].isnan().any())  # (0 x inf)
    out[hit, :, dim] = clean[hit, :, dim]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_prompt_infinite_value_seen_beside_a_nan_not_seen(dtype):
    c = make_prompt([200, 90], [200, 210], 2, dtype, seed=29)
    clean, clean_lse = run_prompt(c)
    value = c["value"].clone()
    c["value"][0, 1, 9], c["value"][100, 1, 30] = float("inf"), float("nan")  # seen by all rows, by rows 100 .. 199
    c["value"][200, 0, 9], c["value"][200 + 209, 0] = -float("inf"), float("nan")  # by all, by the last row
    out, lse = run_prompt(c)
    assert bool((out[:200, 1, 9] == float("inf")).all()) and bool(out[100:200, 1, 30].isnan().all())
    assert bool((out[200:289, 0, 9] == -float("inf")).all()) and bool(out[289, 0].isnan().all())
    for rows, h, dims in ((slice(0, 200), 1, 9), (slice(100, 200), 1, 30), (slice(200, 289), 0, 9), (289, 0, slice(None))):
        out[rows, h, dims] = clean[rows, h, dims]
    R.check_prompt(out, lse, c["query"], c["key"], c["key_rope"], value, c["cu_q"], c["cu_k"], SCALE)


@pytest.mark.parametrize("batches", [(64, 32, 8, 1), (70, 9)])
def test_decode_workspace_of_the_largest_batch_is_enough_for_smaller_ones(batches):
    """Allocated once for a batch that is not split itself; smaller ones are."""
    import l20_latent_attention as la

    lens = [(29 * i) % 256 + 1 for i in range(batches[0])]
    ws = None
    for n in batches:
        c = make_decode(lens[:n], 16, rank=256, seed=37)
        if ws is None:
            ws = la.allocate_l20_paged_latent_workspace(c["query"], c["cache"], 256, kv_rank=256)
        check_decode(c, *run_decode(c, workspace=ws, max_seq_len=256))


def test_outputs_beside_their_inputs_and_over_them():
    """Interleaved with the query, row by row or head by head, is fine; any shared byte is refused."""
    import l20_latent_attention as la

    c = make_decode([300, 40, 7], 6, q_len=2, seed=38)
    want, want_lse = run_decode(c)
    rows, heads = c["query"].shape[:2]
    by_head = torch.zeros(rows, heads, 576 + 512, dtype=torch.bfloat16, device="cuda")
    by_row = torch.zeros(rows, heads * (576 + 512), dtype=torch.bfloat16, device="cuda")
    for query, output in ((by_head[..., :576], by_head[..., 576:]),
                          (by_row[:, :heads * 576].view(rows, heads, 576), by_row[:, heads * 576:].view(rows, heads, 512)),
                          (by_row[:, heads * 512:].view(rows, heads, 576), by_row[:, :heads * 512].view(rows, heads, 512))):
        query.copy_(c["query"])
        out, lse = run_decode({**c, "query": query}, output=output)
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(query, c["query"])
    for output in (c["query"][..., 64:], c["query"][..., :512], c["query"][..., 16:528],
                   by_head.view(rows, -1)[:, 8:8 + heads * 512].view(rows, heads, 512)):
        with pytest.raises(RuntimeError, match="output must not"):
            run_decode({**c, "query": c["query"] if output.shape[2] == 512 and output.stride(1) == 576 else by_head[..., :576]}, output=output)
    p = make_prompt([90, 30], [90, 30], 3, seed=39)
    want, _ = run_prompt(p)
    both = torch.zeros(120, 3, 192 + 128, dtype=torch.bfloat16, device="cuda")
    both[..., :192] = p["query"]
    out, _ = run_prompt({**p, "query": both[..., :192]}, output=both[..., 192:])
    assert torch.equal(out, want) and torch.equal(both[..., :192], p["query"])
    for output in (p["query"][..., 64:], p["value"], p["key"]):
        with pytest.raises(RuntimeError, match="output must not"):
            run_prompt(p, output=output)


@pytest.mark.parametrize("lens,keys", [([200, 70], [200, 333]), ([260], [4000])], ids=["whole", "split"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_prompt_infinite_value_of_a_small_weight(lens, keys, dtype, causal):
    """A weight of about 2^-33 of the largest, which is 0 in fp16: an infinite value is infinite in the sum all the same,
    a NaN a NaN."""
    c = make_prompt(lens, keys, 2, dtype, seed=41)
    c["query"][..., 0] = 8.0
    c["key"][..., 0] = 0.0
    firsts = c["cu_k"].tolist()[:-1]
    for k0 in firsts:
        c["key"][k0 + 1, :, 0] = -40.0
    clean, clean_lse = run_prompt(c, causal)
    value = c["value"].clone()
    for k0 in firsts:
        c["value"][k0 + 1, 1, 9], c["value"][k0 + 1, 0, 127], c["value"][k0 + 2, 0, 64] = float("inf"), -float("inf"), float("nan")
    out, lse = run_prompt(c, causal)
    for q0, q1, n in zip(c["cu_q"].tolist(), c["cu_q"][1:].tolist(), [k - q for q, k in zip(lens, keys)]):
        # (the first row of a prompt without cached keys sees key 0 alone, its second keys 0 and 1)
        inf0, nan0 = (q0 + max(1 - n, 0), q0 + max(2 - n, 0)) if causal else (q0, q0)
        assert bool((out[inf0:q1, 1, 9] == float("inf")).all()) and bool((out[inf0:q1, 0, 127] == -float("inf")).all())
        assert bool(out[nan0:q1, 0, 64].isnan().all())
        for rows, h, dim in ((slice(inf0, q1), 1, 9), (slice(inf0, q1), 0, 127), (slice(nan0, q1), 0, 64)):
            out[rows, h, dim] = clean[rows, h, dim]
    R.check_prompt(out, lse, c["query"], c["key"], c["key_rope"], value, c["cu_q"], c["cu_k"], SCALE, causal)
