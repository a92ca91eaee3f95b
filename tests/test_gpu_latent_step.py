"""GPU: a serving loop over latent attention -- block tables, cache producer, prompt attention, then decode steps
with requests that finish and pages that are used again -- against float64 over the tokens themselves."""

import pytest
import torch

import latent_ref as R

pytestmark = pytest.mark.gpu
SCALE, RANK, HEADS, PAGE = 192 ** -0.5, 512, 6, 32


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_prompts_then_decode_steps(fp8):
    import l20_block_tables as bt
    import l20_latent_attention as la

    dtype, cap, width, pool = torch.bfloat16, 4, 8, 14
    g = torch.Generator().manual_seed(40)
    theta = torch.rand(400, 32, generator=g, dtype=torch.float64) * 6.28
    cs = torch.cat([theta.cos(), theta.sin()], -1).float().cuda()
    weight = (1 + torch.randn(RANK, generator=g) / 8).to(dtype).cuda()
    scale = 1 / 32.0 if fp8 else 1.0
    cache = torch.full((pool, PAGE, RANK + 64), float("nan")).to(torch.float8_e4m3fn if fp8 else dtype).cuda()
    table = torch.full((cap, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, generator=g).to(torch.int32).cuda()
    count = torch.tensor([pool], dtype=torch.int32, device="cuda")
    cached = torch.zeros(cap, dtype=torch.int32, device="cuda")
    lens, cu = torch.zeros_like(cached), torch.zeros(cap + 1, dtype=torch.int32, device="cuda")
    rows = [torch.zeros(0, RANK + 64, dtype=torch.float64, device="cuda") for _ in range(cap)]
    ws = la.allocate_l20_paged_latent_workspace(torch.empty(cap, HEADS, RANK + 64, dtype=dtype, device="cuda"), cache, width * PAGE)

    # (new tokens of each request, -1: it is finished and its place is given to a new one)
    steps = [[70, 33, 1, 100]] + [[1, 1, 1, 1]] * 3 + [[1, -1, 1, -1], [0, 90, 1, 64]] + [[1] * 4] * 4
    for new in steps:
        n = sum(max(x, 0) for x in new)
        tokens = n + 2  # two rows of padding
        slots, positions = (torch.empty(tokens, dtype=torch.int64, device="cuda") for _ in range(2))
        bt.l20_build_block_tables(cached, torch.tensor(new, dtype=torch.int32, device="cuda"), table, free, count, slots,
                                  positions, cu, lens, PAGE)
        down = torch.randn(tokens, RANK + 64, generator=g).to(dtype).cuda()
        query = torch.randn(tokens, HEADS, RANK + 64, generator=g).to(dtype).cuda()
        la.l20_latent_rope_and_cache(query[..., RANK:], down[:, :RANK], down[:, RANK:], positions, cs, True, cache, slots,
                                     norm_weight=weight, cache_scale=scale)
        row = down
        if fp8:
            row = (down.float() / scale).clamp(-448, 448).to(cache.dtype).float() * scale
        at, expect = 0, []
        for b, x in enumerate(new):
            rows[b] = rows[b][:0] if x < 0 else torch.cat([rows[b], row[at:at + max(x, 0)].double()])
            at += max(x, 0)
            expect.append(rows[b].shape[0])
        assert lens.tolist() == expect
        cached.copy_(lens)
        if max(new) > 1:
            continue
        # decode: one row a request (a request without a new token keeps a row of its own too)
        first = cu[:-1].long().clamp_max(tokens - 1)
        q = query[first].contiguous()
        lse = torch.empty(cap, HEADS, device="cuda")
        out = la.l20_paged_latent_attention(q, cache, table, lens, softmax_scale=SCALE, cache_scale=scale,
                                            max_seq_len=width * PAGE, workspace=ws, lse=lse)
        for b in range(cap):
            seen = torch.ones(HEADS, rows[b].shape[0], dtype=torch.bool, device="cuda")
            want = R.attend(q[b].double(), rows[b], rows[b][:, :RANK], seen, SCALE, dtype)
            R.assert_rows(out[b], lse[b], *want, f"request {b}")
    assert int(count) == pool - sum(-(-n // PAGE) for n in lens.tolist())
