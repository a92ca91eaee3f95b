"""GPU: beam search's selection against every candidate in float64 and plain Python."""

import math

import pytest
import torch

import beam_ref as R

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")
    import l20_beam_search  # noqa: F401


def filled(requests, beams):
    """Outputs that hold something else."""
    import l20_beam_search as bs

    out = bs.BeamSearchStep.empty(requests, beams, "cuda")
    for t in out:
        t.fill_(-77)
    return out


def inputs(requests, beams, vocab, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = (scale * torch.randn(requests, beams, vocab, generator=g)).to(dtype)
    return logits, -3 * torch.rand(requests, beams, generator=g)


def compare(out, logits, scores, ends):
    """logits [requests, beams, vocab] and scores on the CPU."""
    want = R.beam_step(logits, scores, list(ends))
    assert want[6] > 1e-6, "the inputs leave the order to the last digits"
    for at, name in enumerate(("tokens", "parents", "scores", "ended_tokens", "ended_parents", "ended_scores")):
        got = out[at].tolist()
        if name.endswith("scores"):
            for r, (mine, theirs) in enumerate(zip(got, want[at])):
                for x, y in zip(mine, theirs):
                    assert x == y if math.isinf(y) else abs(x - y) <= R.score_bound(y, logits.shape[2]), (name, r, x, y)
        else:
            assert got == want[at], name
    return want


def check(logits, scores, ends=(), **kw):
    import l20_beam_search as bs

    out = bs.l20_beam_search_step(logits.cuda(), scores.cuda(), end_tokens=list(ends),
                                  out=filled(*scores.shape), **kw)
    torch.cuda.synchronize()
    return compare(out, logits, scores, ends)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 511, 512, 513, 2047, 2048, 2049, 5001, 16385])
def test_vocabularies(dtype, vocab):
    logits, scores = inputs(3, 4, vocab, DTYPES[dtype], seed=vocab)
    check(logits, scores, ends=[vocab // 2, 0] if vocab > 2 else [])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [3, 5, 255, 257, 259, 260, 261, 508, 517, 770, 1023, 2303, 2305, 2309, 8190, 8451])
def test_rows_that_end_inside_a_load(dtype, vocab):
    """The last tokens are the best, and what lies behind each row would take all of it."""
    import l20_beam_search as bs

    logits, scores = inputs(2, 3, vocab, DTYPES[dtype], seed=vocab + 1)
    for back in range(1, min(vocab, 4)):
        logits[:, :, vocab - back] += 13 - back
    hold = torch.full((2, 3, vocab + 7), math.nan, dtype=DTYPES[dtype], device="cuda")
    hold[:, :, :vocab] = logits.cuda()
    out = bs.l20_beam_search_step(hold[:, :, :vocab], scores.cuda(), end_tokens=[vocab - 1], out=filled(2, 3))
    torch.cuda.synchronize()
    want = compare(out, logits, scores, [vocab - 1])
    assert any(vocab - 1 in row for row in want[3])


@pytest.mark.parametrize("beams", [1, 2, 3, 5, 8, 16, 31, 32])
@pytest.mark.parametrize("ends", [0, 1, 8])
def test_beams_and_end_tokens(beams, ends):
    logits, scores = inputs(3, beams, 1500, torch.bfloat16, seed=10 * beams + ends)
    tokens = [5 * e + 1 for e in range(ends)]
    logits[:, :, tokens] += 7  # likely: they lead many rows
    check(logits, scores, tokens)


@pytest.mark.parametrize("beams,vocab,ends", [(32, 40000, 8), (20, 66000, 1), (32, 20, 3), (17, 18, 1), (32, 40, 8), (9, 200000, 0)])
def test_many_beams_over_long_and_short_vocabularies(beams, vocab, ends):
    """More entries than a wave's list holds, joined from several runs; fewer tokens than beams."""
    logits, scores = inputs(2, beams, vocab, torch.bfloat16, seed=7 * beams + vocab)
    tokens = [(2 * e + 1) % vocab for e in range(ends)]
    logits[:, ::3, tokens] += 6
    check(logits, scores, tokens)


def test_end_tokens_that_are_none():
    """Outside the vocabulary, below it, and named twice."""
    logits, scores = inputs(2, 3, 100, torch.float16, seed=4)
    logits[:, :, 9] += 8
    check(logits, scores, [9, 9, 100, -1, 2 ** 31 - 1])


@pytest.mark.parametrize("requests,beams", [(1, 1), (1, 32), (70, 1), (40, 5)])
def test_numbers_of_rows(requests, beams):
    logits, scores = inputs(requests, beams, 4100, torch.bfloat16, seed=requests + beams)
    check(logits, scores, [17])


def test_rows_without_candidates():
    """Masked throughout, a NaN, an infinity, dead beams of several kinds: no candidate of theirs, and none of the
    others lost.  What a dead beam's row holds does not matter."""
    inf, nan = math.inf, math.nan
    for dtype in DTYPES.values():
        logits, scores = inputs(7, 4, 3000, dtype, seed=3)
        logits[0, 1] = -inf
        logits[1, 0, 2999] = nan
        logits[1, 2, 5] = inf
        logits[1, 3, 1000:] = -inf
        scores[2] = torch.tensor([-1.0, -inf, inf, nan])
        logits[2, 1:] = nan
        scores[3] = -inf
        logits[4] = -inf
        logits[4, 2, [10, 2500]] = torch.tensor([1.0, 0.0]).to(dtype)  # two candidates for four beams
        logits[5] = nan
        logits[6, 0, :2500] = nan
        want = check(logits, scores, [2500])
        assert want[0][3] == [-1] * 4 and want[0][4][0] == 10 and want[0][4][1:] == [-1] * 3 and want[3][4][0] == 2500


@pytest.mark.parametrize("vocab", [40, 515, 2500, 6001])
def test_ties_go_to_the_lower_beam_and_token(vocab):
    """Equal rows of equal beams (at odd offsets too), equal logits, and whole rows of one value."""
    logits, scores = inputs(3, 4, vocab, torch.bfloat16, seed=vocab)
    logits[0, :] = logits[0, :1]
    scores[0] = scores[0, 0]
    logits[1] = 0.25
    scores[1] = -1.0
    logits[2, :, : vocab // 2] = 3.0
    scores[2, 1:] -= 1.5
    want = check(logits, scores, [1])
    assert want[1][1] == [0, 0, 0, 0] and want[0][1] == [0, 2, 3, 4] and want[3][1] == [1, -1, -1, -1]


def test_minus_zero_ties_with_zero():
    logits = torch.zeros(1, 1, 100)
    logits[0, 0, ::2] = -0.0
    assert check(logits, torch.zeros(1, 1), [0])[0] == [[1]]


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_values(dtype):
    """The type's lowest value as a mask, large logits of both signs, and scores far from zero."""
    d = DTYPES[dtype]
    logits, scores = inputs(3, 3, 2600, d, seed=8)
    logits[0, :, 100:] = torch.finfo(d).min
    big = {"bf16": 2.0 ** 120, "fp16": 60000.0, "fp32": 2.0 ** 126}[dtype]
    logits[1] = -big
    logits[1, 0, 7], logits[1, 1, 2599], logits[1, 2, 0] = big, big, -big / 2
    scores[1] = torch.tensor([-1.0, -2.0, -3.0])
    scores[2] = torch.tensor([-1e30, -1e30, -3e38])
    import l20_beam_search as bs

    out = bs.l20_beam_search_step(logits[:2].cuda(), scores[:2].cuda(), out=filled(2, 3))
    compare(out, logits[:2], scores[:2], [])
    # 1e30 swallows the logits: equal scores, so the lower beam, then its higher logits
    out = bs.l20_beam_search_step(logits[2:].cuda(), scores[2:].cuda(), out=filled(1, 3))
    best = sorted(range(2600), key=lambda t: (-float(logits[2, 0, t]), t))[:3]
    assert out.tokens.tolist() == [best] and out.parents.tolist() == [[0] * 3]
    assert out.scores.cpu().equal(torch.full((1, 3), -1e30))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("level", [-300.0, 5.0, 300.0, 60000.0])
def test_rows_that_begin_masked(dtype, level):
    """Nothing finite, or only the type's lowest value, in the first 40000 tokens; logits far from zero behind them."""
    d = DTYPES[dtype]
    if level == 60000.0 and dtype != "fp16":
        level = 2.0 ** 22
    logits, scores = inputs(4, 2, 50000, d, seed=77)
    step = {"bf16": 2.0 ** -7, "fp16": 2.0 ** -10, "fp32": 2.0 ** -23}[dtype] * abs(level)
    late = level + step * torch.randint(-20, 20, (4, 2, 10000), generator=torch.Generator().manual_seed(1))
    logits[:, :, 40000:] = late.to(d)
    logits[0, :, :40000] = -math.inf
    logits[1, :, :40000] = torch.finfo(d).min
    logits[2, 0, :49990] = -math.inf
    logits[2, 1, :49990] = torch.finfo(d).min
    logits[3, 0] = torch.finfo(d).min
    logits[3, 0, 45000] = level
    logits[3, 1, 1:] = -math.inf
    check(logits, scores, [49999])


@pytest.mark.parametrize("order", ["rising", "falling", "blocks"])
def test_orders_that_pass_every_threshold(order):
    x = torch.arange(9000.0) / 1000
    x = {"rising": x, "falling": x.flip(0), "blocks": x.view(9, 1000).flip(0).reshape(-1)}[order]
    logits = torch.stack([x, x * 0.9 + 0.01]).unsqueeze(0).contiguous()
    check(logits, torch.tensor([[-1.0, -1.3]]), [8999])


def test_layouts():
    """Padded rows, beams outside requests, rows at every alignment, one request's strides that say nothing."""
    import l20_beam_search as bs

    logits, scores = inputs(3, 4, 2111, torch.bfloat16, seed=20)
    want = None
    for kind in range(6):
        hold = torch.full((40000,), math.nan, dtype=logits.dtype, device="cuda")
        if kind < 4:
            view = hold[kind:].as_strided((3, 4, 2111), (4 * 2200, 2200 + (kind % 2) * 3, 1))
        elif kind == 4:
            view = hold.as_strided((3, 4, 2111), (2200, 3 * 2200, 1))
        else:
            view = hold[1:].as_strided((12, 2111), (2113, 1))
        view.copy_(logits.view(view.shape))
        s = torch.full((3, 9), 5.0, device="cuda")[:, ::2][:, :4] if kind % 2 else torch.empty(4, 3, device="cuda").t()
        s.copy_(scores)
        out = bs.l20_beam_search_step(view, s, end_tokens=[3], out=filled(3, 4))
        if want is None:
            compare(out, logits, scores, [3])
            want = [t.clone() for t in out]
        assert all(a.equal(b) for a, b in zip(out, want)), kind
    x = logits[:1, :1].cuda()
    out = bs.l20_beam_search_step(x.as_strided((1, 1, 2111), (1, 7, 1)), scores[:1, :1].cuda(), out=filled(1, 1))
    compare(out, logits[:1, :1], scores[:1, :1], [])


def test_scores_in_place_and_smaller_batches_in_one_workspace():
    import l20_beam_search as bs

    logits, scores = inputs(9, 4, 8000, torch.float16, seed=31)
    x = logits.cuda()
    ws = bs.allocate_l20_beam_search_workspace(x, scores.cuda(), end_tokens=[1])
    for n in (9, 4, 1, 7):
        s = scores[:n].cuda()
        out = filled(n, 4)._replace(scores=s)
        ws.fill_(255)
        bs.l20_beam_search_step(x[:n], s, end_tokens=[1], out=out, workspace=ws)
        compare(out, logits[:n], scores[:n], [1])


def test_no_requests():
    import l20_beam_search as bs

    out = bs.l20_beam_search_step(torch.zeros(0, 50, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert out.tokens.shape == (0, 4)


def test_wide_rows_and_many_rows():
    """A vocabulary beyond any tokenizer's in few rows, and more rows than the chip holds waves, against torch in 64
    bits (with the same order of ties: a stable sort of each row)."""
    import l20_beam_search as bs

    for requests, beams, vocab, dtype in ((1, 2, 3_000_017, torch.float32), (700, 8, 2500, torch.bfloat16)):
        g = torch.Generator(device="cuda").manual_seed(vocab)
        x = (2 * torch.randn(requests, beams, vocab, generator=g, device="cuda")).to(dtype)
        s = -3 * torch.rand(requests, beams, generator=g, device="cuda")
        out = bs.l20_beam_search_step(x, s)
        total = torch.log_softmax(x.double(), -1) + s.double()[..., None]
        best, at = total.flatten(1).sort(dim=-1, descending=True, stable=True)
        gaps = best[:, :beams] - best[:, 1:beams + 1]
        other = at[:, :beams] // vocab != at[:, 1:beams + 1] // vocab
        sure = ~(other & (gaps < 1e-6)).any(-1)  # (a request in thousands may hang on the last digits)
        assert sure.float().mean() > 0.99
        assert out.tokens[sure].equal(at[sure, :beams] % vocab) and out.parents[sure].equal((at[sure, :beams] // vocab).int())
        assert ((out.scores.double() - best[:, :beams]).abs() <= 2.0 ** -24 * best[:, :beams].abs() +
                2.0 ** -23 * (4 + math.log(vocab))).all()


def test_rows_beyond_32_bits():
    """Logits whose rows lie further apart than 2^31 elements, and more rows than are counted."""
    import l20_beam_search as bs

    logits, scores = inputs(2, 2, 5000, torch.bfloat16, seed=60)
    view = torch.empty(3 * (1 << 31) // 2 + 3 * (1 << 30) + 5000, dtype=torch.bfloat16, device="cuda").as_strided(
        (2, 2, 5000), (3 * (1 << 30), 3 * (1 << 29), 1))
    view.copy_(logits)
    compare(bs.l20_beam_search_step(view, scores.cuda(), out=filled(2, 2)), logits, scores, [])
    del view
    g = torch.Generator(device="cuda").manual_seed(61)
    x = torch.randn(9000, 1, 300, generator=g, device="cuda")
    s = torch.rand(9000, 1, generator=g, device="cuda")
    s[::3] = -math.inf
    out = bs.l20_beam_search_step(x, s, out=filled(9000, 1))
    assert out.tokens.equal(torch.where(s > -math.inf, x.argmax(-1), -1)) and out.parents.equal((s > -math.inf).int() - 1)


def test_graph_and_another_stream():
    """A captured step whose scores advance in place: replays equal eager calls on copies, also beside eager work."""
    import l20_beam_search as bs

    logits, scores = inputs(5, 4, 9001, torch.bfloat16, seed=50)
    x, s = logits.cuda(), scores.cuda()
    eager = s.clone()
    out = filled(5, 4)._replace(scores=s)
    ws = bs.allocate_l20_beam_search_workspace(x, s, end_tokens=[2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        bs.l20_beam_search_step(x, s.clone(), end_tokens=[2], workspace=ws)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bs.l20_beam_search_step(x, s, end_tokens=[2], out=out, workspace=ws)
    s.copy_(scores)
    for step in range(4):
        x.add_(0.5 * torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(step)).to(x.dtype))
        want = bs.l20_beam_search_step(x, eager, end_tokens=[2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(a.equal(b) for a, b in zip(out, want))
        eager = want.scores.clone()


def test_two_streams_at_once():
    """Calls on two streams, each with its workspace and outputs, of different sizes: as alone."""
    import l20_beam_search as bs

    cases = []
    for n, (requests, beams, vocab) in enumerate(((40, 4, 30000), (3, 8, 90000))):
        logits, scores = inputs(requests, beams, vocab, torch.float16, seed=90 + n)
        x, s = logits.cuda(), scores.cuda()
        cases.append((x, s, filled(requests, beams), bs.allocate_l20_beam_search_workspace(x, s, end_tokens=[4]),
                      bs.l20_beam_search_step(x, s, end_tokens=[4]), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for x, s, out, ws, _, stream in cases:
            with torch.cuda.stream(stream):
                bs.l20_beam_search_step(x, s, end_tokens=[4], out=out, workspace=ws)
    torch.cuda.synchronize()
    for _, _, out, _, want, _ in cases:
        assert all(a.equal(b) for a, b in zip(out, want))


def test_refusals():
    import l20_beam_search as bs

    x, s = torch.zeros(6, 100, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad, message in (((x[:5], s), "logits must be"), ((x.double(), s), "bf16, fp16 or fp32"), ((x, s.double()), "fp32"),
                         ((x.t().contiguous().t(), s), "contiguous"), ((x, s[0]), "requests, beams"),
                         ((torch.zeros(66, 9, device="cuda"), torch.zeros(2, 33, device="cuda")), "1 to 32")):
        with pytest.raises(RuntimeError, match=message):
            bs.l20_beam_search_step(*bad)
    with pytest.raises(RuntimeError, match="at most 8 end tokens"):
        bs.l20_beam_search_step(x, s, end_tokens=list(range(9)))
    with pytest.raises(RuntimeError, match="workspace is missing"):
        bs.l20_beam_search_step(x, s, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    out = bs.BeamSearchStep.empty(2, 3, "cuda")
    with pytest.raises(RuntimeError, match="tokens must be"):
        bs.l20_beam_search_step(x, s, out=out._replace(tokens=out.parents))
    with pytest.raises(RuntimeError, match="lie apart"):
        bs.l20_beam_search_step(x, s, out=out._replace(ended_tokens=out.tokens))
    with pytest.raises(RuntimeError, match="not lie over an input"):
        bs.l20_beam_search_step(x, s, out=out._replace(ended_scores=x.view(-1)[:6].view(2, 3)))


# --------------------------------------------------------------------------- accuracy of a row's log-sum-exp
def lse_bound(x):
    """How far the log-sum-exp of each row of `x` (float64) may be off.  A term is exp2 of an fp32 exponent e relative to a
    reference that no value exceeds by more than 4 ln 2 (a sum of eight terms up to 2^4), so |e| <= max(4, (top - x) log2 e):
    half a step of e, and log2 e halves of one for the difference that it is made of (no larger steps), times ln 2; the
    distance of log2 e from the further of the two floats around it, 1e-7, times that difference and ln 2; exp2 itself
    (one step: 2^-23); three additions (2^-24 each).  The rest is in 64 bits.  The terms' errors weigh as the terms do; 1 %
    for products of them."""
    top = x.amax(-1, keepdim=True)
    weight = (x - torch.logsumexp(x, -1, keepdim=True)).exp()
    e = ((top - x) * math.log2(math.e)).clamp_min(4.0)
    half = torch.exp2(e.log2().ceil() - 25)  # of the steps of (2^(n-1), 2^n]
    apart = 1e-7 * math.log(2) * (e / math.log2(math.e))
    return 1.01 * (weight * ((1 + math.log2(math.e)) * math.log(2) * half + apart + 2.0 ** -23 + 3 * 2.0 ** -24)).sum(-1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0.0, 100.0, -100.0])
@pytest.mark.parametrize("late", [True, False], ids=["best late", "spread"])
@pytest.mark.parametrize("rows,vocab", [(200, 150000), (800, 30000)], ids=["three runs", "one run"])
def test_log_sum_exp_to_its_last_digits(dtype, offset, late, rows, vocab):
    """Each row's best score, moved next to 0, where 32 bits show 1e-10: what is left is the error of lse.  Rows whose best
    token comes last, 0 to 16 above all before it, and rows without one; far from zero too, where log2 e has to be good to
    more than 32 bits."""
    import l20_beam_search as bs

    g = torch.Generator(device="cuda").manual_seed(rows + int(offset))
    x = offset + 2 * torch.randn(rows, 1, vocab, generator=g, device="cuda")
    if late:
        at = torch.randint(vocab - vocab // 8, vocab, (rows, 1, 1), generator=g, device="cuda")
        gap = 16 * torch.rand(rows, 1, 1, generator=g, device="cuda")
        x.scatter_(2, at, x.amax(-1, keepdim=True) + gap)
    x = x.to(DTYPES[dtype])
    wide = x.double()
    lse, best = torch.logsumexp(wide, -1), wide.amax(-1)
    scores = (lse - best).float()
    out = bs.l20_beam_search_step(x, scores, out=filled(rows, 1))
    want = scores.double() + (best - lse)
    off = (out.scores.double() - want).abs()
    assert out.tokens.equal(wide.argmax(-1)) and (out.parents == 0).all()
    over = float((off / (2.0 ** -24 * want.abs() + lse_bound(wide))).max())
    assert over <= 1, f"errors up to {float(off.max()):.2g}, {float(off.mean()):.2g} on average"


# --------------------------------------------------------------------------- workgroups shared out over the live rows
LIVE = {"all": lambda r, w: True, "scattered": lambda r, w: (7 * r + 3 * w) % 5 > 1, "one beam a request": lambda r, w: w == r % 3,
        "one row": lambda r, w: (r, w) == (41, 2), "whole requests": lambda r, w: r % 9 == 4, "the last": lambda r, w: r > 66,
        "none": lambda r, w: False}


@pytest.mark.parametrize("live", LIVE)
@pytest.mark.parametrize("dtype,flat", [("bf16", True), ("bf16", False), ("fp32", False)], ids=["bf16", "bf16 strided", "fp32 strided"])
def test_runs_shared_out_over_live_rows(live, dtype, flat):
    """More rows than there are workgroups for the runs that live ones may get: every number of live rows, so that lists and
    sums lie further apart than they are filled.  What the workspace holds before does not matter."""
    import l20_beam_search as bs

    requests, beams, vocab, ends = 69, 4, 30000, [17, 29999]
    rows, most = requests * beams, min(64, (-(-vocab // 2048) + 3) // 4)
    spread = 3 * torch.cuda.get_device_properties(0).multi_processor_count
    assert rows % 64 and max(spread // rows, 1) < most, "the rows are not shared out"
    logits, scores = inputs(requests, beams, vocab, DTYPES[dtype], seed=len(live))
    logits[:, ::2, 17] += 9
    logits[:, 1, 29999] += 10
    dead = torch.tensor([[not LIVE[live](r, w) for w in range(beams)] for r in range(requests)])
    scores[dead] = -math.inf
    scores[::2] = torch.where(dead[::2], math.nan, scores[::2])
    logits[dead] = math.nan  # (nothing of it matters)
    s = scores.cuda() if flat else torch.full((beams, 2 * requests), 3.0, device="cuda")[:, ::2].t().copy_(scores)
    x = logits.cuda()
    ws = bs.allocate_l20_beam_search_workspace(x, s, end_tokens=ends)
    out = None
    for fill in (255, 0, 85):
        ws.fill_(fill)
        got = bs.l20_beam_search_step(x, s, end_tokens=ends, out=filled(requests, beams), workspace=ws)
        torch.cuda.synchronize()
        assert out is None or all(a.equal(b) for a, b in zip(got, out))
        out = got
    if dead.all():
        assert all((t == v).all() for t, v in zip(out, (-1, -1, -math.inf) * 2))
    else:
        compare(out, logits, scores, ends)


def test_one_workspace_for_rows_shared_out_and_not():
    """The same workspace for a batch whose rows are shared out, smaller ones that get all their runs, and dead ones."""
    import l20_beam_search as bs

    logits, scores = inputs(130, 4, 20000, torch.bfloat16, seed=5)
    x, full = logits.cuda(), scores.cuda()
    ws = bs.allocate_l20_beam_search_workspace(x, full, end_tokens=[3])
    for n, step in ((130, 1), (2, 1), (130, 3), (40, 1), (130, 50)):
        s = full[:n].clone()
        s[:, 1:][torch.arange(n) % step > 0] = -math.inf
        got = bs.l20_beam_search_step(x[:n], s, end_tokens=[3], out=filled(n, 4), workspace=ws)
        compare(got, logits[:n], s.cpu(), [3])
