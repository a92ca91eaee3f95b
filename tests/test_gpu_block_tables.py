"""GPU: block tables, slot maps and positions against the same rules in plain Python (whole numbers: equal)."""

import random

import pytest
import torch

import latent_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")
    import l20_block_tables  # noqa: F401


def t32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(cached, new, page, spare, width=None, free_cells=8, seed=0):
    rng = random.Random(seed)
    held = [-(-max(c, 0) // page) for c in cached]
    width = width or max(-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)) + 1
    ids = list(range(sum(held) + spare))
    rng.shuffle(ids)
    table = []
    for n in held:
        row, ids = ids[:min(n, width)], ids[n:]
        table.append(row + [-9] * (width - len(row)))
    free = ids + [-5] * (sum(held) + free_cells)
    return {"cached": cached, "new": new, "table": table, "free": free, "count": len(ids), "page": page}


def run(c, tokens, in_place=False):
    import l20_block_tables as bt

    dev = {"cached": t32(c["cached"]), "new": t32(c["new"]), "table": t32(c["table"]), "free": t32(c["free"]),
           "count": t32([c["count"]]), "left": t32([-1])}
    n = len(c["cached"])
    slots, positions = (torch.full((tokens,), -77, dtype=torch.int64, device="cuda") for _ in range(2))
    cu, lens = t32([-1] * (n + 1)), t32([-1] * n)
    bt.l20_build_block_tables(dev["cached"], dev["new"], dev["table"], dev["free"], dev["count"], slots, positions, cu, lens,
                              c["page"], **({} if in_place else {"free_count_out": dev["left"]}))
    torch.cuda.synchronize()
    left = dev["count"] if in_place else dev["left"]
    return {"table": dev["table"].tolist(), "free": dev["free"].tolist(), "left": int(left), "slots": slots.tolist(),
            "positions": positions.tolist(), "cu": cu.tolist(), "seq_lens": lens.tolist()}


def check(c, tokens, **kw):
    got = run(c, tokens, **kw)
    want = R.block_tables(c["cached"], c["new"], c["table"], c["free"], c["count"], tokens, c["page"])
    for name in want:
        assert got[name] == want[name], name
    return want


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("extra", [0, 5])
def test_edges_of_pages(page, extra):
    cached = [0, 1, page - 1, page, page + 1, 3 * page, 0, 7]
    new = [1, page - 1, 1, 1, 2 * page, 0, 3 * page + 1, page]
    check(make(cached, new, page, spare=60), sum(new) + extra)


def test_finished_requests_give_their_pages_to_the_others():
    want = check(make([100, 64, 17, 0, 33], [-1, 200, -1, 90, 1], 16, spare=2), 300)
    assert want["seq_lens"] == [0, 64, 0, 0, 34]  # 2 + 7 + 2 pages; 13 wanted by the second, so none is taken
    want = check(make([100, 64, 17, 0, 33], [-1, 100, -1, 60, 1], 16, spare=2), 300)
    assert want["seq_lens"] == [0, 164, 0, 60, 34] and want["left"] == 0


def test_pages_run_out_in_order():
    want = check(make([16, 16, 16, 15, 0], [17, 40, 1, 1, 16], 16, spare=4), 80)
    assert want["seq_lens"] == [33, 16, 16, 16, 0] and want["left"] == 2


def test_rows_and_slots_that_do_not_fit():
    c = make([0, 30, 0, 5, 9], [20, 100, 3, 10, 40], 16, spare=60, width=4)
    want = check(c, 140)
    assert want["seq_lens"][1] == 30 and want["seq_lens"][4] == 9  # beyond the table row; beyond the slots
    check(c, 0)
    check(c, 1)


def test_negative_cached_lengths_and_a_full_stack():
    c = make([50, 20], [-1, -4], 16, spare=0, free_cells=0)
    c["free"] = c["free"][:3]  # room for three of the six pages that come back
    check(c, 4)
    check(make([-3, 5], [20, 2], 16, spare=6), 30)


def test_count_in_place():
    check(make([0, 31, 40], [40, 2, -1], 16, spare=9), 50, in_place=True)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    rng = random.Random(seed)
    n = rng.choice([1, 3, 70, 1000, 2500])
    top = rng.choice([1, 40, 300]) if n > 100 else rng.choice([40, 3000])
    cached = [rng.randint(0, top * 2) for _ in range(n)]
    new = [rng.choice([-1, 0, 1, 1, rng.randint(0, top)]) for _ in range(n)]
    page = rng.choice([16, 32, 80])
    need = sum(max(x, 0) for x in new) // page + n
    c = make(cached, new, page, spare=rng.choice([need, need // 2 + 1]), seed=seed)
    check(c, max(1, sum(max(x, 0) for x in new) + rng.choice([-3, 0, 9])))


def test_most_requests_and_one_long_prompt():
    n = 8192
    check(make([15] * n, [2] * n, 16, spare=n, width=3), 2 * n)
    check(make([0, 100000], [70000, 1], 16, spare=4500), 70001)


def test_replayed_step_by_step():
    """A captured decode step: lengths and stack advance in device memory; every replay equals the plain rules."""
    import l20_block_tables as bt

    cached, page = [14, 3, 31, 0], 16
    c = make(cached, [1] * 4, page, spare=30, width=8)
    dev = {k: t32(c[k]) for k in ("cached", "new", "table", "free")}
    count, slots, positions = t32([c["count"]]), torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    cu, lens = t32([0] * 5), t32([0] * 4)

    def step():
        bt.l20_build_block_tables(dev["cached"], dev["new"], dev["table"], dev["free"], count, slots, positions, cu, lens, page)
        dev["cached"].copy_(lens)

    saved = dev["cached"].clone(), dev["table"].clone(), dev["free"].clone(), count.clone()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, s in zip((dev["cached"], dev["table"], dev["free"], count), saved):
        t.copy_(s)
    table, free, left = c["table"], c["free"], c["count"]
    for _ in range(40):
        want = R.block_tables(cached, [1] * 4, table, free, left, 6, page)
        graph.replay()
        torch.cuda.synchronize()
        assert slots.tolist() == want["slots"] and positions.tolist() == want["positions"]
        assert dev["table"].tolist() == want["table"] and int(count) == want["left"] and lens.tolist() == want["seq_lens"]
        cached, table, free, left = want["seq_lens"], want["table"], want["free"], want["left"]


def test_no_requests():
    import l20_block_tables as bt

    none, left, cu = t32([]), t32([0]), t32([9])
    slots, positions = torch.full((5,), 7, device="cuda"), torch.full((5,), 7, device="cuda")
    bt.l20_build_block_tables(none, none, t32([]).reshape(0, 4), t32([3, 1, 2]), t32([2]), slots, positions, cu, none, 16,
                              free_count_out=left)
    torch.cuda.synchronize()
    assert int(left) == 2 and cu.tolist() == [0] and slots.tolist() == [-1] * 5 and positions.tolist() == [0] * 5


def test_refusals():
    import l20_block_tables as bt

    c = make([1], [1], 16, spare=3)
    d = {k: t32(c[k]) for k in ("cached", "new", "table", "free")}
    i64 = torch.zeros(2, dtype=torch.int64, device="cuda")
    count, cu, lens = t32([3]), t32([0, 0]), t32([0])
    ok = [d["cached"], d["new"], d["table"], d["free"], count, i64, i64.clone(), cu, lens]

    def bad(match, page=16, **change):
        args = list(ok)
        for k, v in change.items():
            args[int(k[1:])] = v
        with pytest.raises(RuntimeError, match=match):
            bt.l20_build_block_tables(*args, page)

    bad("page size", page=24)
    bad("int32 \\[requests\\]", a1=d["new"].long())
    bad("block table", a2=d["table"].long())
    bad("int64 \\[tokens\\]", a5=i64.int())
    bad("requests \\+ 1", a7=t32([0]))
    bad("must not be cached_lens", a8=d["cached"])
    bad("same device", a4=count.cpu())
    bad("at most 8192", a0=t32([0] * 9000))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 4096])
@pytest.mark.parametrize("tokens", [40, 5000], ids=["one", "two"])
def test_lengths_up_to_the_largest(page, tokens):
    """Cached lengths around 2^30 and up to 2^31 - 1 exceed every row: such requests are not served and take no page,
    finished ones give back the pages their rows have, and the others are as without them."""
    large = [2 ** 30 - 2 * page, 2 ** 30 - page, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 5, 2 ** 30 + page, 2 ** 31 - 2 * page, 2 ** 31 - 2, 2 ** 31 - 1]
    cached, new = [], []
    for n in large:
        cached += [n, n, n, 5]
        new += [1, -1, 0, page]
    rows = len(cached)
    free = list(range(4 * rows, 4 * rows + 3 * rows))
    table = [[4 * b + k for k in range(4)] for b in range(rows)]
    c = {"cached": cached, "new": new, "table": table, "free": free + [-5] * (4 * rows), "count": len(free), "page": page}
    assert sum(max(n, 0) for n in new) >= 40
    want = check(c, tokens)
    assert [want["seq_lens"][b] for b in (0, 1, 2)] == [large[0], 0, large[0]]
