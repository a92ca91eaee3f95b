"""GPU: rows that follow their parents, compaction of the pool and copies of pages against the same rules in plain
Python (whole numbers and bytes: equal)."""

import random

import pytest
import torch

import beam_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")
    import l20_block_tables  # noqa: F401


def t32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(groups, beams, page, longest, spare, seed, lens=None, shared=0.6):
    """A pool in the middle of a search: each group's rows share a prefix, sometimes more of it among themselves."""
    rng = random.Random(seed)
    width = -(-longest // page) + 2
    table, all_lens, shares, used = [], [], {}, 0

    def page_of(holders):
        nonlocal used
        shares[used] = holders - 1
        used += 1
        return used - 1

    for g in range(groups):
        rows = []
        n = rng.randint(0, longest) if lens is None else lens[g]
        mine = [n if rng.random() < 0.8 else rng.randint(0, longest) for _ in range(beams)] if lens is None else [n] * beams
        full = min(mine) // page
        common = rng.randint(0, full) if rng.random() < shared else 0
        head = [page_of(beams) for _ in range(common)]
        for m in mine:
            held = -(-m // page)
            rows.append(head + [page_of(1) for _ in range(held - common)] + [-9] * (width - held))
        table += rows
        all_lens += mine
    pages = used + spare
    number = list(range(pages))
    rng.shuffle(number)
    free = number[used:]
    rng.shuffle(free)
    return {"table": [[number[v] if v >= 0 else v for v in r] for r in table], "lens": all_lens,
            "shares": [shares.get(number.index(v), 0) for v in range(pages)] if pages < 400 else
            [x for _, x in sorted((number[v], shares.get(v, 0)) for v in range(pages))],
            "free": free + [-5] * (used + 7), "count": len(free), "page": page}


def parents_of(groups, beams, seed, released=0.2):
    rng = random.Random(1000 + seed)
    return [[-1] * beams if rng.random() < released else [rng.choice([-1, *range(beams)] if rng.random() < 0.1 else range(beams))
                                                          for _ in range(beams)] for _ in range(groups)]


def on_device(c):
    dev = {k: t32(c[k]) for k in ("table", "lens", "shares", "free")}
    dev["count"] = t32([c["count"]])
    return dev


def listed(copies):
    n, short = copies.count.tolist()
    src, dst, tokens = copies.src.tolist(), copies.dst.tolist(), copies.tokens.tolist()
    assert set(src[n:]) <= {-1} and set(dst[n:]) <= {-1} and set(tokens[n:]) <= {0}
    return list(zip(src[:n], dst[:n], tokens[:n])), short


def check_reorder(c, parents, **kw):
    import l20_block_tables as bt

    dev = on_device(c)
    copies = bt.l20_reorder_block_tables(t32(parents), dev["table"], dev["lens"], dev["shares"], dev["free"], dev["count"],
                                         c["page"], **kw)
    torch.cuda.synchronize()
    want = R.reorder(parents, c["table"], c["lens"], c["shares"], c["free"], c["count"], c["page"])
    pairs, short = listed(copies)
    for name, got, expect in (("table", dev["table"].tolist(), want[0]), ("lens", dev["lens"].tolist(), want[1]),
                              ("shares", dev["shares"].tolist(), want[2]), ("free", dev["free"].tolist(), want[3]),
                              ("count", int(dev["count"]), want[4]), ("pairs", pairs, want[5]), ("short", short, want[6])):
        assert got == expect, name
    return dict(zip(("table", "lens", "shares", "free", "count"), want), page=c["page"], pairs=want[5], short=want[6])


def held_once(c):
    """Holders, shares and stack agree: no page is lost and none is in two places."""
    holders = {}
    for r, n in zip(c["table"], c["lens"]):
        for v in r[:R.pages_of(n, c["page"], len(r))]:
            holders[v] = holders.get(v, 0) + 1
    free = c["free"][:c["count"]]
    assert len(set(free)) == len(free) and not set(free) & set(holders)
    assert sorted([*free, *holders]) == list(range(len(c["shares"])))
    assert all(c["shares"][v] == n - 1 for v, n in holders.items()) and all(c["shares"][v] == 0 for v in free)


@pytest.mark.parametrize("beams", [1, 2, 3, 8, 17, 32])
@pytest.mark.parametrize("page", [16, 48])
def test_reorder_random(beams, page):
    for seed in range(4):
        groups = random.Random(seed).choice([1, 2, 9])
        c = pool(groups, beams, page, longest=page * 7, spare=groups * beams + 3, seed=seed)
        held_once(c)
        held_once(check_reorder(c, parents_of(groups, beams, seed)))


def test_reorder_edges_of_pages():
    """Lengths around a page's end: a page that is not full is copied, a full one is not, no page at all."""
    lens = [0, 1, 15, 16, 17, 31, 32, 160, 159]
    c = pool(9, 4, 16, longest=160, spare=40, seed=2, lens=lens)
    after = check_reorder(c, [[2, 2, 0, 2]] * 9)
    held_once(after)
    assert sorted({t for _, _, t in after["pairs"]}) == [1, 15] and len(after["pairs"]) == 2 * 5
    held_once(check_reorder(after, [[3, 1, 1, 1]] * 9))


def test_reorder_keeps_a_page_in_its_own_row():
    c = pool(1, 4, 16, longest=20, spare=9, seed=1, lens=[20], shared=0.0)
    after = check_reorder(c, [[2, 2, 2, 0]])
    assert after["table"][2] == c["table"][2] and [s for s, _, _ in after["pairs"]] == [c["table"][2][1]] * 2
    after = check_reorder(c, [[3, 3, 0, 0]])  # neither parent stays: their first children keep
    assert after["table"][0] == c["table"][3] and after["table"][2] == c["table"][0]


def test_reorder_of_a_prompt_into_its_beams_and_back():
    c = pool(3, 5, 16, longest=100, spare=40, seed=6, lens=[100, 64, 7])
    first = check_reorder(c, [[-1, -1, 4, -1, -1]] * 3)
    held_once(first)
    forked = check_reorder(first, [[2] * 5] * 3)
    held_once(forked)
    assert len(forked["pairs"]) == 8
    gone = check_reorder(forked, [[-1] * 5] * 3)
    held_once(gone)
    assert gone["count"] == len(gone["shares"])


def test_reorder_shares_between_groups():
    """Two groups hold one prefix (a cached prompt): it stays until the last row lets go."""
    table = [[4, 2, 9, -1], [4, 2, 8, -1], [4, 2, 7, -1], [4, 2, 6, -1]]
    shares = [0] * 10
    shares[4] = shares[2] = 3
    c = {"table": table, "lens": [40] * 4, "shares": shares, "free": [0, 1, 3, 5, -1, -1, -1, -1, -1, -1], "count": 4, "page": 16}
    held_once(c)
    one = check_reorder(c, [[-1, -1], [1, -1]])
    held_once(one)
    assert one["shares"][4] == 0 and one["count"] == 7
    both = check_reorder(c, [[-1, -1], [-1, -1]])
    held_once(both)
    assert both["free"][:10] == [0, 1, 3, 5, 2, 4, 6, 7, 8, 9]
    held_once(check_reorder(c, [[1, 1], [0, 0]]))


def test_reorder_when_pages_run_out():
    c = pool(4, 4, 16, longest=40, spare=5, seed=3, lens=[40, 40, 40, 40], shared=0.0)
    c["count"] = 0
    after = check_reorder(c, [[0, 0, 1, 2], [0, 0, 0, 0], [3, 2, 1, 0], [1, 1, 2, 3]])  # gives up as much as it needs
    assert after["short"] == 0
    first = check_reorder(c, [[0, -1, -1, -1]] * 4)
    first["count"] = 4
    after = check_reorder(first, [[0, 0, 0, 0]] * 4)
    assert len(after["pairs"]) == 4 and after["short"] == 8
    assert sum(r.count(-1) for r in after["table"]) == 8


@pytest.mark.parametrize("groups", [1, 20], ids=["one launch", "two"])
def test_reorder_that_forks_again_needs_the_pages_it_gave_up(groups):
    """A step with fewer running beams gives their pages back; one that has all beams again takes a page for each beam that
    it gains, and a row without one is counted where others took them meanwhile."""
    c = pool(groups, 4, 16, longest=20, spare=0, seed=17, lens=[20] * groups, shared=0.0)
    fewer = check_reorder(c, [[0, 1, -1, -1]] * groups)
    held_once(fewer)
    assert fewer["count"] == 4 * groups and not fewer["pairs"] and fewer["short"] == 0
    for left in (0, 1, 2 * groups - 1, 2 * groups):  # what others left on the stack
        after = check_reorder(dict(fewer, count=left), [[0, 0, 1, 1]] * groups)
        assert len(after["pairs"]) == left and after["short"] == 2 * groups - left
        assert sum(r[1] == -1 for r in after["table"]) == after["short"]
    # as many running beams as before: what a step takes it has given up
    same = check_reorder(dict(c, count=0), [[0, 0, 1, 1]] * groups)
    assert same["short"] == 0 and len(same["pairs"]) == 2 * groups


@pytest.mark.parametrize("groups,beams", [(3, 4), (20, 5)], ids=["one launch", "two"])
def test_reorder_takes_a_page_for_each_beam_that_it_gains(groups, beams):
    """Beams of one length with a page each that is not full: whatever the parents, a step is short of exactly the pages
    that it gains live rows and that the stack does not hold."""
    rng = random.Random(23)
    c = pool(groups, beams, 16, longest=15, spare=0, seed=beams, lens=[1 + g % 15 for g in range(groups)], shared=0.0)
    for left in (0, 1, 3, 7):
        state, live = c, groups * beams
        for most in (2, beams, 1, beams):
            parents = []
            for g in range(groups):
                alive = [q for q in range(beams) if state["lens"][g * beams + q]]
                now = rng.randint(1, most)
                parents.append([rng.choice(alive) if i < now else -1 for i in range(beams)])
            gained = sum(q >= 0 for row in parents for q in row) - live
            after = check_reorder(dict(state, count=min(left, state["count"])), parents)
            assert after["short"] == max(0, gained - min(left, state["count"]))
            state = check_reorder(state, parents)
            held_once(state)
            assert state["short"] == 0
            live += gained


@pytest.mark.parametrize("groups", [2, 20], ids=["one launch", "two"])
def test_reorder_children_of_a_row_without_its_last_page(groups):
    """What found no page has none to copy from either: its children get the same number, masked as it is, and take no
    page from the pool, whose contents would be another's."""
    c = pool(groups, 4, 16, longest=40, spare=0, seed=8, lens=[40] * groups, shared=0.0)
    first = check_reorder(c, [[0, -1, -1, -1]] * groups)
    first["count"] = 0
    short = check_reorder(first, [[0, 0, 0, 0]] * groups)
    assert short["short"] == 3 * groups and not short["pairs"]
    short["free"], short["count"] = [v for v in range(len(c["shares"])) if not any(v in r[:3] for r in short["table"])], 2 * groups
    after = check_reorder(short, [[2, 2, 3, 2]] * groups)
    assert after["short"] == 0 and not after["pairs"]
    assert all(r[2] == -1 for r in after["table"])
    back = check_reorder(after, [[-1, -1, -1, -1]] * groups)
    assert back["count"] == after["count"] + 2 * groups
    # a number beyond the pool is no page either, and lies in a column where the child held another one
    c["table"][1][2] = 10 ** 7
    odd = check_reorder(c, [[1, 1, 1, 3]] + [[0, 1, 2, 3]] * (groups - 1))
    assert [r[2] for r in odd["table"][:3]] == [10 ** 7] * 3 and not odd["pairs"]


def test_reorder_with_bad_numbers():
    """Numbers outside the pool in table, stack and parents, negative lengths, rows longer than the table, a stack too
    small for what comes back: nothing is read or written out of bounds, and the rules hold."""
    c = pool(3, 3, 16, longest=60, spare=6, seed=4, lens=[60, 55, 30], shared=0.0)
    c["table"][0][1], c["table"][4][0], c["table"][7][1] = 10 ** 6, -3, -2 ** 31
    c["free"][c["count"] - 2] = len(c["shares"])
    c["lens"][2], c["lens"][8] = -5, 2 ** 31 - 1
    c["free"] = c["free"][:c["count"] + 2]
    check_reorder(c, [[0, 0, 2], [1, 7, 1], [-4, 1, 1]])
    one = check_reorder(c, [[0, -1, -1], [-1, 1, -1], [1, -1, -1]])
    for k in range(1, one["count"], 2):
        one["free"][k] = (-1, len(c["shares"]), 10 ** 9)[k % 3]
    after = check_reorder(one, [[0, 0, 0], [1, 1, 1], [0, 0, 0]])
    assert after["short"] >= 2 and after["pairs"]
    c["count"] = -3
    check_reorder(c, [[0, 0, 0]] * 3)
    c["count"] = 10 ** 6
    check_reorder(c, [[0, 0, 0]] * 3)
    c["count"], c["free"] = 0, [-1]
    check_reorder(c, [[-1, -1, -1]] * 3)


def test_reorder_large():
    """Long rows, the most rows, and a pool of more pages than one pass of the bitmap holds."""
    c = pool(24, 4, 16, longest=5000, spare=120, seed=11)
    held_once(check_reorder(c, parents_of(24, 4, 11)))
    c = pool(256, 32, 16, longest=40, spare=8192, seed=12)
    held_once(check_reorder(c, parents_of(256, 32, 12)))
    c = pool(2, 2, 16, longest=90, spare=5, seed=13)
    far = 1_200_000
    moved = {v: far + v if v % 3 else v for v in range(len(c["shares"]))}
    c["table"] = [[moved.get(v, v) for v in r] for r in c["table"]]
    c["free"] = [moved.get(v, v) for v in c["free"]]
    shares = [0] * (far + 100)
    for v, s in enumerate(c["shares"]):
        shares[moved[v]] = s
    c["shares"] = shares
    check_reorder(c, [[1, 1], [-1, -1]])
    check_reorder(c, [[-1, -1], [-1, -1]])


@pytest.mark.parametrize("spare", [9000, 300_000], ids=["one bitmap", "two"])
def test_reorder_more_lists_than_are_looked_at_together(spare):
    """The most rows, in more column blocks than one pass over the lists of freed pages takes (4096), short and long ones:
    pages come back, and copies are taken, in both passes."""
    rng = random.Random(spare)
    lens = [4780 + g % 16 if g % 97 == 3 or g > 1020 else rng.randint(0, 60) for g in range(1024)]
    c = pool(1024, 8, 16, longest=4796, spare=spare, seed=14, lens=lens)
    assert 1024 * -(-len(c["table"][0]) // 64) > 4096 and (len(c["shares"]) > 1 << 18) == (spare > 9000)
    after = check_reorder(c, parents_of(1024, 8, 14))
    held_once(after)
    freed = {v for v in after["free"][:after["count"]]} - {v for v in c["free"][:c["count"]]}
    rows = [r for r, n in enumerate(c["lens"]) for v in c["table"][r][:R.pages_of(n, 16, 302)] if v in freed]
    assert min(rows) < 8 * 800 and max(rows) > 8 * 1000  # (lists of a group lie together, 5 a group)
    held_once(check_reorder(after, [[-1] * 8] * 1024))


def test_reorder_row_strides_and_no_groups():
    import l20_block_tables as bt

    c = pool(2, 3, 16, longest=50, spare=9, seed=5)
    wide = torch.full((6, 40), -8, dtype=torch.int32, device="cuda")
    n = len(c["table"][0])
    wide[:, :n] = t32(c["table"])
    dev = on_device(c)
    bt.l20_reorder_block_tables(t32([[1, 0, 0], [2, 2, 2]]), wide[:, :n], dev["lens"], dev["shares"], dev["free"], dev["count"], 16)
    want = R.reorder([[1, 0, 0], [2, 2, 2]], c["table"], c["lens"], c["shares"], c["free"], c["count"], 16)
    assert wide[:, :n].tolist() == want[0] and (wide[:, n:] == -8).all()
    empty = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    copies = bt.l20_reorder_block_tables(empty.view(0, 4), empty, empty[:, 0].contiguous(), dev["shares"], dev["free"], dev["count"], 16)
    assert copies.count.tolist() == [0, 0] and int(dev["count"]) == want[4]


@pytest.mark.parametrize("pages", [1 << 18, (1 << 18) + 1, 300_000, 600_000])
def test_reorder_no_groups_of_a_large_pool(pages):
    """Nothing to do, but the copies still say so; around the number of pages that one launch's bitmap holds."""
    import l20_block_tables as bt

    empty = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    shares, free, count = torch.zeros(pages, dtype=torch.int32, device="cuda"), t32([4, 9, pages - 1]), t32([2])
    copies = bt.PageCopies.empty(5, "cuda")
    for t in copies:
        t.fill_(99)
    bt.l20_reorder_block_tables(empty, empty, empty[:, 0].contiguous(), shares, free, count, 16, copies=copies)
    assert copies.src.tolist() == copies.dst.tolist() == [-1] * 5 and copies.tokens.tolist() == [0] * 5
    assert copies.count.tolist() == [0, 0] and count.tolist() == [2] and free.tolist() == [4, 9, pages - 1]
    assert int(shares.abs().sum()) == 0


def test_reorder_replayed_with_the_block_tables():
    """A captured step -- append a token, follow the parents -- whose state advances in device memory; every replay
    equals the plain rules, with eager work between."""
    import l20_block_tables as bt
    import latent_ref as L

    page, beams, groups = 16, 3, 4
    c = pool(groups, beams, page, longest=40, spare=60, seed=9)
    c["table"] = [r + [-9] * 8 for r in c["table"]]
    rows, width = groups * beams, len(c["table"][0])
    dev, fresh, parents = on_device(c), t32([1] * rows), t32([[0, 1, 2]] * groups)
    slots, positions = (torch.zeros(rows, dtype=torch.int64, device="cuda") for _ in range(2))
    cu, lens = t32([0] * (rows + 1)), t32([0] * rows)
    copies = bt.PageCopies.empty(rows + 2, "cuda")
    ws = bt.allocate_l20_reorder_workspace(parents, dev["table"])

    def step():
        bt.l20_build_block_tables(dev["lens"], fresh, dev["table"], dev["free"], dev["count"], slots, positions, cu, lens, page)
        bt.l20_reorder_block_tables(parents, dev["table"], lens, dev["shares"], dev["free"], dev["count"], page, copies=copies,
                                    workspace=ws)
        dev["lens"].copy_(lens)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k, v in on_device(c).items():
        dev[k].copy_(v)
    rng = random.Random(3)
    for n in range(25):
        mine = [[rng.randrange(beams) for _ in range(beams)] for _ in range(groups)]
        if n == 12:
            mine[1] = [-1] * beams
        parents.copy_(t32(mine))
        ws.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        built = L.block_tables(c["lens"], [1] * rows, c["table"], c["free"], c["count"], rows, page)
        want = R.reorder(mine, built["table"], built["seq_lens"], c["shares"], built["free"], built["left"], page)
        c.update(zip(("table", "lens", "shares", "free", "count"), want))
        assert dev["table"].tolist() == c["table"] and dev["lens"].tolist() == c["lens"] and dev["shares"].tolist() == c["shares"]
        assert dev["free"].tolist() == c["free"] and int(dev["count"]) == c["count"] and listed(copies) == (want[5], want[6])
        held_once(c)
    assert width * page > max(c["lens"])


def test_two_pools_on_two_streams():
    """Calls on two pools, of one launch and of two, each on its stream with its workspace: as alone."""
    import l20_block_tables as bt

    runs = []
    for groups, beams, spare in ((3, 4, 60), (40, 3, 400)):
        c = pool(groups, beams, 16, longest=100, spare=spare, seed=groups)
        steps = [parents_of(groups, beams, 50 + n, released=0.05) for n in range(6)]
        sent, dev, stream = [t32(p) for p in steps], on_device(c), torch.cuda.Stream()
        runs.append((c, steps, sent, dev, stream, bt.allocate_l20_reorder_workspace(sent[0], dev["table"]),
                     [bt.PageCopies.empty(groups * beams, "cuda") for _ in steps]))
    torch.cuda.synchronize()
    for n in range(6):
        for _, _, sent, dev, stream, ws, copies in runs:
            with torch.cuda.stream(stream):
                bt.l20_reorder_block_tables(sent[n], dev["table"], dev["lens"], dev["shares"], dev["free"], dev["count"], 16,
                                            copies=copies[n], workspace=ws)
    torch.cuda.synchronize()
    for c, steps, _, dev, _, _, copies in runs:
        for parents, pairs in zip(steps, copies):
            want = R.reorder(parents, c["table"], c["lens"], c["shares"], c["free"], c["count"], 16)
            c.update(zip(("table", "lens", "shares", "free", "count"), want))
            assert listed(pairs) == (want[5], want[6])
        held_once(c)
        for k in ("table", "lens", "shares", "free"):
            assert dev[k].tolist() == c[k], k
        assert int(dev["count"]) == c["count"]


# --------------------------------------------------------------------------- compaction
def check_compact(c, limit, room=None):
    import l20_block_tables as bt

    dev = on_device(c)
    copies = None if room is None else bt.PageCopies.empty(room, "cuda")
    copies = bt.l20_compact_pages(limit, dev["table"], dev["lens"], dev["shares"], dev["free"], dev["count"], c["page"], copies=copies)
    torch.cuda.synchronize()
    want = R.compact(limit, c["table"], c["lens"], c["shares"], c["free"], c["count"], c["page"], copies.src.shape[0])
    pairs, left = listed(copies)
    for name, got, expect in (("table", dev["table"].tolist(), want[0]), ("shares", dev["shares"].tolist(), want[1]),
                              ("free", dev["free"].tolist(), want[2]), ("count", int(dev["count"]), want[3]),
                              ("pairs", pairs, want[4]), ("left", left, want[5])):
        assert got == expect, name
    assert dev["lens"].tolist() == c["lens"]
    return dict(c, table=want[0], shares=want[1], free=want[2], count=want[3]), pairs, left


@pytest.mark.parametrize("page", [16, 80])
@pytest.mark.parametrize("spare", [0, 1, 30, 400])
def test_compact_random(page, spare):
    for seed in range(3):
        c = pool(5, 3, page, longest=page * 9, spare=spare, seed=seed)
        used = len(c["shares"]) - c["count"]
        for limit in (used, used + spare // 2, len(c["shares"]), used // 2, 0):
            after, pairs, left = check_compact(c, limit)
            if limit >= used:
                assert left == 0 and after["count"] == limit - used
                assert all(v < limit for r, n in zip(after["table"], after["lens"]) for v in r[:R.pages_of(n, page, len(r))])


def test_compact_room_rows_and_bad_numbers():
    c = pool(4, 2, 16, longest=100, spare=90, seed=8)
    used = len(c["shares"]) - c["count"]
    _, pairs, left = check_compact(c, used, room=3)
    assert len(pairs) == 3 and left > 0
    check_compact(c, used, room=0)
    c["table"][0][0], c["table"][3][0] = -7, 10 ** 7
    c["free"][0], c["free"][1], c["free"][2] = -2, 10 ** 7, c["free"][3]
    c["lens"][1], c["lens"][2] = -1, 2 ** 31 - 1
    check_compact(c, used)
    c["count"] = 10 ** 6
    check_compact(c, used)
    c["count"] = -1
    check_compact(c, used)


def test_compact_large_pool():
    c = pool(40, 4, 16, longest=4000, spare=30000, seed=21)
    used = len(c["shares"]) - c["count"]
    after, _, left = check_compact(c, used + 5)
    assert left == 0 and after["count"] == 5
    c = pool(10, 4, 16, longest=2000, spare=700_000, seed=22)  # more than one thread takes a page of
    used = len(c["shares"]) - c["count"]
    for limit in (used + 400_000, used, 300):
        check_compact(c, limit)


def test_compact_no_rows_and_graph():
    import l20_block_tables as bt

    empty = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    shares, free, count = t32([0] * 40), t32([30, 3, 20, 5]), t32([4])
    copies = bt.l20_compact_pages(20, empty, empty[:, 0].contiguous(), shares, free, count, 16)
    assert copies.count.tolist() == [0, 0] and int(count) == 2 and free.tolist()[:2] == [5, 3]
    c = pool(3, 3, 16, longest=90, spare=50, seed=30)
    limit = len(c["shares"]) - c["count"] + 2
    dev, saved = on_device(c), on_device(c)
    copies, ws = bt.PageCopies.empty(60, "cuda"), bt.allocate_l20_compact_workspace(dev["shares"])

    def step():
        for k, v in saved.items():
            dev[k].copy_(v)
        bt.l20_compact_pages(limit, dev["table"], dev["lens"], dev["shares"], dev["free"], dev["count"], 16, copies=copies, workspace=ws)

    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (*dev.values(), *copies)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        ws.fill_(-1)
        for t in (*dev.values(), *copies):
            t.fill_(99)
        graph.replay()
        torch.cuda.synchronize()
        assert all(a.equal(b) for a, b in zip((*dev.values(), *copies), want))


# --------------------------------------------------------------------------- copies
def random_bytes(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * n), generator=g, dtype=torch.uint8)
    return raw.view(dtype).cuda()


def raw(t):
    return t.contiguous().view(torch.uint8).cpu()


def check_copy(caches, src, dst, tokens=None, count=None):
    import l20_block_tables as bt

    want = [raw(c).clone() for c in caches]
    n = len(src) if count is None else min(max(count[0], 0), len(src))
    for w in want:
        before = w.clone()
        for k in range(n):
            if 0 <= src[k] < w.shape[0] and 0 <= dst[k] < w.shape[0]:
                m = w.shape[1] if tokens is None else min(max(tokens[k], 0), w.shape[1])
                w[dst[k], :m] = before[src[k], :m]
    bt.l20_copy_pages(bt.PageCopies(t32(src), t32(dst), None if tokens is None else t32(tokens), None if count is None else t32(count)),
                      caches)
    torch.cuda.synchronize()
    for i, (c, w) in enumerate(zip(caches, want)):
        assert raw(c).equal(w), i


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.uint8], ids=["e4m3", "bf16", "fp32", "u8"])
@pytest.mark.parametrize("inside", [(16, 4, 128), (32, 576), (16, 1, 5), (48, 3, 7), (1, 8), (16, 2, 64, 2)], ids=str)
def test_copy_layouts(dtype, inside):
    src, dst = [3, 11, 0, 7], [1, 2, 9, 10]
    for tokens in (None, [inside[0], 1, 0, min(15, inside[0])]):
        caches = [random_bytes((12, *inside), dtype, seed) for seed in range(3)]
        check_copy(caches, src, dst, tokens)


def test_copy_views():
    """Keys and values side by side, heads outside tokens, padded rows, rows at odd offsets, tokens innermost."""
    src, dst, tokens = [5, 0, 2], [1, 4, 3], [16, 3, 9]
    both = random_bytes((6, 2, 16, 4, 64), torch.float8_e4m3fn, 1)
    check_copy(list(both.unbind(1)), src, dst, tokens)
    check_copy(list(random_bytes((6, 4, 16, 128), torch.bfloat16, 2).permute(0, 2, 1, 3).unsqueeze(0)), src, dst, tokens)
    check_copy([random_bytes((6, 16, 3, 80), torch.bfloat16, 3)[..., :64]], src, dst, tokens)
    check_copy([random_bytes((6, 16, 3, 9), torch.uint8, 4)[..., 1:8]], src, dst, tokens)
    check_copy([random_bytes((6, 4, 64, 16), torch.bfloat16, 5).permute(0, 3, 1, 2)], src, dst, tokens)
    check_copy([random_bytes((6, 4, 64, 16), torch.bfloat16, 5).permute(0, 3, 1, 2)], src, dst)
    check_copy([random_bytes((4, 6, 16, 32), torch.float16, 6).permute(1, 2, 0, 3)], src, dst, tokens)  # heads outside pages
    check_copy([random_bytes((6, 32, 40), torch.float16, 7)[:, ::2, :24]], src, dst, tokens)


@pytest.mark.parametrize("page,dim", [(64, 128), (64, 576), (256, 128), (64, 132), (80, 130)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.bfloat16, torch.uint8], ids=["e4m3", "bf16", "u8"])
def test_copy_runs_inside_a_page(page, dim, dtype):
    """A page of several runs of bytes, each by itself: heads outside tokens, whole and in part (tokens that end inside a
    load of 16 bytes, and runs longer than what a workgroup takes at once); heads outside the pages; padded heads."""
    src, dst, tokens = [5, 0, 2, 6], [1, 4, 3, 7], [page, 3, 41, 0]
    heads = 3

    def held(*shape):
        return random_bytes(shape, dtype, page + dim)

    for view in (held(8, heads, page, dim).permute(0, 2, 1, 3), held(heads, 8, page, dim).permute(1, 2, 0, 3),
                 held(8, heads, page + 3, dim)[:, :, :page].permute(0, 2, 1, 3), held(8, heads + 1, page, dim)[:, 1:].permute(0, 2, 1, 3),
                 held(8, 2, heads, page, dim)[:, 1].permute(0, 2, 1, 3)):
        assert view.shape[1:] == (page, heads, dim)
        check_copy([view], src, dst, tokens)
        check_copy([view], dst, src)
    caches = [held(8, heads, page, dim).permute(0, 2, 1, 3) for _ in range(3)]
    check_copy(caches, src, dst, tokens, [2, 0])


def test_copy_many_caches_and_mixed_layouts():
    caches = [random_bytes((8, 16, 2, 64), torch.float8_e4m3fn, s) for s in range(70)]
    caches += [random_bytes((8, 16, 576), torch.bfloat16, s) for s in range(3)] + [random_bytes((5, 32, 8), torch.float32, 9)]
    check_copy(caches, [4, 1, 7], [2, 3, 0], [5, 16, 11], [2, 0])
    check_copy(caches, [4, 1, 7], [2, 3, 0], [5, 16, 11])
    check_copy([], [1], [0])


def test_copy_counts_and_bad_pages():
    for count in ([0, 5], [-2, 0], [3, 0], [99, 0]):
        check_copy([random_bytes((9, 16, 64), torch.bfloat16, 1)], [0, 8, 9, -1, 2], [4, 5, 6, 7, 9], [16, 40, 3, 3, 3], count)
    check_copy([random_bytes((9, 16, 64), torch.bfloat16, 1)], [], [])
    check_copy([random_bytes((9, 16, 64), torch.bfloat16, 1)], [3, 2 ** 31 - 1, -2 ** 31], [3, 0, 1], [-5, 2, 2])


def test_copy_large_pages_beyond_32_bits():
    """Pages whose bytes lie beyond 2^32 of their cache."""
    cache = torch.zeros(70000, 64, 1024, dtype=torch.uint8, device="cuda")  # 4.6 GB
    cache[69999] = random_bytes((64, 1024), torch.uint8, 1)
    import l20_block_tables as bt

    bt.l20_copy_pages(bt.PageCopies(t32([69999, 69999]), t32([3, 66000]), t32([64, 20])), [cache])
    assert cache[3].equal(cache[69999]) and cache[66000, :20].equal(cache[69999, :20]) and int(cache[66000, 20:].sum()) == 0


def test_copy_in_a_graph_and_on_another_stream():
    import l20_block_tables as bt

    caches = [random_bytes((9, 16, 4, 64), torch.bfloat16, s) for s in range(4)]
    copies = bt.PageCopies.empty(4, "cuda")
    for t, v in zip(copies, ([0, 1, 2, -1], [3, 4, 5, -1], [16, 7, 1, 0], [3, 0])):
        t.copy_(t32(v))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        bt.l20_copy_pages(copies, caches)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bt.l20_copy_pages(copies, caches)
    for n in range(3):
        caches[n][:3].copy_(random_bytes((3, 16, 4, 64), torch.bfloat16, 20 + n))
        want = [raw(c).clone() for c in caches]
        for w in want:
            for s, d, m in ((0, 3, 16), (1, 4, 7), (2, 5, 1)):
                w[d, :m] = w[s, :m]
        graph.replay()
        torch.cuda.synchronize()
        assert all(raw(c).equal(w) for c, w in zip(caches, want))


def test_refusals():
    import l20_block_tables as bt

    i = t32([0] * 8)
    with pytest.raises(RuntimeError, match="block table must be int32"):
        bt.l20_reorder_block_tables(i.view(2, 4), i.long().view(8, 1), i, i, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="a row of the block table each"):
        bt.l20_reorder_block_tables(i.view(2, 4)[:1], i.view(8, 1), i, i, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="a pair a row"):
        bt.l20_reorder_block_tables(i.view(2, 4), i.view(8, 1), i, i, i, i[:1], 16, copies=bt.PageCopies.empty(7, "cuda"))
    with pytest.raises(RuntimeError, match="page size"):
        bt.l20_compact_pages(4, i.view(8, 1), i, i, i, i[:1], 20)
    with pytest.raises(RuntimeError, match="limit must be"):
        bt.l20_compact_pages(9, i.view(8, 1), i, i, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="workspace is missing"):
        bt.l20_compact_pages(4, i.view(8, 1), i, i, i, i[:1], 16, workspace=i[:1])
    with pytest.raises(RuntimeError, match="must be \\[pages, page"):
        bt.l20_copy_pages(bt.PageCopies(i, i), [i])
    with pytest.raises(RuntimeError, match="parts overlap"):
        bt.l20_copy_pages(bt.PageCopies(i, i), [i.view(8, 1, 1).expand(8, 16, 4)])
    with pytest.raises(RuntimeError, match="pages overlap"):
        bt.l20_copy_pages(bt.PageCopies(i, i), [torch.zeros(900, device="cuda").as_strided((5, 16, 8), (64, 8, 1))])
    with pytest.raises(RuntimeError, match="too many strides"):
        bt.l20_copy_pages(bt.PageCopies(i, i), [torch.zeros(3, 16, 5, 6, 7, 8, device="cuda")[:, ::2, ::2, ::2, ::2, ::2]])
