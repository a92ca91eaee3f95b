"""The measured cases of beam search over the paged cache.

Kinds of case (``kind``):

* ``beam``    -- one step's selection: the best continuations of each request's beams over the vocabulary;
* ``reorder`` -- block-table rows follow their parents: pages shared, copied on write, given back;
* ``copy``    -- the contents of pages, in the caches of all layers at once;
* ``compact`` -- pages held beyond a limit move below it, and tables, shares and the free stack with them.

``own`` chooses between the plain form of an operator (torch operations; scores in 64 bits, since the order of
candidates of different beams hangs on their last digits) and the framework's calls.
"""

import math
import os
import random
import sys

import torch

own = False

if os.path.join(os.getcwd(), "single-gpu-inference-lab_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "single-gpu-inference-lab_amd"))

_TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
CACHE_VALUES = 1 << 24  # random values that a cache is filled with, again and again


def _beam(name, requests, beams, vocab, **over):
    case = {"name": name, "kind": "beam", "requests": requests, "beams": beams, "vocab": vocab, "dtype": "bf16",
            "ends": 1, "first": False, "masked": 0.0, "stride": vocab}
    case.update(over)
    return case


def _reorder(name, groups, beams, lo, hi, **over):
    case = {"name": name, "kind": "reorder", "groups": groups, "beams": beams, "lo": lo, "hi": hi, "page": 16,
            "suffix": 64, "released": 0.0}
    case.update(over)
    return case


def _copy(name, pairs, layers, **over):
    case = {"name": name, "kind": "copy", "pairs": pairs, "layers": layers, "heads": 4, "dim": 128, "page": 16,
            "dtype": "bf16", "whole": False, "pool": 2 * pairs + 64}
    case.update(over)
    return case


def _compact(name, rows, lo, hi, pool, **over):
    case = {"name": name, "kind": "compact", "rows": rows, "lo": lo, "hi": hi, "pool": pool, "page": 16, "above": 0.5}
    case.update(over)
    return case


def listed():
    return [
        # One request, four beams, a small vocabulary: all latency.
        _beam("beam_1x4_v32000", 1, 4, 32000),
        # Odd vocabulary and rows, fp16, two end tokens, a tenth of the rows constrained to a few tokens.
        _beam("beam_16x5_v50257_fp16", 16, 5, 50257, dtype="fp16", ends=2, masked=0.1),
        # A serving step of 64 requests; rows padded, as a tensor-parallel head leaves them.
        _beam("beam_64x4_v128256", 64, 4, 128256, stride=128512),
        # The largest step: 1024 rows, streaming.
        _beam("beam_128x8_v152064", 128, 8, 152064),
        # The first step after the prompts, fp32 logits: one live beam a request.
        _beam("beam_first_64x8_fp32", 64, 8, 152064, dtype="fp32", first=True),
        # The beams of a few short requests: all latency.
        _reorder("reorder_4x4_short", 4, 4, 40, 400),
        # A serving step on long contexts that share their prompts.
        _reorder("reorder_64x4_8k", 64, 4, 4000, 8000),
        # Wide beams on pages of 64, a quarter of the requests finished and given back.
        _reorder("reorder_24x16_release", 24, 16, 1000, 6000, page=64, suffix=300, released=0.25),
        # What a step copies: the last pages of a few beams, keys and values of 28 layers, fp8.
        _copy("copy_step_12_fp8", 12, 28, dtype="e4m3"),
        # What a compaction moves: whole pages, bf16.
        _copy("copy_whole_512", 512, 28, whole=True),
        # A small pool.
        _compact("compact_16x2k", 16, 100, 2000, 4096),
        # A full serving pool, half of it held, shrunk to that half.
        _compact("compact_256x8k", 256, 500, 8000, 200000),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["beam"] * 5 + ["reorder"] * 3 + ["copy"] * 2 + ["compact"] * 2)
    while True:
        if kind == "beam":
            case = {"kind": kind, "requests": _log_int(rng, 1, 256), "beams": rng.choice([1, 2, 3, 4, 4, 5, 8, 10, 16, 32]),
                    "vocab": _log_int(rng, 200, 200000), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    "ends": rng.choice([0, 1, 1, 2, 4]), "first": rng.random() < 0.2, "masked": rng.choice([0.0, 0.0, 0.2])}
            case["stride"] = case["vocab"] + rng.choice([0, 0, 1, 8, 64])
            if case["requests"] * case["beams"] * case["vocab"] * _SIZE[case["dtype"]] <= 300_000_000:
                return case
        elif kind == "reorder":
            case = {"kind": kind, "groups": _log_int(rng, 1, 256), "beams": rng.choice([1, 2, 4, 4, 5, 8, 16, 32]), "lo": 1,
                    "hi": _log_int(rng, 8, 32768), "page": rng.choice([16, 16, 32, 64]), "suffix": _log_int(rng, 8, 1000),
                    "released": rng.choice([0.0, 0.0, 0.1, 0.5])}
            case["lo"] = max(1, case["hi"] // rng.randint(1, 16))
            if case["groups"] * case["beams"] <= 1024 and case["groups"] * case["beams"] * case["hi"] <= 400_000 * case["page"]:
                return case
        elif kind == "copy":
            case = {"kind": kind, "pairs": _log_int(rng, 1, 512), "layers": rng.choice([1, 4, 24, 28, 32]),
                    "heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 16, 32, 64]),
                    "dtype": rng.choice(["e4m3", "bf16", "fp16"]), "whole": rng.random() < 0.3}
            case["pool"] = 2 * case["pairs"] + rng.randint(1, 300)
            row = case["heads"] * case["dim"] * _SIZE[case["dtype"]] * case["page"] * 2 * case["layers"]
            if row * case["pairs"] <= 450_000_000 and row * case["pool"] <= 2_000_000_000:
                return case
        else:
            case = {"kind": kind, "rows": _log_int(rng, 1, 512), "lo": 1, "hi": _log_int(rng, 16, 16384),
                    "page": rng.choice([16, 16, 32, 64]), "above": rng.choice([0.0, 0.1, 0.5, 0.9])}
            case["lo"] = max(1, case["hi"] // rng.randint(1, 16))
            cells = case["rows"] * -(-case["hi"] // case["page"])
            case["pool"] = cells * rng.randint(2, 4) + 64
            if cells <= 130_000 and case["pool"] <= 400_000:
                return case


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_beam(case, seed):
    g = _gen(seed)
    r, w, v, rows = case["requests"], case["beams"], case["vocab"], case["requests"] * case["beams"]
    ends = [int(e) for e in torch.randperm(v, generator=torch.Generator().manual_seed(7))[:case["ends"]]]
    hold = torch.empty(rows, case["stride"], dtype=_TYPE[case["dtype"]], device="cuda")
    for at in range(0, rows, 128):
        hold[at:at + 128] = 2.5 * torch.randn(hold[at:at + 128].shape, generator=g, device="cuda")
    logits = hold[:, :v]
    # a text that may end here: the end tokens of some rows are likely
    for e in ends:
        logits[:, e] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.3, 11.0, -2.0).to(logits.dtype)
    if case["masked"]:  # constrained rows: a few tokens are allowed, fewer than there are beams in some
        tight = torch.rand(rows, generator=g, device="cuda") < case["masked"]
        allowed = torch.randint(0, v, (rows, 3), generator=g, device="cuda")
        keep = torch.zeros(rows, v, dtype=torch.bool, device="cuda").scatter_(1, allowed, True)
        logits.masked_fill_(tight[:, None] & ~keep, -math.inf)
    scores = -4 - 2 * torch.rand(r, w, generator=g, device="cuda")
    if case["first"]:
        scores[:, 1:] = -math.inf
        scores[:, 0] = 0.0
    shape = dict(device="cuda", dtype=torch.int64)
    out = [torch.zeros(r, w, **shape), torch.zeros(r, w, **shape).int(), torch.zeros(r, w, device="cuda"),
           torch.zeros(r, w, **shape), torch.zeros(r, w, **shape).int(), torch.zeros(r, w, device="cuda")]
    return {"logits": logits, "scores": scores, "ends": ends, "end_ids": torch.tensor(ends, **shape), "out": out, "kept": {}}


def _pack(parts):
    """The int32 tensors of a state as views of one buffer, and a copy of it: every pass starts from the same state."""
    flat = torch.cat([torch.tensor(p, dtype=torch.int32).flatten() if not torch.is_tensor(p) else p.int().flatten()
                      for p in parts.values()]).cuda()
    views, at = {}, 0
    for name, p in parts.items():
        shape = p.shape if torch.is_tensor(p) else torch.tensor(p).shape
        views[name] = flat[at:at + shape.numel()].view(shape)
        at += shape.numel()
    return dict(views, state=flat, saved=flat.clone())


def _lens(case, count):
    """Lengths are the case's own, so that pools and tables are as large for every seed; pages and parents are the seed's."""
    rng = random.Random(4000 + count)
    return [rng.randint(case["lo"], case["hi"]) for _ in range(count)]


def _prepare_reorder(case, seed):
    """Groups of beams in the middle of their search: one prompt's full pages shared by all beams, then for each beam
    pages of its own."""
    g = torch.Generator().manual_seed(seed)
    n, w, page = case["groups"], case["beams"], case["page"]
    lens = torch.tensor(_lens(case, n))
    width = -(-(case["hi"] + 256) // page)
    held = (lens + page - 1) // page
    shared = (lens - torch.tensor(case["suffix"])).clamp_min(0) // page
    col = torch.arange(width)
    own_cell = (col >= shared[:, None]) & (col < held[:, None])
    common = col < shared[:, None]
    cells = torch.cat([common[:, None], own_cell[:, None].expand(n, w, width)], 1)  # the shared row, then each beam's
    pages = torch.where(cells, cells.flatten().cumsum(0).view(cells.shape) - 1, -1)
    used = int(cells.sum())
    pool = used + n * w + 64
    perm = torch.randperm(pool, generator=g)
    table = torch.where(common[:, None], pages[:, :1], pages[:, 1:])
    shares = torch.zeros(pool, dtype=torch.int64)
    shares[perm[pages[:, 0][common]]] = w - 1
    table = torch.where(table >= 0, perm[table.clamp_min(0)], -1)
    parents = torch.randint(0, w, (n, w), generator=g)
    gone = torch.rand(n, generator=g) < case["released"]
    parents[gone] = -1
    free = torch.full((pool,), -1)
    free[:pool - used] = perm[used:]
    s = _pack({"table": table.view(n * w, width), "lens": lens[:, None].expand(n, w).reshape(-1), "shares": shares,
               "free": free, "count": [pool - used]})
    s["parents"] = parents.int().cuda()
    s["copies"] = [torch.zeros(n * w, dtype=torch.int32, device="cuda") for _ in range(3)]
    s["copies"].append(torch.zeros(2, dtype=torch.int32, device="cuda"))
    return dict(s, kept={})


def _prepare_copy(case, seed):
    g = _gen(seed)
    dtype, pairs, pool = _TYPE[case["dtype"]], case["pairs"], case["pool"]
    # one allocation for the caches of all layers, keys and values apart; each layer holds its own two views
    hold = torch.empty(2 * case["layers"], pool, case["page"], case["heads"], case["dim"], dtype=dtype, device="cuda")
    values = torch.randn(CACHE_VALUES, generator=g, device="cuda").to(dtype)
    flat = hold.view(-1)
    for at in range(0, flat.numel(), CACHE_VALUES):
        flat[at:at + CACHE_VALUES] = values[:flat.numel() - at]
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:2 * pairs].int().cuda()
    tokens = torch.full((pairs,), case["page"], dtype=torch.int32)
    if not case["whole"]:
        tokens = torch.randint(1, case["page"], (pairs,), generator=torch.Generator().manual_seed(case["pairs"]))
    return {"hold": hold, "caches": list(hold), "src": ids[:pairs].clone(), "dst": ids[pairs:].clone(),
            "tokens": tokens.int().cuda(), "count": torch.tensor([pairs, 0], dtype=torch.int32, device="cuda")}


def _prepare_compact(case, seed):
    g = torch.Generator().manual_seed(seed)
    rows, page, pool = case["rows"], case["page"], case["pool"]
    lens = torch.tensor(_lens(case, rows))
    width = -(-case["hi"] // page) + 1
    held = (lens + page - 1) // page
    cell = torch.arange(width) < held[:, None]
    used = int(cell.sum())
    limit = int(used * 1.05) + 16  # the pool shrinks to a little more than what is held
    # a share `above` of the held pages lies beyond the limit
    above = min(int(used * case["above"]), pool - limit)
    high = limit + torch.randperm(pool - limit, generator=g)
    low = torch.randperm(limit, generator=g)
    mine = torch.cat([high[:above], low[:used - above]])[torch.randperm(used, generator=g)]
    rest = torch.cat([high[above:], low[used - above:]])
    rest = rest[torch.randperm(rest.numel(), generator=g)]
    table = torch.full((rows, width), -1)
    table[cell] = mine
    shares = torch.zeros(pool, dtype=torch.int64)
    if rows > 1:  # the second row shares the first one's full pages
        common = int(min(lens[0], lens[1])) // page
        rest = torch.cat([rest, table[1, :common].clone()])
        table[1, :common] = table[0, :common]
        shares[table[0, :common]] = 1
    free = torch.full((pool,), -1)
    free[:rest.numel()] = rest
    s = _pack({"table": table, "lens": lens, "shares": shares, "free": free, "count": [rest.numel()]})
    s["limit"] = limit
    s["copies"] = [torch.zeros(used, dtype=torch.int32, device="cuda") for _ in range(3)]
    s["copies"].append(torch.zeros(2, dtype=torch.int32, device="cuda"))
    return dict(s, kept={})


_PREPARE = {"beam": _prepare_beam, "reorder": _prepare_reorder, "copy": _prepare_copy, "compact": _prepare_compact}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, seed), case=case)


# --------------------------------------------------------------------------- plain forms
def _places(chosen, slots):
    """The slot of each chosen entry along the last dimension, in order; `slots` for the others."""
    at = chosen.long().cumsum(-1) - 1
    return torch.where(chosen & (at < slots), at, slots)


def _plain_beam(s):
    logits, ends = s["logits"], s["end_ids"]
    r, w = s["scores"].shape
    v = logits.shape[1]
    x = logits.double()
    top = x.amax(dim=-1, keepdim=True)
    lse = top + (x - top).exp_().sum(dim=-1, keepdim=True).log()
    # the best of each beam, ties to the lowest token: unique whole numbers, the logit's order first
    bits = logits.float().view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 31) + (v - 1 - torch.arange(v, device=x.device))
    k = min(v, w + len(s["ends"]))
    token = (v - 1 - key.topk(k, dim=-1).values % (1 << 31)).view(r, w * k)
    beam = torch.arange(w, device=x.device).repeat_interleave(k).expand(r, w * k)
    score = s["scores"].double()[..., None] + (x.gather(1, token.view(r * w, k)) - lse).view(r, w, k)
    score = score.view(r, w * k)
    score = torch.where(score.float().isfinite(), score, -math.inf)
    score, order = score.sort(dim=-1, descending=True, stable=True)
    token, beam = token.gather(1, order), beam.gather(1, order)
    live = score > -math.inf
    is_end = (token[..., None] == ends).any(-1)
    rank = torch.arange(w * k, device=x.device)
    out = s["out"]
    for at, chosen in ((0, live & ~is_end), (3, live & is_end & (rank < w))):
        place = _places(chosen, w)
        for o, value, none in ((out[at], token, -1), (out[at + 1], beam, -1), (out[at + 2], score, -math.inf)):
            padded = torch.full((r, w + 1), none, dtype=value.dtype, device=x.device)
            o.copy_(padded.scatter_(1, place, value)[:, :w])


def _plain_reorder(s):
    s["state"].copy_(s["saved"])
    page, parents = s["case"]["page"], s["parents"].long()
    (n, w), width, pool, cells = parents.shape, s["table"].shape[1], s["shares"].shape[0], s["free"].shape[0]
    dev = parents.device
    table, lens = s["table"].long().view(n, w, width), s["lens"].long().view(n, w)
    alive = (parents >= 0) & (parents < w)
    p = torch.where(alive, parents, 0)
    new_lens = torch.where(alive, lens.gather(1, p), 0)
    held, new_held = ((x + page - 1) // page for x in (lens, new_lens))
    # the child that keeps the parent's last page: the one in its place, else the first
    i = torch.arange(w, device=dev)
    known = torch.where(alive, parents, -1)
    first = (known[:, :, None] == known[:, None, :]).long().argmax(dim=-1)
    keeper = torch.where(known.gather(1, p) == p, p, first)
    copied = alive & (new_lens % page != 0) & (keeper != i) & (new_lens // page < width)
    col = torch.arange(width, device=dev)
    fresh = copied[..., None] & (col == (new_lens // page)[..., None])
    new = table.gather(1, p[..., None].expand(n, w, width))
    follows = (col < new_held[..., None]) & ~fresh
    none = torch.tensor(pool, device=dev)
    gained = torch.where(follows & (new >= 0) & (new < pool), new, none).flatten()
    lost = torch.where((col < held[..., None]) & (table >= 0) & (table < pool), table, none).flatten()
    one = torch.ones_like(gained)
    change = torch.zeros(pool + 1, dtype=torch.long, device=dev).scatter_add_(0, gained, one).scatter_add_(0, lost, -one)[:pool]
    shares = s["shares"].long() + change
    freed = (change != 0) & (shares == -1)
    s["shares"].copy_(torch.where(freed, 0, shares))
    # the pages that nobody holds go on top of the stack, then the copies take theirs from it
    count = s["count"].long().clamp(0, cells)
    place = torch.where(freed, count + freed.long().cumsum(0) - 1, cells).clamp_max(cells)
    stack = torch.cat([s["free"].long(), none[None]]).scatter(0, place, torch.arange(pool, device=dev))
    have = (count + freed.sum()).clamp_max(cells)
    k = copied.flatten().long().cumsum(0) - 1
    got = stack[(have - 1 - k).clamp(0, cells - 1)]
    served = copied.flatten() & (k < have) & (got >= 0) & (got < pool)
    got = torch.where(served, got, -1)
    source = new.gather(2, (new_lens // page).clamp_max(width - 1)[..., None]).flatten()
    s["table"].copy_(torch.where(fresh, got.view(n, w, 1), torch.where(follows, new, table)).view(n * w, width))
    s["lens"].copy_(new_lens.flatten())
    s["free"].copy_(stack[:cells])
    s["count"].copy_(have - copied.sum().clamp_max(have))
    at = _places(served, n * w)
    for o, value, fill in zip(s["copies"], (source, got, (new_lens % page).flatten()), (-1, -1, 0)):
        o.copy_(torch.full((n * w + 1,), fill, device=dev).scatter(0, at, value)[:-1])
    s["copies"][3].copy_(torch.stack([served.sum(), copied.sum() - served.sum()]))


def _plain_copy(s):
    hold = s["hold"] if s["hold"].element_size() > 1 else s["hold"].view(torch.uint8)  # (fp8 has no indexing)
    src, dst = s["src"].long(), s["dst"].long()
    used = torch.arange(hold.shape[2], device=src.device) < s["tokens"][:, None]
    hold[:, dst] = torch.where(used[:, :, None, None], hold[:, src], hold[:, dst])


def _plain_compact(s):
    s["state"].copy_(s["saved"])
    page, limit = s["case"]["page"], s["limit"]
    (rows, width), pool, cells = s["table"].shape, s["shares"].shape[0], s["free"].shape[0]
    dev = s["table"].device
    table, ids = s["table"].long(), torch.arange(pool, device=dev)
    held = torch.arange(width, device=dev) < ((s["lens"].long() + page - 1) // page)[:, None]
    known = held & (table >= 0) & (table < pool)
    mark = torch.zeros(pool + 1, dtype=torch.bool, device=dev).scatter_(0, torch.where(known, table, pool).flatten(), True)[:pool]
    stack = s["free"].long()
    listed_free = (torch.arange(cells, device=dev) < s["count"]) & (stack >= 0) & (stack < limit)
    free = torch.zeros(pool + 1, dtype=torch.bool, device=dev).scatter_(0, torch.where(listed_free, stack, pool), True)[:pool]
    high = mark & (ids >= limit)
    room = s["copies"][0].shape[0]
    moves = torch.minimum(high.sum(), free.sum()).clamp_max(room)
    src_at, dst_at = high.long().cumsum(0) - 1, free.long().cumsum(0) - 1
    moved, taken = high & (src_at < moves), free & (dst_at < moves)
    empty = torch.full((pool + 1,), -1, device=dev)
    src = empty.scatter(0, torch.where(moved, src_at, pool), ids)
    dst = empty.scatter(0, torch.where(taken, dst_at, pool), ids)
    to = torch.where(moved, dst[src_at.clamp_min(0)], ids)
    s["table"].copy_(torch.where(known, to[table.clamp(0, pool - 1)], table))
    shares = s["shares"].long()
    s["shares"].copy_(torch.cat([torch.where(moved, 0, shares), shares[:1]]).scatter(0, torch.where(moved, to, pool), shares)[:pool])
    # what is still free below the limit, the lowest on top
    left = free.sum() - moves
    place = torch.where(free & ~taken, free.sum() - 1 - dst_at, cells)
    s["free"].copy_(torch.cat([stack, stack[:1]]).scatter(0, place, ids)[:cells])
    s["count"].copy_(left)
    s["copies"][0].copy_(src[:room])
    s["copies"][1].copy_(dst[:room])
    s["copies"][2].copy_(torch.where(torch.arange(room, device=dev) < moves, page, 0))
    s["copies"][3].copy_(torch.stack([moves, high.sum() - moves]))


_PLAIN = {"beam": _plain_beam, "reorder": _plain_reorder, "copy": _plain_copy, "compact": _plain_compact}


# --------------------------------------------------------------------------- the framework's calls
def _own_beam(s):
    from l20_beam_search import BeamSearchStep, allocate_l20_beam_search_workspace, l20_beam_search_step

    kept = s["kept"]
    if not kept:
        kept["out"] = BeamSearchStep(*s["out"])
        kept["workspace"] = allocate_l20_beam_search_workspace(s["logits"], s["scores"], end_tokens=s["ends"])
    l20_beam_search_step(s["logits"], s["scores"], end_tokens=s["ends"], out=kept["out"], workspace=kept["workspace"])


def _own_reorder(s):
    from l20_block_tables import PageCopies, allocate_l20_reorder_workspace, l20_reorder_block_tables

    kept = s["kept"]
    if not kept:
        kept["copies"] = PageCopies(*s["copies"])
        kept["workspace"] = allocate_l20_reorder_workspace(s["parents"], s["table"])
    s["state"].copy_(s["saved"])
    l20_reorder_block_tables(s["parents"], s["table"], s["lens"], s["shares"], s["free"], s["count"], s["case"]["page"],
                             copies=kept["copies"], workspace=kept["workspace"])


def _own_copy(s):
    from l20_block_tables import PageCopies, l20_copy_pages

    l20_copy_pages(PageCopies(s["src"], s["dst"], s["tokens"], s["count"]), s["caches"])


def _own_compact(s):
    from l20_block_tables import PageCopies, allocate_l20_compact_workspace, l20_compact_pages

    kept = s["kept"]
    if not kept:
        kept["copies"] = PageCopies(*s["copies"])
        kept["workspace"] = allocate_l20_compact_workspace(s["shares"])
    s["state"].copy_(s["saved"])
    l20_compact_pages(s["limit"], s["table"], s["lens"], s["shares"], s["free"], s["count"], s["case"]["page"],
                      copies=kept["copies"], workspace=kept["workspace"])


_OWN = {"beam": _own_beam, "reorder": _own_reorder, "copy": _own_copy, "compact": _own_compact}


def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "beam":
        return s["out"]
    if kind == "copy":  # bytes are moved as they are; those of fp8 caches are compared as whole numbers
        return [s["hold"] if s["hold"].element_size() > 1 else s["hold"].view(torch.uint8)]
    return [s[k] for k in ("table", "lens", "shares", "free", "count")] + s["copies"]


def run(state):
    (_OWN if own else _PLAIN)[state["case"]["kind"]](state)
    return _outputs(state)


# --------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "beam":
        rows = case["requests"] * (1 if case["first"] else case["beams"])
        return {"bytes": rows * case["vocab"] * _SIZE[case["dtype"]] + 36 * case["requests"] * case["beams"],
                "flops": 4 * rows * case["vocab"]}
    if kind == "reorder":
        cells = sum(-(-n // case["page"]) for n in _lens(case, case["groups"])) * case["beams"]
        rows = case["groups"] * case["beams"]
        return {"bytes": 4 * cells + 28 * rows, "flops": 2 * cells}
    if kind == "copy":
        tokens = case["pairs"] * (case["page"] if case["whole"] else case["page"] // 2)
        moved = tokens * case["heads"] * case["dim"] * _SIZE[case["dtype"]] * 2 * case["layers"]
        return {"bytes": 2 * moved + 12 * case["pairs"], "flops": 0}
    cells = sum(-(-n // case["page"]) for n in _lens(case, case["rows"]))
    moves = int(cells * case["above"])
    return {"bytes": 4 * cells + 4 * (case["pool"] - cells) + moves * 32, "flops": 2 * cells}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The scores, from whole sorted rows of log-probabilities, and the values of copied pages; everything else is
    whole numbers."""
    if case["kind"] == "copy" and case["dtype"] != "e4m3":
        s = _prepare_copy(case, seed)
        values = s["hold"].double()
        for src, dst, tokens in zip(s["src"].tolist(), s["dst"].tolist(), s["tokens"].tolist()):
            values[:, dst, :tokens] = values[:, src, :tokens]
        return [values]
    if case["kind"] != "beam":
        return None
    s = _prepare_beam(case, seed)
    r, w = s["scores"].shape
    v = case["vocab"]
    running = torch.full((r, w), -math.inf, dtype=torch.float64, device="cuda")
    ended = torch.full((r, w), -math.inf, dtype=torch.float64, device="cuda")
    is_end = torch.zeros(v, dtype=torch.bool, device="cuda")
    is_end[s["end_ids"]] = True
    for q in range(r):
        x = s["logits"][q * w:(q + 1) * w].double()
        total = torch.log_softmax(x, dim=-1) + s["scores"][q].double()[:, None]
        total = torch.where(total.isnan(), -math.inf, total)
        best = total.masked_fill(is_end, -math.inf).flatten().sort(descending=True).values[:w]
        running[q, :best.numel()] = best
        value, at = total.flatten().sort(descending=True, stable=True)
        hit = value[:w][is_end[at[:w] % v] & (value[:w] > -math.inf)]
        ended[q, :hit.numel()] = hit
    return [None, None, running, None, None, ended]
