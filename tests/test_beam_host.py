"""Beam search's selection and the page pool's operators on CPU: mirrors of the argument blocks, every refusal of the C
ABI's checks, workspace sizes, the references' own pins, and the Python functions without a GPU.  No kernel is
launched here."""

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

import beam_ref as R
import l20_pd_cabi as cabi

INCLUDE = Path(__file__).resolve().parents[1] / "include"
FAKE = 0x10000  # never dereferenced
STRUCTS = {
    "l20_pd_reorder_args": ("l20_block_tables.h", cabi.L20PdReorderArgs),
    "l20_pd_compact_args": ("l20_block_tables.h", cabi.L20PdCompactArgs),
    "l20_pd_copy_args": ("l20_block_tables.h", cabi.L20PdCopyArgs),
    "l20_pd_beam_step_args": ("l20_beam_search.h", cabi.L20PdBeamStepArgs),
}


@pytest.mark.parametrize("name", STRUCTS)
def test_mirrors_have_the_headers_fields_in_order(name):
    header, mirror = STRUCTS[name]
    text = re.sub(r"/\*.*?\*/", "", (INCLUDE / header).read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    want = []
    for line in body.split(";"):
        m = re.match(r"\s*(const )?(void|float|int32_t|int64_t)\b(.*)", line.strip(), re.S)
        if not m:
            continue
        for item in m.group(3).split(","):
            kind = ctypes.c_void_p if "*" in item else {"float": ctypes.c_float, "int32_t": ctypes.c_int32,
                                                        "int64_t": ctypes.c_int64}[m.group(2)]
            want.append((item.replace("*", "").replace("const", "").strip(), kind))
    assert list(mirror._fields_) == want


KEEP = []  # host arrays behind the arguments


def beam_args():
    a = cabi.L20PdBeamStepArgs()
    for i, name in enumerate(("logits", "scores", "tokens", "parents", "scores_out", "ended_tokens", "ended_parents",
                              "ended_scores", "workspace")):
        setattr(a, name, FAKE << (2 * i))
    a.l_stride_request, a.l_stride_beam, a.dtype = 4 * 1000, 1000, cabi.L20_PD_BF16
    a.s_stride_request, a.s_stride_beam = 4, 1
    a.requests, a.beams, a.vocab, a.num_end_tokens = 6, 4, 1000, 2
    ends = (ctypes.c_int32 * 2)(3, 9)
    KEEP.append(ends)
    a.end_tokens = ctypes.cast(ends, ctypes.c_void_p)
    a.workspace_bytes = 1 << 20
    return a


def pool_args(kind):
    a = kind()
    for i, name in enumerate(("block_table", "seq_lens", "page_shares", "free_pages", "free_count", "src", "dst", "tokens",
                              "count", "workspace")):
        setattr(a, name, FAKE * (i + 1))
    a.bt_stride_row, a.table_pages, a.pages, a.pool, a.room, a.page_size = 30, 30, 500, 500, 40, 16
    a.workspace_bytes = 1 << 20
    return a


def reorder_args():
    a = pool_args(cabi.L20PdReorderArgs)
    a.parents, a.groups, a.beams = FAKE * 20, 5, 4
    return a


def compact_args():
    a = pool_args(cabi.L20PdCompactArgs)
    a.limit, a.rows = 300, 20
    return a


def copy_args():
    a = cabi.L20PdCopyArgs()
    a.src, a.dst, a.tokens, a.count, a.room = FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 7
    caches = (ctypes.c_void_p * 3)(FAKE * 5, FAKE * 6, FAKE * 7)
    KEEP.append(caches)
    a.caches, a.num_caches = ctypes.cast(caches, ctypes.c_void_p), 3
    a.pages, a.stride_page = 50, 16 * 1024
    a.size0, a.stride0, a.size1, a.size2, a.inner, a.token_level = 16, 1024, 1, 1, 1024, 0
    return a


CHECKS = {"beam_step": beam_args, "reorder_tables": reorder_args, "compact_pages": compact_args, "copy_pages": copy_args}


def check(kind, args):
    rc = getattr(cabi.load(), f"l20_pd_{kind}_check")(ctypes.byref(args))
    return rc, cabi.last_error()


@pytest.mark.parametrize("kind", CHECKS)
def test_well_formed_arguments_pass(kind):
    assert check(kind, CHECKS[kind]()) == (0, "")
    assert getattr(cabi.load(), f"l20_pd_{kind}_check")(None) != 0 and "null argument block" in cabi.last_error()


BAD = [
    ("beam_step", dict(dtype=7), "bf16, fp16 or fp32"),
    ("beam_step", dict(beams=0), "1 to 32 beams"),
    ("beam_step", dict(beams=33), "1 to 32 beams"),
    ("beam_step", dict(num_end_tokens=9), "at most 8 end tokens"),
    ("beam_step", dict(num_end_tokens=-1), "at most 8 end tokens"),
    ("beam_step", dict(vocab=0), "must be positive"),
    ("beam_step", dict(requests=-1), "must be positive"),
    ("beam_step", dict(vocab=(1 << 30) + 1), "vocabulary too large"),
    ("beam_step", dict(requests=(1 << 18) + 1), "2^20 beams"),
    ("beam_step", dict(end_tokens=0), "null tensor pointer"),
    ("beam_step", dict(logits=0), "null tensor pointer"),
    ("beam_step", dict(ended_scores=0), "null tensor pointer"),
    ("beam_step", dict(logits=FAKE + 1), "aligned to their type"),
    ("beam_step", dict(logits=FAKE + 2, dtype=cabi.L20_PD_FP32), "aligned to their type"),
    ("reorder_tables", dict(beams=0), "1 to 32 beams"),
    ("reorder_tables", dict(beams=33), "1 to 32 beams"),
    ("reorder_tables", dict(groups=2049), "8192 rows"),
    ("reorder_tables", dict(groups=-1), "8192 rows"),
    ("reorder_tables", dict(page_size=24), "page size"),
    ("reorder_tables", dict(page_size=8192), "page size"),
    ("reorder_tables", dict(table_pages=0), "must not be empty"),
    ("reorder_tables", dict(pages=0), "must not be empty"),
    ("reorder_tables", dict(pool=0), "must not be empty"),
    ("reorder_tables", dict(pages=(1 << 30) + 1), "too large"),
    ("reorder_tables", dict(table_pages=1 << 26, bt_stride_row=1 << 26), "too large"),
    ("reorder_tables", dict(room=19), "a pair a row"),
    ("reorder_tables", dict(parents=0), "null tensor pointer"),
    ("reorder_tables", dict(count=0), "null tensor pointer"),
    ("reorder_tables", dict(bt_stride_row=29), "rows overlap"),
    ("compact_pages", dict(rows=8193), "8192 rows"),
    ("compact_pages", dict(page_size=0), "page size"),
    ("compact_pages", dict(table_pages=0), "must not be empty"),
    ("compact_pages", dict(limit=-1), "limit must be"),
    ("compact_pages", dict(pages=(1 << 30) + 1), "too large"),
    ("compact_pages", dict(limit=501), "limit must be"),
    ("compact_pages", dict(room=-1), "room must not"),
    ("compact_pages", dict(src=0), "null tensor pointer"),
    ("compact_pages", dict(page_shares=0), "null tensor pointer"),
    ("compact_pages", dict(bt_stride_row=0), "rows overlap"),
    ("compact_pages", dict(pool=(1 << 30) + 1), "too large"),
    ("copy_pages", dict(room=-1), "must not be negative"),
    ("copy_pages", dict(num_caches=-1), "must not be negative"),
    ("copy_pages", dict(pages=0), "must not be empty"),
    ("copy_pages", dict(size1=0), "must not be empty"),
    ("copy_pages", dict(inner=0), "must not be empty"),
    ("copy_pages", dict(token_level=3), "token level"),
    ("copy_pages", dict(token_level=-2), "token level"),
    ("copy_pages", dict(stride0=1000), "parts overlap"),
    ("copy_pages", dict(stride0=0), "parts overlap"),
    ("copy_pages", dict(size1=4, stride1=1024), "parts overlap"),
    ("copy_pages", dict(stride_page=0), "pages overlap"),
    ("copy_pages", dict(stride_page=16 * 1024 - 1024), "pages overlap"),
    ("copy_pages", dict(size0=4, stride0=16 * 1024, size1=16, stride1=1024, token_level=1, stride_page=32 * 1024), "pages overlap"),
    ("copy_pages", dict(size0=1 << 22), "page too large"),
    ("copy_pages", dict(inner=1 << 41), "page too large"),
    ("copy_pages", dict(dst=0), "null tensor pointer"),
    ("copy_pages", dict(caches=0), "null tensor pointer"),
]


@pytest.mark.parametrize("case", BAD, ids=[f"{k}-{'_'.join(c)}-{i}" for i, (k, c, _) in enumerate(BAD)])
def test_refusals(case):
    kind, change, message = case
    args = CHECKS[kind]()
    for name, value in change.items():
        setattr(args, name, value)
    rc, error = check(kind, args)
    assert rc != 0 and message in error, error


@pytest.mark.parametrize("change,message", [
    (dict(size0=1, token_level=-1, inner=1 << 34, size2=1 << 30, stride2=1 << 34, pages=1), "page too large"),  # 2^64 bytes: 0
    (dict(size0=1, token_level=-1, inner=1 << 33, size1=4, stride1=1 << 63 - 2, size2=1 << 29, stride2=1 << 33, pages=1), "page too large"),
    (dict(size0=1 << 30, stride0=1 << 38, inner=1, token_level=-1, pages=1), "page too large"),
    (dict(size0=2, stride0=1 << 41, inner=1, token_level=-1, pages=1), "page too large"),
    (dict(pages=1 << 30, stride_page=1 << 36), "cache too large"),
    (dict(pages=1 << 31, stride_page=1 << 14), "cache too large"),
    (dict(pages=2, stride_page=(1 << 63) - 1), "cache too large"),
], ids=str)
def test_sizes_whose_products_pass_64_bits_are_refused(change, message):
    args = copy_args()
    for name, value in change.items():
        setattr(args, name, value)
    rc, error = check("copy_pages", args)
    assert rc != 0 and message in error, error


def test_the_largest_caches_pass():
    """A page of 2^31 - 16 bytes, and pages that reach a terabyte."""
    args = copy_args()
    args.size0, args.inner, args.token_level, args.pages = 1, (1 << 31) - 16, -1, 512
    args.stride_page = 1 << 31
    assert check("copy_pages", args) == (0, "")


def test_pages_may_lie_inside_other_levels():
    """Heads outside pages: a page is in pieces, and no two share bytes."""
    args = copy_args()
    args.size0, args.stride0, args.size1, args.stride1, args.token_level = 4, 50 * 16 * 1024, 16, 1024, 1
    assert check("copy_pages", args) == (0, "")


def test_nothing_to_do_needs_no_pointers():
    for kind, empty in (("beam_step", dict(requests=0, logits=0, scores=0, tokens=0)),
                        ("reorder_tables", dict(groups=0, parents=0, block_table=0, seq_lens=0, src=0, table_pages=0)),
                        ("compact_pages", dict(rows=0, block_table=0, seq_lens=0, table_pages=0)),
                        ("compact_pages", dict(room=0, src=0, dst=0, tokens=0)),
                        ("copy_pages", dict(room=0, src=0)), ("copy_pages", dict(num_caches=0, caches=0))):
        args = CHECKS[kind]()
        for name, value in empty.items():
            setattr(args, name, value)
        assert check(kind, args) == (0, ""), kind


@pytest.mark.parametrize("kind", ["beam_step", "reorder_tables", "compact_pages"])
@pytest.mark.parametrize("change", [dict(workspace=0), dict(workspace_bytes=64), dict(workspace=FAKE * 64 + 2)], ids=["none", "small", "odd"])
def test_calls_refuse_bad_workspaces(kind, change):
    args = CHECKS[kind]()
    for name, value in change.items():
        setattr(args, name, value)
    rc = getattr(cabi.load(), f"l20_pd_{kind}")(ctypes.byref(args), None)
    assert rc == cabi.L20_PD_EINVAL and "workspace is missing, misaligned or too small" in cabi.last_error()


@pytest.mark.parametrize("change", [
    dict(tokens=FAKE + 8),  # over the logits
    dict(ended_scores=FAKE + 2 * (23 * 1000 + 999)),  # the last logit
    dict(parents=FAKE << 2),  # over the scores
    dict(scores_out=(FAKE << 2) + 4),  # over the scores, but not they themselves
    dict(scores_out=FAKE << 2, s_stride_request=8),  # in another layout
    dict(ended_tokens=FAKE << 4),  # over the tokens
    dict(workspace=(FAKE << 8) + 64),
], ids=range(7))
def test_beam_step_refuses_outputs_over_others(change):
    args = beam_args()
    for name, value in change.items():
        setattr(args, name, value)
    rc = cabi.load().l20_pd_beam_step(ctypes.byref(args), None)
    assert rc == cabi.L20_PD_EINVAL and ("must not lie over" in cabi.last_error() or "must lie apart" in cabi.last_error())


@pytest.mark.parametrize("kind", ["reorder_tables", "compact_pages"])
@pytest.mark.parametrize("change", [
    dict(seq_lens=FAKE + 4 * (30 * 19 + 29)),  # the table's last cell
    dict(page_shares=FAKE * 4 - 4),  # ends in the stack
    dict(dst=FAKE * 6),
    dict(count=FAKE * 5 - 4),
    dict(workspace=FAKE * 8 + 156),
    dict(free_count=FAKE * 2 + 76),
], ids=range(6))
def test_page_calls_refuse_tensors_over_others(kind, change):
    args = CHECKS[kind]()
    for name, value in change.items():
        setattr(args, name, value)
    rc = getattr(cabi.load(), f"l20_pd_{kind}")(ctypes.byref(args), None)
    assert rc == cabi.L20_PD_EINVAL and "must lie apart" in cabi.last_error()


def test_workspaces_are_enough_for_smaller_calls():
    lib, a = cabi.load(), beam_args()
    for beams, vocab, ends in ((1, 1, 0), (4, 152064, 1), (32, 50257, 8), (5, 2049, 2), (32, 200, 8)):
        a.beams, a.vocab, a.num_end_tokens = beams, vocab, ends
        sizes = []
        for a.requests in [*range(1, 300), 1000, 4096, 30000]:
            sizes.append(lib.l20_pd_beam_step_workspace(ctypes.byref(a)))
        assert sizes == sorted(sizes) and sizes[0] > 0
    for name, values in (("vocab", [*range(1, 40), *range(40, 300000, 777)]), ("beams", range(1, 33)), ("num_end_tokens", range(9))):
        a = beam_args()
        sizes = []
        for value in values:
            setattr(a, name, value)
            sizes.append(lib.l20_pd_beam_step_workspace(ctypes.byref(a)))
        assert sizes == sorted(sizes), name
    r = reorder_args()
    sizes = []
    for r.groups in range(1, 50):
        r.table_pages = 10 * r.groups
        sizes.append(lib.l20_pd_reorder_tables_workspace(ctypes.byref(r)))
    assert sizes == sorted(sizes)
    c = compact_args()
    assert lib.l20_pd_compact_pages_workspace(ctypes.byref(c)) == 12 * 16  # two bits and an int a 32 pages
    for name in ("beam_step", "reorder_tables", "compact_pages"):
        assert getattr(lib, f"l20_pd_{name}_workspace")(None) == 0


def test_functions_refuse_cpu_tensors():
    import l20_beam_search as bs
    import l20_block_tables as bt

    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="l20_beam_search_step requires an MI355X"):
        bs.l20_beam_search_step(torch.zeros(4, 10), torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="l20_reorder_block_tables requires an MI355X"):
        bt.l20_reorder_block_tables(i.view(2, 2), i.view(4, 1), i, i, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="l20_compact_pages requires an MI355X"):
        bt.l20_compact_pages(2, i.view(4, 1), i, i, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="l20_copy_pages requires an MI355X"):
        bt.l20_copy_pages(bt.PageCopies(i, i), [torch.zeros(4, 16, 8)])


def test_fake_implementations_return_nothing():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import l20_beam_search as bs
    import l20_block_tables as bt

    with FakeTensorMode():
        out = bs.BeamSearchStep.empty(2, 3, "cuda")
        x = torch.empty(6, 100, device="cuda")
        ws = torch.empty(100, dtype=torch.uint8, device="cuda")
        assert torch.ops.l20_stack.beam_search_step(x, out.scores, [1], *out, ws) is None
        i = torch.empty(6, dtype=torch.int32, device="cuda")
        copies = bt.PageCopies.empty(6, "cuda")
        assert torch.ops.l20_stack.reorder_block_tables(i.view(2, 3), i.view(6, 1), i, i, i, i[:1], 16, *copies, i) is None
        assert torch.ops.l20_stack.compact_pages(2, i.view(6, 1), i, i, i, i[:1], 16, *copies, i) is None
        assert torch.ops.l20_stack.copy_pages(*copies, [torch.empty(6, 16, 8, device="cuda")]) is None


# --------------------------------------------------------------------------- the references themselves
def test_beam_reference_on_known_answers():
    """Probabilities 1/2, 1/4, 1/8, 1/8 of one beam, 1/4 each of the other: the products in order."""
    x = torch.tensor([[[0.5, 0.25, 0.125, 0.125], [0.25] * 4]], dtype=torch.float64).log()
    c = torch.tensor([[math.log(0.5), math.log(0.75)]])
    tokens, parents, scores, *_ = R.beam_step(x, c, [])
    assert tokens == [[0, 0]] and parents == [[0, 1]]  # 1/4, then 3/16 with the lowest token
    assert scores[0] == pytest.approx([math.log(0.25), math.log(3 / 16)], rel=1e-6)
    tokens, parents, _, ended, ended_parents, _, _ = R.beam_step(x, c, [0])
    assert (tokens, parents) == ([[1, 2]], [[1, 1]]) and (ended, ended_parents) == ([[0, 0]], [[0, 1]])


def test_reorder_reference_on_a_fork_and_its_end():
    table, lens, shares, free = [[0, 1, -1], [-1, -1, -1]], [20, 0], [0] * 6, [5, 4, 3, 2, -1, -1]
    t, n, s, f, count, pairs, short = R.reorder([[0, 0]], table, lens, shares, free, 4, 16)
    assert t == [[0, 1, -1], [0, 2, -1]] and n == [20, 20] and s == [1, 0, 0, 0, 0, 0]
    assert pairs == [(1, 2, 4)] and count == 3 and short == 0
    t, n, s, f, count, pairs, short = R.reorder([[1, -1]], t, n, s, f, count, 16)
    assert t[0] == [0, 2, -1] and n == [20, 0] and s == [0] * 6 and pairs == [] and f[:count] == [5, 4, 3, 1]
    _, n, s, f, count, _, _ = R.reorder([[-1, -1]], t, n, s, f, count, 16)
    assert n == [0, 0] and sorted(f[:count]) == list(range(6)) and s == [0] * 6
