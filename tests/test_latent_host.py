"""Latent attention and the block-table builder on CPU: mirrors of the argument blocks, every refusal of the C ABI's
checks, workspace sizes, and the Python functions without a GPU.  No kernel is launched here."""

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

import l20_pd_cabi as cabi

INCLUDE = Path(__file__).resolve().parents[1] / "include"
FAKE = 0x10000  # never dereferenced
STRUCTS = {
    "l20_pd_latent_write_args": ("l20_latent_attention.h", cabi.L20PdLatentWriteArgs),
    "l20_pd_latent_args": ("l20_latent_attention.h", cabi.L20PdLatentArgs),
    "l20_pd_latent_prompt_args": ("l20_latent_attention.h", cabi.L20PdLatentPromptArgs),
    "l20_pd_block_tables_args": ("l20_block_tables.h", cabi.L20PdBlockTablesArgs),
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
            want.append((item.replace("*", "").strip(), kind))
    assert list(mirror._fields_) == want


def write_args():
    a = cabi.L20PdLatentWriteArgs()
    a.query = a.query_out = a.latent = a.latent_out = a.key = a.key_out = a.norm_weight = FAKE
    a.q_stride_token, a.q_stride_head, a.qo_stride_token, a.qo_stride_head = 16 * 192, 192, 16 * 576, 576
    a.l_stride_token, a.lo_stride_token, a.k_stride_token, a.ko_stride_token = 576, 512, 576, 64
    a.num_heads, a.dtype = 16, cabi.L20_PD_BF16
    a.positions = a.cos_sin_cache = a.slot_mapping = a.cache = FAKE
    a.cs_stride_position, a.max_position, a.cs_dtype = 64, 1000, cabi.L20_PD_FP32
    a.norm_eps, a.cache_scale = 1e-6, 0.5
    a.c_stride_page, a.c_stride_token, a.num_pages, a.page_size = 16 * 576, 576, 100, 16
    a.cache_dtype = cabi.L20_PD_KV_FP8_E4M3
    a.num_tokens, a.rank, a.rope_dim = 50, 512, 64
    return a


def paged_args():
    a = cabi.L20PdLatentArgs()
    a.query = a.cache = a.block_table = a.seq_lens = a.workspace = FAKE
    a.output = 2 * FAKE
    a.q_stride_row, a.q_stride_head, a.dtype = 16 * 576, 576, cabi.L20_PD_BF16
    a.c_stride_page, a.c_stride_token, a.num_pages, a.page_size = 64 * 576, 576, 100, 64
    a.cache_dtype, a.cache_scale = cabi.L20_PD_KV_FP8_E4M3, 0.5
    a.bt_stride_row, a.table_pages = 40, 40
    a.o_stride_row, a.o_stride_head = 16 * 512, 512
    a.workspace_bytes, a.softmax_scale = 1 << 40, 0.07
    a.batch, a.q_len, a.num_heads, a.rank, a.rope_dim, a.max_seq_len = 8, 2, 16, 512, 64, 2560
    return a


def prompt_args():
    a = cabi.L20PdLatentPromptArgs()
    a.query = a.key = a.key_rope = a.value = a.cu_q = a.cu_k = FAKE
    a.output = 2 * FAKE
    a.q_stride_token, a.q_stride_head = 8 * 192, 192
    a.k_stride_token = a.v_stride_token = 8 * 256
    a.k_stride_head = a.v_stride_head = 256
    a.kr_stride_token, a.dtype = 64, cabi.L20_PD_BF16
    a.o_stride_token, a.o_stride_head = 8 * 128, 128
    a.softmax_scale, a.causal, a.total_q, a.total_k = 0.07, 1, 300, 500
    a.batch, a.num_heads, a.max_q_len, a.head_dim, a.rope_dim, a.value_dim = 3, 8, 200, 128, 64, 128
    return a


def table_args():
    a = cabi.L20PdBlockTablesArgs()
    for i, name in enumerate(("cached_lens", "new_lens", "block_table", "free_pages", "free_count", "free_count_out",
                              "slots", "positions", "cu_lens", "seq_lens")):
        setattr(a, name, FAKE * (i + 1))
    a.bt_stride_row, a.table_pages, a.pool, a.num_slots, a.batch, a.page_size = 30, 30, 500, 700, 20, 16
    return a


CHECKS = {"latent_write": write_args, "paged_latent": paged_args, "latent_prompt": prompt_args, "block_tables": table_args}


def check(kind, args):
    lib = cabi.load()
    rc = getattr(lib, f"l20_pd_{kind}_check")(ctypes.byref(args))
    return rc, cabi.last_error()


@pytest.mark.parametrize("kind", CHECKS)
def test_well_formed_arguments_pass(kind):
    assert check(kind, CHECKS[kind]()) == (0, "")
    lib = cabi.load()
    assert getattr(lib, f"l20_pd_{kind}_check")(None) != 0 and "null argument block" in cabi.last_error()


BAD = [
    ("latent_write", dict(dtype=cabi.L20_PD_FP32), "bf16 or fp16"),
    ("latent_write", dict(cs_dtype=9), "cos_sin_cache must be"),
    ("latent_write", dict(cache_dtype=cabi.L20_PD_KV_FP16), "model dtype"),
    ("latent_write", dict(cache_dtype=cabi.L20_PD_KV_FP8_E5M2), "model dtype"),
    ("latent_write", dict(rank=384), "rank 256 or 512"),
    ("latent_write", dict(rope_dim=32), "64 rotary dims"),
    ("latent_write", dict(num_tokens=-1), "must be positive"),
    ("latent_write", dict(num_heads=0), "must be positive"),
    ("latent_write", dict(page_size=24), "page size"),
    ("latent_write", dict(page_size=8192), "page size"),
    ("latent_write", dict(num_pages=0), "no pages"),
    ("latent_write", dict(cache_scale=0.0), "cache scale"),
    ("latent_write", dict(cache_scale=math.inf), "cache scale"),
    ("latent_write", dict(norm_eps=-1.0), "epsilon"),
    ("latent_write", dict(norm_eps=math.nan), "epsilon"),
    ("latent_write", dict(max_position=0), "no rows"),
    ("latent_write", dict(query_out=0), "null tensor pointer"),
    ("latent_write", dict(slot_mapping=0), "null tensor pointer"),
    ("latent_write", dict(num_tokens=1 << 30), "too many query rows"),
    ("latent_write", dict(num_tokens=40_000_000), "too many query rows"),  # 2^32 threads
    ("latent_write", dict(latent=FAKE + 2), "16-byte aligned"),
    ("latent_write", dict(l_stride_token=577), "16-byte aligned"),
    ("latent_write", dict(q_stride_head=190), "16-byte aligned"),
    ("latent_write", dict(c_stride_token=570), "latent cache rows"),
    ("paged_latent", dict(dtype=cabi.L20_PD_FP32), "bf16 or fp16"),
    ("paged_latent", dict(cache_dtype=cabi.L20_PD_KV_FP16), "query's dtype"),
    ("paged_latent", dict(rank=128), "rank 256 or 512"),
    ("paged_latent", dict(rope_dim=128), "64 rotary dims"),
    ("paged_latent", dict(page_size=40), "page size"),
    ("paged_latent", dict(batch=-1), "must be positive"),
    ("paged_latent", dict(q_len=0), "must be positive"),
    ("paged_latent", dict(max_seq_len=-5), "must be positive"),
    ("paged_latent", dict(num_heads=40000), "65535 query rows"),
    ("paged_latent", dict(batch=70000), "65535 sequences"),
    ("paged_latent", dict(softmax_scale=0.0), "softmax_scale"),
    ("paged_latent", dict(softmax_scale=math.nan), "softmax_scale"),
    ("paged_latent", dict(cache_scale=-1.0), "cache scale"),
    ("paged_latent", dict(num_pages=0), "must have pages"),
    ("paged_latent", dict(table_pages=0), "must have pages"),
    ("paged_latent", dict(table_pages=1 << 25), "too many tokens"),
    ("paged_latent", dict(batch=65535, table_pages=16385), "too many tokens"),  # the sum of the costs: 31 bits
    ("paged_latent", dict(num_pages=1 << 31), "too many pages"),
    ("paged_latent", dict(c_stride_page=65 * 576), "contiguous"),
    ("paged_latent", dict(seq_lens=0), "null tensor pointer"),
    ("paged_latent", dict(c_stride_token=1 << 26, c_stride_page=1 << 32), "stride out of range"),
    ("paged_latent", dict(query=FAKE + 8), "query rows must be 16-byte"),
    ("paged_latent", dict(cache=FAKE + 8), "latent cache rows must be 16-byte"),
    ("paged_latent", dict(o_stride_head=514), "output rows"),
    ("latent_prompt", dict(dtype=cabi.L20_PD_FP32), "bf16 or fp16"),
    ("latent_prompt", dict(head_dim=64), "128 key, 64 rotary"),
    ("latent_prompt", dict(value_dim=192), "128 key, 64 rotary"),
    ("latent_prompt", dict(num_heads=0), "must be positive"),
    ("latent_prompt", dict(total_k=-1), "must be positive"),
    ("latent_prompt", dict(total_q=1 << 31), "too many tokens"),
    ("latent_prompt", dict(batch=1 << 20, num_heads=128), "units"),
    ("latent_prompt", dict(softmax_scale=-1.0), "softmax_scale"),
    ("latent_prompt", dict(value=0), "null tensor pointer"),
    ("latent_prompt", dict(cu_k=0), "null tensor pointer"),
    ("latent_prompt", dict(k_stride_token=1 << 24), "strides out of range"),
    ("latent_prompt", dict(v_stride_token=-8), "strides out of range"),
    ("latent_prompt", dict(key_rope=FAKE + 4), "16-byte aligned"),
    ("latent_prompt", dict(output=FAKE + 4), "8-byte aligned"),
    ("block_tables", dict(batch=8193), "8192 requests"),
    ("block_tables", dict(batch=-1), "8192 requests"),
    ("block_tables", dict(page_size=20), "page size"),
    ("block_tables", dict(table_pages=0), "must not be empty"),
    ("block_tables", dict(pool=0), "must not be empty"),
    ("block_tables", dict(num_slots=-1), "must not be empty"),
    ("block_tables", dict(free_count=0), "null tensor pointer"),
    ("block_tables", dict(slots=0), "null tensor pointer"),
    ("block_tables", dict(seq_lens=FAKE), "seq_lens must not be"),
    ("block_tables", dict(bt_stride_row=0), "rows overlap"),
    ("paged_latent", dict(output=FAKE), "must not be the query"),
    ("latent_prompt", dict(output=FAKE), "must not be the query"),
]


@pytest.mark.parametrize("case", BAD, ids=[f"{k}-{'_'.join(c)}-{i}" for i, (k, c, _) in enumerate(BAD)])
def test_refusals(case):
    kind, change, message = case
    args = CHECKS[kind]()
    for name, value in change.items():
        setattr(args, name, value)
    rc, error = check(kind, args)
    assert rc != 0 and message in error, error


def test_nothing_to_do_needs_no_pointers():
    for kind, empty in (("latent_write", dict(num_tokens=0, latent=0, key=0, positions=0, slot_mapping=0)),
                        ("paged_latent", dict(batch=0, query=0, output=0, seq_lens=0)),
                        ("latent_prompt", dict(total_q=0, query=0, output=0)),
                        ("latent_prompt", dict(total_k=0, key=0, value=0, key_rope=0)),
                        ("block_tables", dict(num_slots=0, slots=0, positions=0)),
                        ("block_tables", dict(batch=0, cached_lens=0, new_lens=0, block_table=0, seq_lens=0, table_pages=0))):
        args = CHECKS[kind]()
        for name, value in empty.items():
            setattr(args, name, value)
        assert check(kind, args) == (0, ""), kind


def test_workspace_sizes():
    """Two parts a run and row block, each RANK + 2 floats a row, and the runs of a sequence."""
    lib = cabi.load()
    a = paged_args()  # 2 x 16 rows, 8 x 40 tiles of 64 tokens on 256 CUs: 128 runs for each of two blocks of 16 rows
    assert lib.l20_pd_paged_latent_workspace(ctypes.byref(a), 256) == 2 * 128 * 32 * 514 * 4 + 8 * 8
    a.max_seq_len = 1 << 20  # long work: 256 runs, 32 rows together
    assert lib.l20_pd_paged_latent_workspace(ctypes.byref(a), 256) == 2 * 256 * 32 * 514 * 4 + 8 * 8
    a.max_seq_len = 64  # one tile a sequence: not split
    assert lib.l20_pd_paged_latent_workspace(ctypes.byref(a), 256) == 0
    p = prompt_args()
    assert lib.l20_pd_latent_prompt_workspace(ctypes.byref(p), 256) == 0  # few tiles of keys
    p.total_k = 3 * 5000
    assert lib.l20_pd_latent_prompt_workspace(ctypes.byref(p), 256) == 2 * 512 * 128 * 130 * 4 + 3 * 8 * 2 * 8
    p.num_heads = 1 << 12  # blocks of rows enough to fill the chip
    assert lib.l20_pd_latent_prompt_workspace(ctypes.byref(p), 256) == 0
    p = prompt_args()  # one long sequence among many: the join's grid would be mostly empty
    p.batch, p.num_heads, p.max_q_len, p.total_q, p.total_k = 64, 32, 1 << 17, 1 << 17, 1 << 18
    assert lib.l20_pd_latent_prompt_workspace(ctypes.byref(p), 256) == 0
    assert lib.l20_pd_latent_prompt_workspace(None, 256) == 0 and lib.l20_pd_paged_latent_workspace(None, 256) == 0


def test_functions_refuse_cpu_tensors():
    import l20_block_tables as bt
    import l20_latent_attention as la

    x, i = torch.zeros(4, 16, 576, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="l20_paged_latent_attention requires an MI355X"):
        la.l20_paged_latent_attention(x, x, i.view(4, 1), i, softmax_scale=1.0)
    with pytest.raises(RuntimeError, match="l20_latent_prompt_attention requires an MI355X"):
        la.l20_latent_prompt_attention(x[..., :192], x[..., :128], x[:, 0, :64], x[..., :128], i, i, 4)
    with pytest.raises(RuntimeError, match="l20_latent_rope_and_cache requires an MI355X"):
        la.l20_latent_rope_and_cache(None, x[:, 0, :512], x[:, 0, 512:], i.long(), x[:, 0, :64], True, x, i.long())
    with pytest.raises(RuntimeError, match="l20_build_block_tables requires an MI355X"):
        bt.l20_build_block_tables(i, i, i.view(4, 1), i, i[:1], i.long(), i.long(), torch.zeros(5, dtype=torch.int32), i, 16)


def test_fake_implementations_keep_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import l20_latent_attention  # noqa: F401

    with FakeTensorMode():
        q = torch.empty(8, 16, 576, dtype=torch.bfloat16, device="cuda")
        cache = torch.empty(9, 16, 576, dtype=torch.bfloat16, device="cuda")
        out, i = torch.empty(8, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(8, dtype=torch.int32, device="cuda")
        got = torch.ops.l20_stack.paged_latent_attention_out(q, cache, i.view(8, 1), i, out, None, 1.0, 1.0, 16)
        assert got.shape == out.shape


@pytest.mark.parametrize("heads,q_len", [(1, 1), (16, 1), (28, 4), (28, 5), (64, 1), (128, 3)])
@pytest.mark.parametrize("cache", [cabi.L20_PD_KV_FP8_E4M3, cabi.L20_PD_KV_BF16], ids=["e4m3", "model"])
@pytest.mark.parametrize("cus", [256, 64])
def test_workspace_of_a_batch_is_enough_for_smaller_ones(heads, q_len, cache, cus):
    """A step of a serving loop may have fewer sequences, and a shorter bound, than what was allocated for."""
    lib, a = cabi.load(), paged_args()
    a.num_heads, a.q_len, a.cache_dtype = heads, q_len, cache

    def size(batch, length):
        a.batch, a.max_seq_len = batch, length
        return lib.l20_pd_paged_latent_workspace(ctypes.byref(a), cus)

    for length in (16, 64, 128, 256, 512, 1000, 4096, 131072):
        sizes = [size(b, length) for b in [*range(1, 280), 500, 1000, 4096]]
        assert sizes == sorted(sizes)
    for batch in (1, 2, 8, 32, 64, 200, 1000):
        sizes = [size(batch, n) for n in [*range(0, 4096, 16), 8192, 65536, 1 << 19]]
        assert sizes == sorted(sizes)


OVER = [
    ("paged_latent", dict(output=FAKE + 128, o_stride_row=16 * 576, o_stride_head=576)),  # query[..., 64:]
    ("paged_latent", dict(output=FAKE + 2 * 512, o_stride_row=16 * 576, o_stride_head=576)),  # the last 64 dims alone
    ("paged_latent", dict(output=FAKE + 2 * (15 * 16 * 576 + 15 * 576) + 2 * 568)),  # the last row's last dims
    ("paged_latent", dict(query=FAKE << 8, output=(FAKE << 8) - 2 * (16 * 16 * 512 - 4))),  # the other end
    ("paged_latent", dict(batch=1, q_len=1, num_heads=1, output=FAKE + 1144, o_stride_row=0, o_stride_head=0)),
    ("latent_prompt", dict(output=FAKE + 128, o_stride_token=8 * 192, o_stride_head=192)),
    ("latent_prompt", dict(query=FAKE << 8, value=FAKE << 12, output=FAKE << 12, o_stride_token=8 * 256, o_stride_head=256)),
    ("latent_prompt", dict(query=FAKE << 8, key=FAKE << 12, output=(FAKE << 12) + 8, o_stride_token=8 * 256, o_stride_head=256)),
    ("latent_prompt", dict(query=FAKE << 8, key_rope=FAKE << 12, output=(FAKE << 12) + 500 * 128 - 8)),
]


@pytest.mark.parametrize("kind,change", OVER, ids=[f"{k}-{i}" for i, (k, _) in enumerate(OVER)])
def test_calls_refuse_outputs_over_their_inputs(kind, change):
    """Bytes shared with an input, whatever the two views' strides: refused before anything is launched."""
    args = CHECKS[kind]()
    for name, value in change.items():
        setattr(args, name, value)
    lib = cabi.load()
    rc = getattr(lib, f"l20_pd_{kind}")(ctypes.byref(args), None)
    assert rc == cabi.L20_PD_EINVAL and "output must not lie over" in cabi.last_error()


APART = dict(query=FAKE << 8, query_out=FAKE << 9, latent=FAKE << 10, latent_out=FAKE << 11, key=FAKE << 12, key_out=FAKE << 13)


@pytest.mark.parametrize("change", [
    dict(latent_out=FAKE << 10),  # another row stride
    dict(latent_out=(FAKE << 10) + 16, lo_stride_token=576),
    dict(key=(FAKE << 10) + 1024, key_out=(FAKE << 10) + 1024 - 112, ko_stride_token=576),  # over the latent
    dict(query_out=(FAKE << 8) + 2 * 16),  # (strides of an absorbed query)
    dict(query_out=FAKE << 8, qo_stride_token=16 * 192, qo_stride_head=64),
    dict(query_out=(FAKE << 12) - 2 * 16 * 576),
], ids=range(6))
def test_cache_producer_refuses_outputs_over_other_inputs(change):
    args = write_args()
    for name, value in {**APART, **change}.items():
        setattr(args, name, value)
    rc = cabi.load().l20_pd_latent_rope_and_cache(ctypes.byref(args), None)
    assert rc == cabi.L20_PD_EINVAL and "its input itself or lie apart" in cabi.last_error()
