"""GPU: the latent cache producer against plain arithmetic, bit for bit where nothing is summed (RoPE, the fp8
quantiser, the rows' places), within half a step of the type where the norm's sum has an order of its own."""

import pytest
import torch

import latent_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X GPU")
    import l20_latent_attention  # noqa: F401


def make(tokens, heads, rank=512, dtype=torch.bfloat16, cs_dtype=torch.bfloat16, fp8=False, page=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    theta = torch.rand(500, 32, generator=g, dtype=torch.float64) * 6.28
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[::7] = -1
    cache_dtype = torch.float8_e4m3fn if fp8 else dtype
    return {"query": torch.randn(tokens, heads, 192, generator=g).to(dtype).cuda()[..., 128:],
            "down": torch.randn(tokens, rank + 64, generator=g).to(dtype).cuda(),
            "positions": torch.randint(0, 500, (tokens,), generator=g).cuda(),
            "cs": torch.cat([theta.cos(), theta.sin()], -1).to(cs_dtype).cuda(), "slots": slots.cuda(), "rank": rank,
            "weight": (1 + torch.randn(rank, generator=g) / 5).to(dtype).cuda(),
            "cache": torch.full((pages, page, rank + 64), 2.0).to(cache_dtype).cuda(), "scale": 1 / 50.0 if fp8 else 1.0}


def rope(x, cs, positions, neox):
    """x [..., 64] in fp32, each product and the sum rounded to fp32."""
    c, s = cs[positions].float().chunk(2, dim=-1)
    if x.dim() == 3:
        c, s = c[:, None], s[:, None]
    dtype, x = x.dtype, x.float()
    if neox:
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2).to(dtype)


def stored(c, latent, key):
    """The cache after the write of `latent` and `key`, as raw values of its type."""
    want = c["cache"].clone()
    flat = want.view(-1, want.shape[-1])
    row = torch.cat([latent, key], -1)
    live = (c["slots"] >= 0) & (c["slots"] < flat.shape[0])
    if want.dtype == torch.float8_e4m3fn:
        row = (row.float() / c["scale"]).clamp(-448, 448).to(torch.float8_e4m3fn)
        flat.view(torch.uint8)[c["slots"][live]] = row.view(torch.uint8)[live]
    else:
        flat[c["slots"][live]] = row[live]
    return want


def call(c, neox, norm, **kw):
    import l20_latent_attention as la

    la.l20_latent_rope_and_cache(c["query"], c["down"][:, :c["rank"]], c["down"][:, c["rank"]:], c["positions"], c["cs"], neox,
                                 c["cache"], c["slots"], norm_weight=c["weight"] if norm else None, norm_eps=EPS,
                                 cache_scale=c["scale"], **kw)
    torch.cuda.synchronize()


SHAPES = [(1, 16, 512, 16), (37, 3, 512, 48), (64, 128, 256, 16), (515, 28, 512, 64), (9, 1, 256, 4096)]


@pytest.mark.parametrize("shape", SHAPES, ids=[f"t{s[0]}_h{s[1]}_r{s[2]}_p{s[3]}" for s in SHAPES])
@pytest.mark.parametrize("neox", [True, False], ids=["neox", "pairs"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("dtype,cs,fp8", [(torch.bfloat16, torch.bfloat16, False), (torch.float16, torch.float32, True),
                                          (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, False)],
                         ids=["bf16", "fp16_e4m3", "bf16_e4m3", "fp16"])
def test_write_out_of_place(shape, neox, norm, dtype, cs, fp8):
    tokens, heads, rank, page = shape
    c = make(tokens, heads, rank, dtype, cs, fp8, page, seed=tokens + heads)
    kept = c["query"].clone(), c["down"].clone()
    outs = {"query_out": torch.zeros(tokens, heads, rank + 64, dtype=dtype, device="cuda")[..., rank:],
            "latent_out": torch.empty(tokens, rank, dtype=dtype, device="cuda"),
            "key_rope_out": torch.empty(tokens, 64, dtype=dtype, device="cuda")}
    before = c["cache"].clone()
    call(c, neox, norm, **outs)
    assert torch.equal(c["query"], kept[0]) and torch.equal(c["down"], kept[1])
    assert torch.equal(outs["query_out"], rope(c["query"], c["cs"], c["positions"], neox))
    key = rope(c["down"][:, rank:], c["cs"], c["positions"], neox)
    assert torch.equal(outs["key_rope_out"], key)
    x = c["down"][:, :rank]
    if norm:
        # one rounding of T; fp32: rank additions, the root, the division and two products
        x = x.double()
        want = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * c["weight"].double()
        tol = want.abs() * (R.half(dtype) + (rank + 8) * 2.0 ** -24) + 2.0 ** -25
        assert bool(((outs["latent_out"].double() - want).abs() <= tol).all())
    else:
        assert torch.equal(outs["latent_out"], x)
    got, c["cache"] = c["cache"], before
    want = stored(c, outs["latent_out"], key)
    view = torch.uint8 if fp8 else torch.int16
    assert torch.equal(got.view(view), want.view(view))


def test_write_in_place_and_without_a_query():
    c = make(70, 5, seed=3)
    d = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    d["query"] = c["query"].clone()
    outs = {"query_out": torch.empty_like(d["query"]), "latent_out": torch.empty(70, 512, dtype=torch.bfloat16, device="cuda"),
            "key_rope_out": torch.empty(70, 64, dtype=torch.bfloat16, device="cuda")}
    call(d, True, True, **outs)
    call(c, True, True)
    assert torch.equal(c["query"], outs["query_out"])
    assert torch.equal(c["down"], torch.cat([outs["latent_out"], outs["key_rope_out"]], -1))
    assert torch.equal(c["cache"], d["cache"])
    e = make(70, 5, seed=3)
    e["query"] = None
    call(e, True, True)
    assert torch.equal(e["down"], c["down"]) and torch.equal(e["cache"], c["cache"])


def test_write_slots_and_positions_out_of_range():
    """Slots beyond the cache are not stored; positions outside the table take its first or last row."""
    c = make(20, 2, seed=4)
    total = c["cache"].shape[0] * 16
    c["slots"][1], c["slots"][2], c["slots"][3] = total, 2 ** 40, -(2 ** 40)
    c["positions"][4], c["positions"][5] = -3, 10 ** 12
    out = {"query_out": torch.empty_like(c["query"]), "latent_out": torch.empty(20, 512, dtype=torch.bfloat16, device="cuda"),
           "key_rope_out": torch.empty(20, 64, dtype=torch.bfloat16, device="cuda")}
    before = c["cache"].clone()
    call(c, True, False, **out)
    pos = c["positions"].clamp(0, 499)
    key = rope(c["down"][:, 512:], c["cs"], pos, True)
    assert torch.equal(out["key_rope_out"], key)
    got, c["cache"] = c["cache"], before
    assert torch.equal(got, stored(c, c["down"][:, :512], key))


def test_write_refusals():
    import l20_latent_attention as la

    c = make(8, 2, seed=5)
    lat, key = c["down"][:, :512], c["down"][:, 512:]
    rest = (c["positions"], c["cs"], True, c["cache"], c["slots"])
    with pytest.raises(RuntimeError, match="rank 256 or 512"):
        la.l20_latent_rope_and_cache(None, lat[:, :384], key, *rest)
    with pytest.raises(RuntimeError, match="key_rope"):
        la.l20_latent_rope_and_cache(None, lat, key[:4], *rest)
    with pytest.raises(RuntimeError, match="FP16 and BF16"):
        la.l20_latent_rope_and_cache(None, lat.float(), key.float(), *rest)
    with pytest.raises(RuntimeError, match="int64"):
        la.l20_latent_rope_and_cache(None, lat, key, c["positions"].int(), *rest[1:])
    with pytest.raises(RuntimeError, match="norm_weight"):
        la.l20_latent_rope_and_cache(None, lat, key, *rest, norm_weight=c["weight"].float())
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        la.l20_latent_rope_and_cache(None, torch.zeros(8, 513, dtype=torch.bfloat16, device="cuda")[:, 1:], key, *rest)
    with pytest.raises(RuntimeError, match="query_out needs query_rope"):
        la.l20_latent_rope_and_cache(None, lat, key, *rest, query_out=c["query"])


def test_one_token_of_any_stride():
    """The stride of a dimension of size 1 says nothing: a transposed column, here."""
    import l20_latent_attention as la

    c = make(1, 1, seed=12)
    c["slots"].fill_(3)
    want = {k: c[k].clone() for k in ("down", "query", "cache")}
    la.l20_latent_rope_and_cache(want["query"], want["down"][:, :512], want["down"][:, 512:], c["positions"], c["cs"], True,
                                 want["cache"], c["slots"])
    down, query = c["down"].as_strided((1, 576), (1, 1)), c["query"].clone().as_strided((1, 1, 64), (1, 3, 1))
    la.l20_latent_rope_and_cache(query, down[:, :512], down[:, 512:], c["positions"], c["cs"], True, c["cache"], c["slots"])
    torch.cuda.synchronize()
    assert torch.equal(down, want["down"]) and torch.equal(query, want["query"]) and torch.equal(c["cache"], want["cache"])


def test_on_another_stream_and_in_a_graph():
    c = make(40, 6, fp8=True, seed=13)
    outs = {"query_out": torch.empty(40, 6, 64, dtype=torch.bfloat16, device="cuda"),
            "latent_out": torch.empty(40, 512, dtype=torch.bfloat16, device="cuda"),
            "key_rope_out": torch.empty(40, 64, dtype=torch.bfloat16, device="cuda")}
    call(c, True, True, **outs)
    want = {k: v.clone() for k, v in {**outs, "cache": c["cache"].view(torch.uint8)}.items()}
    import l20_latent_attention as la

    def step():
        la.l20_latent_rope_and_cache(c["query"], c["down"][:, :512], c["down"][:, 512:], c["positions"], c["cs"], True,
                                     c["cache"], c["slots"], norm_weight=c["weight"], norm_eps=EPS, cache_scale=c["scale"], **outs)

    def wiped():
        for v in outs.values():
            v.zero_()
        c["cache"].view(torch.uint8).flatten(0, 1)[c["slots"].clamp_min(0)] = 9

    def same():
        torch.cuda.synchronize()
        live = c["slots"][c["slots"] >= 0]
        return all(torch.equal(v, want[k]) for k, v in outs.items()) and torch.equal(
            c["cache"].view(torch.uint8).flatten(0, 1)[live], want["cache"].flatten(0, 1)[live])

    side = torch.cuda.Stream()
    wiped()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        wiped()
        graph.replay()
        assert same()


@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [True, False], ids=["e4m3", "model"])
def test_values_that_are_not_finite(norm, dtype, fp8):
    """The cache holds what the outputs hold: a NaN stays one in an fp8 cache too, an infinity becomes its largest value."""
    c = make(30, 3, dtype=dtype, cs_dtype=torch.float32, fp8=fp8, seed=14)
    nan, inf = float("nan"), float("inf")
    for t, col, x in ((1, 5, nan), (2, 7, inf), (3, 9, -inf), (4, 512 + 3, nan), (5, 512 + 40, inf), (6, 0, -nan), (6, 1, inf),
                      (8, 511, nan), (8, 512 + 63, -inf)):
        c["down"][t, col] = x
    outs = {"query_out": torch.empty_like(c["query"]), "latent_out": torch.empty(30, 512, dtype=dtype, device="cuda"),
            "key_rope_out": torch.empty(30, 64, dtype=dtype, device="cuda")}
    before = c["cache"].clone()
    call(c, True, norm, **outs)
    key = rope(c["down"][:, 512:], c["cs"], c["positions"], True)
    assert torch.equal(key.isnan(), outs["key_rope_out"].isnan())
    assert torch.equal(key.nan_to_num(9.0), outs["key_rope_out"].nan_to_num(9.0))
    rows = outs["latent_out"].isnan()
    assert bool(rows[1, 5]) and bool(rows[6, 0]) and bool(rows[8, 511]) and bool(rows[1].all()) == norm
    got, c["cache"] = c["cache"].float(), before
    want = stored(c, outs["latent_out"], key).float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0))


def test_write_into_the_gaps_of_the_inputs():
    """Outputs interleaved with the inputs share nothing with them; ones in another layout of the same memory do."""
    import l20_latent_attention as la

    def parts():
        c = make(40, 3, seed=15)
        wide = torch.zeros(40, 2 * 576, dtype=torch.bfloat16, device="cuda")
        wide[:, :576] = c["down"]
        return c, wide

    c, wide = parts()
    call(c, True, True)
    d, wide = parts()
    d["down"] = wide[:, :576]
    kept = wide[:, :576].clone()
    call(d, True, True, latent_out=wide[:, 576:1088], key_rope_out=wide[:, 1088:])
    assert torch.equal(wide[:, 576:], c["down"]) and torch.equal(wide[:, :576], kept) and torch.equal(c["cache"], d["cache"])
    with pytest.raises(RuntimeError, match="its input itself or lie apart"):
        call(d, True, False, latent_out=wide.view(-1)[:40 * 512].view(40, 512))
    with pytest.raises(RuntimeError, match="its input itself or lie apart"):
        call(d, True, True, key_rope_out=wide[:, 448:512])
