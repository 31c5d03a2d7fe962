"""Decode attention over 8-bit caches, and with capped scores and a distance bias over every kind of cache, against the plain
64-bit form.

Tolerances.  The output is rounded once (half of finfo.eps, relative).  Before that: a score is off by 2^-22 of the magnitude of
its terms, capped ones by 2^-21 of the cap, so a probability by that relative amount; sums in fp32 add a few 2^-24.  With the
scores' magnitudes here (below 100) that is 100 x 2^-21 = 5e-5 of the values' magnitude, which is below 8."""
import math

import numpy as np
import pytest
import torch

from attention_plain import attention, e4m3, scale_of, to_e4m3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from inference_b200 import ops as _ops
    assert _ops.has_cuda() and _ops.device_sm_version(0) == 100, "needs a B200"
    return _ops


def cache_case(heads, kv, dim, block, lens, dtype, seed=0, fp8=True):
    g = torch.Generator().manual_seed(seed)
    batch, per = len(lens), max(1, -(-max(lens) // block))
    blocks = batch * per + 2
    q = (1.5 * torch.randn(batch, heads, dim, generator=g)).to(dtype)
    k, v = (torch.randn(blocks, block, kv, dim, generator=g) for _ in range(2))
    # blocks of very different sizes
    v *= torch.exp2(torch.randint(-3, 3, (blocks, 1, kv, 1), generator=g).float())
    tables = torch.randperm(blocks, generator=g)[: batch * per].to(torch.int32).view(batch, per)
    c = dict(q=q, tables=tables, lens=torch.tensor(lens, dtype=torch.int32))
    for n, x in (("k", k), ("v", v)):
        if fp8:
            scales = torch.tensor([[scale_of(float(x[i, :, h].abs().max())) for h in range(kv)] for i in range(blocks)])
            c[n + "_cache"], c[n + "_scales"] = to_e4m3(x / scales[:, None, :, None]), scales
        else:
            c[n + "_cache"] = x.to(dtype)
    return c


def values(c, name, b):
    """[len, kv, dim] of a sequence in 64 bits."""
    blocks = c["tables"][b].long()
    x = c[name + "_cache"][blocks]
    x = e4m3(x) * c[name + "_scales"][blocks][:, None, :, None].double() if name + "_scales" in c else x.double()
    return x.flatten(0, 1)[: int(c["lens"][b])]


def want_of(c, scale, cap=0.0, slopes=None, holes=None):
    out = []
    for b in range(c["q"].shape[0]):
        k, v = values(c, "k", b), values(c, "v", b)
        n = k.shape[0]
        seen = None
        if holes is not None:
            seen = ~holes[b][:n][None, :]
            if n and not bool(seen.any()):
                out.append(torch.zeros(1, *c["q"].shape[1:], dtype=torch.float64))
                continue
        out.append(attention(c["q"][b:b + 1], k, v, scale, cap, slopes, seen, torch.tensor([n - 1])))
    return torch.cat(out)


def call(ops, c, scale, **kw):
    d = {n: t.cuda() for n, t in c.items()}
    if "slopes" in kw:
        kw["alibi_slopes"] = kw.pop("slopes").cuda()
    if "k_scales" in d:
        return ops.paged_attn_decode_fp8(d["q"], d["k_cache"], d["v_cache"], d["k_scales"], d["v_scales"], d["tables"], d["lens"], scale, **kw)
    return ops.paged_attn_decode(d["q"], d["k_cache"], d["v_cache"], d["tables"], d["lens"], scale, **kw)


def close(got, want, dtype, atol=4e-4):
    want = want.cpu()
    f = torch.finfo(dtype)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= want.abs() * (f.eps / 2) * 1.01 + atol).all()), float((err - want.abs() * f.eps / 2).max())


SHAPES = [
    # heads, kv_heads, dim, block, lengths
    (32, 8, 128, 16, [1, 17, 129]),
    (8, 8, 64, 16, [0, 16, 15, 64, 65, 300]),
    (7, 1, 128, 32, [63, 1, 0, 200]),                 # seven rows
    (9, 1, 64, 16, [127, 128, 129]),                  # nine query heads of a KV head: three CTAs of three
    (24, 2, 256, 48, [500, 48, 49]),                  # a block size between powers of two
    (16, 8, 256, 16, [33, 1000, 5]),
    (4, 1, 64, 64, [int(x) for x in range(0, 300, 7)]),
    (16, 2, 128, 16, [30000, 1, 64 * 40]),            # a pair spread over many CTAs beside short ones
    (8, 1, 128, 16, [20000]),
]
IDS = [str(i) for i in range(len(SHAPES))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_8_bit_caches(ops, dtype, shape):
    heads, kv, dim, block, lens = shape
    c = cache_case(heads, kv, dim, block, lens, dtype, seed=dim + len(lens))
    scale = dim ** -0.5
    got = call(ops, c, scale)
    close(got, want_of(c, scale), dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((got[b] == 0).all())


@pytest.mark.parametrize("cap,bias", [(0.0, True), (4.0, False), (30.0, True)])
@pytest.mark.parametrize("kind", ["fp8", "bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form", [0, 1, 2], ids=["auto", "cuda_cores", "tensor_cores"])
def test_capped_scores_and_distance_bias(ops, kind, cap, bias, form):
    dtype = {"fp16": torch.float16, "fp32": torch.float32}.get(kind, torch.bfloat16)
    if form and kind in ("fp8", "fp32"):
        pytest.skip("one form only")
    ops.set_option("attn_path", form)
    try:
        for heads, kv, dim, block, lens in SHAPES[:7:2] + SHAPES[7:]:
            c = cache_case(heads, kv, dim, block, lens, dtype, seed=heads, fp8=kind == "fp8")
            c["q"] = (4 * c["q"].float()).to(dtype)     # scores that reach the cap
            kw = dict(softcap=cap)
            slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads) if bias else None
            if bias:
                slopes[heads // 2] = -0.001
                kw["slopes"] = slopes
            got = call(ops, c, dim ** -0.5, **kw)
            # (fp32 caches: scores off by 2^-22 of their magnitude times the values')
            close(got, want_of(c, dim ** -0.5, cap, slopes), dtype)
    finally:
        ops.set_option("attn_path", 0)


@pytest.mark.parametrize("heads,kv,dim,lens", [(16, 8, 128, [900, 0, 1000, 1, 128, 129, 700] * 2), (8, 8, 64, [300] * 50 + [0, 777]),
                                               (4, 2, 256, [64 * i for i in range(1, 41)])], ids=["few", "many", "large"])
def test_shares_that_end_with_the_sequences(ops, heads, kv, dim, lens):
    """More units of tokens than CTAs, fewer (sequence, head) pairs than CTAs: up to three units each."""
    c = cache_case(heads, kv, dim, 16, lens, torch.bfloat16, seed=len(lens))
    close(call(ops, c, dim ** -0.5), want_of(c, dim ** -0.5), torch.bfloat16)


def test_without_cap_and_bias_it_is_the_plain_call(ops):
    for lens in ([40, 300], [9000, 16000, 1]):
        c = cache_case(32, 8, 128, 16, lens, torch.bfloat16, fp8=False)
        assert torch.equal(call(ops, c, 0.1), call(ops, c, 0.1, slopes=torch.zeros(32)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_holes_in_the_table(ops, dtype):
    c = cache_case(8, 2, 128, 32, [100, 40, 5000, 33], dtype, seed=4)
    holes = []
    c2 = dict(c, tables=c["tables"].clone())
    for b, js in enumerate(([1], [0, 1], [3, 100, 101, 156], [1])):
        h = torch.zeros(c["tables"].shape[1] * 32, dtype=torch.bool)
        for i, j in enumerate(js):
            c2["tables"][b, j] = -1 if i % 2 == 0 else c["k_cache"].shape[0] + i
            h[j * 32:(j + 1) * 32] = True
        holes.append(h)
    got = call(ops, c2, 0.09)
    close(got, want_of(c, 0.09, holes=holes), dtype)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_lies_behind_a_sequence_is_not_read_into_it(ops, dtype):
    """NaN bytes in every row that is no token's, NaN scales on blocks that are nobody's."""
    lens = [40, 5000, 1, 0, 16]
    c = cache_case(8, 2, 64, 16, lens, dtype, seed=6)
    want = want_of(c, 0.125)
    used = torch.zeros(c["k_cache"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[int(c["tables"][b, t // 16]), t % 16] = True
    for n in ("k", "v"):
        c[n + "_cache"][~used] = 0x7F
        c[n + "_scales"][~used.any(1)] = float("nan")
    close(call(ops, c, 0.125), want, dtype)


def test_nan_in_the_cache_reaches_its_own_heads_only(ops):
    c = cache_case(8, 4, 64, 16, [50, 3000], torch.bfloat16, seed=3)
    c["v_cache"][int(c["tables"][0, 1]), 2, 1, 5] = 0x7F
    c["k_cache"][int(c["tables"][1, 70]), 2, 3, 5] = 0xFF
    got = call(ops, c, 0.125)
    nan = torch.isnan(got).cpu()
    want = torch.zeros_like(nan)
    want[0, 2:4, 5] = True
    want[1, 6:8] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_far_apart_and_queries_of_any_size(ops, dtype):
    """Blocks whose scales differ by 2^40, scales of zero, a query row of 2^-60 and one of 2^12."""
    c = cache_case(4, 2, 128, 16, [64, 200], dtype, seed=9)
    c["v_scales"][::3] *= 2.0 ** 20
    c["v_scales"][1::3] *= 2.0 ** -20
    c["v_scales"][2] = 0
    if dtype == torch.bfloat16:
        c["q"][0, 0] *= 2.0 ** -60
    c["q"][0, 1] *= 2.0 ** 10
    want = want_of(c, 0.0884)
    got = call(ops, c, 0.0884).cpu().double()
    ok = want.abs() <= torch.finfo(dtype).max
    size = torch.stack([values(c, "v", b).abs().amax(0).repeat_interleave(2, 0) for b in range(2)])
    # the scores of head (0, 1) are some 2^10 x 5: probabilities to 2^-9
    size[0, 1] *= 40
    assert bool(((got - want).abs()[ok] <= (want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + size * 5e-5)[ok]).all())


def test_large_batches_odd_query_addresses_and_out(ops):
    lens = [(i * 37) % 90 for i in range(1030)]          # more sequences than the evenly cut form takes
    c = cache_case(2, 1, 64, 16, lens, torch.bfloat16, seed=4)
    got = call(ops, c, 0.125)
    close(got, want_of(c, 0.125), torch.bfloat16)
    d = {n: t.cuda() for n, t in c.items()}
    buf = torch.zeros(d["q"].numel() + 1, dtype=torch.bfloat16, device="cuda")
    buf[1:] = d["q"].flatten()
    out = torch.empty_like(d["q"])
    again = ops.paged_attn_decode_fp8(buf[1:].view(d["q"].shape), d["k_cache"], d["v_cache"], d["k_scales"], d["v_scales"], d["tables"],
                                      d["lens"], 0.125, out=out)
    assert again is out and torch.equal(out, got)


def test_graphs_and_streams_share_no_scratch(ops):
    cs = [cache_case(16, 2, 128, 16, lens, torch.bfloat16, seed=i) for i, lens in enumerate(([20000, 300], [9000, 16000]))]
    ds = [{n: t.cuda() for n, t in c.items()} for c in cs]
    run = lambda d, **kw: ops.paged_attn_decode_fp8(d["q"], d["k_cache"], d["v_cache"], d["k_scales"], d["v_scales"], d["tables"], d["lens"],
                                                    0.1, **kw)
    want = [run(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros_like(want[0]) for _ in range(3)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, out, d in zip(graphs, outs, ds):
        with torch.cuda.graph(g, stream=streams[2]):
            run(d, out=out)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        run(ds[0], out=outs[2], stream=streams[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(outs[2], want[0])
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,block", [(32, 8, 128, 16), (8, 8, 64, 16), (4, 2, 256, 16), (8, 2, 128, 32)])
def test_every_step_has_its_blocks_scales(ops, dtype, heads, kv, dim, block):
    """Scales that differ from block to block and are no powers of two, over many steps of every warp, again and again."""
    c = cache_case(heads, kv, dim, block, [4101, 700, 33], dtype, seed=dim + block)
    g = torch.Generator().manual_seed(1)
    for n in ("k_scales", "v_scales"):
        c[n] = c[n] * (0.4 + 1.6 * torch.rand(c[n].shape, generator=g))
    got = call(ops, c, dim ** -0.5)
    # values up to some 40
    close(got, want_of(c, dim ** -0.5), dtype, atol=2e-3)
    for _ in range(20):
        assert torch.equal(call(ops, c, dim ** -0.5), got)


@pytest.mark.parametrize("kind", ["fp8", "bf16", "fp16"])
@pytest.mark.parametrize("form", [0, 1, 2], ids=["auto", "cuda_cores", "tensor_cores"])
@pytest.mark.parametrize("cap", [3e4, 1e6, 1e9])
def test_caps_far_above_the_scores(ops, kind, form, cap):
    """A score's error goes by the score, not by the cap: 2^-20 of it at most, which the default tolerance has room for."""
    if form and kind == "fp8":
        pytest.skip("one form only")
    dtype = torch.float16 if kind == "fp16" else torch.bfloat16
    ops.set_option("attn_path", form)
    try:
        for heads, kv, dim, block, lens in SHAPES[:6]:
            c = cache_case(heads, kv, dim, block, lens, dtype, seed=heads, fp8=kind == "fp8")
            close(call(ops, c, dim ** -0.5, softcap=cap), want_of(c, dim ** -0.5, cap), dtype)
    finally:
        ops.set_option("attn_path", 0)


@pytest.mark.parametrize("kind", ["fp8", "bf16", "fp16"])
@pytest.mark.parametrize("form", [1, 2], ids=["cuda_cores", "tensor_cores"])
def test_scores_around_the_cap_of_every_size(ops, kind, form):
    """Caps from a hundredth of the scores to a hundred times them: every part of the curve."""
    dtype = torch.float16 if kind == "fp16" else torch.bfloat16
    ops.set_option("attn_path", form)
    try:
        for cap in (0.05, 0.7, 3.0, 9.0, 40.0, 500.0):
            c = cache_case(8, 2, 128, 16, [40, 700, 3], dtype, seed=int(cap * 100), fp8=kind == "fp8")
            close(call(ops, c, 0.1, softcap=cap), want_of(c, 0.1, cap), dtype)
    finally:
        ops.set_option("attn_path", 0)


@pytest.mark.parametrize("power", [100, 116, 120, -100, -120])
def test_query_rows_at_the_ends_of_bf16(ops, power):
    """A row near 2^power under a scale near its inverse: scores like anybody's."""
    c = cache_case(4, 2, 128, 16, [64, 200], torch.bfloat16, seed=5)
    c["q"] = c["q"].clamp(-4, 4)
    c["q"][:, 1] *= 2.0 ** power
    scale = 2.0 ** -power * 0.0884
    want, got = want_of(c, scale), call(ops, c, scale)
    if power < 0:      # the other rows' scores are without bounds there
        want, got = want[:, 1:2], got[:, 1:2]
    close(got, want, torch.bfloat16)


@pytest.mark.parametrize("cap,bias", [(50.0, False), (2000.0, False), (0.0, True), (2000.0, True)])
def test_fp32_caches_to_fp32s_own_bound(ops, cap, bias):
    """Short sequences whose weights are of one size, so that a score's error shows.  Bound: a score's sum of 64 products of
    fp32 in a tree of at most 16 steps, 2^-20 of the products' magnitude; tanhf 2^-22, the bias 2^-23 and the exponential 2^-22
    of theirs; a weight twice that, times the spread of the values; sums and the output's rounding 8 x 2^-24 of the largest value."""
    lens = [2, 3, 5, 9, 17, 31]
    c = cache_case(4, 2, 64, 16, lens, torch.float32, seed=2, fp8=False)
    scale = 0.03
    slopes = torch.tensor([0.5, 0.01, 0.1, -0.02]) if bias else None
    kw = dict(softcap=cap, **(dict(slopes=slopes) if bias else {}))
    got, want = call(ops, c, scale, **kw).cpu().double(), want_of(c, scale, cap, slopes).cpu()
    rough = []
    for b, n in enumerate(lens):
        k, v = values(c, "k", b), values(c, "v", b)
        size = (c["q"][b].double().abs()[:, None] * k.repeat_interleave(2, 1).abs().permute(1, 0, 2)).sum(-1) * scale     # [heads, n]
        far = torch.arange(n - 1, -1, -1).double()
        score = 2.0 ** -20 * size + 2.0 ** -22 * size + (slopes.abs()[:, None].double() * far * 2.0 ** -23 if bias else 0.0)
        top = v.abs().amax(0).repeat_interleave(2, 0)                                                                    # [heads, dim]
        bound = 2 * (score.amax(1)[:, None] + 2.0 ** -22) * top + 8 * 2.0 ** -24 * top
        assert bool(((got[b] - want[b]).abs() <= bound).all()), (b, float(((got[b] - want[b]).abs() / bound).max()))
        if cap:    # what 1 - 2 / (1 + e^2x) in fp32 would give: off by more than the bound somewhere at the larger cap
            x = (torch.einsum("hd,nhd->hn", c["q"][b].double(), k.repeat_interleave(2, 1)) * scale / cap).float()
            s = (cap * (1 - 2 / (1 + torch.exp2(x * 2.885390081777927)))).double()
            s = s - (slopes[:, None].double() * far if bias else 0.0)
            off = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), v.repeat_interleave(2, 1))
            rough.append(bool(((off - want[b]).abs() > bound).any()))
    assert cap != 2000.0 or any(rough)
