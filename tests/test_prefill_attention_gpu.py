"""prefill_attn against the plain 64-bit form.

Tolerance: P is rounded to the operands' type, half a step per term, so the weighted sum is off by eps / 2 of sum p |v| at most;
the output is rounded once, eps / 2 of itself; scores and sums in fp32 add 5e-5 of the largest |v| (scores below 100 good to
2^-21 of their magnitude)."""
import pytest
import torch

from attention_plain import attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from inference_b200 import ops as _ops
    assert _ops.has_cuda() and _ops.device_sm_version(0) == 100, "needs a B200"
    return _ops


def inputs(lens, heads, kv, dim, dtype, seed=0, lead=0, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = lead + sum(lens) + tail
    qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=g, device="cuda").to(dtype)
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    return qkv[:, :heads] * 2, qkv[:, heads:heads + kv], qkv[:, heads + kv:], cu


def check(got, q, k, v, cu, scale, cap=0.0, slopes=None, prefix=None, vmax=8.0):
    eps = torch.finfo(q.dtype).eps
    for b in range(len(cu) - 1):
        r = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        lim = (i + 1).clamp(min=int(prefix[b]) if prefix is not None else 0)
        seen = i[None, :] < lim[:, None]
        want = attention(q[r], k[r], v[r], scale, cap, slopes, seen, i)
        size = attention(q[r], k[r], v[r].abs(), scale, cap, slopes, seen, i)
        err = (got[r].double() - want).abs()
        bound = eps / 2 * 1.02 * (want.abs() + size) + 5e-5 * vmax
        assert bool((err <= bound).all()), (b, float((err - bound).max()), float(err.max()))


SHAPES = [
    # heads, kv_heads, dim, lengths
    (2, 1, 128, [1]),
    (4, 2, 128, [1, 127, 128, 129]),
    (3, 3, 128, [300, 5, 257, 255, 256]),                    # 256 rows of a head per CTA
    (8, 2, 64, [0, 130, 0, 0, 385, 2]),                      # prompts without tokens
    (5, 1, 64, [513, 64]),
    (2, 2, 256, [200, 1, 64, 63, 65, 500]),
    (8, 1, 256, [129]),
    (6, 2, 128, [1000]),
    (4, 1, 64, [i % 7 for i in range(100)]),                 # more prompts than a warp has lanes
]
IDS = [str(i) for i in range(len(SHAPES))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_causal(ops, dtype, shape):
    heads, kv, dim, lens = shape
    q, k, v, cu = inputs(lens, heads, kv, dim, dtype, seed=len(lens), lead=3, tail=2)
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5, out=out)
    assert got is out and ops.device_status()[0] == 0
    check(got, q, k, v, cu, dim ** -0.5)
    assert bool((got[:3] == 7).all()) and bool((got[cu[-1]:] == 7).all())


@pytest.mark.parametrize("cap,bias,prefix", [(5.0, False, None), (0.0, True, 1), (20.0, True, 2), (0.0, False, 2)])
@pytest.mark.parametrize("shape", SHAPES[2:8], ids=IDS[2:8])
def test_caps_biases_and_prefixes(ops, cap, bias, prefix, shape):
    heads, kv, dim, lens = shape
    q, k, v, cu = inputs(lens, heads, kv, dim, torch.bfloat16, seed=heads)
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if bias else None
    pre = None
    if prefix == 1:
        pre = torch.tensor([max(1, n // 3) for n in lens], dtype=torch.int32, device="cuda")
    elif prefix == 2:     # everything, nothing, more than the prompt has, something in the middle of a block
        pre = torch.tensor([[n, 0, n + 1000, 150, -5][i % 5] for i, n in enumerate(lens)], dtype=torch.int32, device="cuda")
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5, softcap=cap, alibi_slopes=slopes,
                           prefix_lens=pre)
    check(got, q, k, v, cu, dim ** -0.5, cap, slopes, pre)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prompts_and_growing_maxima(ops, dtype):
    """Keys that grow along the prompt: the running maximum is passed by more than 2^8 again and again."""
    heads, kv, dim, lens = 4, 2, 128, [2500, 700]
    q, k, v, cu = inputs(lens, heads, kv, dim, dtype, seed=1)
    k = (k.float() * torch.linspace(0.1, 8, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5)
    # scores up to some 400 here: probabilities to 400 x 2^-21
    check(got, q, k, v, cu, dim ** -0.5, vmax=32.0)


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_that_are_not_positive(ops, scale):
    q, k, v, cu = inputs([200, 70], 2, 2, 64, torch.bfloat16, seed=2)
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), scale)
    check(got, q, k, v, cu, scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_another_prompts_infinities_and_nan_do_not_matter(ops, dim):
    lens = [100, 50, 300, 129]
    q, k, v, cu = (t.clone() if torch.is_tensor(t) else t for t in inputs(lens, 4, 2, dim, torch.bfloat16, seed=3, tail=60))
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    clean = ops.prefill_attn(q, k, v, cu_t, 0.1)
    for t in (q, k, v):
        t[cu[1]:cu[2]] = float("nan")
        t[cu[1]:cu[2], :, ::2] = float("inf")
        t[cu[4]:] = float("nan")
    got = ops.prefill_attn(q, k, v, cu_t, 0.1)
    for b in (0, 2, 3):
        assert torch.equal(got[cu[b]:cu[b + 1]], clean[cu[b]:cu[b + 1]])
    k[cu[2] + 200:cu[3]] = float("nan")     # keys that earlier tokens do not see
    again = ops.prefill_attn(q, k, v, cu_t, 0.1)
    assert torch.equal(again[cu[2]:cu[2] + 200], clean[cu[2]:cu[2] + 200])
    assert bool(torch.isnan(again[cu[2] + 200:cu[3]]).all())


def test_streams_graphs_and_views(ops):
    lens = [700, 33]
    q, k, v, cu = inputs(lens, 8, 4, 128, torch.bfloat16, seed=4)
    q = q.contiguous()
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    want = ops.prefill_attn(q, k, v, cu_t, 0.09)
    assert torch.equal(want, ops.prefill_attn(q, k.contiguous(), v.contiguous(), cu_t, 0.09))
    outs = [torch.zeros_like(want) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.prefill_attn(q, k, v, cu_t, 0.09, out=outs[0])
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        ops.prefill_attn(q, k, v, cu_t, 0.09, out=outs[1], stream=streams[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        for o in outs:
            o.zero_()


@pytest.mark.parametrize("lens", [[77, 400, 130, 600, 1, 0, 333], [0, 129, 0], [(i * 37) % 150 for i in range(32)],
                                  [(i * 37) % 90 for i in range(45)], [700, 700]], ids=["ragged", "one", "32", "45", "even"])
@pytest.mark.parametrize("heads,kv,dim,mod", [(32, 8, 64, True), (27, 9, 128, False), (40, 20, 128, True), (26, 13, 256, False)])
def test_more_tiles_than_sms_in_any_order(ops, heads, kv, dim, mod, lens):
    """One to a dozen CTAs per SM, pairs of heads and of row tiles, batches of more prompts than a warp has lanes."""
    q, k, v, cu = inputs(lens, heads, kv, dim, torch.float16, seed=heads, lead=5, tail=1)
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if mod else None
    pre = torch.tensor([i % 4 * 60 for i in range(len(lens))], dtype=torch.int32, device="cuda") if mod else None
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5, softcap=15.0 if mod else 0.0,
                           alibi_slopes=slopes, prefix_lens=pre, out=out)
    check(got, q, k, v, cu, dim ** -0.5, 15.0 if mod else 0.0, slopes, pre)
    assert bool((got[:5] == 7).all()) and bool((got[cu[-1]:] == 7).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_two_rounds_of_shared_tiles(ops, dim):
    """Prompts long enough that one tile per CTA pays with up to two CTAs per SM, the longest first."""
    lens = [1152, 1300, 1, 2200]
    q, k, v, cu = inputs(lens, 7, 7, dim, torch.bfloat16, seed=dim, lead=2)
    slopes = torch.rand(7, device="cuda")
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5, alibi_slopes=slopes)
    check(got, q, k, v, cu, dim ** -0.5, 0.0, slopes)


@pytest.mark.parametrize("dim", [64, 128])
def test_few_tiles_whose_blocks_of_keys_two_warpgroups_share(ops, dim):
    """Growing and falling keys: the maximum lies in an even or an odd block, or moves; one to twelve blocks."""
    for n, factor in ((1500, lambda t: t * 8), (1500, lambda t: (1 - t) * 8), (1281, lambda t: 1 + 7 * (t > 0.9)),
                      (129, lambda t: 1 + 0 * t), (256, lambda t: 1 + 7 * (t < 0.5))):
        q, k, v, cu = inputs([n], 4, 1, dim, torch.bfloat16, seed=n)
        k = (k.float() * factor(torch.linspace(0, 1, n, device="cuda"))[:, None, None]).bfloat16()
        got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5)
        # scores up to some 400 here: probabilities to 400 x 2^-21
        check(got, q, k, v, cu, dim ** -0.5, vmax=32.0)


def test_warps_of_a_tile_that_are_a_block_apart(ops):
    """Head size 256, whose warps may be a block ahead of one another: rows of one warp whose maximum grows often, the others' not."""
    q, k, v, cu = inputs([2000], 32, 16, 256, torch.float16, seed=32, lead=5, tail=1)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    q = q.clone()
    q[5::3] *= 4
    for _ in range(3):
        check(ops.prefill_attn(q, k, v, cu_t, 0.0625), q, k, v, cu, 0.0625, vmax=32.0)


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (27, 9, 128), (4, 1, 128), (3, 3, 64), (16, 8, 256)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_score_buffers_are_written_again_behind_the_products_that_read_them(ops, heads, kv, dim, cap):
    """Up to 18 blocks of keys whose probabilities lie over the scores: the formula's values, and the same bits every time."""
    q, k, v, cu = inputs([2200, 700], heads, kv, dim, torch.bfloat16, seed=dim)
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    got = ops.prefill_attn(q, k, v, cu_t, dim ** -0.5, softcap=cap)
    check(got, q, k, v, cu, dim ** -0.5, cap)
    for _ in range(20):
        assert torch.equal(ops.prefill_attn(q, k, v, cu_t, dim ** -0.5, softcap=cap), got)


@pytest.mark.parametrize("heads,kv", [(4, 2), (24, 12), (27, 9)])      # few tiles, pairs of heads, pairs of row tiles
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_capped_scores_that_a_token_does_not_see_do_not_change_its_bits(ops, dim, heads, kv):
    """Scores within the cap in the prompts that are looked at; far beyond it, infinite or NaN in the others and behind."""
    lens = [100, 50, 300, 129]
    q, k, v, cu = (t.clone() if torch.is_tensor(t) else t for t in inputs(lens, heads, kv, dim, torch.float16, seed=3, tail=60))
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    call = lambda: ops.prefill_attn(q, k, v, cu_t, 0.1, softcap=50.0)
    clean = call()
    for t in (q, k):
        t[cu[1]:cu[2]] *= 100
        t[cu[4]:] *= 100
    for value in (None, float("inf"), float("nan")):
        if value is not None:
            q[cu[1]:cu[2]] = value
            k[cu[4]:] = value
        got = call()
        for b in (0, 2, 3):
            assert torch.equal(got[cu[b]:cu[b + 1]], clean[cu[b]:cu[b + 1]]), (value, b)
    k[cu[2] + 200:cu[3]] *= 100             # keys that earlier tokens do not see (a warp has the rows 192 .. 223)
    assert torch.equal(call()[cu[2]:cu[2] + 192], clean[cu[2]:cu[2] + 192])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_within_and_beyond_the_cap_side_by_side(ops, dim):
    """Rows of one warp of which every third has scores up to some ten times the cap."""
    q, k, v, cu = inputs([400, 37, 129], 6, 2, dim, torch.bfloat16, seed=dim)
    q = q.clone()
    q[::3] *= 32
    slopes = torch.rand(6, device="cuda") / 8
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5, softcap=10.0, alibi_slopes=slopes)
    check(got, q, k, v, cu, dim ** -0.5, 10.0, slopes)


@pytest.mark.parametrize("heads,kv", [(27, 9), (16, 16), (9, 3)])
@pytest.mark.parametrize("cap,bias,prefix", [(0.0, False, False), (20.0, False, False), (0.0, True, True), (20.0, True, True)])
@pytest.mark.parametrize("lens", [[300, 1, 513, 700, 256, 897], [129, 255, 385, 1024, 640], [1600, 1300, 130, 2100]], ids=["a", "b", "c"])
def test_pairs_of_row_tiles_of_head_size_64_with_unequal_ends(ops, heads, kv, cap, bias, prefix, lens):
    """Two tiles of one head whose blocks of keys differ in number, the second one without rows (n % 256 in 1 .. 128) or with some."""
    q, k, v, cu = inputs(lens, heads, kv, 64, torch.bfloat16, seed=heads + len(lens), lead=1)
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if bias else None
    pre = torch.tensor([[0, n, 200, 130, n // 2, n + 7][i % 6] for i, n in enumerate(lens)], dtype=torch.int32, device="cuda") if prefix else None
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.125, softcap=cap, alibi_slopes=slopes, prefix_lens=pre)
    assert ops.device_status()[0] == 0
    check(got, q, k, v, cu, 0.125, cap, slopes, pre)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (32, 8, 128), (4, 2, 256)])
@pytest.mark.parametrize("cap", [3e4, 1e6, 1e9])
def test_caps_far_above_the_scores(ops, heads, kv, dim, cap):
    """The polynomial is off by 2^-18 of a score there: 3e-5 of scores up to 16, of which the bound has 5e-5 of the largest value."""
    q, k, v, cu = inputs([300, 37, 700], heads, kv, dim, torch.float16, seed=dim)
    q, k = q.clamp(-4, 4), k.clamp(-2, 2)
    got = ops.prefill_attn(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), dim ** -0.5 / 2, softcap=cap)
    check(got, q, k, v, cu, dim ** -0.5 / 2, cap)
