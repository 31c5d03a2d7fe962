"""rope_append_kv and rope_append_kv_fp8 against plain 64-bit forms.

Tolerances: the fraction of a turn is rounded once to fp32 and sine and cosine are good to 2 ulp, so both are off by 2^-21 at
most, and a rotated value by (|x| + |y|) 2^-20 before its one rounding to its type (half of finfo.eps, relative)."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from attention_plain import e4m3, places, rotated, scale_of, to_e4m3

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    from inference_b200 import ops as _ops
    assert _ops.has_cuda() and _ops.device_sm_version(0) == 100, "needs a B200"
    return _ops


def case(dtype, new, lens, heads, kv_heads, dim, block, seed=0, fp8=False, lead=0, tail=0, single=False):
    """Inputs on the GPU; `lead` / `tail`: rows that are nobody's in front and behind."""
    g = torch.Generator().manual_seed(seed)
    batch, per = len(new), max(1, -(-max(lens) // block))
    blocks = batch * per + 2
    tokens = lead + sum(new) + tail
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g)
    qkv[:, heads, 1] *= 40
    qkv = qkv.to(dtype).cuda()
    tables = torch.randperm(blocks, generator=g)[: batch * per].to(torch.int32).view(batch, per)
    cu = [lead]
    for n in new:
        cu.append(cu[-1] + n)
    s = dict(q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:], tables=tables.cuda(),
             lens=torch.tensor(lens, dtype=torch.int32).cuda(), cu=None if single else torch.tensor(cu, dtype=torch.int32).cuda())
    shape = (blocks, block, kv_heads, dim)
    if fp8:
        for n in ("k", "v"):
            s[n + "_cache"] = torch.randint(0, 126, shape, generator=g, dtype=torch.uint8).cuda()
            s[n + "_scales"] = torch.exp2(torch.randint(-9, -4, (blocks, kv_heads), generator=g).float()).cuda()
    else:
        s["k_cache"], s["v_cache"] = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
    return s, cu


def call(ops, s, rotary, base=10000.0, yarn=1.0, **kw):
    args = [s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"]]
    if "k_scales" in s:
        return ops.rope_append_kv_fp8(*args, s["k_scales"], s["v_scales"], s["tables"], s["lens"], rotary, base=base, yarn_factor=yarn,
                                      cu_seqlens=s["cu"], **kw)
    return ops.rope_append_kv(*args, s["tables"], s["lens"], rotary, base=base, yarn_factor=yarn, cu_seqlens=s["cu"], **kw)


def check_rotated(got, x, pos, rotary, base, yarn, dtype):
    """got, x: [heads, dim] of one token."""
    want = rotated(x, pos, rotary, base, yarn)
    half, mag = rotary // 2, x.double().abs().clone()
    pair = mag[:, :half] + mag[:, half:rotary]
    mag[:, :half], mag[:, half:rotary] = pair, pair
    mag[:, rotary:] = 0
    f = torch.finfo(dtype)
    bound = mag * 2.0 ** -20 + want.abs() * (f.eps / 2) * (1 + 2.0 ** -10) + f.smallest_normal * f.eps / 2
    assert bool(((got.double() - want).abs() <= bound).all()), (pos, float((got.double() - want).abs().max()))


SHAPES = [
    # new tokens, lengths with them, heads, kv_heads, dim, block, rotary
    ([1], [1], 8, 2, 128, 16, 128),
    ([3, 17, 1, 40], [3, 30, 100, 41], 4, 4, 64, 16, 64),        # runs over block borders, into partly filled blocks
    ([33, 0, 64], [33, 5, 64], 6, 2, 256, 32, 64),               # a sequence without new tokens
    ([100, 20], [130, 20], 9, 3, 64, 48, 32),                    # several chunks of a block; a block size between powers of two
    ([5, 16], [21, 16], 2, 1, 128, 16, 0),                       # no rotation
    ([7], [300000], 2, 1, 64, 16, 64),                           # far positions
    ([6, 50], [70, 50], 3, 1, 64, 64, 20),                       # a rotary part that 16-byte pieces do not divide
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("fp8", [False, True])
def test_values_places_and_untouched_rows(ops, dtype, shape, fp8):
    new, lens, heads, kv, dim, block, rotary = shape
    s, cu = case(dtype, new, lens, heads, kv, dim, block, seed=sum(new), fp8=fp8, lead=2, tail=3)
    before = {n: s[n].cpu().clone() for n in s if n.endswith(("cache", "scales"))}
    tokens = s["q"].shape[0]
    q_out = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device="cuda")
    k_out = torch.full((tokens, kv, dim), 7.0, dtype=dtype, device="cuda")
    assert call(ops, s, rotary, base=500000.0, yarn=0.75, q_out=q_out, k_out=k_out) is q_out
    torch.cuda.synchronize()
    q, k, v, tables = s["q"].cpu(), s["k"].cpu(), s["v"].cpu(), s["tables"].cpu()
    q_got, k_got = q_out.cpu(), k_out.cpu()
    mine = torch.zeros(tokens, dtype=torch.bool)
    stored = {}
    for t, pos, blk, off in places(cu, lens, tables, block, before["k_cache"].shape[0]):
        mine[t] = True
        check_rotated(q_got[t], q[t], pos, rotary, 500000.0, 0.75, dtype)
        check_rotated(k_got[t], k[t], pos, rotary, 500000.0, 0.75, dtype)
        stored.setdefault(blk, []).append((off, t, pos))
    assert bool((q_got[~mine] == 7).all()) and bool((k_got[~mine] == 7).all())
    if not fp8:
        want_k, want_v = before["k_cache"], before["v_cache"]
        for blk, rows in stored.items():
            for off, t, _ in rows:
                want_k[blk, off], want_v[blk, off] = k_got[t], v[t]
        assert torch.equal(s["k_cache"].cpu(), want_k) and torch.equal(s["v_cache"].cpu(), want_v)
        return
    for name, x, turn in (("k", k, rotary), ("v", v, 0)):
        cache, scales = s[name + "_cache"].cpu(), s[name + "_scales"].cpu()
        old_cache, old_scales = before[name + "_cache"], before[name + "_scales"]
        for blk in range(cache.shape[0]):
            if blk not in stored:
                assert torch.equal(cache[blk], old_cache[blk]) and torch.equal(scales[blk], old_scales[blk])
                continue
            rows = stored[blk]
            first, last = min(r[0] for r in rows), max(r[0] for r in rows)
            assert torch.equal(cache[blk, last + 1:], old_cache[blk, last + 1:])     # what lies behind is left alone
            want = torch.stack([rotated(x[t], pos, turn, 500000.0, 0.75) for _, t, pos in rows])
            for h in range(kv):
                amax, got = float(want[:, h].abs().max()), float(scales[blk, h])
                if first > 0 and got == float(old_scales[blk, h]):
                    assert amax <= 448 * got * (1 + 2.0 ** -18)
                    assert torch.equal(cache[blk, :first, h], old_cache[blk, :first, h])
                else:
                    assert got in (scale_of(amax * (1 - 2.0 ** -18)), scale_of(amax * (1 + 2.0 ** -18)))
                    if first > 0:   # grown: the bytes before moved
                        assert got > float(old_scales[blk, h])
                        moved = to_e4m3(e4m3(old_cache[blk, :first, h]) * float(old_scales[blk, h]) / got)
                        assert torch.equal(cache[blk, :first, h], moved)
                # half a step of E4M3 (2^-4 relative, 2^-10 s below its normal range), beside the rotation's error (its
                # pair is below 2 x 448 s)
                val = torch.stack([e4m3(cache[blk, off, h].contiguous()) * got for off, _, _ in rows])
                bound = want[:, h].abs() * 2.0 ** -4 + got * 2.0 ** -10 + 896 * got * 2.0 ** -20
                assert bool(((val - want[:, h]).abs() <= bound).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_one_token_per_sequence_needs_no_list(ops, dtype, fp8):
    lens = [1, 16, 17, 33, 250, 0, 32]
    a, _ = case(dtype, [1] * 7, lens, 8, 2, 128, 16, seed=3, fp8=fp8, single=True)
    b = {n: t.clone() if t is not None else None for n, t in a.items()}
    b["cu"] = torch.arange(8, dtype=torch.int32, device="cuda")
    ka, kb = torch.zeros(7, 2, 128, dtype=dtype, device="cuda"), torch.zeros(7, 2, 128, dtype=dtype, device="cuda")
    qa, qb = torch.zeros(7, 8, 128, dtype=dtype, device="cuda"), torch.zeros(7, 8, 128, dtype=dtype, device="cuda")
    call(ops, a, 128, q_out=qa, k_out=ka)
    call(ops, b, 128, q_out=qb, k_out=kb)
    assert torch.equal(qa, qb) and torch.equal(ka, kb)
    for n in a:
        if n.endswith(("cache", "scales")):
            assert torch.equal(a[n], b[n]), n
    assert bool((qa[5] == 0).all()) and bool((qa[4] != 0).any())


@pytest.mark.parametrize("fp8", [False, True])
def test_token_by_token_gives_what_a_prompt_gives(ops, fp8):
    """Of the same values: 16-bit caches bit for bit; 8-bit ones have the last scale, and their bytes are within one further
    rounding of E4M3's subnormals."""
    n, heads, kv, dim = 41, 4, 2, 64
    s, _ = case(torch.bfloat16, [n], [n], heads, kv, dim, 16, seed=5, fp8=fp8)
    whole = {k: t.clone() for k, t in s.items()}
    q_whole = call(ops, whole, dim)
    for t in range(n):
        one = dict(s, q=s["q"][t:t + 1], k=s["k"][t:t + 1], v=s["v"][t:t + 1], cu=None,
                   lens=torch.tensor([t + 1], dtype=torch.int32, device="cuda"))
        assert torch.equal(call(ops, one, dim)[0], q_whole[t])
    for name in ("k", "v"):
        if not fp8:
            assert torch.equal(s[name + "_cache"], whole[name + "_cache"])
            continue
        assert torch.equal(s[name + "_scales"], whole[name + "_scales"])
        a, b = (e4m3(c[name + "_cache"].cpu()) for c in (s, whole))
        used = s["tables"].cpu()[0, : -(-n // 16)].long()
        a, b = a[used].flatten(0, 1)[:n], b[used].flatten(0, 1)[:n]
        # each move to another scale may round a subnormal by half a step of 2^-9; a handful of moves per block
        assert bool(((a - b).abs() <= (b.abs() < 2.0 ** -5) * 8 * 2.0 ** -10).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_entries_that_are_no_block_and_positions_beyond_the_table(ops, fp8):
    s, cu = case(torch.float16, [20, 30, 4], [20, 30, 2], 4, 2, 64, 16, seed=8, fp8=fp8)
    s["tables"][0, 1], s["tables"][1, 0] = -1, s["k_cache"].shape[0]
    s["lens"][1] = 45     # the last positions lie beyond the table (2 entries of 16)
    before = {n: s[n].clone() for n in s if n.endswith(("cache", "scales"))}
    q_out = torch.full((54, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    k_out = torch.full((54, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    call(ops, s, 64, q_out=q_out, k_out=k_out)
    q_got, lens = q_out.cpu(), [20, 45, 2]
    stored, mine = {}, set()
    for t, pos, blk, off in places(cu, lens, s["tables"].cpu(), 16, s["k_cache"].shape[0]):
        mine.add(t)
        check_rotated(q_got[t], s["q"][t].cpu(), pos, 64, 10000.0, 1.0, torch.float16)
        check_rotated(k_out[t].cpu(), s["k"][t].cpu(), pos, 64, 10000.0, 1.0, torch.float16)
        if blk is not None:
            stored.setdefault(blk, []).append(off)
    assert len(mine) == 52 and bool((q_out[50:52] == 7).all())    # two tokens more than their sequence is long
    changed = set()
    for blk in range(s["k_cache"].shape[0]):
        if not torch.equal(s["v_cache"][blk], before["v_cache"][blk]) or not torch.equal(s["k_cache"][blk], before["k_cache"][blk]):
            changed.add(blk)
    assert changed == set(stored)


def test_not_finite_values_set_no_scale(ops):
    s, _ = case(torch.bfloat16, [16], [16], 2, 2, 64, 16, seed=2, fp8=True)
    s["v"][3, 0, 5], s["v"][4, 0, 6], s["v"][5, 0, 7] = float("inf"), float("-inf"), float("nan")
    s["v"][:, 1] = 0
    call(ops, s, 64)
    blk = int(s["tables"][0, 0])
    v = s["v"][:, 0].float()
    amax = float(v[torch.isfinite(v)].abs().max())
    assert float(s["v_scales"][blk, 0]) == scale_of(amax) and float(s["v_scales"][blk, 1]) == 2.0 ** -100
    got = e4m3(s["v_cache"][blk, :, 0].cpu().contiguous())
    assert float(got[3, 5]) == 448 and float(got[4, 6]) == -448 and bool(torch.isnan(got[5, 7])) and int(torch.isnan(got).sum()) == 1
    assert bool((s["v_cache"][blk, :, 1] & 0x7F == 0).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_in_place_unaligned_rows_and_another_stream(ops, fp8):
    s, _ = case(torch.bfloat16, [30, 1], [30, 18], 4, 2, 64, 16, seed=4, fp8=fp8)
    want = {n: t.clone() for n, t in s.items()}
    k_want = torch.empty_like(want["k"], memory_format=torch.contiguous_format)
    q_want = call(ops, want, 64, k_out=k_want)
    # rows that begin at odd elements, tokens at an odd stride
    odd = torch.zeros(31, 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    odd[:, 1:] = torch.cat([s["q"], s["k"], s["v"]], 1).reshape(31, -1)
    rows = odd[:, 1:].unflatten(1, (8, 64))
    t = dict({n: x.clone() for n, x in s.items()}, q=rows[:, :4], k=rows[:, 4:6], v=rows[:, 6:])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(ops, t, 64, q_out=t["q"], k_out=t["k"], stream=stream)
    stream.synchronize()
    assert torch.equal(t["q"], q_want) and torch.equal(t["k"], k_want)
    for n in s:
        if n.endswith(("cache", "scales")):
            assert torch.equal(t[n], want[n]), n


def test_many_heads_many_sequences_and_a_replayed_graph(ops):
    lens = [(i * 7) % 90 + 1 for i in range(1500)]
    s, cu = case(torch.float16, [1] * 1500, lens, 70, 70, 64, 16, seed=6, fp8=True)
    ref = {n: t.clone() for n, t in s.items()}
    q_ref = call(ops, dict(ref, cu=None), 64)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q_ref)
    keep = {n: s[n].clone() for n in s if n.endswith(("cache", "scales"))}
    with torch.cuda.graph(graph):
        call(ops, s, 64, q_out=out)
    for n, t in keep.items():
        s[n].copy_(t)
    for _ in range(2):          # the second time the same tokens are stored again: nothing changes
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, q_ref)
        for n in keep:
            assert torch.equal(s[n], ref[n]), n


def test_angles_of_far_positions(ops):
    """A position of a million at the highest frequency: fp32 products of the two would be off by 0.03 rad."""
    pos = 1_000_000
    for dtype in TYPES:
        x = torch.zeros(1, 1, 64, dtype=dtype, device="cuda")
        x[..., 0] = 1
        cache = torch.zeros(1, 16, 1, 64, dtype=dtype, device="cuda")
        tables = torch.zeros(1, 70000, dtype=torch.int32, device="cuda")
        got = ops.rope_append_kv(x, x, x, cache, cache.clone(), tables, torch.tensor([pos + 1], dtype=torch.int32, device="cuda"), 64)
        check_rotated(got[0].cpu(), x[0].cpu(), pos, 64, 10000.0, 1.0, dtype)


def unaligned_first_call(dtype, rotary):
    """Rows at odd elements, heads of 128: against the 64-bit form (run in a process of its own, as its first append)."""
    from inference_b200 import ops
    s, cu = case(dtype, [20, 1], [20, 18], 4, 2, 128, 16, seed=rotary, fp8=True)
    odd = torch.zeros(21, 8 * 128 + 1, dtype=dtype, device="cuda")
    odd[:, 1:] = torch.cat([s["q"], s["k"], s["v"]], 1).reshape(21, -1)
    rows = odd[:, 1:].unflatten(1, (8, 128))
    s.update(q=rows[:, :4], k=rows[:, 4:6], v=rows[:, 6:])
    k_out = torch.zeros(21, 2, 128, dtype=dtype, device="cuda")
    q_got = call(ops, s, rotary, k_out=k_out).cpu()
    for t, pos, blk, off in places(cu, [20, 18], s["tables"].cpu(), 16, s["k_cache"].shape[0]):
        check_rotated(q_got[t], s["q"][t].cpu(), pos, rotary, 10000.0, 1.0, dtype)
        check_rotated(k_out[t].cpu(), s["k"][t].cpu(), pos, rotary, 10000.0, 1.0, dtype)
        scale = s["v_scales"][blk].cpu()[:, None].double()
        stored = e4m3(s["v_cache"][blk, off].cpu()) * scale
        want = s["v"][t].cpu().double()
        assert bool(((stored - want).abs() <= want.abs() * 2.0 ** -4 + scale * 2.0 ** -10).all())


@pytest.mark.parametrize("dtype,rotary", [("bfloat16", 128), ("float16", 128), ("bfloat16", 124), ("float16", 122)])
def test_unaligned_rows_of_128_in_the_first_call_of_a_process(dtype, rotary):
    """Shared memory just below 48 KB beside the kernel's own: whether it is granted must not depend on what ran before."""
    code = f"import test_kv_append_gpu as t, torch; t.unaligned_first_call(torch.{dtype}, {rotary})"
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.dirname(here)])
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=path), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32), (256, 48)])
def test_alignment_and_the_kind_of_cache_do_not_show_in_the_rotated_rows(ops, dtype, dim, block):
    """Caches of the operands' type and E4M3 ones, rows on 16-byte addresses and at odd elements: the same rotated bits."""
    new, lens, heads, kv = [70, 1, 33], [100, 9, 33], 6, 3
    results = []
    for fp8 in (False, True):
        s, _ = case(dtype, new, lens, heads, kv, dim, block, seed=dim, fp8=fp8)
        for odd in (False, True):
            t = {n: x.clone() for n, x in s.items()}
            if odd:
                wide = torch.zeros(104, (heads + 2 * kv) * dim + 1, dtype=dtype, device="cuda")
                wide[:, 1:] = torch.cat([s["q"], s["k"], s["v"]], 1).reshape(104, -1)
                rows = wide[:, 1:].unflatten(1, (heads + 2 * kv, dim))
                t.update(q=rows[:, :heads], k=rows[:, heads:heads + kv], v=rows[:, heads + kv:])
            k_out = torch.zeros(104, kv, dim, dtype=dtype, device="cuda")
            q = call(ops, t, dim, k_out=k_out)
            results.append((q, k_out))
            if odd:
                assert all(torch.equal(t[n], last[n]) for n in t if n.endswith(("cache", "scales")))
            last = t
    for q, k_out in results[1:]:
        assert torch.equal(q, results[0][0]) and torch.equal(k_out, results[0][1])
