"""The attention path as a serving program runs it: projections' output -> cache append -> attention over the prompt, then steps of
one token per sequence.  Every attention result is compared with the plain 64-bit form over what the append left (rotated queries,
cache rows); what the append leaves is the subject of test_kv_append_gpu.py.  And the refusals and give-up paths that need a GPU."""
import ctypes as C

import pytest
import torch

from attention_plain import attention, e4m3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from inference_b200 import ops as _ops
    assert _ops.has_cuda() and _ops.device_sm_version(0) == 100, "needs a B200"
    return _ops


def history(cache, scales, table, length):
    blocks = table.long()
    x = cache[blocks]
    x = e4m3(x) * scales[blocks][:, None, :, None].double() if scales is not None else x.double()
    return x.flatten(0, 1)[:length]


def near(got, want, size, dtype, probabilities_rounded):
    """One rounding of the output, half of eps each for rounded probabilities, 5e-5 for scores and sums in fp32 (values below 8)."""
    eps = torch.finfo(dtype).eps
    bound = eps / 2 * 1.02 * (want.abs() + (size if probabilities_rounded else 0)) + 4e-4
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,heads,kv,dim,cap,bias", [(torch.bfloat16, 8, 2, 128, 0.0, False), (torch.float16, 6, 3, 64, 20.0, True),
                                                         (torch.bfloat16, 4, 1, 256, 0.0, True)])
def test_prompts_then_steps(ops, dtype, heads, kv, dim, cap, bias, fp8):
    g = torch.Generator(device="cuda").manual_seed(dim)
    prompts, block, steps = [37, 1, 160, 16], 16, 18
    batch, per = len(prompts), -(-(max(prompts) + steps) // block)
    blocks = batch * per + 1
    tables = torch.randperm(blocks, device="cuda", generator=g)[: batch * per].to(torch.int32).view(batch, per)
    kind = torch.uint8 if fp8 else dtype
    k_cache, v_cache = (torch.full((blocks, block, kv, dim), 77 if fp8 else 7.0, dtype=kind, device="cuda") for _ in range(2))
    scales = [torch.full((blocks, kv), 3.0, device="cuda") for _ in range(2)] if fp8 else None
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if bias else None
    scale = dim ** -0.5

    def project(n):
        qkv = torch.randn(n, heads + 2 * kv, dim, device="cuda", generator=g).to(dtype)
        return qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]

    def store(q, k, v, lens, **kw):
        if fp8:
            return ops.rope_append_kv_fp8(q, k, v, k_cache, v_cache, *scales, tables, lens, dim, base=5e5, **kw)
        return ops.rope_append_kv(q, k, v, k_cache, v_cache, tables, lens, dim, base=5e5, **kw)

    cu = [0]
    for n in prompts:
        cu.append(cu[-1] + n)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    q, k, v = project(cu[-1])
    turned = torch.empty(cu[-1], kv, dim, dtype=dtype, device="cuda")
    q = store(q, k, v, lens, cu_seqlens=cu_t, k_out=turned)
    got = ops.prefill_attn(q, turned, v, cu_t, scale, softcap=cap, alibi_slopes=slopes)
    for b in range(batch):
        r = slice(cu[b], cu[b + 1])
        i = torch.arange(prompts[b], device="cuda")
        seen = i[None, :] <= i[:, None]
        near(got[r], attention(q[r], turned[r], v[r], scale, cap, slopes, seen, i),
             attention(q[r], turned[r], v[r].abs(), scale, cap, slopes, seen, i), dtype, True)
    for step in range(steps):
        lens += 1
        q, k, v = project(batch)
        q = store(q, k, v, lens)
        if fp8:
            got = ops.paged_attn_decode_fp8(q, k_cache, v_cache, *scales, tables, lens, scale, softcap=cap, alibi_slopes=slopes)
        else:
            got = ops.paged_attn_decode(q, k_cache, v_cache, tables, lens, scale, softcap=cap, alibi_slopes=slopes)
        if step % 6:
            continue
        for b in range(batch):
            n = prompts[b] + step + 1
            kk, vv = (history(c, scales[i] if fp8 else None, tables[b], n) for i, c in enumerate((k_cache, v_cache)))
            want = attention(q[b:b + 1], kk, vv, scale, cap, slopes, None, torch.tensor([n - 1], device="cuda"))
            near(got[b:b + 1], want, None, dtype, False)


def test_refusals_on_the_gpu_leave_the_outputs_alone(ops):
    from inference_b200 import _capi
    h = torch.zeros(6, 8, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(6, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    byte = torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device="cuda")
    scales, tables = torch.zeros(4, 2, device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    lens, cu = torch.ones(6, dtype=torch.int32, device="cuda"), torch.zeros(7, dtype=torch.int32, device="cuda")
    for error, f in [
            (ValueError, lambda: ops.rope_append_kv(h, k, k[:, :, :32], cache, cache, tables, lens, 64)),
            (ValueError, lambda: ops.rope_append_kv(h, k, k, cache, cache.float(), tables, lens, 64)),
            (ValueError, lambda: ops.rope_append_kv(h, k, k, cache, cache, tables, lens[:5], 64)),
            (ValueError, lambda: ops.rope_append_kv(h, k, k, cache, cache, tables, lens, 64, cu_seqlens=cu[:6])),
            (ValueError, lambda: ops.rope_append_kv(h, k, k, cache, cache, tables.long(), lens, 64)),
            (ValueError, lambda: ops.rope_append_kv(h.transpose(0, 1).contiguous().transpose(0, 1), k, k, cache, cache, tables, lens, 64)),
            (ops.InferopError, lambda: ops.rope_append_kv(h, k, k, cache, cache, tables, lens, 63)),
            (ops.InferopError, lambda: ops.rope_append_kv(h[:0], k[:0], k[:0], cache, cache, tables[:0], lens[:0], 64)),
            (ValueError, lambda: ops.rope_append_kv_fp8(h, k, k, byte, byte, scales[:3], scales, tables, lens, 64)),
            (ValueError, lambda: ops.rope_append_kv_fp8(h, k, k, cache, cache, scales, scales, tables, lens, 64)),
            (ops.InferopError, lambda: ops.rope_append_kv_fp8(h, k, k, byte.view(8, 8, 2, 64), byte.view(8, 8, 2, 64), scales.repeat(2, 1),
                                                              scales.repeat(2, 1), tables, lens, 64)),
            (ValueError, lambda: ops.paged_attn_decode(h, cache, cache, tables, lens, 0.1, alibi_slopes=scales[0])),
            (ops.InferopError, lambda: ops.paged_attn_decode(h, cache, cache, tables, lens, 0.1, softcap=-1.0)),
            (ValueError, lambda: ops.paged_attn_decode_fp8(h, byte, byte, scales, scales.half(), tables, lens, 0.1)),
            (ValueError, lambda: ops.paged_attn_decode_fp8(h, byte, byte[:3], scales, scales, tables, lens, 0.1)),
            (ValueError, lambda: ops.paged_attn_decode_fp8(h, byte, byte, scales, scales, tables, lens, 0.1, out=h[:5])),
            (ops.InferopError, lambda: ops.paged_attn_decode_fp8(h, byte, byte, scales, scales, tables, lens, 0.1, softcap=float("nan"))),
            (ValueError, lambda: ops.prefill_attn(h, k, k, cu.long(), 0.1)),
            (ValueError, lambda: ops.prefill_attn(h, k, k, cu, 0.1, prefix_lens=lens[:3])),
            (ValueError, lambda: ops.prefill_attn(h, k, k.half(), cu, 0.1)),
            (ops.InferopError, lambda: ops.prefill_attn(h, k, k, cu[:1], 0.1)),
            (ops.InferopError, lambda: ops.prefill_attn(h.view(-1)[4:4 + 5 * 512].view(5, 8, 64), k[:5], k[:5], cu[:2], 0.1))]:
        with pytest.raises(error):
            f()
    torch.cuda.synchronize()
    for t in (h, cache, byte, scales):
        assert bool((t == 0).all())


def test_lists_that_are_not_in_order_stay_in_bounds(ops):
    """Lengths and offsets that no caller means: whatever they give, nothing outside the tensors is touched."""
    h = torch.randn(40, 4, 64, device="cuda").bfloat16()
    k = torch.randn(40, 2, 64, device="cuda").bfloat16()
    guard = torch.full((20, 16, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cache, byte = guard[5:15], torch.zeros(20, 16, 2, 64, dtype=torch.uint8, device="cuda")[5:15]
    scales, tables = torch.ones(10, 2, device="cuda"), torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4) - 1
    for cu in ([0, 50, 20, 40], [-5, 10, 10, 41], [40, 0, 0, 0], [10, 20, 15, 39], [7, 7, 7, 7]):
        for lens in ([30, 10, 5], [-1, 2 ** 31 - 1, 0], [1000, 3, -2 ** 31]):
            cu_t, lens_t = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, lens))
            ops.rope_append_kv(h, k, k, cache, cache, tables, lens_t, 64, cu_seqlens=cu_t)
            ops.rope_append_kv_fp8(h, k, k, byte, byte, scales, scales, tables, lens_t, 64, cu_seqlens=cu_t)
            ops.prefill_attn(h, k, k, cu_t, 0.1, prefix_lens=lens_t)
            ops.paged_attn_decode_fp8(h[:3], byte, byte, scales, scales, tables, lens_t, 0.1)
    torch.cuda.synchronize()
    assert bool((guard[:5] == 7).all()) and bool((guard[15:] == 7).all()) and ops.device_status()[0] == 0


@pytest.mark.parametrize("what,sites", [("prefill", {0x141, 0x142, 0x241, 0x242, 0x243, 0x244, 0x341, 0x342}), ("decode", {0x351})])
def test_waits_run_out_cleanly_and_the_next_call_is_right(ops, what, sites):
    """No load is issued (a test hook), so nothing can arrive: every role gives up after a millisecond, and says where."""
    from inference_b200 import _capi
    q = torch.randn(200, 4, 128, device="cuda").bfloat16()
    k = torch.randn(200, 2, 128, device="cuda").bfloat16()
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    byte = torch.randint(0, 100, (13, 16, 2, 128), dtype=torch.uint8, device="cuda")
    scales, tables = torch.ones(13, 2, device="cuda") / 64, torch.arange(13, dtype=torch.int32, device="cuda").view(1, 13)
    lens = torch.tensor([200], dtype=torch.int32, device="cuda")
    if what == "prefill":
        call = lambda: ops.prefill_attn(q, k, k, cu, 0.1)
    else:
        call = lambda: ops.paged_attn_decode_fp8(q[:1], byte, byte, scales, scales, tables, lens, 0.1)
    want = call()
    assert ops.device_status()[0] == 0
    rec = (C.c_uint32 * 4)()
    try:
        ops.set_option("wait_budget_us", 1000)
        ops.set_option("debug_no_loads", 1)
        call()
        rc = _capi.lib.inferop_device_status(rec, 1)
        assert rc == _capi.ERR_DEVICE_WAIT and rec[0] in sites, (rc, [hex(v) for v in rec])
    finally:
        ops.set_option("debug_no_loads", 0)
        ops.set_option("wait_budget_us", 0)
    assert torch.equal(call(), want) and ops.device_status()[0] == 0


def test_two_devices_or_one(ops):
    """A tensor of another device than the first one's is refused before anything is launched."""
    h = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.prefill_attn(h, k, k.cpu(), torch.zeros(2, dtype=torch.int32, device="cuda"), 0.1)
    with pytest.raises(ValueError):
        ops.prefill_attn(h, k, k, torch.zeros(2, dtype=torch.int32), 0.1)


@pytest.mark.parametrize("fp8", [False, True])
def test_caches_whose_offsets_pass_32_bits(ops, fp8):
    """Blocks at the end of caches of more than 2^32 elements: append, then attention, against 64 bits."""
    kv, dim, block = 8, 256, 16
    blocks = 2 ** 32 // (block * kv * dim) + 8
    if torch.cuda.mem_get_info()[0] < 5 * blocks * block * kv * dim:
        pytest.skip("needs 22 GB")
    kind = torch.uint8 if fp8 else torch.bfloat16
    k_cache, v_cache = (torch.empty(blocks, block, kv, dim, dtype=kind, device="cuda") for _ in range(2))
    scales = [torch.zeros(blocks, kv, device="cuda") for _ in range(2)] if fp8 else None
    tables = torch.tensor([[blocks - 1, blocks - 3, 0], [blocks - 2, 1, blocks - 4]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(76, h, dim, generator=g, device="cuda").bfloat16() for h in (8, kv, kv))
    lens, cu = torch.tensor([40, 36], dtype=torch.int32, device="cuda"), torch.tensor([0, 40, 76], dtype=torch.int32, device="cuda")
    if fp8:
        q = ops.rope_append_kv_fp8(q, k, v, k_cache, v_cache, *scales, tables, lens, dim, cu_seqlens=cu)[[39, 75]]
        got = ops.paged_attn_decode_fp8(q, k_cache, v_cache, *scales, tables, lens, dim ** -0.5)
    else:
        q = ops.rope_append_kv(q, k, v, k_cache, v_cache, tables, lens, dim, cu_seqlens=cu)[[39, 75]]
        got = ops.paged_attn_decode(q, k_cache, v_cache, tables, lens, dim ** -0.5, softcap=50.0)
    for b, n in enumerate((40, 36)):
        kk, vv = (history(c, scales[i] if fp8 else None, tables[b], n) for i, c in enumerate((k_cache, v_cache)))
        near(got[b:b + 1], attention(q[b:b + 1], kk, vv, dim ** -0.5, 0.0 if fp8 else 50.0, None, None, None), None, torch.bfloat16, False)
        first = cu[b].item()
        if fp8:
            step = scales[1][tables[b].long()][:, None].expand(3, block, kv).reshape(-1, kv)[:n, :, None].double()
            bound = v[first:first + n].double().abs() / 16 + step * 2.0 ** -10    # half a step of E4M3, half a step of its subnormals
            assert bool(((vv - v[first:first + n].double()).abs() <= bound).all())
        else:
            assert torch.equal(vv, v[first:first + n].double())


@pytest.mark.parametrize("dim,cap", [(64, 0.0), (64, 20.0), (128, 0.0), (256, 0.0)])
def test_prompt_waits_run_out_cleanly_with_two_tiles_per_cta(ops, dim, cap):
    """More tiles than SMs: pairs of tiles (taking turns where scores are capped), or the form of the largest heads."""
    from inference_b200 import _capi
    q = torch.randn(300, 80, dim, device="cuda").half()
    k = torch.randn(300, 40, dim, device="cuda").half()
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    want = ops.prefill_attn(q, k, k, cu, 0.1, softcap=cap)
    rec = (C.c_uint32 * 4)()
    try:
        ops.set_option("wait_budget_us", 1000)
        ops.set_option("debug_no_loads", 1)
        ops.prefill_attn(q, k, k, cu, 0.1, softcap=cap)
        rc = _capi.lib.inferop_device_status(rec, 1)
        assert rc == _capi.ERR_DEVICE_WAIT and rec[0] in {0x241, 0x242, 0x341, 0x342}, (rc, [hex(v) for v in rec])
    finally:
        ops.set_option("debug_no_loads", 0)
        ops.set_option("wait_budget_us", 0)
    assert torch.equal(ops.prefill_attn(q, k, k, cu, 0.1, softcap=cap), want) and ops.device_status()[0] == 0


def test_native_calls_take_the_plain_forms_and_give_the_general_ones_bits(ops):
    from inference_b200 import _capi
    fast = _capi.fast
    if not fast.__name__.endswith("_fastcall"):
        pytest.skip("no native module for this torch")
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(50, h, 64, generator=g, device="cuda").bfloat16() for h in (6, 2, 2))
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens, cu = torch.tensor([30, 20], dtype=torch.int32, device="cuda"), torch.tensor([0, 30, 50], dtype=torch.int32, device="cuda")
    slopes = torch.rand(6, device="cuda")
    for fp8 in (False, True):
        results = []
        for form in (0, 1):
            kind = torch.uint8 if fp8 else torch.bfloat16
            kc, vc = (torch.zeros(8, 16, 2, 64, dtype=kind, device="cuda") for _ in range(2))
            ks, vs = (torch.zeros(8, 2, device="cuda") for _ in range(2)) if fp8 else (None, None)
            if form == 0:
                turned = fast.rope_append(q, k, v, kc, vc, ks, vs, tables, lens, 64, 1e4, 1.0, cu, None)
                one = turned[[29, 49]].contiguous()
                got = fast.paged_attn_decode_scored(one, kc, vc, ks, vs, tables, lens, 0.1, 5.0, slopes)
            else:
                append = ops.rope_append_kv_fp8 if fp8 else ops.rope_append_kv
                turned = append(q, k, v, kc, vc, *((ks, vs) if fp8 else ()), tables, lens, 64, cu_seqlens=cu, q_out=torch.empty_like(q))
                one = turned[[29, 49]].contiguous()
                decode = ops.paged_attn_decode_fp8 if fp8 else ops.paged_attn_decode
                got = decode(one, kc, vc, *((ks, vs) if fp8 else ()), tables, lens, 0.1, softcap=5.0, alibi_slopes=slopes,
                             out=torch.empty_like(one))
            results.append((turned, kc, vc, got))
        for a, b in zip(*results):
            assert torch.is_tensor(a) and torch.equal(a, b)
    assert torch.equal(fast.prefill_attn(q, k, v, cu, 0.1, 0.0, slopes, lens),
                       ops.prefill_attn(q, k, v, cu, 0.1, alibi_slopes=slopes, prefix_lens=lens, out=torch.empty_like(q)))
