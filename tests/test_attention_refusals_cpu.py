"""What the cache appends, the 8-bit and scored decode attention and the prompt attention refuse, without a GPU: the C entry
points check before any device work, the Python ones before the C call."""
import pytest
import torch

from inference_b200 import _capi, ops

NAN, INF = float("nan"), float("inf")


def append(fp8=False, **kw):
    a = dict(q_out=16, q_out_stride=1024, k_out=16, k_out_stride=256, k_cache=16, v_cache=16, q=16, q_stride=1024, k=16, k_stride=256,
             v=16, v_stride=256, tables=16, lens=16, cu=16, dt=2, tokens=4, batch=2, heads=8, kv_heads=2, dim=128, rotary=128, block=16,
             blocks=10, per=4, base=1e4, yarn=1.0, k_scales=16, v_scales=16)
    a.update(kw)
    head = [a["q_out"], a["q_out_stride"], a["k_out"], a["k_out_stride"], a["k_cache"], a["v_cache"]]
    tail = [a[n] for n in ("q", "q_stride", "k", "k_stride", "v", "v_stride", "tables", "lens", "cu", "dt", "tokens", "batch", "heads",
                           "kv_heads", "dim", "rotary", "block", "blocks", "per", "base", "yarn")] + [None]
    if fp8:
        return _capi.lib.inferop_rope_append_kv_fp8(*head, a["k_scales"], a["v_scales"], *tail)
    return _capi.lib.inferop_rope_append_kv(*head, *tail)


def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")


@pytest.mark.parametrize("fp8", [False, True])
def test_appends(fp8):
    no_gpu()
    assert append(fp8) == _capi.ERR_NO_DEVICE          # a well-formed call gets as far as the device
    assert append(fp8, k_out=None, k_out_stride=0) == _capi.ERR_NO_DEVICE
    assert append(fp8, cu=None, tokens=2) == _capi.ERR_NO_DEVICE
    assert append(fp8, rotary=0) == _capi.ERR_NO_DEVICE
    for bad in (dict(tokens=0), dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(dim=96), dict(rotary=-2), dict(rotary=130),
                dict(rotary=63), dict(block=0), dict(blocks=0), dict(per=0), dict(cu=None), dict(base=0.0), dict(base=NAN), dict(base=INF),
                dict(yarn=NAN), dict(yarn=INF), dict(q_stride=1023), dict(k_stride=255), dict(v_stride=0), dict(q_out_stride=-1),
                dict(k_out_stride=255)):
        assert append(fp8, **bad) == _capi.ERR_SHAPE, bad
    for bad in (-1, 3):
        assert append(fp8, dt=bad) == _capi.ERR_DTYPE
    assert append(fp8, per=1 << 28) == _capi.ERR_LIMIT
    assert append(fp8, tokens=1 << 31) == _capi.ERR_LIMIT
    for name in ("q", "k", "v", "q_out", "k_cache", "v_cache", "tables", "lens"):
        assert append(fp8, **{name: None}) == _capi.ERR_POINTER, name
    for bad in (dict(k_cache=24), dict(v_cache=8), dict(tables=18), dict(lens=17), dict(cu=18), dict(q=17), dict(k=19), dict(v=17),
                dict(k_out=17), dict(q_out=17), dict(q=18, dt=0)):
        assert append(fp8, **bad) == _capi.ERR_POINTER, bad
    if fp8:
        assert append(True, block=24) == _capi.ERR_SHAPE
        assert append(True, k_scales=18) == append(True, v_scales=17) == _capi.ERR_POINTER
        assert append(True, k_scales=None) == _capi.ERR_POINTER and append(True, v_scales=None) == _capi.ERR_POINTER


def test_scored_and_8_bit_decode():
    no_gpu()
    lib = _capi.lib

    def scored(dt=2, cap=5.0, heads=8):
        return lib.inferop_paged_attn_decode_scored(16, 16, 16, 16, 16, 16, dt, 1, heads, 4, 128, 16, 4, 0.1, cap, None, None)

    def fp8(dt=2, cap=0.0, heads=8, dim=128, block=16, blocks=10, scales=16, cache=16, per=4):
        return lib.inferop_paged_attn_decode_fp8(16, 16, cache, 16, scales, 16, 16, 16, dt, 1, heads, 4, dim, block, blocks, per, 0.1, cap,
                                                 None, None)

    assert scored() == scored(dt=0) == fp8() == fp8(dt=1) == fp8(block=48) == _capi.ERR_NO_DEVICE
    for cap in (-1.0, NAN, INF, 1e-40):   # (0.1 / 1e-40 is no number of fp32's)
        assert scored(cap=cap) == fp8(cap=cap) == _capi.ERR_SHAPE
    assert scored(heads=6) == fp8(heads=6) == _capi.ERR_SHAPE
    assert scored(dt=3) == fp8(dt=3) == fp8(dt=0) == _capi.ERR_DTYPE
    assert fp8(dim=32) == fp8(block=8) == fp8(block=0) == fp8(blocks=0) == _capi.ERR_SHAPE
    assert fp8(scales=18) == _capi.ERR_POINTER
    assert fp8(scales=None) == fp8(cache=None) == fp8(cache=24) == _capi.ERR_POINTER
    assert fp8(block=1 << 20, blocks=1 << 11) == fp8(per=1 << 28) == _capi.ERR_LIMIT


def test_prompt_attention():
    no_gpu()

    def call(out=16, qs=1024, ks=512, vs=512, os=1024, q=16, cu=16, dt=2, tokens=4, batch=1, heads=8, kv=4, dim=128, cap=0.0):
        return _capi.lib.inferop_prefill_attn(out, os, q, qs, 16, ks, 16, vs, cu, None, dt, tokens, batch, heads, kv, dim, 0.1, cap, None,
                                              None)

    assert call() == call(dt=1) == call(qs=1536) == _capi.ERR_NO_DEVICE
    for bad in (dict(tokens=0), dict(batch=0), dict(heads=6), dict(dim=96), dict(cap=-1.0), dict(cap=NAN), dict(cap=1e-40), dict(qs=1016), dict(ks=504),
                dict(vs=504), dict(os=1016)):
        assert call(**bad) == _capi.ERR_SHAPE, bad
    assert call(dt=0) == call(dt=3) == _capi.ERR_DTYPE
    for bad in (dict(q=None), dict(out=None), dict(cu=None), dict(cu=18), dict(q=24), dict(qs=1028), dict(os=1025)):
        assert call(**bad) == _capi.ERR_POINTER, bad
    assert call(tokens=1 << 31) == _capi.ERR_LIMIT


def test_python_calls_refuse_tensors_that_are_not_on_a_gpu_or_have_other_types():
    z = torch.zeros
    q, k, cache = z(4, 8, 64), z(4, 2, 64), z(10, 16, 2, 64)
    tables, lens = z(2, 4, dtype=torch.int32), z(2, dtype=torch.int32)
    byte, scales = z(10, 16, 2, 64, dtype=torch.uint8), z(10, 2)
    h = q.bfloat16()
    for f in (lambda: ops.rope_append_kv(q, k, k, cache, cache, tables, lens, 64),
              lambda: ops.rope_append_kv(q[0], k, k, cache, cache, tables, lens, 64),
              lambda: ops.rope_append_kv(q.double(), k, k, cache, cache, tables, lens, 64),
              lambda: ops.rope_append_kv_fp8(q, k, k, byte, byte, scales, scales, tables, lens, 64),
              lambda: ops.paged_attn_decode(q, cache, cache, tables, lens, 0.1, softcap=5.0),
              lambda: ops.paged_attn_decode_fp8(h, byte, byte, scales, scales, tables, lens, 0.1),
              lambda: ops.paged_attn_decode_fp8(q, byte, byte, scales, scales, tables, lens, 0.1),
              lambda: ops.prefill_attn(h, k.bfloat16(), k.bfloat16(), lens, 0.1),
              lambda: ops.prefill_attn(q, k, k, lens, 0.1)):
        with pytest.raises(ValueError):
            f()


def test_native_calls_leave_what_is_not_plain_to_the_general_form():
    fast = _capi.fast
    assert fast.rope_append(*[None] * 14) is None
    assert fast.paged_attn_decode_scored(*[None] * 10) is None
    assert fast.prefill_attn(*[None] * 8) is None
    assert fast.prefill_attn(1, 2) is None


def test_decode_lists_queries_and_outputs_off_their_elements():
    """Every form of the decode attention, plain scores included: refused on the host, not a misaligned address on the device."""
    no_gpu()

    def call(form, dt=2, out=16, q=16, tables=16, lens=16, slopes=16):
        head, tail = [out, q, 16, 16], [tables, lens, dt, 1, 8, 4, 128, 16]
        if form == "plain":
            return _capi.lib.inferop_paged_attn_decode(*head, *tail, 4, 0.1, None)
        if form == "scored":
            return _capi.lib.inferop_paged_attn_decode_scored(*head, *tail, 4, 0.1, 0.0, slopes, None)
        return _capi.lib.inferop_paged_attn_decode_fp8(*head, 16, 16, *tail, 10, 4, 0.1, 0.0, slopes, None)

    for form in ("plain", "scored", "fp8"):
        assert call(form) == call(form, out=18, q=22) == _capi.ERR_NO_DEVICE
        for bad in (dict(tables=18), dict(tables=17), dict(lens=18), dict(lens=19), dict(q=17), dict(out=21)):
            assert call(form, **bad) == _capi.ERR_POINTER, (form, bad)
        if form != "plain":
            assert call(form, slopes=18) == _capi.ERR_POINTER
        if form != "fp8":
            assert call(form, dt=0, out=20, q=24) == _capi.ERR_NO_DEVICE
            assert call(form, dt=0, q=18) == call(form, dt=0, out=18) == _capi.ERR_POINTER


def test_caps_whose_units_fp32_cannot_hold():
    """Above 1e30 the cap to base 2, or a score in units of it, leaves fp32's range (3e38 gave NaN, 1e38 equal weights)."""
    no_gpu()
    lib = _capi.lib
    for cap, want in ((1e30, _capi.ERR_NO_DEVICE), (2e30, _capi.ERR_SHAPE), (1e38, _capi.ERR_SHAPE), (3e38, _capi.ERR_SHAPE)):
        assert lib.inferop_paged_attn_decode_scored(16, 16, 16, 16, 16, 16, 2, 1, 8, 4, 128, 16, 4, 0.1, cap, None, None) == want
        assert lib.inferop_paged_attn_decode_fp8(16, 16, 16, 16, 16, 16, 16, 16, 2, 1, 8, 4, 128, 16, 10, 4, 0.1, cap, None, None) == want
        assert lib.inferop_prefill_attn(16, 1024, 16, 1024, 16, 512, 16, 512, 16, None, 2, 4, 1, 8, 4, 128, 0.1, cap, None, None) == want
