"""Performance cases of the attention path's newer operators, from the projections to the attention's output.

  append      rope_append_kv: queries and keys rotated, keys and values stored in a paged cache of the operands' type
  append_fp8  rope_append_kv_fp8: the same into E4M3 caches with one scale per cache block and KV head
  decode_fp8  paged_attn_decode_fp8: one query token per sequence over such caches
  decode      paged_attn_decode with capped scores and / or a bias that falls with distance, caches of the operands' type
  prefill     prefill_attn: whole prompts, packed one behind the other, causal, with an optional prefix that every token of
              a prompt sees, a cap and a distance bias

`own` False: plain torch operations in 32 bits (positions, angles and quantised values in 64); True: the library's calls.
Caches, scales, block tables and lengths are what a serving program keeps; the projections' output is its input.  Sizes are
those of the benchmark and the tests (32 query heads over 8 KV heads of 128, blocks of 16 tokens) and such as lie around them.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_E4M3 = torch.float8_e4m3fn
_LOG2_MIN = -100          # the smallest scale of a block is 2^-100


def listed():
    return [
        # a small decode batch stores its tokens: all latency
        _append("append_decode_b8", 8, 1, 1000),
        # a batch of ragged prompts of a model with 28 heads, rotated keys kept for the attention over the prompts
        _append("append_prompts_t8192_h28_fp16", 5, 8192, 0, heads=28, kv_heads=4, dtype="fp16", k_out=True, ragged=True),
        # a decode batch appends into partly filled 8-bit blocks
        _append("append_fp8_decode_b128", 128, 1, 2000, fp8=True, ragged=True),
        # a long prompt into an 8-bit cache, half of the head rotated
        _append("append_fp8_prompt_t16384", 1, 16384, 0, fp8=True, rotary=64, k_out=True),
        # one short conversation on 8-bit caches: latency
        _decode("decode_fp8_b1_len777", 1, 777, fp8=True),
        # the steady state of a serving step: the caches' bytes bound it
        _decode("decode_fp8_b64_len4096", 64, 4096, fp8=True),
        # one very long document, all heads on one KV head: the work has to be split along the tokens
        _decode("decode_fp8_b1_len65536_mqa_fp16", 1, 65536, heads=8, kv_heads=1, dim=64, block=64, dtype="fp16", fp8=True),
        # capped scores, large heads, ragged lengths
        _decode("decode_cap_b32_len3000_d256", 32, 3000, heads=16, kv_heads=8, dim=256, cap=50.0, ragged=True),
        # a distance bias and no grouping of heads, a few sequences, fp32 caches
        _decode("decode_bias_b3_len2000_fp32", 3, 2000, heads=16, kv_heads=16, dim=64, bias=True, dtype="fp32", ragged=True),
        # two short prompts: latency
        _prefill("prefill_b2_t150", 2, 150, ragged=True),
        # one long prompt: the matrix products bound it
        _prefill("prefill_b1_t8192", 1, 8192),
        # packed prompts with a shared-prefix mask, capped scores and a distance bias, head size 64
        _prefill("prefill_b7_t6000_cap_bias_d64_fp16", 7, 6000, heads=16, kv_heads=4, dim=64, cap=30.0, bias=True, prefix=200,
                 dtype="fp16", ragged=True),
    ]


def _append(name, batch, tokens, past, heads=32, kv_heads=8, dim=128, rotary=None, block=16, dtype="bf16", fp8=False, k_out=False,
            ragged=False):
    """tokens: new tokens of all sequences together where past is 0, else each sequence's; past: tokens before them."""
    return dict(name=name, kind="append_fp8" if fp8 else "append", batch=batch, tokens=tokens, past=past, heads=heads,
                kv_heads=kv_heads, dim=dim, rotary=dim if rotary is None else rotary, block=block, dtype=dtype, k_out=k_out,
                ragged=ragged)


def _decode(name, batch, length, heads=32, kv_heads=8, dim=128, block=16, dtype="bf16", fp8=False, cap=0.0, bias=False, ragged=False):
    return dict(name=name, kind="decode_fp8" if fp8 else "decode", batch=batch, length=length, heads=heads, kv_heads=kv_heads,
                dim=dim, block=block, dtype=dtype, cap=cap, bias=bias, ragged=ragged)


def _prefill(name, batch, tokens, heads=32, kv_heads=8, dim=128, dtype="bf16", cap=0.0, bias=False, prefix=0, ragged=False):
    return dict(name=name, kind="prefill", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, cap=cap,
                bias=bias, prefix=prefix, ragged=ragged)


_HEADS = [(32, 8, 128), (28, 4, 128), (16, 16, 64), (16, 8, 256), (12, 4, 64), (8, 1, 128), (40, 8, 128), (9, 3, 64), (6, 2, 256)]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice(_HEADS)
    kind = rng.choice(["append", "append_fp8", "decode_fp8", "decode", "prefill"])
    shape = dict(heads=heads, kv_heads=kv_heads, dim=dim)
    ragged = rng.random() < 0.6
    if kind.startswith("append"):
        fp8 = kind == "append_fp8"
        dtype = rng.choice(["bf16", "fp16"] if fp8 else ["bf16", "fp16", "fp32"])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        block = rng.choice([16, 16, 32, 64])
        if rng.random() < 0.5:
            case = _append("", _log_uniform(rng, 1, 256), 1, _log_uniform(rng, 1, 4000), fp8=fp8, **shape, rotary=rotary, block=block,
                           dtype=dtype, ragged=ragged)
        else:
            batch = _log_uniform(rng, 1, 16)
            tokens = max(batch, _log_uniform(rng, 30, 8000))
            case = _append("", batch, tokens, 0, fp8=fp8, **shape, rotary=rotary, block=block, dtype=dtype, k_out=True, ragged=ragged)
    elif kind.startswith("decode"):
        fp8 = kind == "decode_fp8"
        batch = _log_uniform(rng, 1, 200)
        length = _log_uniform(rng, 1, min(60000, 64 * 4096 * 8 * 128 // 2 // (batch * kv_heads * dim)))
        plain = fp8 and rng.random() < 0.6
        cap = 0.0 if plain else rng.choice([0.0, 30.0, 50.0])
        bias = not plain and (cap == 0.0 or rng.random() < 0.3)
        dtype = rng.choice(["bf16", "fp16"] if fp8 else ["bf16", "fp16", "bf16", "fp32"])
        case = _decode("", batch, length, **shape, block=rng.choice([16, 16, 32, 64]), dtype=dtype, fp8=fp8, cap=cap, bias=bias,
                       ragged=ragged)
    else:
        batch = _log_uniform(rng, 1, 16)
        tokens = max(batch, _log_uniform(rng, 20, 5000))
        case = _prefill("", batch, tokens, **shape, dtype=rng.choice(["bf16", "fp16"]), cap=rng.choice([0.0, 0.0, 50.0]),
                        bias=rng.random() < 0.25, prefix=rng.choice([0, 0, 64, 100000]), ragged=ragged)
    del case["name"]
    return case


# --------------------------------------------------------------------------- lengths
def _fraction(i):
    """A spread of fractions in [0.04, 1), the same for every call."""
    return 0.04 + 0.96 * ((i * 2654435761 + 12345) % (1 << 32)) / float(1 << 32)


def _lengths(case):
    """Host lists: new tokens of each sequence (appends, prompts), and its length with them."""
    batch = case["batch"]
    if case["kind"].startswith("decode"):
        lens = [max(1, int(case["length"] * _fraction(i))) if case["ragged"] else case["length"] for i in range(batch)]
        return [1] * batch, lens
    if case.get("past", 0) > 0:
        past = [int(case["past"] * _fraction(i)) if case["ragged"] else case["past"] for i in range(batch)]
        return [case["tokens"]] * batch, [p + case["tokens"] for p in past]
    # one total over all sequences: every one has a token, the rest by fractions
    rest = case["tokens"] - batch
    weights = [_fraction(i) if case["ragged"] else 1.0 for i in range(batch)]
    ends = [int(rest * sum(weights[: i + 1]) / sum(weights)) for i in range(batch)]
    ends[-1] = rest
    new = [1 + ends[i] - (ends[i - 1] if i else 0) for i in range(batch)]
    return new, list(new)


def _pairs(case):
    """(query, key) pairs that a prompt's mask leaves."""
    return sum(sum(max(i + 1, min(n, case["prefix"])) for i in range(n)) for n in _lengths(case)[0])


def work(case):
    new, lens = _lengths(case)
    e, heads, kv, dim = _BYTES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    t, kind = sum(new), case["kind"]
    if kind.startswith("append"):
        read = t * (heads + 2 * kv) * dim * e
        stored = 2 * t * kv * dim * (1 if kind == "append_fp8" else e)
        return {"bytes": read + stored + t * heads * dim * e + (t * kv * dim * e if case["k_out"] else 0), "flops": 3 * t * (heads + kv) * case["rotary"]}
    if kind.startswith("decode"):
        c = 1 if kind == "decode_fp8" else e
        return {"bytes": 2 * sum(lens) * kv * dim * c + 2 * case["batch"] * heads * dim * e, "flops": 4 * sum(lens) * heads * dim}
    return {"bytes": 2 * t * (heads + kv) * dim * e, "flops": 4 * _pairs(case) * heads * dim}


# --------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _scale_log2(amax):
    """The exponent of the smallest power of two s with amax <= 448 s, no less than _LOG2_MIN."""
    mantissa, exponent = torch.frexp(amax.double())          # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    up = (mantissa > 0.875).to(exponent.dtype)               # 448 = 0.875 2^9
    return torch.where(amax > 0, exponent - 9 + up, torch.full_like(exponent, _LOG2_MIN)).clamp(min=_LOG2_MIN)


def _quantised_cache(x):
    """x [blocks, block, kv_heads, dim] -> E4M3 bytes and fp32 scales [blocks, kv_heads]."""
    log2 = _scale_log2(x.abs().amax(dim=(1, 3)))
    scales = torch.exp2(log2.float())
    q = (x / scales[:, None, :, None]).clamp(-448, 448).to(_E4M3)
    return q.view(torch.uint8), scales


def prepare(case, seed):
    g = _generator(seed)
    new, lens = _lengths(case)
    dt, heads, kv, dim = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=g)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s = dict(case=dict(case))
    if case["kind"] == "prefill":
        # as rope_append_kv leaves them: queries and keys on their own, values inside the projection's output
        t = sum(new)
        qkv = rand(t, heads + 2 * kv, dim).to(dt)
        s["q"], s["k"], s["v"] = (2 * qkv[:, :heads].float()).to(dt), qkv[:, heads:heads + kv].contiguous(), qkv[:, heads + kv:]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu"], s["scale"] = i32(cu), dim ** -0.5
        s["prefix"] = i32([min(case["prefix"], 10 * (i + 1) + case["prefix"] // 2) for i in range(len(new))]) if case["prefix"] else None
    else:
        block = case["block"]
        per = -(-max(lens) // block)
        blocks = case["batch"] * per + 3                    # a few blocks are nobody's
        s["tables"] = torch.randperm(blocks, device="cuda", generator=g)[: case["batch"] * per].to(torch.int32).view(case["batch"], per)
        s["lens"] = i32(lens)
        k, v = 1.5 * rand(blocks, block, kv, dim), rand(blocks, block, kv, dim)
        k[..., dim // 3] *= 4                               # a channel that stands out, as keys have them
        if case["kind"].endswith("fp8"):
            s["k_cache"], s["k_scales"] = _quantised_cache(k)
            s["v_cache"], s["v_scales"] = _quantised_cache(v)
        else:
            s["k_cache"], s["v_cache"] = k.to(dt), v.to(dt)
        if case["kind"].startswith("append"):
            t = sum(new)
            qkv = rand(t, heads + 2 * kv, dim)
            qkv[:, heads:heads + kv, dim // 3] *= 6
            qkv = qkv.to(dt)
            s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
            cu = [0]
            for n in new:
                cu.append(cu[-1] + n)
            s["cu"] = None if case["past"] > 0 and case["tokens"] == 1 else i32(cu)   # one token per sequence needs no list
            s["base"] = 500000.0
            s["k_out"] = torch.empty((t, kv, dim), dtype=dt, device="cuda") if case["k_out"] else None
        else:
            s["q"], s["scale"] = (1.5 * rand(case["batch"], heads, dim)).to(dt), dim ** -0.5
    if case.get("bias"):
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads).float()
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    kind = s["case"]["kind"]
    if kind.startswith("append"):
        return _run_append(s, kind.endswith("fp8"))
    if kind.startswith("decode"):
        return _own_decode(s, kind.endswith("fp8")) if own else _plain_decode(s)
    return _own_prefill(s) if own else _plain_prefill(s)


def _run_append(s, fp8):
    q = _own_append(s, fp8) if own else _plain_append(s, fp8)
    out = {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if fp8:   # the caches as the values that their bytes stand for, in units of the scales beside them
        out.update(k_cache=s["k_cache"].view(_E4M3), v_cache=s["v_cache"].view(_E4M3), k_scales=s["k_scales"], v_scales=s["v_scales"])
    if s["k_out"] is not None:
        out["k"] = s["k_out"]
    return out


def _own_append(s, fp8):
    from inference_b200 import ops
    if fp8:
        return ops.rope_append_kv_fp8(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["tables"],
                                      s["lens"], s["case"]["rotary"], base=s["base"], cu_seqlens=s["cu"], k_out=s["k_out"])
    return ops.rope_append_kv(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["case"]["rotary"],
                              base=s["base"], cu_seqlens=s["cu"], k_out=s["k_out"])


def _own_decode(s, fp8):
    from inference_b200 import ops
    cap, slopes = s["case"]["cap"], s.get("slopes")
    if fp8:
        return ops.paged_attn_decode_fp8(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["tables"], s["lens"],
                                         s["scale"], softcap=cap, alibi_slopes=slopes)
    return ops.paged_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["scale"], softcap=cap, alibi_slopes=slopes)


def _own_prefill(s):
    from inference_b200 import ops
    return ops.prefill_attn(s["q"], s["k"], s["v"], s["cu"], s["scale"], softcap=s["case"]["cap"], alibi_slopes=s.get("slopes"),
                            prefix_lens=s["prefix"])


def _token_places(s):
    """Of every new token: its sequence, its position, its cache block and the offset in it."""
    t = s["q"].shape[0]
    rows = torch.arange(t, device="cuda")
    if s["cu"] is None:
        seq, pos = rows, s["lens"].long() - 1
    else:
        cu = s["cu"].long()
        seq = torch.searchsorted(cu[1:], rows, right=True)
        pos = s["lens"].long()[seq] - (cu[seq + 1] - rows)
    block = s["k_cache"].shape[1]
    return pos, s["tables"].long()[seq, pos // block], pos % block


def _rotated(x, pos, rotary, base):
    """x [tokens, heads, dim], pairs (i, i + rotary / 2) turned by pos base^(-2 i / rotary); in 64 bits."""
    x, half = x.double(), rotary // 2
    angle = pos.double()[:, None] * base ** (-torch.arange(half, device="cuda", dtype=torch.float64) * 2 / rotary)
    c, n = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat([a * c - b * n, b * c + a * n, x[..., rotary:]], -1)


def _plain_append(s, fp8):
    dt, (pos, block, offset) = s["q"].dtype, _token_places(s)
    rotary, base = s["case"]["rotary"], s["base"]
    q, k = _rotated(s["q"], pos, rotary, base).to(dt), _rotated(s["k"], pos, rotary, base)
    if s["k_out"] is not None:
        s["k_out"].copy_(k.to(dt))
    if fp8:
        _plain_store_fp8(s["k_cache"], s["k_scales"], k, block, offset)
        _plain_store_fp8(s["v_cache"], s["v_scales"], s["v"].double(), block, offset)
    else:
        s["k_cache"][block, offset] = k.to(dt)
        s["v_cache"][block, offset] = s["v"]
    return q


def _plain_store_fp8(cache, scales, x, block, offset):
    """A block whose offset 0 is among the new tokens begins anew; the others keep their scale or grow it, and then the tokens
    before the new ones are quantised again."""
    size = cache.shape[1]
    places = torch.zeros(cache.shape[0], dtype=torch.int64, device="cuda")
    first = (places + size).scatter_reduce_(0, block, offset, "amin")
    amax = torch.zeros(scales.shape, device="cuda").scatter_reduce_(0, block[:, None].expand(-1, x.shape[1]), x.abs().amax(-1).float(), "amax")
    wanted = torch.where((first < size)[:, None], torch.exp2(_scale_log2(amax).float()), torch.zeros_like(scales))
    scale = torch.where((first == 0)[:, None], wanted, torch.maximum(scales, wanted))
    before = (torch.arange(size, device="cuda") < first[:, None])[:, :, None, None]
    values = cache.view(_E4M3).float()
    values = torch.where(before, values * scales[:, None, :, None] / scale[:, None, :, None], values)
    values[block, offset] = (x / scale[block][..., None]).float()
    cache.copy_(values.clamp(-448, 448).to(_E4M3).view(torch.uint8))
    scales.copy_(scale)


def _plain_decode(s):
    q, tables, lens, case = s["q"].float(), s["tables"].long(), s["lens"].long(), s["case"]
    batch, heads, dim = q.shape
    kv = s["k_cache"].shape[2]
    if case["kind"] == "decode_fp8":
        gather = lambda c, sc: (s[c].view(_E4M3)[tables].float() * s[sc][tables][:, :, None, :, None]).reshape(batch, -1, kv, dim)
    else:
        gather = lambda c, sc: s[c][tables].float().reshape(batch, -1, kv, dim)
    k, v = gather("k_cache", "k_scales"), gather("v_cache", "v_scales")
    x = torch.matmul(q.view(batch, kv, heads // kv, dim), k.permute(0, 2, 3, 1)).view(batch, heads, -1) * s["scale"]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    t = torch.arange(x.shape[-1], device="cuda")
    if case["bias"]:
        x = x - s["slopes"][:, None] * (lens[:, None] - 1 - t).float()[:, None, :]
    x = x.masked_fill((t >= lens[:, None])[:, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, kv, heads // kv, -1), v.permute(0, 2, 1, 3)).view(batch, heads, dim)
    return out.to(s["q"].dtype)


def _plain_prefill(s):
    case, cu = s["case"], s["cu"].long()
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    t, heads, dim = q.shape
    kv = k.shape[1]
    x = torch.matmul(q.permute(1, 0, 2).reshape(kv, -1, dim), k.permute(1, 2, 0)).view(heads, t, t) * s["scale"]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    rows = torch.arange(t, device="cuda")
    doc = torch.searchsorted(cu[1:], rows, right=True)
    at = rows - cu[doc]
    if case["bias"]:
        x = x - s["slopes"][:, None, None] * (at[:, None] - at[None, :]).abs().float()
    seen = at[None, :] <= at[:, None]
    if s["prefix"] is not None:
        seen = seen | (at[None, :] < s["prefix"].long()[doc][:, None])
    x = x.masked_fill(~(seen & (doc[:, None] == doc[None, :])), -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(kv, -1, t), v.permute(1, 0, 2)).view(heads, t, dim)
    return out.permute(1, 0, 2).contiguous().to(s["q"].dtype)


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lengths(case)
    return _exact_append(s, new, lens) if case["kind"].startswith("append") else \
        _exact_decode(s, lens) if case["kind"].startswith("decode") else _exact_prefill(s, new)


def _exact_turned(x, first, rotary, base):
    """x [n, heads, dim] at positions first, first + 1, ... as complex numbers times e^(i angle)."""
    half = rotary // 2
    z = torch.complex(x[..., :half], x[..., half:rotary])
    freq = torch.tensor([math.pow(base, -2.0 * i / rotary) for i in range(half)], device="cuda", dtype=torch.float64)
    angle = torch.outer(torch.arange(first, first + x.shape[0], device="cuda", dtype=torch.float64), freq)
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    return torch.cat([z.real, z.imag, x[..., rotary:]], dim=-1)


def _exact_append(s, new, lens):
    case, block = s["case"], s["case"]["block"]
    fp8 = case["kind"] == "append_fp8"
    tables = s["tables"].tolist()
    q, k = s["q"].double(), s["k"].double()
    out = {"q": torch.empty_like(q), "k_cache": None, "v_cache": None}
    if fp8:
        # (which side of a border of E4M3 a value falls to is not a question of 64 bits: the bytes have no value here)
        scales = {n: s[n].double().clone() for n in ("k_scales", "v_scales")}
        out.update(scales)
    else:
        out.update(k_cache=s["k_cache"].double(), v_cache=s["v_cache"].double())
    turned = torch.empty_like(k)
    row = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        first = length - n
        part = slice(row, row + n)
        out["q"][part] = _exact_turned(q[part], first, case["rotary"], s["base"])
        turned[part] = _exact_turned(k[part], first, case["rotary"], s["base"])
        for j in range(first // block, (length - 1) // block + 1):
            lo, hi = max(first, j * block), min(length, (j + 1) * block)
            rows = slice(row + lo - first, row + hi - first)
            where, at = tables[b][j], slice(lo - j * block, hi - j * block)
            for name, x in (("k", turned[rows]), ("v", s["v"][rows].double())):
                if fp8:
                    amax = x.abs().amax(dim=(0, 2))
                    wanted = torch.exp2(torch.ceil(torch.log2(torch.clamp(amax / 448, min=2.0 ** _LOG2_MIN))))
                    scales[name + "_scales"][where] = wanted if lo == j * block else torch.maximum(wanted, scales[name + "_scales"][where])
                else:
                    out[name + "_cache"][where, at] = x
        row += n
    if s["k_out"] is not None:
        out["k"] = turned
    return out


def _exact_attention(q, k, v, scale, cap, bias, seen):
    """q [n, heads, dim], k / v [m, kv_heads, dim]; bias [heads, n, m] or None; seen [n, m]: one head at a time."""
    out = torch.empty_like(q)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        x = (q[:, h] @ k[:, h // group].T) * scale
        if cap:
            x = cap * torch.tanh(x / cap)
        if bias is not None:
            x = x + bias(h)
        out[:, h] = torch.softmax(torch.where(seen, x, torch.full_like(x, -math.inf)), dim=-1) @ v[:, h // group]
    return out


def _exact_decode(s, lens):
    case, out = s["case"], []
    for b, length in enumerate(lens):
        blocks = s["tables"][b, : -(-length // case["block"])].long()
        cache = []
        for name in ("k", "v"):
            c = s[name + "_cache"][blocks]
            if case["kind"] == "decode_fp8":
                c = c.view(_E4M3).double() * s[name + "_scales"][blocks].double()[:, None, :, None]
            cache.append(c.double().flatten(0, 1)[:length])
        back = torch.arange(length - 1, -1, -1, device="cuda", dtype=torch.float64)[None, :]
        bias = (lambda h: -s["slopes"][h].double() * back) if case["bias"] else None
        out.append(_exact_attention(s["q"][b:b + 1].double(), *cache, s["scale"], case["cap"], bias, torch.ones_like(back, dtype=torch.bool)))
    return torch.cat(out)


def _exact_prefill(s, new):
    case, out, row = s["case"], [], 0
    prefix = [0] * len(new) if s["prefix"] is None else s["prefix"].tolist()
    for n, shared in zip(new, prefix):
        q, k, v = (s[x][row:row + n].double() for x in ("q", "k", "v"))
        i = torch.arange(n, device="cuda")
        seen = i[None, :] < torch.clamp(i + 1, min=shared)[:, None]
        far = (i[:, None] - i[None, :]).abs().double()
        bias = (lambda h: -s["slopes"][h].double() * far) if case["bias"] else None
        out.append(_exact_attention(q, k, v, s["scale"], case["cap"], bias, seen))
        row += n
    return torch.cat(out)
