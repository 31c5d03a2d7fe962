"""Plain 64-bit forms of the attention path's operators, one token and one head at a time: what the tests compare with."""
import math

import torch


def e4m3(byte_tensor):
    return byte_tensor.view(torch.float8_e4m3fn).double()


def to_e4m3(x):
    """Nearest E4M3 values as bytes, saturating."""
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def scale_of(amax: float) -> float:
    if amax == 0:
        return 2.0 ** -100
    s = 2.0 ** -100
    while amax > 448 * s:
        s *= 2
    return s


def rotated(row, pos, rotary, base, yarn=1.0):
    """row [heads, dim] in 64 bits."""
    out, half = row.double().clone(), rotary // 2
    for i in range(half):
        a = pos * base ** (-2.0 * i / rotary) * yarn
        c, s = math.cos(a), math.sin(a)
        x, y = row[:, i].double(), row[:, i + half].double()
        out[:, i], out[:, i + half] = x * c - y * s, y * c + x * s
    return out


def places(cu, lens, tables, block_size, blocks):
    """(token, position, block or None, offset) of every token that is somebody's."""
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            pos = length - n + i
            if pos < 0:
                continue
            j = pos // block_size
            blk = int(tables[b][j]) if j < len(tables[b]) else -1
            yield cu[b] + i, pos, (blk if 0 <= blk < blocks else None), pos % block_size


def attention(q, k, v, scale, cap=0.0, slopes=None, seen=None, pos=None):
    """q [n, heads, dim] over k / v [m, kv_heads, dim]; seen [n, m] or None; pos: position of each query (default: the last n)."""
    n, heads, dim = q.shape
    m, kv, _ = k.shape
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    if m == 0:
        return out
    pos = torch.arange(m - n, m, device=q.device) if pos is None else pos
    far = (pos[:, None] - torch.arange(m, device=q.device)[None, :]).abs().double()
    for h in range(heads):
        g = h // (heads // kv)
        s = q[:, h].double() @ k[:, g].double().T * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * far
        if seen is not None:
            s = s.masked_fill(~seen, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, g].double()
    return out
