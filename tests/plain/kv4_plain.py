"""A cache in 4 bits and the attention over it, plainly: 64-bit arithmetic, one group, one token, one head after the other."""
import math

import torch

PAGE = 64


def encode(x):
    """float64 [..., d] -> codes [..., d], a and b (bfloat16 as float64) [..., d / 32]."""
    codes, scales, mins = torch.zeros(x.shape, dtype=torch.int64), [], []
    for g in range(x.shape[-1] // 32):
        part = x[..., 32 * g:32 * g + 32]
        low, high = part.min(-1).values, part.max(-1).values
        a = ((high - low) * (16.0 / 15.0)).to(torch.bfloat16).double()
        b = (low - a).to(torch.bfloat16).double()
        bad = ~torch.isfinite(part).all(-1) | (part.abs().amax(-1) > 2.0 ** 127) | ~torch.isfinite(a)
        a, b = torch.where(bad, 0.0, a), torch.where(bad, math.nan, b)
        c = torch.round((part - b[..., None]) * 16.0 / a[..., None] - 16.0).clamp(0, 15)
        codes[..., 32 * g:32 * g + 32] = torch.where((a == 0)[..., None], 0.0, c).long()
        scales.append(a)
        mins.append(b)
    return codes, torch.stack(scales, -1), torch.stack(mins, -1)


def decode(codes, a, b):
    """The values as float64 (each a bfloat16 number)."""
    a, b = a.repeat_interleave(32, -1), b.repeat_interleave(32, -1)
    return (b + a * (1.0 + codes.double() / 16.0)).to(torch.bfloat16).double()


def page_bytes(keys, values):
    """(codes, a, b) of keys and of values, codes [64, d]: the bytes of one key head's part of a page."""
    out = []
    d = keys[0].shape[1]
    for t in range(PAGE):
        for w in range(d // 8):
            word = sum(int(keys[0][t, 8 * w + i]) << 4 * i for i in range(8))
            word = (word << 3 | word >> 29) & 0xFFFFFFFF
            out += [word >> 8 * i & 255 for i in range(4)]
    for t in range(PAGE):
        row = []
        for i in range(d // 2):
            byte = int(values[0][t, 2 * i]) | int(values[0][t, 2 * i + 1]) << 4
            row.append((byte << 3 | byte >> 5) & 255)
        turn = {64: 0, 128: t // 4 % 2, 192: 0, 256: t % 2 + 2 * (t // 4 % 2)}[d]
        for p in range(d // 64):
            out += row[32 * (p ^ turn):32 * (p ^ turn) + 32]
    head = torch.tensor(out, dtype=torch.uint8)
    scales = [torch.stack([a, b], -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten() for _, a, b in (keys, values)]
    return torch.cat([head] + scales)


def project(x, n_heads, n_kv, d, q_w, k_w, eps, cos, sin):
    """float64 [n, (n_heads + 2 n_kv) d] -> q, k, v float64 [n, heads, d], normed and rotated."""
    x = x.view(x.shape[0], n_heads + 2 * n_kv, d)
    q, k, v = x[:, :n_heads], x[:, n_heads:n_heads + n_kv], x[:, n_heads + n_kv:]

    def turn(y, w):
        if w is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        if cos is not None:
            a, b, c, s = y[..., :d // 2], y[..., d // 2:], cos.double()[:, None], sin.double()[:, None]
            y = torch.cat([a * c - b * s, b * c + a * s], -1)
        return y
    return turn(q, q_w), turn(k, k_w), v


def attention(q, keys, values, start, scale):
    """q float64 [new, heads, d] at positions start .., keys and values float64 [kv_heads, length, d].  Returns the result, and per row the weighted sum
    of |v| and the largest sum of |q k| scale: what errors are measured by."""
    new, H, d = q.shape
    group = H // keys.shape[0]
    out, size, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(new, H, 1, dtype=torch.float64)
    for i in range(new):
        end = start + i + 1
        for h in range(H):
            k, v = keys[h // group, :end], values[h // group, :end]
            p = torch.softmax(k @ q[i, h] * scale, 0)
            out[i, h], size[i, h] = p @ v, p @ v.abs()
            reach[i, h] = (k.abs() @ q[i, h].abs()).max() * abs(scale)
    return out, size, reach
