"""The 8-bit cache in 64 bits on the CPU: its form, and attention over it.  Written from the definitions, without the framework."""
import math

import torch

LARGEST, MIN_EXP, NAN = 448.0, -119, 255
MOST = 240.0 * 2.0 ** 120                  # the largest number held: the next one is past the largest of 32 bits


def decode_table():
    out = torch.empty(256, dtype=torch.float64)
    for b in range(256):
        sign, e, m = -1.0 if b & 128 else 1.0, (b >> 3) & 15, b & 7
        out[b] = math.nan if b & 127 == 127 else sign * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return out


TABLE = decode_table()


def quantise(x):
    """(values of e4m3, exponent bytes) of rows x [..., dim]."""
    x = torch.where(torch.isfinite(x), x.double().clamp(-MOST, MOST), x.double())
    bad = ~torch.isfinite(x).all(-1)
    a = torch.where(bad, 0.0, x.abs().amax(-1))
    e = torch.full(a.shape, MIN_EXP)
    while bool((a > LARGEST * torch.exp2(e.double())).any()):
        e += (a > LARGEST * torch.exp2(e.double())).long()
    y = torch.where(bad[..., None], 0.0, x) / torch.exp2(e.double())[..., None]
    grid = torch.cat([TABLE[:127], TABLE[126:127]])                     # 0 .. 448 in order; the nearest of two neighbours
    at = torch.searchsorted(grid[:127].contiguous(), y.abs().contiguous()).clamp_max(126)
    low, high = grid[(at - 1).clamp_min(0)], grid[at]
    up = (high - y.abs() < y.abs() - low) | ((high - y.abs() == y.abs() - low) & (at % 2 == 0))     # (even: the last mantissa bit is 0)
    v = torch.where((at == 0) | up, high, low) * torch.sign(y)
    return v, torch.where(bad, NAN, e + 127)


def values(v, exps):
    """What e4m3 values and exponent bytes stand for."""
    return v * torch.where(exps == NAN, math.nan, torch.exp2(exps.double() - 127))[..., None]


def held(pages, exps, table_row, upto):
    """[positions, kv heads, dim] of one request; rows of a position without a page are not there (second result: which are)."""
    P = pages.shape[2]
    pos = torch.arange(upto)
    ids = table_row[pos // P].long()
    there = ids >= 0
    ids = ids.clamp_min(0)
    v = TABLE[pages.view(torch.uint8)[ids, :, pos % P].long()]
    return values(v, exps[ids, :, pos % P].long()), there


def attention(q, k, v, there, positions, heads, window, scale, softcap):
    """q [tokens, heads, dim], k and v [positions, kv heads, dim]; (results, sum of weights times |v|, the largest
    |scale| * sum |q_i k_i|), each [tokens, heads, dim] or a number."""
    out, mag, most = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0.0
    group = heads // k.shape[1]
    q = q.double()
    for t, p in enumerate(positions):
        lo = max(0, p - window + 1) if window else 0
        at = torch.arange(lo, p + 1)
        at = at[there[lo:p + 1]]
        if not at.numel():
            continue
        for h in range(heads):
            kk, vv = k[at, h // group], v[at, h // group]
            s = kk @ q[t, h] * scale
            most = max(most, float(torch.nan_to_num((kk.abs() @ q[t, h].abs()).amax() * abs(scale))))
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            w = torch.softmax(s, 0)
            out[t, h], mag[t, h] = w @ vv, w @ vv.abs()
    return out, mag, most
