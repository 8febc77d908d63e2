"""Plain implementation of the cache held in 4 bits, in float64 on the CPU: the rows' codes and numbers, the bytes of a pool, and
attention over them.  It shares no code with the package."""
import math

import torch


def bf16(x):
    """x (float64) rounded to the values of bfloat16 (through float32, whose own rounding only counts within 2^-24 of a border)."""
    return x.float().bfloat16().double()


def hold(x):
    """Rows x [..., hd] in float64 -> (codes int64, step, zero [..., 1])."""
    x = x.double()
    zero = bf16(x.amin(-1, keepdim=True))
    step = bf16((x.amax(-1, keepdim=True) - zero).clamp_min(0.0) / 15.0)
    code = torch.where(step > 0, torch.round((x - zero) / torch.where(step > 0, step, 1.0)), 0.0).clamp(0, 15).long()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, 0, code), torch.where(bad, math.nan, step), torch.where(bad, math.nan, zero)


def held(x):
    """What the rows stand for."""
    code, step, zero = hold(x)
    return zero + step * code.double()


def pool_bytes(k, v):
    """k, v [pages, kv heads, page size, hd] -> uint8 [pages, kv heads, page size * (hd + 8)]."""
    out = []
    numbers = []
    for x in (k, v):
        code, step, zero = hold(x)
        out.append((code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8).flatten(2))
        numbers += [step, zero]
    params = torch.cat(numbers, dim=-1).float().bfloat16().contiguous().view(torch.uint8)
    return torch.cat(out + [params.flatten(2)], dim=-1).contiguous()


def rows_of(pool, page, hd):
    """uint8 pool (CPU) -> (k, v) float64 [pages, kv heads, page size, hd], by loops over the bytes' places."""
    P, nkv, _ = pool.shape
    got = []
    params = pool[..., page * hd:].reshape(P, nkv, page, 8)
    for j in range(2):
        codes = pool[..., j * page * hd // 2:(j + 1) * page * hd // 2].reshape(P, nkv, page, hd // 2).long()
        x = torch.zeros(P, nkv, page, hd, dtype=torch.float64)
        x[..., 0::2] = (codes % 16).double()
        x[..., 1::2] = (codes // 16).double()
        pair = params[..., 4 * j:4 * j + 4].contiguous().view(torch.bfloat16).double()
        got.append(pair[..., 1:2] + pair[..., 0:1] * x)
    return got


def sequence(rows, table_row, length):
    """[pages, kv heads, page, hd] -> [length, kv heads, hd] of the sequence with this list of pages."""
    page = rows.shape[2]
    pages = [int(p) for p in table_row[:-(-length // page)]]
    return torch.cat([rows[p].transpose(0, 1) for p in pages])[:length]


def attend(q, k, v, pos, scale, window=0):
    """One query [nh, hd] over k, v [T, nkv, hd] up to position pos; NaN rows count for those that see them only."""
    nh, nkv = q.shape[0], k.shape[1]
    lo = max(0, pos - window + 1) if window > 0 else 0
    out = torch.zeros(nh, v.shape[2], dtype=torch.float64)
    for h in range(nh):
        g = h // (nh // nkv)
        s = (k[lo:pos + 1, g].double() @ q[h].double()) * scale
        w = torch.softmax(s, 0)
        out[h] = w @ v[lo:pos + 1, g].double()
    return out
