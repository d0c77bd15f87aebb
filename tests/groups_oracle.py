"""Float64 forms of attention over shared prefixes, of decode attention over pages and its weights, with bounds on what the kernels may be off.

Bounds count roundings at half a step relative to the value: bf16 2^-8, f16 2^-11.  Float32 arithmetic (scores, exponentials, sums) is given 2^-16 of each
term: a score of 128 products is off by at most 128 * 2^-24 * sum |q k| * scale, sum |q k| * scale <= 60 for the tests' inputs, and so is 2^score by 2^-11 at the very worst
and 2^-16 with the errors' square root of 128; the tests' tolerances for weights use the former, those of bf16 results are far above either."""
import math

import torch

BF16, F16, F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -16


def attend(q, k, v, seen, scale, dout=None):
    """q [n, D], k and v [m, D] float64, seen [n, m].  (out, bound of out [, dq, dk, dv, their bounds]) for weights in bf16."""
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    o, a = p @ v, p @ v.abs()
    bound = (BF16 + F32) * (a + o.abs())
    if dout is None:
        return o, bound
    dp, delta = dout @ v.t(), (dout * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # of the weights' rounding in out, and of out's, through delta; of float32 in p
    e = (dout.abs() * (bound + BF16 * o.abs())).sum(-1, keepdim=True)
    eds = BF16 * ds.abs() + p * e + F32 * p * (dp.abs() + delta.abs() + (dout.abs() @ v.abs().t()))
    dq, dk, dv = ds @ k * scale, ds.t() @ q * scale, p.t() @ dout
    bounds = (eds @ k.abs() * scale, eds.t() @ q.abs() * scale, (BF16 + F32) * (p.t() @ dout.abs()))
    return o, bound, dq, dk, dv, *bounds


def packed(q, k, v, groups, scale, dout=None):
    """groups: [[prefix length, length, ...], ...] of consecutive sequences.  {name: (value, bound)}; rows of no sequence are 0 with bound 0."""
    q, k, v = (x.double() for x in (q, k, v))
    share = q.shape[1] // k.shape[1]
    out = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for lens in groups:
        parts, row = [], at
        for i, n in enumerate(lens):
            parts.append((row, n, 0 if i == 0 else lens[0]))
            row += n
        for row0, n, extra in parts:
            if n == 0:
                continue
            own = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
            seen = torch.cat([own.new_ones(n, extra), own], 1)
            idx = torch.cat([torch.arange(at, at + extra, device=q.device), torch.arange(row0, row0 + n, device=q.device)])
            for h in range(q.shape[1]):
                rows, kh = slice(row0, row0 + n), h // share
                r = attend(q[rows, h], k[idx, kh], v[idx, kh], seen, scale, None if dout is None else dout[rows, h].double())
                out["out"][0][rows, h], out["out"][1][rows, h] = r[0], r[1]
                if dout is not None:
                    out["dq"][0][rows, h], out["dq"][1][rows, h] = r[2], r[5]
                    for name, d, b in (("dk", r[3], r[6]), ("dv", r[4], r[7])):
                        out[name][0][idx, kh] += d
                        out[name][1][idx, kh] += b
        at = row
    return out


def page_rows(st, table, n):
    """Keys and values [Hkv, n, D] in float64 of the first n tokens of a page table (bf16 pages, or e4m3 with scales and values transposed)"""
    pages = table[:(n + 15) // 16].long()
    k, v = st["k"][pages], st["v"][pages]
    if st["ks"] is not None:
        k = k.view(torch.float8_e4m3fn).double() * st["ks"][pages].double()[..., None]
        v = v.reshape(*v.shape[:2], 128, 16).view(torch.float8_e4m3fn).double().transpose(2, 3) * st["vs"][pages].double()[..., None]
    return tuple(x.double().transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, v))


def decode_row(q, k, v, scale, fp8):
    """q [Hq, D], k and v [Hkv, n, D]: (out, bound, weights [Hkv, n] summed over a kv head's query heads, their bound)"""
    q = q.double().view(k.shape[0], -1, q.shape[-1])
    n = k.shape[1]
    if n == 0:
        return torch.zeros(q.shape[0] * q.shape[1], q.shape[2], dtype=torch.float64, device=q.device), 0.0, q.new_zeros(k.shape[0], 0), q.new_zeros(k.shape[0], 0)
    p = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
    o, a = p @ v, p @ v.abs()
    # weights in bf16; or, times the values' scales and at least 2^8, in f16, whose steps are 2^-24 where it is denormal
    bound = (F16 + F32) * a + BF16 * o.abs() + n * 2.0 ** -25 * 448.0 / 256.0 if fp8 else (BF16 + F32) * (a + o.abs())
    worst = (q.abs() @ k.abs().transpose(1, 2)).amax() * scale * 128 * 2.0 ** -24 * 2 + 2.0 ** -20
    return o.flatten(0, 1), bound.flatten(0, 1), p.sum(1), p.sum(1) * worst
