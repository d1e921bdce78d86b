"""How far attention that reads 8-bit codes itself may be from 64 bits: a bound from the roundings that it makes, per row and channel,
for the tests.  (`plain_quantized.attend` has a coarser one, for every way of attending to such a cache.)"""
import math

import torch

from plain_quantized import BLOCK, PAGE


def held(codes, scales, pages, n):
    """(codes, scale of each position) of the first n positions of a sequence, float64 [n, heads, size] and [n, heads]."""
    at = torch.arange(n)
    page = torch.as_tensor(pages).long()[at // PAGE]
    return codes[page, :, at % PAGE].double(), scales[page, :, at % PAGE // BLOCK].double()


def attend_codes(q, keys, values, start, *, scale, window=0, chunk=0, float32):
    """q [n, heads, hd] float64 (positions start..), keys and values as `held` gives them -> (result, bound) [n, heads, hd].

    The roundings: a row of q to whole numbers of 2^-16 (float32: 2^-24) of its largest one, half a unit each; scores, their
    arguments and powers in float32, a few roundings each; a weight times its value's scale to one float16 number, 2^-11 relative
    (float32: to two, 2^-22), and no finer than 2^-30 of the row's largest such product; float32 sums, in bfloat16 of codes
    that have 1152 added to them; the result to its type, 2^-8 (2^-24) relative."""
    (kc, ks), (vc, vs) = keys, values
    n, heads, hd = q.shape
    rep = heads // kc.shape[1]
    out, bound = torch.zeros(n, heads, hd, dtype=torch.float64), torch.zeros(n, heads, hd, dtype=torch.float64)
    for t in range(n):
        pos = start + t
        low = max(0, pos - window + 1) if window else 0
        low = max(low, pos - pos % chunk) if chunk else low
        for h in range(heads):
            k = (kc[low:pos + 1, h // rep] * ks[low:pos + 1, h // rep, None])
            c, s = vc[low:pos + 1, h // rep], vs[low:pos + 1, h // rep]
            row = q[t, h]
            score = k @ row * scale
            p = torch.softmax(score, dim=0)
            off = k.abs().sum(dim=1) * float(row.abs().max()) * (2.0 ** -23.9 if float32 else 2.0 ** -15.9) * scale
            off = off + score.abs() * 2.0 ** -20 + (k.abs() @ row.abs()) * scale * 2.0 ** -22
            slip = 2 * math.expm1(float(off.max())) + (2.0 ** -20 if float32 else 2.0 ** -10.9)
            w = p * s
            size = w @ c.abs()
            sums = (len(p) / BLOCK + 16) * 2.0 ** -23 * size + 2.0 ** -30 * float(w.max()) * c.abs().sum(dim=0)
            if not float32:
                sums = sums + 2.0 ** -21 * 1152 * w.sum()
            out[t, h] = w @ c
            bound[t, h] = slip * size + sums + (2.0 ** -22 if float32 else 2.0 ** -8) * out[t, h].abs()
    return out, bound


def attend_pages(q, keys, values, start, *, scale, window=0, chunk=0, apart):
    """The same for bfloat16 prompts, whose keys and values go by way of 16-bit pages: float16 numbers, 2^-11 relative and no finer than
    2^-32 of the sequence's largest scale, and weights to 2^-11, no finer than 2^-31 of the row's largest; or, where scales lie
    `apart`, all three to bfloat16's 2^-8."""
    (kc, ks), (vc, vs) = keys, values
    n, heads, hd = q.shape
    rep = heads // kc.shape[1]
    unit, page_floor, weight_floor = (2.0 ** -8, 0.0, 0.0) if apart else (2.0 ** -11, 2.0 ** -32, 2.0 ** -31)
    out, bound = torch.zeros(n, heads, hd, dtype=torch.float64), torch.zeros(n, heads, hd, dtype=torch.float64)
    for t in range(n):
        pos = start + t
        low = max(0, pos - window + 1) if window else 0
        low = max(low, pos - pos % chunk) if chunk else low
        for h in range(heads):
            k = kc[low:pos + 1, h // rep] * ks[low:pos + 1, h // rep, None]
            v = vc[low:pos + 1, h // rep] * vs[low:pos + 1, h // rep, None]
            row = q[t, h]
            score = k @ row * scale
            p = torch.softmax(score, dim=0)
            off = ((k.abs() @ row.abs()) * (1.01 * unit) + row.abs().sum() * page_floor * float(ks[:, h // rep].max())) * scale + score.abs() * 2.0 ** -20
            slip = 2 * math.expm1(float(off.max())) + 2.05 * unit + (len(p) + 32) * 2.0 ** -23
            out[t, h] = p @ v
            bound[t, h] = (slip * (p @ v.abs()) + weight_floor * float(p.max()) * v.abs().sum(dim=0) + page_floor * float(vs[:, h // rep].max())
                           + 2.0 ** -8 * out[t, h].abs())
    return out, bound
