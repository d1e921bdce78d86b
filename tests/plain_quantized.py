"""Plain implementations of a cache in 8 bits, of attention over it and of token log probabilities, for the tests: loops over
sequences, blocks and heads on the CPU, codes in the formula's own 32-bit arithmetic, everything else in 64 bits."""
import math

import torch

PAGE, BLOCK = 64, 16
TINY = 2.0 ** -126
STEP = float(torch.tensor(1.0, dtype=torch.float32) / torch.tensor(127.0, dtype=torch.float32))


def turned(x, cos, sin, style):
    """x [.., size] float32 with its first 2 * len(cos) channels rotated; every product and sum rounded once."""
    rot = 2 * cos.numel()
    y = x.clone()
    if rot == 0:
        return y
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if style == 0 else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    if style == 0:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, w
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, w
    return y


def put(codes, scales, rows, start, pages):
    """rows [n, heads, size] float32 into positions start.. of a sequence with these pages; codes [pages, heads, 64, size] and
    scales [pages, heads, 4] change in place."""
    n, heads, _ = rows.shape
    for base in range(start // BLOCK * BLOCK, start + n, BLOCK):
        lo, hi = max(base, start), min(base + BLOCK, start + n)
        if lo >= hi:
            continue
        page, block = int(pages[base // PAGE]), base % PAGE // BLOCK
        for h in range(heads):
            new = rows[lo - start:hi - start, h]
            fine = bool(torch.isfinite(new).all())
            had = scales[page, h, block].clone() if lo > base else torch.zeros(())
            s = torch.nan_to_num(new, nan=0.0, posinf=0.0, neginf=0.0).abs().max() * torch.tensor(STEP)
            s = torch.maximum(torch.where(s < TINY, 0.0, s), had)
            if not fine or bool(torch.isnan(had)):
                s = torch.tensor(math.nan)
            inverse = 1.0 / s if bool(s > 0) else torch.zeros(())
            tile = codes[page, h, base % PAGE:base % PAGE + BLOCK]
            if bool(s > had):
                tile[:lo - base] = torch.round(tile[:lo - base].float() * (had * inverse)).to(torch.int8)
            new = torch.nan_to_num(new, nan=0.0, posinf=0.0, neginf=0.0) if not bool(s > 0) else new
            tile[lo - base:hi - base] = torch.round(new * inverse).to(torch.int8)
            scales[page, h, block] = s


def values(codes, scales, pages, n):
    """float32 [n, heads, size]: what the first n positions of a sequence with these pages hold."""
    out = [codes[int(pages[p // PAGE]), :, p % PAGE].float() * scales[int(pages[p // PAGE]), :, p % PAGE // BLOCK][:, None] for p in range(n)]
    return torch.stack(out) if out else torch.zeros(0, codes.shape[1], codes.shape[3])


def attend(q, k, v, start, *, scale, window=0, chunk=0, unit, step):
    """q [n, heads, hd] (positions start..), k, v [start + n, kv, .] float64 -> (result, bound) [n, heads, v_hd].  `bound`: how far an
    implementation may be that rounds weights, values and results to relative `unit` each and whose scores are off by `step`
    times sum |q k| scale: a score's error is a relative error of its weight, which enters numerator and denominator."""
    n, heads, _ = q.shape
    kv = k.shape[1]
    out, bound = torch.zeros(n, heads, v.shape[2], dtype=torch.float64), torch.zeros(n, heads, v.shape[2], dtype=torch.float64)
    for t in range(n):
        pos = start + t
        low = max(0, pos - window + 1) if window else 0
        low = max(low, pos - pos % chunk) if chunk else low
        for h in range(heads):
            keys, vals = k[low:pos + 1, h // (heads // kv)], v[low:pos + 1, h // (heads // kv)]
            p = torch.softmax(keys @ q[t, h] * scale, dim=0)
            worst = float((keys.abs() @ q[t, h].abs()).max()) * scale * step
            out[t, h] = p @ vals
            bound[t, h] = (3 * unit + 2 * worst + len(p) * 2.0 ** -24) * (p @ vals.abs())
    return out, bound


def logprobs(x, targets, top):
    """(logprob, entropy, ids, their log probabilities) of one row in 64 bits; ids by value, then by id."""
    x = x.double().cpu()
    if bool(torch.isnan(x).any()) or not bool(torch.isfinite(x.max())):
        logp, entropy = torch.full_like(x, math.nan), math.nan
    else:
        logp = torch.log_softmax(x, dim=0)
        entropy = float(-(logp.exp() * logp.clamp(min=-1e30)).sum())
    order = sorted(range(len(x)), key=lambda i: (-math.inf if math.isnan(x[i]) else -float(x[i]), i))[:top] if top and len(x) < 2000 else \
        torch.sort(x, descending=True, stable=True)[1][:top].tolist()
    one = float(logp[targets]) if 0 <= targets < len(x) else math.nan
    return one, entropy, order, logp[order]
