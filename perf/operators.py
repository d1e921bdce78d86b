"""The operators that a cache in 8 bits and the scoring of tokens are timed on: quantising keys and values as they are
written and reading them back, attention over such a cache, and log probabilities of given tokens.

Every case is one pass through an operator, on tensors as the layers of a model hand them over.

    listed()            the cases
    draw(rng)           one more of the same ranges
    prepare(case, seed) what the caller has in hand: rows of a projection, a cache with its page table, logits
    run(state)          one pass, in plain torch operations (`own` false) or by the library's operator (`own` true)
    work(case)          the bytes and operations a pass cannot do without
    exact(case, seed)   the same results in 64 bits

The cache: pages of 64 positions, a page holding a dense [64, head size] tile of 8-bit codes for every kv head, and one
32-bit scale for every 16 positions of a head (keys and values apart).  A code c of a block with the scale s stands for
s * c.  Positions that are written into a block that already holds some keep its scale if they fit, and otherwise raise it
and round the block's older codes to the new one.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE, BLOCK = 64, 16
TINY = 2.0 ** -126                    # the smallest scale: a block that is all smaller than 127 of it holds zeros

# (query heads, kv heads, head size, rotary base, vocabulary) of the models that the library's own workloads name
SHAPES = {
    "qwen2-0.5b": (14, 2, 64, 1e6, 151936),
    "qwen2-1.5b": (12, 2, 128, 1e6, 151936),
    "qwen2.5-3b": (16, 2, 128, 1e6, 151936),
    "qwen2.5-7b": (28, 4, 128, 1e6, 152064),
    "llama3-8b": (32, 8, 128, 5e5, 128256),
    "lulisun-2k": (16, 4, 128, 1e4, 32000),
}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _write(name, model, dtype, n, shortest, longest, fresh, style="half"):
    """n sequences hold between shortest and longest positions after the step, the last `fresh` of each (all, if it has
    fewer) brought by it."""
    case = {"op": "write", "model": model, "dtype": dtype, "sequences": n, "shortest": shortest, "longest": longest,
            "fresh": fresh, "style": style}
    return dict(case, name=name) if name else case


def _read(name, model, dtype, n, shortest, longest):
    case = {"op": "read", "model": model, "dtype": dtype, "sequences": n, "shortest": shortest, "longest": longest}
    return dict(case, name=name) if name else case


def _attend(name, model, dtype, n, shortest, longest, fresh, window=0):
    case = {"op": "attend", "model": model, "dtype": dtype, "sequences": n, "shortest": shortest, "longest": longest,
            "fresh": fresh, "window": window}
    return dict(case, name=name) if name else case


def _score(name, rows, vocab, dtype, top, banned, room=0):
    case = {"op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "banned": banned, "room": room}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a server's ordinary step: one position for each of eight sequences of unequal length, most in the middle of a block
        _write("write step x8", "qwen2.5-7b", "bfloat16", 8, 128, 2048, 1),
        # a handful of short and odd prompts that arrived together
        _write("write prompts x7", "qwen2-1.5b", "bfloat16", 7, 9, 2047, 2047),
        # a conversation of a 32-bit run is taken up again with a few hundred tokens, in the middle of a block
        _write("write turn x2 f32", "qwen2-0.5b", "float32", 2, 1500, 1777, 333),
        # a long sequence is read back whole, to be moved or to be worked on by another kernel
        _read("read 31999", "llama3-8b", "bfloat16", 1, 31999, 31999),
        # one user waiting for the next token of a small model: the smallest call
        _attend("token 0.5b x1", "qwen2-0.5b", "bfloat16", 1, 437, 437, 1),
        # a full batch: 64 sequences of unequal length
        _attend("token 8b x64", "llama3-8b", "bfloat16", 64, 128, 2048, 1),
        # two users with a long document each
        _attend("token 7b x2 long", "qwen2.5-7b", "bfloat16", 2, 27000, 31999, 1),
        # drafted tokens are checked: a few new ones per sequence, in the 32-bit run, over a window
        _attend("drafts x4 f32", "qwen2-1.5b", "float32", 4, 700, 3001, 5, 1024),
        # a prompt of the benchmark's length, over what was just written
        _attend("prompt 7b 2048", "qwen2.5-7b", "bfloat16", 1, 2048, 2048, 2048),
        # the token that was just sampled for one user, with the alternatives that an interface shows
        _score("score 1", 1, 151936, "float32", 5, 0.0),
        # a batch whose grammar bans most tokens, logits in 16 bits and in rows wider than the vocabulary
        _score("score 61 banned", 61, 128256, "bfloat16", 20, 0.9, 64),
        # a text of 2,048 tokens is scored: every token but the first
        _score("score 2047", 2047, 152064, "float32", 1, 0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "score", "score"])
    model = rng.choice(sorted(SHAPES))
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "score":
        vocab = rng.choice([151936, 152064, 128256, 32000, _log(rng, 1000, 150000)])
        rows = _log(rng, 1, 2047)
        return _score(None, rows, vocab, rng.choice(["float32", "float32", "bfloat16"]), rng.choice([0, 1, 5, 20]),
                      rng.choice([0.0, 0.0, 0.3, 0.95]), rng.choice([0, 0, 1, 64]))
    if op == "read":
        total = _log(rng, 64, 31999)
        n = min(rng.choice([1, 2, 8]), total)
        return _read(None, model, dtype, n, max(1, total // n // rng.randint(1, 8)), total // n)
    if op == "write":
        if rng.random() < 0.5:
            longest = _log(rng, 16, 2048)
            return _write(None, model, dtype, _log(rng, 1, 64), max(1, longest // rng.randint(1, 12)), longest, rng.choice([1, 1, 2, 5]),
                          rng.choice(["half", "interleaved"]))
        total = _log(rng, 12, 4096)
        n = min(total, rng.choice([1, 2, 3, 5, 8]))
        longest = max(1, total // n)
        return _write(None, model, dtype, n, max(1, longest // rng.randint(1, 12)), longest, max(1, longest // rng.choice([1, 1, 3])),
                      rng.choice(["half", "interleaved"]))
    window = rng.choice([0, 0, 0, 512, 1024])
    kind = rng.choice(["token", "token", "few", "prompt"])
    if kind == "prompt":
        total = _log(rng, 12, 1700)
        n = min(total, rng.choice([1, 1, 2, 5]))
        longest = max(1, total // n)
        return _attend(None, model, dtype, n, max(1, longest // rng.randint(1, 12)), longest, longest if rng.random() < 0.7 else max(1, longest // 3),
                       window)
    total = _log(rng, 32, 64000)
    n = min(total // 32, _log(rng, 1, 64))
    longest = min(31999, total // n)
    return _attend(None, model, dtype, n, max(1, longest // rng.randint(1, 12)), longest, 1 if kind == "token" else rng.randint(2, 8), window)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Positions of every sequence behind the step and new ones among them: fixed by the case, the first one the longest."""
    rng = random.Random("%(sequences)d %(shortest)d %(longest)d" % case)
    after = [case["longest"]] + [rng.randint(case["shortest"], case["longest"]) for _ in range(case["sequences"] - 1)]
    return after, [min(n, case.get("fresh", n)) for n in after]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)


def _geometry(case, seed):
    """Host side: lengths, pages in no order, slots in no order."""
    after, fresh = _lengths(case)
    rng = random.Random(seed * 31 + 5)
    pages = [-(-n // PAGE) for n in after]
    pool = sum(pages) + 3
    numbers = list(range(pool))
    rng.shuffle(numbers)
    slots = list(range(len(after) + 2))
    rng.shuffle(slots)
    table = torch.zeros(len(slots), max(pages), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[slots[b], :n] = torch.tensor(numbers[at:at + n], dtype=torch.int32)
        at += n
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    start = [n - f for n, f in zip(after, fresh)]
    cu = [0]
    for f in fresh:
        cu.append(cu[-1] + f)
    pos = torch.cat([torch.arange(s, n, dtype=torch.int32) for s, n in zip(start, after)]).to(DEVICE)
    seq = torch.cat([torch.full((f,), b, dtype=torch.int32) for b, f in enumerate(fresh)]).to(DEVICE)
    return {"pool": pool, "page_table": table.to(DEVICE), "seq_slot": ints(slots[:len(after)]), "seq_start": ints(start),
            "seq_len": ints(after), "cu_seqlens": ints(cu), "token_pos": pos, "token_seq": seq, "n_tokens": cu[-1],
            "n_seqs": len(after), "max_new": max(fresh), "max_len": max(after), "total": sum(after)}


def _channels(g, kv, hd):
    """Channels of unequal size, as keys have them: a few several times the others."""
    return torch.exp(0.7 * torch.randn(kv, 1, hd, generator=g, device=DEVICE))


def _held(x):
    """Codes int8 and scales float32 of x [pages, kv heads, PAGE, head size], every block's scale its largest value / 127."""
    b = x.view(*x.shape[:2], PAGE // BLOCK, BLOCK, x.shape[3])
    scale = b.abs().amax(dim=(3, 4)) * (1.0 / 127.0)
    codes = torch.round(b * (1.0 / scale)[..., None, None])
    return codes.to(torch.int8).view(x.shape), scale.contiguous()


def _cache(geo, g, kv, hd):
    shape = (geo["pool"], kv, PAGE, hd)
    k, k_scale = _held(torch.randn(shape, generator=g, device=DEVICE) * _channels(g, kv, hd))
    v, v_scale = _held(torch.randn(shape, generator=g, device=DEVICE))
    return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


def _angles(hd, base, n, dtype):
    theta = base ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEVICE) / hd)
    angle = torch.arange(n, dtype=torch.float64, device=DEVICE)[:, None] * theta[None, :]
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


def _logits(case, g):
    """Rows as a head leaves them: a few tokens well above the rest; banned ones at minus infinity."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.empty(rows, vocab + case["room"], dtype=DTYPES[case["dtype"]], device=DEVICE)
    for at in range(0, rows, 256):
        n = min(256, rows - at)
        part = 2.5 * torch.randn(n, vocab, generator=g, device=DEVICE)
        part.scatter_add_(1, torch.randint(0, vocab, (n, 8), generator=g, device=DEVICE), 12.0 * torch.rand(n, 8, generator=g, device=DEVICE))
        if case["banned"]:
            part.masked_fill_(torch.rand(n, vocab, generator=g, device=DEVICE) < case["banned"], -math.inf)
        x[at:at + n, :vocab] = part
    if case["room"]:
        x[:, vocab:] = 0.0
    x = x[:, :vocab]
    # half of the tokens are the likeliest ones, as in a text that the model could have written
    best = x.float().argmax(dim=1)
    other = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
    target = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.5, best, other)
    return x, target.to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    if case["op"] == "score":
        s["logits"], s["targets"] = _logits(case, g)
        return s
    heads, kv, hd, base, _ = SHAPES[case["model"]]
    dtype = DTYPES[case["dtype"]]
    geo = _geometry(case, seed)
    s |= geo
    s |= _cache(geo, g, kv, hd)
    if case["op"] == "write":
        rows = torch.randn(geo["n_tokens"], heads + 2 * kv, hd, generator=g, device=DEVICE)
        rows[:, heads:heads + kv] *= _channels(g, kv, hd)[:, 0]
        s["qkv"] = rows.view(geo["n_tokens"], -1).to(dtype)
        s["q_out"] = torch.empty(geo["n_tokens"], heads * hd, dtype=dtype, device=DEVICE)
        s["cos"], s["sin"] = _angles(hd, base, geo["max_len"], torch.float32)
        # what is read back: the blocks that the step touches, whole sequences' rows one behind the other
        first = geo["seq_start"] // BLOCK * BLOCK
    else:
        first = torch.zeros_like(geo["seq_start"])
    if case["op"] == "attend":
        s["q"] = torch.randn(geo["n_tokens"], heads * hd, generator=g, device=DEVICE).to(dtype)
        s["out"] = torch.empty(geo["n_tokens"], heads * hd, dtype=dtype, device=DEVICE)
        return s
    count = geo["seq_len"] - first
    s["first"] = first
    s["cu_rows"] = torch.cat([count.new_zeros(1), count.cumsum(0, dtype=torch.int32)])
    n = int(s["cu_rows"][-1])
    s["row_seq"] = torch.repeat_interleave(torch.arange(geo["n_seqs"], dtype=torch.int32, device=DEVICE), count, output_size=n)
    s["row_pos"] = torch.arange(n, dtype=torch.int32, device=DEVICE) - s["cu_rows"][s["row_seq"]] + first[s["row_seq"]]
    s["k_rows"] = torch.empty(n, kv, hd, dtype=dtype, device=DEVICE)
    s["v_rows"] = torch.empty(n, kv, hd, dtype=dtype, device=DEVICE)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _turned(x, cos, sin, style):
    """x [T, heads, head size] float32 turned by rows of the tables [T, 1, head size / 2]."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if style == "interleaved" else (x[..., :half], x[..., half:])
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.stack([u, w], dim=-1).flatten(-2) if style == "interleaved" else torch.cat([u, w], dim=-1)


def _put(codes, scales, rows, block, offset, begun):
    """Rows [T, kv, hd] float32 into a cache, in place.  block [T]: number of each row's block (page * 4 + block of the page),
    offset [T]: its place there, begun [T]: whether the block holds earlier positions of the sequence."""
    pages, kv, _, hd = codes.shape
    per = PAGE // BLOCK
    at = block.long()
    top = torch.zeros(pages * per, kv, device=rows.device).index_reduce_(0, at, rows.abs().amax(dim=2), "amax")
    touched = torch.zeros(pages * per, 1, device=rows.device, dtype=torch.bool).index_fill_(0, at, True)
    kept = torch.zeros(pages * per, 1, device=rows.device, dtype=torch.bool).index_put_((at,), begun[:, None])
    old = scales.transpose(1, 2).reshape(pages * per, kv)
    had = torch.where(kept, old, torch.zeros_like(old))
    new = top * (1.0 / 127.0)
    new = torch.where(new < TINY, torch.zeros_like(new), new).maximum(had)
    inverse = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))
    # older codes of the touched blocks at the new scale
    held = codes.view(pages, kv, per, BLOCK, hd).permute(0, 2, 1, 3, 4).reshape(pages * per, kv, BLOCK, hd)
    again = torch.where((new > had)[..., None, None], torch.round(held.float() * (had * inverse)[..., None, None]), held.float()).to(torch.int8)
    held = torch.where((touched & kept)[:, :, None, None], again, held)
    held[at, :, offset.long()] = torch.round(rows * inverse[at][..., None]).to(torch.int8)
    codes.copy_(held.view(pages, per, kv, BLOCK, hd).permute(0, 2, 1, 3, 4).reshape(codes.shape))
    scales.copy_(torch.where(touched, new, old).view(pages, per, kv).transpose(1, 2))


def _values(codes, scales, page, offset):
    """float32 [rows, kv, hd]: what the cache holds at these pages and offsets."""
    page, offset = page.long(), offset.long()
    return codes[page, :, offset].float() * scales[page, :, offset // BLOCK][..., None]


def _pages(s, seq, pos):
    return s["page_table"][s["seq_slot"][seq.long()].long(), (pos // PAGE).long()]


def _plain_read(s):
    page, offset = _pages(s, s["row_seq"], s["row_pos"]), s["row_pos"] % PAGE
    s["k_rows"].copy_(_values(s["k"], s["k_scale"], page, offset))
    s["v_rows"].copy_(_values(s["v"], s["v_scale"], page, offset))
    return {"k": s["k_rows"], "v": s["v_rows"]}


def _plain_write(s):
    case = s["case"]
    heads, kv, hd, _, _ = SHAPES[case["model"]]
    x = s["qkv"].float().view(s["n_tokens"], heads + 2 * kv, hd)
    pos = s["token_pos"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["q_out"].copy_(_turned(x[:, :heads], cos, sin, case["style"]).reshape(s["n_tokens"], -1))
    offset = s["token_pos"] % PAGE
    block = _pages(s, s["token_seq"], s["token_pos"]) * (PAGE // BLOCK) + offset // BLOCK
    begun = s["token_pos"] // BLOCK * BLOCK < s["seq_start"][s["token_seq"].long()]
    _put(s["k"], s["k_scale"], _turned(x[:, heads:heads + kv], cos, sin, case["style"]), block, offset % BLOCK, begun)
    _put(s["v"], s["v_scale"], x[:, heads + kv:], block, offset % BLOCK, begun)
    return {"q": s["q_out"], **_plain_read(s)}


def _plain_attend(s):
    case = s["case"]
    heads, kv, hd, _, _ = SHAPES[case["model"]]
    n, longest, fresh = s["n_seqs"], s["max_len"], s["max_new"]
    key = torch.arange(longest, device=DEVICE)
    page = s["page_table"][s["seq_slot"].long()][:, key // PAGE]                    # [n, longest]
    # [n, kv, longest, hd]; positions behind a sequence's end come from page 0 and are masked
    k = _values(s["k"], s["k_scale"], page, (key % PAGE).expand(n, -1)).transpose(1, 2)
    v = _values(s["v"], s["v_scale"], page, (key % PAGE).expand(n, -1)).transpose(1, 2)
    row = torch.arange(s["n_tokens"], device=DEVICE)
    seq = s["token_seq"].long()
    place = row - s["cu_seqlens"][seq]
    q = torch.zeros(n, fresh, heads * hd, device=DEVICE)
    q[seq, place] = s["q"].float()
    q = q.view(n, fresh, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)         # rows: head, then token
    score = (q @ k.transpose(2, 3)).view(n, kv, heads // kv, fresh, longest) * (1.0 / math.sqrt(hd))
    pos = s["seq_start"][:, None] + torch.arange(fresh, device=DEVICE)
    seen = key <= pos[..., None]
    if case["window"]:
        seen = seen & (key > pos[..., None] - case["window"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(dim=-1, keepdim=True))
    weight = weight / weight.sum(dim=-1, keepdim=True)
    o = (weight.view(n, kv, -1, longest) @ v).view(n, heads, fresh, hd)
    s["out"].copy_(o.permute(0, 2, 1, 3).reshape(n, fresh, -1)[seq, place])
    return s["out"]


def _plain_score(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(dim=1, keepdim=True)
    logp = x - m - torch.log(z)
    p = e / z
    out = {"logprob": logp.gather(1, s["targets"].long()[:, None])[:, 0],
           "entropy": -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=1)}
    if top:
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]     # stable: ties of the logits to the lowest id
        out |= {"top_ids": ids.to(torch.int32), "top_logprobs": logp.gather(1, ids)}
    return out


# ---- the library's operators ------------------------------------------------------------------------------------------
def _layer(s):
    """The cache as the library's operators take it, made of the caller's tensors once."""
    if "layer" not in s:
        from rust_inference_b200.kernels import quantized_cache
        s["layer"] = quantized_cache.QuantizedPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s["layer"]


def _own_read(s):
    from rust_inference_b200.kernels import quantized_cache
    quantized_cache.read(_layer(s), s["k_rows"], s["v_rows"], s["page_table"], s["seq_slot"], s["first"], s["seq_len"],
                         max_len=s["max_len"], cu_rows=s["cu_rows"])
    return {"k": s["k_rows"], "v": s["v_rows"]}


def _own_write(s):
    from rust_inference_b200.kernels import quantized_cache
    heads, kv, hd, _, _ = SHAPES[s["case"]["model"]]
    quantized_cache.write(s["qkv"], s["q_out"], s["cos"], s["sin"], _layer(s), s["page_table"], s["seq_slot"], s["seq_start"],
                          s["cu_seqlens"], n_heads=heads, n_kv_heads=kv, head_dim=hd, max_new=s["max_new"],
                          style=1 if s["case"]["style"] == "interleaved" else 0)
    return {"q": s["q_out"], **_own_read(s)}


def _context(s):
    """The step as the library's layers know it, made of the caller's arrays once; scratch buffers live in its workspace."""
    if "context" not in s:
        from rust_inference_b200.engine.context import StepContext, Workspace
        s["context"] = StepContext(
            n_tokens=s["n_tokens"], n_seqs=s["n_seqs"], token_ids=s["token_pos"], token_pos=s["token_pos"], token_seq=s["token_seq"],
            seq_slot=s["seq_slot"], seq_start=s["seq_start"], seq_len=s["seq_len"], cu_seqlens=s["cu_seqlens"],
            logit_rows=s["cu_seqlens"], n_logit_rows=0, max_new=s["max_new"], max_len=s["max_len"], all_single=s["max_new"] == 1,
            page_table=s["page_table"], page_size=PAGE, dtype=s["q"].dtype, device=s["q"].device, workspace=Workspace(s["q"].device))
    return s["context"]


def _own_attend(s):
    from rust_inference_b200.kernels import attention
    heads, kv, hd, _, _ = SHAPES[s["case"]["model"]]
    return attention.attention(s["q"], _layer(s), s["out"], _context(s), n_heads=heads, n_kv_heads=kv, head_dim=hd,
                               scale=1.0 / math.sqrt(hd), window=s["case"]["window"])


def _own_score(s):
    from rust_inference_b200.kernels import ops
    found = ops.token_logprobs(s["logits"], s["targets"], top=s["case"]["top"])
    out = {"logprob": found.logprob, "entropy": found.entropy}
    if s["case"]["top"]:
        out |= {"top_ids": found.top_ids, "top_logprobs": found.top_logprobs}
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"write": _own_write, "read": _own_read, "attend": _own_attend, "score": _own_score}[op](state)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "score": _plain_score}[op](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    heads, kv, hd, _, _ = SHAPES[case["model"]]
    item = DTYPES[case["dtype"]].itemsize
    after, fresh = _lengths(case)
    scales = 4.0 / BLOCK
    if case["op"] == "read":
        n = sum(after)
        return {"bytes": 2 * n * kv * (hd * (1 + item) + scales), "flops": 2 * n * kv * hd}
    if case["op"] == "write":
        n = sum(fresh)
        # of the blocks that a step touches: the older positions' codes read, the new ones' written, all read back
        rows = sum(f + (a - f) % BLOCK for a, f in zip(after, fresh))
        return {"bytes": n * (heads + 2 * kv) * hd * item + n * heads * hd * item + n * 4 * hd + 2 * rows * kv * (hd * (1 + item) + scales),
                "flops": n * (heads + kv) * hd * 3 + 2 * n * kv * hd * 3 + 2 * rows * kv * hd}
    keys = pairs = 0
    for a, f in zip(after, fresh):
        w = case["window"] or a
        keys += min(a, w + f - 1)
        pairs += sum(min(p + 1, w) for p in range(a - f, a))
    return {"bytes": 2 * sum(fresh) * heads * hd * item + 2 * keys * kv * (hd + scales), "flops": 4.0 * pairs * heads * hd}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        parts = []
        for at in range(0, case["rows"], 64):
            x, t = s["logits"][at:at + 64].double(), s["targets"][at:at + 64].long()
            logp = x - torch.logsumexp(x, dim=1, keepdim=True)
            p = torch.exp(logp)
            one = {"logprob": logp[torch.arange(len(t), device=DEVICE), t], "entropy": -(p * logp.clamp(min=-1e30)).sum(dim=1)}
            if case["top"]:
                one["top_logprobs"] = logp.topk(case["top"], dim=1).values
            parts.append(one)
        out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
        return {**out, "top_ids": None} if case["top"] else out
    heads, kv, hd, base, _ = SHAPES[case["model"]]
    after, fresh = _lengths(case)
    rep = heads // kv
    table, slot = s["page_table"].cpu(), s["seq_slot"].cpu()

    def held(name, b, upto):
        """[kv, upto, hd] float64: what the cache holds of sequence b before the step."""
        pages = table[int(slot[b]), :-(-upto // PAGE)].long().to(DEVICE)
        codes = s[name][pages].double().view(len(pages), kv, PAGE // BLOCK, BLOCK, hd) * s[name + "_scale"][pages].double()[..., None, None]
        return codes.reshape(len(pages), kv, PAGE, hd).transpose(0, 1).reshape(kv, -1, hd)[:, :upto]

    if case["op"] == "read":
        got = [[held(name, b, n).transpose(0, 1) for b, n in enumerate(after)] for name in "kv"]
        return {"k": torch.cat(got[0]), "v": torch.cat(got[1])}
    if case["op"] == "attend":
        outs, at = [], 0
        for b, (n, f) in enumerate(zip(after, fresh)):
            k, v = held("k", b, n), held("v", b, n)
            q = s["q"][at:at + f].double().view(f, kv, rep, hd)
            at += f
            pos = torch.arange(n - f, n, device=DEVICE)
            seen = torch.arange(n, device=DEVICE)[None] <= pos[:, None]
            if case["window"]:
                seen &= torch.arange(n, device=DEVICE)[None] > pos[:, None] - case["window"]
            o = torch.empty(f, kv, rep, hd, dtype=torch.float64, device=DEVICE)
            for h in range(kv):
                score = torch.einsum("trd,nd->trn", q[:, h], k[h]) / math.sqrt(hd)
                o[:, h] = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), dim=-1) @ v[h]
            outs.append(o.reshape(f, -1))
        return torch.cat(outs)
    # write: keys turned in 64 bits by the 32-bit angles' tables; a block's values after the step, block by block
    x = s["qkv"].double().view(-1, heads + 2 * kv, hd)
    cos, sin = s["cos"].double()[s["token_pos"].long()][:, None], s["sin"].double()[s["token_pos"].long()][:, None]
    turned = _exact_turned(x[:, :heads + kv], cos, sin, case["style"])
    rows = {"k": turned[:, heads:], "v": x[:, heads + kv:]}
    out = {"q": turned[:, :heads].reshape(len(x), -1), "k": [], "v": []}
    for name in "kv":
        at = 0
        for b, (n, f) in enumerate(zip(after, fresh)):
            new = rows[name][at:at + f]
            at += f
            pages = table[int(slot[b])]
            for first in range((n - f) // BLOCK * BLOCK, n, BLOCK):
                page, block = int(pages[first // PAGE]), first % PAGE // BLOCK
                lo, hi = max(first, n - f), min(first + BLOCK, n)
                part = new[lo - (n - f):hi - (n - f)].transpose(0, 1)
                older = s[name][page, :, block * BLOCK:block * BLOCK + lo - first]
                size = (part.abs().amax(dim=(1, 2), keepdim=True) / 127.0)
                size = torch.where(size < TINY, 0.0, size).float().double()
                if lo > first:
                    was = s[name + "_scale"][page, :, block].double()[:, None, None]
                    size = torch.maximum(size, was)
                    older = torch.where(size > was, torch.round(older.double() * was / size), older.double())
                codes = torch.cat([older.double(), torch.round(part / torch.where(size > 0, size, 1.0))], dim=1)
                out[name].append((codes * size).transpose(0, 1))
        out[name] = torch.cat(out[name])
    return out


def _exact_turned(x, cos, sin, style):
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) if style == "interleaved" else torch.complex(*x.chunk(2, dim=-1))
    z = z * torch.complex(cos, sin)
    return torch.view_as_real(z).flatten(-2) if style == "interleaved" else torch.cat([z.real, z.imag], dim=-1)
