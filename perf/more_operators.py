"""The operators that weights in microscaled 4-bit floating point are timed on: holding a matrix in 4 bits, the root-mean-square
norm that adds what a layer adds to the stream and leaves its result in microscaled 8 bits, the product of 8-bit rows with a 4-bit
matrix, and the gated feed-forward that chains them.

Every case is one pass through an operator, on tensors as the layers of a model hand them over.

    listed()            the cases
    draw(rng)           one more of the same ranges
    prepare(case, seed) what the caller has in hand: the stream, a layer's matrices (in 4 bits already, but where that is measured)
    run(state)          one pass, in plain torch operations (`own` false) or by the library's operators (`own` true)
    work(case)          the bytes and operations a pass cannot do without
    exact(case, seed)   the same results in 64 bits

Microscaled numbers: 32 consecutive ones along a row share a power of two, 2^e, the smallest for which the largest of them is at most
the largest number of the type: 6 for four bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), 448 for eight (four bits of exponent,
three of mantissa).  Each is rounded to the nearest number of the type times 2^e, ties to the even one.  A row's last block may be shorter.
A matrix in 4 bits comes as its codes [N, ceil(K / 2)] (number 2i in the low half of byte i; sign, then the place in the list above)
and its exponents plus 127, [N, ceil(K / 32)].
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 32
EPS = 1e-6

# (hidden size, intermediate size, columns of q, k and v together) of the models that the library's own workloads name
SHAPES = {
    "qwen2-0.5b": (896, 4864, 1152),
    "qwen2-1.5b": (1536, 8960, 2048),
    "qwen2.5-3b": (2048, 11008, 2560),
    "qwen2.5-7b": (3584, 18944, 4608),
    "llama3-8b": (4096, 14336, 6144),
}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _named(case, name):
    return dict(case, name=name) if name else case


def _hold(name, dtype, n, k):
    return _named({"op": "hold", "dtype": dtype, "n": n, "k": k}, name)


def _norm(name, dtype, rows, k):
    return _named({"op": "norm", "dtype": dtype, "rows": rows, "k": k}, name)


def _project(name, dtype, rows, n, k, bias):
    return _named({"op": "project", "dtype": dtype, "rows": rows, "n": n, "k": k, "bias": bias}, name)


def _feed(name, rows, hidden, inner):
    return _named({"op": "feed", "dtype": "bfloat16", "rows": rows, "k": hidden, "inner": inner}, name)


def listed():
    return [
        # a small model is loaded: one of its square matrices
        _hold("hold 0.5b o", "bfloat16", 896, 896),
        # a matrix of odd sizes from a file in 32 bits: a short last block in every row
        _hold("hold odd f32", "float32", 3001, 1333),
        # the largest matrix of a layer
        _hold("hold 7b down", "bfloat16", 3584, 18944),
        # a server's ordinary step: the attention's result joins the stream, and the feed-forward's input leaves
        _norm("norm 7b x8", "bfloat16", 8, 3584),
        # the same of a prompt
        _norm("norm 8b 2047", "bfloat16", 2047, 4096),
        # one user waiting for the next token of a small model: the smallest call
        _project("qkv 0.5b x1", "bfloat16", 1, 1152, 896, True),
        # the output projection of a batch of eight
        _project("o 7b x8", "bfloat16", 8, 3584, 3584, False),
        # a full batch
        _project("qkv 8b x61", "bfloat16", 61, 6144, 4096, False),
        # a conversation of a 32-bit run is taken up again with a few hundred tokens
        _project("qkv 3b 333 f32", "float32", 333, 2560, 2048, True),
        # whole feed-forwards, from the stream to what joins it: one user, a batch, a prompt of the benchmark's length
        _feed("feed 1.5b x1", 1, 1536, 8960),
        _feed("feed 7b x8", 8, 3584, 18944),
        _feed("feed 7b 2048", 2048, 3584, 18944),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["hold", "norm", "project", "project", "feed", "feed"])
    hidden, inner, qkv = SHAPES[rng.choice(sorted(SHAPES))]
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    odd = rng.random() < 0.4
    if op == "hold":
        n, k = rng.choice([(qkv, hidden), (hidden, inner), (inner, hidden)])
        return _hold(None, dtype, _log(rng, 100, 8000), _log(rng, 40, 8000)) if odd else _hold(None, dtype, n, k)
    if op == "norm":
        return _norm(None, dtype, _log(rng, 1, 2048), _log(rng, 40, 8000) if odd else hidden)
    rows = rng.choice([1, 2, 7, 8, _log(rng, 1, 128), _log(rng, 1, 128), _log(rng, 129, 2048)])
    if op == "feed":
        return _feed(None, rows, _log(rng, 300, 3500), _log(rng, 700, 12000)) if odd else _feed(None, rows, hidden, inner)
    n, k = rng.choice([(qkv, hidden), (hidden, hidden), (hidden, inner)])
    if odd:
        n, k = _log(rng, 100, 12000), _log(rng, 40, 12000)
    return _project(None, dtype, rows, n, k, rng.random() < 0.5)


# ---- microscaled numbers in plain operations --------------------------------------------------------------------------
STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_FOUR, MOST_EIGHT = (0.75, 3), (0.875, 9)           # 6 and 448 as p * 2^e


def _two(e):
    """2^e as a float64, for integers e of -1022 to 1023."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _blocks(x):
    """x [rows, k] as [rows, blocks, 32], zeros behind the end of a row."""
    rows, k = x.shape
    n = -(-k // BLOCK)
    if n * BLOCK > k:
        x = torch.cat([x, x.new_zeros(rows, n * BLOCK - k)], dim=1)
    return x.view(rows, n, BLOCK)


def _exponent(b, part, shift):
    """[rows, blocks, 1]: the smallest e with max |b| <= part * 2^(shift + e), which is the type's largest number times 2^e."""
    p, e = torch.frexp(b.abs().amax(dim=2, keepdim=True))
    return (e - shift + (p > part)).clamp(-127, 127)


def _rounded(y, least, mantissa):
    """y to the nearest number with so many bits of mantissa, exponents from `least` on; ties to even."""
    _, e = torch.frexp(y)
    step = _two((e - 1).clamp(min=least) - mantissa).to(y.dtype)
    return torch.round(y / step) * step


def _in_eight(x):
    """x [rows, k] as the microscaled 8-bit numbers nearest to it."""
    b = _blocks(x)
    s = _two(_exponent(b, *MOST_EIGHT)).to(x.dtype)
    return (_rounded(b / s, -6, 3) * s).flatten(1)[:, :x.shape[1]]


def _in_four(x):
    b = _blocks(x)
    s = _two(_exponent(b, *MOST_FOUR)).to(x.dtype)
    return (_rounded(b / s, 0, 1) * s).flatten(1)[:, :x.shape[1]]


def _packed(x):
    """Codes and exponents of x [n, k] float32 in 4 bits, a few thousand rows at a time."""
    codes, scales = [], []
    for part in x.split(2048):
        b = _blocks(part)
        e = _exponent(b, *MOST_FOUR)
        y = _rounded(b / _two(e).float(), 0, 1)
        place = torch.bucketize(y.abs(), torch.tensor(STEPS, device=x.device)) + torch.where(torch.signbit(y) & (y != 0), 8, 0)
        place = place.to(torch.uint8).flatten(1)
        codes.append((place[:, 0::2] | place[:, 1::2] << 4)[:, :-(-x.shape[1] // 2)])
        scales.append((e[:, :, 0] + 127).to(torch.uint8))
    return torch.cat(codes).contiguous(), torch.cat(scales).contiguous()


def _unpacked(m, dtype=torch.float32):
    """The numbers [n, k] that a packed matrix stands for."""
    codes, scales, k = m
    table = torch.tensor(STEPS + tuple(-v for v in STEPS), dtype=dtype, device=codes.device)
    y = table[torch.stack([codes & 15, codes >> 4], dim=2).flatten(1).int()][:, :k]
    return (_blocks(y) * _two(scales.int() - 127).to(dtype)[:, :, None]).flatten(1)[:, :k]


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 29)


def _rows(g, rows, k):
    """Activations: channels of unequal size, a few several times the others."""
    return torch.randn(rows, k, generator=g, device=DEVICE) * torch.exp(0.7 * torch.randn(k, generator=g, device=DEVICE))


def _matrix(g, n, k):
    return torch.randn(n, k, generator=g, device=DEVICE) * (1.0 / math.sqrt(k))


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    dtype, k = DTYPES[case["dtype"]], case["k"]
    if case["op"] == "hold":
        s["w"] = _matrix(g, case["n"], k).to(dtype)
        return s
    rows = case["rows"]
    if case["op"] == "project":
        n = case["n"]
        s["x"] = _rows(g, rows, k).to(dtype)
        s["w"] = (*_packed(_matrix(g, n, k)), k)
        s["bias"] = torch.randn(n, generator=g, device=DEVICE) if case["bias"] else None
        s["out"] = torch.empty(rows, n, dtype=dtype, device=DEVICE)
        return s
    s["stream"] = _rows(g, rows, k)
    s["branch"] = _rows(g, rows, k).to(dtype)
    s["weight"] = 1.0 + 0.1 * torch.randn(k, generator=g, device=DEVICE)
    s["total"] = torch.empty(rows, k, device=DEVICE)
    s["out"] = torch.empty(rows, k, dtype=torch.bfloat16, device=DEVICE)
    if case["op"] == "feed":
        s["gate"], s["up"] = ((*_packed(2.0 * _matrix(g, case["inner"], k)), k) for _ in range(2))
        s["down"] = (*_packed(_matrix(g, k, case["inner"])), case["inner"])
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _plain_norm(s):
    """The stream with the branch added, and its norm, both [rows, k]; the norm in 64 bits, because it is rounded to few."""
    total = s["stream"] + s["branch"].float()
    x = total.double()
    return total, x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["weight"].double()


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        return _own(s, op)
    if op == "hold":
        return _in_four(s["w"].float()).to(s["w"].dtype)
    if op == "project":
        y = _in_eight(s["x"].float()) @ _unpacked(s["w"]).t()
        s["out"].copy_(y if s["bias"] is None else y + s["bias"])
        return s["out"]
    total, h = _plain_norm(s)
    s["total"].copy_(total)
    if op == "norm":
        s["out"].copy_(_in_eight(h))
        return {"total": s["total"], "normed": s["out"]}
    x = _in_eight(h).float()
    gate, up = x @ _unpacked(s["gate"]).t(), x @ _unpacked(s["up"]).t()
    s["out"].copy_(_in_eight(gate / (1.0 + torch.exp(-gate)) * up) @ _unpacked(s["down"]).t())
    return {"total": s["total"], "out": s["out"]}


# ---- the library's operators ------------------------------------------------------------------------------------------
def _held(s, name):
    """A matrix as the library's products take it, laid out of the caller's codes once."""
    key = "held " + name
    if key not in s:
        from rust_inference_b200.kernels import microscaled
        s[key] = microscaled.Matrix.of_codes(*s[name])
    return s[key]


def _scratch(s, name, rows, k):
    """8-bit rows that a caller keeps between its calls."""
    key = "rows " + name
    if key not in s:
        from rust_inference_b200.kernels import microscaled
        s[key] = microscaled.Rows(rows, k, DEVICE)
    return s[key]


def _context(s, rows, dtype):
    """The step as the library's layers know it, made once; the products' scratch lives in its workspace."""
    if "context" not in s:
        from rust_inference_b200.engine.context import StepContext, Workspace
        ints = torch.zeros(rows + 1, dtype=torch.int32, device=DEVICE)
        s["context"] = StepContext(
            n_tokens=rows, n_seqs=rows, token_ids=ints, token_pos=ints, token_seq=ints, seq_slot=ints, seq_start=ints, seq_len=ints,
            cu_seqlens=ints, logit_rows=ints, n_logit_rows=0, max_new=1, max_len=1, all_single=True, page_table=ints[None], page_size=64,
            dtype=dtype, device=ints.device, workspace=Workspace(ints.device))
    return s["context"]


def _own(s, op):
    from rust_inference_b200.kernels import linear, microscaled
    case = s["case"]
    if op == "hold":
        return microscaled.values(microscaled.Matrix.of(s["w"]), s["w"].dtype)
    rows, k = case["rows"], case["k"]
    ctx = _context(s, rows, DTYPES[case["dtype"]])
    if op == "project":
        linear.project(s["x"], _held(s, "w"), s["out"], ctx, bias=s["bias"])
        return s["out"]
    normed = _scratch(s, "normed", rows, k)
    microscaled.rmsnorm(s["stream"], s["weight"], EPS, normed, branch=s["branch"], total=s["total"])
    if op == "norm":
        microscaled.values(normed, torch.bfloat16, out=s["out"])
        return {"total": s["total"], "normed": s["out"]}
    act = _scratch(s, "act", rows, case["inner"])
    linear.gated(normed, _held(s, "gate"), _held(s, "up"), act, ctx)
    linear.project(act, _held(s, "down"), s["out"], ctx)
    return {"total": s["total"], "out": s["out"]}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    item, k = DTYPES[case["dtype"]].itemsize, case["k"]

    def four(n, width):
        return n * (-(-width // 2) + -(-width // BLOCK))

    if case["op"] == "hold":
        return {"bytes": 2 * case["n"] * k * item, "flops": 4 * case["n"] * k}
    rows = case["rows"]
    if case["op"] == "project":
        n = case["n"]
        return {"bytes": rows * (k + n) * item + four(n, k) + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    norm = {"bytes": rows * k * (4 + item + 4 + 2) + 4 * k, "flops": 8 * rows * k}
    if case["op"] == "norm":
        return norm
    inner = case["inner"]
    return {"bytes": norm["bytes"] + 2 * four(inner, k) + four(k, inner), "flops": norm["flops"] + 6 * rows * k * inner}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------
def _nearest(x, numbers, most):
    """x [rows, k] float64 as the microscaled numbers nearest to it: `numbers` are the type's that are not negative, in order, of which
    every second one is even."""
    numbers = torch.tensor(numbers, dtype=torch.float64, device=x.device)
    middle = (numbers[1:] + numbers[:-1]) / 2
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        top = part.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / most))
        e = torch.where(top > most * torch.exp2(e), e + 1, torch.where(top <= most * torch.exp2(e - 1), e - 1, e)).clamp(-127, 127)
        a = part.abs() * torch.exp2(-e)
        low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)      # they differ where a is a middle
        place = torch.where(low % 2 == 0, low, high)
        out[:, at:at + BLOCK] = torch.copysign(numbers[place], part) * torch.exp2(e)
    return out


EIGHT = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
FOUR = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _stands_for(m):
    """A packed matrix in 64 bits, number by number of a byte."""
    codes, scales, k = m
    signed = torch.tensor(FOUR + [-v for v in FOUR], dtype=torch.float64, device=codes.device)
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    out[:, 0::2] = signed[(codes % 16).int()]
    out[:, 1::2] = signed[(codes // 16).int()]
    out = out[:, :k]
    return out * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "hold":
        return _nearest(s["w"].double(), FOUR, 6.0)
    if case["op"] == "project":
        y = torch.einsum("tk,nk->tn", _nearest(s["x"].double(), EIGHT, 448.0), _stands_for(s["w"]))
        return y if s["bias"] is None else y + s["bias"].double()
    total = s["stream"].double() + s["branch"].double()
    held = total.float().double()                                # the stream is held in 32 bits
    h = held / torch.sqrt(torch.linalg.vecdot(held, held)[:, None] / case["k"] + EPS) * s["weight"].double()
    h = _nearest(h, EIGHT, 448.0)
    if case["op"] == "norm":
        return {"total": total, "normed": h}
    z = torch.einsum("tk,nk->tn", h, _stands_for(s["gate"]))
    z = z * torch.sigmoid(z) * torch.einsum("tk,nk->tn", h, _stands_for(s["up"]))
    return {"total": total, "out": torch.einsum("tk,nk->tn", _nearest(z, EIGHT, 448.0), _stands_for(s["down"]))}
