"""The cache in 8 bits, kernel by kernel, against `plain_quantized`: codes and scales bit by bit, values read back, and attention
over it within bounds that follow from the roundings each path makes."""
import math

import pytest
import torch

import plain_quantized as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _qc():
    from rust_inference_b200.kernels import quantized_cache
    return quantized_cache


class Step:
    """Sequences (positions before, new tokens) over shuffled pages and slots, with the arrays of a step on the device."""

    def __init__(self, runs, n_kv, hd, v_hd=None, seed=0):
        self.runs, self.n_kv, self.hd, self.v_hd = runs, n_kv, hd, hd if v_hd is None else v_hd
        g = torch.Generator().manual_seed(seed)
        counts = [-(-(s + n) // plain.PAGE) for s, n in runs]
        pool = sum(counts) + 2
        order, self.slots = torch.randperm(pool, generator=g), torch.randperm(len(runs) + 1, generator=g)[:len(runs)]
        self.table = torch.zeros(len(runs) + 1, max(counts + [1]), dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[self.slots[b], :c] = order[at:at + c].int()
            at += c
        self.layer = _qc().empty_layer(pool, n_kv, hd, self.v_hd, device=DEV)
        # pages that other sequences have used: whatever codes and scales they left
        for t in (self.layer.k, self.layer.v):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g).to(torch.int8))
        for t in (self.layer.k_scale, self.layer.v_scale):
            t.copy_(torch.rand(t.shape, generator=g) + 0.5)
            t[-1] = math.nan
        self.arrays(runs)

    def arrays(self, runs):
        self.runs = runs
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.seq_start, self.seq_len = ints([s for s, _ in runs]), ints([s + n for s, n in runs])
        cu = [0]
        for _, n in runs:
            cu.append(cu[-1] + n)
        self.cu, self.cu_seqlens, self.n_tokens = cu, ints(cu), cu[-1]
        self.token_pos = ints([p for s, n in runs for p in range(s, s + n)])
        self.token_seq = ints([b for b, (_, n) in enumerate(runs) for _ in range(n)])
        self.page_table, self.seq_slot = self.table.to(DEV), self.slots.int().to(DEV)
        self.max_new, self.max_len = max(n for _, n in runs), max(s + n for s, n in runs)

    def pages(self, b):
        return self.table[self.slots[b]]

    def host(self):
        return [t.cpu().clone() for t in (self.layer.k, self.layer.v, self.layer.k_scale, self.layer.v_scale)]

    def fill(self, seed=1):
        """Earlier positions of every sequence, as the plain implementation writes them."""
        g = torch.Generator().manual_seed(seed)
        k, v, ks, vs = self.host()
        for b, (start, _) in enumerate(self.runs):
            if start:
                plain.put(k, ks, torch.randn(start, self.n_kv, self.hd, generator=g), 0, self.pages(b))
                plain.put(v, vs, torch.randn(start, self.n_kv, self.v_hd, generator=g), 0, self.pages(b))
        for to, t in zip((self.layer.k, self.layer.v, self.layer.k_scale, self.layer.v_scale), (k, v, ks, vs)):
            to.copy_(t)

    def context(self, dtype):
        from rust_inference_b200.engine.context import StepContext, Workspace
        return StepContext(n_tokens=self.n_tokens, n_seqs=len(self.runs), token_ids=self.token_pos, token_pos=self.token_pos,
                           token_seq=self.token_seq, seq_slot=self.seq_slot, seq_start=self.seq_start, seq_len=self.seq_len,
                           cu_seqlens=self.cu_seqlens, logit_rows=self.cu_seqlens, n_logit_rows=0, max_new=self.max_new,
                           max_len=self.max_len, all_single=all(n == 1 for _, n in self.runs), page_table=self.page_table,
                           page_size=plain.PAGE, dtype=dtype, device=torch.device(DEV), workspace=Workspace(DEV))


def _tables(positions, rot):
    theta = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * theta
    return angle.cos().float(), angle.sin().float()


def _write(step, rows, *, n_heads, rot, style, bias=None, clear=False, q_dtype=None, v_hd=None):
    cos, sin = _tables(max(step.max_len, 1), rot)
    src = rows.to(DEV)
    q = torch.zeros(step.n_tokens, n_heads * step.hd, dtype=q_dtype or rows.dtype, device=DEV)
    _qc().write(src, q, cos.to(DEV) if rot else None, sin.to(DEV) if rot else None, step.layer, step.page_table, step.seq_slot,
                step.seq_start, step.cu_seqlens, n_heads=n_heads, n_kv_heads=step.n_kv, head_dim=step.hd, v_head_dim=step.v_hd,
                max_new=max(step.max_new, 1), style=style, rot_dims=rot, bias=None if bias is None else bias.to(DEV), clear=clear)
    return q, src


def _check_written(step, rows, before, q, *, n_heads, rot, style, bias=None):
    """Codes, scales and queries against the plain implementation, bit by bit."""
    k, v, ks, vs = before
    cos, sin = _tables(max(step.max_len, 1), rot)
    x = rows.float()[:, :(n_heads + step.n_kv) * step.hd + step.n_kv * step.v_hd]
    if bias is not None:
        x = x + bias[:x.shape[1]]
    heads = x[:, :(n_heads + step.n_kv) * step.hd].reshape(step.n_tokens, -1, step.hd)
    pos = step.token_pos.cpu().long()
    heads = torch.stack([plain.turned(heads[t], cos[pos[t]], sin[pos[t]], style) for t in range(step.n_tokens)])
    vals = x[:, (n_heads + step.n_kv) * step.hd:].reshape(step.n_tokens, step.n_kv, step.v_hd)
    assert torch.equal(q.cpu(), heads[:, :n_heads].reshape(step.n_tokens, -1).to(q.dtype))
    for b, (start, n) in enumerate(step.runs):
        a, e = step.cu[b], step.cu[b + 1]
        plain.put(k, ks, heads[a:e, n_heads:], start, step.pages(b))
        plain.put(v, vs, vals[a:e], start, step.pages(b))
    got = step.host()
    for g, w in zip(got[:2], (k, v)):
        assert torch.equal(g, w)
    for g, w in zip(got[2:], (ks, vs)):
        assert torch.equal(g.view(torch.int32) * ~g.isnan(), w.view(torch.int32) * ~w.isnan()) and torch.equal(g.isnan(), w.isnan())


RUNS = {
    "single": [(0, 1), (15, 1), (16, 1), (63, 1), (64, 1), (200, 1), (7, 1)],
    "few": [(0, 2), (14, 5), (62, 3), (127, 1), (48, 16)],
    "prompts": [(0, 70), (0, 1), (0, 16), (5, 33), (100, 29), (0, 0), (31, 0)],
    "long": [(0, 333)],
}


@pytest.mark.parametrize("runs", sorted(RUNS))
@pytest.mark.parametrize("n_heads, n_kv, hd, v_hd, rot, style, dtype", [
    (4, 2, 64, 64, 64, 0, torch.bfloat16), (4, 2, 64, 64, 64, 1, torch.float32), (7, 1, 128, 128, 128, 0, torch.bfloat16),
    (6, 3, 128, 128, 128, 1, torch.bfloat16), (2, 2, 128, 128, 128, 0, torch.float32), (6, 2, 24, 24, 24, 0, torch.bfloat16),
    (2, 1, 96, 32, 48, 0, torch.float32), (4, 2, 64, 128, 32, 1, torch.bfloat16), (4, 2, 128, 128, 0, 0, torch.bfloat16)])
def test_write(runs, n_heads, n_kv, hd, v_hd, rot, style, dtype):
    step = Step(RUNS[runs], n_kv, hd, v_hd)
    step.fill()
    g = torch.Generator().manual_seed(3)
    rows = (torch.randn(step.n_tokens, (n_heads + n_kv) * hd + n_kv * v_hd, generator=g) * 1.5).to(dtype)
    before = step.host()
    q, _ = _write(step, rows, n_heads=n_heads, rot=rot, style=style)
    _check_written(step, rows, before, q, n_heads=n_heads, rot=rot, style=style)


@pytest.mark.parametrize("sequences", [80, 110])
@pytest.mark.parametrize("n_heads, hd, dtype", [(30, 64, torch.bfloat16), (32, 128, torch.float32)])
def test_write_of_many_sequences(sequences, n_heads, hd, dtype):
    """More query heads than the SMs have warps for at once, one per warp; the last block of heads not full."""
    runs = [((7 * i) % 45, 1 + (i % 9 == 0)) for i in range(sequences)]
    step = Step(runs, 8, hd)
    step.fill()
    rows = torch.randn(step.n_tokens, (n_heads + 16) * hd, generator=torch.Generator().manual_seed(5)).to(dtype)
    before = step.host()
    q, _ = _write(step, rows, n_heads=n_heads, rot=hd, style=0)
    _check_written(step, rows, before, q, n_heads=n_heads, rot=hd, style=0)


@pytest.mark.parametrize("hd, q_dtype", [(64, torch.bfloat16), (128, torch.float32), (40, torch.bfloat16)])
@pytest.mark.parametrize("runs", ["single", "prompts"])
def test_write_from_sums_with_a_bias(runs, hd, q_dtype):
    """float32 sums of a product that was cut over K, wider than the heads: the bias is added, the sums that were used are zeroed."""
    step = Step(RUNS[runs], 2, hd)
    step.fill()
    g = torch.Generator().manual_seed(4)
    cols = 8 * hd
    rows, bias = torch.randn(step.n_tokens, cols + 8, generator=g), torch.randn(cols + 8, generator=g)
    before = step.host()
    q, src = _write(step, rows, n_heads=4, rot=hd, style=0, bias=bias, clear=True, q_dtype=q_dtype)
    _check_written(step, rows, before, q, n_heads=4, rot=hd, style=0, bias=bias)
    assert not src[:, :cols].any() and torch.equal(src[:, cols:].cpu(), rows[:, cols:])


@pytest.mark.parametrize("hd", [64, 128, 24])
def test_rows_off_a_16_byte_boundary(hd):
    step = Step(RUNS["few"], 2, hd)
    step.fill()
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(step.n_tokens, 8 * hd + 3, generator=g).to(torch.bfloat16)       # an odd row length
    before = step.host()
    q, _ = _write(step, rows, n_heads=4, rot=hd, style=0)
    _check_written(step, rows, before, q, n_heads=4, rot=hd, style=0)


@pytest.mark.parametrize("hd", [64, 128, 24])
def test_a_block_grows_token_by_token(hd):
    """Forty single tokens, most larger than the one before: scales grow, older codes are rounded again, and every value
    stays within half a step of the final scale for each time its block grew, plus its own half step."""
    step = Step([(0, 1), (9, 1)], 2, hd)
    step.fill()
    g = torch.Generator().manual_seed(6)
    written = {b: [] for b in range(2)}
    for t in range(40):
        if t:
            step.arrays([(s + 1, 1) for s, _ in step.runs]) if step.runs[0][0] + 2 <= 64 else None
        rows = torch.randn(2, 8 * hd, generator=g) * (1.0 + 0.3 * t)
        before = step.host()
        q, _ = _write(step, rows, n_heads=4, rot=0, style=0)
        _check_written(step, rows, before, q, n_heads=4, rot=0, style=0)
        for b in range(2):
            written[b].append(rows[b, 4 * hd:].view(4, hd))
    k, v, ks, vs = step.host()
    for b, first in ((0, 0), (1, 9)):
        rows = torch.stack(written[b])
        for codes, scales, want in ((k, ks, rows[:, :2]), (v, vs, rows[:, 2:])):
            got = plain.values(codes, scales, step.pages(b), first + 40)[first:]
            s = torch.stack([scales[int(step.pages(b)[p // 64]), :, p % 64 // 16] for p in range(first, first + 40)])
            assert ((got - want).abs() <= (0.5 * 17 + 1e-3) * s[..., None]).all()


@pytest.mark.parametrize("hd", [64, 128, 24])
def test_values_that_are_no_numbers(hd):
    """A NaN or an infinity marks its block for good, and the next sequence on the page starts afresh; tiny values are zeros."""
    step = Step([(3, 2), (16, 18), (0, 4), (0, 3)], 2, hd)
    step.fill()
    g = torch.Generator().manual_seed(7)
    rows = torch.randn(step.n_tokens, 8 * hd, generator=g)
    rows[0, 4 * hd + 1] = math.nan              # sequence 0: key head 0
    rows[2 + 17, 7 * hd + 5] = -math.inf        # sequence 1: value head 1 of its second block
    rows[20:24] *= 1e-39                        # sequence 2: below every scale
    rows[24:27] *= 1e37                         # sequence 3: near the largest numbers
    before = step.host()
    q, _ = _write(step, rows, n_heads=4, rot=0, style=0)
    _check_written(step, rows, before, q, n_heads=4, rot=0, style=0)
    assert step.layer.k_scale[step.pages(0)[0].item(), 0, 0].isnan() and step.layer.v_scale[step.pages(1)[0].item(), 1, 2].isnan()
    assert not step.layer.k_scale[step.pages(2)[0].item(), :, 0].any()
    step.arrays([(5, 1), (34, 1), (0, 5), (3, 1)])        # the marked blocks go on, sequence 2's pages are given to another
    rows = torch.randn(step.n_tokens, 8 * hd, generator=g)
    before = step.host()
    q, _ = _write(step, rows, n_heads=4, rot=0, style=0)
    _check_written(step, rows, before, q, n_heads=4, rot=0, style=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd, v_hd", [(64, 64), (128, 128), (24, 24), (96, 32)])
def test_read(hd, v_hd, dtype):
    step = Step([(130, 1), (0, 64), (1, 0), (63, 1), (0, 0), (17, 3)], 3, hd, v_hd)
    step.fill()
    step.arrays([(s + n, 0) for s, n in step.runs])
    first = torch.tensor([64, 0, 0, 63, 0, 16], dtype=torch.int32)
    lens = step.seq_len.cpu()
    n = (lens - first).clamp_min(0)
    # sequences without new tokens were filled up to their start
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0).int()])
    k = torch.full((int(cu[-1]), 3, hd), 7.0, dtype=dtype, device=DEV)
    v = torch.full((int(cu[-1]), 3, v_hd), 7.0, dtype=dtype, device=DEV)
    _qc().read(step.layer, k, v, step.page_table, step.seq_slot, first.to(DEV), step.seq_len, max_len=step.max_len, cu_rows=cu.to(DEV))
    codes = step.host()
    kp = torch.full(step.layer.k.shape, 7.0, dtype=dtype, device=DEV)
    vp = torch.full(step.layer.v.shape, 7.0, dtype=dtype, device=DEV)
    _qc().read(step.layer, kp, vp, step.page_table, step.seq_slot, first.to(DEV), step.seq_len, max_len=step.max_len)
    for c, s, rows, whole in ((codes[0], codes[2], k, kp), (codes[1], codes[3], v, vp)):
        want = torch.full(whole.shape, 7.0, dtype=dtype)
        for b in range(len(step.runs)):
            every = plain.values(c, s, step.pages(b), int(lens[b])).to(dtype)
            assert torch.equal(rows[int(cu[b]):int(cu[b + 1])].cpu(), every[int(first[b]):])
            for at in range(int(first[b]) // 64 * 64, int(lens[b]), 64):
                page = int(step.pages(b)[at // 64])
                part = every[at:at + 64].transpose(0, 1).clone()
                part[:, :max(0, int(first[b]) - at)] = 0
                want[page] = 0
                want[page, :, :part.shape[1]] = part
        assert torch.equal(whole.cpu(), want)


# relative rounding of weights, values and results; error of a score relative to sum |q k| scale
UNITS = {torch.bfloat16: (2.0 ** -9, 2.0 ** -9), torch.float32: (2.0 ** -21, 2.0 ** -20)}

ATTEND = {
    "single": [(0, 1), (15, 1), (63, 1), (64, 1), (300, 1), (128, 1)],
    "one": [(436, 1)],
    "few": [(0, 3), (14, 5), (126, 4), (250, 2)],
    "mixed": [(0, 1), (77, 6), (64, 0), (190, 1)],
    "prompts": [(0, 90), (0, 1), (33, 50), (0, 17)],
}


@pytest.mark.parametrize("limits", [{}, {"window": 50}, {"chunk": 48}, {"window": 1}], ids=str)
@pytest.mark.parametrize("runs", sorted(ATTEND))
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", [
    (4, 2, 64, torch.bfloat16), (14, 2, 64, torch.float32), (7, 1, 128, torch.bfloat16), (8, 8, 128, torch.float32),
    (16, 1, 128, torch.bfloat16), (40, 2, 128, torch.bfloat16), (6, 2, 24, torch.bfloat16), (4, 1, 96, torch.float32)])
def test_attention(runs, n_heads, n_kv, hd, dtype, limits):
    from rust_inference_b200.kernels import attention
    step = Step(ATTEND[runs], n_kv, hd)
    step.arrays([(s + n, 0) for s, n in ATTEND[runs]])
    step.fill()
    step.arrays(ATTEND[runs])
    g = torch.Generator().manual_seed(8)
    q = torch.randn(step.n_tokens, n_heads * hd, generator=g).to(dtype)
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(hd)
    attention.attention(q.to(DEV), step.layer, out, step.context(dtype), n_heads=n_heads, n_kv_heads=n_kv, head_dim=hd, scale=scale,
                        out_scale=0.5, **limits)
    k, v, ks, vs = step.host()
    for b, (start, n) in enumerate(step.runs):
        a, e = step.cu[b], step.cu[b + 1]
        keys, vals = (plain.values(c, s, step.pages(b), start + n).double() for c, s in ((k, ks), (v, vs)))
        unit, slip = UNITS[dtype]
        want, bound = plain.attend(q[a:e].double().view(n, n_heads, hd), keys, vals, start, scale=scale, unit=unit, step=slip, **limits)
        off = (out[a:e].cpu().double().view(n, n_heads, hd) - 0.5 * want).abs()
        assert (off <= 0.5 * bound).all(), float((off / bound).max())


@pytest.mark.parametrize("runs", sorted(ATTEND))
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", [
    (14, 2, 64, torch.float32), (7, 1, 128, torch.bfloat16), (16, 1, 128, torch.float32), (16, 1, 64, torch.bfloat16), (40, 2, 128, torch.bfloat16),
    (7, 1, 64, torch.bfloat16), (4, 1, 128, torch.float32)])
def test_attention_in_wide_tiles(runs, n_heads, n_kv, hd, dtype):
    """What the host knows of the lengths decides which tiles of rows a step is cut into, not what comes out: a step that might be long."""
    from rust_inference_b200.kernels import quantized_cache as qc
    step = Step(ATTEND[runs], n_kv, hd)
    step.arrays([(s + n, 0) for s, n in ATTEND[runs]])
    step.fill()
    step.arrays(ATTEND[runs])
    step.max_len = 1 << 24
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(hd)
    qc.attend_step(q.to(DEV), step.layer, out, qc.step_of(step.context(dtype), n_heads, n_kv, hd), scale, 0, 1.0)
    k, v, ks, vs = step.host()
    for b, (start, n) in enumerate(step.runs):
        a, e = step.cu[b], step.cu[b + 1]
        keys, vals = (plain.values(c, s, step.pages(b), start + n).double() for c, s in ((k, ks), (v, vs)))
        unit, slip = UNITS[dtype]
        want, bound = plain.attend(q[a:e].double().view(n, n_heads, hd), keys, vals, start, scale=scale, unit=unit, step=slip)
        off = (out[a:e].cpu().double().view(n, n_heads, hd) - want).abs()
        assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype, runs", [
    (8, 2, 64, torch.float32, [(57, 1003), (900, 700)]), (4, 1, 128, torch.float32, [(0, 1700)]),
    (32, 8, 128, torch.bfloat16, [(1000 + 37 * i, 16 - i % 5) for i in range(12)]), (14, 2, 64, torch.bfloat16, [(2900 - i, 16) for i in range(10)]),
    (32, 8, 128, torch.bfloat16, [(31990, 1)]), (4, 1, 64, torch.bfloat16, [((37 * i) % 200, int(i % 7 != 3)) for i in range(301)]),
    (2, 2, 128, torch.float32, [((91 * i) % 333, 1 + i % 3) for i in range(140)])])
def test_attention_of_many_rows_and_keys(n_heads, n_kv, hd, dtype, runs, window):
    """Steps that fill the SMs for long, and of more sequences than a block has threads; some of their tokens."""
    from rust_inference_b200.kernels import attention
    step = Step(runs, n_kv, hd)
    for t in (step.layer.k_scale, step.layer.v_scale):
        t.uniform_(0.004, 0.016, generator=torch.Generator(DEV).manual_seed(3))
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(10)).to(dtype)
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(hd)
    attention.attention(q.to(DEV), step.layer, out, step.context(dtype), n_heads=n_heads, n_kv_heads=n_kv, head_dim=hd, scale=scale, window=window)
    assert out.isfinite().all()
    k, v, ks, vs = step.host()
    unit, slip = UNITS[dtype]
    for b, (start, n) in list(enumerate(runs))[::max(1, len(runs) // 10) if len(runs) > 100 else 1][:3 if len(runs) < 100 else None]:
        keys, vals = (plain.values(c, s, step.pages(b), start + n).double() for c, s in ((k, ks), (v, vs)))
        for t in sorted({0, n // 3, n // 2, n - 1}) if n else ():
            row, pos = step.cu[b] + t, start + t
            want, bound = plain.attend(q[row:row + 1].double().view(1, n_heads, hd), keys[:pos + 1], vals[:pos + 1], pos, scale=scale, unit=unit,
                                       step=slip, window=window)
            off = (out[row].cpu().double().view(1, n_heads, hd) - want).abs()
            assert (off <= bound).all(), (b, t, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_over_codes_off_a_16_byte_boundary(dtype):
    """Such a layer is read back."""
    from rust_inference_b200.kernels import attention
    qc = _qc()
    step = Step([(77, 3), (10, 1)], 2, 64)
    step.arrays([(80, 0), (11, 0)])
    step.fill()
    step.arrays([(77, 3), (10, 1)])
    codes = [torch.empty(t.numel() + 1, dtype=torch.int8, device=DEV)[1:].view(t.shape).copy_(t) for t in (step.layer.k, step.layer.v)]
    moved = qc.QuantizedPages(*codes, step.layer.k_scale, step.layer.v_scale)
    q = torch.randn(step.n_tokens, 8 * 64, device=DEV).to(dtype)
    got, want = torch.empty_like(q), torch.empty_like(q)
    for layer, out in ((moved, got), (step.layer, want)):
        attention.attention(q, layer, out, step.context(dtype), n_heads=8, n_kv_heads=2, head_dim=64, scale=0.125)
    assert (got.float() - want.float()).abs().max() <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-4) * want.float().abs().max()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_past_what_it_does_not_see(hd, dtype):
    """Codes and scales behind a sequence's end, and blocks before the window, may hold anything; a seen block that is marked
    as no number makes the result NaN, and only for who sees it."""
    from rust_inference_b200.kernels import attention
    step = Step([(100, 1), (40, 2), (150, 1)], 1, hd)
    step.arrays([(101, 0), (42, 0), (151, 0)])
    step.fill()
    step.arrays([(100, 1), (40, 2), (150, 1)])
    for t in (step.layer.k_scale, step.layer.v_scale):
        t[step.pages(0)[1].item(), :, 3] = math.nan              # positions 112..127: behind the end of sequence 0
        t[step.pages(1)[0].item(), :, 3] = 1e30                  # positions 48..63: behind the end of sequence 1
        t[step.pages(2)[0].item(), :, 0] = math.nan              # positions 0..15: before sequence 2's window
    q = torch.randn(step.n_tokens, 4 * hd, device=DEV).to(dtype)
    out = torch.empty(step.n_tokens, 4 * hd, dtype=dtype, device=DEV)
    call = dict(n_heads=4, n_kv_heads=1, head_dim=hd, scale=0.1)
    attention.attention(q, step.layer, out, step.context(dtype), window=100, **call)
    assert out.isfinite().all()
    attention.attention(q, step.layer, out, step.context(dtype), **call)
    assert out[:3].isfinite().all() and out[3].isnan().all()


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_past_what_they_do_not_see(hd, dtype, window):
    """The same for prompts of many rows: who does not see a marked block is as without it, and who does is no number."""
    from rust_inference_b200.kernels import attention
    runs = [(0, 130), (37, 90), (0, 50)]
    step = Step(runs, 2, hd)
    step.arrays([(s + n, 0) for s, n in runs])
    step.fill()
    step.arrays(runs)
    q = torch.randn(step.n_tokens, 8 * hd, device=DEV).to(dtype)
    call = dict(n_heads=8, n_kv_heads=2, head_dim=hd, scale=0.1, window=window)
    want = torch.empty_like(q)
    attention.attention(q, step.layer, want, step.context(dtype), **call)
    assert want.isfinite().all()
    step.layer.k_scale[step.pages(0)[1].item(), 0, 0] = math.nan         # sequence 0: positions 64..79 of kv head 0
    step.layer.v_scale[step.pages(1)[1].item(), 1, 1] = math.nan         # sequence 1: positions 80..95 of kv head 1
    step.layer.v_scale[step.pages(2)[0].item(), :, 3] = math.nan         # sequence 2: its last block
    got = torch.empty_like(q)
    attention.attention(q, step.layer, got, step.context(dtype), **call)
    bad = torch.zeros(step.n_tokens, 8, dtype=torch.bool)
    for b, head, low, high in ((0, 0, 64, 80), (1, 1, 80, 96), (2, 0, 48, 64), (2, 1, 48, 64)):
        start, n = runs[b]
        for t in range(n):
            pos = start + t
            first = max(0, pos - window + 1) if window else 0
            if pos >= low and first < high:
                bad[step.cu[b] + t, 4 * head:4 * head + 4] = True
    got, want = got.view(-1, 8, hd).cpu(), want.view(-1, 8, hd).cpu()
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], want[~bad]) or (got[~bad].float() - want[~bad].float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


def test_attention_of_large_and_small_queries_and_scales():
    """Queries, keys and values far from one: the float32 result stays as near as the sums allow."""
    from rust_inference_b200.kernels import attention
    for size_q, size_k, size_v in ((1e-20, 1e20, 1e-25), (1e15, 1e-15, 1e20), (1e3, 1e-3, 1.0)):
        step = Step([(90, 1), (30, 2)], 2, 128)
        step.arrays([(91, 0), (32, 0)])
        step.fill()
        step.arrays([(90, 1), (30, 2)])
        step.layer.k_scale.mul_(size_k)
        step.layer.v_scale.mul_(size_v)
        q = torch.randn(step.n_tokens, 4 * 128, device=DEV) * size_q
        out = torch.empty_like(q)
        attention.attention(q, step.layer, out, step.context(torch.float32), n_heads=4, n_kv_heads=2, head_dim=128, scale=0.09)
        k, v, ks, vs = step.host()
        for b, (start, n) in enumerate(step.runs):
            a, e = step.cu[b], step.cu[b + 1]
            keys, vals = (plain.values(c, s, step.pages(b), start + n).double() for c, s in ((k, ks), (v, vs)))
            unit, slip = UNITS[torch.float32]
            want, bound = plain.attend(q[a:e].double().cpu().view(n, 4, 128), keys, vals, start, scale=0.09, unit=unit, step=slip)
            assert ((out[a:e].cpu().double().view(n, 4, 128) - want).abs() <= bound).all()


def test_refusals():
    from rust_inference_b200.kernels.ops import KernelError
    qc = _qc()
    step = Step([(0, 4)], 2, 64)
    rows = torch.zeros(4, 8 * 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(4, 4 * 64, dtype=torch.bfloat16, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(4, 64))

    def write(src=rows, q_out=q, c=cos, s=sin, layer=step.layer, table=step.page_table, start=step.seq_start, **other):
        qc.write(src, q_out, c, s, layer, table, step.seq_slot, start, step.cu_seqlens,
                 **dict(dict(n_heads=4, n_kv_heads=2, head_dim=64, max_new=4), **other))

    write()
    bad = [dict(src=rows[:, :-1]), dict(src=rows[:, :7 * 64].contiguous()), dict(src=rows.half()), dict(q_out=q.float()),
           dict(c=cos.double()), dict(c=cos[:, :31].contiguous()), dict(table=step.page_table.long()), dict(start=step.seq_start.cpu()),
           dict(head_dim=32), dict(n_kv_heads=1), dict(style=2), dict(bias=torch.zeros(8 * 64, device=DEV, dtype=torch.bfloat16)),
           dict(rot_dims=63, c=cos[:, :31].contiguous(), s=sin[:, :31].contiguous()), dict(src=rows.cpu())]
    for case in bad:
        with pytest.raises(KernelError):
            write(**case)
    n = step.layer                              # layers of another make are refused when they are put together
    for tensors in [(n.k.float(), n.v, n.k_scale, n.v_scale), (n.k, n.v, n.k_scale[:, :, :2].contiguous(), n.v_scale),
                    (n.k, n.v, n.k_scale, n.v_scale.double()), (n.k.cpu(), n.v, n.k_scale, n.v_scale), (n.k, n.v[:1], n.k_scale, n.v_scale),
                    (n.k[:, :, ::2], n.v[:, :, ::2], n.k_scale, n.v_scale), (n.k.transpose(1, 2), n.v, n.k_scale, n.v_scale)]:
        with pytest.raises(KernelError):
            qc.QuantizedPages(*tensors)
    k = torch.zeros(4, 2, 64, device=DEV)
    call = dict(max_len=4, cu_rows=step.cu_seqlens)
    qc.read(step.layer, k, k.clone(), step.page_table, step.seq_slot, step.seq_start, step.seq_len, **call)
    for out in (k.half(), k[:, :1].contiguous(), k.transpose(0, 1), torch.zeros(4, 2, 32, device=DEV)):
        with pytest.raises(KernelError):
            qc.read(step.layer, out, out, step.page_table, step.seq_slot, step.seq_start, step.seq_len, **call)
    with pytest.raises(KernelError):            # without cu_rows: the cache's shape
        qc.read(step.layer, k, k.clone(), step.page_table, step.seq_slot, step.seq_start, step.seq_len, max_len=4)
