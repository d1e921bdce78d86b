"""Weights in microscaled 4 bits, rows in 8 and their products against 64-bit arithmetic.

Tolerances.  What is held is exact: the nearest numbers, ties to even, bit for bit; float32 and bfloat16 hold them.  A norm is formed in
64 bits and rounded once to 24 before it is rounded to 4 bits of mantissa, so a result is as near to the exact norm y as the nearest number,
but for 2^-22 |y|.  A product's terms are exact (4 + 2 bits of mantissa, powers of two); the tensor cores add 32 of them, aligned, to a
float32 sum, K / 32 times, each time off by at most a unit in the last place (2^-23) of what has been added up in magnitude, and a handful
of pieces of K and a bias join the same way: (K / 32 + 16) 2^-23 sum |x w|, and half a step of the result's type."""
import math

import pytest
import torch

import plain_microscaled as plain

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def spread(n, k, seed, dtype=torch.float32, wide=6.0):
    """Numbers whose blocks lie powers of two apart."""
    g = gen(seed)
    x = torch.randn(n, k, generator=g) * torch.exp2(wide * torch.randn(n, -(-k // 32), generator=g).repeat_interleave(32, 1)[:, :k])
    return x.to(dtype)


def context(dtype=torch.bfloat16):
    from rust_inference_b200.engine.context import StepContext, Workspace
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    return StepContext(n_tokens=1, n_seqs=1, token_ids=i, token_pos=i, token_seq=i, seq_slot=i, seq_start=i, seq_len=i, cu_seqlens=i, logit_rows=i,
                       n_logit_rows=0, max_new=1, max_len=1, all_single=True, page_table=i[None], page_size=64, dtype=dtype, device=i.device,
                       workspace=Workspace(i.device))


def check_status():
    from rust_inference_b200.kernels import tcgen05
    torch.cuda.synchronize()
    tcgen05.check_status()


SIZES = [(1, 1), (1, 31), (2, 32), (3, 33), (5, 127), (129, 128), (31, 129), (300, 1000), (257, 4096), (130, 2052)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", SIZES)
def test_held_numbers_are_the_nearest(n, k, dtype):
    from rust_inference_b200.kernels import microscaled
    x = spread(n, k, 1000 * n + k, dtype)
    for held, numbers in ((microscaled.Matrix.of(x.to(DEV)), plain.FOUR), (microscaled.quantize(x.to(DEV)), plain.EIGHT)):
        want = plain.nearest(x, numbers)
        for out in (torch.float32, torch.bfloat16):
            got = microscaled.values(held, out)
            assert got.dtype == out and torch.equal(got.double().cpu(), want)


def test_ties_borders_and_numbers_that_are_none():
    from rust_inference_b200.kernels import microscaled
    rows = []
    for numbers in (plain.FOUR, plain.EIGHT):
        t = torch.tensor(numbers, dtype=torch.float64)
        mid = (t[1:] + t[:-1]) / 2
        for e in (0.0, -20.0, 50.0, -100.0):
            for v in (t, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)):
                for part in (v * 2.0 ** e).split(31):
                    row = torch.zeros(32, dtype=torch.float64)
                    row[0] = numbers[-1] * 2.0 ** e                      # the type's largest: the power of two is 2^e
                    row[1:1 + len(part)] = part
                    rows += [row, -row]
        for top in (numbers[-1] * (1 + 2.0 ** -23), numbers[-1], numbers[-1] * (1 - 2.0 ** -23)):
            row = torch.full((32,), 0.3, dtype=torch.float64)
            row[7] = top
            rows.append(row)
    rows += [torch.zeros(32).double(), torch.full((32,), 1e-45).double(), torch.full((32,), 2.0 ** -126).double(), torch.full((32,), 3.4e38).double(),
             torch.arange(32).double() * 1e-40, torch.arange(32).double() * 2.0 ** -128]
    for bad in (math.inf, -math.inf, math.nan):
        row = torch.arange(32).double()
        row[5] = bad
        rows.append(row)
    x = torch.stack(rows).float()
    for held, numbers in ((microscaled.Matrix.of(x.to(DEV)), plain.FOUR), (microscaled.quantize(x.to(DEV)), plain.EIGHT)):
        want, got = plain.nearest(x, numbers).float(), microscaled.values(held, torch.float32).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_rows_apart_and_off_a_boundary():
    from rust_inference_b200.kernels import microscaled
    for dtype in (torch.float32, torch.bfloat16):
        wide = spread(70, 401, 3, dtype).to(DEV)
        for x in (wide[:, :256], wide[:, 1:257], wide[3:, 100:399], wide[::2, :64], wide.t()):
            want4, want8 = plain.nearest(x.cpu(), plain.FOUR), plain.nearest(x.cpu(), plain.EIGHT)
            assert torch.equal(microscaled.values(microscaled.Matrix.of(x)).double().cpu(), want4)
            if x.stride(1) == 1:
                assert torch.equal(microscaled.values(microscaled.quantize(x)).double().cpu(), want8)


@pytest.mark.parametrize("n,k", [(1, 1), (3, 63), (130, 257), (256, 384)])
def test_matrix_from_a_files_codes(n, k):
    from rust_inference_b200.kernels import microscaled
    x = spread(n, k, 5)
    want = plain.nearest(x, plain.FOUR)
    codes, exponents = plain.codes_of(want, k)
    if k % 2:
        codes[:, -1] |= 0x70                                # what lies behind a row's end says nothing
    m = microscaled.Matrix.of_codes(codes.to(DEV), exponents.to(DEV), k)
    assert torch.equal(microscaled.values(m).double().cpu(), want)
    other = microscaled.Matrix.of(want.float().to(DEV))    # the same rule on the same numbers (3.2 becomes 3, which is 6 times half as much)
    assert torch.equal(m.exponents, other.exponents) and torch.equal(m.codes, other.codes)


@pytest.mark.parametrize("branch", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 31), (2, 896), (9, 1333), (3, 4096), (5, 8960), (2, 18944), (700, 260)])
def test_norm(n, k, branch):
    from rust_inference_b200.kernels import microscaled
    g = gen(n * k)
    x = 3 * torch.randn(n, k, generator=g) + 0.5
    b = None if branch is None else torch.randn(n, k, generator=g).to(branch)
    w = 1 + 0.2 * torch.randn(k, generator=g)
    want_total, y = plain.rmsnorm(x, b, w, 1e-5)
    near = plain.nearest(y, plain.EIGHT)
    rows = microscaled.Rows(n, k)
    for total in ("none", "other", "same"):
        xd = x.to(DEV)
        to = {"none": None, "other": torch.full_like(xd, math.nan), "same": xd}[total]
        microscaled.rmsnorm(xd, w.to(DEV), 1e-5, rows, branch=None if b is None else b.to(DEV), total=to)
        if to is not None:
            assert torch.equal(to.cpu(), want_total)
        got = microscaled.values(rows).double().cpu()
        assert ((got - y).abs() <= (near - y).abs() + 2.0 ** -22 * y.abs()).all()


def exact_product(x, w):
    """x W^T and the sum of its terms' magnitudes, 64 bits."""
    x, w = plain.nearest(x, plain.EIGHT).to(DEV), plain.nearest(w, plain.FOUR).to(DEV)
    return x @ w.t(), x.abs() @ w.abs().t()


def bound(k, mass, y, dtype):
    return (k / 32 + 16) * 2.0 ** -23 * mass + HALF_STEP[dtype] * y.abs()


PRODUCTS = [(1, 1, 1), (1, 128, 128), (2, 130, 64), (1, 896, 896), (7, 1000, 1333), (8, 3584, 3584), (16, 257, 2048), (17, 640, 384), (33, 129, 4097),
            (64, 2560, 2048), (61, 300, 8960), (100, 129, 640), (127, 1152, 896), (128, 256, 512), (129, 200, 300), (200, 5000, 256), (333, 2560, 2048),
            (1000, 640, 1536), (3, 40000, 160), (5, 128, 18944), (130, 41000, 200)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, dtype):
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context(dtype)
    x, w = spread(m, k, 11 * m + k, dtype, 1.0), spread(n, k, 13 * n + k, wide=1.0)
    b = torch.randn(n, generator=gen(n)).to(DEV)
    y, mass = exact_product(x, w)
    held = microscaled.Matrix.of(w.to(DEV))
    xd = x.to(DEV)
    for bias in (None, b):
        out = torch.full((m, n), math.nan, dtype=dtype, device=DEV)
        linear.project(xd, held, out, ctx, bias=bias)
        want = y if bias is None else y + bias.double()
        assert ((out.double() - want).abs() <= bound(k, mass + (0 if bias is None else bias.double().abs()), want, dtype)).all()
    start = torch.randn(m, n, generator=gen(m)).to(DEV)
    out = start.clone()
    linear.into_residual(microscaled.quantize(xd), held, out, ctx)
    want = y + start.double()
    assert ((out.double() - want).abs() <= bound(k, mass + start.double().abs(), want, torch.float32)).all()
    again = start.clone()
    linear.into_residual(xd, held, again, ctx)
    assert torch.equal(out, again)
    check_status()


@pytest.mark.parametrize("form", [None, "bounded"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4864, 896), (8, 1000, 1333), (9, 18944, 256), (16, 300, 2048), (31, 640, 640), (64, 1100, 512), (100, 256, 2048),
                                   (128, 700, 300), (129, 200, 300), (333, 1500, 640), (700, 129, 1000), (200, 20000, 130), (128, 25000, 129)])
def test_gated_and_into_eight_bits(m, n, k, form):
    from rust_inference_b200.kernels import linear, microscaled, ops
    ctx = context()
    x = spread(m, k, 3 * m + k, wide=0.5)
    wg, wu = (spread(n, k, s + n + k, wide=0.5) / math.sqrt(k) for s in (1, 2))
    f = None if form is None else ops.gate_form(alpha=1.702, limit=1.5, shift=1.0, device=DEV)
    g, gm = exact_product(x, wg)
    u, um = exact_product(x, wu)
    want = plain.gate(g, u, f)
    # gate and up are off by so much, and the gate's slope is 1.1 at most in size (alpha = 1.702: 1.1 too); a few units in the last place of float32 beside it
    eg, eu = ((k / 32 + 16) * 2.0 ** -23 * v for v in (gm, um))
    up = u.abs() + 1 if f is not None else u.abs()
    off = 1.2 * eg * (up + eu) + g.abs() * eu + 2.0 ** -20 * (g.abs() * up)
    held = [microscaled.Matrix.of(w.to(DEV)) for w in (wg, wu)]
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), math.nan, dtype=dtype, device=DEV)
        linear.gated(x.to(DEV), *held, out, ctx, form=f)
        assert ((out.double() - want).abs() <= off + HALF_STEP[dtype] * want.abs() * 1.01).all()
    rows = microscaled.Rows(m, n)
    rows.codes.fill_(255)
    linear.gated(x.to(DEV), *held, rows, ctx, form=f)
    got = microscaled.values(rows).double()
    # a block's step follows its largest number: half a step is 2^-4 of a number, or 2^-10 times 2^e, which is at most the block's largest / 224
    near = plain.nearest(want.cpu(), plain.EIGHT).to(DEV)
    wide = torch.nn.functional.pad(want.abs() + off, (0, -n % 32)).view(m, -1, 32).amax(dim=2, keepdim=True).expand(-1, -1, 32).reshape(m, -1)[:, :n]
    assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * wide / 224) + off * 1.1).all()
    assert float((got != near).double().mean()) < 0.01
    # behind a row's end there are zeros, for the next product
    if n % 128:
        assert not rows.codes.view(m, -1)[:, n:].any()
    # and the next product reads them as they lie
    wd = spread(200, n, 9, wide=0.5)
    down = microscaled.Matrix.of(wd.to(DEV))
    out = torch.empty(m, 200, dtype=torch.float32, device=DEV)
    linear.project(rows, down, out, ctx)
    w8 = plain.nearest(wd, plain.FOUR).to(DEV)
    y, mass = got @ w8.t(), got.abs() @ w8.abs().t()
    assert ((out.double() - y).abs() <= bound(n, mass, y, torch.float32)).all()
    check_status()


@pytest.mark.parametrize("m", [1, 9, 130, 600])
def test_activated(m):
    from rust_inference_b200.kernels import linear, microscaled, ops
    ctx = context()
    x, w = spread(m, 500, m, wide=0.5), spread(390, 500, 77, wide=0.5) / 20
    form = torch.tensor(ops.RELU_SQUARED_FORM, dtype=torch.float32, device=DEV)
    y, mass = exact_product(x, w)
    want = y.clamp(min=0) ** 2
    off = (500 / 32 + 16) * 2.0 ** -23 * mass
    off = 2 * off * (y.abs() + off) + 2.0 ** -21 * want
    held = microscaled.Matrix.of(w.to(DEV))
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, 390), math.nan, dtype=dtype, device=DEV)
        linear.activated(x.to(DEV), held, out, ctx, form)
        assert ((out.double() - want).abs() <= off + HALF_STEP[dtype] * want * 1.01).all()
    rows = microscaled.Rows(m, 390)
    linear.activated(x.to(DEV), held, rows, ctx, form)
    got = microscaled.values(rows).double()
    assert float((got != plain.nearest(want.cpu(), plain.EIGHT).to(DEV)).double().mean()) < 0.01
    check_status()


@pytest.mark.parametrize("m", [3, 130, 600])
def test_numbers_that_are_none_stay_where_they_are(m):
    """A NaN or an infinity makes its token's results, or its feature's, NaN, and no others."""
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context(torch.float32)
    x, w = spread(m, 300, 1, wide=0.5), spread(260, 300, 2, wide=0.5)
    x[1, 7], x[2, 299], w[5, 0], w[259, 100] = math.nan, math.inf, -math.inf, math.nan
    out = torch.zeros(m, 260, dtype=torch.float32, device=DEV)
    linear.project(x.to(DEV), microscaled.Matrix.of(w.to(DEV)), out, ctx)
    bad = torch.zeros(m, 260, dtype=torch.bool)
    bad[1:3] = True
    bad[:, [5, 259]] = True
    assert torch.equal(torch.isnan(out).cpu(), bad) and torch.isfinite(out.cpu()[~bad]).all()
    y, mass = exact_product(x.nan_to_num(0, 0, 0), w.nan_to_num(0, 0, 0))
    good = ~bad.to(DEV)
    assert ((out.double() - y).abs() <= bound(300, mass, y, torch.float32))[good].all()
    rows = microscaled.Rows(m, 260)
    linear.gated(x.to(DEV), microscaled.Matrix.of(w.to(DEV)), microscaled.Matrix.of(w.to(DEV)), rows, ctx)
    got = microscaled.values(rows).cpu()
    blocks = torch.zeros(m, 260, dtype=torch.bool)
    blocks[1:3] = True
    blocks[:, 0:32] = True
    blocks[:, 256:260] = True
    assert torch.equal(torch.isnan(got), blocks)
    check_status()


@pytest.mark.parametrize("up", [-120, -60, 0, 60, 110])
def test_far_powers_of_two(up):
    """Powers of two far apart cancel in the product, also where each alone is near float32's ends."""
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context(torch.float32)
    x, w = spread(5, 256, 3, wide=0.5), spread(130, 256, 4, wide=0.5)
    out = torch.empty(5, 130, dtype=torch.float32, device=DEV)
    linear.project((x * 2.0 ** up).to(DEV), microscaled.Matrix.of((w * 2.0 ** -up).to(DEV)), out, ctx)
    y, mass = exact_product(x * 2.0 ** up, w * 2.0 ** -up)
    assert ((out.double() - y).abs() <= bound(256, mass, y, torch.float32)).all()


def test_results_off_a_boundary_and_in_wider_memory():
    """Results that begin off a 16-byte boundary; what lies before and behind them stays."""
    from rust_inference_b200.kernels import linear, microscaled
    for m in (2, 40, 300, 1000):
        x, w = spread(m, 256, 5, wide=0.5), spread(256, 256, 6, wide=0.5)
        y, mass = exact_product(x, w)
        held, xd = microscaled.Matrix.of(w.to(DEV)), x.to(DEV)
        for dtype in (torch.bfloat16, torch.float32):
            ctx = context(dtype)
            room = torch.full((m * 256 + 9,), 7.0, dtype=dtype, device=DEV)
            out = room[1:1 + m * 256].view(m, 256)
            linear.project(xd, held, out, ctx)
            assert ((out.double() - y).abs() <= bound(256, mass, y, dtype)).all()
            if dtype is torch.float32:
                linear.into_residual(xd, held, out, ctx)
                assert ((out.double() - 2 * y).abs() <= bound(256, 2 * mass, 2 * y, dtype)).all()
            assert float(room[0]) == 7.0 and (room[1 + m * 256:] == 7.0).all()
    # plain rows off a boundary, and rows apart
    w = spread(70, 64, 8, wide=0.5)
    held = microscaled.Matrix.of(w.to(DEV))
    wide = spread(3, 200, 9, wide=0.5).to(DEV)
    for x in (wide[:, :64], wide[:, 3:67], wide[:, 8:72], wide[:1, 1:65], wide[::2, :64]):
        out = torch.empty(x.shape[0], 70, dtype=torch.float32, device=DEV)
        linear.project(x, held, out, context(torch.float32))
        y, mass = exact_product(x.cpu(), w)
        assert ((out.double() - y).abs() <= bound(64, mass, y, torch.float32)).all()
    check_status()


def test_no_tokens():
    from rust_inference_b200.kernels import linear, microscaled
    held = microscaled.Matrix.of(torch.ones(5, 40, device=DEV))
    out = torch.empty(0, 5, dtype=torch.bfloat16, device=DEV)
    assert linear.project(torch.empty(0, 40, dtype=torch.bfloat16, device=DEV), held, out, context()) is out


@pytest.mark.parametrize("m", [1, 8, 40, 200, 700])
def test_a_run_of_them_captured_and_again(m):
    """What a decoder's feed-forward does with them, the stream on its way through: against 64 bits, the same bits every time, captured, replayed over
    other inputs, and on another stream."""
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context()
    k, inner = 640, 1100
    weight = (1 + 0.1 * torch.randn(k, generator=gen(1))).to(DEV)
    wg, wu, wd = spread(inner, k, 2, wide=0.3) / 12, spread(inner, k, 3, wide=0.3) / 12, spread(k, inner, 4, wide=0.3) / 16
    g, u, d = (microscaled.Matrix.of(w.to(DEV)) for w in (wg, wu, wd))
    normed, act = microscaled.Rows(m, k), microscaled.Rows(m, inner)
    stream, branch = torch.empty(m, k, device=DEV), torch.empty(m, k, dtype=torch.bfloat16, device=DEV)
    total = torch.empty(m, k, device=DEV)

    def step():
        microscaled.rmsnorm(stream, weight, 1e-6, normed, branch=branch, total=total)
        linear.gated(normed, g, u, act, ctx)
        linear.into_residual(act, d, total, ctx)

    def fill(seed):
        stream.copy_(2 * torch.randn(m, k, generator=gen(seed)))
        branch.copy_(torch.randn(m, k, generator=gen(seed + 1)))

    def want():
        t, y = plain.rmsnorm(stream, branch, weight, 1e-6)
        h = plain.nearest(y, plain.EIGHT)
        w4 = [plain.nearest(w, plain.FOUR) for w in (wg, wu, wd)]
        a = plain.gate(h @ w4[0].t(), h @ w4[1].t())
        a8 = plain.nearest(a, plain.EIGHT)
        off = (a - a8).abs() @ w4[2].abs().t()
        return t.double() + a8 @ w4[2].t(), off

    fill(10)
    step()
    first = total.clone()
    y, off = want()
    # a number of the gate's next to the middle of two falls to the other side now and then: a step instead of none, one of a thousand at most
    assert ((first.double().cpu() - y).abs() <= 0.25 * off + 1e-4 * y.abs() + 1e-5).all()
    for _ in range(3):
        step()
        assert torch.equal(total, first)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        step()
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(total, first)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for seed in (20, 10, 30):
        fill(seed)
        graph.replay()
        replayed = total.clone()
        step()
        assert torch.equal(replayed, total)
        if seed == 10:
            assert torch.equal(replayed, first)
    check_status()


def test_a_matrix_is_read_right_behind_its_making():
    """Products begin their reads of a matrix before the kernel before them has ended: not before the matrix is there."""
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context()
    x = microscaled.quantize(spread(2, 4096, 1, wide=0.5).to(DEV))
    ws = [spread(4096, 4096, 40 + i, torch.bfloat16, wide=0.5).to(DEV) for i in range(2)]
    want = []
    for w in ws:
        m = microscaled.Matrix.of(w)
        torch.cuda.synchronize()
        want.append(linear.project(x, m, torch.empty(2, 4096, dtype=torch.float32, device=DEV), ctx))
    for turn in range(20):
        m = microscaled.Matrix.of(ws[turn % 2])                    # (in the memory of the one before)
        out = linear.project(x, m, torch.empty(2, 4096, dtype=torch.float32, device=DEV), ctx)
        assert torch.equal(out, want[turn % 2])
        del m


def test_refusals():
    from rust_inference_b200.kernels import linear, microscaled, ops
    KE = ops.KernelError
    ctx = context()
    w = microscaled.Matrix.of(torch.ones(40, 64, device=DEV))
    x = torch.ones(3, 64, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(3, 40, dtype=torch.bfloat16, device=DEV)
    f32 = torch.empty(3, 40, device=DEV)
    rows = microscaled.quantize(x)
    bad = [
        lambda: linear.project(x[:, :63], w, out, ctx), lambda: linear.project(x, w, out[:2], ctx), lambda: linear.project(x, w, out.t(), ctx),
        lambda: linear.project(x.half(), w, out, ctx), lambda: linear.project(x, w, out.half(), ctx), lambda: linear.project(x.cpu(), w, out, ctx),
        lambda: linear.project(x, w, out, ctx, bias=torch.ones(39, device=DEV)), lambda: linear.project(x, w, out, ctx, bias=torch.ones(40, device=DEV).half()),
        lambda: linear.into_residual(x, w, out, ctx), lambda: linear.into_residual(x, w, microscaled.Rows(3, 40), ctx),
        lambda: linear.gated(x, w, microscaled.Matrix.of(torch.ones(41, 64, device=DEV)), out, ctx),
        lambda: linear.gated(x, w, torch.ones(40, 64, device=DEV), out, ctx), lambda: linear.logits(x, w, f32, ctx, silu_cols=torch.ones(1, device=DEV)),
        lambda: linear.project(rows, microscaled.Matrix.of(torch.ones(64, 64, device=DEV)), rows, ctx),
        lambda: linear.project(rows, w, microscaled.Rows(3, 41), ctx), lambda: microscaled.quantize(x, microscaled.Rows(4, 64)),
        lambda: microscaled.product(x, w, out, ctx, bias=torch.ones(40, device=DEV), add=True), lambda: microscaled.product(x, w, out, ctx, form=torch.ones(5, device=DEV)),
        lambda: microscaled.Matrix.of(torch.ones(0, 4, device=DEV)), lambda: microscaled.Matrix.of(torch.ones(4, device=DEV)),
        lambda: microscaled.Matrix.of(torch.ones(4, 4, dtype=torch.float16, device=DEV)), lambda: microscaled.Rows(0, 4), lambda: microscaled.Rows(4, 0),
        lambda: microscaled.Rows(4, 64, codes=torch.zeros(4, dtype=torch.uint8, device=DEV)),
        lambda: microscaled.Rows(1, 64, codes=torch.zeros(129, dtype=torch.uint8, device=DEV)[1:]),
        lambda: microscaled.rmsnorm(x, torch.ones(64, device=DEV), 1e-5, rows), lambda: microscaled.rmsnorm(x.float(), torch.ones(63, device=DEV), 1e-5, rows),
        lambda: microscaled.rmsnorm(x.float(), torch.ones(64, device=DEV), 1e-5, microscaled.Rows(2, 64)),
        lambda: microscaled.rmsnorm(x.float(), torch.ones(64, device=DEV), 1e-5, rows, branch=x[:2]),
        lambda: microscaled.rmsnorm(x.float(), torch.ones(64, device=DEV), 1e-5, rows, total=torch.empty(3, 64, dtype=torch.bfloat16, device=DEV)),
        lambda: microscaled.values(rows, torch.float16), lambda: microscaled.values(w, torch.float32, out=torch.empty(64, 40, device=DEV)),
        lambda: microscaled.Matrix.of_codes(torch.zeros(4, 5, dtype=torch.uint8, device=DEV), torch.zeros(4, 1, dtype=torch.uint8, device=DEV), 12),
        lambda: microscaled.Matrix.of_codes(torch.zeros(4, 6, dtype=torch.uint8, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV), 12),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KE):
            call()
            pytest.fail(f"call {i} was not refused")
    # memory that a call reads and writes at different places
    room = torch.zeros(4 * 64 + 64, device=DEV)
    stream = room[:3 * 64].view(3, 64)
    with pytest.raises(KE, match="apart"):
        microscaled.rmsnorm(stream, torch.ones(64, device=DEV), 1e-5, rows, total=room[64:4 * 64].view(3, 64))
    square = microscaled.Matrix.of(torch.ones(64, 64, device=DEV))
    with pytest.raises(KE, match="apart"):
        linear.project(x, square, x, ctx)
    check_status()


def test_a_files_codes_on_another_device_than_the_current_one(monkeypatch):
    from rust_inference_b200.kernels import microscaled, ops
    codes, exponents = torch.zeros(4, 6, dtype=torch.uint8, device=DEV), torch.zeros(4, 1, dtype=torch.uint8, device=DEV)
    microscaled.Matrix.of_codes(codes, exponents, 12)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ops.KernelError, match="current device"):
        microscaled.Matrix.of_codes(codes, exponents, 12)


@pytest.mark.parametrize("n,k", [(896, 896), (1536, 1536), (2048, 2048), (3584, 3584), (1152, 904), (200, 8)])
def test_a_few_plain_rows_are_what_rows_in_eight_bits_are(n, k):
    """However a product comes by its rows, its results are the same to the bit."""
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context()
    held = microscaled.Matrix.of(spread(n, k, n + k, wide=1.0).to(DEV))
    for m in (1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 13, 16, 17):
        for dtype in (torch.bfloat16, torch.float32):
            x = spread(m, k + 8, 3 * m + k, dtype, 2.0).to(DEV)[:, :k]
            out, again = (torch.full((m, n), math.nan, device=DEV) for _ in range(2))
            linear.logits(x, held, out, ctx)
            linear.logits(microscaled.quantize(x), held, again, ctx)
            assert torch.equal(out, again)
            rows, from_rows = microscaled.Rows(m, n), microscaled.Rows(m, n)
            linear.gated(x, held, held, rows, ctx)
            linear.gated(microscaled.quantize(x), held, held, from_rows, ctx)
            assert torch.equal(microscaled.values(rows), microscaled.values(from_rows))
    check_status()


@pytest.fixture(params=["pairs of SMs", "single SMs"])
def one_kernel(request):
    from rust_inference_b200.kernels import microscaled
    microscaled.set_pairs(1 if request.param == "pairs of SMs" else 1 << 30)
    yield
    microscaled.set_pairs()


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (2, 130, 64), (61, 300, 8960), (129, 200, 300), (200, 5000, 256), (257, 385, 129), (333, 2560, 2048), (1000, 640, 1536),
                                   (130, 41000, 200), (513, 20100, 136)])
def test_either_kernel_takes_every_product(one_kernel, m, n, k):
    for dtype in (torch.bfloat16, torch.float32):
        test_product(m, n, k, dtype)
    if n < 10000:
        test_gated_and_into_eight_bits(m, n, k, "bounded")


@pytest.mark.parametrize("m", [1, 130, 600])
def test_either_kernel_applies_every_activation(one_kernel, m):
    test_activated(m)


def test_two_streams_at_once():
    """Products of either kernel and a plain bfloat16 one, side by side on two streams: results as alone."""
    from rust_inference_b200.kernels import linear, microscaled
    sides = []
    for s, (m, hidden, inner) in enumerate(((8, 2048, 5632), (300, 1536, 4096))):
        ctx = context()
        ws = [spread(n, k, 7 * s + n + k, torch.bfloat16, 0.3).to(DEV) / math.sqrt(k) for n, k in ((hidden, hidden), (inner, hidden), (inner, hidden), (hidden, inner))]
        held, weight = [microscaled.Matrix.of(w) for w in ws], linear.Weight(ws[0])
        x = spread(m, hidden, s, torch.bfloat16, 0.3).to(DEV)
        act, outs = microscaled.Rows(m, inner), [torch.empty(m, hidden, dtype=d, device=DEV) for d in (torch.bfloat16, torch.float32, torch.bfloat16)]

        def run(ctx=ctx, x=x, held=held, weight=weight, act=act, outs=outs):
            linear.project(x, held[0], outs[0], ctx)
            linear.gated(outs[0], held[1], held[2], act, ctx)
            linear.logits(act, held[3], outs[1], ctx)
            linear.project(x, weight, outs[2], ctx)
        sides.append((run, outs))
    alone = []
    for run, outs in sides:
        run()
        alone.append([o.clone() for o in outs])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    for _ in range(20):
        for _ in range(5):
            for (run, _), stream in zip(sides, streams):
                with torch.cuda.stream(stream):
                    run()
        torch.cuda.synchronize()
        for (_, outs), want in zip(sides, alone):
            for o, w in zip(outs[:2], want):
                assert torch.equal(o, w)
            assert ((outs[2] - want[2]).abs() <= 2.0 ** -6 * want[2].abs() + 2.0 ** -6).all()       # (its pieces of K may meet in any order)
    check_status()


def test_more_numbers_than_31_bits_count():
    from rust_inference_b200.kernels import linear, microscaled
    ctx = context()
    n, k, m = 40000, 96, 60000
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(m, k, generator=g, device=DEV)
    w = microscaled.Matrix.of(torch.randn(n, k, generator=g, device=DEV))
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    last = torch.empty(77, n, dtype=torch.bfloat16, device=DEV)
    linear.project(x[-77:], w, last, ctx)
    for pairs in (1, 1 << 30):
        microscaled.set_pairs(pairs)
        try:
            out[-77:] = math.nan
            linear.project(x, w, out, ctx)
        finally:
            microscaled.set_pairs()
        # either sum is off by (96 / 32 + 16) 2^-23 of what is added up (about 60, 200 at most); then a step of the result's type
        assert ((out[-77:].float() - last.float()).abs() <= 2.0 ** -7 * last.float().abs() + 2 * 19 * 2.0 ** -23 * 200).all()
    # rows in 8 bits of them, and read back
    rows = microscaled.quantize(out)
    assert torch.equal(microscaled.values(rows, torch.bfloat16)[-77:], microscaled.values(microscaled.quantize(out[-77:]), torch.bfloat16))
    del out
    other = microscaled.Rows(m, n)
    linear.gated(x, w, w, other, ctx)
    few = microscaled.Rows(77, n)
    linear.gated(x[-77:], w, w, few, ctx)
    a, b = microscaled.values(other, torch.bfloat16)[-77:].float(), microscaled.values(few, torch.bfloat16).float()
    # a code apart (2^-3 of a number, or 2^-9 times 2^e, which is at most the block's largest / 224), and twice that where e is one apart
    wide = b.abs().view(77, -1, 32).amax(dim=2, keepdim=True).expand(-1, -1, 32).reshape(77, n)
    assert ((a - b).abs() <= 2.0 ** -3 * b.abs() + 2.0 ** -8 * wide / 224).all() and float((a != b).float().mean()) < 1e-3
    del other, rows
    # a matrix of as many, and a norm of as many
    wide = torch.randn(m, n, dtype=torch.bfloat16, generator=g, device=DEV)
    held = microscaled.Matrix.of(wide)
    assert torch.equal(microscaled.values(held, torch.bfloat16)[-77:], microscaled.values(microscaled.Matrix.of(wide[-77:]), torch.bfloat16))
    y = torch.randn(3, n, generator=g, device=DEV)
    got = torch.empty(3, m, device=DEV)
    linear.logits(y, held, got, ctx)
    y8, w4 = microscaled.values(microscaled.quantize(y)).double(), microscaled.values(microscaled.Matrix.of(wide[-128:])).double()
    want, mass = y8 @ w4.t(), y8.abs() @ w4.abs().t()
    assert ((got[:, -128:].double() - want).abs() <= bound(n, mass, want, torch.float32)).all()
    del held
    stream = wide.float()
    rows = microscaled.rmsnorm(stream, torch.ones(n, device=DEV), 1e-6, microscaled.Rows(m, n), branch=wide, total=stream)
    again = microscaled.rmsnorm(wide[-77:].float() * 2, torch.ones(n, device=DEV), 1e-6, microscaled.Rows(77, n))
    assert torch.equal(microscaled.values(rows, torch.bfloat16)[-77:], microscaled.values(again, torch.bfloat16))
    assert torch.equal(stream[-77:], wide[-77:].float() * 2)
    check_status()


@pytest.mark.parametrize("n,k", [(2, 8191), (3, 8321), (2, 20001), (400, 129), (400, 4099), (310, 9003)])
def test_norm_of_odd_rows_longer_than_a_block_holds(n, k):
    """Rows off every boundary, the second part of which is read again; nothing behind the last row is written."""
    from rust_inference_b200.kernels import microscaled
    for branch in (None, torch.bfloat16, torch.float32):
        test_norm(n, k, branch)
    g = gen(n + k)
    room = torch.full((n * k + 64,), 7.0, device=DEV)
    stream = room[1:n * k + 1].view(n, k)                      # 4 bytes off a boundary
    x, b, w = torch.randn(n, k, generator=g), torch.randn(n, k, generator=g).bfloat16(), 1 + 0.1 * torch.randn(k, generator=g)
    stream.copy_(x)
    a, e = microscaled.Rows.sizes(n, k)
    codes, exponents = torch.full((a + 64,), 9, dtype=torch.uint8, device=DEV), torch.full((e + 64,), 9, dtype=torch.uint8, device=DEV)
    rows = microscaled.Rows(n, k, codes=codes, exponents=exponents)
    microscaled.rmsnorm(stream, w.to(DEV), 1e-5, rows, branch=b.to(DEV), total=stream)
    want, y = plain.rmsnorm(x, b, w, 1e-5)
    assert torch.equal(stream.cpu(), want) and room[0] == 7.0 and (room[n * k + 1:] == 7.0).all() and (codes[a:] == 9).all() and (exponents[e:] == 9).all()
    near = plain.nearest(y, plain.EIGHT)
    assert ((microscaled.values(rows).double().cpu() - y).abs() <= (near - y).abs() + 2.0 ** -22 * y.abs()).all()
    # the same memory for holding and reading back
    held = microscaled.quantize(stream, rows)
    out = torch.full((n * k + 64,), 5.0, device=DEV)
    microscaled.values(held, torch.float32, out=out[3:n * k + 3].view(n, k))
    assert torch.equal(out[3:n * k + 3].view(n, k).double().cpu(), plain.nearest(want, plain.EIGHT)) and (out[:3] == 5.0).all() and (out[n * k + 3:] == 5.0).all()
    assert (codes[a:] == 9).all() and (exponents[e:] == 9).all()


@pytest.mark.parametrize("call", ["linear.project(torch.ones(20, 64, dtype=torch.bfloat16, device='cuda'), w, torch.empty(20, 8, dtype=torch.bfloat16, device='cuda'), ctx)",
                                  "microscaled.values(w)", "microscaled.quantize(torch.ones(3, 7, device='cuda'))",
                                  "microscaled.rmsnorm(torch.ones(2, 64, device='cuda'), torch.ones(64, device='cuda'), 1e-6, microscaled.Rows(2, 64))"])
def test_each_call_as_a_process_first_one(call):
    """A matrix from a file's codes, and then any of the others: nothing has to have been called before."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys; sys.path[:0] = [%r, %r]\nimport torch\nfrom test_microscaled_gpu import context\n"
            "from rust_inference_b200.kernels import linear, microscaled\nctx = context()\n"
            "w = microscaled.Matrix.of_codes(torch.full((8, 32), 34, dtype=torch.uint8, device='cuda'), torch.full((8, 2), 127, dtype=torch.uint8, device='cuda'), 64)\n"
            "%s\ntorch.cuda.synchronize()\n" % (os.path.dirname(here), here, call))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
