"""Log probabilities of given tokens, entropy and alternatives, against `plain_quantized.logprobs` in 64 bits."""
import math

import pytest
import torch

import plain_quantized as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from rust_inference_b200.kernels import ops
    return ops


def _check(x, targets, top, got=None):
    got = _ops().token_logprobs(x, targets, top=top) if got is None else got
    rows, vocab = x.shape
    # the sum over the row in 32 bits: runs of at most vocab / 256 terms, then trees; exponentials and their arguments
    unit = (vocab / 256 + 32) * 2.0 ** -24
    for r in range(rows):
        logp, entropy, ids, best = plain.logprobs(x[r], int(targets[r]), top)
        pairs = [(float(got.logprob[r]), logp), (float(got.entropy[r]), entropy)]
        if top:
            assert got.top_ids[r].tolist() == ids
            pairs += list(zip(got.top_logprobs[r].tolist(), best.tolist()))
        else:
            assert got.top_ids is None and got.top_logprobs is None
        for one, want in pairs:
            if math.isfinite(want):
                assert abs(one - want) <= unit * (2 + abs(want))
            else:
                assert (math.isnan(one) and math.isnan(want)) or one == want


def _rows(rows, vocab, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 9.0
    return x.to(dtype).to(DEV), torch.randint(0, vocab, (rows,), generator=g).int().to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (3, 2, 2), (5, 31, 31), (1, 100, 64), (70, 1000, 5), (2, 1023, 20), (1, 32001, 20),
                                              (9, 32000, 1), (1, 151936, 5), (33, 128256, 20), (300, 5003, 3), (4, 152064, 0)])
def test_rows(rows, vocab, top, dtype):
    x, targets = _rows(rows, vocab, dtype)
    _check(x, targets, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("left, right", [(0, 1), (1, 0), (3, 61), (8, 8)])
@pytest.mark.parametrize("vocab", [997, 33000])
def test_rows_inside_wider_ones(left, right, vocab, dtype):
    """Rows that begin and end off every boundary; what lies beside them is larger than anything in them."""
    x, targets = _rows(6, left + vocab + right, dtype, seed=2)
    x[:, :left] = 1e30
    x[:, left + vocab:] = math.nan
    _check(x[:, left:left + vocab], (targets % vocab).contiguous(), 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1500, 40000])
def test_rows_of_every_kind(vocab, dtype):
    lowest = torch.finfo(dtype).min
    x, targets = _rows(14, vocab, dtype, seed=3)
    x[0, ::2] = -math.inf                         # every other token banned
    x[1] = -math.inf                              # nothing left
    x[2, :] = -math.inf
    x[2, vocab // 2] = 1.5                        # one token left
    x[3, 7] = math.nan
    x[4, vocab - 1] = math.inf
    x[5, 3:] = lowest                             # banned by the type's lowest value
    x[6] = lowest                                 # all of them: a uniform distribution
    x[7] = 2.0                                    # all equal
    x[8, 100:400] = 20.0                          # many equal at the top
    x[9] = 0.0
    x[9, 1::2] = -0.0                             # equal numbers
    x[10] *= 1e4                                  # far apart
    x[11, 5] = torch.finfo(dtype).max
    x[12, :] = -math.inf
    x[12, [3, 900]] = -1e30                       # two left, far below
    targets[12], targets[13], targets[2] = 900, -1, 0
    _check(x, targets, 12)
    targets[:] = vocab
    assert _ops().token_logprobs(x, targets).logprob.isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab, top", [(310, 35003, 5), (150, 50257, 3), (40, 100001, 5), (9, 70000, 0), (1, 151936, 20)])
def test_rows_of_many_turns(rows, vocab, top, dtype):
    """Rows that a block goes over in several turns, in clusters of several sizes, and more rows than the SMs hold two of."""
    x, targets = _rows(rows, vocab, dtype, seed=6)
    some = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:12].tolist()
    found = _ops().token_logprobs(x, targets, top=top)
    _check(x[some], targets[some], top, type(found)(*[None if f is None else f[some] for f in found]))


def test_many_rows_and_no_rows():
    x, targets = _rows(1500, 257, torch.float32, seed=4)
    whole = _ops().token_logprobs(x, targets, top=4)
    part = _ops().token_logprobs(x[700:703], targets[700:703].contiguous(), top=4)
    for a, b in zip(whole, part):
        assert torch.equal(a[700:703], b)
    none = _ops().token_logprobs(x[:0], targets[:0], top=4)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 4)


def test_on_another_stream():
    x, targets = _rows(8, 50000, torch.float32, seed=5)
    want = _ops().token_logprobs(x, targets, top=3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _ops().token_logprobs(x, targets, top=3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from rust_inference_b200.kernels.ops import KernelError
    ops = _ops()
    x, t = _rows(4, 100, torch.float32)
    for bad in [(x.half(), t, 1), (x.cpu(), t, 1), (x, t.long(), 1), (x, t[:3], 1), (x, t, 101), (x, t, -1), (x.t(), t, 1), (x[0], t, 1),
                (x[:, ::2], t, 1), (torch.zeros(4, 2000, device=DEV), t, 65)]:
        with pytest.raises(KernelError):
            ops.token_logprobs(bad[0], bad[1], top=bad[2])
