"""How steps over a cache in 8 bits go in which sequences bring different numbers of tokens (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

from rust_inference_b200.kernels import attention


def _reads(runs, heads=32, kv=8, hd=128, span=0, known=True):
    ctx = SimpleNamespace(n_seqs=len(runs), max_new=max(n for _, n in runs), page_table=torch.zeros(len(runs), 1024), extras={})
    if known:
        ctx.host_starts, ctx.host_counts = [s for s, _ in runs], [n for _, n in runs]
    return attention.reads_codes(ctx, False, heads, kv, hd, span)


@pytest.mark.parametrize("heads, kv, hd", [(32, 8, 128), (28, 4, 128), (14, 2, 64)])
def test_many_single_tokens_beside_a_short_prompt(heads, kv, hd):
    """All of the many long sequences would be copied for the sake of one with a few tokens more."""
    for runs in ([(2000, 1)] * 63 + [(0, 17)], [(2000, 1)] * 63 + [(0, 500)], [(2000, 1)] * 8 + [(0, 40)] * 8, [(2000, 1)] * 63 + [(4000, 100)]):
        assert _reads(runs, heads, kv, hd)


@pytest.mark.parametrize("heads, kv, hd", [(32, 8, 128), (28, 4, 128), (14, 2, 64)])
def test_prompts(heads, kv, hd):
    for runs in ([(0, 2048)], [(0, 300)] * 7, [(2000, 1)] * 63 + [(29000, 1000)], [(2000, 1)] * 63 + [(0, 4000)], [(100, 1)] * 7 + [(0, 1000)]):
        assert not _reads(runs, heads, kv, hd)


def test_windows_shorten_what_is_copied():
    runs = [(30000, 1)] * 20 + [(0, 1200)]
    assert _reads(runs) and not _reads(runs, span=100) and not _reads(runs, span=-128)


def test_without_the_hosts_numbers():
    assert not _reads([(2000, 1)] * 63 + [(0, 17)], known=False) and _reads([(0, 64)], known=False) and not _reads([(0, 65)], known=False)


def test_other_numbers_in_the_place_of_those_that_were_judged():
    ctx = SimpleNamespace(n_seqs=2, max_new=900, page_table=torch.zeros(2, 1024), extras={}, host_starts=[0, 0], host_counts=[900, 900])
    assert not attention.reads_codes(ctx, False, 32, 8)
    ctx.host_starts, ctx.host_counts, ctx.max_new = [60000, 60000], [20, 20], 20
    assert attention.reads_codes(ctx, False, 32, 8)
