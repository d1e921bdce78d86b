"""What the cache in 8 bits and the scores decide on the host (no GPU)."""
import os
import re

import pytest
import torch

from rust_inference_b200.cache.sequence_cache import KVRequest, SequenceCache
from rust_inference_b200.cache.pager import CacheError
from rust_inference_b200.cli import CliError, parse_args
from rust_inference_b200.engine.engine import resolve_cache_dtype
from rust_inference_b200.kernels import build, ops
from rust_inference_b200.kernels.ops import KernelError


def _source(name):
    with open(os.path.join(build.CSRC, name)) as f:
        return f.read()


def test_the_entry_points_arguments_are_those_of_the_sources():
    """What the extension calls by address has the arguments, in kind and order, that the kernel libraries declare."""
    def kinds(args):
        return "".join("p" if "*" in a or "cudaStream_t" in a else "l" if "long long" in a else "f" if a.split()[0] == "float" else "i"
                       for a in args.split(","))

    for name, (_, module, fn) in ops._NATIVE.items():
        declared = re.search(r"RI_API int " + fn + r"\(([^)]*)\)", _source(build.MODULES[module])).group(1)
        called = re.search(r"typedef int " + name.capitalize() + r"Fn\(([^)]*)\)", _source("native_calls.cpp")).group(1)
        assert kinds(called) == kinds(declared), fn


def test_the_extension_refuses_what_it_cannot_take():
    """On the host: tensors that lie there, and arguments that are no tensors, are an error with a message, not a crash."""
    calls = build.load_extension("native_calls")
    for fn, count in (("write", 18), ("read", 12), ("attend", 7), ("logprobs", 4), ("bind", 4)):
        with pytest.raises((RuntimeError, TypeError)):
            getattr(calls, fn)(*[None] * count)
        with pytest.raises(RuntimeError):
            getattr(calls, fn)()
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the device"):
        calls.logprobs(x, t, 1, 64)
    with pytest.raises((RuntimeError, TypeError)):
        calls.logprobs(x, t, "one", 64)
    assert calls.launches() == 0


def test_cache_dtype_names():
    assert resolve_cache_dtype(None) is None and resolve_cache_dtype("same") is None
    assert resolve_cache_dtype("int8") is torch.int8 and resolve_cache_dtype(torch.int8) is torch.int8
    for bad in ("int4", "float8", torch.uint8, 8):
        with pytest.raises(ValueError):
            resolve_cache_dtype(bad)


def test_requests_that_are_not_kept_in_8_bits():
    with pytest.raises(CacheError, match="8 bits"):
        SequenceCache([KVRequest(2, 64)], max_tokens=64, max_seq_len=64, dtype=torch.float32, device="cpu", kv_dtype=torch.int8)
    with pytest.raises(CacheError, match="8 bits"):
        SequenceCache([(KVRequest(2, 64, quantizable=True), KVRequest(1, 40, None, 32, True))], max_tokens=64, max_seq_len=64,
                      dtype=torch.float32, device="cpu", kv_dtype=torch.int8)
    with pytest.raises(ValueError, match="int8"):
        SequenceCache([], max_tokens=64, max_seq_len=64, dtype=torch.float32, device="cpu", kv_dtype=torch.float16)
    with pytest.raises(KernelError, match="CUDA"):              # there is no path on the host
        SequenceCache([KVRequest(2, 64, quantizable=True)], max_tokens=64, max_seq_len=64, dtype=torch.float32, device="cpu", kv_dtype=torch.int8)
    # whether a request may be kept so is no part of what tells requests apart
    assert KVRequest(2, 64, quantizable=True) == KVRequest(2, 64) and hash(KVRequest(2, 64, quantizable=True)) == hash(KVRequest(2, 64))


def test_flags(tmp_path):
    base = ["--model", str(tmp_path), "--prompt", "1,2"]
    assert parse_args(base)["cache_dtype"] is None and parse_args(base)["score"] is None
    a = parse_args(base + ["--cache-dtype", "int8", "--score", "5"])
    assert a["cache_dtype"] == "int8" and a["score"] == 5
    for bad in (["--cache-dtype", "fp8"], ["--score", "-1"], ["--score", "65"], ["--score", "x"]):
        with pytest.raises(CliError):
            parse_args(base + bad)


def test_which_steps_read_the_codes():
    from types import SimpleNamespace
    from rust_inference_b200.kernels import attention

    def reads(n_seqs, max_new, f32=False, heads=32, kv=8, pages=64):
        return attention.reads_codes(SimpleNamespace(n_seqs=n_seqs, max_new=max_new, page_table=torch.zeros(n_seqs, pages), extras={}), f32, heads, kv)

    assert reads(1, 1) and reads(64, 1) and reads(64, 16) and reads(1, 64) and reads(1, 512, heads=4, kv=4)
    assert not reads(64, 17) and not reads(1, 65) and not reads(8, 2048)
    assert reads(8, 2048, f32=True) and reads(64, 2048, f32=True, pages=512)
    assert not reads(64, 4096, f32=True, pages=2048)            # more units than 31 bits count: read back
