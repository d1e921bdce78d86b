"""Numbers of heads that are none, over a cache in 8 bits: refused, where they would lead before the arrays."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from rust_inference_b200.kernels import build, quantized_cache as qc
from rust_inference_b200.kernels.ops import KernelError


def test_writing():
    calls = build.load_extension("native_calls")
    x, t = torch.zeros(1, 512), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="negative number of heads"):
        calls.write(x, None, None, None, (0, 0, 0, 0, 2, 64, 64), t[None], t, t, t, -1, 2, 64, 64, 1, 0, 0, None, False)


def test_a_step():
    step = SimpleNamespace(page_table=torch.zeros(1, 1, dtype=torch.int32), seq_slot=torch.zeros(1, dtype=torch.int32), max_new=1, extras={}, max_len=1)
    for heads, kv in ((-4, 2), (0, 2), (4, -2), (4, 0), (5, 2)):
        with pytest.raises(KernelError, match="heads"):
            qc.step_of(step, heads, kv, 64)


def test_the_libraries():
    """The entry points themselves: nothing is looked at before the numbers are (no array is given)."""
    lib, null = build.load("attention_quantized"), ctypes.c_void_p(None)
    i = ctypes.c_int
    for heads, kv in ((-4, 2), (0, 2), (4, -2), (4, 0)):
        args = [null, i(1), i(256), null, null, null, null, null, i(1), null, null, null, null, i(256), i(1), i(1), i(1), i(heads), i(kv), i(64),
                ctypes.c_float(1.0), i(0), ctypes.c_float(1.0), null, ctypes.c_longlong(0), null, null]
        assert lib.ri_attention_quantized(*args) != 0 and lib.ri_attention_quantized_form(1, 1, 1, 1, heads, kv, 64, 0) == -1
    lib = build.load("quantized_cache")
    for heads, kv in ((-4, 2), (4, -2), (4, 0), (-1, 65536)):
        args = [null, i(1), i(512), null, i(0), null, i(1), null, null, null, i(1), null, null, null, null, null, null, null, i(1), i(1), i(1),
                i(heads), i(kv), i(64), i(64), i(0), i(0), null]
        assert lib.ri_quantized_write(*args) != 0
