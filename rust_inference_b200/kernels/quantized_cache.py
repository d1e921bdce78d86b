"""A cache of keys and values in 8 bits: writing into it, reading it back.

A cache layer (`QuantizedPages`) holds int8 codes [pages, kv heads, 64, head size] and one float32 scale for every `BLOCK`
positions of a page and kv head, [pages, kv heads, 64 / BLOCK], keys and values apart; a code c stands for scale * c.
`write` says how rows become codes (csrc/quantized_cache.cu has the formulas).  Attention over such a layer is
`kernels.attention.attention`, which takes it in the place of a layer in the run dtype.

    layer = quantized_cache.empty_layer(pages, kv_heads, head_dim)
    quantized_cache.write(qkv, q, cos, sin, layer, page_table, seq_slot, seq_start, cu_seqlens, n_heads=..., ...)
    attention.attention(q, layer, out, ctx, n_heads=..., ...)
    quantized_cache.read(layer, k, v, page_table, seq_slot, seq_first, seq_len, max_len=..., cu_rows=...)
"""
from __future__ import annotations

import functools
from ctypes import c_int

import torch

from .build import load
from .ops import RI_BF16, RI_F32, KernelError, _call, _p, _stream, native

PAGE_SIZE, BLOCK = 64, 16


class QuantizedPages:
    """One layer: k, v int8 [pages, kv heads, 64, head size] (values may have a head size of their own), k_scale, v_scale
    float32 [pages, kv heads, 4], contiguous and on one device.  The tensors are looked at here, once, and stay the layer's."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "request", "sizes", "native", "aligned", "device")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, request=None):
        for t in (k, v, k_scale, v_scale):
            if not t.is_cuda or t.device != k.device:
                raise KernelError("a quantized layer's tensors lie on one CUDA device; this library has no CPU path")
        if not (k.dtype == torch.int8 and v.dtype == torch.int8 and k.is_contiguous() and v.is_contiguous() and k.dim() == 4
                and v.dim() == 4 and k.shape[2] == PAGE_SIZE and v.shape[:3] == k.shape[:3]):
            raise KernelError(f"a quantized layer's codes are contiguous int8 [pages, kv heads, {PAGE_SIZE}, head size]")
        scales = (k.shape[0], k.shape[1], PAGE_SIZE // BLOCK)
        for t in (k_scale, v_scale):
            if not (t.dtype == torch.float32 and t.is_contiguous() and tuple(t.shape) == scales):
                raise KernelError(f"a quantized layer's scales are contiguous float32 {list(scales)}")
        self.k, self.v, self.k_scale, self.v_scale, self.request = k, v, k_scale, v_scale, request
        self.sizes = (k.shape[1], k.shape[3], v.shape[3])           # kv heads, head size, value head size
        # as the native calls take it: addresses, then sizes
        self.native = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *self.sizes)
        self.aligned = k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0
        self.device = k.device


def empty_layer(n_pages: int, n_kv_heads: int, head_dim: int, v_head_dim: int | None = None, device="cuda") -> QuantizedPages:
    shape, scales = (n_pages, n_kv_heads, PAGE_SIZE), (n_pages, n_kv_heads, PAGE_SIZE // BLOCK)
    return QuantizedPages(torch.zeros(*shape, head_dim, dtype=torch.int8, device=device),
                          torch.zeros(*shape, head_dim if v_head_dim is None else v_head_dim, dtype=torch.int8, device=device),
                          torch.zeros(scales, dtype=torch.float32, device=device), torch.zeros(scales, dtype=torch.float32, device=device))


def is_quantized(layer) -> bool:
    return type(layer) is QuantizedPages


def _index(what: str, t: torch.Tensor, least: int) -> int:
    """The address of an index array of at least so many entries."""
    if not (t.dtype is torch.int32 and t.is_cuda and t.numel() >= least and t.is_contiguous()):
        raise KernelError(f"{what}: index arrays are contiguous int32 on the device, {least} entries or more here")
    return t.data_ptr()


def _need(good: bool, what: str, message: str) -> None:
    if not good:
        raise KernelError(f"{what}: {message}")


def write(src: torch.Tensor, q_out: torch.Tensor | None, cos, sin, layer: QuantizedPages, page_table: torch.Tensor, seq_slot, seq_start,
          cu_seqlens, *, n_heads: int, n_kv_heads: int, head_dim: int, max_new: int, v_head_dim: int | None = None, style: int = 0,
          rot_dims: int | None = None, bias: torch.Tensor | None = None, clear: bool = False) -> None:
    """A step's projection [T, q heads | k heads | v heads (or more columns)] to where it goes: queries, rotated, into q_out
    [T, n_heads * head_dim], keys, rotated, and values into the cache as codes.  Sequence b of slot seq_slot[b] holds seq_start[b]
    positions before the step and brings the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, at most max_new.  cos, sin: float32
    [positions, rot_dims / 2]; rot_dims 0: nothing is rotated; style 0: pairs (i, i + rot_dims / 2), 1: pairs (2i, 2i + 1).
    src may be float32 beside a bfloat16 q_out: the sums of a product that was cut over K, with `bias` (float32 [columns]) still to
    be added, and `clear` leaves them zeroed.  q_out None: the q columns are not looked at (`cos`, `sin` then turn keys only)."""
    native("write")(src, q_out, cos, sin, layer.native, page_table, seq_slot, seq_start, cu_seqlens, n_heads, n_kv_heads, head_dim,
                    head_dim if v_head_dim is None else v_head_dim, max_new, style, head_dim if rot_dims is None else rot_dims, bias, clear)


def read(layer: QuantizedPages, k_out: torch.Tensor, v_out: torch.Tensor, page_table: torch.Tensor, seq_slot, seq_first, seq_len, *,
         max_len: int, cu_rows: torch.Tensor | None = None, seen_span: int | None = None, out_pages: int = 0) -> tuple:
    """The values of the positions seq_first[b] .. seq_len[b] - 1 of every sequence b, in float32 or bfloat16.  With cu_rows, k_out
    and v_out are [rows, kv heads, head size] and sequence b's rows begin at cu_rows[b]; without, they have the cache's shape and
    the pages that hold these positions are filled (zeros elsewhere in them), the others left alone; with out_pages they are
    [sequences * out_pages, kv heads, 64, head size] instead, and a sequence's i-th page is the i-th of its own.  max_len: no
    sequence is longer.  seen_span: reading begins at the first key that a query at position seq_first[b] sees, of all keys (0), the last so many
    (> 0) or its own block of -span positions (< 0)."""
    native("read")(layer.native, k_out, v_out, page_table, seq_slot, seq_first, seq_len, max_len, cu_rows, layer.k.shape[0],
                   0 if seen_span is None else 1, seen_span or 0, out_pages)
    return k_out, v_out


def widen(layer: QuantizedPages, k_out: torch.Tensor, v_out: torch.Tensor, factors: torch.Tensor, page_table: torch.Tensor, seq_slot,
          seq_start, seq_len, *, max_len: int, span: int = 0, out_pages: int = 0) -> None:
    """The pages that a step's queries see as float16 numbers for `attention_tc.prefill_half`: k_out, v_out float16 of the cache's
    shape (or with out_pages for each sequence, as for `read`), and factors float32 [sequences, 2, kv heads] that keys and values are to be multiplied by; where scales
    lie too far apart for float16, the pages hold bfloat16 numbers instead and the keys' factor is -1.  What is outside a sequence's
    seen blocks is 0; a block that is no number is that in its keys."""
    what = "quantized_cache.widen"
    n_kv, hd, v_hd = layer.sizes
    n_seqs = seq_slot.numel()
    _need(layer.aligned and v_hd == hd and hd in (64, 128), what, "heads of 64 or 128 channels, keys and values alike")
    _need(k_out.is_cuda and v_out.is_cuda and k_out.dtype == v_out.dtype == torch.float16 and k_out.is_contiguous() and v_out.is_contiguous()
          and k_out.shape == v_out.shape == (n_seqs * out_pages if out_pages else layer.k.shape[0], *layer.k.shape[1:]), what,
          "outputs must be float16 of the cache's shape, or so many pages for each sequence")
    _need(factors.is_cuda and factors.dtype == torch.float32 and factors.is_contiguous() and factors.numel() >= 2 * n_seqs * n_kv, what,
          "factors must be float32 [sequences, 2, kv heads]")
    _need(page_table.dim() == 2, what, "the page table must be int32 [slots, pages]")
    for t, least in ((page_table, 1), (seq_slot, n_seqs), (seq_start, n_seqs), (seq_len, n_seqs)):
        _index(what, t, least)
    _call("quantized_cache", "ri_quantized_widen", _p(layer.k), _p(layer.v), _p(layer.k_scale), _p(layer.v_scale), _p(k_out), _p(v_out),
          _p(factors), _p(page_table), c_int(page_table.shape[1]), _p(seq_slot), _p(seq_start), _p(seq_len), c_int(n_seqs), c_int(max_len),
          c_int(n_kv), c_int(hd), c_int(span), c_int(out_pages), _stream())


@functools.lru_cache(maxsize=None)
def attention_workspace(n_heads: int, n_kv_heads: int, head_dim: int, max_new: int) -> tuple:
    """(float32 numbers of scratch, int32 counters) that `attend_step` wants; the counters are zero when it begins, and when it ends."""
    blocks = int(load("attention_quantized").ri_attention_quantized_blocks())
    return 2 * blocks * min(16, max_new * (n_heads // n_kv_heads)) * (head_dim + 4), 4 * 2 * blocks


def attention_counts(n_seqs: int, pages: int, max_new: int, n_heads: int, n_kv_heads: int) -> bool:
    """Whether `attend_step`'s units (pages of a kv head, for 8 rows) of a step over up to so many pages per sequence are counted in 31
    bits.  (An item counts as eight pages more.)"""
    return n_seqs * (pages + 8) * n_kv_heads * ((max_new * (n_heads // n_kv_heads) + 7) // 8) < 1 << 31


class _Step:
    """What the calls of a step have in common: its arrays' addresses and sizes, looked at once."""

    __slots__ = ("native", "kept", "max_new", "longest", "calls")

    def __init__(self, ctx, n_heads, n_kv_heads, head_dim):
        what = "quantized_cache.attend_step"
        table, n_seqs = ctx.page_table, ctx.seq_slot.numel()
        _need(n_kv_heads > 0 and n_heads > 0 and n_heads % n_kv_heads == 0 and head_dim in (64, 128) and table.dim() == 2, what,
              f"{n_heads} heads of {head_dim} over {n_kv_heads}, or a page table that is not [slots, pages]")
        self.max_new, self.longest = ctx.max_new, _longest(ctx)
        self.calls = set()                                      # (span, dtype) of the layers' calls
        floats, ints = attention_workspace(n_heads, n_kv_heads, head_dim, ctx.max_new)
        part = ctx.buffer("quantized_part", (floats,), torch.float32)
        arrived = ctx.zeroed_buffer("quantized_arrived", (ints,), torch.int32)
        self.native = (_index(what, table, 1), table.shape[1], _index(what, ctx.seq_slot, n_seqs), _index(what, ctx.seq_start, n_seqs),
                       _index(what, ctx.cu_seqlens, n_seqs + 1), n_seqs, ctx.max_new, n_heads, n_kv_heads, head_dim, part.data_ptr(), part.numel(),
                       _index(what, arrived, ints), self.longest)
        self.kept = (table, ctx.seq_slot, ctx.seq_start, ctx.cu_seqlens, ctx.workspace, part, arrived)     # whose addresses these are

    def stands(self, ctx) -> bool:
        """Whether the step still has the arrays, the scratch and the sizes that were looked at."""
        kept = self.kept
        return (kept[2] is ctx.seq_start and kept[3] is ctx.cu_seqlens and kept[1] is ctx.seq_slot and kept[0] is ctx.page_table
                and kept[4] is ctx.workspace and self.max_new == ctx.max_new and self.longest == _longest(ctx))


def _longest(ctx) -> int:
    """The keys of the step's longest sequence, as far as the host knows them (a captured step has a bound of its own)."""
    return ctx.extras.get("longest", ctx.max_len)


def step_of(ctx, n_heads: int, n_kv_heads: int, head_dim: int) -> _Step:
    """`attend_step`'s view of a step (`engine.context.StepContext`), made by the first layer that asks, and again if the step has
    been given other arrays, scratch or sizes since."""
    key = ("quantized", n_heads, n_kv_heads, head_dim)
    step = ctx.extras.get(key)
    if step is None or not step.stands(ctx):
        step = ctx.extras[key] = _Step(ctx, n_heads, n_kv_heads, head_dim)
    return step


def attend_step(q, layer: QuantizedPages, out, step: _Step, scale: float, span: int, out_scale: float) -> torch.Tensor:
    """Attention of every token of the step over its slot's cached keys, straight from the codes (csrc/attention_quantized.cu), for heads
    of 64 or 128.  q: float32 or bfloat16 rows whose leading columns are the queries, rotated; out: rows of q's dtype; span: > 0 the
    last so many keys, < 0 the keys of the query's own block of -span positions, 0 all."""
    step.calls.add((span, q.dtype))
    return native("attend")(q, layer.native, out, step.native, scale, span, out_scale)


def step_forms(ctx, longest: int) -> dict:
    """Which kernels the calls of a step so far would launch if its longest sequence had so many keys."""
    form = load("attention_quantized").ri_attention_quantized_form
    return {(key, call): form(*(c_int(v) for v in (RI_F32 if call[1] is torch.float32 else RI_BF16, step.kept[1].numel(), step.max_new, longest,
                                                   *key[1:], call[0])))
            for key, step in ctx.extras.items() if type(step) is _Step for call in step.calls}
