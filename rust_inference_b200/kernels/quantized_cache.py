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
from ctypes import c_float, c_int
from dataclasses import dataclass

import torch

from .build import load
from .ops import _call, _need, _need_cuda, _p, _stream, dtype_code

PAGE_SIZE, BLOCK = 64, 16


@dataclass
class QuantizedPages:
    """One layer: k, v int8 [pages, kv heads, 64, head size] (values may have a head size of their own), k_scale, v_scale
    float32 [pages, kv heads, 4]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    request: object = None


def empty_layer(n_pages: int, n_kv_heads: int, head_dim: int, v_head_dim: int | None = None, device="cuda") -> QuantizedPages:
    shape, scales = (n_pages, n_kv_heads, PAGE_SIZE), (n_pages, n_kv_heads, PAGE_SIZE // BLOCK)
    return QuantizedPages(torch.zeros(*shape, head_dim, dtype=torch.int8, device=device),
                          torch.zeros(*shape, head_dim if v_head_dim is None else v_head_dim, dtype=torch.int8, device=device),
                          torch.zeros(scales, dtype=torch.float32, device=device), torch.zeros(scales, dtype=torch.float32, device=device))


def is_quantized(layer) -> bool:
    return isinstance(layer, QuantizedPages)


def _need_layer(layer: QuantizedPages, n_kv_heads: int, head_dim: int, v_head_dim: int, what: str) -> None:
    k, v = layer.k, layer.v
    _need_cuda(k, v, layer.k_scale, layer.v_scale)
    _need(k.dtype == torch.int8 and v.dtype == torch.int8 and k.is_contiguous() and v.is_contiguous() and k.dim() == 4 and v.dim() == 4
          and k.shape[1:] == (n_kv_heads, PAGE_SIZE, head_dim) and v.shape[1:] == (n_kv_heads, PAGE_SIZE, v_head_dim)
          and k.shape[0] == v.shape[0], f"{what}: codes must be contiguous int8 [pages, {n_kv_heads}, {PAGE_SIZE}, head size]")
    scales = (k.shape[0], n_kv_heads, PAGE_SIZE // BLOCK)
    for t in (layer.k_scale, layer.v_scale):
        _need(t.dtype == torch.float32 and t.is_contiguous() and tuple(t.shape) == scales, f"{what}: scales must be float32 {list(scales)}")


def _need_int32(what: str, *tensors) -> None:
    for t in tensors:
        _need(t is None or (t.dtype == torch.int32 and t.is_contiguous()), f"{what}: index arrays must be contiguous int32")


def write(src: torch.Tensor, q_out: torch.Tensor | None, cos, sin, layer: QuantizedPages, page_table: torch.Tensor, seq_slot, seq_start,
          cu_seqlens, *, n_heads: int, n_kv_heads: int, head_dim: int, max_new: int, v_head_dim: int | None = None, style: int = 0,
          rot_dims: int | None = None, bias: torch.Tensor | None = None, clear: bool = False) -> None:
    """A step's projection [T, q heads | k heads | v heads (or more columns)] to where it goes: queries, rotated, into q_out
    [T, n_heads * head_dim], keys, rotated, and values into the cache as codes.  Sequence b of slot seq_slot[b] holds seq_start[b]
    positions before the step and brings the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, at most max_new.  cos, sin: float32
    [positions, rot_dims / 2]; rot_dims 0: nothing is rotated; style 0: pairs (i, i + rot_dims / 2), 1: pairs (2i, 2i + 1).
    src may be float32 beside a bfloat16 q_out: the sums of a product that was cut over K, with `bias` (float32 [columns]) still to
    be added, and `clear` leaves them zeroed.  q_out None: the q columns are not looked at (`cos`, `sin` then turn keys only)."""
    what = "quantized_cache.write"
    v_hd = head_dim if v_head_dim is None else int(v_head_dim)
    rot = head_dim if rot_dims is None else int(rot_dims)
    _need_cuda(src, q_out, cos, sin, page_table, seq_slot, seq_start, cu_seqlens, bias)
    _need_layer(layer, n_kv_heads, head_dim, v_hd, what)
    _need_int32(what, page_table, seq_slot, seq_start, cu_seqlens)
    n_seqs = seq_slot.numel()
    cols = (n_heads + n_kv_heads) * head_dim + n_kv_heads * v_hd
    _need(src.dim() == 2 and src.is_contiguous() and src.shape[1] >= cols, f"{what}: a contiguous [tokens, {cols} or more] is wanted")
    _need(seq_start.numel() >= n_seqs and cu_seqlens.numel() > n_seqs, f"{what}: one start per sequence and one offset more")
    _need(q_out is None or (q_out.is_contiguous() and q_out.shape == (src.shape[0], n_heads * head_dim)
                            and (q_out.dtype == src.dtype or src.dtype == torch.float32)), f"{what}: q_out must be [tokens, heads * head size]")
    _need(rot == 0 or (cos.dtype == sin.dtype == torch.float32 and cos.shape[1] == rot // 2 and sin.shape == cos.shape
                       and cos.is_contiguous() and sin.is_contiguous()), f"{what}: tables must be float32 [positions, rotated channels / 2]")
    _need(bias is None or (bias.dtype == torch.float32 and bias.is_contiguous() and bias.numel() >= cols), f"{what}: bias must be float32 [columns]")
    _call("quantized_cache", "ri_quantized_write", _p(src), c_int(dtype_code(src.dtype)), c_int(src.shape[1]), _p(bias),
          c_int(1 if clear else 0), _p(q_out), c_int(dtype_code(src.dtype if q_out is None else q_out.dtype)), _p(cos), _p(sin),
          _p(page_table), c_int(page_table.shape[1]), _p(seq_slot), _p(seq_start), _p(cu_seqlens), _p(layer.k), _p(layer.v),
          _p(layer.k_scale), _p(layer.v_scale), c_int(n_seqs), c_int(max_new), c_int(n_heads), c_int(n_kv_heads), c_int(head_dim),
          c_int(v_hd), c_int(rot), c_int(style), _stream())


def read(layer: QuantizedPages, k_out: torch.Tensor, v_out: torch.Tensor, page_table: torch.Tensor, seq_slot, seq_first, seq_len, *,
         max_len: int, cu_rows: torch.Tensor | None = None, seen_span: int | None = None) -> tuple:
    """The values of the positions seq_first[b] .. seq_len[b] - 1 of every sequence b, in float32 or bfloat16.  With cu_rows, k_out
    and v_out are [rows, kv heads, head size] and sequence b's rows begin at cu_rows[b]; without, they have the cache's shape and
    the pages that hold these positions are filled (zeros elsewhere in them), the others left alone.  max_len: no sequence is
    longer.  seen_span: reading begins at the first key that a query at position seq_first[b] sees, of all keys (0), the last so many
    (> 0) or its own block of -span positions (< 0)."""
    what = "quantized_cache.read"
    n_kv, hd, v_hd = layer.k.shape[1], layer.k.shape[3], layer.v.shape[3]
    _need_cuda(k_out, v_out, page_table, seq_slot, seq_first, seq_len, cu_rows)
    _need_layer(layer, n_kv, hd, v_hd, what)
    _need_int32(what, page_table, seq_slot, seq_first, seq_len, cu_rows)
    n_seqs = seq_slot.numel()
    _need(seq_first.numel() >= n_seqs and seq_len.numel() >= n_seqs and (cu_rows is None or cu_rows.numel() >= n_seqs),
          f"{what}: one entry per sequence")
    _need(k_out.dtype == v_out.dtype and k_out.is_contiguous() and v_out.is_contiguous(), f"{what}: outputs of one dtype, contiguous")
    if cu_rows is None:
        _need(k_out.shape == layer.k.shape and v_out.shape == layer.v.shape, f"{what}: without cu_rows the outputs have the cache's shape")
    else:
        _need(k_out.dim() == 3 and k_out.shape[1:] == (n_kv, hd) and v_out.shape == (k_out.shape[0], n_kv, v_hd),
              f"{what}: with cu_rows the outputs are [rows, kv heads, head size]")
    _call("quantized_cache", "ri_quantized_read", _p(layer.k), _p(layer.v), _p(layer.k_scale), _p(layer.v_scale), _p(k_out), _p(v_out),
          c_int(dtype_code(k_out.dtype)), _p(page_table), c_int(page_table.shape[1]), _p(seq_slot), _p(seq_first), _p(seq_len),
          _p(cu_rows), c_int(n_seqs), c_int(max_len), c_int(n_kv), c_int(hd), c_int(v_hd),
          c_int(0 if seen_span is None else 1), c_int(seen_span or 0), _stream())
    return k_out, v_out


@functools.lru_cache(maxsize=None)
def _attention_blocks(device: int) -> int:
    return int(load("attention_quantized").ri_attention_quantized_blocks())


def attention_workspace(n_tokens: int, n_heads: int, n_kv_heads: int, head_dim: int, max_new: int) -> tuple:
    """(float32 numbers of scratch, int32 counters) that `attention` wants for a step of n_tokens; the counters are zero when it
    begins, and when it ends."""
    cap = min(16, max_new * (n_heads // n_kv_heads))
    return 2 * _attention_blocks(torch.cuda.current_device()) * cap * (head_dim + 4), n_tokens * n_heads


def attention_supports(dtype: torch.dtype, head_dim: int, v_head_dim: int | None) -> bool:
    """The sizes that `attention` takes."""
    return dtype in (torch.float32, torch.bfloat16) and head_dim in (64, 128) and v_head_dim in (None, head_dim)


def attention(q: torch.Tensor, layer: QuantizedPages, out: torch.Tensor, page_table: torch.Tensor, seq_slot, seq_start, cu_seqlens, *,
              n_heads: int, n_kv_heads: int, head_dim: int, max_new: int, scale: float, part: torch.Tensor, arrived: torch.Tensor,
              span: int = 0, out_scale: float = 1.0) -> torch.Tensor:
    """Attention of every token of the step over its slot's cached keys, straight from the codes (csrc/attention_quantized.cu): for
    steps of few tokens per sequence, and for float32.  q: rows whose leading n_heads * head_dim columns are the queries, rotated;
    span: > 0 the last so many keys, < 0 the keys of the query's own block of -span positions; part, arrived: `attention_workspace`."""
    what = "quantized_cache.attention"
    _need_cuda(q, out, page_table, seq_slot, seq_start, cu_seqlens, part, arrived)
    _need_layer(layer, n_kv_heads, head_dim, head_dim, what)
    _need_int32(what, page_table, seq_slot, seq_start, cu_seqlens, arrived)
    n_seqs = seq_slot.numel()
    _need(q.dtype == out.dtype and attention_supports(q.dtype, head_dim, None) and q.dim() == 2 and out.dim() == 2 and q.stride(1) == 1
          and out.stride(1) == 1 and q.shape[0] == out.shape[0] and min(q.shape[1], out.shape[1]) >= n_heads * head_dim,
          f"{what}: queries and result must be float32 or bfloat16 [tokens, heads * 64 or 128]")
    _need(n_heads % n_kv_heads == 0 and seq_start.numel() >= n_seqs and cu_seqlens.numel() > n_seqs, f"{what}: heads, or entries per sequence")
    floats, ints = attention_workspace(q.shape[0], n_heads, n_kv_heads, head_dim, max_new)
    _need(part.dtype == torch.float32 and part.is_contiguous() and part.numel() >= floats and arrived.numel() >= ints, f"{what}: scratch too small")
    _call("attention_quantized", "ri_attention_quantized", _p(q), c_int(dtype_code(q.dtype)), c_int(q.stride(0)), _p(layer.k), _p(layer.v),
          _p(layer.k_scale), _p(layer.v_scale), _p(page_table), c_int(page_table.shape[1]), _p(seq_slot), _p(seq_start), _p(cu_seqlens),
          _p(out), c_int(out.stride(0)), c_int(n_seqs), c_int(max_new), c_int(n_heads), c_int(n_kv_heads), c_int(head_dim), c_float(scale),
          c_int(span), c_float(out_scale), _p(part), _p(arrived), c_int(_attention_blocks(torch.cuda.current_device())), _stream())
    return out
