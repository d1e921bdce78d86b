"""Weights in microscaled 4-bit floating point, and the 8-bit rows that they are multiplied with.

32 consecutive numbers of a row share a power of two, the smallest for which none of them exceeds the type's largest number times it, and
each is kept as the nearest number of the type times that power, ties to the even one: in a matrix (`Matrix`) 4 bits, +-{0, 0.5, 1, 1.5, 2, 3,
4, 6}, in rows of activations (`Rows`) 8, with four bits of exponent and three of mantissa, up to 448.  csrc/microscaled.cuh has the layout.
A block that holds an infinity or a NaN stands for 32 NaNs.

    w = microscaled.Matrix.of(t)                                  # [n, k] float32 or bfloat16, once, when a model is loaded
    w = microscaled.Matrix.of_codes(codes, exponents, k)          # from a file that holds such numbers already
    microscaled.rmsnorm(stream, weight, eps, rows, branch=b, total=stream)
    linear.project(rows, w, out, ctx)                             # and the others of `kernels.linear`: rows in 8 bits, or plain
    linear.gated(rows, w_gate, w_up, more_rows, ctx)              # ones, which are brought to 8 bits first
    microscaled.values(w, torch.bfloat16)                         # what is held, as plain numbers
"""
from __future__ import annotations

from ctypes import c_double, c_int, c_longlong, c_void_p

import torch

from . import ops
from .build import load
from .ops import KernelError, _call, _need, _p, _stream, dtype_code

_current_device = getattr(ops, "_current_device", torch.cuda.current_device)

BLOCK, SPAN, PIECE = 32, 128, 512
OUT_BF16, OUT_F32, OUT_ROWS, OUT_ADD = 0, 1, 2, 3
_KIND = {torch.bfloat16: OUT_BF16, torch.float32: OUT_F32}


def _spans(k: int) -> int:
    return -(-k // SPAN)


def _here(what: str, *tensors) -> None:
    """The tensors lie on the current device, whose stream the kernels go to."""
    for t in tensors:
        if t is not None and not (t.is_cuda and t.device.index == _current_device()):
            raise KernelError(f"{what}: a tensor that is not on the current CUDA device; this library has no CPU path")


def _encode(codes: torch.Tensor, exponents: torch.Tensor, rows: int, spans: int, bits: int, box: int) -> torch.Tensor:
    m = torch.empty(256, dtype=torch.uint8)           # CPU allocations are 64-byte aligned
    _call("gemm_microscaled", "ri_mx_encode", c_void_p(m.data_ptr()), _p(codes), _p(exponents), c_longlong(rows), c_int(spans), c_int(bits), c_int(box))
    ops._launches -= 1                                # encoding a map launches nothing
    return m


class Matrix:
    """A weight matrix [n, k] in 4 bits, for the products of `kernels.linear`."""

    __slots__ = ("n", "k", "spans", "codes", "exponents", "device", "_map")

    def __init__(self, n: int, k: int, codes: torch.Tensor, exponents: torch.Tensor):
        self.n, self.k, self.spans = n, k, _spans(k)
        self.codes, self.exponents, self.device, self._map = codes, exponents, codes.device, None

    @classmethod
    def of(cls, t: torch.Tensor) -> "Matrix":
        """The matrix nearest to t [n, k], float32 or bfloat16, whose rows may lie apart."""
        _need(t.dim() == 2 and t.shape[0] > 0 and t.shape[1] > 0, "microscaled.Matrix: a matrix [n, k] of at least one number is wanted")
        _here("microscaled.Matrix", t)
        if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1]:
            t = t.contiguous()
        n, k = t.shape
        m = cls._empty(n, k, t.device)
        _call("microscaled", "ri_mx_hold", _p(t), c_int(dtype_code(t.dtype)), c_int(4), c_longlong(n), c_longlong(k), c_longlong(t.stride(0)), _p(m.codes),
              _p(m.exponents), _stream())
        return m

    @classmethod
    def _empty(cls, n, k, device) -> "Matrix":
        spans = _spans(k)
        # exponents of rows behind the last one, in its piece of 128, are read beside it and have no effect: zeros, so that they are numbers
        return cls(n, k, torch.empty(n, spans * SPAN // 2, dtype=torch.uint8, device=device),
                   torch.zeros(-(-n // 128), spans, PIECE, dtype=torch.uint8, device=device))

    @classmethod
    def of_codes(cls, codes: torch.Tensor, exponents: torch.Tensor, k: int) -> "Matrix":
        """From codes uint8 [n, ceil(k / 2)], number 2i in the low half of byte i (the sign, then the place among 0, 0.5, 1, 1.5, 2, 3, 4, 6),
        and exponents plus 127, uint8 [n, ceil(k / 32)] (255: NaN)."""
        n = codes.shape[0]
        _need(codes.dtype == torch.uint8 and exponents.dtype == torch.uint8 and n > 0 and k > 0 and tuple(codes.shape) == (n, -(-k // 2))
              and tuple(exponents.shape) == (n, -(-k // BLOCK)), "microscaled.Matrix: codes uint8 [n, ceil(k / 2)] and exponents uint8 [n, ceil(k / 32)] are wanted")
        _here("microscaled.Matrix", codes, exponents)
        m = cls._empty(n, k, codes.device)
        m.codes.zero_()
        m.codes[:, :codes.shape[1]] = codes
        if k % 2:
            m.codes[:, k // 2] &= 15
        spans = m.spans
        wide = torch.zeros(m.exponents.shape[0] * 128, spans * 4, dtype=torch.uint8, device=codes.device)
        wide[:n, :exponents.shape[1]] = exponents
        m.exponents.copy_(wide.view(-1, 4, 32, spans, 4).permute(0, 3, 2, 1, 4).reshape(-1, spans, PIECE))
        return m

    @property
    def shape(self):
        return self.n, self.k

    def bytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def map(self) -> torch.Tensor:
        if self._map is None:
            self._map = _encode(self.codes, self.exponents, self.n, self.spans, 4, 128)
        return self._map


class Rows:
    """Room for rows [n, k] in 8 bits, which a norm, a product or `quantize` fills and products read.  `codes` and `exponents`: buffers of
    the caller's own, uint8 and of `Rows.sizes(n, k)` bytes at least."""

    __slots__ = ("n", "k", "spans", "codes", "exponents", "device", "_maps")

    def __init__(self, n: int, k: int, device="cuda", codes: torch.Tensor | None = None, exponents: torch.Tensor | None = None):
        _need(n > 0 and k > 0, "microscaled.Rows: at least one row of at least one number")
        a, b = self.sizes(n, k)
        codes = torch.empty(a, dtype=torch.uint8, device=device) if codes is None else codes
        exponents = torch.empty(b, dtype=torch.uint8, device=device) if exponents is None else exponents
        for t, least in ((codes, a), (exponents, b)):
            _need(t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous() and t.numel() >= least and t.device == codes.device and t.data_ptr() % 32 == 0,
                  "microscaled.Rows: buffers are contiguous uint8 on one CUDA device, on a 32-byte boundary and of Rows.sizes(n, k) bytes")
        self.n, self.k, self.spans = n, k, _spans(k)
        self.codes, self.exponents, self.device, self._maps = codes, exponents, codes.device, {}

    @staticmethod
    def sizes(n: int, k: int) -> tuple:
        """Bytes of the codes and of the exponents."""
        return n * _spans(k) * SPAN, -(-n // 128) * _spans(k) * PIECE

    @property
    def shape(self):
        return self.n, self.k

    def map(self, box: int) -> torch.Tensor:
        m = self._maps.get(box)
        if m is None:
            m = self._maps[box] = _encode(self.codes, self.exponents, self.n, self.spans, 8, box)
        return m


def quantize(x: torch.Tensor, out: Rows | None = None) -> Rows:
    """x [n, k], float32 or bfloat16, rows apart or not, in 8 bits."""
    _need(x.dim() == 2 and (x.stride(1) == 1 or x.shape[1] == 1) and (x.stride(0) >= x.shape[1] or x.shape[0] == 1),
          "microscaled.quantize: rows [n, k] whose numbers lie side by side are wanted")
    n, k = x.shape
    if out is None:
        out = Rows(n, k, x.device)
    _need((out.n, out.k) == (n, k), "microscaled.quantize: out holds other rows")
    _here("microscaled.quantize", x, out.codes)
    _call("microscaled", "ri_mx_hold", _p(x), c_int(dtype_code(x.dtype)), c_int(8), c_longlong(n), c_longlong(k), c_longlong(max(x.stride(0), k)), _p(out.codes),
          _p(out.exponents), _stream())
    return out


def values(held, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The numbers [n, k] that a `Matrix` or `Rows` stands for, in float32 or bfloat16 (which hold them exactly, but for results that
    the type has no room for)."""
    if out is None:
        out = torch.empty(held.n, held.k, dtype=dtype, device=held.device)
    _need(tuple(out.shape) == (held.n, held.k) and out.is_contiguous() and out.dtype == dtype, "microscaled.values: out is contiguous [n, k] of the dtype asked for")
    _here("microscaled.values", out, held.codes)
    _call("microscaled", "ri_mx_values", _p(held.codes), _p(held.exponents), c_int(dtype_code(dtype)), c_int(4 if type(held) is Matrix else 8),
          c_longlong(held.n), c_longlong(held.k), _p(out), _stream())
    return out


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: Rows, *, branch: torch.Tensor | None = None,
            total: torch.Tensor | None = None) -> Rows:
    """total = x + branch (x alone without a branch), and out = total / sqrt(mean(total^2) + eps) * weight in 8 bits.  x and weight
    float32, x [n, k]; branch float32 or bfloat16; total float32, x itself or another array, or None where it is not wanted."""
    n, k = out.n, out.k
    _need(x.dtype == torch.float32 and tuple(x.shape) == (n, k) and x.is_contiguous() and weight.dtype == torch.float32 and weight.numel() == k
          and weight.is_contiguous(), "microscaled.rmsnorm: x must be float32 [n, k] as out, weight float32 [k]")
    _need(branch is None or (tuple(branch.shape) == (n, k) and branch.is_contiguous()), "microscaled.rmsnorm: a branch [n, k] is wanted")
    _need(total is None or (total.dtype == torch.float32 and tuple(total.shape) == (n, k) and total.is_contiguous()), "microscaled.rmsnorm: total must be float32 [n, k]")
    _here("microscaled.rmsnorm", x, weight, branch, total, out.codes)
    _call("microscaled", "ri_mx_rmsnorm", _p(x), _p(branch), c_int(dtype_code(branch.dtype if branch is not None else torch.float32)), _p(weight), _p(total),
          c_longlong(n), c_longlong(k), c_double(eps), _p(out.codes), _p(out.exponents), _stream())
    return out


def rows_of(x, ctx, k: int) -> Rows:
    """x as rows in 8 bits: itself, or plain rows brought to them in the step's scratch."""
    if type(x) is Rows:
        return x
    return quantize(x, ctx.workspace.rows("mx_rows", x.shape[0], k))


def product(x, w: Matrix, out, ctx, *, w2: Matrix | None = None, bias=None, form=None, act=None, add: bool = False):
    """out = x W^T + bias; with `act` an activation of it (`ops.whole_act_form`); with w2 the gated form of x W^T and x W2^T (`form`:
    `ops.gate_form`, None: silu); with `add` out<float32> += x W^T.  x: `Rows`, or plain rows; out: plain rows, or (not with `add`) `Rows`."""
    what = "microscaled.product"
    n_tok = x.shape[0]
    _need(type(w) is Matrix and x.shape[1] == w.k, "microscaled.product: rows and matrix have another number of columns")
    _need(w2 is None or (type(w2) is Matrix and w2.shape == w.shape), "microscaled.product: the second matrix must be as the first")
    _need((bias is not None) + (act is not None) + (w2 is not None) + add <= 1 and (form is None or w2 is not None),
          "microscaled.product: a bias, an activation, a gate and an addition are not combined")
    _need(tuple(out.shape) == (n_tok, w.n), "microscaled.product: out must be [tokens, features]")
    if n_tok == 0:
        return out
    constants = bias
    if bias is not None:
        _need(bias.dtype == torch.float32 and bias.numel() == w.n and bias.is_contiguous(), "microscaled.product: bias must be float32 [features]")
    if form is not None:
        constants = ops.whole_gate_form(form)
        _need(constants.dtype == torch.float32 and constants.numel() == 5, "microscaled.product: a gate form is five float32 constants")
    if act is not None:
        constants = ops.whole_act_form(act)
        _need(constants.dtype == torch.float32 and constants.numel() == 4, "microscaled.product: an activation's form is four float32 constants")
    if type(out) is Rows:
        _need(not add, "microscaled.product: nothing is added to rows in 8 bits")
        kind, to, to_exp, to_spans = OUT_ROWS, out.codes, out.exponents, out.spans
    else:
        _need(out.is_contiguous() and out.dtype in _KIND and (not add or out.dtype == torch.float32), "microscaled.product: out must be contiguous float32 or bfloat16 (float32 where sums are added)")
        kind, to, to_exp, to_spans = OUT_ADD if add else _KIND[out.dtype], out, None, 0
    rows = rows_of(x, ctx, w.k)
    _need(to is not rows.codes, "microscaled.product: rows cannot be their own product")
    _here(what, rows.codes, w.codes, w2.codes if w2 is not None else None, to, constants)
    from .tcgen05 import status_word
    box = load("gemm_microscaled").ri_mx_box(c_int(n_tok), c_int(w.n), c_int(w.spans), c_int(1 if w2 is not None else 0))
    _call("gemm_microscaled", "ri_mx_gemm", c_void_p(w.map().data_ptr()), c_void_p(w2.map().data_ptr() if w2 is not None else 0),
          c_void_p(rows.map(box).data_ptr()), _p(w.exponents), _p(w2.exponents if w2 is not None else None), _p(rows.exponents), _p(constants),
          c_int(1 if w2 is not None else 0), c_int(1 if act is not None else 0), c_int(kind), _p(to), _p(to_exp), c_int(to_spans), c_int(n_tok), c_int(w.n),
          c_int(w.spans), c_void_p(status_word().data_ptr()), _stream())
    return out
