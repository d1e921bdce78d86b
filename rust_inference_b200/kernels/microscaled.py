"""Weights in microscaled 4-bit floating point, and the 8-bit rows that they are multiplied with.

32 consecutive numbers of a row share a power of two, the smallest for which none of them exceeds the type's largest number times it, and
each is kept as the nearest number of the type times that power, ties to the even one: in a matrix (`Matrix`) 4 bits, +-{0, 0.5, 1, 1.5, 2, 3,
4, 6}, in rows of activations (`Rows`) 8, with four bits of exponent and three of mantissa, up to 448.  csrc/microscaled.cuh has the layout.
A block that holds an infinity or a NaN stands for 32 NaNs.  Whatever a product with a `Matrix` reads is in 8 bits then, in a float32 run too.

    w = microscaled.Matrix.of(t)                                  # [n, k] float32 or bfloat16, once, when a model is loaded
    w = microscaled.Matrix.of_codes(codes, exponents, k)          # from a file that holds such numbers already
    microscaled.rmsnorm(stream, weight, eps, rows, branch=b, total=stream)
    linear.project(rows, w, out, ctx)                             # and the others of `kernels.linear`: rows in 8 bits, or plain
    linear.gated(rows, w_gate, w_up, more_rows, ctx)              # ones, which are brought to 8 bits first
    microscaled.values(w, torch.bfloat16)                         # what is held, as plain numbers
"""
from __future__ import annotations

import functools
from ctypes import c_int, c_longlong, c_void_p, cast

import torch

from . import ops
from .build import load
from .ops import KernelError, _call, _need, _p, _stream, native

BLOCK, SPAN, PIECE = 32, 128, 512


def _spans(k: int) -> int:
    return -(-k // SPAN)


@functools.lru_cache(maxsize=None)
def _held_bytes() -> int:
    fn = load("microscaled").ri_mx_held_bytes
    fn.restype = c_longlong
    return fn()


def _describe(codes: torch.Tensor, exponents: torch.Tensor, n: int, k: int, bits: int) -> torch.Tensor:
    """What the entry points are given of something held, in host memory."""
    at = torch.empty(_held_bytes(), dtype=torch.uint8)           # CPU allocations are 64-byte aligned
    _call("microscaled", "ri_mx_make", c_void_p(at.data_ptr()), _p(codes), _p(exponents), c_longlong(n), c_longlong(k), c_int(bits), c_int(codes.device.index))
    ops._launches -= 1                                           # (launches nothing)
    return at


@functools.lru_cache(maxsize=None)
def _maker():
    native("mx_hold")                                            # names the entry points that it takes
    from .build import load_extension
    fn, make, size = load_extension("native_calls").mx_matrix, cast(load("microscaled").ri_mx_make, c_void_p).value, _held_bytes()
    return lambda t: fn(t, make, size)


class _NotPlain(KernelError, AttributeError):
    pass


class _Held:
    """What matrices and rows have in common: they are no tensors, and a kernel that would take them for one refuses them."""

    __slots__ = ()

    def __getattr__(self, name):
        raise _NotPlain(f"microscaled.{type(self).__name__} has no {name!r}: it is multiplied by the products of `kernels.linear` with matrices in 4 bits, "
                        "not given to operators that take tensors (`microscaled.values` makes one of it)")


class Matrix(_Held):
    """A weight matrix [n, k] in 4 bits, for the products of `kernels.linear`."""

    __slots__ = ("n", "k", "spans", "codes", "exponents", "device", "_described", "native")

    def __init__(self, n: int, k: int, codes: torch.Tensor, exponents: torch.Tensor):
        self.n, self.k, self.spans = n, k, _spans(k)
        self.codes, self.exponents, self.device = codes, exponents, codes.device
        self._described = _describe(codes, exponents, n, k, 4)
        self.native = self._described.data_ptr()

    @classmethod
    def of(cls, t: torch.Tensor) -> "Matrix":
        """The matrix nearest to t [n, k], float32 or bfloat16, whose rows may lie apart."""
        n, k = t.shape if t.dim() == 2 else (0, 0)
        _need(n > 0 and k > 0 and t.dtype in (torch.float32, torch.bfloat16),
              "microscaled.Matrix: a matrix [n, k] of at least one number, float32 or bfloat16, is wanted")
        ops._need_cuda(t)
        if not t.is_contiguous() and ((t.stride(1) != 1 and k > 1) or t.stride(0) < k):
            t = t.contiguous()
        m = cls.__new__(cls)
        m.codes, m.exponents, m._described = _maker()(t)
        m.n, m.k = n, k
        m.spans, m.device, m.native = _spans(k), t.device, m._described.data_ptr()
        return m

    @classmethod
    def _empty(cls, n, k, device) -> "Matrix":
        spans = _spans(k)
        # rows behind the last one, in its tile of 128, are read beside it and have no effect
        return cls(n, k, torch.zeros(-(-n // 128), spans, 128, SPAN // 2, dtype=torch.uint8, device=device),
                   torch.zeros(-(-n // 128), spans, PIECE, dtype=torch.uint8, device=device))

    @classmethod
    def of_codes(cls, codes: torch.Tensor, exponents: torch.Tensor, k: int) -> "Matrix":
        """From codes uint8 [n, ceil(k / 2)], number 2i in the low half of byte i (the sign, then the place among 0, 0.5, 1, 1.5, 2, 3, 4, 6),
        and exponents plus 127, uint8 [n, ceil(k / 32)] (255: NaN)."""
        n = codes.shape[0] if codes.dim() == 2 else 0
        _need(codes.dtype == torch.uint8 and exponents.dtype == torch.uint8 and n > 0 and k > 0 and tuple(codes.shape) == (n, -(-k // 2))
              and tuple(exponents.shape) == (n, -(-k // BLOCK)), "microscaled.Matrix: codes uint8 [n, ceil(k / 2)] and exponents uint8 [n, ceil(k / 32)] are wanted")
        ops._need_cuda(codes, exponents)
        _need(codes.device.index == torch.cuda.current_device() and exponents.device == codes.device, "microscaled.Matrix: codes and exponents lie on the current device")
        m = cls._empty(n, k, codes.device)
        spans, tiles = m.spans, m.exponents.shape[0]
        wide = torch.zeros(tiles * 128, spans * 64, dtype=torch.uint8, device=codes.device)
        wide[:n, :codes.shape[1]] = codes
        if k % 2:
            wide[:, k // 2] &= 15
        m.codes.copy_(wide.view(tiles, 128, spans, 64).transpose(1, 2))
        wide = torch.zeros(tiles * 128, spans * 4, dtype=torch.uint8, device=codes.device)
        wide[:n, :exponents.shape[1]] = exponents
        m.exponents.copy_(wide.view(-1, 4, 32, spans, 4).permute(0, 3, 2, 1, 4).reshape(-1, spans, PIECE))
        _call("microscaled", "ri_mx_settle", _stream())
        return m

    @property
    def shape(self):
        return self.n, self.k

    def bytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


class Rows(_Held):
    """Room for rows [n, k] in 8 bits, which a norm, a product or `quantize` fills and products read.  `codes` and `exponents`: buffers of
    the caller's own, uint8 and of `Rows.sizes(n, k)` bytes at least."""

    __slots__ = ("n", "k", "spans", "codes", "exponents", "device", "_described", "native")

    def __init__(self, n: int, k: int, device="cuda", codes: torch.Tensor | None = None, exponents: torch.Tensor | None = None):
        _need(n > 0 and k > 0, "microscaled.Rows: at least one row of at least one number")
        a, b = self.sizes(n, k)
        ops._need_cuda(codes, exponents)
        _need(codes is not None or torch.device(device).type == "cuda", "microscaled.Rows: rows lie on a CUDA device; this library has no CPU path")
        codes = torch.empty(a, dtype=torch.uint8, device=device) if codes is None else codes
        exponents = torch.empty(b, dtype=torch.uint8, device=codes.device) if exponents is None else exponents
        for t, least in ((codes, a), (exponents, b)):
            _need(t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous() and t.numel() >= least and t.device == codes.device and t.data_ptr() % 32 == 0,
                  "microscaled.Rows: buffers are contiguous uint8 on one CUDA device, on a 32-byte boundary and of Rows.sizes(n, k) bytes")
        self.n, self.k, self.spans = n, k, _spans(k)
        self.codes, self.exponents, self.device = codes, exponents, codes.device
        self._described = _describe(codes, exponents, n, k, 8)
        self.native = self._described.data_ptr()

    @staticmethod
    def sizes(n: int, k: int) -> tuple:
        """Bytes of the codes and of the exponents."""
        return n * _spans(k) * SPAN, -(-n // 128) * _spans(k) * PIECE

    @property
    def shape(self):
        return self.n, self.k


def quantize(x: torch.Tensor, out: Rows | None = None) -> Rows:
    """x [n, k], float32 or bfloat16, rows apart or not, in 8 bits."""
    if out is None:
        _need(x.dim() == 2, "microscaled.quantize: rows [n, k] are wanted")
        ops._need_cuda(x)
        out = Rows(*x.shape, x.device)
    _need(type(out) is Rows, "microscaled.quantize: out must be Rows")
    native("mx_hold")(x, out.native)
    return out


def values(held, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The numbers [n, k] that a `Matrix` or `Rows` stands for, in float32 or bfloat16 (which hold them exactly, but for results that
    the type has no room for)."""
    _need(type(held) is Matrix or type(held) is Rows, "microscaled.values: a Matrix or Rows are wanted")
    if out is None:
        _need(dtype in (torch.float32, torch.bfloat16), "microscaled.values: float32 or bfloat16 is wanted")
        return native("mx_values")(held.native, None, dtype is torch.bfloat16, held.n, held.k)
    _need(out.dtype is dtype, "microscaled.values: out is of the dtype asked for")
    native("mx_values")(held.native, out)
    return out


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: Rows, *, branch: torch.Tensor | None = None,
            total: torch.Tensor | None = None) -> Rows:
    """total = x + branch (x alone without a branch), and out = total / sqrt(mean(total^2) + eps) * weight in 8 bits.  x and weight
    float32, x [n, k]; branch float32 or bfloat16; total float32, x itself or another array, or None where it is not wanted."""
    _need(type(out) is Rows, "microscaled.rmsnorm: out must be Rows")
    native("mx_rmsnorm")(x, branch, weight, total, eps, out.native)
    return out


def product(x, w: Matrix, out, ctx, *, w2: Matrix | None = None, bias=None, form=None, act=None, add: bool = False):
    """out = x W^T + bias; with `act` an activation of it (`ops.whole_act_form`); with w2 the gated form of x W^T and x W2^T (`form`:
    `ops.gate_form`, None: silu); with `add` out<float32> += x W^T.  x: `Rows`, or plain rows, which are brought to 8 bits in the step's
    scratch; out: plain rows, or (not with `add`) `Rows`."""
    if type(w) is not Matrix or (w2 is not None and type(w2) is not Matrix):
        raise KernelError("microscaled.product: matrices in 4 bits are wanted")
    if type(x) is Rows:
        rows, x = x, None
    else:
        shape = x.shape
        if len(shape) != 2 or shape[0] == 0:
            _need(len(shape) == 2 and shape[1] == w.k and tuple(out.shape) == (0, w.n), "microscaled.product: rows [tokens, k] and a result [tokens, features] are wanted")
            return out
        rows = ctx.workspace.rows("mx_rows", shape[0], w.k)
    if (bias is not None) + (act is not None) + (w2 is not None) + add > 1 or (form is not None and w2 is None):
        raise KernelError("microscaled.product: a bias, an activation, a gate and an addition are not combined")
    constants = bias if bias is not None else ops.whole_act_form(act) if act is not None else ops.whole_gate_form(form) if form is not None else None
    held = type(out) is Rows
    _product()(x, rows.native, w.native, 0 if w2 is None else w2.native, constants, act is not None, add, None if held else out,
                         out.native if held else 0, _status_address())
    return out


@functools.lru_cache(maxsize=None)
def _product():
    native("mx_hold")                                            # brings plain rows to 8 bits where the product does not
    return native("mx_product")


@functools.lru_cache(maxsize=None)
def _status_address() -> int:
    from .tcgen05 import status_word
    return status_word().data_ptr()


def set_pairs(tokens: int = 0) -> None:
    """Products of at least so many tokens run on pairs of SMs, others do not; 0: whichever takes less time (for tests and comparisons)."""
    load("gemm_microscaled").ri_mx_set_pairs(c_int(tokens))
