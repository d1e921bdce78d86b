"""Microscaled operators refuse results that share memory with what they read (other blocks would read what the first ones have written).  The entry points
look at addresses and sizes before anything else, so that made-up ones, which nobody reads, do here; what lies apart gets as far as asking for a device."""
import ctypes
from ctypes import c_double, c_int, c_longlong, c_void_p

import pytest
import torch

from rust_inference_b200.kernels import build, microscaled

BASE = 1 << 32
NOWHERE = 1 << 20            # no such device: no call gets beyond that, on a machine with GPUs either
F32, BF16 = 0, 1


class Library:
    def __init__(self, module):
        self.lib = build.load(module)
        self.lib.ri_last_error.restype = ctypes.c_char_p

    def refuses(self, name, *args):
        assert getattr(self.lib, name)(*args) != 0
        return "apart" in self.lib.ri_last_error().decode()


@pytest.fixture(scope="module")
def numbers():
    return Library("microscaled")


@pytest.fixture(scope="module")
def products():
    return Library("gemm_microscaled")


def sizes(n, k, bits):
    spans = -(-k // 128)
    return (-(-n // 128) * 128 * 64 if bits == 4 else n * 128) * spans, -(-n // 128) * spans * 512


def make(numbers, n, k, bits, codes, exponents):
    at = torch.empty(microscaled._held_bytes(), dtype=torch.uint8)
    if numbers.lib.ri_mx_make(c_void_p(at.data_ptr()), c_void_p(codes), c_void_p(exponents), c_longlong(n), c_longlong(k), c_int(bits), c_int(NOWHERE)) != 0:
        return None
    return at


def p(at):
    return c_void_p(at.data_ptr() if isinstance(at, torch.Tensor) else at)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,k", [(1, 1), (130, 300)])
def test_codes_and_exponents(numbers, n, k, bits):
    a, b = sizes(n, k, bits)
    for exponents, fine in ((BASE + a, True), (BASE + a - 32, False), (BASE, False), (BASE - b, True), (BASE - b + 32, False)):
        assert (make(numbers, n, k, bits, BASE, exponents) is not None) == fine
        assert fine or "apart" in numbers.lib.ri_last_error().decode()


def around(start, size, mine, step=32):
    """Places of `mine` bytes, and whether they lie apart from `size` bytes from `start` on."""
    return [(start - mine, True), (start - mine + step, False), (start, False), (start + size - step, False), (start + size, True)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,item", [(F32, 4), (BF16, 2)])
def test_holding_and_reading_back(numbers, bits, dtype, item):
    n, k, ld = 40, 264, 300
    a, b = sizes(n, k, bits)
    held = make(numbers, n, k, bits, BASE, BASE + (1 << 24))
    for start, size in ((BASE, a), (BASE + (1 << 24), b)):
        for at, fine in around(start, size, ((n - 1) * ld + k) * item):
            assert numbers.refuses("ri_mx_hold", p(at), c_int(dtype), c_longlong(n), c_longlong(k), c_longlong(ld), p(held), p(0)) != fine
        for at, fine in around(start, size, n * k * item):
            assert numbers.refuses("ri_mx_values", p(held), c_int(dtype), c_longlong(n), c_longlong(k), p(at), p(0)) != fine


@pytest.mark.parametrize("which", ["x", "branch", "weight", "total"])
def test_norm(numbers, which):
    n, k = 40, 264
    a, b = sizes(n, k, 8)
    held = make(numbers, n, k, 8, BASE, BASE + (1 << 24))
    mine = {"x": n * k * 4, "branch": n * k * 2, "weight": k * 4, "total": n * k * 4}
    for start, size in ((BASE, a), (BASE + (1 << 24), b)):
        for at, fine in around(start, size, mine[which]):
            args = {"x": 2 * BASE, "branch": 3 * BASE, "weight": 4 * BASE, "total": 5 * BASE, which: at}
            assert numbers.refuses("ri_mx_rmsnorm", p(args["x"]), p(args["branch"]), c_int(BF16), p(args["weight"]), p(args["total"]), c_longlong(n), c_longlong(k),
                                   c_double(1e-5), p(held), p(0)) != fine


def test_norm_without_branch_and_total(numbers):
    held = make(numbers, 4, 64, 8, BASE, BASE + (1 << 24))
    assert not numbers.refuses("ri_mx_rmsnorm", p(2 * BASE), p(0), c_int(0), p(3 * BASE), p(0), c_longlong(4), c_longlong(64), c_double(1e-5), p(held), p(0))


@pytest.mark.parametrize("into_rows", [False, True])
@pytest.mark.parametrize("which", ["rows", "plain", "w", "w2", "constants"])
def test_product(numbers, products, which, into_rows):
    m, n, k, ld = 9, 200, 264, 280
    held = lambda rows, bits, i: make(numbers, rows, k, bits, i * BASE, i * BASE + (1 << 24))  # noqa: E731
    x, w, w2 = held(m, 8, 2), held(n, 4, 3), held(n, 4, 4)
    plain, constants = 5 * BASE, 6 * BASE
    regions = {"rows": [(2 * BASE, sizes(m, k, 8)[0]), (2 * BASE + (1 << 24), sizes(m, k, 8)[1])], "w": [(3 * BASE, sizes(n, k, 4)[0]), (3 * BASE + (1 << 24), sizes(n, k, 4)[1])],
               "w2": [(4 * BASE, sizes(n, k, 4)[0]), (4 * BASE + (1 << 24), sizes(n, k, 4)[1])], "plain": [(plain, ((m - 1) * ld + k) * 2)], "constants": [(constants, 20)]}

    def call(out, to):
        return products.refuses("ri_mx_product", p(x), p(plain), c_int(BF16), c_longlong(m), c_longlong(k), c_longlong(ld), p(w), p(w2), p(constants), c_longlong(5),
                                c_int(0), c_int(0), p(out), c_int(F32), c_longlong(m if out else 0), c_longlong(n if out else 0), p(to), p(0), p(0))

    a, b = sizes(m, n, 8)
    for start, size in regions[which]:
        if not into_rows:
            for at, fine in around(start, size, m * n * 4, 4):
                assert call(at, 0) != fine
            continue
        start, end = start // 32 * 32, -(-(start + size) // 32) * 32
        for at, fine in around(start, end - start, a):
            assert call(0, make(numbers, m, n, 8, at, 7 * BASE)) != fine
        for at, fine in around(start, end - start, b):
            assert call(0, make(numbers, m, n, 8, 7 * BASE, at)) != fine
