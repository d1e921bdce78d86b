// Microscaled numbers: 32 consecutive numbers of a row share a power of two, 2^e, whose exponent is kept as the byte e + 127, and each
// is kept as the nearest number of a small type times 2^e (ties to the even one): four bits, +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, or eight
// (e4m3, up to 448).  e is the smallest exponent, -127 at least, for which nothing in the block exceeds the type's largest number times 2^e.
// A block with an infinity or a NaN among its numbers has the byte 255 and stands for 32 NaNs.
//
// [n, k] such numbers are held with k rounded up to whole `SPAN`s of 128, zeros behind a row's end.  Rows in 8 bits: codes [n, span count * 128].
// A matrix in 4 bits, whose n is rounded up to whole 128s too, lies as the products read it, a tile of 128 rows and a span, 8 KB, after the other,
// [row / 128][span][128][64 bytes], number 2i in the low half of byte i (in rows as long as the matrix's, a tile would be 128 pieces of 64 bytes that
// lie far apart: two large matrices for 8 tokens 2 to 3% slower).  Exponents lie in the order in which the tensor cores' scale registers take them: one piece of 512
// bytes for every 128 rows and span, [row / 128][span], the exponent of row r and the span's block j (0..3) at (r % 32) * 16 + r % 128 / 32 * 4 + j.
#pragma once

#include "common.cuh"

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <new>

namespace ri {
namespace mx {

constexpr int BLOCK = 32;              // numbers that share an exponent
constexpr int SPAN = 128;              // numbers of a row that one step of a product takes
constexpr int PIECE = 512;             // bytes of exponents of 128 rows and one span

// A matrix or rows as the entry points take them: host memory of the caller's, made by `ri_mx_make` once, beside the device's buffers.  The
// products' tensor maps are encoded when they are first wanted, a pair (codes, exponents) for every 16 rows of a box.
struct Held {
    uint8_t *codes, *exponents;
    int n, k, n_spans, bits, device;
    std::atomic<uint32_t> made;            // which of the maps are there
    alignas(64) unsigned char maps[8][256];
};

__host__ __device__ __forceinline__ int spans(int k) { return (k + SPAN - 1) / SPAN; }

// Whether two pieces of memory (or none, where one is null) have no byte in common.
inline bool apart(const void* a, long long a_bytes, const void* b, long long b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a == nullptr || b == nullptr || x + (uintptr_t)a_bytes <= y || y + (uintptr_t)b_bytes <= x;
}
inline long long code_bytes(long long n, int n_spans, int bits) { return (bits == 4 ? (n + 127) / 128 * 128 * (SPAN / 2) : n * SPAN) * n_spans; }
inline long long exponent_bytes(long long n, int n_spans) { return (n + 127) / 128 * n_spans * PIECE; }
inline bool apart(const Held* h, const void* p, long long bytes) {
    return apart(h->codes, code_bytes(h->n, h->n_spans, h->bits), p, bytes) && apart(h->exponents, exponent_bytes(h->n, h->n_spans), p, bytes);
}
inline bool apart(const Held* a, const Held* b) {
    return apart(a, b->codes, code_bytes(b->n, b->n_spans, b->bits)) && apart(a, b->exponents, exponent_bytes(b->n, b->n_spans));
}
inline long long item_bytes(int dtype) { return dtype == RI_BF16 ? 2 : 4; }
__device__ __forceinline__ size_t exponent_at(int row, int block, int n_spans) {
    return ((size_t)(row >> 7) * n_spans + (block >> 2)) * PIECE + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// The byte of the code of row `row` and column c.
template <int BITS>
__device__ __forceinline__ size_t code_at(int row, int c, int n_spans) {
    if (BITS == 8) return (size_t)row * n_spans * SPAN + c;
    return (((size_t)(row >> 7) * n_spans + (c >> 7)) * 128 + (row & 127)) * (SPAN / 2) + (c & 127) / 2;
}

// The exponent byte of a block whose largest magnitude has these bits (a float's, so that a NaN's are larger than any number's).  The
// largest number of the type is 1.5 * 2^2 or 1.75 * 2^8.
template <int BITS>
__device__ __forceinline__ uint32_t exponent_byte(uint32_t largest) {
    constexpr uint32_t MOST = BITS == 4 ? 0x400000u : 0x600000u, UP = BITS == 4 ? 2u : 8u;
    const uint32_t e = largest >> 23;
    if (e == 255u) return 255u;
    const uint32_t want = e + ((largest & 0x7fffffu) > MOST ? 1u : 0u);
    return e == 0u || want < UP ? 0u : want - UP;       // (a subnormal number is far below 2^-127 times the type's largest)
}
// 2^-e, which brings a block's numbers to the type (0 for the byte 255, whose codes say nothing)
__device__ __forceinline__ float to_type(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
// 2^e
__device__ __forceinline__ float from_type(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// The codes of eight numbers (already times 2^-e): a word of four bits each.
__device__ __forceinline__ uint32_t four_bits(const float* y) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_E2M1, cudaRoundNearest) << (8 * i);
    return w;
}
__device__ __forceinline__ uint32_t eight_bits(const float* y) {       // of four numbers
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}
// Two codes, in the low halves of a word's halves, as bfloat16 numbers: exponent and mantissa in place, times the difference of the
// exponents' biases.  (Only shifts and products, whose rate conversions do not have.)
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
__device__ __forceinline__ uint32_t as_word(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __nv_bfloat162 eight_to_bf162(uint32_t w) { return __hmul2(as_bf162((w & 0x00800080u) << 8 | (w & 0x007f007fu) << 4), as_bf162(0x7b807b80u)); }
__device__ __forceinline__ __nv_bfloat162 four_to_bf162(uint32_t w) { return __hmul2(as_bf162((w & 0x00080008u) << 12 | (w & 0x00070007u) << 6), as_bf162(0x7e807e80u)); }
// 2^e and 2^-e
__device__ __forceinline__ __nv_bfloat162 from_type_bf162(uint32_t byte) {
    const uint32_t h = byte == 255u ? 0x7fc0u : byte == 0u ? 0x0040u : byte << 7;
    return as_bf162(h | h << 16);
}
__device__ __forceinline__ __nv_bfloat162 to_type_bf162(uint32_t byte) {
    const uint32_t h = byte == 255u ? 0u : (254u - byte) << 7;
    return as_bf162(h | h << 16);
}
__device__ __forceinline__ uint8_t eight_bits_of_one(float y) { return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3); }

}  // namespace mx
}  // namespace ri
