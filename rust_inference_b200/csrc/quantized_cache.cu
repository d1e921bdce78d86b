// A cache of keys and values in 8 bits: writing into it and reading it back.
//
// Pages of 64 positions as in the other caches, [page][kv head][64][head size], of codes int8 in -127..127, and one float32
// scale for every 16 positions of a page and kv head ([page][kv head][4]), keys and values apart.  A code c of a block with the
// scale s stands for s * c.
//
// Writing rows x into a block (keys after their rotation in float32; each product and each sum of it rounded once, so that
// the codes are a matter of the formula and not of what the compiler contracts):
//   a = max |x| over the block's new rows and channels,  s_new = a * (1 / 127), 0 where that is no normal number
//   the block holds earlier positions of the sequence:  s = max(s_old, s_new), and if that is larger than s_old
//       the older codes become rint(c * (s_old * (1 / s)))
//   else: s = s_new, whatever the page held for another sequence
//   c = rint(x * (1 / s)), all zero where s = 0
// A block that is given an infinity or a NaN gets the scale NaN and keeps it: all of it reads as NaN, until the page is given to
// another sequence.  A block's older codes are rounded again whenever its scale grows, at most half a step of the new
// scale each time.
#include "common.cuh"

#include <cuda_fp16.h>
#include <float.h>

using namespace ri;

namespace {

constexpr int PAGE = 64, BLOCK = 16, PER_PAGE = PAGE / BLOCK;
constexpr int THREADS = 128;

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

struct Written {                 // where a projection's columns go
    void* src;                   // [tokens][ld]: q heads, k heads, v heads
    int ld;
    const float* bias;           // [ld] or null
    int clear;                   // leave zeros in src behind (float32 accumulators of a product that was cut over K)
    void* q_out;                 // [tokens][n_heads * hd], rotated; null: no queries
    const float *cos_t, *sin_t;  // [positions][rot / 2]
    const int *page_table, *seq_slot, *seq_start, *cu_seqlens;
    int max_pages;
    int8_t *kc, *vc;
    float *ks, *vs;
    int n_heads, n_kv, hd, v_hd, rot, style;
    int n_seqs, runs;            // blocks of positions per sequence, at most; 0: counted through, sequence by sequence
};

// a pair of channels turned, every product and sum rounded once
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
    const float x0 = a, x1 = b;
    a = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
    b = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
}

// A position block of a step: rows lo..hi-1 of the sequence's positions base..base+15
struct Run { int seq, base, lo, hi, row0; };
__device__ __forceinline__ int runs_of(int start, int n) { return n > 0 ? (start + n - 1) / BLOCK - start / BLOCK + 1 : 0; }
__device__ __forceinline__ bool run_of(const Written& w, int i, Run& r) {
    r.seq = w.runs ? i / w.runs : w.n_seqs;
    int nth = w.runs ? i % w.runs : i;
    if (w.runs == 0) {                              // a lane per sequence
        const int lane = threadIdx.x & 31;
        for (int s0 = 0; s0 < w.n_seqs; s0 += 32) {
            const int s = s0 + lane;
            const int mine = s < w.n_seqs ? runs_of(w.seq_start[s], w.cu_seqlens[s + 1] - w.cu_seqlens[s]) : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int before = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += before;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > nth);
            if (past) {
                const int at = __ffs(past) - 1;
                r.seq = s0 + at;
                nth -= __shfl_sync(0xffffffffu, upto - mine, at);
                break;
            }
            nth -= __shfl_sync(0xffffffffu, upto, 31);
        }
        if (r.seq == w.n_seqs) return false;
    }
    const int first = w.cu_seqlens[r.seq], n = w.cu_seqlens[r.seq + 1] - first, start = w.seq_start[r.seq];
    r.base = (start / BLOCK + nth) * BLOCK;
    r.lo = max(r.base, start);
    r.hi = min(r.base + BLOCK, start + n);
    r.row0 = first + r.lo - start;
    return r.lo < r.hi;
}

// Any head sizes, any number of rotated channels, any alignment: a block of threads per (position block, head), which goes over
// its rows twice.
template <typename TS, typename TQ>
__global__ void __launch_bounds__(THREADS) write_any_kernel(Written w) {
    __shared__ float scratch[33];
    Run r;
    const bool some = run_of(w, blockIdx.x, r);
    let_next_kernel_start();
    wait_for_previous_kernels();
    if (!some) return;
    const int part = blockIdx.y;                    // k heads, v heads, q heads
    const bool is_k = part < w.n_kv, is_v = !is_k && part < 2 * w.n_kv;
    const int head = is_k ? part : (is_v ? part - w.n_kv : part - 2 * w.n_kv);
    const int size = is_v ? w.v_hd : w.hd, rot = is_v ? 0 : w.rot;
    const int col = is_k ? (w.n_heads + head) * w.hd : (is_v ? (w.n_heads + w.n_kv) * w.hd + head * w.v_hd : head * w.hd);
    TS* src = reinterpret_cast<TS*>(w.src);
    const int half = rot / 2, pairs = size / 2, n = (r.hi - r.lo) * pairs;

    // the i-th pair of channels of the row's head, rotated
    auto pair = [&](int row, int i, int& d0, int& d1, float& y0, float& y1) {
        const bool turned = i < half;
        d0 = turned && w.style == 0 ? i : (turned ? 2 * i : rot + 2 * (i - half));
        d1 = turned && w.style == 0 ? i + half : d0 + 1;
        const TS* at = src + (size_t)(r.row0 + row) * w.ld + col;
        const float x0 = to_f32<TS>(at[d0]) + (w.bias ? w.bias[col + d0] : 0.f);
        const float x1 = to_f32<TS>(at[d1]) + (w.bias ? w.bias[col + d1] : 0.f);
        y0 = x0;
        y1 = x1;
        if (turned) {
            const float c = w.cos_t[(size_t)(r.lo + row) * half + i], s = w.sin_t[(size_t)(r.lo + row) * half + i];
            rotate(y0, y1, c, s);
        }
    };
    auto cleared = [&](int row, int d0, int d1) {
        if (!w.clear) return;
        TS* at = src + (size_t)(r.row0 + row) * w.ld + col;
        at[d0] = at[d1] = from_f32<TS>(0.f);
    };
    int d0, d1;
    float y0, y1;
    if (!is_k && !is_v) {
        TQ* q = reinterpret_cast<TQ*>(w.q_out);
        for (int i = threadIdx.x; i < n; i += THREADS) {
            pair(i / pairs, i % pairs, d0, d1, y0, y1);
            TQ* at = q + (size_t)(r.row0 + i / pairs) * w.n_heads * w.hd + head * w.hd;
            at[d0] = from_f32<TQ>(y0);
            at[d1] = from_f32<TQ>(y1);
            cleared(i / pairs, d0, d1);
        }
        return;
    }
    const int slot = w.seq_slot[r.seq];
    if (!RI_BLOCK_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) || !RI_BLOCK_IN_RANGE(r.base / PAGE, w.max_pages, RI_CHECK_PAGE_INDEX)) return;
    const int page = w.page_table[(size_t)slot * w.max_pages + r.base / PAGE];
    if (!RI_BLOCK_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE)) return;
    const size_t tile = (size_t)page * w.n_kv + head;
    int8_t* codes = (is_k ? w.kc : w.vc) + (tile * PAGE + r.base % PAGE) * size;
    float* scale = (is_k ? w.ks : w.vs) + tile * PER_PAGE + r.base % PAGE / BLOCK;

    float a = 0.f;
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        pair(i / pairs, i % pairs, d0, d1, y0, y1);
        a = fmaxf(a, fmaxf(fabsf(y0), fabsf(y1)));
        bad |= !(fabsf(y0) <= FLT_MAX && fabsf(y1) <= FLT_MAX);
    }
    a = block_max(a, scratch);
    bad = __syncthreads_or(bad);
    const float had = r.base < r.lo ? *scale : 0.f;
    float s = a * (1.f / 127.f);
    s = fmaxf(s < FLT_MIN ? 0.f : s, had);
    if (bad || had != had) s = __int_as_float(0x7fffffff);
    const float inv = s > 0.f ? 1.f / s : 0.f;
    if (s > had) {
        const float f = had * inv;
        for (int i = threadIdx.x; i < (r.lo - r.base) * size; i += THREADS) codes[i] = (int8_t)__float2int_rn((float)codes[i] * f);
    }
    for (int i = threadIdx.x; i < n; i += THREADS) {
        pair(i / pairs, i % pairs, d0, d1, y0, y1);
        int8_t* at = codes + (r.lo - r.base + i / pairs) * size;
        at[d0] = (int8_t)__float2int_rn(y0 * inv);
        at[d1] = (int8_t)__float2int_rn(y1 * inv);
        cleared(i / pairs, d0, d1);
    }
    __syncthreads();                                // every thread has read the old scale
    if (threadIdx.x == 0) *scale = s;
}

// Heads of 64 or 128 whose channels are all rotated, or none, on 16-byte boundaries: two warps take eight rows each of a position
// block of one head (four heads to a block of threads, which read the same angles), each lane four pairs of channels of every second
// or fourth row; keys and values stay in registers between their maximum and their codes.  Angles are read before the wait for the
// kernel before.  What bounds it is memory: 8 prompts of 2,047 tokens (32 heads over 8 of 128) 75.7 us, 4.9 TB/s.
// How a lane's pairs lie in a head: (i, i + HD/2), or (2i, 2i + 1) for i = 4 lane' .. + 4; unrotated heads as the second.
template <typename T> struct Four;                 // four neighbouring numbers as they lie in memory
template <> struct Four<float> {
    float4 v;
    __device__ __forceinline__ void get(const float* p) { v = load_written(p); }
    __device__ __forceinline__ void open(float* f) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
};
template <> struct Four<__nv_bfloat16> {
    uint32_t x, y;
    __device__ __forceinline__ void get(const __nv_bfloat16* p) { asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "l"(p) : "memory"); }
    __device__ __forceinline__ void open(float* f) const {
        f[0] = __uint_as_float(x << 16), f[1] = __uint_as_float(x & 0xffff0000u);
        f[2] = __uint_as_float(y << 16), f[3] = __uint_as_float(y & 0xffff0000u);
    }
};
template <typename T> __device__ __forceinline__ void put4(T* p, const float* f);
template <> __device__ __forceinline__ void put4<float>(float* p, const float* f) { *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(f); }
template <> __device__ __forceinline__ void put4<__nv_bfloat16>(__nv_bfloat16* p, const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    uint2 v;
    v.x = *reinterpret_cast<const uint32_t*>(&a), v.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = v;
}
__device__ __forceinline__ uint32_t four_codes(const float* f, float inverse) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v |= (uint32_t)(__float2int_rn(f[i] * inverse) & 255) << (8 * i);
    return v;
}
__device__ __forceinline__ uint32_t rounded_again(uint32_t codes, float factor) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v |= (uint32_t)(__float2int_rn((float)(int8_t)(codes >> (8 * i)) * factor) & 255) << (8 * i);
    return v;
}

constexpr int HEADS = 4, HALF = BLOCK / 2;          // heads of a block of threads; rows of a warp

template <typename TS, typename TQ, int HD>
__global__ void __launch_bounds__(64 * HEADS, 4) write_kernel(Written w, int kv_blocks, int q_each) {
    constexpr int LANES = HD / 8, STRIDE = 32 / LANES, TURNS = HALF / STRIDE;      // lanes per row, rows per turn, turns
    __shared__ float most[2 * HEADS];
    __shared__ __align__(16) float angles[2][BLOCK][HD / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, sub = lane / LANES;
    let_next_kernel_start();
    Run r;
    const bool some = run_of(w, blockIdx.x, r);
    // the first blocks: k heads, v heads; then q heads
    const bool kv = (int)blockIdx.y < kv_blocks;
    const int part = kv ? (int)blockIdx.y * HEADS + (warp >> 1) : ((int)blockIdx.y - kv_blocks) * HEADS * q_each + (warp >> 1);
    const bool is_k = kv && part < w.n_kv;
    const int head = kv && !is_k ? part - w.n_kv : part;
    const bool here = some && part < (kv ? 2 * w.n_kv : w.n_heads);
    int col = !kv ? head * HD : (is_k ? w.n_heads + head : w.n_heads + w.n_kv + head) * HD;
    const bool turned = (is_k || !kv) && w.rot != 0, apart = turned && w.style == 0;
    const int d0 = apart ? 4 * l : 8 * l, d1 = d0 + (apart ? HD / 2 : 4);          // this lane's channels: four from d0, four from d1
    const int lo = r.lo - r.base, hi = r.hi - r.base, row0 = (warp & 1) * HALF + sub;      // the block's new rows; this lane's first row
    auto mine = [&](int turn) { return row0 + turn * STRIDE >= lo && row0 + turn * STRIDE < hi; };
    // the rows' angles (cosines, then sines), once for the block's heads
    if (some && w.rot != 0) {
        const size_t at = (size_t)(r.base + lo) * (HD / 2);
        for (int i = threadIdx.x; i < (hi - lo) * (HD / 8); i += 64 * HEADS) {
            reinterpret_cast<float4*>(angles[0][lo])[i] = reinterpret_cast<const float4*>(w.cos_t + at)[i];
            reinterpret_cast<float4*>(angles[1][lo])[i] = reinterpret_cast<const float4*>(w.sin_t + at)[i];
        }
    }
    bool there = false;
    int page = 0;
    if (kv && here) {
        const int slot = w.seq_slot[r.seq];
        // checked build: a slot, a page index or a page outside is recorded and nothing is written
        there = RI_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) && RI_IN_RANGE(r.base / PAGE, w.max_pages, RI_CHECK_PAGE_INDEX);
        if (there) page = w.page_table[(size_t)slot * w.max_pages + r.base / PAGE];
        there = there && RI_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE);
    }
    wait_for_previous_kernels();
    if (!some) return;
    TS* src = reinterpret_cast<TS*>(w.src) + ((ptrdiff_t)r.row0 - lo + row0) * w.ld + col;     // this lane's row of turn 0 (looked at from row lo on)

    Four<TS> raw[TURNS][2];
    auto get = [&](const TS* from) {
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
            if (mine(k)) {
                raw[k][0].get(from + (ptrdiff_t)k * STRIDE * w.ld + d0);
                raw[k][1].get(from + (ptrdiff_t)k * STRIDE * w.ld + d1);
            }
    };
    if (here) get(src);
    __syncthreads();                                // the angles are there
    auto finish = [&](int k, float* y) {            // bias, rotation, zeros behind
        raw[k][0].open(y);
        raw[k][1].open(y + 4);
        if (w.clear) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            TS* at = src + (ptrdiff_t)k * STRIDE * w.ld;
            put4<TS>(at + d0, zero);
            put4<TS>(at + d1, zero);
        }
        if (w.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] += w.bias[col + d0 + i], y[4 + i] += w.bias[col + d1 + i];
        }
        if (!turned) return;
        __align__(16) float c[4], s[4];
        *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(&angles[0][row0 + k * STRIDE][4 * l]);
        *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(&angles[1][row0 + k * STRIDE][4 * l]);
        if (apart) {
#pragma unroll
            for (int i = 0; i < 4; ++i) rotate(y[i], y[4 + i], c[i], s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) rotate(y[2 * i], y[2 * i + 1], c[i], s[i]);
        }
    };
    if (!kv) {
        // as many q heads as the launch gives a warp, four apart: the same rows and angles
        TQ* q = reinterpret_cast<TQ*>(w.q_out) + ((ptrdiff_t)r.row0 - lo + row0) * w.n_heads * HD + head * HD;
        for (int n = 0; n < q_each && part + n * HEADS < w.n_heads; ++n) {
#pragma unroll
            for (int k = 0; k < TURNS; ++k)
                if (mine(k)) {
                    float y[8];
                    finish(k, y);
                    TQ* at = q + (ptrdiff_t)k * STRIDE * w.n_heads * HD;
                    put4<TQ>(at + d0, y);
                    put4<TQ>(at + d1, y + 4);
                }
            src += HEADS * HD;
            col += HEADS * HD;
            if (n + 1 < q_each && part + (n + 1) * HEADS < w.n_heads) get(src);
            q += HEADS * HD;
        }
        return;
    }
    float y[TURNS][8];
    if (here) {
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
            if (mine(k)) finish(k, y[k]);
    }
    // the largest value, over the two warps of the rows' block; an infinity where one is no number
    float a = 0.f;
    bool fine = true;
    if (here) {
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
            if (mine(k)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a = fmaxf(a, fabsf(y[k][i]));
                    fine &= fabsf(y[k][i]) <= FLT_MAX;
                }
            }
    }
    a = warp_max(a);
    if (!__all_sync(0xffffffffu, fine)) a = INFINITY;
    if (lane == 0) most[warp] = a;
    const size_t tile = (size_t)page * w.n_kv + head;
    int8_t* codes = (is_k ? w.kc : w.vc) + (tile * PAGE + r.base % PAGE) * HD;
    float* scale = (is_k ? w.ks : w.vs) + tile * PER_PAGE + r.base % PAGE / BLOCK;
    const float had = there && lo > 0 ? *scale : 0.f;
    __syncthreads();                                // both warps' maxima are there, and both have read the old scale
    if (!there) return;
    a = fmaxf(a, most[warp ^ 1]);
    float s = a * (1.f / 127.f);
    s = fmaxf(s < FLT_MIN ? 0.f : s, had);
    if (!(a <= FLT_MAX) || had != had) s = __int_as_float(0x7fffffff);
    const float inverse = s > 0.f ? 1.f / s : 0.f;
    if (s > had && lo > 0) {
        for (int k = 0, row = row0; k < TURNS && row < lo; ++k, row += STRIDE) {
            uint32_t* at = reinterpret_cast<uint32_t*>(codes + row * HD);
            at[d0 / 4] = rounded_again(at[d0 / 4], had * inverse);
            at[d1 / 4] = rounded_again(at[d1 / 4], had * inverse);
        }
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        if (!mine(k)) continue;
        uint32_t* at = reinterpret_cast<uint32_t*>(codes + (row0 + k * STRIDE) * HD);
        at[d0 / 4] = four_codes(y[k], inverse);
        at[d1 / 4] = four_codes(y[k] + 4, inverse);
    }
    if (lane == 0 && warp % 2 == 0) *scale = s;
}

// The same for steps of one token per sequence: a warp for each head, a lane for two (four) of its channels, nothing to meet for.  What
// bounds it is the latency of its loads, which are all on their way at once, and of its instructions where the other kernels
// of a step have had theirs in the cache: so few of them: inside a step of 1, 8 and 64
// sequences (28 heads over 4 of 128, from sums with a bias) 2.3, 2.5 and 2.7 us, where the kernel above takes 6.4, 5.8 and 7.5; alone, 8 and 64
// sequences (32 over 8) 1.7 and 2.0, and 2.2 and 3.3.
constexpr int ONE_WARPS = 4;
template <int N, typename T> struct Few;           // N neighbouring numbers
template <> struct Few<2, float> {
    static __device__ __forceinline__ void get(const float* p, float* f) { asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(f[0]), "=f"(f[1]) : "l"(p) : "memory"); }
    static __device__ __forceinline__ void put(float* p, const float* f) { *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]); }
};
template <> struct Few<1, float> {
    static __device__ __forceinline__ void get(const float* p, float* f) { asm volatile("ld.global.f32 %0, [%1];" : "=f"(f[0]) : "l"(p) : "memory"); }
    static __device__ __forceinline__ void put(float* p, const float* f) { *p = f[0]; }
};
template <> struct Few<2, __nv_bfloat16> {
    static __device__ __forceinline__ void get(const __nv_bfloat16* p, float* f) {
        uint32_t v;
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
        f[0] = __uint_as_float(v << 16), f[1] = __uint_as_float(v & 0xffff0000u);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, const float* f) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(f[0], f[1]); }
};
template <> struct Few<1, __nv_bfloat16> {
    static __device__ __forceinline__ void get(const __nv_bfloat16* p, float* f) {
        unsigned short v;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
        f[0] = __uint_as_float((uint32_t)v << 16);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, const float* f) { *p = __float2bfloat16_rn(f[0]); }
};

template <typename TS, typename TQ, int HD>
__global__ void __launch_bounds__(32 * ONE_WARPS) write_one_kernel(Written w) {
    constexpr int N = HD / 64;                      // channels from d0 on, and from d1 on
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seq = blockIdx.x;
    const int part = (int)blockIdx.y * ONE_WARPS + warp;                               // k heads, v heads, q heads
    let_next_kernel_start();
    const bool is_k = part < w.n_kv, kv = part < 2 * w.n_kv;
    const int head = is_k ? part : (kv ? part - w.n_kv : part - 2 * w.n_kv);
    const int row = w.cu_seqlens[seq], pos = w.seq_start[seq], lo = pos % BLOCK;
    const bool here = part < 2 * w.n_kv + (w.q_out ? w.n_heads : 0) && w.cu_seqlens[seq + 1] > row;
    const int col = !kv ? head * HD : (is_k ? w.n_heads + head : w.n_heads + w.n_kv + head) * HD;
    const bool turned = (is_k || !kv) && w.rot != 0, apart = turned && w.style == 0;
    const int d0 = apart ? N * lane : 2 * N * lane, d1 = apart ? HD / 2 + N * lane : d0 + N;
    float c[N], sn[N], b[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = 1.f, sn[i] = b[i] = b[N + i] = 0.f;
    bool there = false;
    int page = 0;
    if (here) {
        if (turned) {
            Few<N, float>::get(w.cos_t + (size_t)pos * (HD / 2) + N * lane, c);
            Few<N, float>::get(w.sin_t + (size_t)pos * (HD / 2) + N * lane, sn);
        }
        if (w.bias != nullptr)
            for (int i = 0; i < N; ++i) b[i] = w.bias[col + d0 + i], b[N + i] = w.bias[col + d1 + i];
        if (kv) {
            const int slot = w.seq_slot[seq];
            // checked build: a slot, a page index or a page outside is recorded and nothing is written
            there = RI_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) && RI_IN_RANGE(pos / PAGE, w.max_pages, RI_CHECK_PAGE_INDEX);
            if (there) page = w.page_table[(size_t)slot * w.max_pages + pos / PAGE];
            there = there && RI_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE);
        }
    }
    wait_for_previous_kernels();
    if (!here) return;
    TS* src = reinterpret_cast<TS*>(w.src) + (size_t)row * w.ld + col;
    float y[2 * N];
    Few<N, TS>::get(src + d0, y);
    Few<N, TS>::get(src + d1, y + N);
    // the block's earlier positions: their scale, and their codes, sixteen bytes at a time
    constexpr int OLD = BLOCK * HD / 512;
    const size_t tile = (size_t)page * w.n_kv + head;
    int8_t* codes = (is_k ? w.kc : w.vc) + (tile * PAGE + pos % PAGE / BLOCK * BLOCK) * HD;
    float* scale = (is_k ? w.ks : w.vs) + tile * PER_PAGE + pos % PAGE / BLOCK;
    float had = 0.f;
    uint4 old[OLD];
    auto earlier = [&](int k) { return (k * 512 + lane * 16) / HD < lo; };
    if (there && lo > 0) {
        had = *scale;
#pragma unroll
        for (int k = 0; k < OLD; ++k)
            if (earlier(k)) old[k] = *reinterpret_cast<const uint4*>(codes + k * 512 + lane * 16);
    }
    if (w.clear) {
        const float zero[N] = {};
        Few<N, TS>::put(src + d0, zero);
        Few<N, TS>::put(src + d1, zero);
    }
    if (w.bias != nullptr)
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) y[i] += b[i];
    if (turned) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (apart || N == 1) rotate(y[i], y[N + i], c[i], sn[i]);
            else rotate(y[2 * i], y[2 * i + 1], c[i], sn[i]);
        }
    }
    if (!kv) {
        TQ* q = reinterpret_cast<TQ*>(w.q_out) + ((size_t)row * w.n_heads + head) * HD;
        Few<N, TQ>::put(q + d0, y);
        Few<N, TQ>::put(q + d1, y + N);
        return;
    }
    if (!there) return;
    float a = 0.f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        a = fmaxf(a, fabsf(y[i]));
        fine &= fabsf(y[i]) <= FLT_MAX;
    }
    a = warp_max(a);
    float s = a * (1.f / 127.f);
    s = fmaxf(s < FLT_MIN ? 0.f : s, had);
    if (!__all_sync(0xffffffffu, fine) || had != had) s = __int_as_float(0x7fffffff);
    const float inverse = s > 0.f ? 1.f / s : 0.f;
    if (s > had && lo > 0) {
        const float f = had * inverse;
#pragma unroll
        for (int k = 0; k < OLD; ++k)
            if (earlier(k))
                *reinterpret_cast<uint4*>(codes + k * 512 + lane * 16) =
                    make_uint4(rounded_again(old[k].x, f), rounded_again(old[k].y, f), rounded_again(old[k].z, f), rounded_again(old[k].w, f));
    }
    int8_t* to = codes + lo * HD;
#pragma unroll
    for (int i = 0; i < N; ++i) to[d0 + i] = (int8_t)__float2int_rn(y[i] * inverse), to[d1 + i] = (int8_t)__float2int_rn(y[N + i] * inverse);
    if (lane == 0) *scale = s;
}

// Reading back: a block of threads takes a page of one kv head, keys and values, as many codes per thread and turn as make sixteen
// bytes of values (a warp then writes whole sectors).  What bounds it is memory: 31,999 positions of 8 heads of 128 to bfloat16 36.8 us,
// 5.4 TB/s, 82% of what a copy reaches.  (Registers for 6 blocks per SM in bfloat16 and 7 in float32: with 8 in bfloat16 seven prompts of up
// to 2,047 tokens take 21.5 us with their writing instead of 20.7; with 6 in float32 8 sequences of 500 to 4,000 41.9 instead of 41.0.)
// ROWS: to rows of a sequence's own (cu_rows); else to pages.
constexpr int READERS = 256;
struct Read {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    void *k_out, *v_out;
    const int *page_table, *seq_slot, *seq_first, *seq_len, *cu_rows;   // cu_rows null: out has the cache's pages
    int max_pages, n_kv, hd, v_hd, pages;                              // pages: of a sequence, at most
    int out_pages;                                                     // 0: a page goes where it lies; else sequence b's i-th to b * out_pages + i
    int seen, span;                                                    // seen: from the first key that position seq_first sees (span)
};

template <typename T, bool VEC, bool ROWS>
__device__ __forceinline__ void read_tile(const Read& r, const int8_t* codes, const float* scales, T* out, int size, int head, int page,
                                          int out_page, int base, int first, int len, int row_of_0) {
    const size_t tile = (size_t)page * r.n_kv + head;
    T* const own = out + ((size_t)out_page * r.n_kv + head) * PAGE * size;             // (pages)
    codes += tile * PAGE * size;
    scales += tile * PER_PAGE;
    constexpr int PER = VEC ? 16 / sizeof(T) : 1, AT_ONCE = VEC ? 4 : 1;             // codes that make sixteen bytes of values; pieces at once
    for (int e0 = threadIdx.x * PER; e0 < PAGE * size; e0 += AT_ONCE * READERS * PER) {
        uint2 c[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int e = e0 + k * READERS * PER;
            if (e >= PAGE * size) break;
            if (PER == 8) c[k] = *reinterpret_cast<const uint2*>(codes + e);
            else if (PER == 4) c[k].x = *reinterpret_cast<const uint32_t*>(codes + e);
            else c[k].x = (uint8_t)codes[e];
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int e = e0 + k * READERS * PER;
            if (e >= PAGE * size) break;
            const int row = e / size, d = e % size, pos = base + row;
            const bool there = pos >= first && pos < len;    // the rest of a page reads as zeros
            if (ROWS && !there) continue;
            T* const to = ROWS ? out + ((ptrdiff_t)(row_of_0 + pos) * r.n_kv + head) * size + d : own + e;
            const float s = scales[row / BLOCK];
            __align__(16) float v[8];
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = there ? s * (float)(int8_t)((i < 4 ? c[k].x : c[k].y) >> (8 * (i & 3))) : 0.f;
            if (PER == 8) *reinterpret_cast<uint4*>(to) = pack8(v);
            else if (PER == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(v);
            else *to = from_f32<T>(v[0]);
        }
    }
}

template <typename T, bool VEC, bool ROWS>
__global__ void __launch_bounds__(READERS, sizeof(T) == 2 ? 6 : 7) read_kernel(Read r) {
    let_next_kernel_start();
    const int seq = blockIdx.x / r.pages, head = blockIdx.y;
    const int first = r.seen ? first_visible_key(r.seq_first[seq], r.span) : r.seq_first[seq], len = r.seq_len[seq];
    const int index = first / PAGE + (int)(blockIdx.x % r.pages), base = index * PAGE;
    const int row_of_0 = ROWS ? r.cu_rows[seq] - first : 0;            // the row of position 0, if it had one
    wait_for_previous_kernels();
    if (base >= len) return;
    const int slot = r.seq_slot[seq];
    if (!RI_BLOCK_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) || !RI_BLOCK_IN_RANGE(index, r.max_pages, RI_CHECK_PAGE_INDEX)) return;
    const int page = r.page_table[(size_t)slot * r.max_pages + index];
    if (!RI_BLOCK_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE)) return;
    const int out_page = r.out_pages ? seq * r.out_pages + index : page;
    read_tile<T, VEC, ROWS>(r, r.kc, r.ks, reinterpret_cast<T*>(r.k_out), r.hd, head, page, out_page, base, first, len, row_of_0);
    read_tile<T, VEC, ROWS>(r, r.vc, r.vs, reinterpret_cast<T*>(r.v_out), r.v_hd, head, page, out_page, base, first, len, row_of_0);
}

// A cache's pages for the prompts' attention (attention_tcgen05.cu): as float16 numbers over a power of two of their own per
// sequence and kv head, the one that brings the largest scale of the blocks that are read to [2^7, 2^8).  A block of threads takes
// a page of one kv head and finds that scale for itself (four numbers a page).  What a sequence does not see, before its first
// seen block and behind its end, is 0.  A block that is no number is that in its keys, whose scores a row that does not see them
// leaves out, and 0 in its values, which every row's sum runs over.
// Float16 has no finer numbers than 2^-32 of the largest scale, and the attention no finer weights than 2^-31 of a row's largest: with
// scales more than 2^12 apart the small ones, of rows that may not see the large ones, would be rounded by those.  Such a sequence's kv
// head gets bfloat16 numbers, which have the same 8 bits everywhere, and the factors -1 and 1, which say so.
struct Widen {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    __half *k_out, *v_out;
    float* factors;              // [sequences][2][kv heads]
    const int *page_table, *seq_slot, *seq_start, *seq_len;
    int max_pages, n_kv, pages, span;
    int out_pages;               // as in Read
};
constexpr int WIDENERS = 256;

__device__ __forceinline__ float power_above(float scale) {            // 2^e with scale / 2^e in [2^7, 2^8); 1 for no scale
    const int e = (int)(__float_as_uint(scale) >> 23) - 127 - 7;
    return scale > 0.f ? __uint_as_float((uint32_t)(127 + max(e, -126)) << 23) : 1.f;
}

constexpr unsigned APART = 12u << 23;              // as far apart as float16 numbers serve, as the bits of powers of two

template <int HD>
__global__ void __launch_bounds__(WIDENERS) widen_kernel(Widen w) {
    __shared__ uint4 found[WIDENERS / 32];          // the largest and the smallest scale of a warp's blocks, of keys and of values, by their bits
    __shared__ float scales[2][PER_PAGE];
    let_next_kernel_start();
    const int seq = blockIdx.x / w.pages, head = blockIdx.y, tid = threadIdx.x;
    const int start = w.seq_start[seq], len = w.seq_len[seq];
    const int first = first_visible_key(start, w.span) / BLOCK, last = (len - 1) / BLOCK;      // blocks that are seen
    const int index = first / PER_PAGE + (int)(blockIdx.x % w.pages), end = last / PER_PAGE + 1;
    const int slot = w.seq_slot[seq];
    wait_for_previous_kernels();
    if (len <= start || index >= end) return;
    if (!RI_BLOCK_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) || !RI_BLOCK_IN_RANGE(end - 1, w.max_pages, RI_CHECK_PAGE_INDEX)) return;
    const int* pages = w.page_table + (size_t)slot * w.max_pages;
    const int page = pages[index];
    if (!RI_BLOCK_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE)) return;
    const size_t tile = (size_t)page * w.n_kv + head, out_tile = w.out_pages ? ((size_t)seq * w.out_pages + index) * w.n_kv + head : tile;
    constexpr int TURNS = PAGE * HD / 8 / WIDENERS;
    uint2 k[TURNS], v[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        k[i] = reinterpret_cast<const uint2*>(w.kc + tile * PAGE * HD)[tid + i * WIDENERS];
        v[i] = reinterpret_cast<const uint2*>(w.vc + tile * PAGE * HD)[tid + i * WIDENERS];
    }
    uint4 range = make_uint4(0u, ~0u, 0u, ~0u);     // (positive numbers are in the order of their bits; zeros and what is no number are left out)
    for (int b = first + tid; b <= last; b += WIDENERS) {
        const int p = pages[b / PER_PAGE];
        if (!RI_IN_LIMIT(p, RI_LIMIT_PAGES, RI_CHECK_PAGE)) continue;
        const size_t at = ((size_t)p * w.n_kv + head) * PER_PAGE + b % PER_PAGE;
        const float ks = w.ks[at], vs = w.vs[at];
        if (ks > 0.f) range.x = max(range.x, __float_as_uint(ks)), range.y = min(range.y, __float_as_uint(ks));
        if (vs > 0.f) range.z = max(range.z, __float_as_uint(vs)), range.w = min(range.w, __float_as_uint(vs));
    }
    range = make_uint4(__reduce_max_sync(0xffffffffu, range.x), __reduce_min_sync(0xffffffffu, range.y), __reduce_max_sync(0xffffffffu, range.z),
                       __reduce_min_sync(0xffffffffu, range.w));
    if (tid % 32 == 0) found[tid / 32] = range;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WIDENERS / 32; ++i) {
        const uint4 f = found[i];
        range = make_uint4(max(range.x, f.x), min(range.y, f.y), max(range.z, f.z), min(range.w, f.w));
    }
    const bool apart = (range.x != 0u && range.x - range.y > APART) || (range.z != 0u && range.z - range.w > APART);
    const float k_unit = apart ? 1.f : power_above(__uint_as_float(range.x)), v_unit = apart ? 1.f : power_above(__uint_as_float(range.z));
    if (tid < PER_PAGE) {
        const int b = index * PER_PAGE + tid;
        const bool seen = b >= first && b <= last;
        const float ks = seen ? w.ks[tile * PER_PAGE + tid] : 0.f, vs = seen ? w.vs[tile * PER_PAGE + tid] : 0.f;
        scales[0][tid] = vs != vs ? vs : ks / k_unit;
        scales[1][tid] = vs != vs ? 0.f : vs / v_unit;
    }
    if (index == first / PER_PAGE && tid == 0) {
        w.factors[(size_t)(2 * seq) * w.n_kv + head] = apart ? -1.f : k_unit;
        w.factors[(size_t)(2 * seq + 1) * w.n_kv + head] = v_unit;
    }
    __syncthreads();
    auto widened = [&](const uint2& c, float s, bool there) {
        uint4 o;
        __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = (i < 2 ? c.x : c.y) >> (16 * (i & 1));
            const float x = there ? s * (float)(int8_t)two : 0.f, y = there ? s * (float)(int8_t)(two >> 8) : 0.f;
            if (apart) reinterpret_cast<__nv_bfloat162*>(h)[i] = __floats2bfloat162_rn(x, y);
            else h[i] = __floats2half2_rn(x, y);
        }
        return o;
    };
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int e = tid + i * WIDENERS, row = e / (HD / 8);
        const bool there = index * PAGE + row < len;
        reinterpret_cast<uint4*>(w.k_out + out_tile * PAGE * HD)[e] = widened(k[i], scales[0][row / BLOCK], there);
        reinterpret_cast<uint4*>(w.v_out + out_tile * PAGE * HD)[e] = widened(v[i], scales[1][row / BLOCK], there);
    }
}

}  // namespace

// The pages that a step's queries see (all keys, or a span of them: first_visible_key) as float16 numbers, and
// float32 factors [n_seqs][2][n_kv] that keys and values are to be multiplied by (keys' -1: bfloat16 numbers, as they are).  out_pages 0: the outputs have the cache's shape; else
// they are [n_seqs * out_pages, ...], and a sequence's i-th page is that one's own (max_len / 64 rounded up or more).  Heads of
// 64 or 128; max_len: no sequence is longer.
RI_API int ri_quantized_widen(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* k_out, void* v_out, float* factors,
                              const int* page_table, int max_pages, const int* seq_slot, const int* seq_start, const int* seq_len,
                              int n_seqs, int max_len, int n_kv, int hd, int span, int out_pages, cudaStream_t stream) {
    if (n_seqs <= 0 || max_len <= 0) return 0;
    if (hd != 64 && hd != 128) return fail("quantized_widen: heads of %d channels (64 or 128 wanted)", hd);
    if (n_kv > 65535) return fail("quantized_widen: %d kv heads are too many", n_kv);
    if (!aligned16(kc) || !aligned16(vc) || !aligned16(k_out) || !aligned16(v_out)) return fail("quantized_widen: pages must lie on 16-byte boundaries");
    const int pages = (max_len + PAGE - 1) / PAGE;
    if ((long long)pages * n_seqs > 0x7fffffff) return fail("quantized_widen: %d sequences of %d positions are too many", n_seqs, max_len);
    if (out_pages < 0 || (out_pages > 0 && out_pages < pages)) return fail("quantized_widen: %d pages for %d positions", out_pages, max_len);
    const Widen w = {kc, vc, ks, vs, (__half*)k_out, (__half*)v_out, factors, page_table, seq_slot, seq_start, seq_len, max_pages, n_kv, pages, span, out_pages};
    const dim3 grid((unsigned)(pages * n_seqs), (unsigned)n_kv);
    auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, grid, dim3(WIDENERS), 0, stream, w), "quantized_widen"); };
    return hd == 64 ? launch(widen_kernel<64>) : launch(widen_kernel<128>);
}

// src [tokens, ld] of src_dtype holds q heads, k heads, v heads (plus bias where one is given); queries, rotated, go to q_out
// [tokens, n_heads * hd] of q_dtype, keys and values into the cache.  `rot` channels of q and k are rotated (0: none), style 0:
// pairs (i, i + rot / 2), style 1: pairs (2i, 2i + 1).  n_tokens: rows of src; max_new: the most tokens that a sequence brings.  clear: src is left zeroed.
RI_API int ri_quantized_write(void* src, int src_dtype, int ld, const float* bias, int clear, void* q_out, int q_dtype, const float* cos_t,
                              const float* sin_t, const int* page_table, int max_pages, const int* seq_slot, const int* seq_start,
                              const int* cu_seqlens, int8_t* kc, int8_t* vc, float* ks, float* vs, int n_tokens, int n_seqs, int max_new, int n_heads,
                              int n_kv, int hd, int v_hd, int rot, int style, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return 0;
    if (hd <= 0 || v_hd <= 0 || hd % 2 || v_hd % 2) return fail("quantized_write: heads of %d and %d channels (even numbers wanted)", hd, v_hd);
    if (rot < 0 || rot % 2 || rot > hd) return fail("quantized_write: %d rotated channels of a head of %d", rot, hd);
    if (style != 0 && style != 1) return fail("quantized_write: unknown style %d", style);
    if (n_heads < 0 || n_kv <= 0 || n_heads + 2ll * n_kv > 65535) return fail("quantized_write: %d heads and %d kv heads", n_heads, n_kv);
    // Blocks of positions: so many per sequence, or, where most sequences bring far fewer tokens than the longest, counted through (a warp
    // then walks the sequences' lengths, but fewer blocks of threads find nothing to do): 16 sequences of 1 to 2,047 tokens 28.1 us by
    // sequence, 25.9 counted through; 2 of 1 to 333 3.41 and 3.30.
    const long long each = (max_new + 2 * BLOCK - 2) / BLOCK, counted = n_tokens / BLOCK + 2ll * n_seqs;
    const bool direct = each * n_seqs <= counted;
    if ((direct ? each * n_seqs : counted) > 0x7fffffff) return fail("quantized_write: %d sequences of %d tokens are too many", n_seqs, max_new);
    const int runs = (int)(direct ? each * n_seqs : counted);
    const Written w = {src, ld, bias, clear, q_out, cos_t, sin_t, page_table, seq_slot, seq_start, cu_seqlens, max_pages, kc, vc, ks, vs,
                       n_heads, n_kv, hd, v_hd, rot, style, n_seqs, direct ? (int)each : 0};
    const int heads = 2 * n_kv + (q_out ? n_heads : 0);
    const int item = src_dtype == RI_F32 ? 4 : 2;
    if ((hd == 64 || hd == 128) && v_hd == hd && (rot == 0 || rot == hd) && ld * item % 16 == 0 && aligned16(src) && aligned16(q_out) &&
        aligned16(cos_t) && aligned16(sin_t) && aligned16(kc) && aligned16(vc)) {
        using B = __nv_bfloat16;
        if (max_new == 1) {
            const dim3 one((unsigned)n_seqs, (unsigned)((heads + ONE_WARPS - 1) / ONE_WARPS));
            auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, one, dim3(32 * ONE_WARPS), 0, stream, w), "quantized_write"); };
            if (src_dtype == RI_F32 && q_dtype == RI_F32) return hd == 64 ? launch(write_one_kernel<float, float, 64>) : launch(write_one_kernel<float, float, 128>);
            if (src_dtype == RI_F32 && q_dtype == RI_BF16) return hd == 64 ? launch(write_one_kernel<float, B, 64>) : launch(write_one_kernel<float, B, 128>);
            if (src_dtype == RI_BF16 && q_dtype == RI_BF16) return hd == 64 ? launch(write_one_kernel<B, B, 64>) : launch(write_one_kernel<B, B, 128>);
        }
        // A warp takes one q head, or two or four of the same rows (address arithmetic and the angles' reads are then shared): one while the
        // SMs hold the grid at once, four blocks each; two up to twice as much.  One, two and four, us (steps of one token are not here):
        //   32 heads over 8 of 128:  16 sequences of 2 tokens (384 blocks at one) 2.3, 2.5, 2.9;  32 (768) 3.1, 2.8, 3.5;  64 (1,536) 5.2, 4.7, 4.7;
        //     2,047 tokens (1,548) 12.6, 12.0, 13.6;  3 times 1,000 (2,304) 17.6, 16.7, 16.7;  8 times 2,047 (12,384) 83.5, 76.7, 75.5
        //   28 over 4:  64 sequences of 5 (1,152) 4.7, 4.2, 4.7;  2,047 tokens (1,161) 9.3, 9.3, 9.8;  8 times 2,047 (9,288) 61.5, 56.0, 54.7
        const int kv_blocks = (2 * n_kv + HEADS - 1) / HEADS;
        const auto blocks_for = [&](int each) { return q_out ? (n_heads + HEADS * each - 1) / (HEADS * each) : 0; };
        const auto waves = [&](int each) { return (long long)runs * (kv_blocks + blocks_for(each)) / (4.f * sm_count()); };
        const int q_each = waves(1) <= 1.f ? 1 : (waves(2) <= 2.f ? 2 : 4);
        const int q_blocks = blocks_for(q_each);
        const dim3 grid((unsigned)runs, (unsigned)(kv_blocks + q_blocks));
        auto launch = [&](auto kernel) {
            return check_launch(launch_dependent(kernel, grid, dim3(64 * HEADS), 0, stream, w, kv_blocks, q_each), "quantized_write");
        };
        if (src_dtype == RI_F32 && q_dtype == RI_F32) return hd == 64 ? launch(write_kernel<float, float, 64>) : launch(write_kernel<float, float, 128>);
        if (src_dtype == RI_F32 && q_dtype == RI_BF16) return hd == 64 ? launch(write_kernel<float, B, 64>) : launch(write_kernel<float, B, 128>);
        if (src_dtype == RI_BF16 && q_dtype == RI_BF16) return hd == 64 ? launch(write_kernel<B, B, 64>) : launch(write_kernel<B, B, 128>);
    }
    const dim3 grid((unsigned)runs, (unsigned)heads);
    auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, grid, dim3(THREADS), 0, stream, w), "quantized_write"); };
    if (src_dtype == RI_F32 && q_dtype == RI_F32) return launch(write_any_kernel<float, float>);
    if (src_dtype == RI_F32 && q_dtype == RI_BF16) return launch(write_any_kernel<float, __nv_bfloat16>);
    if (src_dtype == RI_BF16 && q_dtype == RI_BF16) return launch(write_any_kernel<__nv_bfloat16, __nv_bfloat16>);
    return fail("quantized_write: unknown dtypes %d, %d", src_dtype, q_dtype);
}

// Values of the positions seq_first..seq_len - 1 of every sequence (seen: from the first key that a query at seq_first sees within
// `span`, see first_visible_key).  cu_rows null: k_out, v_out get whole pages (zeros elsewhere in them), out_pages as in
// ri_quantized_widen; else they are [rows, kv heads, head size] and sequence b's rows begin at cu_rows[b].
// max_len: no sequence is longer.
RI_API int ri_quantized_read(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* k_out, void* v_out, int dtype,
                             const int* page_table, int max_pages, const int* seq_slot, const int* seq_first, const int* seq_len,
                             const int* cu_rows, int n_seqs, int max_len, int n_kv, int hd, int v_hd, int seen, int span, int out_pages, cudaStream_t stream) {
    if (n_seqs <= 0 || max_len <= 0) return 0;
    if (n_kv > 65535) return fail("quantized_read: %d kv heads are too many", n_kv);
    const int pages = (max_len + PAGE - 1) / PAGE;
    if ((long long)pages * n_seqs > 0x7fffffff) return fail("quantized_read: %d sequences of %d positions are too many", n_seqs, max_len);
    if (out_pages < 0 || (out_pages > 0 && out_pages < pages)) return fail("quantized_read: %d pages for %d positions", out_pages, max_len);
    const Read r = {kc, vc, ks, vs, k_out, v_out, page_table, seq_slot, seq_first, seq_len, cu_rows, max_pages, n_kv, hd, v_hd, pages, out_pages, seen, span};
    const dim3 grid((unsigned)(pages * n_seqs), (unsigned)n_kv);
    const bool vec = hd % 8 == 0 && v_hd % 8 == 0 && aligned16(kc) && aligned16(vc) && aligned16(k_out) && aligned16(v_out);
    auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, grid, dim3(READERS), 0, stream, r), "quantized_read"); };
    auto form = [&](auto rows_kernel, auto pages_kernel) { return cu_rows != nullptr ? launch(rows_kernel) : launch(pages_kernel); };
    using B = __nv_bfloat16;
    if (dtype == RI_F32) return vec ? form(read_kernel<float, true, true>, read_kernel<float, true, false>) : form(read_kernel<float, false, true>, read_kernel<float, false, false>);
    if (dtype == RI_BF16) return vec ? form(read_kernel<B, true, true>, read_kernel<B, true, false>) : form(read_kernel<B, false, true>, read_kernel<B, false, false>);
    return fail("quantized_read: unknown dtype %d", dtype);
}

RI_DEFINE_LAST_ERROR()
