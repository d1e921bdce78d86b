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

#include <float.h>

using namespace ri;

namespace {

constexpr int PAGE = 64, BLOCK = 16, PER_PAGE = PAGE / BLOCK;
constexpr int THREADS = 128;

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
    int runs;                    // blocks of positions per sequence, at most
};

// A position block of a step: rows lo..hi-1 of the sequence's positions base..base+15
struct Run { int seq, base, lo, hi, row0; };
__device__ __forceinline__ bool run_of(const Written& w, int i, Run& r) {
    r.seq = i / w.runs;
    const int first = w.cu_seqlens[r.seq], n = w.cu_seqlens[r.seq + 1] - first, start = w.seq_start[r.seq];
    r.base = (start / BLOCK + i % w.runs) * BLOCK;
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
            y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
            y1 = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
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

// Reading back: a block of threads takes a page of one kv head, keys and values, sixteen codes per thread and turn.  What
// bounds it is memory.
struct Read {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    void *k_out, *v_out;
    const int *page_table, *seq_slot, *seq_first, *seq_len, *cu_rows;   // cu_rows null: out has the cache's pages
    int max_pages, n_kv, hd, v_hd, pages;                              // pages: of a sequence, at most
    int seen, span;                                                    // seen: from the first key that position seq_first sees (span)
};

template <typename T> __device__ __forceinline__ void put16(T* to, const float* v);
template <> __device__ __forceinline__ void put16<float>(float* to, const float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(to)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
template <> __device__ __forceinline__ void put16<__nv_bfloat16>(__nv_bfloat16* to, const float* v) {
    reinterpret_cast<uint4*>(to)[0] = pack8(v);
    reinterpret_cast<uint4*>(to)[1] = pack8(v + 8);
}

template <typename T, bool VEC>
__device__ __forceinline__ void read_tile(const Read& r, const int8_t* codes, const float* scales, T* out, int size, int head, int page,
                                          int base, int first, int len, int seq) {
    const size_t tile = (size_t)page * r.n_kv + head;
    codes += tile * PAGE * size;
    scales += tile * PER_PAGE;
    const int step = VEC ? 16 : 1;
    for (int e = threadIdx.x * step; e < PAGE * size; e += blockDim.x * step) {
        const int row = e / size, d = e % size, pos = base + row;
        T* to;
        if (r.cu_rows != nullptr) {
            if (pos < first || pos >= len) continue;
            to = out + ((size_t)(r.cu_rows[seq] + pos - first) * r.n_kv + head) * size + d;
        } else {
            to = out + tile * PAGE * size + e;
        }
        const float s = scales[row / BLOCK];
        const bool there = pos >= first && pos < len;    // the rest of a page reads as zeros
        if (VEC) {
            const int4 c = *reinterpret_cast<const int4*>(codes + e);
            __align__(16) float v[16];
            const int8_t* b = reinterpret_cast<const int8_t*>(&c);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = there ? s * (float)b[i] : 0.f;
            put16<T>(to, v);
        } else {
            *to = from_f32<T>(there ? s * (float)codes[e] : 0.f);
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) read_kernel(Read r) {
    let_next_kernel_start();
    const int seq = blockIdx.x / r.pages, head = blockIdx.y;
    const int first = r.seen ? first_visible_key(r.seq_first[seq], r.span) : r.seq_first[seq], len = r.seq_len[seq];
    const int index = first / PAGE + (int)(blockIdx.x % r.pages), base = index * PAGE;
    wait_for_previous_kernels();
    if (base >= len) return;
    const int slot = r.seq_slot[seq];
    if (!RI_BLOCK_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) || !RI_BLOCK_IN_RANGE(index, r.max_pages, RI_CHECK_PAGE_INDEX)) return;
    const int page = r.page_table[(size_t)slot * r.max_pages + index];
    if (!RI_BLOCK_IN_LIMIT(page, RI_LIMIT_PAGES, RI_CHECK_PAGE)) return;
    read_tile<T, VEC>(r, r.kc, r.ks, reinterpret_cast<T*>(r.k_out), r.hd, head, page, base, first, len, seq);
    read_tile<T, VEC>(r, r.vc, r.vs, reinterpret_cast<T*>(r.v_out), r.v_hd, head, page, base, first, len, seq);
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

// src [tokens, ld] of src_dtype holds q heads, k heads, v heads (plus bias where one is given); queries, rotated, go to q_out
// [tokens, n_heads * hd] of q_dtype, keys and values into the cache.  `rot` channels of q and k are rotated (0: none), style 0:
// pairs (i, i + rot / 2), style 1: pairs (2i, 2i + 1).  max_new: the most tokens that a sequence brings.  clear: src is left zeroed.
RI_API int ri_quantized_write(void* src, int src_dtype, int ld, const float* bias, int clear, void* q_out, int q_dtype, const float* cos_t,
                              const float* sin_t, const int* page_table, int max_pages, const int* seq_slot, const int* seq_start,
                              const int* cu_seqlens, int8_t* kc, int8_t* vc, float* ks, float* vs, int n_seqs, int max_new, int n_heads,
                              int n_kv, int hd, int v_hd, int rot, int style, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return 0;
    if (hd <= 0 || v_hd <= 0 || hd % 2 || v_hd % 2) return fail("quantized_write: heads of %d and %d channels (even numbers wanted)", hd, v_hd);
    if (rot < 0 || rot % 2 || rot > hd) return fail("quantized_write: %d rotated channels of a head of %d", rot, hd);
    if (style != 0 && style != 1) return fail("quantized_write: unknown style %d", style);
    if (n_heads + 2 * n_kv > 65535) return fail("quantized_write: %d heads are too many", n_heads + 2 * n_kv);
    const int runs = (max_new + 2 * BLOCK - 2) / BLOCK;
    if ((long long)runs * n_seqs > 0x7fffffff) return fail("quantized_write: %d sequences of %d tokens are too many", n_seqs, max_new);
    const Written w = {src, ld, bias, clear, q_out, cos_t, sin_t, page_table, seq_slot, seq_start, cu_seqlens, max_pages, kc, vc, ks, vs,
                       n_heads, n_kv, hd, v_hd, rot, style, runs};
    const dim3 grid((unsigned)(runs * n_seqs), (unsigned)(2 * n_kv + (q_out ? n_heads : 0)));
    auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, grid, dim3(THREADS), 0, stream, w), "quantized_write"); };
    if (src_dtype == RI_F32 && q_dtype == RI_F32) return launch(write_any_kernel<float, float>);
    if (src_dtype == RI_F32 && q_dtype == RI_BF16) return launch(write_any_kernel<float, __nv_bfloat16>);
    if (src_dtype == RI_BF16 && q_dtype == RI_BF16) return launch(write_any_kernel<__nv_bfloat16, __nv_bfloat16>);
    return fail("quantized_write: unknown dtypes %d, %d", src_dtype, q_dtype);
}

// Values of the positions seq_first..seq_len - 1 of every sequence (seen: from the first key that a query at seq_first sees within
// `span`, see first_visible_key).  cu_rows null: k_out, v_out have the cache's shape and get whole pages (zeros elsewhere in them); else they are [rows, kv heads, head size] and sequence b's rows begin at cu_rows[b].
// max_len: no sequence is longer.
RI_API int ri_quantized_read(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* k_out, void* v_out, int dtype,
                             const int* page_table, int max_pages, const int* seq_slot, const int* seq_first, const int* seq_len,
                             const int* cu_rows, int n_seqs, int max_len, int n_kv, int hd, int v_hd, int seen, int span, cudaStream_t stream) {
    if (n_seqs <= 0 || max_len <= 0) return 0;
    if (n_kv > 65535) return fail("quantized_read: %d kv heads are too many", n_kv);
    const int pages = (max_len + PAGE - 1) / PAGE;
    if ((long long)pages * n_seqs > 0x7fffffff) return fail("quantized_read: %d sequences of %d positions are too many", n_seqs, max_len);
    const Read r = {kc, vc, ks, vs, k_out, v_out, page_table, seq_slot, seq_first, seq_len, cu_rows, max_pages, n_kv, hd, v_hd, pages, seen, span};
    const dim3 grid((unsigned)(pages * n_seqs), (unsigned)n_kv);
    const bool vec = hd % 16 == 0 && v_hd % 16 == 0 && aligned16(kc) && aligned16(vc) && aligned16(k_out) && aligned16(v_out);
    auto launch = [&](auto kernel) { return check_launch(launch_dependent(kernel, grid, dim3(256), 0, stream, r), "quantized_read"); };
    if (dtype == RI_F32) return vec ? launch(read_kernel<float, true>) : launch(read_kernel<float, false>);
    if (dtype == RI_BF16) return vec ? launch(read_kernel<__nv_bfloat16, true>) : launch(read_kernel<__nv_bfloat16, false>);
    return fail("quantized_read: unknown dtype %d", dtype);
}

RI_DEFINE_LAST_ERROR()
