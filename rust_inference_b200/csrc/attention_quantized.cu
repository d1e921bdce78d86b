// Attention over a cache in 8 bits (quantized_cache.cu) for steps of few query rows: single tokens, drafted tokens, short
// continuations; head sizes 64 and 128.  It reads codes and scales as they lie in the cache, each once per 16 query rows.
//
// The mathematics.  With key codes c_j of scale s_j, value codes d_j of scale t_j, both the same for the 16 positions of a block:
//   score_j = scale s_j (q . c_j),  out = sum_j w_j t_j d_j / sum_j w_j,  w_j = 2^(score_j log2 e - m)
// over the keys 0..pos of the token's slot within its span (common.cuh: first_visible_key).  Codes are whole numbers up to 127, so
// as float16 numbers they are exact, and the products run on the tensor cores (m16n8k16, float32 sums) without a rounding of keys
// or values:
//   - a row of q is brought to [2^14, 2^15) by a power of two and cut into one float16 number per channel, for float32
//     queries into two (the second holds what the first left over).  A bfloat16 number has 8 significant bits, float16 has 11:
//     the first one is exact, down to 2^-28 of the row's largest number;
//   - a weight times 2^14 times t_j over the largest t so far of the warp is at most 2^14: as float16 it is rounded to
//     2^-12 relative (two numbers for float32: 2^-23), whatever its size down to 2^-28 of the largest.  The sums run
//     in units of that t; when a larger one comes, they are brought to it as they are to a new maximum.
//
// The work.  A unit is one page (64 keys) of one kv head for a tile of 16 rows (row = token * n_rep + head of the kv head).  The
// units of a step, sequence by sequence, are cut into equal runs, one per thread block: however unequal the sequences are, all
// blocks have the same to read.  A block's four warps take 16 keys of each page each, every warp with a ring of its own that
// cp.async fills (no barrier inside a run).  An item (sequence, kv head, tile) that lies in one block is finished there; one that
// spreads over several is written as partial sums, and the block that arrives last (a counter per item) adds them up in the
// order of the blocks, so that the result does not depend on who was last.
//
// Fragments come straight from 16-byte reads of shared memory, because the order of a contraction's terms is free: lane (g, t) of
// a product holds of key g the channels t HD/4 .. + HD/4, of its four keys (2t, 2t + 1, 2t + 8, 2t + 9) the channels g HD/8 ..
// + HD/8, and of the result's row g the channels t HD/4 .. + HD/4 again.
#include "common.cuh"

#include <cuda_fp16.h>

using namespace ri;

namespace {

constexpr int PAGE = 64, BLOCK = 16, WARPS = 4, THREADS = 32 * WARPS, ROWS = 16, STAGES = 4;
constexpr float BIAS = 14.f;                     // weights are formed times 2^14

struct Args {
    const void* q;
    int q_ld, q_vec;
    const int8_t *kc, *vc;
    const float *ks, *vs;
    const int *page_table, *seq_slot, *seq_start, *cu_seqlens;
    int max_pages, n_seqs;
    void* out;
    int out_ld, out_vec;
    int n_rep, n_kv;
    float scale;
    int span;
    float out_scale;
    float* part;                                 // [2 * blocks][rows_cap][HD]
    float4* stat;                                // [2 * blocks][rows_cap]: maximum, sum, unit of the sums
    int* arrived;                                // per item, zero between calls
    int rows_cap;                                // rows of a tile that any item fills
};

// Where an item lies
struct Item {
    int seq, head, tile;                         // kv head, tile of rows
    int low, end;                                // its pages
    int first_tok, start, n_rows, tiles;
};

__device__ __forceinline__ int pages_of(const Args& a, int start, int n_tok, int& low) {
    low = first_visible_key(start, a.span) / PAGE;
    return n_tok > 0 ? (start + n_tok - 1) / PAGE + 1 - low : 0;
}
__device__ __forceinline__ int units_of(const Args& a, int seq) {
    const int n = a.cu_seqlens[seq + 1] - a.cu_seqlens[seq];
    int low;
    return pages_of(a, a.seq_start[seq], n, low) * a.n_kv * ((n * a.n_rep + ROWS - 1) / ROWS);
}
__device__ __forceinline__ void enter(const Args& a, int seq, Item& it) {
    it.seq = seq;
    it.first_tok = a.cu_seqlens[seq];
    const int n = a.cu_seqlens[seq + 1] - it.first_tok;
    it.start = a.seq_start[seq];
    it.n_rows = n * a.n_rep;
    it.tiles = (it.n_rows + ROWS - 1) / ROWS;
    it.end = pages_of(a, it.start, n, it.low) + it.low;
}
// the item after this one (there is one)
__device__ __forceinline__ void next_item(const Args& a, Item& it) {
    if (++it.tile < it.tiles) return;
    it.tile = 0;
    if (++it.head < a.n_kv) return;
    it.head = 0;
    do enter(a, it.seq + 1, it); while (it.n_rows == 0);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Sixteen-byte pieces lie in lines of 128 bytes; piece p of line l at p ^ swizzle(l), so that the reads below meet no bank twice.
template <int HD> __device__ __forceinline__ int swizzle(int line) { return HD == 128 ? line & 7 : (line & 3) << 1; }

// two codes (bytes `pick` of w, offset by 128) as float16 numbers: 1024 + code + 128 by its bits, less 1152
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t pick) {
    const uint32_t u = __byte_perm(w, 0x64646464u, pick);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T> __device__ __forceinline__ void load4(const T* p, bool vec, float* f);
template <> __device__ __forceinline__ void load4<float>(const float* p, bool vec, float* f) {
    if (vec) {
        *reinterpret_cast<float4*>(f) = load_written(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const volatile float*>(p + i);
    }
}
template <> __device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, bool vec, float* f) {
    uint2 v;
    if (vec) {
        asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
    } else {
        const volatile uint16_t* h = reinterpret_cast<const volatile uint16_t*>(p);
        v.x = h[0] | ((uint32_t)h[1] << 16);
        v.y = h[2] | ((uint32_t)h[3] << 16);
    }
    f[0] = __uint_as_float(v.x << 16);
    f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16);
    f[3] = __uint_as_float(v.y & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void store4(T* p, bool vec, const float4& v);
template <> __device__ __forceinline__ void store4<float>(float* p, bool vec, const float4& v) {
    if (vec) *reinterpret_cast<float4*>(p) = v;
    else p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
}
template <> __device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, bool vec, const float4& v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    if (vec) {
        uint2 u;
        u.x = *reinterpret_cast<const uint32_t*>(&a);
        u.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(p) = u;
    } else {
        p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
    }
}

// What several partial results of a row are weighted with: maxima m, sums l, units s of their values
__device__ __forceinline__ float merge_weight(float m, float top) { return exp2f(m - (top == -INFINITY ? 0.f : top)); }
__device__ __forceinline__ float unit_ratio(float s, float most) { return s == most ? 1.f : s / most; }      // (both 0: 1; s NaN never is the unit)

template <int HD> constexpr int RING_BYTES = WARPS * STAGES * (2 * BLOCK * HD + 16);
template <int HD> int smem_bytes(int rows_cap) { return RING_BYTES<HD> + WARPS * rows_cap * (HD + 4) * 4 + WARPS * ROWS * 16; }

template <int HD, typename T, int TERMS>
__global__ void __launch_bounds__(THREADS)
attn_quantized_kernel(const Args a) {
    constexpr int KS = HD / 16;                  // steps of a score's contraction
    constexpr int NT = HD / 8;                   // column tiles of the result
    constexpr int TILE = BLOCK * HD;             // bytes of 16 keys
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int sums[THREADS + 1];
    __shared__ int found[2];
    __shared__ int last_here;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    let_next_kernel_start();

    // ---- this block's run of units ----
    const int per = (a.n_seqs + THREADS - 1) / THREADS;
    int mine = 0;
    for (int s = tid * per; s < min((tid + 1) * per, a.n_seqs); ++s) mine += units_of(a, s);
    sums[tid + 1] = mine;
    if (tid == 0) sums[0] = 0;
    __syncthreads();
    if (warp == 0) {                             // running sums of the 128 numbers, four per lane
        int v[4], run = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = run += sums[4 * lane + 1 + i];
        int before = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += w;
        }
        before -= run;
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[4 * lane + 1 + i] = v[i] + before;
    }
    __syncthreads();
    const long long total = sums[THREADS];
    const int blocks = (int)min((long long)gridDim.x, total), me = blockIdx.x;
    if (me >= blocks) {
        wait_for_previous_kernels();             // (who waits for this kernel waits for those before it too)
        return;
    }
    const int u0 = (int)(total * me / blocks), u1 = (int)(total * (me + 1) / blocks);
    if (sums[tid] <= u0 && u0 < sums[tid + 1]) {
        int at = sums[tid], s = tid * per;
        for (int n; at + (n = units_of(a, s)) <= u0; ++s) at += n;
        found[0] = s;
        found[1] = at;
    }
    __syncthreads();
    Item it;
    enter(a, found[0], it);
    int page;
    {
        const int within = u0 - found[1], n = it.end - it.low;
        page = it.low + within % n;
        it.tile = within / n % it.tiles;
        it.head = within / n / it.tiles;
    }
    wait_for_previous_kernels();

    // ---- the ring ----
    unsigned char* ring = smem + warp * STAGES * (2 * TILE + 16);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    Item ahead = it;
    int ahead_page = page, ahead_u = u0, ahead_slot = 0;
    auto number_of = [&](const Item& i, int p) {
        const int slot = a.seq_slot[i.seq];
        // checked build: a slot or a page index outside is recorded, page 0 read in its place
        if (!RI_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT) || !RI_IN_RANGE(p, a.max_pages, RI_CHECK_PAGE_INDEX)) return 0;
        return a.page_table[(size_t)slot * a.max_pages + p];
    };
    int ahead_number = number_of(ahead, ahead_page);
    auto fetch = [&]() {
        if (ahead_u < u1) {
            const int base = ahead_page * PAGE + warp * BLOCK;
            // 16 keys that no row of the sequence sees are left out
            if (base <= ahead.start + (ahead.n_rows - 1) / a.n_rep && base + BLOCK > first_visible_key(ahead.start, a.span)) {
                int number = ahead_number;
                if (!RI_IN_LIMIT(number, RI_LIMIT_PAGES, RI_CHECK_PAGE)) number = 0;    // checked build: recorded, read from a page that exists
                const size_t tile = (size_t)number * a.n_kv + ahead.head;
                const int8_t* k = a.kc + (tile * PAGE + warp * BLOCK) * HD;
                const int8_t* v = a.vc + (tile * PAGE + warp * BLOCK) * HD;
                const uint32_t to = ring_at + ahead_slot * (2 * TILE + 16);
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    const int piece = i * 32 + lane, line = piece >> 3;
                    const uint32_t at = to + (line * 8 + ((piece & 7) ^ swizzle<HD>(line))) * 16;
                    copy16(at, k + piece * 16);
                    copy16(at + TILE, v + piece * 16);
                }
                if (lane < 2) copy4(to + 2 * TILE + 4 * lane, (lane ? a.vs : a.ks) + tile * (PAGE / BLOCK) + warp);
            }
            if (++ahead_u < u1) {
                if (++ahead_page == ahead.end) {
                    next_item(a, ahead);
                    ahead_page = ahead.low;
                }
                ahead_number = number_of(ahead, ahead_page);
            }
            ahead_slot = ahead_slot + 1 == STAGES ? 0 : ahead_slot + 1;
        }
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch();

    float* so = reinterpret_cast<float*>(smem + RING_BYTES<HD>);                       // [WARPS][rows_cap][HD + 4]
    float4* sml = reinterpret_cast<float4*>(so + WARPS * a.rows_cap * (HD + 4));       // [WARPS][ROWS]
    int slot = 0;
    for (int u = u0; u < u1;) {
        // ---- an item's part in this block: pages page .. stop - 1 ----
        const int stop = min(it.end, page + (u1 - u));
        const int row0 = it.tile * ROWS, here = min(ROWS, it.n_rows - row0);
        const bool whole = page == it.low && stop == it.end;
        const int item_u0 = u - (page - it.low), item_n = it.end - it.low;

        // queries: rows g and g + 8 of the tile, as float16 numbers
        uint32_t qa[TERMS][KS][4];
        float unit[2];                           // what a score's sum is multiplied by (without the keys' scale)
        int pos[2], low[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + g + 8 * r;
            const bool there = row < it.n_rows;
            pos[r] = there ? it.start + row / a.n_rep : -1;
            low[r] = there ? first_visible_key(pos[r], a.span) : 0;
            float x[KS][4], top = 0.f;
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(it.first_tok + (there ? row / a.n_rep : 0)) * a.q_ld +
                           (size_t)(it.head * a.n_rep + (there ? row % a.n_rep : 0)) * HD + t * (HD / 4);
#pragma unroll
            for (int i = 0; i < KS; ++i) load4<T>(src + 4 * i, a.q_vec, x[i]);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) top = fmaxf(top, fabsf(x[i][c]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the power of two that brings the largest number to [2^14, 2^15); numbers below 2^-112 are brought less far
            const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);
            const float up = __uint_as_float((uint32_t)(127 + 14 - min(e, 127)) << 23), down = __uint_as_float((uint32_t)max(127 - 14 + e, 1) << 23);
            unit[r] = down * (a.scale * 1.4426950408889634f);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float y0 = x[i][2 * h] * up, y1 = x[i][2 * h + 1] * up;
                    const uint32_t first = pack(y0, y1);
                    qa[0][i][2 * h + r] = first;
                    if (TERMS == 2) {
                        const float2 f = unpack(first);
                        qa[TERMS - 1][i][2 * h + r] = pack(y0 - f.x, y1 - f.y);
                    }
                }
        }

        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, most = 0.f, inverse = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        const int last_pos = it.start + (row0 + here - 1) / a.n_rep;
        const int first_pos = it.start + row0 / a.n_rep, first_key = first_visible_key(first_pos, a.span);
        const int last_low = first_visible_key(last_pos, a.span);

        for (; page < stop; ++page, ++u) {
            __syncwarp();                        // every lane has read what the next copies overwrite
            fetch();
            copies_wait<STAGES - 1>();
            __syncwarp();
            const unsigned char* kt = ring + slot * (2 * TILE + 16);
            const unsigned char* vt = kt + TILE;
            const float* scales = reinterpret_cast<const float*>(kt + 2 * TILE);
            slot = slot + 1 == STAGES ? 0 : slot + 1;
            const int base = page * PAGE + warp * BLOCK;
            if (base > last_pos || base + BLOCK <= first_key) continue;

            // scores of 16 rows and 16 keys
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
                uint32_t w[KS];
                const int key = 8 * j + g;
#pragma unroll
                for (int i = 0; i < KS / 4; ++i) {
                    const int line = HD == 128 ? key : key >> 1, piece = HD == 128 ? 2 * t + i : (key & 1) * 4 + t;
                    *reinterpret_cast<uint4*>(w + 4 * i) = *reinterpret_cast<const uint4*>(kt + (line * 8 + (piece ^ swizzle<HD>(line))) * 16);
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const uint32_t c = w[i] ^ 0x80808080u;
                    const uint32_t b0 = halves(c, 0x4140), b1 = halves(c, 0x4342);
#pragma unroll
                    for (int x = 0; x < TERMS; ++x) mma(s[j], qa[x][i], b0, b1);
                }
            }
            const float k_scale = scales[0], v_scale = scales[1];
            const bool edge = base + BLOCK - 1 > first_pos || base < last_low || here < ROWS;
            float alpha[2];
            bool moved = false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = k_scale * unit[r];
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int key = base + 8 * j + 2 * t + c;
                        float& v = s[j][2 * r + c];
                        v *= f;
                        if (edge && !(key <= pos[r] && key >= low[r])) v = -INFINITY;
                        top = fmaxf(top, v);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m[r], top), ref = m_new == -INFINITY ? 0.f : m_new;
                alpha[r] = exp2f(m[r] - ref);
                moved |= m_new != m[r];
                m[r] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& v = s[j][2 * r + c];
                        v = exp2f(v - (ref - BIAS));
                        sum += v;
                    }
                l[r] = l[r] * alpha[r] + sum;
            }
            if (v_scale > most) {                // a larger unit for the sums (of this warp: all lanes alike)
                const float f = most * (1.f / v_scale);
                alpha[0] *= f;
                alpha[1] *= f;
                moved = true;
                most = v_scale;
                inverse = 1.f / v_scale;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][0] *= alpha[0];
                    o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1];
                    o[i][3] *= alpha[1];
                }
            }
            // weights in units of `most`, as one or two float16 numbers
            const float ratio = v_scale == most ? 1.f : v_scale * inverse;
            uint32_t pa[TERMS][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float y0 = s[j][2 * r] * ratio, y1 = s[j][2 * r + 1] * ratio;
                    if (edge) {                  // an unseen key's weight is 0 also beside a scale that is no number
                        const int key = base + 8 * j + 2 * t;
                        if (!(key <= pos[r] && key >= low[r])) y0 = 0.f;
                        if (!(key + 1 <= pos[r] && key + 1 >= low[r])) y1 = 0.f;
                    }
                    const uint32_t first = pack(y0, y1);
                    pa[0][2 * j + r] = first;
                    if (TERMS == 2) {
                        const float2 f = unpack(first);
                        pa[TERMS - 1][2 * j + r] = pack(y0 - f.x, y1 - f.y);
                    }
                }
            // values: four keys of this lane, four channels at a time
            uint32_t w[4][HD / 32];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int key = 2 * t + (k & 1) + (k >> 1) * 8;
                if (HD == 128) {
                    *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(vt + (key * 8 + (g ^ swizzle<HD>(key))) * 16);
                } else {
                    const int line = key >> 1, piece = (key & 1) * 4 + (g >> 1);
                    *reinterpret_cast<uint2*>(w[k]) =
                        *reinterpret_cast<const uint2*>(vt + (line * 8 + (piece ^ swizzle<HD>(line))) * 16 + (g & 1) * 8);
                }
            }
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t pick = h ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(w[0][i], w[1][i], pick) ^ 0x80808080u, y = __byte_perm(w[2][i], w[3][i], pick) ^ 0x80808080u;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t b0 = halves(x, c ? 0x4342 : 0x4140), b1 = halves(y, c ? 0x4342 : 0x4140);
#pragma unroll
                        for (int n = 0; n < TERMS; ++n) mma(o[4 * i + 2 * h + c], pa[n], b0, b1);
                    }
                }
            }
        }

        // ---- the four warps' parts together ----
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int row = g + 8 * r;
            if (t == 0) sml[warp * ROWS + row] = make_float4(m[r], l[r], most, 0.f);
            if (row < here) {
                // columns 2t and 2t + 1 of the tiles are the channels (2t) HD/8 + i and (2t + 1) HD/8 + i
                float* to = so + (warp * a.rows_cap + row) * (HD + 4) + t * (HD / 4);
#pragma unroll
                for (int i = 0; i < NT; i += 4) {
                    *reinterpret_cast<float4*>(to + i) = make_float4(o[i][2 * r], o[i + 1][2 * r], o[i + 2][2 * r], o[i + 3][2 * r]);
                    *reinterpret_cast<float4*>(to + NT + i) =
                        make_float4(o[i][2 * r + 1], o[i + 1][2 * r + 1], o[i + 2][2 * r + 1], o[i + 3][2 * r + 1]);
                }
            }
        }
        __syncthreads();
        auto write = [&](int row, int d, float4 v, float sum, float s) {
            const float inv = 1.f / sum, f = s * a.out_scale;
            v = make_float4(v.x * inv * f, v.y * inv * f, v.z * inv * f, v.w * inv * f);
            row += row0;
            store4<T>(reinterpret_cast<T*>(a.out) + (size_t)(it.first_tok + row / a.n_rep) * a.out_ld +
                      (size_t)(it.head * a.n_rep + row % a.n_rep) * HD + d, a.out_vec, v);
        };
        const int first_block = (int)(((item_u0 + 1ll) * blocks - 1) / total), last_block = (int)(((long long)(item_u0 + item_n) * blocks - 1) / total);
        auto part_of = [&](int b) { return (size_t)(2 * b + (b == first_block && (int)(total * b / blocks) < item_u0 ? 1 : 0)) * a.rows_cap; };
        for (int i = tid; i < here * (HD / 4); i += THREADS) {
            const int row = i / (HD / 4), d = i % (HD / 4) * 4;
            float top = -INFINITY, s = 0.f, sum = 0.f;
            float4 st[WARPS], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                st[w] = sml[w * ROWS + row];
                top = fmaxf(top, st[w].x);
                s = fmaxf(s, st[w].z);
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = merge_weight(st[w].x, top), x = f * unit_ratio(st[w].z, s);
                const float4 p = *reinterpret_cast<const float4*>(so + (w * a.rows_cap + row) * (HD + 4) + d);
                sum = fmaf(st[w].y, f, sum);
                v = make_float4(fmaf(p.x, x, v.x), fmaf(p.y, x, v.y), fmaf(p.z, x, v.z), fmaf(p.w, x, v.w));
            }
            if (whole) {
                write(row, d, v, sum, s);
            } else {
                const size_t at = part_of(me) + row;
                *reinterpret_cast<float4*>(a.part + at * HD + d) = v;
                if (d == 0) a.stat[at] = make_float4(top, sum, s, 0.f);
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            int* arrived = a.arrived + ((size_t)it.first_tok * a.n_rep + it.tile) * a.n_kv + it.head;
            if (tid == 0) last_here = atomicAdd(arrived, 1) == last_block - first_block;
            __syncthreads();
            if (last_here) {
                __threadfence();
                if (tid == 0) *arrived = 0;
                for (int i = tid; i < here * (HD / 4); i += THREADS) {
                    const int row = i / (HD / 4), d = i % (HD / 4) * 4;
                    float top = -INFINITY, s = 0.f, sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int b = first_block; b <= last_block; ++b) {
                        const float4 st = __ldcg(a.stat + part_of(b) + row);
                        top = fmaxf(top, st.x);
                        s = fmaxf(s, st.z);
                    }
                    for (int b = first_block; b <= last_block; ++b) {
                        const size_t at = part_of(b) + row;
                        const float4 st = __ldcg(a.stat + at), p = __ldcg(reinterpret_cast<const float4*>(a.part + at * HD + d));
                        const float f = merge_weight(st.x, top), x = f * unit_ratio(st.z, s);
                        sum = fmaf(st.y, f, sum);
                        v = make_float4(fmaf(p.x, x, v.x), fmaf(p.y, x, v.y), fmaf(p.z, x, v.z), fmaf(p.w, x, v.w));
                    }
                    write(row, d, v, sum, s);
                }
            }
        }
        __syncthreads();                         // the warps' parts have been read
        if (u < u1) {
            next_item(a, it);
            page = it.low;
        }
    }
    copies_wait<0>();
}

int rows_cap(int n_rep, int max_new) { return n_rep * max_new < ROWS ? n_rep * max_new : ROWS; }

template <int HD, typename T, int TERMS>
int launch(const Args& a, int blocks, cudaStream_t stream) {
    static PerDeviceOnce once;
    auto kernel = attn_quantized_kernel<HD, T, TERMS>;
    if (raise_dynamic_smem(kernel, smem_bytes<HD>(ROWS), once, "attention_quantized")) return 1;
    return check_launch(launch_dependent(kernel, dim3((unsigned)blocks), dim3(THREADS), (size_t)smem_bytes<HD>(a.rows_cap), stream, a),
                        "attention_quantized");
}

}  // namespace

// Thread blocks of a step: two per SM
RI_API int ri_attention_quantized_blocks() { return 2 * sm_count(); }

// part: float32 [2 * blocks * min(16, n_rep * max_new) * (hd + 4)]; arrived: int32 [tokens * heads], zero, and left so.
RI_API int ri_attention_quantized(const void* q, int dtype, int q_ld, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs,
                                  const int* page_table, int max_pages, const int* seq_slot, const int* seq_start, const int* cu_seqlens,
                                  void* out, int out_ld, int n_seqs, int max_new, int n_heads, int n_kv, int hd, float scale, int span,
                                  float out_scale, float* part, int* arrived, int blocks, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return 0;
    if (hd != 64 && hd != 128) return fail("attention_quantized: heads of %d channels (64 or 128 wanted)", hd);
    if (n_kv <= 0 || n_heads % n_kv) return fail("attention_quantized: %d heads over %d kv heads", n_heads, n_kv);
    if ((uintptr_t)kc % 16 || (uintptr_t)vc % 16 || (uintptr_t)part % 16) return fail("attention_quantized: codes and scratch must lie on 16-byte boundaries");
    const long long rows = (long long)max_new * (n_heads / n_kv);
    if ((long long)n_seqs * max_pages * n_kv * ((rows + ROWS - 1) / ROWS) > 0x7fffffff || rows > 0x7fffffff)
        return fail("attention_quantized: %d sequences of %d new tokens are too many", n_seqs, max_new);
    Args a = {};
    const int item = dtype == RI_F32 ? 4 : 2;
    a.q = q;
    a.q_ld = q_ld;
    a.q_vec = (uintptr_t)q % (4 * item) == 0 && q_ld % 4 == 0;
    a.kc = kc, a.vc = vc, a.ks = ks, a.vs = vs;
    a.page_table = page_table, a.seq_slot = seq_slot, a.seq_start = seq_start, a.cu_seqlens = cu_seqlens;
    a.max_pages = max_pages;
    a.n_seqs = n_seqs;
    a.out = out;
    a.out_ld = out_ld;
    a.out_vec = (uintptr_t)out % (4 * item) == 0 && out_ld % 4 == 0;
    a.n_rep = n_heads / n_kv;
    a.n_kv = n_kv;
    a.scale = scale;
    a.span = span;
    a.out_scale = out_scale;
    a.rows_cap = rows_cap(a.n_rep, max_new);
    a.stat = reinterpret_cast<float4*>(part);
    a.part = part + (size_t)2 * blocks * a.rows_cap * 4;
    a.arrived = arrived;
    if (dtype == RI_F32) return hd == 64 ? launch<64, float, 2>(a, blocks, stream) : launch<128, float, 2>(a, blocks, stream);
    if (dtype == RI_BF16) return hd == 64 ? launch<64, __nv_bfloat16, 1>(a, blocks, stream) : launch<128, __nv_bfloat16, 1>(a, blocks, stream);
    return fail("attention_quantized: unknown dtype %d", dtype);
}

RI_DEFINE_LAST_ERROR()
