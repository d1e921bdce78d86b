// Attention over a cache in 8 bits (quantized_cache.cu) for steps of few query rows: single tokens, drafted tokens, short
// continuations; head sizes 64 and 128.  It reads codes and scales as they lie in the cache, each once per tile of query rows.
//
// The mathematics.  With key codes c_j of scale s_j, value codes d_j of scale t_j, both the same for the 16 positions of a block:
//   score_j = scale s_j (q . c_j),  out = sum_j w_j t_j d_j / sum_j w_j,  w_j = 2^(score_j log2 e - m)
// over the keys 0..pos of the token's slot within its span (common.cuh: first_visible_key).  Codes enter the tensor cores' products
// exactly, so that keys and values are rounded nowhere:
//   - scores are sums of whole numbers (m16n8k32, int8): a row of q is brought to +-127 256 and rounded to whole numbers of
//     two signed bytes, q = 256 d1 + d0 (float32: +-127 65536, three bytes), 2^-16 (2^-24) of the row's largest
//     number; codes times bytes add up in 32 bits without a rounding.  The codes are operands as they lie in memory;
//   - results are sums of weights in float16 (m16n8k16, float32 sums; for float32 two float16 numbers each, the second what
//     the first left over) times codes.  A row has two references, both whole numbers so that bringing sums to a new one is
//     exact: m, which its scores are measured from and the sum of its weights runs in, and r, the same for score_j log2 e + log2 t_j,
//     which the products of weights and codes run in (out = 2^(r - m) times their quotient).  So w_j t_j is rounded to 2^-11 (2^-22)
//     relative, and no finer than 2^-30 of the row's own largest such product, whatever the values of
//     keys that the row does not see, or gives no weight to.  A code c becomes float16 by its bits: 1024 + 128 + c has the byte c + 128 as its low one.
//     With one number per weight the products are taken of 1152 + c, one byte permutation for two codes, and a product of the same
//     weights with -1152 follows each of them (float32 sums of that size are off by 2^-23 1152 = 1.4e-4 of a code); with two numbers
//     1152 is taken off the codes.
//
// The products are taken with codes as the rows of the MMA, 16 keys (scores) or 16 channels (result), and the query rows as its
// columns, 8 at a time: a code is made a float16 number once for all rows, and the usual 4 to 8 query heads of a kv head fill the
// columns, where they left half of 16 rows empty.
//
// The work.  A unit is one page (64 keys) of one kv head for a tile of 8 or 16 rows (row = token * n_rep + head of the kv head).
// The units of a step, sequence by sequence, are cut into equal runs, one per thread block: however unequal the sequences are,
// all blocks have the same to read (where that is not worth its joins, an item goes to a block whole).  A block's four warps take half of one of two pages each at a time, every warp with a ring of its
// own that cp.async fills (no barrier inside a run).  An item (sequence, kv head, tile) that lies in one block is finished there;
// one that spreads over several is written as partial sums, which the blocks that arrive last (a counter per eight parts) add up
// in the order of the blocks, so that the result does not depend on who was last.  Where few items are short, each gets a cluster of
// blocks instead, which add their parts up through distributed shared memory, a third of what meeting in memory takes.
//
// What it measures (32 heads over 8 of 128, bfloat16): 64 sequences of 128 to 2,048 keys 34.8 us, 4.3 TB/s of codes, 65% of what a copy
// reaches; with the loads alone 31, without the joining of parts too 27.  2 sequences of about 30,000 keys (28 heads over 4) 22.7 us, of
// which 14 for the loads and 8 for the two rounds of joining.  1 sequence of 1,024 keys 5.7 us, 3 of them until the first keys are there.  A
// scheduler issues in 46% of its cycles and the tensor cores are busy in 19%: what bounds the large steps is how many loads are in flight
// beside four blocks' arithmetic per SM (a second buffer for keys and values 38.0 us instead of 36.4, as blocks are then fewer; one for keys
// alone would leave four, and is not measured).
//
// Fragments come straight from 16-byte reads of shared memory, because the order of a contraction's terms, and which channel is which
// row of a product, are free: lane (g, t) holds of the keys g and g + 8 the channels t HD/4 .. + HD/4, of its four keys (2t,
// 2t + 1, 2t + 8, 2t + 9) the channels g HD/8 .. + HD/8, and of the result's rows 2t and 2t + 1 those channels again.
#include "cluster.cuh"

#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>

using namespace ri;

namespace {

constexpr int PAGE = 64, BLOCK = 16, WARPS = 4, THREADS = 32 * WARPS;
constexpr int STEP = 2 * BLOCK;                  // keys that a warp takes at a time
constexpr int MOST_BLOCKS = 5;                   // thread blocks per SM, at most
// What an item costs a block beside its pages (queries fetched, warps joined, the result written), in pages
// (64 sequences of 128 to 2,048 keys, 32 heads over 8: 4 35.8 us, 8 35.3, 12 36.9; 1 of 30,000: 4 23.5, 8 22.7)
constexpr int SETUP = 8;
// Items go to blocks whole where there are no more of them than blocks and the longest has so many pages more at most than each block would
// have of equal runs: what joining costs.  Equal runs and whole items, us, 64 sequences, 32 heads over 8: 250 keys 17.8 and 11.6, 1,024 33.4
// and 29.6; 28 over 4: 500 keys (8 pages for 3.5) 17.9 and 14.5, 700 (11 for 4.8) 19.6 and 18.0, 1,024 (16 for 6.9) 22.6 and 22.9.
constexpr int JOINING = 8;
// What a block has at least: the two pages of one turn, or as many turns as keep an item's parts to eight (64), which are added up in
// one go (two): up to 4 pages (8).
__device__ __forceinline__ int least_pages(int pages, int items) { return pages <= 16 * items ? 2 : (pages <= 256 * items ? 4 : 8); }
// Parts of an item are added up eight at a time: a block that arrives last of eight adds theirs and goes on with seven others
constexpr int GROUP = 8;
// Weights are formed times 2^6 against a reference that follows the row's maximum only when that is 2^8 times ahead: they stay below
// 2^14, which float16 holds, and sums are brought to a new reference a few times per row instead of at most steps.  Weights times their
// values' scales likewise.
constexpr float BIAS = 6.f, AHEAD = 8.f;
constexpr float LOWEST = -1.7e38f;               // the references of a row without keys
// ... of products whose values are all zeros, or below 2^-120: so far below the weights' reference (results of such a size are rounded to 2^-149)
constexpr float BELOW = 126.f;

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
    float4* stat;                                // [2 * blocks][rows_cap]: the weights' reference, their sum, the products' reference
    int* arrived;                                // [4][2 * blocks] (8^4 parts are more than there are blocks), zero between calls
    int places;                                  // 2 * blocks
    int cluster;                                 // blocks of a cluster, one for every item; 1: runs of units
    int rows_cap;                                // rows of a tile that any item fills
};

// Where an item lies
struct Item {
    int seq, head, tile;                         // kv head, tile of rows
    int low, end;                                // its pages
    int first_tok, start, n_rows, tiles;
    int first_key, last_pos;                     // the keys that any row of the sequence sees
    const int* table;                            // its pages' numbers
};

__device__ __forceinline__ int pages_of(const Args& a, int start, int n) {       // (of a sequence with new tokens)
    return (start + n - 1) / PAGE + 1 - first_visible_key(start, a.span) / PAGE;
}
__device__ __forceinline__ void enter(const Args& a, int seq, int first_tok, int n, int start, int slot, int rows, Item& it) {
    it.seq = seq;
    it.first_tok = first_tok;
    it.start = start;
    it.n_rows = n * a.n_rep;
    it.tiles = (it.n_rows + rows - 1) / rows;
    it.first_key = first_visible_key(start, a.span);
    it.last_pos = start + n - 1;
    it.low = it.first_key / PAGE;
    it.end = n > 0 ? it.last_pos / PAGE + 1 : it.low;
    // checked build: a slot outside is recorded, slot 0 read in its place
    if (!RI_IN_LIMIT(slot, RI_LIMIT_SLOTS, RI_CHECK_SLOT)) slot = 0;
    it.table = a.page_table + (size_t)slot * a.max_pages;
}
// the item after this one (there is one)
__device__ __forceinline__ void next_item(const Args& a, int rows, Item& it) {
    if (++it.tile < it.tiles) return;
    it.tile = 0;
    if (++it.head < a.n_kv) return;
    it.head = 0;
    do {
        const int seq = it.seq + 1, first_tok = a.cu_seqlens[seq];
        enter(a, seq, first_tok, a.cu_seqlens[seq + 1] - first_tok, a.seq_start[seq], a.seq_slot[seq], rows, it);
    } while (it.n_rows == 0);
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

// Two codes (bytes `pick` of w, offset by 128) as float16 numbers: 1024 + 128 + code by its bits, and the code itself
__device__ __forceinline__ uint32_t offset_halves(uint32_t w, uint32_t pick) { return __byte_perm(w, 0x64646464u, pick); }
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t pick) {
    const uint32_t u = offset_halves(w, pick);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// an 8 x 8 matrix of 16-bit numbers, two neighbours of a row per lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t w;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w) : "r"(v));
    return w;
}
// 2^x by the hardware's instruction: 2 units in the last place
__device__ __forceinline__ float two_to(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ... of whole numbers up to 127, exactly (what it leaves of a sum that far below another is nothing)
__device__ __forceinline__ float power(float x) { return x < -126.f ? 0.f : __int_as_float(((int)x + 127) << 23); }
__device__ __forceinline__ float log2_of(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the same of whole numbers, 32 terms
__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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

template <int HD> constexpr int OWN_BYTES = 2 * STEP * HD + 16;         // a warp's keys, values, two scales of each
// ... and what it sums up: in the place of its last values (8 rows), or beside them
template <int HD, int NQ> constexpr int PART_BYTES = NQ == 1 ? 0 : 8 * NQ * HD * 4;
template <int HD, int NQ> constexpr int SMEM_BYTES = WARPS * (OWN_BYTES<HD> + PART_BYTES<HD, NQ> + 8 * NQ * 16);

// NQ: tiles of 8 query rows; TERMS: float16 numbers per weight, TERMS + 1 bytes per query channel
// own: every item has a cluster of blocks of its own; else equal runs of units
template <int HD, typename T, int TERMS, int NQ, bool own>
__global__ void __launch_bounds__(THREADS, TERMS * NQ == 1 ? 4 : 2)
attn_quantized_kernel(const Args a) {
    constexpr int ROWS = 8 * NQ;
    constexpr int KS = HD / 16;                  // four-channel pieces of a key per lane
    constexpr int DIGITS = TERMS + 1;
    constexpr int CT = HD / 16;                  // tiles of 16 channels of the result
    constexpr int TILE = BLOCK * HD;             // bytes of 16 keys
    constexpr int OWN = OWN_BYTES<HD>, PART = PART_BYTES<HD, NQ>;
    static_assert(PART > 0 || ROWS * HD * 4 <= 2 * TILE, "a warp's sums fit where its values were");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int sums[THREADS + 1];
    __shared__ int found[6], totals[WARPS][3];
    __shared__ int last_here;
    __shared__ float4 sgroup[GROUP][ROWS];       // statistics of parts that are added up (a cluster's: each block's own first)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    let_next_kernel_start();

    // ---- this block's run of units (lengths, slots and pages are fixed before the step) ----
    const int per = (a.n_seqs + THREADS - 1) / THREADS;
    int mine = 0, mine_items = 0, longest = 0, slot = 0;
    for (int s = tid * per; s < min((tid + 1) * per, a.n_seqs); ++s) {
        const int n = a.cu_seqlens[s + 1] - a.cu_seqlens[s], start = a.seq_start[s];
        const int each = a.n_kv * ((n * a.n_rep + ROWS - 1) / ROWS), pages = n > 0 ? pages_of(a, start, n) : 0;
        if (n > 0) mine += (pages + SETUP) * each;
        mine_items += each;
        longest = max(longest, pages);
        slot = a.seq_slot[s];                    // (in the cache for when it is wanted)
    }
    const int me = blockIdx.x, C = a.cluster;
    if (tid == 0) sums[0] = 0;
    {
        const int units = __reduce_add_sync(0xffffffffu, mine), n = __reduce_add_sync(0xffffffffu, mine_items), most = __reduce_max_sync(0xffffffffu, longest);
        if (lane == 0) totals[warp][0] = units, totals[warp][1] = n, totals[warp][2] = most;
    }
    __syncthreads();
    int total = 0, items = 0;
    longest = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += totals[w][0], items += totals[w][1], longest = max(longest, totals[w][2]);
    const bool one = !own && items <= (int)gridDim.x && longest <= (total - SETUP * items) / (int)gridDim.x + JOINING;
    const int least = least_pages(total - SETUP * items, items), blocks = one ? items : min((int)gridDim.x, (total + least - 1) / least);
    sums[tid + 1] = own || one ? mine_items : mine;
    __syncthreads();
    // a cluster's item is cut into equal runs of whole turns
    auto run_of = [&](int pages) { return max(2, ((pages + C - 1) / C + 1) & ~1); };
    auto leave = [&]() {                         // (who waits for this kernel waits for those before it too)
        wait_for_previous_kernels();
        if (own) cluster_sync(), cluster_sync();
    };
    if (me >= (own ? items * C : blocks)) return leave();
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
    // the first `more` runs have one unit more than `each`
    const int each = total / max(blocks, 1), more = total % max(blocks, 1);
    auto run_start = [&](int b) { return b * each + min(b, more); };
    const int u0 = own ? me / C : (one ? me : run_start(me));
    if (sums[tid] <= u0 && u0 < sums[tid + 1]) {
        int at = sums[tid], s = tid * per, first_tok = a.cu_seqlens[s], n = a.cu_seqlens[s + 1] - first_tok, start = a.seq_start[s];
        auto many = [&]() { return n > 0 ? (own || one ? 1 : pages_of(a, start, n) + SETUP) * a.n_kv * ((n * a.n_rep + ROWS - 1) / ROWS) : 0; };
        for (int units; at + (units = many()) <= u0;) {
            at += units;
            ++s;
            first_tok += n;
            n = a.cu_seqlens[s + 1] - first_tok;
            start = a.seq_start[s];
        }
        found[0] = s, found[1] = at, found[2] = first_tok, found[3] = n, found[4] = start;
        found[5] = per == 1 ? slot : a.seq_slot[s];
    }
    __syncthreads();
    Item it;
    enter(a, found[0], found[2], found[3], found[4], found[5], ROWS, it);
    int page, u, u1;                             // the next page, and its place among the units (its number, with a cluster); the run's end
    {
        const int within = u0 - found[1], n = own || one ? 1 : it.end - it.low + SETUP, at = within % n;
        it.tile = within / n % it.tiles;
        it.head = within / n / it.tiles;
        if (own) {
            const int run = run_of(it.end - it.low);
            u = page = it.low + me % C * run;
            u1 = min(it.end, page + run);
        } else if (one) {
            u = page = it.low;
            u1 = it.end;
        } else {
            page = it.low + max(at - SETUP, 0);
            u = u0 + max(SETUP - at, 0);
            u1 = run_start(me + 1);
        }
    }
    if (u >= u1) return leave();

    // ---- half a page at a time: keys are on their way while values are worked on, values while scores are ----
    unsigned char* kt = smem + warp * OWN;
    unsigned char* vt = kt + 2 * TILE;
    const float* scales = reinterpret_cast<const float*>(kt + 4 * TILE);
    const uint32_t k_to = (uint32_t)__cvta_generic_to_shared(kt);
    // where this lane's pieces go (those of odd runs of 32: 4 pieces further on in the swizzle), and where it reads: keys g and
    // g + 8, pieces 2t and 2t + 1 (64 channels: piece t); keys 2t and 2t + 1 (and 8 on), piece g (64 channels: half of piece g / 2)
    const int put = ((lane >> 3) * 8 + ((lane & 7) ^ swizzle<HD>(lane >> 3))) * 16, put_odd = put ^ (HD == 128 ? 64 : 0);
    const int k_at = HD == 128 ? (g * 8 + ((2 * t) ^ g)) * 16 : ((g >> 1) * 8 + (((g & 1) * 4 + t) ^ swizzle<HD>(g >> 1))) * 16;
    const int v_at = HD == 128 ? (2 * t * 8 + (g ^ (2 * t))) * 16 : (t * 8 + ((g >> 1) ^ swizzle<HD>(t))) * 16 + (g & 1) * 8;
    const int v_at_1 = HD == 128 ? ((2 * t + 1) * 8 + (g ^ (2 * t + 1))) * 16 : (t * 8 + ((4 + (g >> 1)) ^ swizzle<HD>(t))) * 16 + (g & 1) * 8;
    const int my_page = warp >> 1, my_half = (warp & 1) * STEP;
    Item ahead = it;
    // (ahead_u: where the item's pages would begin, also if an earlier block has its first ones)
    int ahead_u = u - (page - it.low), ahead_page = page, ahead_stop = min(it.end, page + (u1 - u));
    auto number_of = [&](const Item& i, int p) {
        if (p >= i.end || !RI_IN_RANGE(p, a.max_pages, RI_CHECK_PAGE_INDEX)) return 0;     // checked build: recorded, page 0 read in its place
        return i.table[p];
    };
    int ahead_number = number_of(ahead, ahead_page + my_page);
    size_t v_tile = 0;                           // where the values lie that belong to the keys fetched last
    bool v_there = false;
    wait_for_previous_kernels();
    auto fetch_keys = [&]() {
        v_there = false;
        if (ahead_page < ahead_stop) {
            const int base = (ahead_page + my_page) * PAGE + my_half;
            // half a page that no row of the sequence sees is left out
            if (ahead_page + my_page < ahead_stop && base <= ahead.last_pos && base + STEP > ahead.first_key) {
                int number = ahead_number;
                if (!RI_IN_LIMIT(number, RI_LIMIT_PAGES, RI_CHECK_PAGE)) number = 0;
                v_there = true;
                v_tile = (size_t)number * a.n_kv + ahead.head;
                const int8_t* k = a.kc + (v_tile * PAGE + my_half) * HD + lane * 16;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) copy16(k_to + (i & 1 ? put_odd : put) + i * 512, k + i * 512);
                if (lane < 2) copy4(k_to + 4 * TILE + 4 * lane, a.ks + v_tile * (PAGE / BLOCK) + my_half / BLOCK + lane);
            }
            ahead_page += 2;
            if (!own && ahead_page >= ahead_stop && ahead_stop == ahead.end && (ahead_u += SETUP + ahead.end - ahead.low) < u1) {
                next_item(a, ROWS, ahead);
                ahead_page = ahead.low;
                ahead_stop = min(ahead.end, ahead.low + (u1 - ahead_u));
            }
            if (ahead_page < ahead_stop) ahead_number = number_of(ahead, ahead_page + my_page);
        }
        copies_commit();
    };
    auto fetch_values = [&]() {
        if (v_there) {
            const int8_t* v = a.vc + (v_tile * PAGE + my_half) * HD + lane * 16;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) copy16(k_to + 2 * TILE + (i & 1 ? put_odd : put) + i * 512, v + i * 512);
            if (lane < 2) copy4(k_to + 4 * TILE + 8 + 4 * lane, a.vs + v_tile * (PAGE / BLOCK) + my_half / BLOCK + lane);
        }
        copies_commit();
    };
    bool begun = false;                          // the first keys are sent for behind the first queries, which would wait for them otherwise

    // a warp's sums [WARPS][ROWS][HD] and their rows' statistics [WARPS][ROWS]
    auto part_at = [&](int w) { return reinterpret_cast<float*>(smem + (PART ? WARPS * OWN + w * PART : w * OWN + 2 * TILE)); };
    float4* sml = reinterpret_cast<float4*>(smem + WARPS * (OWN + PART));
    auto write = [&](const Item& i, int row, int d, float4 v, float sum, float m, float r) {
        const float inv = 1.f / sum, f = power(r - m) * a.out_scale;
        v = make_float4(v.x * inv * f, v.y * inv * f, v.z * inv * f, v.w * inv * f);
        store4<T>(reinterpret_cast<T*>(a.out) + (size_t)(i.first_tok + row / a.n_rep) * a.out_ld + (size_t)(i.head * a.n_rep + row % a.n_rep) * HD + d,
                  a.out_vec, v);
    };
    while (true) {
        // ---- an item's part in this block: pages page .. stop - 1 ----
        const int stop = min(it.end, page + (u1 - u));
        const int row0 = it.tile * ROWS, here = min(ROWS, it.n_rows - row0);
        const bool whole = page == it.low && stop == it.end;
        const int item_u = u - (page - it.low), item_n = it.end - it.low;        // the item's pages among the units

        // queries: bytes of row 8 n + g of the tile
        uint32_t qd[DIGITS][NQ][KS];
        // ... and of the rows 8 n + 2t + r, whose scores this lane has: what a sum of products is multiplied by (without the keys'
        // scale), position and first visible key
        float unit[NQ][2];
        int pos[NQ][2], low[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int row = row0 + 8 * n + g;
            const bool there = row < it.n_rows;
            const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(it.first_tok + (there ? row / a.n_rep : 0)) * a.q_ld +
                           (size_t)(it.head * a.n_rep + (there ? row % a.n_rep : 0)) * HD + t * (HD / 4);
            float x[KS][4], top = 0.f;
            bool fine = true;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                load4<T>(src + 4 * i, a.q_vec, x[i]);
                if (!there) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;       // its scores stay 0, its result is not written
            }
            if (n == 0 && !begun) fetch_keys(), begun = true;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top = fmaxf(top, fabsf(x[i][c]));
                    fine &= fabsf(x[i][c]) < INFINITY;
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            constexpr float MOST = TERMS == 1 ? 127.f * 256.f : 127.f * 65536.f;
            constexpr int HALF = TERMS == 1 ? 0x8080 : 0x808080;               // makes the bytes of a number its signed digits
            const float size = fmaxf(top, 7.9e-31f), up = MOST / size;         // (a row below 2^-100 is 0)
            // a row with an infinity or a NaN has no scores
            float down = size * (1.f / MOST) * (a.scale * 1.4426950408889634f);
            fine = (__ballot_sync(0xffffffffu, fine) >> (lane & 28) & 15u) == 15u;
            if (!fine) down = __int_as_float(0x7fffffff);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t d[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) d[c] = (uint32_t)(__float2int_rn(x[i][c] * up) + HALF) ^ HALF;
                const uint32_t lo01 = __byte_perm(d[0], d[1], 0x5140), lo23 = __byte_perm(d[2], d[3], 0x5140);
                qd[0][n][i] = __byte_perm(lo01, lo23, 0x5410);
                qd[1][n][i] = __byte_perm(lo01, lo23, 0x7632);
                if (DIGITS == 3) qd[DIGITS - 1][n][i] = __byte_perm(__byte_perm(d[0], d[1], 0x0062), __byte_perm(d[2], d[3], 0x0062), 0x5410);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int mine = row0 + 8 * n + 2 * t + r;
                unit[n][r] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + r));
                pos[n][r] = mine < it.n_rows ? it.start + mine / a.n_rep : -1;
                low[n][r] = mine < it.n_rows ? first_visible_key(pos[n][r], a.span) : 0;
            }
        }

        float o[NQ][CT][4], m[NQ][2], r[NQ][2], from_m[NQ][2], l[NQ][2];      // from_m: 2^(m - r)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n][0] = m[n][1] = r[n][0] = r[n][1] = LOWEST;
            from_m[n][0] = from_m[n][1] = 1.f;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < CT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        }
        const int last_pos = it.start + (row0 + here - 1) / a.n_rep;
        const int first_pos = it.start + row0 / a.n_rep, first_key = first_visible_key(first_pos, a.span);
        const int last_low = first_visible_key(last_pos, a.span);

        u += stop - page;
        for (; page < stop; page += 2) {
            __syncwarp();                        // every lane has read the values that the next ones overwrite
            fetch_values();
            copies_wait<1>();
            __syncwarp();                        // the keys are there
            const int base = (page + my_page) * PAGE + my_half;
            if (page + my_page >= stop || base > last_pos || base + STEP <= first_key) {
                fetch_keys();
                copies_wait<1>();                // values that nobody wants have landed before the next ones are sent for
                continue;
            }

            // scores of the keys g (s[..][0], [1]) and g + 8 ([2], [3]) of two blocks for the rows 2t and 2t + 1
            float s[2][NQ][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[2][KS];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < KS / 4; ++i)
                        *reinterpret_cast<uint4*>(w[h] + 4 * i) = *reinterpret_cast<const uint4*>(kt + (i ? k_at ^ 16 : k_at) + h * (TILE / 2) + j * TILE);
                const float k_scale = scales[j];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    int c[DIGITS][4];
#pragma unroll
                    for (int d = 0; d < DIGITS; ++d) c[d][0] = c[d][1] = c[d][2] = c[d][3] = 0;
#pragma unroll
                    for (int i = 0; i < KS; i += 2)
#pragma unroll
                        for (int d = 0; d < DIGITS; ++d) mma_s8(c[d], w[0][i], w[1][i], w[0][i + 1], w[1][i + 1], qd[d][n][i], qd[d][n][i + 1]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float v = (float)(c[1][x] * 256 + c[0][x]);
                        if (DIGITS == 3) v = fmaf((float)c[DIGITS - 1][x], 65536.f, v);
                        s[j][n][x] = v * (k_scale * unit[n][x & 1]);
                    }
                }
            }
            const bool edge = base + STEP - 1 > first_pos || base < last_low;
            __syncwarp();                        // every lane has read the keys
            fetch_keys();
            if (edge) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = base + 16 * j + 8 * (x >> 1) + g;
                            if (!(key <= pos[n][x & 1] && key >= low[n][x & 1])) s[j][n][x] = -INFINITY;
                        }
            }
            copies_wait<1>();
            __syncwarp();                        // the values are there
            // (a block that no row sees has no say)
            const float v0 = edge && !(base <= last_pos && base + BLOCK > first_key) ? 0.f : scales[2];
            const float v1 = edge && !(base + BLOCK <= last_pos && base + STEP > first_key) ? 0.f : scales[3];
            const float log_v0 = log2_of(v0), log_v1 = log2_of(v1);          // a scale that is no number moves no reference
            uint32_t pb[2][TERMS][NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                // whether the rows' references are far behind
                float top[2], product[2];
                bool behind = false;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float top0 = fmaxf(s[0][n][x], s[0][n][2 + x]), top1 = fmaxf(s[1][n][x], s[1][n][2 + x]);
                    top[x] = fmaxf(top0, top1);
                    product[x] = fmaxf(top0 + log_v0, top1 + log_v1);
                    behind |= top[x] > m[n][x] + AHEAD || product[x] > r[n][x] + AHEAD;
                }
                if (__any_sync(0xffffffffu, behind)) {
                    float alpha[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int lanes = 4; lanes < 32; lanes <<= 1) {
                            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], lanes));
                            product[x] = fmaxf(product[x], __shfl_xor_sync(0xffffffffu, product[x], lanes));
                        }
                        const float m_new = fmaxf(m[n][x], ceilf(top[x])), r_new = fmaxf(fmaxf(r[n][x], ceilf(product[x])), m_new - BELOW);
                        l[n][x] *= power(m[n][x] - m_new);
                        alpha[x] = power(r[n][x] - r_new);
                        m[n][x] = m_new;
                        r[n][x] = r_new;
                        from_m[n][x] = power(m_new - r_new);
                    }
#pragma unroll
                    for (int i = 0; i < CT; ++i) {
                        o[n][i][0] *= alpha[0];
                        o[n][i][1] *= alpha[1];
                        o[n][i][2] *= alpha[0];
                        o[n][i][3] *= alpha[1];
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float y[4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float ref = m[n][x] - BIAS, p0 = two_to(s[j][n][x] - ref), p1 = two_to(s[j][n][2 + x] - ref);
                        l[n][x] += p0 + p1;
                        float f = from_m[n][x] * (j ? v1 : v0);
                        f = f > FLT_MAX ? FLT_MAX : f;       // (beside weights of 0)
                        y[x] = p0 * f;
                        y[2 + x] = p1 * f;
                    }
                    if (edge) {                  // an unseen key's weight is 0 also beside a scale that is no number
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = base + 16 * j + 8 * (x >> 1) + g;
                            if (!(key <= pos[n][x & 1] && key >= low[n][x & 1])) y[x] = 0.f;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t first = pack(y[2 * h], y[2 * h + 1]);
                        pb[j][0][n][h] = transposed(first);
                        if (TERMS == 2) {
                            const float2 f = unpack(first);
                            pb[j][TERMS - 1][n][h] = transposed(pack(y[2 * h] - f.x, y[2 * h + 1] - f.y));
                        }
                    }
                }
            }
            // values: four keys of this lane in each block, four channels at a time
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[4][HD / 32];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned char* at = vt + (k & 1 ? v_at_1 : v_at) + (k >> 1) * (TILE / 2) + j * TILE;
                    if (HD == 128) *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(at);
                    else *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(at);
                }
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const uint32_t pick = i & 1 ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(w[0][i / 2], w[1][i / 2], pick) ^ 0x80808080u, y = __byte_perm(w[2][i / 2], w[3][i / 2], pick) ^ 0x80808080u;
                    if (TERMS == 1) {
                        const uint32_t v[4] = {offset_halves(x, 0x4140), offset_halves(x, 0x4342), offset_halves(y, 0x4140), offset_halves(y, 0x4342)};
                        const uint32_t less[4] = {0xe480e480u, 0xe480e480u, 0xe480e480u, 0xe480e480u};       // -1152
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            mma(o[n][i], v, pb[j][0][n][0], pb[j][0][n][1]);
                            mma(o[n][i], less, pb[j][0][n][0], pb[j][0][n][1]);
                        }
                    } else {
                        const uint32_t v[4] = {halves(x, 0x4140), halves(x, 0x4342), halves(y, 0x4140), halves(y, 0x4342)};
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int k = 0; k < TERMS; ++k) mma(o[n][i], v, pb[j][k][n][0], pb[j][k][n][1]);
                    }
                }
            }
        }

        // ---- the four warps' parts together ----
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[n][x];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = 8 * n + 2 * t + x;
                if (g == 0) sml[warp * ROWS + row] = make_float4(m[n][x], sum, r[n][x], 0.f);
                if (row < here) {
                    float* to = part_at(warp) + row * HD + g * (HD / 8);
#pragma unroll
                    for (int i = 0; i < CT; i += 2)
                        *reinterpret_cast<float4*>(to + 2 * i) = make_float4(o[n][i][x], o[n][i][2 + x], o[n][i + 1][x], o[n][i + 1][2 + x]);
                }
            }
        __syncthreads();
        auto block_of = [&](int x) { return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each; };
        const int first_block = block_of(item_u), parts = block_of(item_u + item_n - 1) - first_block + 1;
        // a block has two places: for an item whose pages began before its run (or with it), and for one whose began inside
        const int first_place = 2 * first_block + (run_start(first_block) < item_u ? 1 : 0);
        auto place_of = [&](int part) { return part == 0 ? first_place : 2 * (first_block + part); };
        for (int i = tid; i < here * (HD / 4); i += THREADS) {
            const int row = i / (HD / 4), d = i % (HD / 4) * 4;
            float top = LOWEST, high = LOWEST, sum = 0.f;
            float4 st[WARPS], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                st[w] = sml[w * ROWS + row];
                top = fmaxf(top, st[w].x);
                high = fmaxf(high, st[w].z);
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = power(st[w].x - top), x = power(st[w].z - high);
                const float4 p = *reinterpret_cast<const float4*>(part_at(w) + row * HD + d);
                sum = fmaf(st[w].y, f, sum);
                v = make_float4(fmaf(p.x, x, v.x), fmaf(p.y, x, v.y), fmaf(p.z, x, v.z), fmaf(p.w, x, v.w));
            }
            if (whole) {
                write(it, row0 + row, d, v, sum, top, high);
            } else if (own) {
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(smem) + row * HD + d) = v;       // where the first warp's keys were
                if (d == 0) sgroup[0][row] = make_float4(top, sum, high, 0.f);
            } else {
                const size_t at = (size_t)place_of(me - first_block) * a.rows_cap + row;
                *reinterpret_cast<float4*>(a.part + at * HD + d) = v;
                if (d == 0) a.stat[at] = make_float4(top, sum, high, 0.f);
            }
        }
        if (!own && !whole) {
            int n = parts, index = me - first_block, stride = 1;       // parts of this level, this block's among them, how far apart they lie
            for (int level = 0;; ++level) {
                const int lead = index / GROUP * GROUP, members = min(GROUP, n - lead);
                __syncthreads();                 // all of this block's part is written
                int* arrived = a.arrived + level * a.places + place_of(lead * stride);
                if (tid == 0) {
                    __threadfence();
                    last_here = atomicAdd(arrived, 1) == members - 1;
                    if (last_here) *arrived = 0;
                    __threadfence();
                }
                __syncthreads();
                if (!last_here) break;
                const bool done = n <= GROUP;
                constexpr int TWO = 2;           // places that a thread reads together
                float4 p[TWO][GROUP];
                auto read = [&](int i0) {
#pragma unroll
                    for (int z = 0; z < TWO; ++z) {
                        const int i = i0 + z * THREADS, row = i / (HD / 4), d = i % (HD / 4) * 4;
#pragma unroll
                        for (int x = 0; x < GROUP; ++x) {
                            p[z][x] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (x < members && row < here)
                                p[z][x] = __ldcg(reinterpret_cast<const float4*>(a.part + ((size_t)place_of((lead + x) * stride) * a.rows_cap + row) * HD + d));
                        }
                    }
                };
                // the parts' statistics, one per thread; what each part is weighted with, and the row's own
                float4 st = make_float4(LOWEST, 0.f, LOWEST, 0.f);
                if (tid < GROUP * ROWS && tid / ROWS < members && tid % ROWS < here)
                    st = __ldcg(a.stat + (size_t)place_of((lead + tid / ROWS) * stride) * a.rows_cap + tid % ROWS);
                read(tid);
                if (tid < GROUP * ROWS) sgroup[tid / ROWS][tid % ROWS] = st;
                __syncthreads();
                if (tid < here) {
                    float top = LOWEST, high = LOWEST, sum = 0.f;
                    for (int x = 0; x < members; ++x) top = fmaxf(top, sgroup[x][tid].x), high = fmaxf(high, sgroup[x][tid].z);
                    for (int x = 0; x < members; ++x) {
                        sum = fmaf(sgroup[x][tid].y, power(sgroup[x][tid].x - top), sum);
                        sgroup[x][tid].w = power(sgroup[x][tid].z - high);
                    }
                    sml[tid] = make_float4(top, sum, high, 0.f);
                }
                __syncthreads();
                for (int i0 = tid; i0 < here * (HD / 4); i0 += TWO * THREADS) {
                    if (i0 != tid) read(i0);
#pragma unroll
                    for (int z = 0; z < TWO; ++z) {
                        const int i = i0 + z * THREADS, row = i / (HD / 4), d = i % (HD / 4) * 4;
                        if (row >= here) continue;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int x = 0; x < GROUP; ++x) {
                            const float w = x < members ? sgroup[x][row].w : 0.f;
                            v = make_float4(fmaf(p[z][x].x, w, v.x), fmaf(p[z][x].y, w, v.y), fmaf(p[z][x].z, w, v.z), fmaf(p[z][x].w, w, v.w));
                        }
                        if (done) write(it, row0 + row, d, v, sml[row].y, sml[row].x, sml[row].z);
                        // in the place of the first (its channels are this thread's; its statistics have been read)
                        else *reinterpret_cast<float4*>(a.part + ((size_t)place_of(lead * stride) * a.rows_cap + row) * HD + d) = v;
                    }
                }
                if (done) break;
                if (tid < here) a.stat[(size_t)place_of(lead * stride) * a.rows_cap + tid] = sml[tid];
                n = (n + GROUP - 1) / GROUP;
                index = lead / GROUP;
                stride *= GROUP;
            }
        }
        if (own || stop != it.end || (u += SETUP) >= u1) break;
        __syncthreads();                         // the warps' parts have been read
        next_item(a, ROWS, it);
        page = it.low;
    }
    copies_wait<0>();
    if (!own) return;

    // ---- a cluster's parts: a warp for each row, eight lanes (four times) for their statistics, then one for each four channels ----
    cluster_sync();
    const int run = run_of(it.end - it.low), parts = (it.end - it.low + run - 1) / run, row0 = it.tile * ROWS, here = min(ROWS, it.n_rows - row0);
    for (int row = me % C + parts * warp; parts > 1 && row < here; row += parts * WARPS) {
        const int x8 = lane & 7;
        float4 st = make_float4(LOWEST, 0.f, LOWEST, 0.f), v = make_float4(0.f, 0.f, 0.f, 0.f), p[8];
        if (x8 < parts) st = peer_float4(reinterpret_cast<const float*>(&sgroup[0][row]), x8);
#pragma unroll
        for (int x = 0; x < 8; ++x)
            p[x] = x < parts && 4 * lane < HD ? peer_float4(reinterpret_cast<const float*>(smem) + row * HD + 4 * lane, x) : make_float4(0.f, 0.f, 0.f, 0.f);
        float top = st.x, high = st.z;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        const float w = power(st.z - high);
        float sum = st.y * power(st.x - top);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const float z = __shfl_sync(0xffffffffu, w, x);
            v = make_float4(fmaf(p[x].x, z, v.x), fmaf(p[x].y, z, v.y), fmaf(p[x].z, z, v.z), fmaf(p[x].w, z, v.w));
        }
        if (4 * lane < HD) write(it, row0 + row, 4 * lane, v, sum, top, high);
    }
    cluster_sync();                              // a peer may still be reading this block's part
}

// form, if asked for: which kernel it would be, clusters of eight, of four or runs of units (0, 1, 2), times 4 and NQ; nothing is launched
template <int HD, typename T, int TERMS, int NQ>
int launch(Args a, long long items, long long keys, long long part_floats, int* form, cudaStream_t stream) {
    static PerDeviceOnce once, once_own;
    static std::atomic<int> resident[64][3];
    // (tiles of 16 rows are for steps that do not fit clusters)
    const auto kernel = attn_quantized_kernel<HD, T, TERMS, NQ, false>, kernel_own = attn_quantized_kernel<HD, T, TERMS, NQ, NQ == 1>;
    constexpr int smem = SMEM_BYTES<HD, NQ>;
    if (raise_dynamic_smem(kernel, smem, once, "attention_quantized") || raise_dynamic_smem(kernel_own, smem, once_own, "attention_quantized")) return 1;
    // as many blocks as the device holds at once, in clusters of eight, of four or alone (asked once per device)
    int dev = 0;
    cudaGetDevice(&dev);
    auto held = [&](int which) {
        const int size = which == 2 ? 1 : 8 >> which;
        int n = dev >= 0 && dev < 64 ? resident[dev][which].load(std::memory_order_relaxed) : 0;
        if (n == 0) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)size);
            cfg.blockDim = dim3(THREADS);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)size;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            const cudaError_t e = size == 1 ? cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, THREADS, smem) : cudaOccupancyMaxActiveClusters(&n, kernel_own, &cfg);
            if (e != cudaSuccess || n <= 0) cudaGetLastError(), n = 1;
            n = std::min(size == 1 ? n * sm_count() : n, MOST_BLOCKS * sm_count() / size);
            if (dev >= 0 && dev < 64) resident[dev][which].store(n, std::memory_order_relaxed);
        }
        return n * size;
    };
    // A cluster for each item, of eight blocks or of four, where the device holds them all and nobody takes more than four turns, or eight
    // where there is one sequence (of several the longest holds the others up: with 8 sequences runs of units win once their
    // lengths are half of the longest on average).  With and without, us, 32 heads over 8 of 128: 1 sequence of 1,024 keys 5.7 and 9.1, 4,096
    // 8.9 and 14.1, 8,192 12.9 and 14.4, 16,384 23.0 and 17.3; 8 sequences of 4,096 17.2 and 23.4, 2,048 without 14.6; 16 of 2,048 (fours)
    // 17.5 and 20.9; float32, 4 of 4,096 12.8 and 18.3; 14 heads over 2 of 64: 1 of 437 4.9 and 6.4, 32 of 4,096 11.9 and 17.8.
    auto fits = [&](int size) { return keys <= (long long)(a.n_seqs == 1 ? 8 : 4) * 2 * PAGE * size; };
    const int which = NQ > 1 ? 2 : (8 * items <= held(0) && fits(8) ? 0 : (4 * items <= held(1) && fits(4) ? 1 : 2));
    if (form != nullptr) {
        *form = 4 * which + NQ;
        return 0;
    }
    a.cluster = which == 2 ? 1 : 8 >> which;
    const int blocks = which == 2 ? held(2) : a.cluster * (int)items;
    if (part_floats < 2ll * blocks * a.rows_cap * (HD + 4)) return fail("attention_quantized: scratch of %lld numbers is too small", part_floats);
    a.places = 2 * blocks;
    a.stat = reinterpret_cast<float4*>(a.part);
    a.part += (size_t)2 * blocks * a.rows_cap * 4;
    return launch_cluster("attention_quantized", which == 2 ? kernel : kernel_own, dim3((unsigned)blocks), THREADS, (size_t)smem, a.cluster, stream, a);
}

// a.n_seqs, n_rep, n_kv and span are set; longest: the keys of the longest sequence
int choose(Args a, int dtype, int max_new, int longest, int hd, long long part_floats, int* form, cudaStream_t stream) {
    const long long rows = (long long)max_new * a.n_rep;
    // A tile of 16 rows takes 1.75 times what one of 8 takes, which pays where the step has rows and keys for all of the SMs to be busy for
    // long, 80 pages for 8 rows and more to an SM; below that half as many items to spread over the blocks cost more.  Tiles of 8 and of 16,
    // us: 64 sequences of 1,024 keys, 32 heads over 8 of 128, 4 tokens 58.8 and 55.2 (16,384 pages), 16 tokens 182 and 165; 28 heads over 4, 3
    // tokens (21 rows) 43.9 and 51.4; float32, 1,000 tokens over 4,096 keys 645 and 509; below: 1 sequence of 1,024 keys, 4 tokens
    // 10.3 and 13.6; 4 sequences of 3,000, 12 heads over 2, 4 tokens in float32 15.3 and 20.9 (752 pages).
    const long long tiles = (rows + 7) / 8, wide = (rows + 15) / 16;
    const long long keys = a.span == 0 ? longest : std::min((long long)longest, (long long)max_new + (a.span > 0 ? a.span : -(long long)a.span));
    const int nq = 7 * wide < 4 * tiles && (keys + PAGE - 1) / PAGE * tiles * a.n_seqs * a.n_kv > 80ll * sm_count() ? 2 : 1;
    a.rows_cap = (int)(rows < 8 * nq ? rows : 8 * nq);
    const long long items = a.n_seqs * (nq == 1 ? tiles : wide) * a.n_kv;        // at most
    using B = __nv_bfloat16;
    if (dtype == RI_F32 && nq == 1) return hd == 64 ? launch<64, float, 2, 1>(a, items, keys, part_floats, form, stream) : launch<128, float, 2, 1>(a, items, keys, part_floats, form, stream);
    if (dtype == RI_F32) return hd == 64 ? launch<64, float, 2, 2>(a, items, keys, part_floats, form, stream) : launch<128, float, 2, 2>(a, items, keys, part_floats, form, stream);
    if (dtype == RI_BF16 && nq == 1) return hd == 64 ? launch<64, B, 1, 1>(a, items, keys, part_floats, form, stream) : launch<128, B, 1, 1>(a, items, keys, part_floats, form, stream);
    if (dtype == RI_BF16) return hd == 64 ? launch<64, B, 1, 2>(a, items, keys, part_floats, form, stream) : launch<128, B, 1, 2>(a, items, keys, part_floats, form, stream);
    return fail("attention_quantized: unknown dtype %d", dtype);
}

}  // namespace

// Which kernel `ri_attention_quantized` launches for such a step, as a number; -1 for one that it does not take
RI_API int ri_attention_quantized_form(int dtype, int n_seqs, int max_new, int longest, int n_heads, int n_kv, int hd, int span) {
    if (n_seqs <= 0 || max_new <= 0 || (hd != 64 && hd != 128) || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv) return -1;
    Args a = {};
    a.n_seqs = n_seqs, a.n_rep = n_heads / n_kv, a.n_kv = n_kv, a.span = span;
    int form = -1;
    return choose(a, dtype, max_new, longest, hd, 0, &form, nullptr) ? -1 : form;
}

// Thread blocks of a step, at most
RI_API int ri_attention_quantized_blocks() { return MOST_BLOCKS * sm_count(); }

// part: float32 [2 * blocks * min(16, n_rep * max_new) * (hd + 4)]; arrived: int32 [4 * 2 * blocks], zero, and left so.  longest: the keys of
// the longest sequence as far as the host knows them (what it chooses the tiles by; any number gives the same sums).
RI_API int ri_attention_quantized(const void* q, int dtype, int q_ld, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs,
                                  const int* page_table, int max_pages, const int* seq_slot, const int* seq_start, const int* cu_seqlens,
                                  void* out, int out_ld, int n_seqs, int max_new, int longest, int n_heads, int n_kv, int hd, float scale, int span,
                                  float out_scale, float* part, long long part_floats, int* arrived, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return 0;
    if (hd != 64 && hd != 128) return fail("attention_quantized: heads of %d channels (64 or 128 wanted)", hd);
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv) return fail("attention_quantized: %d heads over %d kv heads", n_heads, n_kv);
    if ((uintptr_t)kc % 16 || (uintptr_t)vc % 16 || (uintptr_t)part % 16) return fail("attention_quantized: codes and scratch must lie on 16-byte boundaries");
    const long long rows = (long long)max_new * (n_heads / n_kv);
    if ((long long)n_seqs * (max_pages + SETUP) * n_kv * ((rows + 7) / 8) > 0x7fffffff || rows > 0x7fffffff)
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
    a.part = part;
    a.arrived = arrived;
    return choose(a, dtype, max_new, longest, hd, part_floats, nullptr, stream);
}

RI_DEFINE_LAST_ERROR()
