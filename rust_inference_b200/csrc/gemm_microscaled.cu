// out[tokens, features] = X[tokens, K] * W[features, K]^T for X in microscaled 8 bits and W in microscaled 4 bits (microscaled.cuh) on the
// 5th-generation tensor cores: tcgen05.mma of kind mxf8f6f4 takes both as they are held, with their exponents from tensor memory, and
// adds in float32.  Nothing is widened in registers: a decode step is a read of its weights, 17/32 of a byte each.
//
// Codes come to shared memory by TMA with 128-byte swizzle: 128 numbers of a row, a span, are one swizzled row of 128 bytes.  Those of four bits
// are spread on the way (16 numbers to 8 bytes and 8 bytes left out, as the tensor cores read them), so that they cost half the memory's
// traffic and none of a warp's instructions; a copy's bytes are counted as they lie in memory.  The exponents of 128 rows and a span are a piece
// of 512 bytes, which a bulk copy brings along and tcgen05.cp puts into four columns of tensor memory, in order with the MMAs that read them.
//
// Two kernels, which are cut differently:
//   few tokens   the MMA's M runs over 128 features and its N over up to 128 tokens (`mx_feature_kernel`).  K is cut over the CTAs of a
//                cluster, whose sums meet in shared memory and are added in the order of the ranks: results do not depend on timing.
//   many         M runs over 256 tokens on a pair of SMs (cta_group::2), N over 256 rows of W (`mx_pair_kernel`).
//
// Epilogues (float32 arithmetic), all written to bfloat16 or float32, and all but the adding one to rows in 8 bits too, for the next product:
//   bias   acc + bias                                     act    act(acc) (`ActForm`, common.cuh)
//   add    out<float32> += acc                            gated  gate(acc, acc2), acc2 = X W2^T (`GateForm`)
// In the first kernel a warp's 32 lanes are a block of the next product's K, in the second a thread's 32 registers are.
//
// Every wait on an mbarrier is bounded, as in the bfloat16 products: a wait that runs out stores a code in the host-visible status word, the
// CTA stops issuing work, waits (bounded) for its own copies in flight, frees its tensor memory and returns.
#include "cluster.cuh"
#include "microscaled.cuh"
#include "tcgen05_common.cuh"

using namespace ri;
using namespace ri::tc;
using namespace ri::mx;

namespace {

constexpr int ROWS = 128;                          // rows of W or of X in a tile of shared memory
constexpr int TILE = ROWS * SPAN;                  // its bytes, a byte a number
constexpr int W_COPIED = TILE / 2;                 // what a copy of 4-bit codes counts
constexpr int MAX_STAGES = 12;
constexpr int THREADS = 320;
constexpr int SMEM_LIMIT = 225 * 1024;
constexpr int CLUSTER_MOST = 8;
constexpr int TOKENS_MOST = 128;                   // of a tile of the first kernel

enum Status { ST_PRODUCER_TIMEOUT = 51, ST_MMA_TIMEOUT = 52, ST_EPILOGUE_TIMEOUT = 53, ST_DRAIN_TIMEOUT = 54 };
constexpr int NEEDS_ROWS = 2;                       // a product's answer to plain rows that have to be in 8 bits before
enum Out { OUT_BF16 = 0, OUT_F32 = 1, OUT_ROWS = 2, OUT_ADD = 3 };

// Instruction descriptor of kind mxf8f6f4: the exponents' byte of A (bits 29, 30) and of B (4, 5) to be set per instruction, types of A and B
// (0: e4m3, 5: e2m1), exponents alone (bit 23), N / 8, M / 16.
__host__ __device__ constexpr uint32_t instruction(int m, int n, int type_a, int type_b) {
    return ((uint32_t)type_a << 7) | ((uint32_t)type_b << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t of_block(uint32_t idesc, int j) { return idesc | ((uint32_t)j << 29) | ((uint32_t)j << 4); }

// Shared-memory descriptor of a piece of exponents: 32 rows of 16 bytes, eight of them 128 bytes, not swizzled.
__device__ __forceinline__ uint64_t piece_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
template <int PAIR>
__device__ __forceinline__ void exponents_to_tmem(uint32_t leader, uint32_t taddr, uint64_t desc) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(leader) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(leader) : "memory");
}
template <int PAIR>
__device__ __forceinline__ void mx_mma(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t exp_a, uint32_t exp_b, bool accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(exp_a), "r"(exp_b), "r"((uint32_t)accumulate), "r"(leader) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(exp_a), "r"(exp_b), "r"((uint32_t)accumulate), "r"(leader) : "memory");
}
// Copies, for a warp that stays together: every lane calls, the one whose `leader` is set issues (in a branch that one lane takes, each took
// 120 clocks to issue, and these products wait for little else).
__device__ __forceinline__ void expect_by(uint32_t leader, uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}"
                 ::"r"(bar), "r"(bytes), "r"(leader) : "memory");
}
__device__ __forceinline__ void load_2d_by(uint32_t leader, uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(leader) : "memory");
}
// A ring's position: the stage, its barrier's parity, and what a look at that barrier, taken a step before, has shown.  (A wait that begins
// when its turn has come costs a step some 60 clocks, also where the barrier has long completed.)
struct Ring {
    uint32_t bars;               // the stages' barriers
    int s;
    uint32_t parity;
    bool seen;
    __device__ __forceinline__ uint32_t bar() const { return bars + 8u * (uint32_t)s; }
    __device__ __forceinline__ bool wait() const { return seen || mbar_wait_warp(bar(), parity); }      // bounded; the same answer for the warp
    // looks at the next stage's barrier before what is issued between the two calls
    __device__ __forceinline__ bool look(int stages) const {
        const bool wraps = s + 1 == stages;
        uint32_t ok;                       // (test_wait: try_wait would stay for a while)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(wraps ? bars : bar() + 8u), "r"(wraps ? parity ^ 1u : parity) : "memory");
        return ok != 0;
    }
    __device__ __forceinline__ void next(int stages, bool looked) {
        if (++s == stages) {
            s = 0;
            parity ^= 1u;
        }
        seen = __all_sync(0xffffffffu, looked);
    }
};
// a piece of exponents into this CTA's shared memory
__device__ __forceinline__ void load_piece_by(uint32_t leader, uint32_t dst, const uint8_t* src, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
                 ::"r"(dst), "l"(src), "r"((uint32_t)PIECE), "r"(bar), "r"(leader) : "memory");
}

// The epilogues' arithmetic.  `constants`: the bias [features], or an activation's or a gate's constants, or null.  Fast exponentials where
// the result is rounded to 8 or 16 bits, accurate ones where it stays in float32.
struct Epilogue {
    const float* constants;
    bool act;
    ActForm af;
    GateForm gf;
};
template <bool DUAL>
__device__ __forceinline__ Epilogue load_epilogue(const float* constants, int act) {
    Epilogue e;
    e.constants = constants;
    e.act = act != 0;
    e.af = (!DUAL && act != 0) ? load_act_form(constants) : ActForm{0.f, 0.f, 0.f};
    e.gf = load_gate_form(DUAL ? constants : nullptr);
    return e;
}
__device__ __forceinline__ float gated_quick(float g, float u, const GateForm& f) {
    g = at_most(g, f.limit);
    u = at_least(at_most(u, f.limit), -f.limit) + f.shift;
    const float inner = f.cubic == 0.f ? 1.f : fmaf(f.cubic * g, g, 1.f);          // (0 times an infinite gate is none)
    return __fdividef(g, 1.f + __expf(-f.alpha * g * inner)) * u * f.mult;
}
// the same with the constants of silu
__device__ __forceinline__ float silu_quick(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }
// `act_quick_f32` (common.cuh) without branches: a warp whose accumulators lie on both sides of zero would go through one after the other
// (256 features of a token took 7 us, 1.5 so)
__device__ __forceinline__ float act_chosen(float z, const ActForm& f) {
    const float series = z * z * fmaf(z, fmaf(z, fmaf(z, 1.f / 120.f, 1.f / 24.f), 1.f / 6.f), 0.5f);
    const float t = z > -0.25f ? series : __expf(z) - 1.f - z;
    const float curved = z > 0.f ? f.ap * z * z : f.an == 0.f ? 0.f : f.an * t;
    return fmaf(f.lin, z, curved);
}
template <bool DUAL, int OUT>
__device__ __forceinline__ float result(float a, float u, float bias, const Epilogue& e) {
    if (OUT == OUT_ADD) return a;
    if (DUAL) return OUT == OUT_F32 ? gated_f32(a, u, e.gf) : gated_quick(a, u, e.gf);
    if (e.act) return OUT == OUT_F32 ? act_f32(a, e.af) : act_chosen(a, e.af);
    return a + bias;
}

// So many of a warp's 32 rows of accumulators from one column on.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t* r) {
    if (N == 4)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
    else if (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
    else
        tmem_ld16(taddr, r);
}

// What a product writes: plain numbers [tokens, features], or rows in 8 bits with `spans` spans and their exponents.
struct Result {
    void* out;
    uint8_t* exponents;
    int n_spans;
};
// What N tokens (t(0), t(1), ...; those that `good` says) have at feature f of the first kernel, whose warp has 32 features that begin at a
// multiple of 32.  The tokens' chains of instructions are independent and without branches, so that they run side by side.
template <int OUT, int N, typename T, typename G>
__device__ __forceinline__ void store_lanes(const Result& r, T t, G good, int f, int n_feat, const float* v) {
    if (OUT == OUT_ROWS) {
        uint32_t byte[N];
#pragma unroll
        for (int j = 0; j < N; ++j) byte[j] = exponent_byte<8>(__reduce_max_sync(0xffffffffu, f < n_feat ? __float_as_uint(v[j]) & 0x7fffffffu : 0u));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint8_t code = eight_bits_of_one(f < n_feat ? v[j] * to_type(byte[j]) : 0.f);
            if (good(j)) reinterpret_cast<uint8_t*>(r.out)[(size_t)t(j) * r.n_spans * SPAN + f] = code;
        }
        if ((f & 31) == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (good(j)) r.exponents[exponent_at(t(j), f >> 5, r.n_spans)] = (uint8_t)byte[j];
        }
    } else if (f < n_feat) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const size_t at = (size_t)t(j) * n_feat + f;
            if (!good(j)) continue;
            if (OUT == OUT_BF16) reinterpret_cast<__nv_bfloat16*>(r.out)[at] = __float2bfloat16_rn(v[j]);
            else if (OUT == OUT_F32) reinterpret_cast<float*>(r.out)[at] = v[j];
            else atomicAdd(reinterpret_cast<float*>(r.out) + at, v[j]);         // one add per number: no order to depend on
        }
    }
}

// Plain rows that a kernel for few tokens brings to 8 bits itself: those whose spans all have a stage of the ring, up to 4 of them, and up to
// PLAIN_MOST where a CTA has no more than 32 spans of all rows together (64 where K is not cut).  The epilogue's warps, which have nothing else to do
// then, read them and write codes and exponents as TMA would have brought them.  (us, plain rows / by a kernel before: [3584, 3584], 7 spans a CTA,
// 1 token 5.1 / 6.4, 4 tokens 5.5 / 5.9, 8 tokens 6.0 / 5.75; [1536, 1536], 2 spans, 16 tokens 4.4 / 5.0; [896, 896], 7 spans, uncut, 8 tokens
// 4.05 / 4.2, 16 tokens 5.2 / 4.4.)
constexpr int PLAIN_MOST = 16;
struct PlainRows {
    const void* at;              // null: rows in 8 bits come by TMA
    int f32, k;
    long long ld;
};

// The CTA's spans, `count` from `begin` on, by 256 threads: eight numbers of a row each, so that sixteen threads have a span of a row, and four a
// block; two reads of a thread are on their way together.
template <typename T>
__device__ __forceinline__ void write_plain(const PlainRows& x, int n_tok, int begin, int count, uint32_t tiles, uint32_t tile_bytes, uint32_t pieces,
                                            uint32_t piece_bytes, int thread) {
    const int items = count * n_tok * 16, chunk = thread & 15;
    const uint32_t of_row = 0xffffu / (uint32_t)n_tok + 1;          // (exact: numbers below 2^10 by at most 16)
    for (int i0 = thread; i0 < items + 15; i0 += 2 * 256) {           // (whole quads go round together: items is a multiple of 16)
        float v[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int q = (i0 + i * 256) >> 4, span = (int)((uint32_t)q * of_row >> 16), row = q - span * n_tok, c = (begin + span) * SPAN + chunk * 8;
            const bool there = span < count && c < x.k;
            if (sizeof(T) == 2) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (there) {
                    const float4 f = load_written(reinterpret_cast<const float*>(reinterpret_cast<const T*>(x.at) + (size_t)row * x.ld + c));
                    w = *reinterpret_cast<const uint4*>(&f);
                }
                unpack8(w, v[i]);
            } else {
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                if (there) {
                    const float* at = reinterpret_cast<const float*>(x.at) + (size_t)row * x.ld + c;
                    a = load_written(at);
                    b = load_written(at + 4);
                }
                v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
                v[i][4] = b.x; v[i][5] = b.y; v[i][6] = b.z; v[i][7] = b.w;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int q = (i0 + i * 256) >> 4, span = (int)((uint32_t)q * of_row >> 16), row = q - span * n_tok;
            if (span >= count) break;
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
            const uint32_t four = 0xfu << (threadIdx.x & 28);
            top = max(top, __shfl_xor_sync(four, top, 1));
            top = max(top, __shfl_xor_sync(four, top, 2));
            const uint32_t byte = exponent_byte<8>(top);
            const float f = to_type(byte);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= f;
            const uint32_t at = tiles + (uint32_t)span * tile_bytes + row * SPAN + (((chunk >> 1) ^ (row & 7)) << 4) + (chunk & 1) * 8;
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(eight_bits(v[i])), "r"(eight_bits(v[i] + 4)) : "memory");
            if ((chunk & 3) == 0)
                asm volatile("st.shared.b8 [%0], %1;" ::"r"(pieces + (uint32_t)span * piece_bytes + row * 16 + (chunk >> 2)), "r"(byte) : "memory");
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Few tokens.  Tiles of 128 features x tn tokens, for a persistent grid of CTAs, or (not gated) each for a cluster whose CTAs share its K.  Warp 0
// issues the copies, warp 1 allocates tensor memory and issues the MMAs, warps 2-9 run the epilogue, two for each quarter of tensor memory's
// lanes, which take turns at TURN tokens.
// What bounds it: the weights' way from memory, where there are enough of them (8 tokens: two matrices [18944, 3584], 72 MB, 14.6 us, 4.9 TB/s; between
// the kernels of a step 12.7 with one token, since the first ring of weights goes out before the wait); else trips: the rows' 1 us after the wait, the last
// span's MMAs and the epilogue 0.5, the cluster's meeting 1.2 ([4608, 3584] 6.0 us, [3584, 3584] 5.5, [3584, 18944] 10.6, [896, 896] 3.0).
// ---------------------------------------------------------------------------------------------
template <bool DUAL, int OUT, int TURN>
__global__ void __launch_bounds__(THREADS, DUAL ? 1 : 2)
mx_feature_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_x,
                  const uint8_t* __restrict__ w_exp, const uint8_t* __restrict__ w2_exp, const uint8_t* x_exp, const PlainRows plain, const float* __restrict__ constants, int act,
                  Result res, int n_tok, int n_feat, int n_spans, int cluster, int stages, int tn, int buffers, int tmem_cols, int recv_at, int* status) {
    constexpr int MATS = DUAL ? 2 : 1;
    const uint32_t tile_bytes = MATS * TILE + tn * SPAN;                          // of a stage's codes
    constexpr uint32_t EXP_BYTES = (MATS + 1) * PIECE;                            // of its exponents
    const uint32_t stage_tx = (uint32_t)(MATS * (W_COPIED + PIECE) + (plain.at == nullptr ? tn * SPAN + PIECE : 0));
    const int acc_cols = MATS * tn;
    const uint32_t idesc = instruction(ROWS, tn, 5, 0);

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
    __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
    __shared__ __align__(8) uint64_t acc_full[2];
    __shared__ __align__(8) uint64_t acc_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag, any_failed;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t exp_base = smem_base + (uint32_t)stages * tile_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quarter = warp & 3, half = (warp - 2) >> 2;      // epilogue warps: the TMEM lanes that a warp may read, and which of the two it is
    const bool clustered = !DUAL && cluster > 1;
    const int rank = clustered ? (int)cluster_rank() : 0;
    const int n_tok_tiles = (n_tok + tn - 1) / tn, n_feat_tiles = (n_feat + ROWS - 1) / ROWS;
    const int total_tiles = n_tok_tiles * n_feat_tiles;
    // a cluster has one tile, a CTA without one its share of them
    const int first = (int)blockIdx.x / cluster;
    const int my_tiles = clustered ? 1 : (first < total_tiles) ? (total_tiles - 1 - first) / (int)gridDim.x + 1 : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), plain.at == nullptr ? 1 : 9);         // the copies', and the writing warps'
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 8);             // one arrival per epilogue warp
        }
        abort_flag = any_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"((uint32_t)tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);
    if (clustered) cluster_arrive();                   // "this CTA runs, its flags are set"
    let_next_kernel_start();

    // token tiles vary fastest, so that CTAs which run together share a tile of W in L2
    auto tile_coords = [&](int i, int& f0, int& t0) {
        const int tile = first + i * (int)gridDim.x;
        f0 = (tile / n_tok_tiles) * ROWS;
        t0 = (tile % n_tok_tiles) * tn;
    };
    const int begin = n_spans * rank / cluster, count = n_spans * (rank + 1) / cluster - begin;       // spans of this CTA: cluster <= n_spans

    if (warp == 0) {
        {                                                        // the whole warp goes through, one lane issues
            const uint32_t leader = elect_one();
            int it = 0;                      // spans issued
            Ring ring{empty0, 0, 1u, true};  // (a barrier's phase before its first counts as completed)
            bool waited = false, alive = true;
            for (int i = 0; i < my_tiles && alive; ++i) {
                int f0, t0;
                tile_coords(i, f0, t0);
                if (abort_flag) break;
                // pieces of exponents of this tile's rows (a tile's tokens are all or the first of one: tn is 128, or there is one tile)
                const uint8_t* we = w_exp + ((size_t)(f0 / ROWS) * n_spans + begin) * PIECE;
                const uint8_t* we2 = DUAL ? w2_exp + ((size_t)(f0 / ROWS) * n_spans + begin) * PIECE : nullptr;
                const uint8_t* xe = x_exp + ((size_t)(t0 / ROWS) * n_spans + begin) * PIECE;
                const int w_row = ((f0 / ROWS) * n_spans + begin) * ROWS;        // the map's, of the tile of the first span
                auto load_w = [&](int at, int j) {
                    const uint32_t bar = full0 + 8u * (uint32_t)at, stage = smem_base + (uint32_t)at * tile_bytes, ex = exp_base + (uint32_t)at * EXP_BYTES;
                    expect_by(leader, bar, stage_tx);
                    load_2d_by(leader, stage, &map_w, bar, 0, w_row + j * ROWS);
                    if (DUAL) load_2d_by(leader, stage + TILE, &map_w2, bar, 0, w_row + j * ROWS);
                    load_piece_by(leader, ex, we + (size_t)j * PIECE, bar);
                    if (DUAL) load_piece_by(leader, ex + PIECE, we2 + (size_t)j * PIECE, bar);
                };
                auto load_x = [&](int at, int j) {
                    if (plain.at != nullptr) return;
                    const uint32_t bar = full0 + 8u * (uint32_t)at;
                    load_2d_by(leader, smem_base + (uint32_t)at * tile_bytes + MATS * TILE, &map_x, bar, (begin + j) * SPAN, t0);
                    load_piece_by(leader, exp_base + (uint32_t)at * EXP_BYTES + MATS * PIECE, xe + (size_t)j * PIECE, bar);
                };
                int j = 0;
                if (!waited) {
                    // the weights are written by no kernel: a ring of them goes out before the wait for the one that makes the rows
                    const int ahead = min(stages, count);
                    for (; j < ahead; ++j) load_w(j, j);
                    wait_for_previous_kernels();
                    waited = true;
                    for (j = 0; j < ahead; ++j) load_x(j, j);
                    it = ahead;
                    if (ahead == stages) ring = Ring{empty0, 0, 0u, false}; else ring.s = ahead;
                }
                for (; j < count; ++j, ++it) {
                    if (!ring.wait()) {
                        if (lane == 0 && !abort_flag) report(status, ST_PRODUCER_TIMEOUT);
                        abort_flag = 1;
                        alive = false;
                        break;
                    }
                    const bool looked = ring.look(stages);
                    load_w(ring.s, j);
                    load_x(ring.s, j);
                    ring.next(stages, looked);
                }
            }
            RI_PHASE_LATEST(1);
            // do not leave, or hand the ring to the cluster, while a copy into it may still be in flight
            for (int j = max(0, it - stages); j < it; ++j)
                if (!mbar_wait_warp(full0 + 8u * (uint32_t)(j % stages), (uint32_t)(j / stages) & 1u)) {
                    if (lane == 0) report(status, ST_DRAIN_TIMEOUT);
                    abort_flag = 1;
                    break;
                }
        }
    } else if (warp == 1) {
        const uint32_t leader = elect_one();                     // the whole warp goes through, one lane issues
        Ring ring{full0, 0, 0u, false};
        bool alive = true;
        const uint64_t desc_w0 = make_smem_desc(smem_base), desc_e0 = piece_desc(exp_base);
        for (int i = 0; i < my_tiles && alive; ++i) {
            int f0, t0;
            tile_coords(i, f0, t0);
            const int buf = buffers == 2 ? i & 1 : 0, round = buffers == 2 ? i >> 1 : i;
            if (!mbar_wait_warp(smem_u32(&acc_empty[buf]), (uint32_t)(round & 1) ^ 1u)) {
                if (lane == 0) report(status, ST_MMA_TIMEOUT);
                abort_flag = 1;
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem_base + (uint32_t)(buf * acc_cols);
            for (int j = 0; j < count; ++j) {
                if (!ring.wait()) {
                    if (lane == 0) report(status, ST_MMA_TIMEOUT);
                    abort_flag = 1;
                    alive = false;
                    break;
                }
                tc_fence_after();
                const bool looked = ring.look(stages);
                // exponents go to one of two sets of columns behind the accumulators, while the MMAs before still read the other
                const uint32_t ex = tmem_base + (uint32_t)(buffers * acc_cols + (j & 1) * (MATS + 1) * 4);
                const uint64_t e = desc_e0 + (uint64_t)((uint32_t)ring.s * (EXP_BYTES >> 4));
#pragma unroll
                for (int m = 0; m <= MATS; ++m) exponents_to_tmem<0>(leader, ex + 4 * m, e + (uint64_t)(m * (PIECE >> 4)));
                const uint64_t w = desc_w0 + (uint64_t)((uint32_t)ring.s * (tile_bytes >> 4)), x = w + (uint64_t)(MATS * (TILE >> 4));
#pragma unroll
                for (int b = 0; b < SPAN / BLOCK; ++b) {
                    mx_mma<0>(leader, acc, w + 2 * b, x + 2 * b, of_block(idesc, b), ex, ex + 4 * MATS, j > 0 || b > 0);
                    if (DUAL) mx_mma<0>(leader, acc + tn, w + (TILE >> 4) + 2 * b, x + 2 * b, of_block(idesc, b), ex + 4, ex + 4 * MATS, j > 0 || b > 0);
                }
                umma_commit_by(leader, empty0 + 8u * (uint32_t)ring.s);
                ring.next(stages, looked);
            }
            umma_commit_by(leader, smem_u32(&acc_full[buf]));
        }
    } else {
        wait_for_previous_kernels();          // `out` may still be read or written by the kernel before
        if (plain.at != nullptr) {                                // (a CTA has one tile then, and count <= stages)
            const uint32_t tiles = smem_base + MATS * TILE, pieces = exp_base + MATS * PIECE;
            if (plain.f32) write_plain<float>(plain, n_tok, begin, count, tiles, tile_bytes, pieces, EXP_BYTES, (int)threadIdx.x - 64);
            else write_plain<__nv_bfloat16>(plain, n_tok, begin, count, tiles, tile_bytes, pieces, EXP_BYTES, (int)threadIdx.x - 64);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // for the tensor cores' reads
            __syncwarp();
            if (lane < count) mbar_arrive(full0 + 8u * (uint32_t)lane);
        }
        const Epilogue e = load_epilogue<DUAL>(constants, act);
        for (int i = 0; i < my_tiles; ++i) {
            int f0, t0;
            tile_coords(i, f0, t0);
            const int buf = buffers == 2 ? i & 1 : 0, round = buffers == 2 ? i >> 1 : i;
            const bool landed = mbar_wait(smem_u32(&acc_full[buf]), (uint32_t)(round & 1));
            if (!landed) {
                if (lane == 0) report(status, ST_EPILOGUE_TIMEOUT);
                abort_flag = 1;
            }
            tc_fence_after();
            __syncwarp();
            if (__any_sync(0xffffffffu, !landed || abort_flag)) break;
            if (clustered) break;                                  // the pieces meet below
            const int f = f0 + quarter * 32 + lane;
            const float b = (!DUAL && !e.act && OUT != OUT_ADD && e.constants != nullptr && f < n_feat) ? e.constants[f] : 0.f;
            const uint32_t trow = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * acc_cols);
#pragma unroll 1
            for (int c0 = half * TURN; c0 < tn; c0 += 2 * TURN) {
                if (t0 + c0 >= n_tok) break;
                uint32_t v[TURN], u[TURN];
                tmem_load<TURN>(trow + c0, v);
                if (DUAL) tmem_load<TURN>(trow + tn + c0, u);
                tmem_wait_ld();
                float r[TURN];
#pragma unroll
                for (int j = 0; j < TURN; ++j) r[j] = result<DUAL, OUT>(__uint_as_float(v[j]), DUAL ? __uint_as_float(u[j]) : 0.f, b, e);
                store_lanes<OUT, TURN>(res, [&](int j) { return t0 + c0 + j; }, [&](int j) { return t0 + c0 + j < n_tok; }, f, n_feat, r);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
        }
    }

    RI_PHASE_LATEST(2);
    if constexpr (!DUAL) if (clustered) {
        // Token c of the tile is finished by the CTA of rank c % cluster: everybody sends it its sums of that token, into `recv`
        // [rank of the sender][c / cluster][128], and it adds them in the order of the ranks.  `recv` lies behind the ring, where both are in
        // the shared memory that there is (`recv_at`), else where the ring was, once nobody's is in use any more.
        // A CTA that gave up says so before; then none of the cluster writes.
        const int held = (tn + cluster - 1) / cluster;
        int f0, t0;
        tile_coords(0, f0, t0);
        const int tokens = min(tn, n_tok - t0);
        float* recv = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)) + recv_at);
        const int fl = quarter * 32 + lane;
        __syncwarp();
        cluster_wait();                                            // the peers run
        if (abort_flag && lane == 0) set_in_all(&any_failed, cluster);
        __syncwarp();
        if (recv_at == 0) cluster_sync();                          // nobody's ring is in use any more
        if (warp >= 2 && !abort_flag) {
            const uint32_t trow = tmem_base + ((uint32_t)(quarter * 32) << 16);
            const float* mine = recv + (size_t)rank * held * ROWS + fl;
#pragma unroll 1
            for (int c0 = half * TURN; c0 < tokens; c0 += 2 * TURN) {
                uint32_t v[TURN];
                tmem_load<TURN>(trow + c0, v);
                tmem_wait_ld();
                int to = c0 % cluster, at = (c0 / cluster) * ROWS;
#pragma unroll
                for (int j = 0; j < TURN; ++j) {
                    if (c0 + j < tokens) store_peer_float(mine + at, (uint32_t)to, __uint_as_float(v[j]));
                    if (++to == cluster) { to = 0; at += ROWS; }
                }
            }
        }
        __syncwarp();
        cluster_sync();                                            // everything sent has arrived
        const bool failed = any_failed != 0;
        const int f = f0 + fl;
        if (warp >= 2 && !failed) {
            const Epilogue e = load_epilogue<false>(constants, act);
            const float b = (!e.act && OUT != OUT_ADD && e.constants != nullptr && f < n_feat) ? e.constants[f] : 0.f;
            constexpr int TOGETHER = 4;
            for (int i = half * TOGETHER; rank + i * cluster < tokens; i += 2 * TOGETHER) {
                const int c = rank + i * cluster, n = min(TOGETHER, (tokens - c + cluster - 1) / cluster);      // tokens c, c + cluster, ...
                float a[TOGETHER] = {};
                const float* from = recv + (size_t)i * ROWS + fl;
#pragma unroll 4
                for (int p = 0; p < cluster; ++p, from += (size_t)held * ROWS) {
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j) {
                        if (j < n) a[j] += from[j * ROWS];
                    }
                }
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) a[j] = result<false, OUT>(a[j], 0.f, b, e);
                store_lanes<OUT, TOGETHER>(res, [&](int j) { return t0 + c + j * cluster; }, [&](int j) { return j < n; }, f, n_feat, a);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    RI_PHASE_LATEST(5);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)tmem_cols) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// Many tokens, on pairs of SMs (tcgen05 cta_group::2).  A tile is 256 tokens x 256 rows of W: 256 features, or the gate rows of 128 and the up
// rows of the same.  Each CTA of the pair holds 128 of the tokens (its half of A and of the accumulator) and 128 of the rows of W (its half of
// B, which the tensor cores of both read), and the exponents of its tokens and of all the rows of W.  The first CTA issues the MMAs.
//
// Two accumulators of 256 columns would leave tensor memory no room for exponents, so the second begins 32 columns before the first ends: an
// epilogue reads the columns that both use first, and says so, and then the MMAs of the next tile may begin.
//
// What bounds it: the clock, which falls to 1.6 GHz under these MMAs, and at it the tensor cores, which are busy for 75 to 87% of the time; the way from
// L2 (8.6 TB/s; without the copies of X an eighth less time), the turn of the accumulators at a tile's end (7% at 28 spans a tile), the epilogue's
// instructions and stores (4 and 3%).  2,048 tokens: gated [18944, 3584] 184 us, 3.0 PFLOP/s, with one kernel for the two matrices and the rows in 8 bits
// that the next product reads; [3584, 18944] onto the stream 100 us, 2.8 PFLOP/s.
// ---------------------------------------------------------------------------------------------
constexpr int PAIR_TOK = 2 * ROWS, PAIR_ROWS = 2 * ROWS;
constexpr int PAIR_EXP = 3 * PIECE;                    // exponents of a stage: 128 tokens, 256 rows of W
constexpr int PAIR_STAGE = 2 * TILE + PAIR_EXP;
constexpr int SECOND_ACC = 224, PAIR_EXP_COL = 480;    // columns: accumulators [0, 256) and [224, 480), two sets of exponents behind them

__device__ __forceinline__ uint32_t in_first_cta(uint32_t local_addr) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(local_addr));
    return a;
}
// A tile into this CTA's shared memory whose arrival is counted by a barrier of the pair's first CTA.
__device__ __forceinline__ void load_2d_pair(uint32_t leader, uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
        ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(leader) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(bar), "h"((uint16_t)3), "r"(leader) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    tmem_ld16(taddr, r);
    tmem_ld16(taddr + 16, r + 16);
}

// 32 features of a token each, from feature f on, as the 32 threads of a warp have computed them for tokens t.. of which `tokens` are there: pieces of
// 16 bytes change places in the warp's 2 KB of shared memory, so that neighbouring threads write neighbouring pieces.
constexpr int EXCHANGE = 2048;
__device__ __forceinline__ uint32_t piece_at(uint32_t room, int token, int piece, int pieces) {
    return room + (uint32_t)(token * pieces + (piece ^ (token * pieces / 8 & (pieces - 1)))) * 16u;
}
template <int PIECES>
__device__ __forceinline__ void spread(uint32_t room, int lane, const uint4* c) {
    __syncwarp();
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(room, lane, q, PIECES)), "r"(c[q].x), "r"(c[q].y), "r"(c[q].z), "r"(c[q].w) : "memory");
    __syncwarp();
}
template <int PIECES>
__device__ __forceinline__ void exchange(uint32_t room, int lane, uint4* c) {
    spread<PIECES>(room, lane, c);
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(c[q].x), "=r"(c[q].y), "=r"(c[q].z), "=r"(c[q].w)
                     : "r"(piece_at(room, q * (32 / PIECES) + lane / PIECES, lane % PIECES, PIECES)) : "memory");
}
template <int OUT>
__device__ __forceinline__ void store_run(const Result& r, int t, int tokens, int f, int n_feat, bool aligned, uint32_t room, int lane, float* v) {
    if (OUT == OUT_ROWS) {
        if (f + 32 > n_feat) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = f + j < n_feat ? v[j] : 0.f;
        }
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        const uint32_t byte = exponent_byte<8>(top);
        const float by = to_type(byte);
        uint4 c[2];
        uint32_t* w = reinterpret_cast<uint32_t*>(c);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = v[4 * q + j] * by;
            w[q] = eight_bits(y);
        }
        exchange<2>(room, lane, c);
        uint8_t* to = reinterpret_cast<uint8_t*>(r.out) + (size_t)(t + lane / 2) * r.n_spans * SPAN + f + lane % 2 * 16;
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (q * 16 + lane / 2 < tokens) *reinterpret_cast<uint4*>(to + (size_t)(q * 16) * r.n_spans * SPAN) = c[q];
        if (lane < tokens) r.exponents[exponent_at(t + lane, f >> 5, r.n_spans)] = (uint8_t)byte;
        return;
    }
    if (aligned && f + 32 <= n_feat) {
        if (OUT == OUT_BF16) {
            uint4 c[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) c[q] = pack8(v + 8 * q);
            exchange<4>(room, lane, c);
            __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(r.out) + (size_t)(t + lane / 4) * n_feat + f + lane % 4 * 8;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q * 8 + lane / 4 < tokens) *reinterpret_cast<uint4*>(to + (size_t)(q * 8) * n_feat) = c[q];
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {                                             // sixteen features at a time
                uint4 c[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) c[q] = *reinterpret_cast<uint4*>(v + 16 * h + 4 * q);
                exchange<4>(room, lane, c);
                float* to = reinterpret_cast<float*>(r.out) + (size_t)(t + lane / 4) * n_feat + f + 16 * h + lane % 4 * 4;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q * 8 + lane / 4 < tokens) {
                        float* at = to + (size_t)(q * 8) * n_feat;
                        if (OUT == OUT_ADD)
                            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(__uint_as_float(c[q].x)),
                                         "f"(__uint_as_float(c[q].y)), "f"(__uint_as_float(c[q].z)), "f"(__uint_as_float(c[q].w)) : "memory");
                        else
                            *reinterpret_cast<uint4*>(at) = c[q];
                    }
            }
        }
        return;
    }
    // rows off a 16-byte boundary, or the last features: a number at a time, those of neighbouring features together (2,048 tokens of [4606, 3584],
    // float32 sums: 157 -> 35 us)
    if constexpr (OUT == OUT_BF16) {
        uint4 c[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = pack8(v + 8 * q);
        spread<4>(room, lane, c);
        uint16_t* to = reinterpret_cast<uint16_t*>(r.out) + (size_t)t * n_feat + f + lane;
#pragma unroll 8
        for (int row = 0; row < 32; ++row) {
            uint16_t y;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(piece_at(room, row, lane / 8, 4) + lane % 8 * 2) : "memory");
            if (row < tokens && f + lane < n_feat) to[(size_t)row * n_feat] = y;
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                                 // sixteen features of two tokens
            spread<4>(room, lane, reinterpret_cast<const uint4*>(v + 16 * h));
            const int at = f + 16 * h + lane % 16;
            float* to = reinterpret_cast<float*>(r.out) + (size_t)(t + lane / 16) * n_feat + at;
#pragma unroll 8
            for (int row = lane / 16; row < 32; row += 2, to += (size_t)2 * n_feat) {
                float y;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(piece_at(room, row, lane % 16 / 4, 4) + lane % 4 * 4) : "memory");
                if (row < tokens && at < n_feat) {
                    if (OUT == OUT_ADD) atomicAdd(to, y);
                    else *to = y;
                }
            }
        }
    }
}

template <bool DUAL, int OUT>
__global__ void __launch_bounds__(THREADS, 1)
mx_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_we, const __grid_constant__ CUtensorMap map_we2, const __grid_constant__ CUtensorMap map_xe,
               const float* __restrict__ constants, int act, Result res, int n_tok, int n_feat, int n_spans, int stages, int* status) {
    constexpr int FEATS = DUAL ? PAIR_ROWS / 2 : PAIR_ROWS;    // features of a tile
    constexpr uint32_t IDESC = instruction(PAIR_TOK, PAIR_ROWS, 0, 5);
    constexpr uint32_t CTA_TX = TILE + W_COPIED + PAIR_EXP;    // bytes of a stage that a CTA's copies count

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];     // used in the first CTA only
    __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
    __shared__ __align__(8) uint64_t acc_full[2];
    __shared__ __align__(8) uint64_t next_bar;                 // first CTA: the epilogues have read the columns that the next tile writes too
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t exp_base = smem_base + (uint32_t)stages * 2 * TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();                      // 0: issues the MMAs
    const int pair = (int)blockIdx.x >> 1, n_pairs = (int)gridDim.x >> 1;
    const int n_tok_tiles = (n_tok + PAIR_TOK - 1) / PAIR_TOK, n_feat_tiles = (n_feat + FEATS - 1) / FEATS;
    const int total_tiles = n_tok_tiles * n_feat_tiles;
    const int my_tiles = (pair < total_tiles) ? (total_tiles - 1 - pair) / n_pairs + 1 : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&acc_full[i]), 1);
        mbar_init(smem_u32(&next_bar), 16);                    // one arrival per epilogue warp of the pair
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();                                        // the partner's barriers stand before anything arrives there
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);
    const uint32_t full0_first = in_first_cta(full0);
    let_next_kernel_start();

    // token tiles vary fastest, so that pairs which run together share the rows of W in L2
    auto tile_coords = [&](int i, int& f0, int& t0) {
        const int item = pair + i * n_pairs;
        t0 = (item % n_tok_tiles) * PAIR_TOK;
        f0 = (item / n_tok_tiles) * FEATS;
    };

    if (warp == 0) {
        {                                                        // the whole warp goes through, one lane issues
            const uint32_t leader = elect_one();
            int it = 0;
            Ring ring{empty0, 0, 1u, true};
            bool alive = true;
            wait_for_previous_kernels();                         // the rows come from the kernel before
            const CUtensorMap* my_w = (DUAL && rank == 1) ? &map_w2 : &map_w;
            const CUtensorMap* second_we = DUAL ? &map_we2 : &map_we;
            const int w_off = DUAL ? 0 : rank * ROWS;
            for (int i = 0; i < my_tiles && alive; ++i) {
                int f0, t0;
                tile_coords(i, f0, t0);
                if (abort_flag) break;
                // pieces of exponents: a row of a map each (beyond the last one: zeros)
                const int w_row = ((f0 + w_off) / ROWS) * n_spans * ROWS;        // the map's, of this CTA's tile of the first span (beyond the last one: zeros)
                const int xe = (t0 / ROWS + rank) * n_spans, we = (f0 / ROWS) * n_spans, we2 = DUAL ? we : we + n_spans;
                for (int j = 0; j < n_spans; ++j, ++it) {
                    if (!ring.wait()) {
                        if (lane == 0 && !abort_flag) report(status, ST_PRODUCER_TIMEOUT);
                        abort_flag = 1;
                        alive = false;
                        break;
                    }
                    const bool looked = ring.look(stages);
                    const uint32_t stage = smem_base + (uint32_t)ring.s * 2 * TILE, ex = exp_base + (uint32_t)ring.s * PAIR_EXP, bar = full0_first + 8u * (uint32_t)ring.s;
                    if (rank == 0) expect_by(leader, full0 + 8u * (uint32_t)ring.s, 2 * CTA_TX);                 // both CTAs' bytes
                    load_2d_pair(leader, stage, &map_x, bar, j * SPAN, t0 + rank * ROWS);
                    load_2d_pair(leader, stage + TILE, my_w, bar, 0, w_row + j * ROWS);
                    load_2d_pair(leader, ex, &map_xe, bar, 0, xe + j);
                    load_2d_pair(leader, ex + PIECE, &map_we, bar, 0, we + j);
                    load_2d_pair(leader, ex + 2 * PIECE, second_we, bar, 0, we2 + j);
                    ring.next(stages, looked);
                }
            }
            // Do not leave while a copy into this CTA's shared memory may still be in flight: a stage whose `empty` barrier has completed
            // again was read by the MMAs, so its copies had landed.
            for (int j = 0; j < stages && it > 0; ++j) {
                if (!ring.wait()) {
                    if (lane == 0) report(status, ST_DRAIN_TIMEOUT);
                    break;
                }
                ring.next(stages, false);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {                                         // the whole warp goes through, one lane issues
            const uint32_t leader = elect_one();
            Ring ring{full0, 0, 0u, false};
            bool alive = true;
            const uint64_t desc_x0 = make_smem_desc(smem_base), desc_e0 = piece_desc(exp_base);
            for (int i = 0; i < my_tiles && alive; ++i) {
                const uint32_t acc = tmem_base + (uint32_t)((i & 1) * SECOND_ACC);
                for (int j = 0; j < n_spans; ++j) {
                    if (!ring.wait()) {
                        if (lane == 0) report(status, ST_MMA_TIMEOUT);
                        abort_flag = 1;
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const bool looked = ring.look(stages);
                    const uint32_t ex = tmem_base + (uint32_t)(PAIR_EXP_COL + (j & 1) * 16);
                    const uint64_t e = desc_e0 + (uint64_t)((uint32_t)ring.s * (PAIR_EXP >> 4));
#pragma unroll
                    for (int m = 0; m < 3; ++m) exponents_to_tmem<1>(leader, ex + 4 * m, e + (uint64_t)(m * (PIECE >> 4)));
                    if (j == 0 && i > 0) {
                        // the columns that the tile before shares have been read, and with them all of the one before that
                        if (!mbar_wait_warp(smem_u32(&next_bar), (uint32_t)(i - 1) & 1u)) {
                            if (lane == 0) report(status, ST_MMA_TIMEOUT);
                            abort_flag = 1;
                            alive = false;
                            break;
                        }
                        tc_fence_after();
                    }
                    const uint64_t x = desc_x0 + (uint64_t)((uint32_t)ring.s * (2 * TILE >> 4)), w = x + (TILE >> 4);
#pragma unroll
                    for (int b = 0; b < SPAN / BLOCK; ++b)
                        mx_mma<1>(leader, acc, x + 2 * b, w + 2 * b, of_block(IDESC, b), ex, ex + 4, j > 0 || b > 0);
                    commit_pair(leader, empty0 + 8u * (uint32_t)ring.s); // frees the stage in both CTAs
                    ring.next(stages, looked);
                }
                commit_pair(leader, smem_u32(&acc_full[i & 1]));
            }
        }
    } else {
        // a thread has a token, and 32 of its features at a time; two warps share a quarter of the tokens and take turns at the runs
        const int lane_base = (warp & 3) * 32, half = (warp - 2) >> 2;
        const uint32_t next_first = in_first_cta(smem_u32(&next_bar));
        wait_for_previous_kernels();
        const Epilogue e = load_epilogue<DUAL>(constants, act);
        const uint32_t room = exp_base + (uint32_t)stages * PAIR_EXP + (uint32_t)(warp - 2) * EXCHANGE;
        const bool aligned = (OUT == OUT_BF16 ? n_feat % 8 == 0 : n_feat % 4 == 0) && (reinterpret_cast<uintptr_t>(res.out) & 15) == 0;
        for (int i = 0; i < my_tiles; ++i) {
            int f0, t0;
            tile_coords(i, f0, t0);
            const bool landed = mbar_wait(smem_u32(&acc_full[i & 1]), (uint32_t)(i >> 1) & 1u);
            if (!landed) {
                if (lane == 0) report(status, ST_EPILOGUE_TIMEOUT);
                abort_flag = 1;
            }
            tc_fence_after();
            __syncwarp();
            if (__any_sync(0xffffffffu, !landed || abort_flag)) break;
            const int t = t0 + rank * ROWS + lane_base;                // the warp's first token
            const uint32_t trow = tmem_base + ((uint32_t)lane_base << 16) + (uint32_t)((i & 1) * SECOND_ACC);
            constexpr int RUNS = FEATS / 32;
#pragma unroll 1
            for (int n = half; n < RUNS; n += 2) {
                // the first accumulator shares its last columns, the second its first: those are read in the first turn
                const int c = ((i & 1) ? n : RUNS - 1 - n) * 32, f = f0 + c;
                alignas(16) float v[32], u[DUAL ? 32 : 1];
                if (!DUAL || (i & 1)) tmem_ld32(trow + c, reinterpret_cast<uint32_t*>(v));
                else tmem_ld32(trow + ROWS + c, reinterpret_cast<uint32_t*>(u));
                if (n == half) {
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_cluster(next_first);
                }
                if (DUAL) {
                    if (i & 1) tmem_ld32(trow + ROWS + c, reinterpret_cast<uint32_t*>(u));
                    else tmem_ld32(trow + c, reinterpret_cast<uint32_t*>(v));
                }
                tmem_wait_ld();
                if (f >= (OUT == OUT_ROWS ? res.n_spans * SPAN : n_feat) || t >= n_tok) continue;           // (of no thread's, or of all)
                if (DUAL && OUT != OUT_F32 && e.constants == nullptr) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = silu_quick(v[j], u[DUAL ? j : 0]);
                } else if (DUAL || e.act) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = result<DUAL, OUT>(v[j], DUAL ? u[j] : 0.f, 0.f, e);
                } else if (OUT != OUT_ADD && e.constants != nullptr) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] += f + j < n_feat ? e.constants[f + j] : 0.f;
                }
                store_run<OUT>(res, t, n_tok - t, f, n_feat, aligned, room, lane, v);
            }
        }
    }

    // nothing of the pair's tensor or shared memory is freed while the partner may still use it
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Codes as a tensor map with a box of a span and `box_rows` rows, 128-byte swizzle, zeros outside: of 8 bits, or of 4 that are spread.
int encode_codes(CUtensorMap* map, const void* ptr, long long rows, int n_spans, int bits, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail("gemm_microscaled: cuTensorMapEncodeTiled is not available from the driver");
    if ((uintptr_t)ptr % 32) return fail("gemm_microscaled: codes must begin on a 32-byte boundary");
    // (a matrix's tiles lie one after the other: rows of a span, 128 for each of them)
    cuuint64_t dims[2] = {(cuuint64_t)(bits == 4 ? 1 : n_spans) * SPAN, bits == 4 ? (cuuint64_t)((rows + ROWS - 1) / ROWS) * n_spans * ROWS : (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)dims[0] * bits / 8};
    cuuint32_t box[2] = {(cuuint32_t)SPAN, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = fn(map, bits == 4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
                    elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("gemm_microscaled: cuTensorMapEncodeTiled failed (code %d)", (int)r);
    return 0;
}

// Exponents as a tensor map whose rows are pieces.
int encode_pieces(CUtensorMap* map, const void* ptr, long long pieces) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail("gemm_microscaled: cuTensorMapEncodeTiled is not available from the driver");
    if ((uintptr_t)ptr % 16) return fail("gemm_microscaled: exponents must begin on a 16-byte boundary");
    cuuint64_t dims[2] = {PIECE / 4, (cuuint64_t)pieces};
    cuuint64_t strides[1] = {PIECE};
    cuuint32_t box[2] = {PIECE / 4, 1};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("gemm_microscaled: cuTensorMapEncodeTiled failed for exponents (code %d)", (int)r);
    return 0;
}

// The tensor maps that a matrix or rows keep: of the codes, with boxes of so many rows, and of the exponents.
struct Maps {
    CUtensorMap codes, exponents;
};
static_assert(sizeof(Maps) == sizeof(Held::maps[0]), "a pair of maps");
int maps_of(Held* h, int box_rows, const Maps** found) {
    const int i = box_rows / 16 - 1;
    Maps* m = reinterpret_cast<Maps*>(h->maps[i]);
    if (!(h->made.load(std::memory_order_acquire) >> i & 1u)) {
        if (int rc = encode_codes(&m->codes, h->codes, h->n, h->n_spans, h->bits, box_rows)) return rc;
        if (int rc = encode_pieces(&m->exponents, h->exponents, (long long)(h->n + ROWS - 1) / ROWS * h->n_spans)) return rc;
        h->made.fetch_or(1u << i, std::memory_order_release);
    }
    *found = m;
    return 0;
}

// How a product is cut: on pairs of SMs, or into tiles of tn tokens with K over the CTAs of a cluster, one or two CTAs to an SM.
struct Plan {
    bool pairs;
    int tn, cluster, per_sm;
};
struct Call {
    Plan plan;
    const Maps *w, *w2, *x;
    const uint8_t *w_exp, *w2_exp, *x_exp;
    PlainRows plain;
    const float* constants;
    int act;
    Result res;
    int n_tok, n_feat, n_spans;
    int* status;
    cudaStream_t stream;
};

int columns(int need) { return need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512; }

int g_pair_tokens = 0;           // > 0: products of at least so many tokens run on pairs of SMs, others do not (tests)

// What a product takes, in units of 10 ns, from measurements of the products of models 896 to 4,096 wide (weights from memory), good to a tenth
// where no other product of the rule is near (tn: tokens of the tile):
//   first kernel, not cut   a round of tiles: 12.5 + 0.066 tn a span, and 100 beside the next one's; once 190 + 1.85 tn
//   cut over clusters       the same for the spans of a CTA; once 320 + 2.2 tn, and the codes at 6 TB/s
//   either, up to 16 tokens 60 more where a CTA's spans are more than its ring holds, but less than two of it: the last are asked for when the rows have
//                           come, and nothing hides their wait ([1536, 1536], 12 spans, ring of 11, 1 token: uncut 4.25 us, clusters of 8 3.5, plain rows
//                           5.2 / 3.75; [4608, 3584], 28 spans: uncut 6.0, clusters of 3 6.0, and a decode step of 8 sequences 5% slower with them)
//   pairs                   a round of tiles: 34 a span, and 90; once 560 (stores of 256 tokens that nothing runs beside)
// So a product of [3584, 3584] (us, first kernel / pairs) with 256 tokens takes 11.9 / 15.5, 1,024: 18.7 / 16.9, 2,048: 31.9 / 27.4, and of
// [3584, 18944] 25.1 / 49.4, 70.5 / 54.1 and 133 / 106; of [2048, 2048] with 64 tokens, not cut / in clusters of four, 5.3 / 5.7, of [3584, 3584]
// 7.5 / 7.1, of [3584, 18944] 30 / 13.1.
Plan plan(int n_tok, int n_feat, int n_spans, bool dual) {
    Plan p;
    p.tn = n_tok >= TOKENS_MOST ? TOKENS_MOST : (n_tok + 15) / 16 * 16;
    p.cluster = p.per_sm = 1;
    const long long sms = sm_count(), feat_tiles = (n_feat + ROWS - 1) / ROWS, tiles = feat_tiles * ((n_tok + p.tn - 1) / p.tn);
    if (dual) {
        // Gated products fill the ring with two matrices, and a cluster's exchange costs them what it saves.  On pairs a tile has twice the
        // tokens and reads them once for both matrices: beyond 128 tokens always (160 tokens, 148 tiles 43.9 / 26.6 us), from 56 where a
        // round is enough (56 tokens, 38 tiles 8.7 / 8.0, 70 tiles 10.75 / 10.75; 96 tokens 11.5 / 8.1, 13.7 / 10.4; 86 tiles, two rounds, 16.1 / 16.7).
        p.pairs = n_tok > TOKENS_MOST || (n_tok >= 56 && 2 * feat_tiles <= sms);
    } else {
        const double span = 12.5 + 0.066 * p.tn, rounds = (double)((tiles + sms - 1) / sms);
        const double meet = 320 + 2.2 * p.tn + (double)n_feat * n_spans * (SPAN / 2) / 6e4;
        const int ring = (SMEM_LIMIT - 1024) / (TILE + p.tn * SPAN + 2 * PIECE);
        auto late = [&](int count) { return p.tn <= 16 && count > ring && count < 2 * ring ? 60 : 0; };
        double best = rounds * (span * n_spans + 100) + 90 + 1.85 * p.tn + late(n_spans);
        for (int c = 2; c <= CLUSTER_MOST && c <= n_spans; ++c) {
            // Clusters of whole SMs lie within groups of SMs, which leaves some over, and those of the next kernel come in while these leave: where
            // there are many, the last find their place late (36 clusters of 4, 9.9 us instead of 6.1), large ones sooner (16 of 7, 12.2 instead
            // of 7.1).
            if (tiles * c > (c > 4 ? sms * 2 / 3 : sms - 20)) continue;
            const double cost = span * ((n_spans + c - 1) / c) + meet + late((n_spans + c - 1) / c);
            if (cost < best) {
                best = cost;
                p.cluster = c;
            }
        }
        // Up to 16 tokens, whose stages are small, twice the CTAs keep more copies in flight where each still has a long piece of K
        // (8 tokens, us, one CTA per SM / two: [3584, 18944] 11.6 / 10.9, [4096, 14336] 10.4 / 10.0, [6144, 4096] 7.3 / 6.9).
        if (n_tok <= 16 && n_spans / p.cluster >= 14) {
            const long long most = 2 * (sms - 10) / tiles;
            const int c = (int)(most < CLUSTER_MOST ? most : CLUSTER_MOST);
            if (c > p.cluster) {
                p.cluster = c;
                p.per_sm = 2;
            }
        }
        const long long pair_tiles = (long long)((n_tok + PAIR_TOK - 1) / PAIR_TOK) * ((n_feat + PAIR_ROWS - 1) / PAIR_ROWS), pairs = sms / 2;
        p.pairs = n_tok > TOKENS_MOST && ((pair_tiles + pairs - 1) / pairs) * (34.0 * n_spans + 90) + 560 < best;
    }
    if (g_pair_tokens > 0) p.pairs = n_tok >= g_pair_tokens;
    if (p.pairs) p.tn = ROWS;
    return p;
}

template <bool DUAL, int OUT, int TURN>
int launch_feature(const Call& c) {
    const Plan& p = c.plan;
    const long long tiles = (long long)((c.n_tok + p.tn - 1) / p.tn) * ((c.n_feat + ROWS - 1) / ROWS);
    if (tiles > 0x7fffffffLL / CLUSTER_MOST) return fail("gemm_microscaled: %lld tiles exceed the index range", tiles);
    auto kernel = mx_feature_kernel<DUAL, OUT, TURN>;
    static PerDeviceOnce configured;
    if (int rc = raise_dynamic_smem(kernel, SMEM_LIMIT, configured, "gemm_microscaled")) return rc;
    constexpr int MATS = DUAL ? 2 : 1;
    const int stage = MATS * TILE + p.tn * SPAN + (MATS + 1) * PIECE;
    const int recv = p.cluster > 1 ? p.cluster * ((p.tn + p.cluster - 1) / p.cluster) * ROWS * 4 : 0;
    const int most = (c.n_spans + p.cluster - 1) / p.cluster;            // spans of a CTA
    // A ring fills the SM, also where a next kernel's could begin in half of it: what is on its way from memory is what these products wait for
    // (8 tokens, a gated product of [18944, 3584]: 102 KB of codes on their way 16.2 us, 51 KB 19.6).
    int stages = ((p.per_sm == 2 ? SMEM_LIMIT / 2 : SMEM_LIMIT) - 1024) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (p.cluster > 1 && stages > most) stages = most;
    const size_t ring = (size_t)stages * stage;
    // what a cluster's CTAs send each other has a place of its own where it is small (a meeting point fewer), else the ring's
    const bool apart = p.cluster > 1 && recv <= 32 * 1024 && ring + recv + 1024 <= (size_t)(p.per_sm == 2 ? SMEM_LIMIT / 2 : SMEM_LIMIT);
    const int recv_at = apart ? (int)ring : 0;
    size_t smem = (apart ? ring + recv : ring > (size_t)recv ? ring : (size_t)recv) + 1024;
    long long ctas = tiles * p.cluster;
    if (p.cluster == 1 && ctas > sm_count()) ctas = sm_count();
    if (c.plain.at != nullptr && (stages < most || ctas < tiles || (c.n_tok > 4 && most * c.n_tok > (p.cluster > 1 ? 32 : 64)))) return NEEDS_ROWS;
    // two accumulators, so that a tile's epilogue runs beside the next one's MMAs, where a CTA has several tiles and the columns suffice
    constexpr int EXP_COLS = 2 * (MATS + 1) * 4;
    const int one = MATS * p.tn + EXP_COLS, two = one + MATS * p.tn;
    const int buffers = (p.cluster == 1 && ctas < tiles && two <= 512) ? 2 : 1;
    const int need = buffers == 2 ? two : one, cols = columns(need);
    if (need > 512 || stages < 1 || smem > (size_t)SMEM_LIMIT) return fail("gemm_microscaled: %d columns of tensor memory, %lld bytes of shared memory", need, (long long)smem);
    // CTAs that wait for others of their cluster must not wait for tensor memory that CTAs of another cluster hold, which may wait likewise:
    // shared memory in proportion to their columns keeps all that an SM takes in within its 512 columns.
    if (p.cluster > 1 && smem < (size_t)cols * 456) smem = (size_t)cols * 456 < SMEM_LIMIT ? (size_t)cols * 456 : SMEM_LIMIT;
    return launch_cluster("gemm_microscaled", kernel, dim3((unsigned)ctas), THREADS, smem, p.cluster, c.stream, c.w->codes, c.w2->codes, c.x->codes, c.w_exp,
                          c.w2_exp, c.x_exp, c.plain, c.constants, c.act, c.res, c.n_tok, c.n_feat, c.n_spans, p.cluster, stages, p.tn, buffers, cols, recv_at, c.status);
}

template <bool DUAL, int OUT>
int launch_pair(const Call& c) {
    constexpr int FEATS = DUAL ? PAIR_ROWS / 2 : PAIR_ROWS;
    const long long tiles = (long long)((c.n_tok + PAIR_TOK - 1) / PAIR_TOK) * ((c.n_feat + FEATS - 1) / FEATS);
    if (tiles > 0x7fffffffLL) return fail("gemm_microscaled: %lld tiles exceed the index range", tiles);
    auto kernel = mx_pair_kernel<DUAL, OUT>;
    static PerDeviceOnce configured;
    if (int rc = raise_dynamic_smem(kernel, SMEM_LIMIT, configured, "gemm_microscaled")) return rc;
    constexpr int ROOM = 8 * EXCHANGE, STAGES = (SMEM_LIMIT - 1024 - ROOM) / PAIR_STAGE;
    static_assert(STAGES <= MAX_STAGES && STAGES >= 2, "a ring of stages");
    long long pairs = sm_count() / 2;
    if (pairs > tiles) pairs = tiles;
    return launch_cluster("gemm_microscaled (pairs of SMs)", kernel, dim3((unsigned)(2 * pairs)), THREADS, (size_t)STAGES * PAIR_STAGE + ROOM + 1024, 2, c.stream,
                          c.w->codes, c.w2->codes, c.x->codes, c.w->exponents, c.w2->exponents, c.x->exponents, c.constants, c.act, c.res, c.n_tok, c.n_feat,
                          c.n_spans, STAGES, c.status);
}

template <bool DUAL, int OUT>
int launch(const Call& c) {
    if (c.plan.pairs) return c.plain.at != nullptr ? NEEDS_ROWS : launch_pair<DUAL, OUT>(c);
    // Up to 16 tokens a turn of the epilogue takes 8, of gated products 4, since a turn costs as much for tokens that are not there; beyond that 16
    // (us, turns of 16 / 8 / 4: gated [18944, 3584] 1 token 15.8 / 14.7 / 14.3, 16 tokens 16.0 / 15.0 / 15.2, 61 19.4 / 19.7 / 19.8; [1152, 896] 1
    // token 3.25 / 3.0 / 3.0, 61 4.0 / 4.0 / 4.2).
    return c.n_tok <= 16 ? launch_feature<DUAL, OUT, DUAL ? 4 : 8>(c) : launch_feature<DUAL, OUT, 16>(c);
}

}  // namespace

// tokens > 0: products of at least so many tokens run on pairs of SMs, others do not; 0: as planned (for comparisons and tests).
RI_API int ri_mx_set_pairs(int tokens) {
    g_pair_tokens = tokens;
    return 0;
}

// out = X W^T with an epilogue: a bias or nothing (`constants` float32 [features] or null); `act`: an activation's four constants; w2 not null:
// the gate's five constants, or null for silu; `add`: added to out.  x, w, w2 and, where the result is rows in 8 bits, out_held are `Held`s; otherwise
// `out` is [out_rows, out_cols] of `out_dtype`.  X is what x holds, or, with `x_plain` not null, the plain rows
// [x->n, x->k] there, `x_ld` numbers apart; the answer is 2, and nothing is done, where they have to be brought to x first.
// `status` is a host-visible int that receives a code if a wait ran out.
RI_API int ri_mx_product(void* x_held, const void* x_plain, int x_dtype, long long x_rows, long long x_cols, long long x_ld, void* w_held, void* w2_held, const float* constants,
                         long long n_constants, int act, int add, void* out, int out_dtype, long long out_rows, long long out_cols, void* out_held,
                         int* status, cudaStream_t stream) {
    Held *x = (Held*)x_held, *w = (Held*)w_held, *w2 = (Held*)w2_held, *to = (Held*)out_held;
    const long long n_tok = x->n;
    // (other CTAs read their rows and matrices while the first ones write)
    const long long out_bytes = out ? out_rows * out_cols * item_bytes(out_dtype) : 0, plain_bytes = x_plain ? ((x_rows - 1) * x_ld + x_cols) * item_bytes(x_dtype) : 0;
    auto from_result = [&](const Held* h) { return h == nullptr || (to ? apart(h, to) : apart(h, out, out_bytes)); };
    auto from_result_bytes = [&](const void* p, long long bytes) { return to ? apart(to, p, bytes) : apart(out, out_bytes, p, bytes); };
    if (!from_result(x) || !from_result(w) || !from_result(w2) || !from_result_bytes(x_plain, plain_bytes) || !from_result_bytes(constants, 4 * n_constants))
        return fail("gemm_microscaled: the result must lie apart from the rows, the matrices and the constants");
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || x->device != device || w->device != device || (w2 && w2->device != device) || (to && to->device != device))
        return fail("gemm_microscaled: rows and matrices lie on the current device");
    if (x->bits != 8 || x->k != w->k || w->bits != 4 || (w2 && (w2->bits != 4 || w2->n != w->n || w2->k != w->k)))
        return fail("gemm_microscaled: rows and a matrix [%d, %d], or two matrices, that do not go together", w->n, w->k);
    if (x_plain && (x_rows != x->n || x_cols != x->k || x_ld < x->k)) return fail("gemm_microscaled: plain rows [%lld, %lld] for [%d, %d]", x_rows, x_cols, x->n, x->k);
    if (to ? (to->bits != 8 || to->n != n_tok || to->k != w->n) : (out_rows != n_tok || out_cols != w->n))
        return fail("gemm_microscaled: the result is [%lld, %d]", n_tok, w->n);
    if (add && (to || out_dtype != RI_F32)) return fail("gemm_microscaled: sums are added to float32 numbers");
    if ((act != 0) + (add != 0) + (w2 != nullptr) > 1 || (add && constants)) return fail("gemm_microscaled: a bias, an activation, a gate and an addition are not combined");
    if ((act && !constants) || (constants && n_constants != (act ? 4 : w2 ? 5 : w->n)))
        return fail("gemm_microscaled: %lld constants of an epilogue", n_constants);
    // plain rows are read in whole eights on 16-byte boundaries
    if (x_plain && (n_tok > PLAIN_MOST || x->k % 8 || (uintptr_t)x_plain % 16 || x_ld * (x_dtype == RI_BF16 ? 2 : 4) % 16)) return NEEDS_ROWS;
    const Plan p = plan((int)n_tok, w->n, w->n_spans, w2 != nullptr);
    Call c;
    c.plan = p;
    if (maps_of(x, p.tn, &c.x) || maps_of(w, ROWS, &c.w) || maps_of(w2 ? w2 : w, ROWS, &c.w2)) return 1;
    c.x_exp = x->exponents;
    c.plain = PlainRows{x_plain, x_dtype != RI_BF16, w->k, x_ld};
    c.w_exp = w->exponents;
    c.w2_exp = w2 ? w2->exponents : nullptr;
    c.constants = constants;
    c.act = act;
    c.res = to ? Result{to->codes, to->exponents, to->n_spans} : Result{out, nullptr, 0};
    c.n_tok = (int)n_tok;
    c.n_feat = w->n;
    c.n_spans = w->n_spans;
    c.status = status;
    c.stream = stream;
    if (w2) {
        if (to) return launch<true, OUT_ROWS>(c);
        return out_dtype == RI_BF16 ? launch<true, OUT_BF16>(c) : launch<true, OUT_F32>(c);
    }
    if (to) return launch<false, OUT_ROWS>(c);
    if (add) return launch<false, OUT_ADD>(c);
    return out_dtype == RI_BF16 ? launch<false, OUT_BF16>(c) : launch<false, OUT_F32>(c);
}

RI_DEFINE_LAST_ERROR()
