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
constexpr int THREADS = 192;
constexpr int SMEM_LIMIT = 225 * 1024;
constexpr int CLUSTER_MOST = 8;
constexpr int TOKENS_MOST = 128;                   // of a tile of the first kernel

enum Status { ST_PRODUCER_TIMEOUT = 51, ST_MMA_TIMEOUT = 52, ST_EPILOGUE_TIMEOUT = 53, ST_DRAIN_TIMEOUT = 54 };
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
// A piece of exponents into this CTA's shared memory.
__device__ __forceinline__ void load_piece(uint32_t dst, const uint8_t* src, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"((uint32_t)PIECE), "r"(bar) : "memory");
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
    g = fminf(g, f.limit);
    u = fmaxf(fminf(u, f.limit), -f.limit) + f.shift;
    return __fdividef(g, 1.f + __expf(-f.alpha * g * fmaf(f.cubic * g, g, 1.f))) * u * f.mult;
}
template <bool DUAL, int OUT>
__device__ __forceinline__ float result(float a, float u, float bias, const Epilogue& e) {
    if (OUT == OUT_ADD) return a;
    if (DUAL) return OUT == OUT_F32 ? gated_f32(a, u, e.gf) : gated_quick(a, u, e.gf);
    if (e.act) return OUT == OUT_F32 ? act_f32(a, e.af) : act_quick_f32(a, e.af);
    return a + bias;
}

// What a product writes: plain numbers [tokens, features], or rows in 8 bits with `spans` spans and their exponents.
struct Result {
    void* out;
    uint8_t* exponents;
    int n_spans;
};
// One number of token t and feature f of the first kernel, whose warp has 32 features that begin at a multiple of 32.
template <int OUT>
__device__ __forceinline__ void store_lane(const Result& r, int t, int f, int n_feat, float v) {
    if (OUT == OUT_ROWS) {
        if (f >= n_feat) v = 0.f;
        const uint32_t byte = exponent_byte<8>(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
        reinterpret_cast<uint8_t*>(r.out)[(size_t)t * r.n_spans * SPAN + f] = eight_bits_of_one(v * to_type(byte));
        if ((f & 31) == 0) r.exponents[exponent_at(t, f >> 5, r.n_spans)] = (uint8_t)byte;
    } else if (f < n_feat) {
        const size_t at = (size_t)t * n_feat + f;
        if (OUT == OUT_BF16) reinterpret_cast<__nv_bfloat16*>(r.out)[at] = __float2bfloat16_rn(v);
        else if (OUT == OUT_F32) reinterpret_cast<float*>(r.out)[at] = v;
        else atomicAdd(reinterpret_cast<float*>(r.out) + at, v);         // one add per number: no order to depend on
    }
}

// ---------------------------------------------------------------------------------------------
// Few tokens.  A persistent grid of tiles of 128 features x tn tokens, or clusters of CTAs that share a tile's K.  Warp 0 issues the copies,
// warp 1 allocates tensor memory and issues the MMAs, warps 2-5 run the epilogue.
// ---------------------------------------------------------------------------------------------
template <bool DUAL, int OUT>
__global__ void __launch_bounds__(THREADS, 1)
mx_feature_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_x,
                  const uint8_t* __restrict__ w_exp, const uint8_t* __restrict__ w2_exp, const uint8_t* x_exp, const float* __restrict__ constants, int act,
                  Result res, int n_tok, int n_feat, int n_spans, int cluster, int stages, int tn, int buffers, int tmem_cols, int* status) {
    constexpr int MATS = DUAL ? 2 : 1;
    const uint32_t tile_bytes = MATS * TILE + tn * SPAN;                          // of a stage's codes
    constexpr uint32_t EXP_BYTES = (MATS + 1) * PIECE;                            // of its exponents
    const uint32_t stage_tx = (uint32_t)(MATS * (W_COPIED + PIECE) + tn * SPAN + PIECE);
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
    const bool clustered = cluster > 1;
    const int rank = clustered ? (int)cluster_rank() : 0;
    const int n_tok_tiles = (n_tok + tn - 1) / tn, n_feat_tiles = (n_feat + ROWS - 1) / ROWS;
    const int total_tiles = n_tok_tiles * n_feat_tiles;
    const int my_tiles = clustered ? 1 : ((int)blockIdx.x < total_tiles) ? (total_tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 4);
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
    auto tile_coords = [&](int i, int& f0, int& t0, int& begin, int& count) {
        if (clustered) {
            f0 = ((int)blockIdx.x / cluster) * ROWS;
            t0 = 0;
            begin = n_spans * rank / cluster;
            count = n_spans * (rank + 1) / cluster - begin;                // >= 1: cluster <= n_spans
            return;
        }
        const int tile = (int)blockIdx.x + i * (int)gridDim.x;
        f0 = (tile / n_tok_tiles) * ROWS;
        t0 = (tile % n_tok_tiles) * tn;
        begin = 0;
        count = n_spans;
    };

    if (warp == 0) {
        if (lane == 0) {
            int it = 0, s = 0;               // spans issued; ring position and pass parity, carried along
            uint32_t ph = 0;
            bool waited = false, alive = true;
            for (int i = 0; i < my_tiles && alive; ++i) {
                int f0, t0, begin, count;
                tile_coords(i, f0, t0, begin, count);
                if (abort_flag) break;
                // pieces of exponents of this tile's rows; a tile's tokens lie within one piece (tn = 128, or a single tile of fewer)
                const uint8_t* we = w_exp + ((size_t)(f0 / ROWS) * n_spans + begin) * PIECE;
                const uint8_t* we2 = DUAL ? w2_exp + ((size_t)(f0 / ROWS) * n_spans + begin) * PIECE : nullptr;
                const uint8_t* xe = x_exp + ((size_t)(t0 / ROWS) * n_spans + begin) * PIECE;
                auto load_w = [&](int at, int j) {
                    const uint32_t bar = full0 + 8u * (uint32_t)at, stage = smem_base + (uint32_t)at * tile_bytes, ex = exp_base + (uint32_t)at * EXP_BYTES;
                    mbar_expect_tx(bar, stage_tx);
                    tma_load_2d(stage, &map_w, bar, (begin + j) * SPAN, f0);
                    if (DUAL) tma_load_2d(stage + TILE, &map_w2, bar, (begin + j) * SPAN, f0);
                    load_piece(ex, we + (size_t)j * PIECE, bar);
                    if (DUAL) load_piece(ex + PIECE, we2 + (size_t)j * PIECE, bar);
                };
                auto load_x = [&](int at, int j) {
                    const uint32_t bar = full0 + 8u * (uint32_t)at, stage = smem_base + (uint32_t)at * tile_bytes, ex = exp_base + (uint32_t)at * EXP_BYTES;
                    tma_load_2d(stage + MATS * TILE, &map_x, bar, (begin + j) * SPAN, t0);
                    load_piece(ex + MATS * PIECE, xe + (size_t)j * PIECE, bar);
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
                    if (ahead == stages) ph = 1; else s = ahead;
                }
                for (; j < count; ++j, ++it) {
                    if (!mbar_wait(empty0 + 8u * s, ph ^ 1u)) {
                        if (!abort_flag) report(status, ST_PRODUCER_TIMEOUT);
                        abort_flag = 1;
                        alive = false;
                        break;
                    }
                    load_w(s, j);
                    load_x(s, j);
                    if (++s == stages) { s = 0; ph ^= 1u; }
                }
            }
            // do not leave, or hand the ring to the cluster, while a copy into it may still be in flight
            for (int j = max(0, it - stages); j < it; ++j)
                if (!mbar_wait(full0 + 8u * (uint32_t)(j % stages), (uint32_t)(j / stages) & 1u)) {
                    report(status, ST_DRAIN_TIMEOUT);
                    abort_flag = 1;
                    break;
                }
        }
    } else if (warp == 1) {
        const uint32_t leader = elect_one();                     // the whole warp goes through, one lane issues
        int s = 0;
        uint32_t ph = 0;
        bool alive = true;
        const uint64_t desc_w0 = make_smem_desc(smem_base), desc_e0 = piece_desc(exp_base);
        for (int i = 0; i < my_tiles && alive; ++i) {
            int f0, t0, begin, count;
            tile_coords(i, f0, t0, begin, count);
            const int buf = buffers == 2 ? i & 1 : 0, round = buffers == 2 ? i >> 1 : i;
            if (!mbar_wait_warp(smem_u32(&acc_empty[buf]), (uint32_t)(round & 1) ^ 1u)) {
                if (lane == 0) report(status, ST_MMA_TIMEOUT);
                abort_flag = 1;
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem_base + (uint32_t)(buf * acc_cols);
            for (int j = 0; j < count; ++j) {
                if (!mbar_wait_warp(full0 + 8u * s, ph)) {
                    if (lane == 0) report(status, ST_MMA_TIMEOUT);
                    abort_flag = 1;
                    alive = false;
                    break;
                }
                tc_fence_after();
                // exponents go to one of two sets of columns behind the accumulators, while the MMAs before still read the other
                const uint32_t ex = tmem_base + (uint32_t)(buffers * acc_cols + (j & 1) * (MATS + 1) * 4);
                const uint64_t e = desc_e0 + (uint64_t)((uint32_t)s * (EXP_BYTES >> 4));
#pragma unroll
                for (int m = 0; m <= MATS; ++m) exponents_to_tmem<0>(leader, ex + 4 * m, e + (uint64_t)(m * (PIECE >> 4)));
                const uint64_t w = desc_w0 + (uint64_t)((uint32_t)s * (tile_bytes >> 4)), x = w + (uint64_t)(MATS * (TILE >> 4));
#pragma unroll
                for (int b = 0; b < SPAN / BLOCK; ++b) {
                    mx_mma<0>(leader, acc, w + 2 * b, x + 2 * b, of_block(idesc, b), ex, ex + 4 * MATS, j > 0 || b > 0);
                    if (DUAL) mx_mma<0>(leader, acc + tn, w + (TILE >> 4) + 2 * b, x + 2 * b, of_block(idesc, b), ex + 4, ex + 4 * MATS, j > 0 || b > 0);
                }
                umma_commit_by(leader, empty0 + 8u * s);
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
            umma_commit_by(leader, smem_u32(&acc_full[buf]));
        }
    } else {
        wait_for_previous_kernels();          // `out` may still be read or written by the kernel before
        const int lane_base = (warp & 3) * 32;                 // the TMEM lanes this warp may read
        const Epilogue e = load_epilogue<DUAL>(constants, act);
        for (int i = 0; i < my_tiles; ++i) {
            int f0, t0, begin, count;
            tile_coords(i, f0, t0, begin, count);
            const int buf = buffers == 2 ? i & 1 : 0, round = buffers == 2 ? i >> 1 : i;
            const bool landed = mbar_wait(smem_u32(&acc_full[buf]), (uint32_t)(round & 1));
            if (!landed) {
                if (lane == 0) report(status, ST_EPILOGUE_TIMEOUT);
                abort_flag = 1;
            }
            tc_fence_after();
            __syncwarp();
            if (__any_sync(0xffffffffu, !landed || abort_flag)) break;
            if (clustered) break;                                  // the pieces of K meet below
            const int f = f0 + lane_base + lane;
            const float b = (!DUAL && !e.act && OUT != OUT_ADD && e.constants != nullptr && f < n_feat) ? e.constants[f] : 0.f;
            const uint32_t trow = tmem_base + ((uint32_t)lane_base << 16) + (uint32_t)(buf * acc_cols);
#pragma unroll 1
            for (int c0 = 0; c0 < tn; c0 += 16) {
                if (t0 + c0 >= n_tok) break;
                uint32_t v[16], u[16];
                tmem_ld16(trow + c0, v);
                if (DUAL) tmem_ld16(trow + tn + c0, u);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (t0 + c0 + j < n_tok)
                        store_lane<OUT>(res, t0 + c0 + j, f, n_feat, result<DUAL, OUT>(__uint_as_float(v[j]), DUAL ? __uint_as_float(u[j]) : 0.f, b, e));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
        }
    }

    if (clustered) {
        // Token c is finished by the CTA of rank c % cluster: everybody sends it its sums of that token, into `recv`
        // [rank of the sender][c / cluster][(gate, up)][128], which lies where the ring was, and it adds them in the order of the ranks.
        // A CTA that gave up says so before; then none of the cluster writes.
        constexpr int SENT = MATS * ROWS;                          // floats per token
        const int held = (n_tok + cluster - 1) / cluster;
        float* recv = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));
        const int fl = (warp & 3) * 32 + lane;
        __syncwarp();
        cluster_wait();                                            // the peers run
        if (abort_flag && lane == 0) set_in_all(&any_failed, cluster);
        __syncwarp();
        cluster_sync();                                            // nobody's ring is in use any more
        const bool failed = any_failed != 0;
        if (warp >= 2 && !failed) {
            const uint32_t trow = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
            const float* mine = recv + (size_t)rank * held * SENT + fl;
#pragma unroll 1
            for (int c0 = 0; c0 < n_tok; c0 += 16) {
                uint32_t v[16], u[16];
                tmem_ld16(trow + c0, v);
                if (DUAL) tmem_ld16(trow + tn + c0, u);
                tmem_wait_ld();
                int to = c0 % cluster, at = (c0 / cluster) * SENT;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (c0 + j >= n_tok) break;
                    store_peer_float(mine + at, (uint32_t)to, __uint_as_float(v[j]));
                    if (DUAL) store_peer_float(mine + at + ROWS, (uint32_t)to, __uint_as_float(u[j]));
                    if (++to == cluster) { to = 0; at += SENT; }
                }
            }
        }
        __syncwarp();
        cluster_sync();                                            // everything sent has arrived
        const int f = ((int)blockIdx.x / cluster) * ROWS + fl;
        if (warp >= 2 && !failed) {
            const Epilogue e = load_epilogue<DUAL>(constants, act);
            const float b = (!DUAL && !e.act && OUT != OUT_ADD && e.constants != nullptr && f < n_feat) ? e.constants[f] : 0.f;
            for (int i = 0, c = rank; c < n_tok; ++i, c += cluster) {
                const float* from = recv + (size_t)i * SENT + fl;
                float a = 0.f, u = 0.f;
                for (int p = 0; p < cluster; ++p, from += (size_t)held * SENT) {
                    a += from[0];
                    if (DUAL) u += from[ROWS];
                }
                store_lane<OUT>(res, c, f, n_feat, result<DUAL, OUT>(a, u, b, e));
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)tmem_cols) : "memory");
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
    cuuint64_t dims[2] = {(cuuint64_t)n_spans * SPAN, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)n_spans * SPAN * bits / 8};
    cuuint32_t box[2] = {(cuuint32_t)SPAN, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = fn(map, bits == 4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
                    elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("gemm_microscaled: cuTensorMapEncodeTiled failed (code %d)", (int)r);
    return 0;
}

struct Call {
    const CUtensorMap *w, *w2, *x;
    const uint8_t *w_exp, *w2_exp, *x_exp;
    const float* constants;
    int act;
    Result res;
    int n_tok, n_feat, n_spans;
    int* status;
    cudaStream_t stream;
};

int columns(int need) { return need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512; }

// How the first kernel cuts a product: tokens of a tile and CTAs of a cluster.
struct Plan {
    int tn, cluster;
};
Plan plan(int n_tok, int n_feat, int n_spans) {
    Plan p;
    p.tn = n_tok >= TOKENS_MOST ? TOKENS_MOST : (n_tok + 15) / 16 * 16;
    p.cluster = 1;
    const long long tiles = (long long)((n_feat + ROWS - 1) / ROWS);
    if (n_tok <= TOKENS_MOST)
        while (p.cluster < CLUSTER_MOST && tiles * (p.cluster + 1) <= sm_count() && n_spans >= 2 * (p.cluster + 1)) ++p.cluster;
    return p;
}

template <bool DUAL, int OUT>
int launch_feature(const Call& c) {
    constexpr int MATS = DUAL ? 2 : 1;
    const Plan p = plan(c.n_tok, c.n_feat, c.n_spans);
    const long long tiles = (long long)((c.n_tok + p.tn - 1) / p.tn) * ((c.n_feat + ROWS - 1) / ROWS);
    if (tiles > 0x7fffffffLL / CLUSTER_MOST) return fail("gemm_microscaled: %lld tiles exceed the index range", tiles);
    auto kernel = mx_feature_kernel<DUAL, OUT>;
    static PerDeviceOnce configured;
    if (int rc = raise_dynamic_smem(kernel, SMEM_LIMIT, configured, "gemm_microscaled")) return rc;
    const int stage = MATS * TILE + p.tn * SPAN + (MATS + 1) * PIECE;
    const int recv = p.cluster > 1 ? p.cluster * ((c.n_tok + p.cluster - 1) / p.cluster) * MATS * ROWS * 4 : 0;
    const int most = (c.n_spans + p.cluster - 1) / p.cluster;            // spans of a tile
    int stages = (SMEM_LIMIT - 1024) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (p.cluster > 1 && stages > most) stages = most;
    const size_t ring = (size_t)stages * stage;
    size_t smem = (ring > (size_t)recv ? ring : (size_t)recv) + 1024;
    long long ctas = p.cluster > 1 ? tiles * p.cluster : tiles;
    if (p.cluster == 1 && ctas > sm_count()) ctas = sm_count();
    const int exps = 2 * (MATS + 1) * 4;
    int buffers = (p.cluster > 1 || ctas == tiles) ? 1 : 2;
    if (buffers * MATS * p.tn + exps > 512) buffers = 1;
    const int cols = columns(buffers * MATS * p.tn + exps);
    // CTAs that wait for others of their cluster must not wait for tensor memory that CTAs of another cluster hold, which may wait likewise:
    // shared memory in proportion to their columns keeps all that an SM takes in within its 512 columns.
    if (p.cluster > 1 && smem < (size_t)cols * 456) smem = (size_t)cols * 456 < SMEM_LIMIT ? (size_t)cols * 456 : SMEM_LIMIT;
    return launch_cluster("gemm_microscaled", kernel, dim3((unsigned)ctas), THREADS, smem, p.cluster, c.stream, *c.w, *c.w2, *c.x, c.w_exp, c.w2_exp, c.x_exp,
                          c.constants, c.act, c.res, c.n_tok, c.n_feat, c.n_spans, p.cluster, stages, p.tn, buffers, cols, c.status);
}

}  // namespace

// The tensor map of codes [rows, spans * 128] of `bits` (4 or 8) bits, into the 128 bytes at `map_out` (64-byte aligned).  box_rows: 128 for
// a matrix, `ri_mx_box` for rows.
RI_API int ri_mx_encode(void* map_out, const void* ptr, long long rows, int n_spans, int bits, int box_rows) {
    if ((uintptr_t)map_out % 64) return fail("gemm_microscaled: tensor map storage must be 64-byte aligned");
    if (rows <= 0 || n_spans <= 0 || (bits != 4 && bits != 8) || box_rows < 8 || box_rows > 256)
        return fail("gemm_microscaled: no map of [%lld, %d] in %d bits with boxes of %d rows", rows, n_spans, bits, box_rows);
    return encode_codes(reinterpret_cast<CUtensorMap*>(map_out), ptr, rows, n_spans, bits, box_rows);
}

// Rows of the box of a product's X.
RI_API int ri_mx_box(int n_tok, int n_feat, int n_spans) { return plan(n_tok, n_feat, n_spans).tn; }

// `kind`: what is written (`Out`); `dual`: gated, with the second matrix; `act`: `constants` are an activation's.  out_exp, out_spans: with rows in 8 bits.
RI_API int ri_mx_gemm(const void* map_w, const void* map_w2, const void* map_x, const void* w_exp, const void* w2_exp, const void* x_exp,
                      const float* constants, int dual, int act, int kind, void* out, void* out_exp, int out_spans, int n_tok, int n_feat, int n_spans,
                      int* status, cudaStream_t stream) {
    if (n_tok <= 0 || n_feat <= 0) return 0;
    if (n_spans <= 0) return fail("gemm_microscaled: rows without numbers");
    if (kind < OUT_BF16 || kind > OUT_ADD || (dual && act) || (kind == OUT_ADD && (dual || act || constants != nullptr)) || (act && constants == nullptr))
        return fail("gemm_microscaled: no epilogue %d (gated %d, activated %d)", kind, dual, act);
    Call c;
    c.w = reinterpret_cast<const CUtensorMap*>(map_w);
    c.w2 = reinterpret_cast<const CUtensorMap*>(dual ? map_w2 : map_w);
    c.x = reinterpret_cast<const CUtensorMap*>(map_x);
    c.w_exp = (const uint8_t*)w_exp;
    c.w2_exp = (const uint8_t*)w2_exp;
    c.x_exp = (const uint8_t*)x_exp;
    c.constants = constants;
    c.act = act;
    c.res = Result{out, (uint8_t*)out_exp, out_spans};
    c.n_tok = n_tok;
    c.n_feat = n_feat;
    c.n_spans = n_spans;
    c.status = status;
    c.stream = stream;
    if (dual) {
        switch (kind) {
            case OUT_BF16: return launch_feature<true, OUT_BF16>(c);
            case OUT_F32: return launch_feature<true, OUT_F32>(c);
            default: return launch_feature<true, OUT_ROWS>(c);
        }
    }
    switch (kind) {
        case OUT_BF16: return launch_feature<false, OUT_BF16>(c);
        case OUT_F32: return launch_feature<false, OUT_F32>(c);
        case OUT_ROWS: return launch_feature<false, OUT_ROWS>(c);
        default: return launch_feature<false, OUT_ADD>(c);
    }
}

RI_DEFINE_LAST_ERROR()
