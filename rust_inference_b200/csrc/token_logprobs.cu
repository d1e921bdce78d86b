// Log probabilities of given tokens, the entropy of the distribution they come from, and its likeliest tokens.
//
// For a row x of logits, with m = max x, z = sum exp(x_i - m) and t = sum exp(x_i - m) (x_i - m):
//   logprob(i) = x_i - m - ln z,   entropy = ln z - t / z.
// Banned tokens (logits of minus infinity) have probability 0 and add nothing.  A row with a NaN or plus infinity, or with
// nothing but minus infinity, has no distribution: all of its results are NaN.  The likeliest tokens are the largest logits in
// descending order, ties in the order of the ids (NaN before all).  A target outside the vocabulary (-1: none) has the log
// probability NaN.
//
// One pass over the row: every thread keeps the maximum of its elements, sixteen bytes at a time, and z and t against a reference
// that moves up with it (m -> m': z' = z a, t' = a (t + z (m - m')), a = exp(m - m')); all of it is float32.
//
// The likeliest `top` tokens without a second pass: four neighbouring threads are a group.  With tau the top-th largest of
// the groups' maxima, at least `top` elements are tau or more, and all of those lie in groups whose maximum is.  Those are about
// `top` groups of 1/128 of a block's part of the row; only they are read again, out of the L2 cache, and the few elements above
// tau, with those equal to it, are put in order by counting.  (Where blocks share a row, tau is taken from 128 maxima too, each
// of a group of every block.)
//
// A row belongs to one block of 512 threads, or, where few rows are long, to a cluster of up to 8, which read each
// other's sums and maxima through distributed shared memory and put their candidates into the first block's.  What bounds
// many rows is memory: 2,047 rows of 152,064 in float32 212 us, 5.9 TB/s, 90% of what a copy reaches.  One row takes what its
// meetings and the few dependent reads take (151,936: 4.1 us, 6.1 with the five likeliest).
#include "cluster.cuh"

#include <float.h>

#include <atomic>

using namespace ri;

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, GROUP = 4, GROUPS = THREADS / GROUP, MOST_TOP = 64, MOST_BLOCKS = 8;
constexpr int ROOM = 1024;                       // elements above tau, and equal to it, that a block's lists hold
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Sums { float m, z, t; };                  // t in units of log2

__device__ __forceinline__ float two_to(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void raise(Sums& s, float m) {
    const float d = (s.m - m) * LOG2E, a = two_to(d);
    s.t = a * fmaf(s.z, fmaxf(d, -1000.f), s.t);
    s.z *= a;
    s.m = m;
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    a.z += b.z;
    a.t += b.t;
    return a;
}
__device__ __forceinline__ void add(Sums& s, float x) {                // s.m is x or more
    const float d = (x - s.m) * LOG2E, e = two_to(d);
    s.z += e;
    s.t = fmaf(e, fmaxf(d, -1000.f), s.t);       // (banned: e = 0; a NaN stays one through e)
}

// sixteen bytes that an earlier kernel writes (see load_written), not kept in L1
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float load1(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float load1(const __nv_bfloat16* p) {
    unsigned short v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
    return __uint_as_float((uint32_t)v << 16);
}
template <typename T> struct Piece;              // sixteen bytes of logits
template <> struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void open(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float most(const uint4& v) {             // (a NaN is left out)
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void open(const uint4& v, float* f) { unpack8(v, f); }
    static __device__ __forceinline__ float most(const uint4& v) {
        const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
        const float2 m = __bfloat1622float2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
        return fmaxf(m.x, m.y);
    }
};

// Larger logits first: whole numbers in their order (0 and -0 are equal, NaN before all)
__device__ __forceinline__ unsigned order(float x) {
    const unsigned u = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ float ordered(unsigned u) {                  // ... and back
    return __uint_as_float(u == 0xffffffffu ? 0x7fffffffu : ((u & 0x80000000u) ? u ^ 0x80000000u : ~u));
}

__device__ __forceinline__ const void* peer(const void* own, int rank) {           // a place in a peer's shared memory
    uint64_t there;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(there) : "l"(own), "r"(rank));
    return reinterpret_cast<const void*>(there);
}

struct __align__(16) Lists {
    unsigned long long found[WARPS];
    unsigned every[GROUPS];                      // the largest of the groups' maxima in the row's blocks
    Sums sums[WARPS];
    Sums block;                                  // of this block's part of the row
    unsigned most[GROUPS];                       // the groups' maxima, in their order
    float m, log_z;                              // of the whole row; log_z NaN: no distribution
    int votes[WARPS];
    unsigned tau;
    int above_n, equal_n, groups_n;
    unsigned above_x[ROOM];
    int above_id[ROOM], equal_id[ROOM], group[GROUPS];
};

// The whole row, ordered by x and id, from the largest on, by one block and one pass per token: where the lists do not hold what is
// above tau (rows whose large logits lie in a few of the groups).
template <typename T>
__device__ void one_by_one(const T* x, int vocab, int top, float m, float log_z, int* ids, float* best, unsigned long long* scratch) {
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long found = 0ull;
        for (int i = threadIdx.x; i < vocab; i += THREADS) {
            const unsigned long long key = ((unsigned long long)order(load1(x + i)) << 32) | (unsigned)~i;
            if ((k == 0 || key < last) && key > found) found = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long w = __shfl_xor_sync(0xffffffffu, found, o);
            found = w > found ? w : found;
        }
        __syncthreads();
        if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = found;
        __syncthreads();
        last = 0ull;
        for (int w = 0; w < WARPS; ++w) last = scratch[w] > last ? scratch[w] : last;
        if (threadIdx.x == 0) {
            const int id = (int)~(unsigned)last;
            ids[k] = id;
            best[k] = load1(x + id) - m - log_z;
        }
    }
}

// PER_SM: blocks that an SM holds
template <typename T, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM)
logprobs_kernel(const T* logits, long long ld, int vocab, const int* targets, int top, float* __restrict__ logprob, float* __restrict__ entropy,
                int* __restrict__ top_ids, float* __restrict__ top_logprobs, int blocks) {
    constexpr int N = Piece<T>::N, AT_ONCE = 4;
    __shared__ Lists s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blocks > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / blocks;
    let_next_kernel_start();
    const T* x = logits + (size_t)row * ld;
    // this block's part of the row, cut at 16-byte boundaries of memory: a head of single elements, pieces, a tail
    const int skew = (int)(((16 - (uintptr_t)x % 16) % 16) / sizeof(T));              // elements before the first boundary
    const int first = min(skew, vocab), pieces = (vocab - first) / N;
    const int p0 = (int)((long long)pieces * rank / blocks), p1 = (int)((long long)pieces * (rank + 1) / blocks);
    const int singles = rank == 0 ? vocab - pieces * N : 0;                            // head and tail, the first block's
    auto single = [&](int i) { return i < first ? i : i + pieces * N; };               // the i-th of them
    const T* body = x + first;
    if (tid == 0) s.above_n = s.equal_n = s.groups_n = 0;
    wait_for_previous_kernels();

    float wanted = 0.f;                          // the target's logit, by the thread that will want it
    if (rank == 0 && tid == THREADS - 32) {
        const int id = targets[row];
        if (id >= 0 && id < vocab) wanted = load1(x + id);
    }
    Sums mine = {-FLT_MAX, 0.f, 0.f};            // (a finite reference: minus infinity less it is minus infinity)
    float most = -INFINITY;
    auto get = [&](uint4 (&v)[AT_ONCE], int p) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
            if (p + k * THREADS < p1) v[k] = load16(body + (size_t)(p + k * THREADS) * N);
    };
    auto take = [&](const uint4 (&v)[AT_ONCE], int p) {
        float higher = -INFINITY;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
            if (p + k * THREADS < p1) higher = fmaxf(higher, Piece<T>::most(v[k]));
        most = fmaxf(most, higher);
        if (higher > mine.m) raise(mine, higher);
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (p + k * THREADS >= p1) break;
            float f[N];
            Piece<T>::open(v[k], f);
#pragma unroll
            for (int i = 0; i < N; ++i) add(mine, f[i]);
        }
    };
    constexpr int TURN = AT_ONCE * THREADS;
    uint4 v[AT_ONCE];
    if (PER_SM == 2) {                           // the next pieces are on their way while these are worked on
        uint4 w[AT_ONCE];
        int p = p0 + tid;
        get(v, p);
        for (; p < p1; p += 2 * TURN) {
            get(w, p + TURN);
            take(v, p);
            get(v, p + 2 * TURN);
            take(w, p + TURN);
        }
    } else {
        for (int p = p0 + tid; p < p1; p += TURN) {
            get(v, p);
            take(v, p);
        }
    }
    for (int i = tid; i < singles; i += THREADS) {
        const float f = load1(x + single(i));
        most = fmaxf(most, f);
        if (f > mine.m) raise(mine, f);
        add(mine, f);
    }
    unsigned key = order(most);
    if (mine.z != mine.z) {                      // a NaN (or an infinity less itself): maxima leave NaN out, the order does not
        for (int p = p0 + tid; p < p1; p += THREADS)
            for (int i = 0; i < N; ++i) key = max(key, order(load1(body + (size_t)p * N + i)));
        for (int i = tid; i < singles; i += THREADS) key = max(key, order(load1(x + single(i))));
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        if (o < GROUP) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        const Sums other = {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.z, o), __shfl_xor_sync(0xffffffffu, mine.t, o)};
        mine = joined(mine, other);
    }
    if (lane == 0) s.sums[warp] = mine;
    if (tid % GROUP == 0) s.most[tid / GROUP] = key;
    __syncthreads();
    if (tid < 32) {
        Sums all = tid < WARPS ? s.sums[tid] : Sums{-FLT_MAX, 0.f, 0.f};
#pragma unroll
        for (int o = 1; o < WARPS; o <<= 1) {
            const Sums other = {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.z, o), __shfl_xor_sync(0xffffffffu, all.t, o)};
            all = joined(all, other);
        }
        if (tid == 0) s.block = all;
    }
    if (blocks > 1) cluster_sync();
    else __syncthreads();
    // ---- the last warp: the row's sums; the others: tau, the top-th largest of the groups' maxima ----
    if (warp == WARPS - 1) {
        Sums all = {-FLT_MAX, 0.f, 0.f};
        if (lane < blocks) all = blocks > 1 ? *reinterpret_cast<const Sums*>(peer(&s.block, lane)) : s.block;
#pragma unroll
        for (int o = 1; o < MOST_BLOCKS; o <<= 1) {
            const Sums other = {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.z, o), __shfl_xor_sync(0xffffffffu, all.t, o)};
            all = joined(all, other);
        }
        if (lane == 0) {
            // no distribution: an infinite maximum, a NaN among the sums, nothing but banned tokens
            const bool none = !(all.m < INFINITY) || !(all.z > 0.f);
            s.m = all.m;
            s.log_z = none ? __int_as_float(0x7fffffff) : logf(all.z);
            if (rank == 0) {
                const int id = targets[row];
                logprob[row] = (id >= 0 && id < vocab ? wanted : __int_as_float(0x7fffffff)) - all.m - s.log_z;
                entropy[row] = s.log_z - all.t * LN2 / all.z;
            }
        }
    }
    if (top == 0) {
        if (blocks > 1) cluster_sync();          // a peer may still be reading this block's sums
        return;
    }
    if (tid < GROUPS) {
        unsigned most_of[MOST_BLOCKS];           // all reads at once
#pragma unroll
        for (int b = 0; b < MOST_BLOCKS; ++b)
            most_of[b] = b == 0 && blocks == 1 ? s.most[tid] : (b < blocks ? *reinterpret_cast<const unsigned*>(peer(s.most + tid, b)) : 0u);
        unsigned largest = most_of[0];
#pragma unroll
        for (int b = 1; b < MOST_BLOCKS; ++b) largest = max(largest, most_of[b]);
        s.every[tid] = largest;
    }
    __syncthreads();
    {                                            // a maximum's place: how many are larger, or as large and earlier (four threads for each)
        const int k = tid / 4, quarter = tid % 4 * (GROUPS / 4);
        const unsigned mine = s.every[k];
        int before = 0;
#pragma unroll
        for (int i = 0; i < GROUPS / 4; i += 4) {
            const int o = quarter + (i + 4 * (tid % 4)) % (GROUPS / 4);        // (the four in different banks)
            const uint4 u = *reinterpret_cast<const uint4*>(s.every + o);
            before += (u.x > mine || (u.x == mine && o < k)) + (u.y > mine || (u.y == mine && o + 1 < k)) +
                      (u.z > mine || (u.z == mine && o + 2 < k)) + (u.w > mine || (u.w == mine && o + 3 < k));
        }
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        if (tid % 4 == 0 && before == top - 1) s.tau = mine;
    }
    __syncthreads();
    const unsigned tau = s.tau;

    // ---- what is above it, and equal to it, in the groups that have any ----
    if (tid < GROUPS && s.most[tid] >= tau) s.group[atomicAdd(&s.groups_n, 1)] = tid;
    __syncthreads();
    Lists& lists = blocks > 1 ? *const_cast<Lists*>(reinterpret_cast<const Lists*>(peer(&s, 0))) : s;       // the first block's
    auto look = [&](float f, int id) {
        const unsigned u = order(f);
        if (u < tau) return;
        if (u > tau) {
            const int at = atomicAdd(&lists.above_n, 1);
            if (at < ROOM) lists.above_x[at] = u, lists.above_id[at] = id;
        } else {
            const int at = atomicAdd(&lists.equal_n, 1);
            if (at < ROOM) lists.equal_id[at] = id;
        }
    };
    constexpr int RUN = GROUP * N;               // neighbouring elements of a group
    for (int i = warp; i < s.groups_n; i += WARPS) {
        const int g = s.group[i];
        // 32 / RUN runs at a time, one element per lane
        const int turn = lane / RUN, within = lane % RUN;
        for (int p = p0 + g * GROUP + turn * THREADS; p < p1; p += 8 * (32 / RUN) * THREADS) {
            float f[8];
            bool there[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int piece = p + k * (32 / RUN) * THREADS + within / N;
                there[k] = piece < p1;
                if (there[k]) f[k] = load1(body + (size_t)piece * N + within % N);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int piece = p + k * (32 / RUN) * THREADS + within / N;
                if (there[k]) look(f[k], first + piece * N + within % N);
            }
        }
    }
    for (int i = tid; i < singles; i += THREADS) look(load1(x + single(i)), single(i));
    if (blocks > 1) cluster_sync();
    else __syncthreads();

    if (rank == 0) {
        // ---- the first block puts them in order ----
        const int above = s.above_n, equal = s.equal_n;
        const bool held = above <= ROOM, ties = equal <= ROOM;         // all that is above; all that is equal
        const float m = s.m, log_z = s.log_z;
        int* ids = top_ids + (size_t)row * top;
        float* best = top_logprobs + (size_t)row * top;
        const float equal_value = ordered(tau) - m - log_z;
        if (!held) {
            one_by_one<T>(x, vocab, top, m, log_z, ids, best, s.found);
        } else {
            for (int i = tid; i < above; i += THREADS) {
                const unsigned u = s.above_x[i];
                const int id = s.above_id[i];
                int place = 0;
                for (int o = 0; o < above; ++o) place += s.above_x[o] > u || (s.above_x[o] == u && s.above_id[o] < id);
                if (place < top) ids[place] = id, best[place] = ordered(u) - m - log_z;
            }
            if (above < top && ties) {
                for (int i = tid; i < equal; i += THREADS) {
                    const int id = s.equal_id[i];
                    int place = above;
                    for (int o = 0; o < equal; ++o) place += s.equal_id[o] < id;
                    if (place < top) ids[place] = id, best[place] = equal_value;
                }
            } else if (above < top) {            // more of them than the list holds (banned tokens, for one): the lowest ids, in their order
                for (int from = 0, place = above; place < top && from < vocab; from += THREADS) {
                    const bool is = from + tid < vocab && order(load1(x + from + tid)) == tau;
                    const unsigned votes = __ballot_sync(0xffffffffu, is);
                    __syncthreads();
                    if (lane == 0) s.votes[warp] = __popc(votes);
                    __syncthreads();
                    int at = place + __popc(votes & ((1u << lane) - 1u));
                    for (int w = 0; w < WARPS; ++w) {
                        if (w < warp) at += s.votes[w];
                        place += s.votes[w];
                    }
                    if (is && at < top) ids[at] = from + tid, best[at] = equal_value;
                }
            }
        }
    }
    // (the first block reads its own lists only: the others may leave)
}

// How many clusters of so many blocks the device holds at once: they lie within groups of SMs, some of which they leave over.  Asked once.
template <typename T>
int clusters_held(int blocks) {
    static std::atomic<int> known[64][MOST_BLOCKS + 1];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    n = known[dev][blocks].load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)blocks);
        cfg.blockDim = dim3(THREADS);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)blocks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, logprobs_kernel<T, 2>, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = 1;
        }
        known[dev][blocks].store(n, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace

// logits [rows] of `vocab` numbers, `ld` apart; targets [rows]; top_ids, top_logprobs [rows, top] (top 0: not written)
RI_API int ri_token_logprobs(const void* logits, int dtype, long long ld, int rows, int vocab, const int* targets, int top, float* logprob,
                             float* entropy, int* top_ids, float* top_logprobs, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || top < 0 || top > vocab || top > MOST_TOP) return fail("token_logprobs: %d alternatives of %d tokens", top, vocab);
    // Blocks per row: what a block does beside its part of the row, and clusters that wait for one another, have to be paid by shorter
    // parts.  So parts of 8,192 logits or more where the blocks leave half of the SMs alone, of 24,000 or more up to as many clusters as the
    // SMs hold at once (a cluster more costs a second round).  With 1, 2, 4 and 8, us, and the five likeliest, bfloat16:
    //   vocabulary 128,256:  1 row 12.8, 9.4, 6.9, 6.2;  48 rows 13.2, 10.5, 10.1, 15.2;  90 rows 18.5, 14.1, 14.8, 23.4;  148 rows 15.2, 14.7, 23.2, 37.1
    //   vocabulary 32,000:   1 row 6.1, 6.1, 5.8, 5.5;   48 rows 6.4, 7.1, 7.5, 12.6;     90 rows 7.9, 8.3, 13.3, 19.4;    148 rows 6.5, 8.7, 17.5, 30.2
    const bool f32 = dtype == RI_F32;
    int blocks = 1;
    for (int b = 2; b <= MOST_BLOCKS; ++b)
        if ((2ll * rows * b <= sm_count() && vocab >= 8192 * b) || (vocab >= 24000 * b && rows <= (f32 ? clusters_held<float>(b) : clusters_held<__nv_bfloat16>(b))))
            blocks = b;
    if ((long long)rows * blocks > 0x7fffffff) return fail("token_logprobs: %d rows are too many", rows);
    auto launch = [&](auto kernel, auto* x) {
        return launch_cluster("token_logprobs", kernel, dim3((unsigned)(rows * blocks)), THREADS, 0, blocks, stream, x, ld, vocab, targets, top,
                              logprob, entropy, top_ids, top_logprobs, blocks);
    };
    // Two blocks per SM whose threads fetch while they work, or, where the rows are more than those, three that do not (their registers
    // hold one turn), us with the five likeliest: vocabulary 151,936, float32, 61 rows 11.9 and 14.0, 148 rows 20.8 and 24.6, 300 rows 49.7 and
    // 39.5, 2,047 rows (the likeliest) 224 and 212.
    const bool many = rows > 2 * sm_count();
    if (dtype == RI_F32) return many ? launch(logprobs_kernel<float, 3>, (const float*)logits) : launch(logprobs_kernel<float, 2>, (const float*)logits);
    if (dtype == RI_BF16) return many ? launch(logprobs_kernel<__nv_bfloat16, 3>, (const __nv_bfloat16*)logits) : launch(logprobs_kernel<__nv_bfloat16, 2>, (const __nv_bfloat16*)logits);
    return fail("token_logprobs: unknown dtype %d", dtype);
}

RI_DEFINE_LAST_ERROR()
