// Log probabilities of given tokens, the entropy of the distribution they come from, and its likeliest tokens.
//
// For a row x of logits, with m = max x, z = sum exp(x_i - m) and t = sum exp(x_i - m) (x_i - m):
//   logprob(i) = x_i - m - ln z,   entropy = ln z - t / z.
// Banned tokens (logits of minus infinity) have probability 0 and add nothing.  A row with a NaN or plus infinity, or with
// nothing but minus infinity, has no distribution: all of its results are NaN.  The likeliest tokens are the largest logits in
// descending order, ties in the order of the ids (NaN before all).  A target outside the vocabulary (-1: none) has the log
// probability NaN.
#include "common.cuh"

using namespace ri;

namespace {

constexpr int THREADS = 1024;

// The order of the alternatives as one number: larger logits first, the lower id among equals (0 and -0 are equal)
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
    unsigned u = __float_as_uint(x + 0.f);
    u = x != x ? 0xffffffffu : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned)~id;
}

__device__ __forceinline__ unsigned long long block_max64(unsigned long long v, unsigned long long* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = threadIdx.x < (blockDim.x >> 5) ? scratch[threadIdx.x] : 0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
            v = w > v ? w : v;
        }
        if (threadIdx.x == 0) scratch[32] = v;
    }
    __syncthreads();
    return scratch[32];
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
logprobs_kernel(const T* __restrict__ logits, long long ld, int vocab, const int* __restrict__ targets, int top, float* __restrict__ logprob,
                float* __restrict__ entropy, int* __restrict__ top_ids, float* __restrict__ top_logprobs) {
    __shared__ float scratch[33];
    __shared__ unsigned long long scratch64[33];
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int row = blockIdx.x;
    const T* x = logits + (size_t)row * ld;
    float m = -INFINITY;
    bool bad = false;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float v = to_f32<T>(x[i]);
        bad |= v != v;
        m = fmaxf(m, v);
    }
    m = block_max(m, scratch);
    bad = __syncthreads_or(bad);
    float z = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float d = fmaxf(to_f32<T>(x[i]) - m, -1000.f), e = expf(d);      // (banned: e = 0, and e d too)
        z += e;
        t = fmaf(e, d, t);
    }
    z = block_sum(z, scratch);
    t = block_sum(t, scratch);
    const float nan = __int_as_float(0x7fffffff);
    bad |= !(fabsf(m) < INFINITY);
    const float lz = bad ? nan : logf(z);
    if (threadIdx.x == 0) {
        const int id = targets[row];
        logprob[row] = id >= 0 && id < vocab ? to_f32<T>(x[id]) - m - lz : nan;
        entropy[row] = lz - t / z;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long best = 0ull;
        for (int i = threadIdx.x; i < vocab; i += THREADS) {
            const unsigned long long key = rank_key(to_f32<T>(x[i]), i);
            if ((k == 0 || key < last) && key > best) best = key;
        }
        last = block_max64(best, scratch64);
        if (threadIdx.x == 0) {
            const int id = (int)~(unsigned)last;
            top_ids[(size_t)row * top + k] = id;
            top_logprobs[(size_t)row * top + k] = to_f32<T>(x[id]) - m - lz;
        }
    }
}

}  // namespace

// logits [rows] of `vocab` numbers, `ld` apart; targets [rows]; top_ids, top_logprobs [rows, top] (top 0: not written)
RI_API int ri_token_logprobs(const void* logits, int dtype, long long ld, int rows, int vocab, const int* targets, int top, float* logprob,
                             float* entropy, int* top_ids, float* top_logprobs, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || top < 0 || top > vocab) return fail("token_logprobs: %d alternatives of %d tokens", top, vocab);
    auto launch = [&](auto kernel, auto* x) {
        return check_launch(launch_dependent(kernel, dim3((unsigned)rows), dim3(THREADS), 0, stream, x, ld, vocab, targets, top, logprob,
                                             entropy, top_ids, top_logprobs), "token_logprobs");
    };
    if (dtype == RI_F32) return launch(logprobs_kernel<float>, (const float*)logits);
    if (dtype == RI_BF16) return launch(logprobs_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits);
    return fail("token_logprobs: unknown dtype %d", dtype);
}

RI_DEFINE_LAST_ERROR()
