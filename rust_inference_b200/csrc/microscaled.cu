// Microscaled numbers (microscaled.cuh) from plain ones and back, and the root-mean-square norm that leaves its result in them.
//
//   ri_mx_hold     a matrix in 4 bits, or rows in 8
//   ri_mx_values   the numbers that either stands for
//   ri_mx_rmsnorm  total = stream + branch;  rows in 8 bits of  total / sqrt(mean(total^2) + eps) * weight
//
// All are bound by memory.  A thread has eight consecutive numbers of a row (16 or 32 bytes in, 4 or 8 out), four neighbouring threads
// a block, whose largest magnitude two exchanges find.
#include "microscaled.cuh"

using namespace ri;
using namespace ri::mx;

namespace {

constexpr int THREADS = 256;

// Eight numbers of a row of k, from column c on; zeros behind its end.  WHOLE: rows are whole 16-byte pieces that begin on a 16-byte boundary.
// (Volatile reads: rows may come from the kernel before, and these stay behind the wait for it.)
template <typename T, bool WHOLE>
__device__ __forceinline__ void load8(const T* row, int c, int k, float* v) {
    if (WHOLE && c < k) {
        if (sizeof(T) == 2) {
            const float4 raw = load_written(reinterpret_cast<const float*>(row + c));
            unpack8(*reinterpret_cast<const uint4*>(&raw), v);
        } else {
            const float4 a = load_written(reinterpret_cast<const float*>(row + c)), b = load_written(reinterpret_cast<const float*>(row + c) + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < k ? to_f32<T>(const_cast<const volatile T*>(row)[c + i]) : 0.f;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16, false>(const __nv_bfloat16* row, int c, int k, float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned short raw = c + i < k ? reinterpret_cast<const volatile unsigned short*>(row)[c + i] : (unsigned short)0;
        v[i] = __uint_as_float((uint32_t)raw << 16);
    }
}

// Eight numbers of one thread, whose block four neighbouring threads hold, to codes and exponent.
template <int BITS>
__device__ __forceinline__ void store8(const float* v, int row, int c, int n_spans, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t four = 0xfu << (threadIdx.x & 28);        // a row's threads come in whole fours, not in whole warps
    top = max(top, __shfl_xor_sync(four, top, 1));
    top = max(top, __shfl_xor_sync(four, top, 2));
    const uint32_t byte = exponent_byte<BITS>(top);
    const float f = to_type(byte);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = v[i] * f;
    const size_t at = (size_t)row * n_spans * SPAN + c;
    if (BITS == 4) {
        *reinterpret_cast<uint32_t*>(codes + at / 2) = four_bits(y);
    } else {
        *reinterpret_cast<uint2*>(codes + at) = make_uint2(eight_bits(y), eight_bits(y + 4));
    }
    if ((c & 31) == 0) exponents[exponent_at(row, c >> 5, n_spans)] = (uint8_t)byte;
}

template <typename T, int BITS, bool WHOLE>
__global__ void __launch_bounds__(THREADS) hold_kernel(const T* x, int k, long long ld, int n_spans, uint32_t groups, uint8_t* codes, uint8_t* exponents) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const uint32_t per_row = n_spans * (SPAN / 8);
    for (uint32_t g = blockIdx.x * THREADS + threadIdx.x; g < groups; g += gridDim.x * THREADS) {
        const int row = (int)(g / per_row), c = (int)(g - (uint32_t)row * per_row) * 8;
        float v[8];
        load8<T, WHOLE>(x + (size_t)row * ld, c, k, v);
        store8<BITS>(v, row, c, n_spans, codes, exponents);
    }
}

template <typename T, int BITS, bool WHOLE>
__global__ void __launch_bounds__(THREADS) values_kernel(const uint8_t* codes, const uint8_t* exponents, int k, int n_spans, uint32_t groups, T* out) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const uint32_t per_row = n_spans * (SPAN / 8);
    for (uint32_t g = blockIdx.x * THREADS + threadIdx.x; g < groups; g += gridDim.x * THREADS) {
        const int row = (int)(g / per_row), c = (int)(g - (uint32_t)row * per_row) * 8;
        if (c >= k) continue;
        const size_t at = (size_t)row * n_spans * SPAN + c;
        const volatile uint32_t* from = reinterpret_cast<const volatile uint32_t*>(codes + (BITS == 4 ? at / 2 : at));
        uint32_t w[2];
        w[0] = from[0];
        if (BITS == 8) w[1] = from[1];
        const float f = from_type(const_cast<const volatile uint8_t*>(exponents)[exponent_at(row, c >> 5, n_spans)]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2_raw h = BITS == 4 ? __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(w[0] >> (8 * i)), __NV_E2M1)
                                            : __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
            const float2 p = __half22float2(__half2(h));
            v[2 * i] = p.x * f;
            v[2 * i + 1] = p.y * f;
        }
        T* to = out + (size_t)row * k + c;
        if (WHOLE) {
            if (sizeof(T) == 2) {
                *reinterpret_cast<uint4*>(to) = pack8(v);
            } else {
                reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
            for (int i = 0; i < 8 && c + i < k; ++i) to[i] = from_f32<T>(v[i]);
        }
    }
}

// A block of threads per row.  Sum of squares, root and factors are in 64 bits: the result is rounded to four bits of mantissa, and what
// lies next to the middle of two numbers should fall as the formula says, not as a sum's last bits do.  (The arithmetic hides behind the
// memory's: see the figures in front of the launch.)  HELD: so many groups of eight per thread stay in registers between the two passes;
// longer rows are read again.
template <typename B, int HELD, bool WHOLE>
__global__ void rmsnorm_kernel(const float* stream, const B* branch, const float* __restrict__ weight, float* total, int k, int n_spans, double eps,
                               uint8_t* codes, uint8_t* exponents) {
    __shared__ double sums[33];
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int row = blockIdx.x, tid = threadIdx.x, threads = blockDim.x, groups = n_spans * (SPAN / 8);
    const float* x = stream + (size_t)row * k;
    const B* add = branch == nullptr ? nullptr : branch + (size_t)row * k;
    float held[HELD][8];
    auto read = [&](int g, float* v) {
        load8<float, WHOLE>(x, g * 8, k, v);
        if (add != nullptr) {
            float b[8];
            load8<B, WHOLE>(add, g * 8, k, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += b[i];
        }
    };
    double sum = 0.0;
    auto square = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fma((double)v[i], (double)v[i], sum);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (tid + h * threads < groups) {
            read(tid + h * threads, held[h]);
            square(held[h]);
        }
    for (int g = tid + HELD * threads; g < groups; g += threads) {
        float v[8];
        read(g, v);
        square(v);
    }
    const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        double s = lane < threads / 32 ? sums[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sums[32] = 1.0 / sqrt(s / (double)k + eps);
    }
    __syncthreads();
    const double r = sums[32];
    auto finish = [&](int g, float* v) {
        const int c = g * 8;
        if (total != nullptr) {
            float* to = total + (size_t)row * k + c;
            if (WHOLE) {
                if (c < k) {
                    reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            } else {
                for (int i = 0; i < 8 && c + i < k; ++i) to[i] = v[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < k ? (float)((double)v[i] * r * (double)weight[c + i]) : 0.f;
        store8<8>(v, row, c, n_spans, codes, exponents);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (tid + h * threads < groups) finish(tid + h * threads, held[h]);
    for (int g = tid + HELD * threads; g < groups; g += threads) {
        float v[8];
        read(g, v);
        finish(g, v);
    }
}

int blocks_for(uint32_t groups) {
    const long long want = ((long long)groups + THREADS - 1) / THREADS, most = 16LL * sm_count();
    return (int)(want < most ? want : most);
}

// Groups of eight numbers of what is held, which must lie on the current device.
int groups_of(const char* what, const Held* h, uint32_t* groups) {
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || device != h->device) return fail("%s: what is held lies on device %d, the current one is %d", what, h->device, device);
    *groups = (uint32_t)((long long)h->n * h->n_spans * (SPAN / 8));
    return 0;
}

template <typename T, int BITS>
int hold(const void* x, int n, int k, long long ld, void* codes, void* exponents, uint32_t groups, cudaStream_t stream) {
    const bool whole = k % 8 == 0 && (ld * (long long)sizeof(T)) % 16 == 0 && (uintptr_t)x % 16 == 0;
    const dim3 grid((unsigned)blocks_for(groups));
    uint8_t *c = (uint8_t*)codes, *e = (uint8_t*)exponents;
    const T* from = (const T*)x;
    return check_launch(whole ? launch_dependent(hold_kernel<T, BITS, true>, grid, dim3(THREADS), 0, stream, from, k, ld, spans(k), groups, c, e)
                              : launch_dependent(hold_kernel<T, BITS, false>, grid, dim3(THREADS), 0, stream, from, k, ld, spans(k), groups, c, e), "mx_hold");
}

template <typename T, int BITS>
int values(const void* codes, const void* exponents, int k, void* out, uint32_t groups, cudaStream_t stream) {
    const bool whole = k % 8 == 0 && (uintptr_t)out % 16 == 0;
    const dim3 grid((unsigned)blocks_for(groups));
    const uint8_t *c = (const uint8_t*)codes, *e = (const uint8_t*)exponents;
    T* to = (T*)out;
    return check_launch(whole ? launch_dependent(values_kernel<T, BITS, true>, grid, dim3(THREADS), 0, stream, c, e, k, spans(k), groups, to)
                              : launch_dependent(values_kernel<T, BITS, false>, grid, dim3(THREADS), 0, stream, c, e, k, spans(k), groups, to), "mx_values");
}

template <typename B>
int norm(const float* x, const void* branch, const float* weight, float* total, int n, int k, double eps, void* codes, void* exponents, cudaStream_t stream) {
    const int groups = spans(k) * (SPAN / 8);
    const bool whole = k % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)branch % 16 == 0 && (uintptr_t)total % 16 == 0;
    constexpr int HELD = 2;
    int threads = ((groups + HELD - 1) / HELD + 31) / 32 * 32;
    if (threads > 512) threads = 512;
    uint8_t *c = (uint8_t*)codes, *e = (uint8_t*)exponents;
    const B* b = (const B*)branch;
    return check_launch(whole ? launch_dependent(rmsnorm_kernel<B, HELD, true>, dim3((unsigned)n), dim3(threads), 0, stream, x, b, weight, total, k, spans(k), eps, c, e)
                              : launch_dependent(rmsnorm_kernel<B, HELD, false>, dim3((unsigned)n), dim3(threads), 0, stream, x, b, weight, total, k, spans(k), eps, c, e),
                        "mx_rmsnorm");
}

}  // namespace

// Bytes of a `Held`, 64-byte aligned.
RI_API long long ri_mx_held_bytes() { return (long long)sizeof(Held); }

// A `Held` at `at`: [n, k] numbers of `bits` bits (4: a matrix, 8: rows) over these buffers of the device `device`.
RI_API int ri_mx_make(void* at, void* codes, void* exponents, long long n, long long k, int bits, int device) {
    if ((uintptr_t)at % 64) return fail("mx_make: 64-byte aligned memory is wanted");
    if (n <= 0 || k <= 0 || k > 0x7fffffffLL - SPAN || (bits != 4 && bits != 8)) return fail("mx_make: no [%lld, %lld] numbers of %d bits", n, k, bits);
    if (n * spans((int)k) > 0x7fffffffLL / (SPAN / 8)) return fail("mx_make: [%lld, %lld] numbers are more than 2^31 eights", n, k);
    if ((uintptr_t)codes % 32 || (uintptr_t)exponents % 32) return fail("mx_make: buffers must begin on a 32-byte boundary");
    Held* h = new (at) Held;
    h->codes = (uint8_t*)codes;
    h->exponents = (uint8_t*)exponents;
    h->n = (int)n;
    h->k = (int)k;
    h->n_spans = spans((int)k);
    h->bits = bits;
    h->device = device;
    h->made.store(0);
    return 0;
}

// x [n, k] (rows `ld` numbers apart) to what is held.
RI_API int ri_mx_hold(const void* x, int dtype, long long n, long long k, long long ld, void* held, cudaStream_t stream) {
    const Held* h = (const Held*)held;
    uint32_t groups;
    if (n != h->n || k != h->k || ld < k) return fail("mx_hold: [%lld, %lld] numbers, rows %lld apart, do not go into [%d, %d]", n, k, ld, h->n, h->k);
    if (int rc = groups_of("mx_hold", h, &groups)) return rc;
    if (dtype == RI_BF16) return h->bits == 4 ? hold<__nv_bfloat16, 4>(x, h->n, h->k, ld, h->codes, h->exponents, groups, stream)
                                              : hold<__nv_bfloat16, 8>(x, h->n, h->k, ld, h->codes, h->exponents, groups, stream);
    return h->bits == 4 ? hold<float, 4>(x, h->n, h->k, ld, h->codes, h->exponents, groups, stream)
                        : hold<float, 8>(x, h->n, h->k, ld, h->codes, h->exponents, groups, stream);
}

// out [n, k]: the numbers that are held.
RI_API int ri_mx_values(const void* held, int dtype, long long n, long long k, void* out, cudaStream_t stream) {
    const Held* h = (const Held*)held;
    uint32_t groups;
    if (n != h->n || k != h->k) return fail("mx_values: [%d, %d] numbers do not go into [%lld, %lld]", h->n, h->k, n, k);
    if (int rc = groups_of("mx_values", h, &groups)) return rc;
    if (dtype == RI_BF16) return h->bits == 4 ? values<__nv_bfloat16, 4>(h->codes, h->exponents, h->k, out, groups, stream)
                                              : values<__nv_bfloat16, 8>(h->codes, h->exponents, h->k, out, groups, stream);
    return h->bits == 4 ? values<float, 4>(h->codes, h->exponents, h->k, out, groups, stream) : values<float, 8>(h->codes, h->exponents, h->k, out, groups, stream);
}

// total = stream + branch (branch null: the stream itself; total null: not kept; it may be the stream), [n, k], and the norm of it times `weight` in 8 bits.
RI_API int ri_mx_rmsnorm(const float* x, const void* branch, int branch_dtype, const float* weight, float* total, long long n, long long k, double eps,
                         void* held, cudaStream_t stream) {
    const Held* h = (const Held*)held;
    uint32_t groups;
    if (n != h->n || k != h->k || h->bits != 8) return fail("mx_rmsnorm: a norm of [%lld, %lld] does not go into [%d, %d] of %d bits", n, k, h->n, h->k, h->bits);
    if (int rc = groups_of("mx_rmsnorm", h, &groups)) return rc;
    return branch_dtype == RI_BF16 ? norm<__nv_bfloat16>(x, branch, weight, total, h->n, h->k, eps, h->codes, h->exponents, stream)
                                   : norm<float>(x, branch, weight, total, h->n, h->k, eps, h->codes, h->exponents, stream);
}

RI_DEFINE_LAST_ERROR()
