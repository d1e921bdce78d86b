// Microscaled numbers (microscaled.cuh) from plain ones and back, and the root-mean-square norm that leaves its result in them.
//
//   ri_mx_hold     a matrix in 4 bits, or rows in 8
//   ri_mx_values   the numbers that either stands for
//   ri_mx_rmsnorm  total = stream + branch;  rows in 8 bits of  total / sqrt(mean(total^2) + eps) * weight
//
// All are bound by memory: [3584, 18944] from bfloat16 to 4 bits 36.5 us (4.7 TB/s), back 31.9 (5.4); the norm of 2,047 rows of 4,096 with a bfloat16
// branch and the total 22 us (4.1; reading, one sum, writing, 3.5 rounds of blocks), without them 17.0, of one row of 896 1.5, of 8 of 3,584 2.4: trips.
// A thread has eight consecutive numbers of a row (16 or 32 bytes in, 4 or 8 out), four neighbouring threads a block, whose largest magnitude two
// exchanges find.
#include "microscaled.cuh"

using namespace ri;
using namespace ri::mx;

namespace {

constexpr int THREADS = 256;

// Eight consecutive numbers of a row.  WHOLE: rows are whole eights that begin on a 16-byte boundary.  (Reads that stay behind the wait for the
// kernel before, which may have written them.)
template <int BYTES> struct Sized { using type = uint32_t; };
template <> struct Sized<2> { using type = uint16_t; };
template <typename T> struct Eight;
template <> struct alignas(16) Eight<float> {
    float v[8];
    // from column c on of a row of k, in whole eights on 16-byte boundaries; zeros behind its end
    __device__ __forceinline__ void load(const float* row, int c, int k) {
        if (c < k) {
            const float4 a = load_written(row + c), b = load_written(row + c + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
    }
    // the largest magnitude, as a float's bits (a NaN's are larger than any number's)
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
        return t;
    }
    __device__ __forceinline__ void scaled(uint32_t byte, float* y) const {          // times 2^-e
        const float f = to_type(byte);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[i] * f;
    }
};
template <> struct alignas(16) Eight<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* row, int c, int k) {
        if (c < k) {
            const float4 a = load_written(reinterpret_cast<const float*>(row + c));
            w[0] = __float_as_uint(a.x); w[1] = __float_as_uint(a.y); w[2] = __float_as_uint(a.z); w[3] = __float_as_uint(a.w);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = 0u;
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) t = __vmaxu2(t, w[i] & 0x7fff7fffu);
        return max(t << 16, t & 0xffff0000u);
    }
    __device__ __forceinline__ void scaled(uint32_t byte, float* y) const {          // (a product that is no normal number any more is 0 in either type)
        const __nv_bfloat162 f = to_type_bf162(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t p = as_word(__hmul2(as_bf162(w[i]), f));
            y[2 * i] = __uint_as_float(p << 16);
            y[2 * i + 1] = __uint_as_float(p & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void add_to(float* v) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] += __uint_as_float(w[i] << 16);
            v[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// The largest of a block's four threads.
__device__ __forceinline__ uint32_t block_top(uint32_t top) {
    const uint32_t four = 0xfu << (threadIdx.x & 28);        // a row's threads come in whole fours, not in whole warps
    top = max(top, __shfl_xor_sync(four, top, 1));
    return max(top, __shfl_xor_sync(four, top, 2));
}

// Rows that are no whole eights on 16-byte boundaries: a warp reads (and writes) 32 neighbouring numbers at a time, eight times, and they change places
// in its part of shared memory, `room`, so that each thread has eight in a row.  ([3584, 18945] bfloat16 to 4 bits 71 -> 51 us and back 193 -> 40;
// the norm of 2,047 rows of 4,097 56 -> 34 us.)
template <typename T> using Bits = typename Sized<sizeof(T)>::type;
template <typename T>
__device__ __forceinline__ void read_apart(const T* row, int c, int k, Bits<T>* raw) {                // c: the first of this thread's numbers
#pragma unroll
    for (int q = 0; q < 8; ++q) raw[q] = c + q * 32 < k ? reinterpret_cast<const volatile Bits<T>*>(row)[c + q * 32] : (Bits<T>)0;
}
template <typename T>
__device__ __forceinline__ void gather(Bits<T>* room, int lane, const Bits<T>* raw, Eight<T>& v) {
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) room[q * 32 + lane] = raw[q];
    __syncwarp();
    v = *reinterpret_cast<const Eight<T>*>(room + lane * 8);
}

// A warp takes a part of a row, GROUPS times 256 numbers, whose reads are on their way together: four where there is much to do, else one.
template <typename T, int BITS, bool WHOLE, int GROUPS>
__global__ void __launch_bounds__(THREADS) hold_kernel(const T* x, int n, int k, long long ld, int n_spans, uint32_t parts, uint32_t items, uint8_t* codes,
                                                       uint8_t* exponents) {
    __shared__ alignas(16) Bits<T> room[WHOLE ? 1 : THREADS / 32][256];
    if (BITS == 8) let_next_kernel_start();                 // (a matrix: see `settle`)
    wait_for_previous_kernels();
    const int lane = threadIdx.x & 31;
    for (uint32_t it = (blockIdx.x * THREADS + threadIdx.x) >> 5; it < items; it += gridDim.x * (THREADS / 32)) {
        const int row = (int)(it / parts), c0 = (int)(it - (uint32_t)row * parts) * (GROUPS * 256) + lane * 8, width = n_spans * SPAN;
        uint8_t* to = codes + code_at<BITS>(row, c0, n_spans);                       // (256 numbers further on: two tiles, or 256 bytes)
        uint8_t* exp_to = exponents + exponent_at(row, c0 >> 5, n_spans);           // (two pieces)
        if (BITS == 4 && row >= n) {               // of a matrix's last 128 rows those that are none
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                if (c0 + i * 256 >= width) break;
                *reinterpret_cast<uint32_t*>(to + i * 2 * 128 * (SPAN / 2)) = 0u;
                if ((lane & 3) == 0) exp_to[i * 2 * PIECE] = 0;
            }
            continue;
        }
        const T* from = x + (size_t)row * ld;
        Eight<T> v[GROUPS];
        if (WHOLE) {
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) v[i].load(from, c0 + i * 256, k);
        } else {
            Bits<T> raw[GROUPS][8];
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) read_apart(from, c0 - lane * 7 + i * 256, k, raw[i]);
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) gather(room[threadIdx.x >> 5], lane, raw[i], v[i]);
        }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            if (c0 + i * 256 >= width) break;
            const uint32_t byte = exponent_byte<BITS>(block_top(v[i].top()));
            float y[8];
            v[i].scaled(byte, y);
            if (BITS == 4) *reinterpret_cast<uint32_t*>(to + i * 2 * 128 * (SPAN / 2)) = four_bits(y);
            else *reinterpret_cast<uint2*>(to + i * 256) = make_uint2(eight_bits(y), eight_bits(y + 4));
            if ((lane & 3) == 0) exp_to[i * 2 * PIECE] = (uint8_t)byte;
        }
    }
}

// The same for reading back, a thread 16 bytes of the result at a time.
template <typename T> struct Sixteen { static constexpr int N = 16 / sizeof(T); };

template <typename T, int BITS, bool WHOLE, int GROUPS>
__global__ void __launch_bounds__(THREADS) values_kernel(const uint8_t* codes, const uint8_t* exponents, int k, int n_spans, uint32_t parts, uint32_t items, T* out) {
    constexpr int N = Sixteen<T>::N, BYTES = N * BITS / 8;          // numbers of a thread, and bytes of their codes: 2, 4 or 8
    __shared__ alignas(16) Bits<T> room[WHOLE ? 1 : THREADS / 32][32 * N];
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int lane = threadIdx.x & 31;
    for (uint32_t it = (blockIdx.x * THREADS + threadIdx.x) >> 5; it < items; it += gridDim.x * (THREADS / 32)) {
        const int row = (int)(it / parts), c0 = (int)(it - (uint32_t)row * parts) * (GROUPS * 32 * N) + lane * N;
        const volatile uint8_t* at = codes + code_at<BITS>(row, c0, n_spans);
        const volatile uint8_t* exp_at = exponents + exponent_at(row, c0 >> 5, n_spans);      // (32 N numbers further on: one or two pieces)
        T* to = out + (size_t)row * k + c0;
        uint32_t w[GROUPS][2] = {}, byte[GROUPS] = {};
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            if (c0 + i * 32 * N >= k) break;
            const volatile uint8_t* from = at + (BITS == 4 ? i * (N / 4) * 128 * (SPAN / 2) : i * 32 * BYTES);
            if (BYTES == 2) w[i][0] = *reinterpret_cast<const volatile uint16_t*>(from);
            else w[i][0] = *reinterpret_cast<const volatile uint32_t*>(from);
            if (BYTES == 8) w[i][1] = *reinterpret_cast<const volatile uint32_t*>(from + 4);
            byte[i] = exp_at[i * (N / 4) * PIECE];
        }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int c = c0 + i * 32 * N;
            if ((WHOLE ? c : c - lane * N) >= k) break;
            __nv_bfloat162 v[N / 2];
#pragma unroll
            for (int q = 0; q < N / 2; ++q)
                v[q] = BITS == 4 ? four_to_bf162((w[i][0] >> (8 * q) & 0xffu) * 0x1001u) : eight_to_bf162(__byte_perm(w[i][q >> 1], 0, q & 1 ? 0x4342 : 0x4140));
            uint4 r;
            uint32_t* p = reinterpret_cast<uint32_t*>(&r);
            if (sizeof(T) == 2) {
                const __nv_bfloat162 f = from_type_bf162(byte[i]);
#pragma unroll
                for (int q = 0; q < N / 2; ++q) p[q] = as_word(__hmul2(v[q], f));
            } else {
                const float f = from_type(byte[i]);
#pragma unroll
                for (int q = 0; q < N / 2; ++q) {
                    p[2 * q] = __float_as_uint(__low2float(v[q]) * f);
                    p[2 * q + 1] = __float_as_uint(__high2float(v[q]) * f);
                }
            }
            T* dst = to + i * 32 * N;
            if (WHOLE) {
                *reinterpret_cast<uint4*>(dst) = r;
            } else {
                __syncwarp();
                *reinterpret_cast<uint4*>(&room[threadIdx.x >> 5][lane * N]) = r;
                __syncwarp();
                Bits<T>* line = reinterpret_cast<Bits<T>*>(dst) - lane * N;
#pragma unroll
                for (int q = 0; q < N; ++q)
                    if (c - lane * N + q * 32 + lane < k) line[q * 32 + lane] = room[threadIdx.x >> 5][q * 32 + lane];
            }
        }
    }
}

// A double as the float towards zero, its last bit set where that is not the double: rounded again to fewer bits it becomes what the double would.
__device__ __forceinline__ uint32_t to_odd(double y) {
    const float f = __double2float_rz(y);
    const uint32_t bits = __float_as_uint(f);
    if (fabs(y) >= 0x1p128) return (bits & 0x80000000u) | 0x7f800000u;
    return bits | ((double)f != y ? 1u : 0u);            // (a NaN too)
}

// A block of threads per row.  Results are what the formula in 64 bits, rounded once, gives: what lies next to the middle of two numbers falls as the
// formula says, not as a sum's last bits do.  The sum of squares and its root are in 64 bits; factors too, but only where 32 leave it open (32 bits
// throughout: 2,047 rows of 4,096 without a branch 17.0 -> 14.8 us, with branch and total 22.1 -> 21.4; 8 of 3,584 2.4 -> 2.0, of which the sum and its root are
// 0.15 and the factors 0.2; one of 896 1.5 -> 1.35.  Beside that the exchanges that find a block's largest are 0.1 to 0.2.  Into bfloat16 the same rows take
// 12.4, 1.5 and 1.1).  HELD: so many groups of eight per thread stay in
// registers between the two passes; longer rows are read again.
template <typename B, int HELD, bool WHOLE>
__global__ void __launch_bounds__(HELD == 1 ? 1024 : 512, HELD == 1 ? 1 : 2) rmsnorm_kernel(const float* stream, const B* branch, const float* __restrict__ weight, float* total, int k,
                                                                                            int n_spans, double inverse, double eps, uint8_t* codes,
                                                                                            uint8_t* exponents) {
    __shared__ double sums[32];
    __shared__ alignas(16) uint32_t rooms[WHOLE ? 1 : HELD == 1 ? 32 : 16][256];
    constexpr uint32_t NEAR = 4;
    let_next_kernel_start();
    const int tid = threadIdx.x, threads = blockDim.x, groups = n_spans * (SPAN / 8);
    const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    uint32_t* room = rooms[WHOLE ? 0 : warp];
    // the groups of a row that a thread has; where they change places, those that its warp has
    auto there = [&](int g) { return (WHOLE ? g : g - lane) < groups; };
    auto weights = [&](int g, float* w) {
        const int c = g * 8;
        if (WHOLE) {
            if (c < k) {
                const float4 a = *reinterpret_cast<const float4*>(weight + c), b = *reinterpret_cast<const float4*>(weight + c + 4);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
                w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = 0.f;
            }
        } else {
            uint32_t raw[8];
            Eight<float> e;
            read_apart(weight, c - lane * 7, k, raw);
            gather(room, lane, raw, e);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = e.v[i];
        }
    };
    auto join = [&](Eight<float>& v, const Eight<B>& b) {
        if constexpr (sizeof(B) == 2) {
            b.add_to(v.v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v.v[i] += b.v[i];
        }
    };
    if (HELD == 1 && blockIdx.x == 0 && tid * 8 < k) asm volatile("prefetch.global.L2 [%0];" ::"l"(weight + tid * 8));   // (while the kernel before ends)
    wait_for_previous_kernels();
    const int row = blockIdx.x;
    auto read = [&](int g, Eight<float>& v) {
        Eight<B> b;
        if (WHOLE) {
            v.load(stream + (size_t)row * k, g * 8, k);
            if (branch != nullptr) b.load(branch + (size_t)row * k, g * 8, k);
        } else {
            uint32_t raw[8];
            Bits<B> more[8];
            read_apart(stream + (size_t)row * k, g * 8 - lane * 7, k, raw);
            if (branch != nullptr) read_apart(branch + (size_t)row * k, g * 8 - lane * 7, k, more);
            gather(room, lane, raw, v);
            if (branch != nullptr) gather(reinterpret_cast<Bits<B>*>(room), lane, more, b);
        }
        if (branch != nullptr) join(v, b);
    };
    double sum = 0.0, more = 0.0;
    auto square = [&](const Eight<float>& v) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            sum = fma((double)v.v[i], (double)v.v[i], sum);
            more = fma((double)v.v[i + 1], (double)v.v[i + 1], more);
        }
    };
    Eight<float> held[HELD];
    float w[HELD][8];
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (there(tid + h * threads)) read(tid + h * threads, held[h]);
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (there(tid + h * threads)) {
            weights(tid + h * threads, w[h]);
            square(held[h]);
        }
    for (int g = tid + HELD * threads; there(g); g += threads) {
        Eight<float> v;
        read(g, v);
        square(v);
    }
    sum += more;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    // every warp adds the warps' sums, in the same order: lanes that are apart by the power of two that holds them have the same
    const int over = warps <= 1 ? 1 : 2 << (31 - __clz(warps - 1)), at = lane & (over - 1);
    double s = at < warps ? sums[at] : 0.0;
    for (int o = over >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const double r = rsqrt(s * inverse + eps);
    const float r32 = (float)r;
    const bool fine = r32 >= 0x1p-126f;
    auto finish = [&](int g, const Eight<float>& v, const float* by) {
        const int c = g * 8;
        if (total != nullptr) {
            float* to = total + (size_t)row * k + c;
            if (WHOLE) {
                if (c < k) {
                    reinterpret_cast<float4*>(to)[0] = make_float4(v.v[0], v.v[1], v.v[2], v.v[3]);
                    reinterpret_cast<float4*>(to)[1] = make_float4(v.v[4], v.v[5], v.v[6], v.v[7]);
                }
            } else {
                __syncwarp();
                *reinterpret_cast<Eight<float>*>(room + lane * 8) = v;
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c - lane * 7 + q * 32 < k) to[q * 32 - lane * 7] = __uint_as_float(room[q * 32 + lane]);
            }
        }
        Eight<float> y;
        auto exact = [&] {
#pragma unroll
            for (int i = 0; i < 8; ++i) y.v[i] = __uint_as_float(to_odd((double)v.v[i] * r * (double)by[i]));
        };
        // In 32 bits first, which is off by three units in the last place at most: that decides, but next to where the exponent or a code changes
        // (one block in 10^5, and one eight in 700, most of these for numbers below the type's 2^-6), and where a factor may be no normal number: with an
        // inverse root or a weight out of the ordinary, and in blocks of nothing above 2^-47 (numbers from the type's 2^-6 on are 2^-15 of the largest at
        // least, so that v r32 is 2^-62 over a weight below 2^64).
        float heavy = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y.v[i] = v.v[i] * r32 * by[i];
            heavy = fmaxf(heavy, fabsf(by[i]));
        }
        uint32_t top = block_top(fine && heavy < 0x1p64f ? y.top() : 0x7f800000u), byte = exponent_byte<8>(top);
        float z[8];
        if ((top & 0x7fffffu) - (0x600000u - NEAR) <= 2u * NEAR || (top >> 23) - 80u > 158u) {  // (the same for a block's four threads)
            exact();
            byte = exponent_byte<8>(block_top(y.top()));
            y.scaled(byte, z);
        } else {
            y.scaled(byte, z);
            uint32_t apart = 0xffffffffu;                 // from the middle of two codes, in units in the last place, plus NEAR
            float least = 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                apart = min(apart, (__float_as_uint(z[i]) + 0x80000u + NEAR) & 0xfffffu);
                least = fminf(least, fabsf(z[i]));
            }
            if (apart <= 2u * NEAR || least < 0x1p-6f) {
                exact();
                y.scaled(byte, z);
            }
        }
        if (!WHOLE && g >= groups) return;
        *reinterpret_cast<uint2*>(codes + (size_t)row * n_spans * SPAN + c) = make_uint2(eight_bits(z), eight_bits(z + 4));
        if ((c & 31) == 0) exponents[exponent_at(row, c >> 5, n_spans)] = (uint8_t)byte;
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (there(tid + h * threads)) finish(tid + h * threads, held[h], w[h]);
    for (int g = tid + HELD * threads; there(g); g += threads) {
        Eight<float> v;
        float by[8];
        read(g, v);
        weights(g, by);
        finish(g, v, by);
    }
}

// Blocks of threads for so many parts of rows, a warp each; where there are many, a few a warp.
int blocks_for(long long items) {
    const long long want = (items + THREADS / 32 - 1) / (THREADS / 32), most = 1LL << 30;
    return (int)(want < most ? want : most);
}

// What is held must lie on the current device.
int on_device(const char* what, const Held* h) {
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || device != h->device) return fail("%s: what is held lies on device %d, the current one is %d", what, h->device, device);
    return 0;
}

// Launches GROUPS = 4 where its warps are at least as many as the device holds at a time, else 1.
template <typename F1, typename F4>
int by_size(int rows, int width, int of_warp, F1 one, F4 four) {
    const uint32_t parts = (width + 4 * of_warp - 1) / (4 * of_warp);
    if ((long long)rows * parts >= 64LL * sm_count()) return four(parts, (uint32_t)rows * parts);
    const uint32_t small = (width + of_warp - 1) / of_warp;
    return one(small, (uint32_t)rows * small);
}

template <typename T, int BITS, bool WHOLE>
int hold(const T* x, long long ld, const Held* h, cudaStream_t stream) {
    // (a matrix is written in whole tiles: rows behind the last one have no effect on a product, and are zeros)
    const int rows = BITS == 4 ? (h->n + 127) & ~127 : h->n;
    auto go = [&](auto kernel, uint32_t parts, uint32_t items) {
        return check_launch(launch_dependent(kernel, dim3((unsigned)blocks_for(items)), dim3(THREADS), 0, stream, x, h->n, h->k, ld, h->n_spans, parts, items, h->codes,
                                             h->exponents), "mx_hold");
    };
    return by_size(rows, h->n_spans * SPAN, 256, [&](uint32_t p, uint32_t i) { return go(hold_kernel<T, BITS, WHOLE, 1>, p, i); },
                   [&](uint32_t p, uint32_t i) { return go(hold_kernel<T, BITS, WHOLE, 4>, p, i); });
}
// Products read their matrices before they wait for the kernel before them.  So the kernel that makes one lets none begin early, and a kernel that
// nothing may overlap follows it, whose end everything behind it waits for.
__global__ void settle_kernel() {}

template <typename T>
int hold(const T* x, long long ld, const Held* h, cudaStream_t stream) {
    const bool whole = h->k % 8 == 0 && (ld * (long long)sizeof(T)) % 16 == 0 && (uintptr_t)x % 16 == 0;
    if (h->bits == 4) {
        if (int rc = whole ? hold<T, 4, true>(x, ld, h, stream) : hold<T, 4, false>(x, ld, h, stream)) return rc;
        settle_kernel<<<1, 1, 0, stream>>>();
        return check_launch("mx_hold");
    }
    return whole ? hold<T, 8, true>(x, ld, h, stream) : hold<T, 8, false>(x, ld, h, stream);
}

template <typename T, int BITS, bool WHOLE>
int values(const Held* h, T* out, cudaStream_t stream) {
    auto go = [&](auto kernel, uint32_t parts, uint32_t items) {
        return check_launch(launch_dependent(kernel, dim3((unsigned)blocks_for(items)), dim3(THREADS), 0, stream, h->codes, h->exponents, h->k, h->n_spans, parts, items, out),
                            "mx_values");
    };
    return by_size(h->n, h->k, 32 * Sixteen<T>::N, [&](uint32_t p, uint32_t i) { return go(values_kernel<T, BITS, WHOLE, 1>, p, i); },
                   [&](uint32_t p, uint32_t i) { return go(values_kernel<T, BITS, WHOLE, 4>, p, i); });
}
template <typename T>
int values(const Held* h, T* out, cudaStream_t stream) {
    const bool whole = h->k % Sixteen<T>::N == 0 && (uintptr_t)out % 16 == 0;
    if (h->bits == 4) return whole ? values<T, 4, true>(h, out, stream) : values<T, 4, false>(h, out, stream);
    return whole ? values<T, 8, true>(h, out, stream) : values<T, 8, false>(h, out, stream);
}

template <typename B, int HELD>
int norm(const float* x, const B* branch, const float* weight, float* total, const Held* h, double eps, int most, cudaStream_t stream) {
    const int groups = h->n_spans * (SPAN / 8);
    const bool whole = h->k % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)branch % 16 == 0 && (uintptr_t)total % 16 == 0 && (uintptr_t)weight % 16 == 0;
    int threads = ((groups + HELD - 1) / HELD + 31) / 32 * 32;
    if (threads > most) threads = most;
    auto go = [&](auto kernel) {
        return check_launch(launch_dependent(kernel, dim3((unsigned)h->n), dim3(threads), 0, stream, x, branch, weight, total, h->k, h->n_spans, 1.0 / h->k, eps, h->codes,
                                             h->exponents), "mx_rmsnorm");
    };
    return whole ? go(rmsnorm_kernel<B, HELD, true>) : go(rmsnorm_kernel<B, HELD, false>);
}
// Few rows are as fast as one of them, which many threads with one group each have sooner (us, one group / two: 8 rows of 3,584 2.4 / 2.7, 148 of
// 4,096 2.6 / 3.25, 296 of them 4.0 / 4.4); many are as fast as the SMs' instructions, of which two groups a thread take fewer (330 of 4,096 5.7 / 5.55,
// 600 8.1 / 7.5, 2,047 20.8 / 17.0, with branch and total 25.6 / 22.1).
template <typename B>
int norm(const float* x, const void* branch, const float* weight, float* total, const Held* h, double eps, cudaStream_t stream) {
    return h->n <= 2 * sm_count() ? norm<B, 1>(x, (const B*)branch, weight, total, h, eps, 1024, stream)
                                  : norm<B, 2>(x, (const B*)branch, weight, total, h, eps, 512, stream);
}

}  // namespace

// Bytes of a `Held`, 64-byte aligned.
RI_API long long ri_mx_held_bytes() { return (long long)sizeof(Held); }

// A `Held` at `at`: [n, k] numbers of `bits` bits (4: a matrix, 8: rows) over these buffers of the device `device`.
RI_API int ri_mx_make(void* at, void* codes, void* exponents, long long n, long long k, int bits, int device) {
    if ((uintptr_t)at % 64) return fail("mx_make: 64-byte aligned memory is wanted");
    if (n <= 0 || k <= 0 || k > 0x7fffffffLL - SPAN || (bits != 4 && bits != 8)) return fail("mx_make: no [%lld, %lld] numbers of %d bits", n, k, bits);
    if ((n + 127) / 128 * 128 * spans((int)k) > 0x7fffffffLL / (SPAN / 8)) return fail("mx_make: [%lld, %lld] numbers are more than 2^31 eights", n, k);
    if ((uintptr_t)codes % 32 || (uintptr_t)exponents % 32) return fail("mx_make: buffers must begin on a 32-byte boundary");
    if (!apart(codes, code_bytes(n, spans((int)k), bits), exponents, exponent_bytes(n, spans((int)k)))) return fail("mx_make: codes and exponents must lie apart");
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
    if (n != h->n || k != h->k || ld < k) return fail("mx_hold: [%lld, %lld] numbers, rows %lld apart, do not go into [%d, %d]", n, k, ld, h->n, h->k);
    if (!apart(h, x, ((n - 1) * ld + k) * item_bytes(dtype))) return fail("mx_hold: the numbers must lie apart from what holds them");
    if (int rc = on_device("mx_hold", h)) return rc;
    return dtype == RI_BF16 ? hold((const __nv_bfloat16*)x, ld, h, stream) : hold((const float*)x, ld, h, stream);
}

// After a matrix has been written by something else than `ri_mx_hold`: see `settle_kernel`.
RI_API int ri_mx_settle(cudaStream_t stream) {
    settle_kernel<<<1, 1, 0, stream>>>();
    return check_launch("mx_settle");
}

// out [n, k]: the numbers that are held.
RI_API int ri_mx_values(const void* held, int dtype, long long n, long long k, void* out, cudaStream_t stream) {
    const Held* h = (const Held*)held;
    if (n != h->n || k != h->k) return fail("mx_values: [%d, %d] numbers do not go into [%lld, %lld]", h->n, h->k, n, k);
    if (!apart(h, out, n * k * item_bytes(dtype))) return fail("mx_values: the numbers must lie apart from what holds them");
    if (int rc = on_device("mx_values", h)) return rc;
    return dtype == RI_BF16 ? values(h, (__nv_bfloat16*)out, stream) : values(h, (float*)out, stream);
}

// total = stream + branch (branch null: the stream itself; total null: not kept; it may be the stream), [n, k], and the norm of it times `weight` in 8 bits.
RI_API int ri_mx_rmsnorm(const float* x, const void* branch, int branch_dtype, const float* weight, float* total, long long n, long long k, double eps,
                         void* held, cudaStream_t stream) {
    const Held* h = (const Held*)held;
    if (n != h->n || k != h->k || h->bits != 8) return fail("mx_rmsnorm: a norm of [%lld, %lld] does not go into [%d, %d] of %d bits", n, k, h->n, h->k, h->bits);
    if (!apart(h, x, n * k * 4) || !apart(h, branch, n * k * item_bytes(branch_dtype)) || !apart(h, weight, k * 4) || !apart(h, total, n * k * 4))
        return fail("mx_rmsnorm: the rows in 8 bits must lie apart from what is read and from the total");
    if (int rc = on_device("mx_rmsnorm", h)) return rc;
    return branch_dtype == RI_BF16 ? norm<__nv_bfloat16>(x, branch, weight, total, h, eps, stream)
                                   : norm<float>(x, branch, weight, total, h, eps, stream);
}

RI_DEFINE_LAST_ERROR()
