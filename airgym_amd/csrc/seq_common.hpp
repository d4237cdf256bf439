// seq_common.hpp - element types and scalar functions shared by the sequence operators (causal_conv.hip, selective_scan.hip,
// policy_loss.hip).  Activations come in float32, bfloat16 or float16; every product and sum is formed in float32 and rounded
// once, to nearest, where a result is stored in its type (the policy loss's bfloat16 gradient a second time where the loss is scaled).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/airgym_hip.h"

namespace {

constexpr long long kMaxThreads = 0xffffffffLL;      // of one launch
constexpr int kMaxSteps = 1 << 30;                   // of a sequence: step indexes run a little past its end

// The last-level cache holds 256 MB.  What a call reads or writes of a buffer below half of that may still be there for the next kernel;
// what it touches of a larger one will mostly be gone by then and only drives out the rest: from here on it is marked as used once.
constexpr long long kCached = 128LL << 20;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// N consecutive elements (at most 16 bytes), kept as they are stored and moved with one access.  The access is aligned to the element
// only - rows of an odd width start anywhere -, which the memory takes at the same speed.
template <int kWords> struct Words;
#define AG_WORDS(n)                                                                  \
    template <> struct Words<n> {                                                    \
        typedef uint32_t any2 __attribute__((ext_vector_type(n), aligned(2)));       \
        typedef uint32_t any4 __attribute__((ext_vector_type(n), aligned(4)));       \
    };
AG_WORDS(2) AG_WORDS(4)
#undef AG_WORDS
template <> struct Words<1> {
    typedef uint32_t any2 __attribute__((aligned(2)));
    typedef uint32_t any4;
};

template <typename T, int N> struct Vec {
    static constexpr int kWords = N * (int)sizeof(T) / 4;
    uint32_t w[kWords ? kWords : 1];
    __device__ __forceinline__ float at(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t v = w[i / 2];
        if (__is_same(T, bf16_t)) return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
        return (float)__builtin_bit_cast(f16_t, (uint16_t)(i & 1 ? v >> 16 : v));
    }
    __device__ __forceinline__ void set(const float* x) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = __float_as_uint(x[k]);
        } else if constexpr (N == 1) {
            w[0] = __builtin_bit_cast(uint16_t, from_f32<T>(x[0]));
        } else {
            typedef T pair __attribute__((ext_vector_type(2)));
            typedef float two __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int k = 0; k < kWords; k++) {
                const two f = {x[2 * k], x[2 * k + 1]};
                w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, pair));
            }
        }
    }
};
// kOnce: nothing reads this again before it has left the caches (a hint to them, nothing else)
#define AG_LOAD(P, p) (kOnce ? __builtin_nontemporal_load((const P*)(p)) : *(const P*)(p))
#define AG_STORE(P, p, v) (kOnce ? __builtin_nontemporal_store(v, (P*)(p)) : (void)(*(P*)(p) = v))
template <typename T, int N, bool kOnce = false> __device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
    constexpr int K = Vec<T, N>::kWords;
    Vec<T, N> c;
    if constexpr (K == 0) c.w[0] = AG_LOAD(uint16_t, p);
    else if constexpr (K == 1) {
        if constexpr (sizeof(T) == 2) c.w[0] = AG_LOAD(Words<1>::any2, p);
        else c.w[0] = AG_LOAD(uint32_t, p);
    } else if constexpr (sizeof(T) == 2) {
        const auto v = AG_LOAD(typename Words<K>::any2, p);
#pragma unroll
        for (int k = 0; k < K; k++) c.w[k] = v[k];
    } else {
        const auto v = AG_LOAD(typename Words<K>::any4, p);
#pragma unroll
        for (int k = 0; k < K; k++) c.w[k] = v[k];
    }
    return c;
}
template <typename T, int N, bool kOnce = false> __device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& c) {
    constexpr int K = Vec<T, N>::kWords;
    if constexpr (K == 0) AG_STORE(uint16_t, p, (uint16_t)c.w[0]);
    else if constexpr (K == 1) {
        if constexpr (sizeof(T) == 2) AG_STORE(Words<1>::any2, p, c.w[0]);
        else AG_STORE(uint32_t, p, c.w[0]);
    } else if constexpr (sizeof(T) == 2) {
        typename Words<K>::any2 v;
#pragma unroll
        for (int k = 0; k < K; k++) v[k] = c.w[k];
        AG_STORE(typename Words<K>::any2, p, v);
    } else {
        typename Words<K>::any4 v;
#pragma unroll
        for (int k = 0; k < K; k++) v[k] = c.w[k];
        AG_STORE(typename Words<K>::any4, p, v);
    }
}
#undef AG_LOAD
#undef AG_STORE

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }       // v_log_f32: 1 ulp
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }        // v_rcp_f32: 1 ulp
__device__ __forceinline__ float exp_hw(float x) { return exp2_hw(x * kLog2e); }
__device__ __forceinline__ float sigmoid(float x) { return rcp_hw(1.0f + exp_hw(-x)); }

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in [0, 1].  log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3: 2 atanh(s) / s is a
// function of q = s^2 in [0, 1/9]; the polynomial of degree 4 through its Chebyshev points is within 4e-9 of it.  Unlike log(1 + e) this
// keeps its RELATIVE accuracy where e is small (steps of 1e-3 and less are what the scan's time step usually is).
__device__ __forceinline__ float softplus_from(float x, float e) {
    const float s = e * rcp_hw(2.0f + e), q = s * s;
    float p = 0.28174657f;
    p = __builtin_fmaf(p, q, 0.27961419f);
    p = __builtin_fmaf(p, q, 0.40024854f);
    p = __builtin_fmaf(p, q, 0.66666316f);
    p = __builtin_fmaf(p, q, 2.0f);
    return __builtin_fmaf(p, s, fmaxf(x, 0.0f));
}
__device__ __forceinline__ float softplus(float x) { return softplus_from(x, exp_hw(-__builtin_fabsf(x))); }
// ... and its slope, the sigmoid, from the same exponential
__device__ __forceinline__ float softplus(float x, float& slope) {
    const float e = exp_hw(-__builtin_fabsf(x)), r = rcp_hw(1.0f + e);
    slope = x < 0.0f ? e * r : r;
    return softplus_from(x, e);
}

// steps of sequence b that count: all T, or its length clamped to what the buffers hold
__device__ __forceinline__ int seq_len(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > T ? T : n);
}

// Sums over the rows of a [rows, n] table, in a fixed order: a column per lane, `Parts` parts of the rows per column (so that a table
// of few columns and many rows still has enough loads in flight), joined through LDS.  `out(i, sum)` puts column i's sum away.
template <int Parts, typename Out>
__global__ __launch_bounds__(64 * Parts) void sum_rows_kernel(const float* table, int rows, long long n, Out out) {
    __shared__ float part[Parts][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long i = (long long)blockIdx.x * 64 + lane;
    const int per = (rows + Parts - 1) / Parts, first = w * per, last = first + per < rows ? first + per : rows;
    float s = 0.0f;
    if (i < n)
#pragma unroll 8
        for (int r = first; r < last; r++) s += table[(long long)r * n + i];
    part[w][lane] = s;
    __syncthreads();
    if (w || i >= n) return;
#pragma unroll
    for (int k = 1; k < Parts; k++) s += part[k][lane];
    out(i, s);
}

// ... and of a table of few rows: a column per thread (several, where columns outnumber what a launch can hold)
template <typename Out>
__global__ __launch_bounds__(256) void sum_few_rows_kernel(const float* table, int rows, long long n, Out out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = 0.0f;
        for (int r = 0; r < rows; r += 4) {                     // four rows' loads at a time, added in order
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = r + k < rows ? table[(long long)(r + k) * n + i] : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) s += v[k];
        }
        out(i, s);
    }
}

// At 256 columns x 1024 rows the split rows take 5 us where a column per thread took 236; at 3 M columns x 4 rows the plain form takes
// half of theirs.
template <typename Out>
inline void launch_sum_rows(const float* table, int rows, long long n, Out out, void* stream) {
    if (rows <= 4 || n >= (1 << 18)) {
        const long long blocks = (n + 255) / 256, most = kMaxThreads / 256;
        hipLaunchKernelGGL((sum_few_rows_kernel<Out>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, (hipStream_t)stream, table, rows, n, out);
        return;
    }
    const dim3 grid((unsigned)((n + 63) / 64));
    if (rows > 64) hipLaunchKernelGGL((sum_rows_kernel<16, Out>), grid, dim3(1024), 0, (hipStream_t)stream, table, rows, n, out);
    else hipLaunchKernelGGL((sum_rows_kernel<4, Out>), grid, dim3(256), 0, (hipStream_t)stream, table, rows, n, out);
}

inline int seq_status() { return hipGetLastError() == hipSuccess ? AG_OK : AG_ERR_HIP; }

}  // namespace

// run CALL with `T` bound to the element type of an ag_dtype; AG_ERR_UNSUPPORTED for any other value
#define AG_FOR_DTYPE(dtype, CALL)                              \
    do {                                                       \
        switch (dtype) {                                       \
            case AG_F32: { using T = float; CALL; } break;     \
            case AG_BF16: { using T = bf16_t; CALL; } break;   \
            case AG_F16: { using T = f16_t; CALL; } break;     \
            default: return AG_ERR_UNSUPPORTED;                \
        }                                                      \
    } while (0)
