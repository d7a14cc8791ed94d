// Shared by the state-space layer's kernels (conv.hip, sscan_*.hip, rmsnorm.hip): activation types and lane sums.
#pragma once
#include "common.h"

#define ASR_F32 0
#define ASR_BF16 1
#define ASR_F16 2

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Activations are held in f32, bf16 or f16 and computed in f32; a store rounds once, to nearest even.
template <typename T> __device__ __forceinline__ float ldf(const T* p) { return (float)*p; }
template <typename T> __device__ __forceinline__ void stf(T* p, float v) { *p = (T)v; }

// V consecutive values as one access (V * sizeof(T) = 16 bytes, or V = 1)
template <typename T, int V> struct Vec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct Vec<T, 1> { typedef T type; };
template <typename T, int V> __device__ __forceinline__ void ldv(const T* p, float* o) {
    if constexpr (V == 1) o[0] = (float)p[0];
    else {
        const typename Vec<T, V>::type v = *(const typename Vec<T, V>::type*)p;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (float)v[e];
    }
}
template <typename T, int V> __device__ __forceinline__ void stv(T* p, const float* o) {
    if constexpr (V == 1) p[0] = (T)o[0];
    else {
        typename Vec<T, V>::type v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)o[e];
        *(typename Vec<T, V>::type*)p = v;
    }
}

// V values from any address that suits T: gfx950 takes 16 bytes at a time from there, and a wave's 1 KiB touches one line more than it has to.
template <typename T, int V> struct AnyV { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T> struct AnyV<T, 1> { typedef T type; };
template <typename T, int V> __device__ __forceinline__ void ldu(const T* p, float* o) {
    const typename AnyV<T, V>::type v = *(const typename AnyV<T, V>::type*)p;
    if constexpr (V == 1) o[0] = (float)v;
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (float)v[e];
    }
}
template <typename T, int V> __device__ __forceinline__ void stu(T* p, const float* o) {
    typename AnyV<T, V>::type v;
    if constexpr (V == 1) v = (T)o[0];
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)o[e];
    }
    *(typename AnyV<T, V>::type*)p = v;
}

// e^-|v| in (0, 1]: the argument's product with log2 e in two floats, the rest as a first-order correction.  Finite for
// every v (a NaN becomes e^-110): the functions below carry v itself on, and with it infinities and NaN.
__device__ __forceinline__ float exp_neg_abs_(float v) {
    const float L2E_HI = 0x1.715476p+0f, L2E_LO = 0x1.4ae0c0p-26f, LN2_ = 0x1.62e430p-1f;
    const float x = fmaxf(-fabsf(v), -110.0f);
    const float hi = x * L2E_HI, lo = __builtin_fmaf(x, L2E_HI, -hi) + x * L2E_LO;
    const float e = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(e, lo * LN2_, e);
}
// 1 / (1 + e^-v) from u = e^-|v|, and by itself.  The plain exponent loses |v| 2^-24 of e^-v: of the sigmoid where it is
// small, of v sigmoid(v) never more than 0.6 * 2^-24 absolute (|v|^2 e^-|v| 2^-24), less than its last rounding near 1.
__device__ __forceinline__ float sigmoid_from_(float v, float u) {
    const float r = __builtin_amdgcn_rcpf(1.0f + u);
    return v < 0.0f ? u * r : r;
}
__device__ __forceinline__ float sigm_(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}
__device__ __forceinline__ float silu_(float z) { return z * sigm_(z); }
// d silu / dz, from z and its sigmoid
__device__ __forceinline__ float dsilu_(float z, float sg) { return sg * (1.0f + z * (1.0f - sg)); }
// log(1 + e^v) = max(v, 0) + log1p(u), u = e^-|v|: no overflow, relative accuracy for very negative v.  log1p(u) = log(w) u / (w - 1)
// with w = 1 + u rounded (Kahan's form: the rounding of w is in both factors), u itself where w = 1.
__device__ __forceinline__ float softplus_from_(float v, float u) {
    const float w = 1.0f + u, d = w - 1.0f;
    const float l = __builtin_amdgcn_logf(w) * 0x1.62e430p-1f;
    return (v < 0.0f ? 0.0f : v) + (d == 0.0f ? u : l * (u * __builtin_amdgcn_rcpf(d)));
}
__device__ __forceinline__ float softplus_(float v) { return softplus_from_(v, exp_neg_abs_(v)); }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// a frame of row b: walking order s -> frame.  Both directions walk the valid frames s = 0 .. len-1.
__device__ __forceinline__ int row_len(const int* lens, int b, int T) {
    if (!lens) return T;
    const int n = lens[b];
    return n < 0 ? 0 : (n > T ? T : n);
}

// out[i] = sum over p of part[p * stride + i], i < n, in a fixed order: the second half of every reduction over rows or
// time.  16 columns x 64 groups of partials per workgroup: few columns and many partials are the usual shape (1024 columns,
// 2048 partials: 39 us with 64 columns x 16 groups).
static __global__ __launch_bounds__(1024) void sum_partials_kernel(const float* __restrict__ part, size_t stride, int P,
                                                                   size_t n, float* __restrict__ out) {
    __shared__ float sm[16][16];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const size_t i = (size_t)blockIdx.x * 16 + c;
    float acc = 0.f;
    if (i < n) {
#pragma unroll 4
        for (int p = g; p < P; p += 64) acc += part[(size_t)p * stride + i];
    }
    acc += __shfl_xor(acc, 16);
    acc += __shfl_xor(acc, 32);
    if ((threadIdx.x & 63) < 16) sm[threadIdx.x >> 6][c] = acc;
    __syncthreads();
    if (threadIdx.x < 16 && i < n) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += sm[k][c];
        out[i] = t;
    }
}
static inline void sum_partials(const float* part, size_t stride, int P, size_t n, float* out, hipStream_t stream) {
    if (n) hipLaunchKernelGGL(sum_partials_kernel, dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, stream, part, stride, P, n,
                              out);
}

static inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
static inline size_t elem_size(int dtype) { return dtype == ASR_F32 ? 4 : 2; }
