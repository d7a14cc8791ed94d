// Global norm over a list of tensors and their scaling by clip(norm, 0, max_norm) / (eps + norm): the arithmetic of
// libs/lasagne_libs/updates.py:845-855 for gradients that do not lie in one buffer.
// The list travels in the kernel arguments (up to TENSORS tensors a launch), so a call needs no copy of a table to the device
// and can be captured.  HBM-bound for large tensors, launch-bound for small ones: a chunk of CHUNK values of one tensor is a
// workgroup's work whatever the sizes in the list, three launches in all for up to TENSORS tensors.
// Squares are summed in double: an f32 square overflows above 1.8e19 and a long f32 sum loses digits.
// Measured, 56 tensors of 148 MB, f32 and bf16: squares 24 us (6.1 TB/s, part of it from the Infinity Cache), the norm 4, scaling
// 47 (6.4 TB/s read and written); the host needs 76 us to prepare such a list, beside them.
#include "seq_common.h"

#define TENSORS 64
#define CHUNK 8192

struct ClipList {
    const void* src[TENSORS];
    void* dst[TENSORS];
    long long size[TENSORS];
    int first[TENSORS + 1];            // first chunk of a tensor
    unsigned char dtype[TENSORS];
    int count;
};

__device__ __forceinline__ int find_tensor(const ClipList& l, int chunk) {
    int lo = 0, hi = l.count - 1;      // the last tensor whose first chunk is <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// 16 bytes at a time at any address that suits T: the results of one type lie behind one another in one buffer.
template <typename T> struct Any16 {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ double chunk_sq(const T* p, int n) {
    constexpr int V = 16 / sizeof(T);
    double acc = 0.0;
    const int nv = n / V;
    for (int i = threadIdx.x; i < nv; i += 256) {
        const typename Any16<T>::type v = *(const typename Any16<T>::type*)(p + i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) acc = __builtin_fma((double)(float)v[e], (double)(float)v[e], acc);
    }
    for (int i = nv * V + threadIdx.x; i < n; i += 256) {
        const double v = (double)ldf(p + i);
        acc = __builtin_fma(v, v, acc);
    }
    return acc;
}

__global__ __launch_bounds__(256) void clip_sq_kernel(ClipList l, double* __restrict__ part) {
    __shared__ double sm[4];
    const int t = find_tensor(l, blockIdx.x);
    const long long at = (long long)(blockIdx.x - l.first[t]) * CHUNK;
    const int n = (int)min((long long)CHUNK, l.size[t] - at);
    double acc;
    if (l.dtype[t] == ASR_F32) acc = chunk_sq((const float*)l.src[t] + at, n);
    else if (l.dtype[t] == ASR_BF16) acc = chunk_sq((const bf16_t*)l.src[t] + at, n);
    else acc = chunk_sq((const f16_t*)l.src[t] + at, n);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

__global__ __launch_bounds__(1024) void clip_norm_kernel(const double* __restrict__ part, int n, float max_norm, float eps,
                                                         float* __restrict__ norm_out, float* __restrict__ mult) {
    __shared__ double sm[16];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) acc += part[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int k = 0; k < 16; ++k) t += sm[k];
        const float nv = (float)sqrt(t);
        norm_out[0] = nv;
        mult[0] = fminf(fmaxf(nv, 0.f), max_norm) / (eps + nv);
    }
}

template <typename T, bool STREAM>
__device__ __forceinline__ void chunk_scale(const T* p, T* q, int n, float m) {
    constexpr int V = 16 / sizeof(T);
    const int nv = n / V;
    for (int i = threadIdx.x; i < nv; i += 256) {
        typename Any16<T>::type v = *(const typename Any16<T>::type*)(p + i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)((float)v[e] * m);
        if constexpr (STREAM) __builtin_nontemporal_store(v, (typename Any16<T>::type*)(q + i * V));
        else *(typename Any16<T>::type*)(q + i * V) = v;
    }
    for (int i = nv * V + threadIdx.x; i < n; i += 256) stf(q + i, ldf(p + i) * m);
}

// STREAM: results that do not stay in the caches.  From 64 MiB on they would push out the inputs that this second pass still has
// to read: with a momentum step behind it that reads the results, 64 / 128 / 256 / 512 MiB of f32 take 122 / 299 / 662 / 1323 us
// instead of 141 / 309 / 678 / 1331; at 32 MiB the step misses them (80 us instead of 67), at 8 MiB there is no difference.
#define STREAM_BYTES (64ll << 20)
template <bool STREAM>
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipList l, const float* __restrict__ mult) {
    const int c = gridDim.x - 1 - blockIdx.x;          // what was read last, first: it is in the caches
    const int t = find_tensor(l, c);
    const long long at = (long long)(c - l.first[t]) * CHUNK;
    const int n = (int)min((long long)CHUNK, l.size[t] - at);
    const float m = mult[0];
    if (l.dtype[t] == ASR_F32) chunk_scale<float, STREAM>((const float*)l.src[t] + at, (float*)l.dst[t] + at, n, m);
    else if (l.dtype[t] == ASR_BF16) chunk_scale<bf16_t, STREAM>((const bf16_t*)l.src[t] + at, (bf16_t*)l.dst[t] + at, n, m);
    else chunk_scale<f16_t, STREAM>((const f16_t*)l.src[t] + at, (f16_t*)l.dst[t] + at, n, m);
}

// ---------------------------------------------------------------- C entry
static long long chunks_of(long long n) { return (n + CHUNK - 1) / CHUNK; }

extern "C" size_t asr_clip_list_ws_bytes(int count, const long long* sizes) {
    if (count <= 0 || !sizes) return 16;
    long long c = 0;
    for (int i = 0; i < count; ++i) c += sizes[i] > 0 ? chunks_of(sizes[i]) : 0;
    return (size_t)c * sizeof(double) + 16;
}

extern "C" int asr_clip_list(int count, const int* dtypes, const void* const* src, void* const* dst,
                             const long long* sizes, float max_norm, float eps, float* norm_out, void* ws,
                             size_t ws_bytes, hipStream_t stream) {
    if (count < 0 || !norm_out || !(max_norm >= 0.f) || !(eps >= 0.f)) return ASR_ERR_ARG;
    if (count && (!dtypes || !src || !dst || !sizes)) return ASR_ERR_ARG;
    long long total = 0, bytes = 0;
    for (int i = 0; i < count; ++i) {
        if (dtypes[i] < ASR_F32 || dtypes[i] > ASR_F16 || sizes[i] < 0) return ASR_ERR_ARG;
        if (sizes[i] && (!src[i] || !dst[i])) return ASR_ERR_ARG;
        if (sizes[i] > (1ll << 40)) return ASR_ERR_LIMIT;
        total += chunks_of(sizes[i]);
        bytes += sizes[i] * (long long)elem_size(dtypes[i]);
    }
    if (total >= (1 << 24)) return ASR_ERR_LIMIT;                // 2^32 work items a launch
    if (!ws || ws_bytes < asr_clip_list_ws_bytes(count, sizes)) return ASR_ERR_WS;
    if ((uintptr_t)ws & 15) return ASR_ERR_ARG;
    double* part = (double*)ws;
    float* mult = (float*)(part + total);
    for (int pass = 0; pass < 2; ++pass) {
        int i = 0;
        double* at = part;
        while (i < count) {
            ClipList l;
            l.count = 0;
            int c = 0;
            for (; i < count && l.count < TENSORS; ++i) {
                if (!sizes[i]) continue;
                l.src[l.count] = src[i]; l.dst[l.count] = dst[i]; l.size[l.count] = sizes[i];
                l.dtype[l.count] = (unsigned char)dtypes[i]; l.first[l.count] = c;
                c += (int)chunks_of(sizes[i]);
                ++l.count;
            }
            if (!l.count) break;
            l.first[l.count] = c;
            if (pass == 0) hipLaunchKernelGGL(clip_sq_kernel, dim3(c), dim3(256), 0, stream, l, at);
            else if (bytes >= STREAM_BYTES)
                hipLaunchKernelGGL(clip_scale_kernel<true>, dim3(c), dim3(256), 0, stream, l, (const float*)mult);
            else hipLaunchKernelGGL(clip_scale_kernel<false>, dim3(c), dim3(256), 0, stream, l, (const float*)mult);
            ASR_CHECK_LAUNCH();
            at += c;
        }
        if (pass == 0) {
            hipLaunchKernelGGL(clip_norm_kernel, dim3(1), dim3(1024), 0, stream, (const double*)part, (int)total, max_norm, eps,
                               norm_out, mult);
            ASR_CHECK_LAUNCH();
        }
    }
    return ASR_OK;
}
