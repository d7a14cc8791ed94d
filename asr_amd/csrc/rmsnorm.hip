// Root-mean-square norm of rows with the residual's addition in front of it, forward and backward.
//   r = x (+ residual),   y = r rstd w,   rstd = 1 / sqrt(mean r^2 + eps)
//   g = dy w,   dr = (g - xhat mean(g xhat)) rstd (+ dres),   dw = sum_rows dy xhat,   xhat = r rstd
// HBM-bound: a pass reads and writes every tensor once, a row stays in registers between its two uses.  r is rounded to the
// activation type when it is stored; y is formed from the unrounded sum, and the backward pass forms that sum again from x and
// the residual (one more read than the stored r would cost, but gradients of what was computed: with the stored r, dw is off by
// the type's half step).  Measured at 36192 rows x 1024, bf16, with a residual: forward 48 us (6.2 TB/s of the 0.30 GB of its four
// tensors, some of them still in the Infinity Cache), backward 77 us (4.8 TB/s of 0.37 GB) and 5 for the parts of dw.
#include "seq_common.h"

// A row is walked in groups of V columns, a lane to a group.  Where n is no multiple of V the last group is moved back to end with
// the row: its first `skip` columns are the group's in front of it too, are left out of its sums, and are stored twice, the same.
// Lanes behind the row stand on that group too (skip >= V: all of it) and store nothing: no branch between a row's loads.
// (Measured before, a value at a time: 36192 x 1001, bf16, 120 us forward and 300 backward.)
struct Group { int c, skip; };
template <int V> __device__ __forceinline__ Group group(int c, int n) {
    const int at = min(c, n - V);
    return Group{at, c - at};
}
template <int V> __device__ __forceinline__ float dot_v(const float (&a)[V], const float (&b)[V], int skip) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s = __builtin_fmaf(a[e], b[e], s);
    if (skip) {
        s = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) s = e < skip ? s : __builtin_fmaf(a[e], b[e], s);
    }
    return s;
}

// WPR waves share a row (1: four rows per workgroup, 4: one).  NV groups of V values per lane are held in registers.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* sm, int w) {
    v = wave_sum(v);
    if constexpr (WPR == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[w] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

template <typename T, int V, int NV, int WPR>
__global__ __launch_bounds__(256) void rms_fwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ res,
                                                      long long ldr, const float* __restrict__ w, int rows, int n,
                                                      float eps, T* __restrict__ y, T* __restrict__ sum,
                                                      float* __restrict__ rstd) {
    __shared__ float sm[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int row = WPR == 1 ? blockIdx.x * 4 + wv : blockIdx.x;
    if (row >= rows) return;                                    // a whole wave, and WPR = 4 has no such row
    const int c0 = (WPR == 1 ? lane : (int)threadIdx.x) * V;
    constexpr int STEP = 64 * WPR * V;
    float v[NV][V];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) ldu<T, V>(x + row * ldx + group<V>(c0 + i * STEP, n).c, v[i]);
    if (res) {
        float q[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) ldu<T, V>(res + row * ldr + group<V>(c0 + i * STEP, n).c, q[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] += q[i][e];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Group k = group<V>(c0 + i * STEP, n);
        if (sum && c0 + i * STEP < n) stu<T, V>(sum + (size_t)row * n + k.c, v[i]);
        sq += dot_v<V>(v[i], v[i], k.skip);
    }
    sq = row_sum<WPR>(sq, sm, wv);
    const float rs = 1.0f / sqrtf(sq / (float)n + eps);
    if (rstd && (WPR == 1 ? lane : (int)threadIdx.x) == 0) rstd[row] = rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * STEP;
        if (c >= n) continue;
        const Group k = group<V>(c, n);
        float o[V], ww[V];
        ldu<float, V>(w + k.c, ww);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[i][e] * rs * ww[e];
        stu<T, V>(y + (size_t)row * n + k.c, o);
    }
}

// Rows longer than the registers hold: a workgroup per row, read twice.
template <typename T, int V>
__global__ __launch_bounds__(256) void rms_fwd_long_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ res,
                                                           long long ldr, const float* __restrict__ w, int n, float eps,
                                                           T* __restrict__ y, T* __restrict__ sum,
                                                           float* __restrict__ rstd) {
    __shared__ float sm[4];
    const size_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    const T* rr = res ? res + row * ldr : nullptr;
    float sq = 0.f;
    const auto sums = [&](int c, float (&v)[V]) {
        ldu<T, V>(xr + c, v);
        if (rr) {
            float q[V];
            ldu<T, V>(rr + c, q);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += q[e];
        }
    };
    for (int c = threadIdx.x * V; c < n; c += 256 * V) {
        const Group k = group<V>(c, n);
        float v[V];
        sums(k.c, v);
        sq += dot_v<V>(v, v, k.skip);
    }
    sq = row_sum<4>(sq, sm, threadIdx.x >> 6);
    const float rs = 1.0f / sqrtf(sq / (float)n + eps);
    if (rstd && threadIdx.x == 0) rstd[row] = rs;
    for (int c = threadIdx.x * V; c < n; c += 256 * V) {
        const Group k = group<V>(c, n);
        float v[V], ww[V];
        sums(k.c, v);
        ldu<float, V>(w + k.c, ww);
        if (sum) stu<T, V>(sum + row * n + k.c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = v[e] * rs * ww[e];
        stu<T, V>(y + row * n + k.c, v);
    }
}

// A workgroup walks rows blockIdx.x, + gridDim.x, ...; a lane owns columns, so its part of dw stays in registers.
template <typename T, int V, int NV, int WPR>
__global__ __launch_bounds__(256) void rms_bwd_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                      long long ldx, const T* __restrict__ res, long long ldr,
                                                      const float* __restrict__ w,
                                                      const float* __restrict__ rstd, const T* __restrict__ dres,
                                                      long long ldd, int rows, int n, T* __restrict__ dx,
                                                      float* __restrict__ part) {
    constexpr int STEP = 64 * WPR * V, RPB = 4 / WPR;
    __shared__ float sm[4];
    __shared__ float s_dw[WPR == 1 ? 3 : 1][WPR == 1 ? NV * V * 64 : 1];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c0 = (WPR == 1 ? lane : (int)threadIdx.x) * V;
    float dw[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[i][e] = 0.f;
    for (int row = blockIdx.x * RPB + (WPR == 1 ? wv : 0); row < rows; row += gridDim.x * RPB) {
        const float rs = rstd[row];
        float g[NV][V], xh[NV][V], dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ldu<T, V>(dy + row * lddy + group<V>(c0 + i * STEP, n).c, g[i]);
            ldu<T, V>(x + row * ldx + group<V>(c0 + i * STEP, n).c, xh[i]);
        }
        if (res) {
            float q[NV][V];
#pragma unroll
            for (int i = 0; i < NV; ++i) ldu<T, V>(res + row * ldr + group<V>(c0 + i * STEP, n).c, q[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) xh[i][e] += q[i][e];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Group k = group<V>(c0 + i * STEP, n);
            float ww[V];
            ldu<float, V>(w + k.c, ww);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[i][e] *= rs;
                dw[i][e] = __builtin_fmaf(g[i][e], xh[i][e], dw[i][e]);
                g[i][e] *= ww[e];
            }
            dot += dot_v<V>(g[i], xh[i], k.skip);
        }
        dot = row_sum<WPR>(dot, sm, wv) / (float)n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = c0 + i * STEP;
            if (c >= n) continue;
            const Group k = group<V>(c, n);
            float o[V], d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = (g[i][e] - xh[i][e] * dot) * rs;
            if (dres) {
                ldu<T, V>(dres + row * ldd + k.c, d);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += d[e];
            }
            stu<T, V>(dx + (size_t)row * n + k.c, o);
        }
    }
    if constexpr (WPR == 1) {                              // the four waves' parts, joined in order
        if (wv) {
#pragma unroll
            for (int i = 0; i < NV * V; ++i) s_dw[wv - 1][i * 64 + lane] = dw[i / V][i % V];
        }
        __syncthreads();
        if (wv) return;
#pragma unroll
        for (int i = 0; i < NV * V; ++i)
            dw[i / V][i % V] = (dw[i / V][i % V] + s_dw[0][i * 64 + lane]) + (s_dw[1][i * 64 + lane] + s_dw[2][i * 64 + lane]);
    }
    float* pp = part + (size_t)blockIdx.x * n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * STEP;
        if (c < n) {
            const Group k = group<V>(c, n);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e >= k.skip) pp[k.c + e] = dw[i][e];
        }
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void rms_bwd_long_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                           long long ldx, const T* __restrict__ res, long long ldr,
                                                           const float* __restrict__ w,
                                                           const float* __restrict__ rstd, const T* __restrict__ dres,
                                                           long long ldd, int rows, int n, T* __restrict__ dx,
                                                           float* __restrict__ part) {
    __shared__ float sm[4];
    float* pp = part + (size_t)blockIdx.x * n;                 // a thread's own columns only: no other thread reads them
    for (int c = threadIdx.x * V; c < n; c += 256 * V)
        for (int e = c; e < min(c + V, n); ++e) pp[e] = 0.f;
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const float rs = rstd[row];
        const auto pair = [&](int c, float (&g)[V], float (&xh)[V]) {        // dy and xhat
            ldu<T, V>(dy + row * lddy + c, g);
            ldu<T, V>(x + row * ldx + c, xh);
            if (res) {
                float q[V];
                ldu<T, V>(res + row * ldr + c, q);
#pragma unroll
                for (int e = 0; e < V; ++e) xh[e] += q[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) xh[e] *= rs;
        };
        float dot = 0.f;
        for (int c = threadIdx.x * V; c < n; c += 256 * V) {
            const Group k = group<V>(c, n);
            float g[V], xh[V], ww[V];
            pair(k.c, g, xh);
            ldu<float, V>(w + k.c, ww);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (e >= k.skip) pp[k.c + e] = __builtin_fmaf(g[e], xh[e], pp[k.c + e]);
                g[e] *= ww[e];
            }
            dot += dot_v<V>(g, xh, k.skip);
        }
        dot = row_sum<4>(dot, sm, threadIdx.x >> 6) / (float)n;
        for (int c = threadIdx.x * V; c < n; c += 256 * V) {
            const Group k = group<V>(c, n);
            float g[V], xh[V], ww[V];
            pair(k.c, g, xh);
            ldu<float, V>(w + k.c, ww);
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = (g[e] * ww[e] - xh[e] * dot) * rs;
            if (dres) {
                ldu<T, V>(dres + row * ldd + k.c, ww);
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] += ww[e];
            }
            stu<T, V>(dx + (size_t)row * n + k.c, g);
        }
    }
}

// ---------------------------------------------------------------- C entries
// How a row is held: 16 bytes at a time (a value at a time where the row is shorter), up to 32 values per lane; a wave per row up
// to 64 * 16 values (no barrier), four waves above, up to 8192 values; nv = 0: the row does not fit the registers.
struct RmsPlan { int nv, wpr; };
static RmsPlan rms_plan(int dtype, int n) {
    const int V = 16 / (int)elem_size(dtype);
    for (int wpr = 1; wpr <= 4; wpr += 3)
        for (int nv = 1; V * nv <= (wpr == 1 ? 16 : 32); nv *= 2)
            if (n <= 64 * wpr * V * nv) return RmsPlan{nv, wpr};
    return RmsPlan{0, 4};
}
static const int RMS_BLOCKS = 1024;
static int rms_blocks(int rows, int wpr) {
    const int need = (rows + 4 / wpr - 1) / (4 / wpr);
    return need < RMS_BLOCKS ? (need > 0 ? need : 1) : RMS_BLOCKS;
}

// up to 16 values per lane with a wave per row, 8 to 32 with four
#define RMS_PICK(CALL) do { constexpr int M_ = 16 / VW;                                                                  \
                            if (n < VW) CALL(1, 1, 1);                                                                   \
                            else if (pl.wpr == 1) { if (pl.nv == 1) CALL(VW, 1, 1); else if (pl.nv == 2) CALL(VW, 2, 1); \
                                                    else CALL(VW, M_, 1); }                                              \
                            else { if (pl.nv < M_) CALL(VW, M_ / 2, 4); else if (pl.nv == M_) CALL(VW, M_, 4);           \
                                   else CALL(VW, 2 * M_, 4); } } while (0)

template <typename T>
static void rms_fwd_t(const RmsPlan& pl, const void* x, long long ldx, const void* res, long long ldr, const float* w,
                      int rows, int n, float eps, void* y, void* sum, float* rstd, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    if (!pl.nv) {
        hipLaunchKernelGGL((rms_fwd_long_kernel<T, VW>), dim3(rows), dim3(256), 0, stream, (const T*)x, ldx, (const T*)res, ldr, w,
                           n, eps, (T*)y, (T*)sum, rstd);
        return;
    }
    const dim3 grid(pl.wpr == 1 ? (rows + 3) / 4 : rows);
#define FWD_(V_, NV_, W_) hipLaunchKernelGGL((rms_fwd_kernel<T, V_, NV_, W_>), grid, dim3(256), 0, stream, (const T*)x, ldx, \
                                             (const T*)res, ldr, w, rows, n, eps, (T*)y, (T*)sum, rstd)
    RMS_PICK(FWD_);
#undef FWD_
}

template <typename T>
static void rms_bwd_t(const RmsPlan& pl, int blocks, const void* dy, long long lddy, const void* x, long long ldx,
                      const void* res, long long ldr, const float* w, const float* rstd, const void* dres, long long ldd, int rows, int n, void* dx,
                      float* part, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    if (!pl.nv) {
        hipLaunchKernelGGL((rms_bwd_long_kernel<T, VW>), dim3(blocks), dim3(256), 0, stream, (const T*)dy, lddy, (const T*)x, ldx,
                           (const T*)res, ldr, w, rstd, (const T*)dres, ldd, rows, n, (T*)dx, part);
        return;
    }
#define BWD_(V_, NV_, W_) hipLaunchKernelGGL((rms_bwd_kernel<T, V_, NV_, W_>), dim3(blocks), dim3(256), 0, stream,          \
                                             (const T*)dy, lddy, (const T*)x, ldx, (const T*)res, ldr, w, rstd, (const T*)dres, ldd, rows, n,   \
                                             (T*)dx, part)
    RMS_PICK(BWD_);
#undef BWD_
}

extern "C" int asr_rms_norm_fwd(int dtype, const void* x, long long ldx, const void* res, long long ldr, const float* w,
                                int rows, int n, float eps, void* y, void* sum, float* rstd, hipStream_t stream) {
    if (dtype < ASR_F32 || dtype > ASR_F16 || rows < 0 || n <= 0 || !w || !(eps >= 0.f)) return ASR_ERR_ARG;
    if (rows >= (1 << 24) || n > (1 << 25)) return ASR_ERR_LIMIT;       // 2^32 work items a launch
    if (rows == 0) return ASR_OK;
    if (!x || !y) return ASR_ERR_ARG;
    const RmsPlan pl = rms_plan(dtype, n);
    if (dtype == ASR_F32) rms_fwd_t<float>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    else if (dtype == ASR_BF16) rms_fwd_t<bf16_t>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    else rms_fwd_t<f16_t>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

// the parts of dw: one per workgroup, as many as a workgroup per row would need (how many rows share one depends on the type)
extern "C" size_t asr_rms_norm_bwd_ws_bytes(int rows, int n) {
    if (rows <= 0 || n <= 0) return 0;
    return (size_t)rms_blocks(rows, 4) * n * sizeof(float);
}

extern "C" int asr_rms_norm_bwd(int dtype, const void* dy, long long lddy, const void* x, long long ldx, const void* res,
                                long long ldr, const float* w, const float* rstd, const void* dres, long long ldd, int rows, int n, void* dx, float* dw,
                                void* ws, size_t ws_bytes, hipStream_t stream) {
    if (dtype < ASR_F32 || dtype > ASR_F16 || rows < 0 || n <= 0 || !w || !dw) return ASR_ERR_ARG;
    if (rows >= (1 << 24) || n > (1 << 25)) return ASR_ERR_LIMIT;       // 2^32 work items a launch
    if (rows && (!dy || !x || !rstd || !dx)) return ASR_ERR_ARG;
    if (rows && (!ws || ws_bytes < asr_rms_norm_bwd_ws_bytes(rows, n))) return ASR_ERR_WS;
    if ((uintptr_t)ws & 15) return ASR_ERR_ARG;
    int P = 0;
    if (rows) {
        const RmsPlan pl = rms_plan(dtype, n);
        const int blocks = rms_blocks(rows, pl.wpr);
        P = blocks;
        if (dtype == ASR_F32) rms_bwd_t<float>(pl, blocks, dy, lddy, x, ldx, res, ldr, w, rstd, dres, ldd, rows, n, dx, (float*)ws, stream);
        else if (dtype == ASR_BF16) rms_bwd_t<bf16_t>(pl, blocks, dy, lddy, x, ldx, res, ldr, w, rstd, dres, ldd, rows, n, dx, (float*)ws, stream);
        else rms_bwd_t<f16_t>(pl, blocks, dy, lddy, x, ldx, res, ldr, w, rstd, dres, ldd, rows, n, dx, (float*)ws, stream);
        ASR_CHECK_LAUNCH();
    }
    sum_partials((const float*)ws, n, P, n, dw, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}
