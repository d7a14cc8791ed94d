// Root-mean-square norm of rows with the residual's addition in front of it, forward and backward.
//   r = x (+ residual),   y = r rstd w,   rstd = 1 / sqrt(mean r^2 + eps)
//   g = dy w,   dr = (g - xhat mean(g xhat)) rstd (+ dres),   dw = sum_rows dy xhat,   xhat = r rstd
// HBM-bound: a pass reads and writes every tensor once, a row stays in registers between its two uses.  r is rounded to the
// activation type when it is stored; y is formed from the unrounded sum, and the backward pass forms that sum again from x and
// the residual (one more read than the stored r would cost, but gradients of what was computed: with the stored r, dw is off by
// the type's half step).  Measured at 36192 rows x 1024, bf16, with a residual: forward 50 us (5.9 TB/s of the 0.30 GB of its four
// tensors, some of them still in the Infinity Cache), backward 81 us (4.6 TB/s of 0.37 GB) and 5 for the parts of dw.
#include "seq_common.h"

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
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * STEP;
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = 0.f;
        if (c < n) {
            ldv<T, V>(x + row * ldx + c, v[i]);
            if (res) {
                float q[V];
                ldv<T, V>(res + row * ldr + c, q);
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] += q[e];
            }
            if (sum) stv<T, V>(sum + (size_t)row * n + c, v[i]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sq = __builtin_fmaf(v[i][e], v[i][e], sq);
    }
    sq = row_sum<WPR>(sq, sm, wv);
    const float rs = 1.0f / sqrtf(sq / (float)n + eps);
    if (rstd && (WPR == 1 ? lane : (int)threadIdx.x) == 0) rstd[row] = rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * STEP;
        if (c >= n) continue;
        float o[V], ww[V];
        ldv<float, V>(w + c, ww);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[i][e] * rs * ww[e];
        stv<T, V>(y + (size_t)row * n + c, o);
    }
}

// Rows longer than the registers hold: a workgroup per row, the sum formed twice.
template <typename T>
__global__ __launch_bounds__(256) void rms_fwd_long_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ res,
                                                           long long ldr, const float* __restrict__ w, int n, float eps,
                                                           T* __restrict__ y, T* __restrict__ sum,
                                                           float* __restrict__ rstd) {
    __shared__ float sm[4];
    const size_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    const T* rr = res ? res + row * ldr : nullptr;
    float sq = 0.f;
    for (int c = threadIdx.x; c < n; c += 256) {
        const float v = ldf(xr + c) + (rr ? ldf(rr + c) : 0.f);
        sq = __builtin_fmaf(v, v, sq);
    }
    sq = row_sum<4>(sq, sm, threadIdx.x >> 6);
    const float rs = 1.0f / sqrtf(sq / (float)n + eps);
    if (rstd && threadIdx.x == 0) rstd[row] = rs;
    for (int c = threadIdx.x; c < n; c += 256) {
        const float v = ldf(xr + c) + (rr ? ldf(rr + c) : 0.f);
        if (sum) stf(sum + row * n + c, v);
        stf(y + row * n + c, v * rs * w[c]);
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
            const int c = c0 + i * STEP;
#pragma unroll
            for (int e = 0; e < V; ++e) g[i][e] = xh[i][e] = 0.f;
            if (c < n) {
                float ww[V];
                ldv<T, V>(dy + row * lddy + c, g[i]);
                ldv<T, V>(x + row * ldx + c, xh[i]);
                if (res) {
                    float q[V];
                    ldv<T, V>(res + row * ldr + c, q);
#pragma unroll
                    for (int e = 0; e < V; ++e) xh[i][e] += q[e];
                }
                ldv<float, V>(w + c, ww);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    xh[i][e] *= rs;
                    dw[i][e] = __builtin_fmaf(g[i][e], xh[i][e], dw[i][e]);
                    g[i][e] *= ww[e];
                    dot = __builtin_fmaf(g[i][e], xh[i][e], dot);
                }
            }
        }
        dot = row_sum<WPR>(dot, sm, wv) / (float)n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = c0 + i * STEP;
            if (c >= n) continue;
            float o[V], d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = (g[i][e] - xh[i][e] * dot) * rs;
            if (dres) {
                ldv<T, V>(dres + row * ldd + c, d);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += d[e];
            }
            stv<T, V>(dx + (size_t)row * n + c, o);
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
        if (c < n)
#pragma unroll
            for (int e = 0; e < V; ++e) pp[c + e] = dw[i][e];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void rms_bwd_long_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                           long long ldx, const T* __restrict__ res, long long ldr,
                                                           const float* __restrict__ w,
                                                           const float* __restrict__ rstd, const T* __restrict__ dres,
                                                           long long ldd, int rows, int n, T* __restrict__ dx,
                                                           float* __restrict__ part) {
    __shared__ float sm[4];
    float* pp = part + (size_t)blockIdx.x * n;                 // this thread's columns only: no other thread reads them
    for (int c = threadIdx.x; c < n; c += 256) pp[c] = 0.f;
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const float rs = rstd[row];
        float dot = 0.f;
        for (int c = threadIdx.x; c < n; c += 256) {
            const float gy = ldf(dy + row * lddy + c), xh = (ldf(x + row * ldx + c) + (res ? ldf(res + row * ldr + c) : 0.f)) * rs;
            pp[c] = __builtin_fmaf(gy, xh, pp[c]);
            dot = __builtin_fmaf(gy * w[c], xh, dot);
        }
        dot = row_sum<4>(dot, sm, threadIdx.x >> 6) / (float)n;
        for (int c = threadIdx.x; c < n; c += 256) {
            const float g = ldf(dy + row * lddy + c) * w[c], xh = (ldf(x + row * ldx + c) + (res ? ldf(res + row * ldr + c) : 0.f)) * rs;
            float o = (g - xh * dot) * rs;
            if (dres) o += ldf(dres + row * ldd + c);
            stf(dx + (size_t)row * n + c, o);
        }
    }
}

// ---------------------------------------------------------------- C entries
static bool al(const void* p, int b) { return ((uintptr_t)p & (b - 1)) == 0; }

// How a row is held: V values at a time when the row's length, strides and addresses allow it, up to 32 values per lane (16 single
// ones); a wave per row up to 64 * 16 values (no barrier), four waves above; wide = 0: the row does not fit the registers.
struct RmsPlan { int vec, nv, wpr, wide; };
static RmsPlan rms_plan(int dtype, int n, bool vec) {
    const int V = vec ? 16 / (int)elem_size(dtype) : 1;
    RmsPlan p{vec, 0, 1, 1};
    const int most = 32 / V > 4 && V > 1 ? 4 : (V == 1 ? 16 : 32 / V);
    for (int wpr = 1; wpr <= 4; wpr += 3)
        for (int nv = 1; nv <= most; nv *= 2)
            if (n <= 64 * wpr * V * nv && (wpr == 4 || V * nv <= 16)) { p.nv = nv; p.wpr = wpr; return p; }
    p.wide = 0;
    return p;
}
static const int RMS_BLOCKS = 1024;
static int rms_blocks(int rows, int wpr) {
    const int need = (rows + 4 / wpr - 1) / (4 / wpr);
    return need < RMS_BLOCKS ? (need > 0 ? need : 1) : RMS_BLOCKS;
}

#define RMS_NV(V_, W_, CALL) switch (pl.nv) { case 1: CALL(V_, 1, W_); break; case 2: CALL(V_, 2, W_); break;   \
                                              case 4: CALL(V_, 4, W_); break; case 8: CALL(V_, 8, W_); break;   \
                                              default: CALL(V_, 16, W_); break; }
#define RMS_NV4(V_, W_, CALL) switch (pl.nv) { case 1: CALL(V_, 1, W_); break; case 2: CALL(V_, 2, W_); break;  \
                                               default: CALL(V_, 4, W_); break; }
#define RMS_PICK(CALL) do { if (pl.vec) { if (pl.wpr == 1) RMS_NV4(VW, 1, CALL) else RMS_NV4(VW, 4, CALL) }     \
                            else { if (pl.wpr == 1) RMS_NV(1, 1, CALL) else RMS_NV(1, 4, CALL) } } while (0)

template <typename T>
static void rms_fwd_t(const RmsPlan& pl, const void* x, long long ldx, const void* res, long long ldr, const float* w,
                      int rows, int n, float eps, void* y, void* sum, float* rstd, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    if (!pl.wide) {
        hipLaunchKernelGGL((rms_fwd_long_kernel<T>), dim3(rows), dim3(256), 0, stream, (const T*)x, ldx, (const T*)res, ldr, w,
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
    if (!pl.wide) {
        hipLaunchKernelGGL((rms_bwd_long_kernel<T>), dim3(blocks), dim3(256), 0, stream, (const T*)dy, lddy, (const T*)x, ldx,
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
    const int e = (int)elem_size(dtype), V = 16 / e;
    const bool vec = n % V == 0 && ldx % V == 0 && (!res || ldr % V == 0) && al(x, 16) && al(res, 16) && al(y, 16) &&
                     al(sum, 16) && al(w, 16);
    const RmsPlan pl = rms_plan(dtype, n, vec);
    if (dtype == ASR_F32) rms_fwd_t<float>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    else if (dtype == ASR_BF16) rms_fwd_t<bf16_t>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    else rms_fwd_t<f16_t>(pl, x, ldx, res, ldr, w, rows, n, eps, y, sum, rstd, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

// the parts of dw: one per workgroup, as many as a workgroup per row would need (how many rows share one depends on alignment)
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
        const int V = 16 / (int)elem_size(dtype);
        const bool vec = n % V == 0 && lddy % V == 0 && ldx % V == 0 && (!res || ldr % V == 0) && (!dres || ldd % V == 0) &&
                         al(dy, 16) && al(x, 16) && al(res, 16) && al(dres, 16) && al(dx, 16) && al(w, 16);
        const RmsPlan pl = rms_plan(dtype, n, vec);
        const int wpr = pl.wide ? pl.wpr : 4, blocks = rms_blocks(rows, wpr);
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
