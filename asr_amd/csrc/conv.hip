// Short causal depthwise convolution over time with an optional SiLU, forward, backward and for single frames.
//   pre[s,d] = bias[d] + sum_k w[d,k] x[s-(K-1)+k, d],   out = silu(pre) or pre
// s counts the valid frames of a row in walking order; s < 0 is the carried state.  HBM-bound: one pass over x (and dout).
// A thread owns V channels (16 bytes) and a run of frames and keeps the K-frame window in registers, so a frame is loaded
// once per run plus the K-1 frames in front of it.
#include "seq_common.h"

struct ConvArgs {
    int T, B, D, reverse, act;
    const int* lens;
    const void* x; long long x_st, x_sb;
    const void* dout; long long do_st, do_sb;
    const float *w, *bias;
    const void* state;          // (K-1,B,D)
    void* out; long long o_st, o_sb;
    void* state_out;            // (K-1,B,D)
    const void* dstate_out;     // (K-1,B,D)
    void *dx, *dstate;          // (T,B,D), (K-1,B,D)
    float* part;                // (runs groups * B, K+1, D)
};

// the input at walking position s (>= -(K-1)) of row b
template <typename T, int V, int K>
__device__ __forceinline__ void load_x(const ConvArgs& p, int s, int len, int b, int d, float* o) {
    if (s >= 0) {
        const int f = p.reverse ? len - 1 - s : s;
        ldv<T, V>((const T*)p.x + f * p.x_st + b * p.x_sb + d, o);
    } else if (p.state) {
        ldv<T, V>((const T*)p.state + ((size_t)(s + K - 1) * p.B + b) * p.D + d, o);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = 0.f;
    }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs p, int run) {
    const int d = (blockIdx.x * 64 + (threadIdx.x & 63)) * V;
    const int b = blockIdx.z;
    const int s0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * run;
    if (d >= p.D) return;
    const int len = row_len(p.lens, b, p.T);
    const int s1 = min(s0 + run, p.T);
    T* out = (T*)p.out + b * p.o_sb + d;
    if (s0 < len) {
        float w[K][V], win[K][V], bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            bias[e] = p.bias ? p.bias[d + e] : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][e] = p.w[(size_t)(d + e) * K + k];
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_x<T, V, K>(p, s0 - (K - 1) + k, len, b, d, win[k]);
        const int se = min(s1, len);
        for (int s = s0; s < se; ++s) {
            load_x<T, V, K>(p, s, len, b, d, win[K - 1]);
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float a = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][e], win[k][e], a);
                y[e] = p.act ? silu_(a) : a;
            }
            stv<T, V>(out + (p.reverse ? len - 1 - s : s) * p.o_st, y);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) win[k][e] = win[k + 1][e];
        }
    }
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = max(s0, len); s < s1; ++s) stv<T, V>(out + s * p.o_st, zero);
    // the carried state: the inputs at the last K-1 walking positions (positions in front of the row stay state rows)
    if (p.state_out && s0 == 0) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            float v[V];
            load_x<T, V, K>(p, len - (K - 1) + k, len, b, d, v);
            stv<T, V>((T*)p.state_out + ((size_t)k * p.B + b) * p.D + d, v);
        }
    }
}

// dx and the parts of dw / db.  A thread walks e = s0 .. s0+run+K-2: it forms dpre[e], adds dpre[e] x to dw for the frames it
// owns (e < s0+run) and, K-1 frames later, has all the terms of dx[e-(K-1)].
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs p, int run) {
    __shared__ float sm[3][K + 1][64 * V];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int d = (blockIdx.x * 64 + lane) * V;
    const int b = blockIdx.z;
    const int s0 = (blockIdx.y * 4 + wv) * run;
    const bool on = d < p.D;
    const int len = row_len(p.lens, b, p.T);
    const int s1 = min(s0 + run, p.T);
    float dw[K + 1][V];
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k][e] = 0.f;
    if (on && (s0 < len || s0 == 0)) {
        float w[K][V], win[K][V], dp[K][V], bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            bias[e] = p.bias ? p.bias[d + e] : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) { w[k][e] = p.w[(size_t)(d + e) * K + k]; dp[k][e] = 0.f; }
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_x<T, V, K>(p, s0 - (K - 1) + k, len, b, d, win[k]);
        const int own = min(s1, len);              // dx rows of this thread: [s0, own), and the state rows if s0 == 0
        for (int q = s0; q < own + K - 1; ++q) {
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) dp[k][e] = dp[k + 1][e];
            if (q < len) {
                float g[V];
                load_x<T, V, K>(p, q, len, b, d, win[K - 1]);
                ldv<T, V>((const T*)p.dout + (p.reverse ? len - 1 - q : q) * p.do_st + b * p.do_sb + d, g);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float a = bias[e];
#pragma unroll
                    for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][e], win[k][e], a);
                    if (p.act) g[e] *= dsilu_(a, sigm_(a));
                    dp[K - 1][e] = g[e];
                    if (q < own) {
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][e] = __builtin_fmaf(g[e], win[k][e], dw[k][e]);
                        dw[K][e] += g[e];
                    }
                }
#pragma unroll
                for (int k = 0; k < K - 1; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) win[k][e] = win[k + 1][e];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) dp[K - 1][e] = 0.f;
            }
            const int s = q - (K - 1);             // dx[s] = sum_j w[K-1-j] dpre[s+j]
            if (s < s0 && s0 != 0) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                o[e] = 0.f;
#pragma unroll
                for (int j = 0; j < K; ++j) o[e] = __builtin_fmaf(w[K - 1 - j][e], dp[j][e], o[e]);
            }
            const int r = s - (len - (K - 1));     // this position's row of the carried-out state
            if (p.dstate_out && r >= 0) {
                float ds[V];
                ldv<T, V>((const T*)p.dstate_out + ((size_t)r * p.B + b) * p.D + d, ds);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += ds[e];
            }
            if (s >= 0) stv<T, V>((T*)p.dx + ((size_t)(p.reverse ? len - 1 - s : s) * p.B + b) * p.D + d, o);
            else if (p.dstate) stv<T, V>((T*)p.dstate + ((size_t)(s + K - 1) * p.B + b) * p.D + d, o);
        }
    }
    if (on) {
        const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int s = max(s0, len); s < s1; ++s) stv<T, V>((T*)p.dx + ((size_t)s * p.B + b) * p.D + d, zero);
    }
    // four runs of a workgroup are joined in order
    if (wv) {
#pragma unroll
        for (int k = 0; k <= K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) sm[wv - 1][k][e * 64 + lane] = dw[k][e];
    }
    __syncthreads();
    if (wv == 0 && on) {
        float* out = p.part + ((size_t)blockIdx.y * gridDim.z + b) * (K + 1) * p.D;
#pragma unroll
        for (int k = 0; k <= K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = dw[k][e] + sm[0][k][e * 64 + lane] + sm[1][k][e * 64 + lane] + sm[2][k][e * 64 + lane];
                // dw as (D,K) rows behind one another, then db
                out[k < K ? (size_t)(d + e) * K + k : (size_t)p.D * K + d + e] = t;
            }
    }
}

// One frame: the window is (state rows, x); the state moves on by one frame in place.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_step_kernel(const T* __restrict__ x, long long x_sb, T* state,
                                                        const float* __restrict__ w, const float* __restrict__ bias,
                                                        int act, T* __restrict__ out, long long o_sb, int B, int D) {
    const int per = D / V;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)B * per) return;
    const int b = (int)(i / per), d = (int)(i % per) * V;
    float win[K][V], y[V];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) ldv<T, V>(state + ((size_t)k * B + b) * D + d, win[k]);
    ldv<T, V>(x + b * x_sb + d, win[K - 1]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float a = bias ? bias[d + e] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[(size_t)(d + e) * K + k], win[k][e], a);
        y[e] = act ? silu_(a) : a;
    }
    stv<T, V>(out + b * o_sb + d, y);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) stv<T, V>(state + ((size_t)k * B + b) * D + d, win[k + 1]);
}

// ---------------------------------------------------------------- C entries
static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool stride_ok(long long st, int V) { return st % V == 0; }

// frames a thread walks: long enough that the K-1 frames read twice cost little, short enough that the chip is full
static const int RUN_FWD = 16, RUN_BWD = 32;
static int run_groups(int T, int run) { return T > 0 ? (T + 4 * run - 1) / (4 * run) : 1; }

#define CONV_K(K_, ...) case K_: { constexpr int K = K_; __VA_ARGS__; break; }
#define CONV_KS(...) switch (k_) { CONV_K(2, __VA_ARGS__) CONV_K(3, __VA_ARGS__) CONV_K(4, __VA_ARGS__) \
                                   CONV_K(5, __VA_ARGS__) CONV_K(6, __VA_ARGS__) CONV_K(7, __VA_ARGS__) \
                                   CONV_K(8, __VA_ARGS__) default: return ASR_ERR_LIMIT; }

template <typename T>
static int conv_fwd_t(const ConvArgs& p, int k_, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    const bool vec = p.D % VW == 0 && al16(p.x) && al16(p.out) && al16(p.state) && al16(p.state_out) &&
                     stride_ok(p.x_st, VW) && stride_ok(p.x_sb, VW) && stride_ok(p.o_st, VW) && stride_ok(p.o_sb, VW);
    const int run = RUN_FWD;
    const int V = vec ? VW : 1;
    const dim3 grid((p.D + 64 * V - 1) / (64 * V), run_groups(p.T, run), p.B);
    if (vec) { CONV_KS(hipLaunchKernelGGL((conv_fwd_kernel<T, VW, K>), grid, dim3(256), 0, stream, p, run)) }
    else { CONV_KS(hipLaunchKernelGGL((conv_fwd_kernel<T, 1, K>), grid, dim3(256), 0, stream, p, run)) }
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}
template <typename T>
static int conv_bwd_t(const ConvArgs& p, int k_, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    const bool vec = p.D % VW == 0 && al16(p.x) && al16(p.dout) && al16(p.state) && al16(p.dstate_out) && al16(p.dx) &&
                     al16(p.dstate) && stride_ok(p.x_st, VW) && stride_ok(p.x_sb, VW) && stride_ok(p.do_st, VW) &&
                     stride_ok(p.do_sb, VW);
    const int run = RUN_BWD;
    const int V = vec ? VW : 1;
    const dim3 grid((p.D + 64 * V - 1) / (64 * V), run_groups(p.T, run), p.B);
    if (vec) { CONV_KS(hipLaunchKernelGGL((conv_bwd_kernel<T, VW, K>), grid, dim3(256), 0, stream, p, run)) }
    else { CONV_KS(hipLaunchKernelGGL((conv_bwd_kernel<T, 1, K>), grid, dim3(256), 0, stream, p, run)) }
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

static int conv_dims_ok(int dtype, int T, int B, int D, int K) {
    if (dtype < ASR_F32 || dtype > ASR_F16 || T < 0 || B < 0 || D <= 0 || K < 2) return ASR_ERR_ARG;
    if (K > 8 || B > 65535 || D > (1 << 24) || T > (1 << 21)) return ASR_ERR_LIMIT;   // grid axes y, z end at 65535
    return ASR_OK;
}

extern "C" int asr_conv_fwd(int dtype, int T, int B, int D, int K, const void* x, long long x_st, long long x_sb,
                            const float* w, const float* bias, const void* state, const int* lens, int act, int reverse,
                            void* out, long long o_st, long long o_sb, void* state_out, hipStream_t stream) {
    if (int e = conv_dims_ok(dtype, T, B, D, K)) return e;
    if (!w || (state_out && state_out == state)) return ASR_ERR_ARG;
    if (B == 0 || (T == 0 && !state_out)) return ASR_OK;
    if (T && (!x || !out)) return ASR_ERR_ARG;
    ConvArgs p{};
    p.T = T; p.B = B; p.D = D; p.reverse = reverse; p.act = act; p.lens = lens; p.x = x; p.x_st = x_st; p.x_sb = x_sb;
    p.w = w; p.bias = bias; p.state = state; p.out = out; p.o_st = o_st; p.o_sb = o_sb; p.state_out = state_out;
    if (dtype == ASR_F32) return conv_fwd_t<float>(p, K, stream);
    if (dtype == ASR_BF16) return conv_fwd_t<bf16_t>(p, K, stream);
    return conv_fwd_t<f16_t>(p, K, stream);
}

extern "C" size_t asr_conv_bwd_ws_bytes(int T, int B, int D, int K) {
    if (T < 0 || B < 0 || D <= 0 || K < 2) return 0;
    return (size_t)run_groups(T, RUN_BWD) * B * (K + 1) * (size_t)D * sizeof(float);
}

extern "C" int asr_conv_bwd(int dtype, int T, int B, int D, int K, const void* dout, long long do_st, long long do_sb,
                            const void* x, long long x_st, long long x_sb, const float* w, const float* bias,
                            const void* state, const int* lens, int act, int reverse, const void* dstate_out, void* dx,
                            float* dwb, void* dstate, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (int e = conv_dims_ok(dtype, T, B, D, K)) return e;
    if (!w || !dwb || (dstate && dstate == dstate_out)) return ASR_ERR_ARG;
    const size_t n = (size_t)D * (K + 1);
    if (T && B && (!x || !dout || !dx)) return ASR_ERR_ARG;
    if (ws_bytes < asr_conv_bwd_ws_bytes(T, B, D, K) || (B && !ws)) return ASR_ERR_WS;
    int P = 0;
    if (B) {
        ConvArgs p{};
        p.T = T; p.B = B; p.D = D; p.reverse = reverse; p.act = act; p.lens = lens; p.x = x; p.x_st = x_st; p.x_sb = x_sb;
        p.dout = dout; p.do_st = do_st; p.do_sb = do_sb; p.w = w; p.bias = bias; p.state = state;
        p.dstate_out = dstate_out; p.dx = dx; p.dstate = dstate; p.part = (float*)ws;
        const int e = dtype == ASR_F32 ? conv_bwd_t<float>(p, K, stream)
                    : dtype == ASR_BF16 ? conv_bwd_t<bf16_t>(p, K, stream) : conv_bwd_t<f16_t>(p, K, stream);
        if (e) return e;
        P = run_groups(T, RUN_BWD) * B;
    }
    sum_partials((const float*)ws, n, P, n, dwb, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

template <typename T>
static int conv_step_t(int B, int D, int k_, const void* x, long long x_sb, void* state, const float* w, const float* bias,
                       int act, void* out, long long o_sb, hipStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    const bool vec = D % VW == 0 && al16(x) && al16(out) && al16(state) && stride_ok(x_sb, VW) && stride_ok(o_sb, VW);
    const size_t n = (size_t)B * (D / (vec ? VW : 1));
    const dim3 grid((unsigned)((n + 255) / 256));
    if (vec) { CONV_KS(hipLaunchKernelGGL((conv_step_kernel<T, VW, K>), grid, dim3(256), 0, stream, (const T*)x, x_sb,
                                           (T*)state, w, bias, act, (T*)out, o_sb, B, D)) }
    else { CONV_KS(hipLaunchKernelGGL((conv_step_kernel<T, 1, K>), grid, dim3(256), 0, stream, (const T*)x, x_sb,
                                       (T*)state, w, bias, act, (T*)out, o_sb, B, D)) }
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

extern "C" int asr_conv_step(int dtype, int B, int D, int K, const void* x, long long x_sb, void* state, const float* w,
                             const float* bias, int act, void* out, long long o_sb, hipStream_t stream) {
    if (int e = conv_dims_ok(dtype, 1, B, D, K)) return e;
    if (!w) return ASR_ERR_ARG;
    if (!B) return ASR_OK;
    if (!x || !state || !out) return ASR_ERR_ARG;
    if (dtype == ASR_F32) return conv_step_t<float>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
    if (dtype == ASR_BF16) return conv_step_t<bf16_t>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
    return conv_step_t<f16_t>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
}
