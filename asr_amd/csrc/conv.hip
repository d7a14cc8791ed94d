// Short causal depthwise convolution over time with an optional SiLU, forward, backward and for single frames.
//   pre[s,d] = bias[d] + sum_k w[d,k] x[s-(K-1)+k, d],   out = silu(pre) or pre
// s counts the valid frames of a row in walking order; s < 0 is the carried state.  HBM-bound: one pass over x (and dout).
// A thread owns V channels and a run of frames and keeps the K-frame window in registers, so a frame is loaded once per run plus
// the K-1 frames in front of it.  Measured at T 4096, B 16, D 2048, bf16, K 4: forward 113 us (4.8 TB/s of the 0.54 GB it has to
// move), backward 210 us (3.8 TB/s of 0.81 GB) and 9 for the parts of dw; one f32 frame of 16 x 1024 channels 2.9 us, the launch.
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

// frames a thread walks: a multiple of K near n
__host__ __device__ constexpr int conv_run(int K, int n) { return (n + K - 1) / K * K; }

// the input at walking position s (>= -(K-1)) of row b
template <typename T, int V, int K>
__device__ __forceinline__ void load_x(const ConvArgs& p, int s, int len, int b, int d, float* o) {
    if (s >= 0) {
        const int f = p.reverse ? len - 1 - s : s;
        ldu<T, V>((const T*)p.x + f * p.x_st + b * p.x_sb + d, o);
    } else if (p.state) {
        ldu<T, V>((const T*)p.state + ((size_t)(s + K - 1) * p.B + b) * p.D + d, o);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = 0.f;
    }
}

template <typename T, int V> using Raw = typename AnyV<T, V>::type;
template <typename T, int V> __device__ __forceinline__ float raw_at(const Raw<T, V>& r, int e) {
    if constexpr (V == 1) return (float)r; else return (float)r[e];
}

// Where D is no multiple of V the last thread's channels are moved back to end with D: the ones that it shares with the thread in
// front are worked out and stored twice, the same.  (Measured before, a channel a thread: T 4096, B 8, D 2047, bf16, K 4, both
// passes, 261 us.)
// Frames are taken K at a time, so that a frame's place in the window (s mod K) is known when the code is compiled and nothing
// is moved from register to register.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs p) {
    const int dg = (blockIdx.x * 64 + (threadIdx.x & 63)) * V, d = min(dg, p.D - V);
    const int b = blockIdx.z;
    constexpr int RUN = conv_run(K, 16);
    const int s0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * RUN;
    if (dg >= p.D) return;
    const int len = row_len(p.lens, b, p.T);
    const int s1 = min(s0 + RUN, p.T);
    T* out = (T*)p.out + b * p.o_sb + d;
    if (s0 < len) {
        float w[K][V], win[K][V], bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            bias[e] = p.bias ? p.bias[d + e] : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][e] = p.w[(size_t)(d + e) * K + k];
        }
        // the frame at s0 + i sits in win[(i + K - 1) % K]
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_x<T, V, K>(p, s0 - (K - 1) + k, len, b, d, win[k]);
        const int se = min(s1, len);
        const auto frame = [&](int s, int j) {
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float a = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][e], win[(j + k) % K][e], a);
                y[e] = p.act ? silu_(a) : a;
            }
            stu<T, V>(out + (p.reverse ? len - 1 - s : s) * p.o_st, y);
        };
        // whole windows: the next one is on its way while one is worked on
        int s = s0;
        Raw<T, V> nx[K];
        const T* px = (const T*)p.x + b * p.x_sb + d;
        const auto fetch = [&](int s) {
#pragma unroll
            for (int j = 0; j < K; ++j) nx[j] = *(const Raw<T, V>*)(px + (p.reverse ? len - 1 - s - j : s + j) * p.x_st);
        };
        if (s + K <= se) fetch(s);
        for (; s + K <= se; s += K) {
            Raw<T, V> cx[K];
#pragma unroll
            for (int j = 0; j < K; ++j) cx[j] = nx[j];
            if (s + 2 * K <= se) fetch(s + K);
#pragma unroll
            for (int j = 0; j < K; ++j) {
#pragma unroll
                for (int e = 0; e < V; ++e) win[(j + K - 1) % K][e] = raw_at<T, V>(cx[j], e);
                frame(s + j, j);
            }
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            if (s + j >= se) break;
            load_x<T, V, K>(p, s + j, len, b, d, win[(j + K - 1) % K]);
            frame(s + j, j);
        }
    }
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = max(s0, len); s < s1; ++s) stu<T, V>(out + s * p.o_st, zero);
    // the carried state: the inputs at the last K-1 walking positions (positions in front of the row stay state rows)
    if (p.state_out && s0 == 0) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            float v[V];
            load_x<T, V, K>(p, len - (K - 1) + k, len, b, d, v);
            stu<T, V>((T*)p.state_out + ((size_t)k * p.B + b) * p.D + d, v);
        }
    }
}

// dx and the parts of dw / db.  A thread walks q = s0 .. s0+run+K-2: it forms dpre[q], adds dpre[q] x to dw for the frames it
// owns (q < s0+run) and, K-1 frames later, has all the terms of dx[q-(K-1)].
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs p) {
    __shared__ float sm[3][K + 1][64 * V];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int dg = (blockIdx.x * 64 + lane) * V, d = min(dg, p.D - V);
    const int b = blockIdx.z;
    constexpr int RUN = conv_run(K, 32);
    const int s0 = (blockIdx.y * 4 + wv) * RUN;
    const bool on = dg < p.D;
    const int len = row_len(p.lens, b, p.T);
    const int s1 = min(s0 + RUN, p.T);
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
        // x and dpre of the frame at s0 + i sit in [(i + K - 1) % K]
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_x<T, V, K>(p, s0 - (K - 1) + k, len, b, d, win[k]);
        const int own = min(s1, len);              // dx rows of this thread: [s0, own), and the state rows if s0 == 0
        const T* pdo = (const T*)p.dout + b * p.do_sb + d;
        // dpre of frame q (its x is in the window) from dout, and its share of dw
        const auto gradient = [&](int j, const float (&g)[V], bool mine) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float a = bias[e], v = g[e];
#pragma unroll
                for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][e], win[(j + k) % K][e], a);
                if (p.act) v *= dsilu_(a, sigm_(a));
                dp[(j + K - 1) % K][e] = v;
                if (mine) {
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k][e] = __builtin_fmaf(v, win[(j + k) % K][e], dw[k][e]);
                    dw[K][e] += v;
                }
            }
        };
        // dx[s], s = q - (K-1): sum_i w[K-1-i] dpre[s+i]
        const auto emit = [&](int s, int j) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                o[e] = 0.f;
#pragma unroll
                for (int i = 0; i < K; ++i) o[e] = __builtin_fmaf(w[K - 1 - i][e], dp[(j + i) % K][e], o[e]);
            }
            const int r = s - (len - (K - 1));     // this position's row of the carried-out state
            if (p.dstate_out && r >= 0) {
                float ds[V];
                ldu<T, V>((const T*)p.dstate_out + ((size_t)r * p.B + b) * p.D + d, ds);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += ds[e];
            }
            if (s >= 0) stu<T, V>((T*)p.dx + ((size_t)(p.reverse ? len - 1 - s : s) * p.B + b) * p.D + d, o);
            else if (p.dstate) stu<T, V>((T*)p.dstate + ((size_t)(s + K - 1) * p.B + b) * p.D + d, o);
        };
        // whole windows: the next one is on its way while one is worked on
        int q = s0;
        Raw<T, V> nx[K], ng[K];
        const T* pxb = (const T*)p.x + b * p.x_sb + d;
        const auto fetch = [&](int q) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const long long f = p.reverse ? len - 1 - q - j : q + j;
                nx[j] = *(const Raw<T, V>*)(pxb + f * p.x_st);
                ng[j] = *(const Raw<T, V>*)(pdo + f * p.do_st);
            }
        };
        if (q + K <= own) fetch(q);
        for (; q + K <= own; q += K) {
            Raw<T, V> cx[K], cg[K];
#pragma unroll
            for (int j = 0; j < K; ++j) { cx[j] = nx[j]; cg[j] = ng[j]; }
            if (q + 2 * K <= own) fetch(q + K);
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float g[V];
#pragma unroll
                for (int e = 0; e < V; ++e) { win[(j + K - 1) % K][e] = raw_at<T, V>(cx[j], e); g[e] = raw_at<T, V>(cg[j], e); }
                gradient(j, g, true);
                if (q + j - (K - 1) >= s0 || s0 == 0) emit(q + j - (K - 1), j);
            }
        }
        // up to K-1 owned frames and the K-1 behind them
        for (; q < own + K - 1; q += K) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (q + j >= own + K - 1) break;
                if (q + j < len) {
                    float g[V];
                    load_x<T, V, K>(p, q + j, len, b, d, win[(j + K - 1) % K]);
                    ldu<T, V>(pdo + (p.reverse ? len - 1 - q - j : q + j) * p.do_st, g);
                    gradient(j, g, q + j < own);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) dp[(j + K - 1) % K][e] = 0.f;
                }
                if (q + j - (K - 1) >= s0 || s0 == 0) emit(q + j - (K - 1), j);
            }
        }
    }
    if (on) {
        const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int s = max(s0, len); s < s1; ++s) stu<T, V>((T*)p.dx + ((size_t)s * p.B + b) * p.D + d, zero);
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
static bool al(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
static bool al16(const void* p) { return al(p, 16); }
static bool stride_ok(long long st, int V) { return st % V == 0; }

// A thread walks 16 frames forward, 32 backward (rounded up to whole windows): the K-1 frames read twice cost little, and the
// chip is full.
static int run_groups(int T, int K, int n) {
    const int run = 4 * conv_run(K, n);
    return T > 0 ? (T + run - 1) / run : 1;
}

#define CONV_K(K_, ...) case K_: { constexpr int K = K_; __VA_ARGS__; break; }
#define CONV_KS(...) switch (k_) { CONV_K(2, __VA_ARGS__) CONV_K(3, __VA_ARGS__) CONV_K(4, __VA_ARGS__) \
                                   CONV_K(5, __VA_ARGS__) CONV_K(6, __VA_ARGS__) CONV_K(7, __VA_ARGS__) \
                                   CONV_K(8, __VA_ARGS__) default: return ASR_ERR_LIMIT; }

// Bytes a thread: 16 forward (8 of a 16-bit type from 6 taps on, whose two windows would not leave registers for two waves per SIMD), 8
// backward: there two windows of x and dout on their way, the windows of x and dpre and the parts of dw are 150 registers at 8
// bytes, 250 at 16 (one wave per SIMD); 4 of a 16-bit type from 6 taps on.  Measured for both passes: backward 8 / 16 / 4 bytes, T 4096,
// B 16, D 2048, bf16, K 4: 339 / 398 / 344 us; T 2262, B 16, D 1024, f32: 135 / 139 / 138 us; the rule for 6 taps and more, T 4096,
// B 8, D 2048, bf16: K 6 205 -> 180 us, K 7 214 -> 211, K 8 366 -> 246.
// Few channels leave most lanes of a wave without any at that width: one value a thread below 24 (32) threads' worth.  T 4096, B 8,
// bf16, K 4, D 99: 35 us at full width, 27 so; D 199: 37.5 and 35.3 (B 64: 166 and 226).
template <typename T>
static int conv_fwd_t(const ConvArgs& p, int k_, hipStream_t stream) {
    CONV_KS(
        constexpr int VW = (sizeof(T) == 2 && K > 5 ? 8 : 16) / sizeof(T);
        const bool vec = p.D >= 24 * VW; const int V = vec ? VW : 1;
        const dim3 grid((p.D + 64 * V - 1) / (64 * V), run_groups(p.T, K, 16), p.B);
        if (vec) hipLaunchKernelGGL((conv_fwd_kernel<T, VW, K>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((conv_fwd_kernel<T, 1, K>), grid, dim3(256), 0, stream, p);)
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}
template <typename T>
static int conv_bwd_t(const ConvArgs& p, int k_, hipStream_t stream) {
    CONV_KS(
        constexpr int VW = (sizeof(T) == 2 && K > 5 ? 4 : 8) / sizeof(T);
        const bool vec = p.D >= 32 * VW; const int V = vec ? VW : 1;
        const dim3 grid((p.D + 64 * V - 1) / (64 * V), run_groups(p.T, K, 32), p.B);
        if (vec) hipLaunchKernelGGL((conv_bwd_kernel<T, VW, K>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((conv_bwd_kernel<T, 1, K>), grid, dim3(256), 0, stream, p);)
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

static int conv_dims_ok(int dtype, int T, int B, int D, int K) {
    if (dtype < ASR_F32 || dtype > ASR_F16 || T < 0 || B < 0 || D <= 0 || K < 2) return ASR_ERR_ARG;
    // grid axes y and z end at 65535, a launch at 2^32 work items
    if (K > 8 || B > 65535 || D > (1 << 20) || T > (1 << 21)) return ASR_ERR_LIMIT;
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
    return (size_t)run_groups(T, K, 32) * B * (K + 1) * (size_t)D * sizeof(float);
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
    if ((uintptr_t)ws & 15) return ASR_ERR_ARG;
    int P = 0;
    if (B) {
        ConvArgs p{};
        p.T = T; p.B = B; p.D = D; p.reverse = reverse; p.act = act; p.lens = lens; p.x = x; p.x_st = x_st; p.x_sb = x_sb;
        p.dout = dout; p.do_st = do_st; p.do_sb = do_sb; p.w = w; p.bias = bias; p.state = state;
        p.dstate_out = dstate_out; p.dx = dx; p.dstate = dstate; p.part = (float*)ws;
        const int e = dtype == ASR_F32 ? conv_bwd_t<float>(p, K, stream)
                    : dtype == ASR_BF16 ? conv_bwd_t<bf16_t>(p, K, stream) : conv_bwd_t<f16_t>(p, K, stream);
        if (e) return e;
        P = run_groups(T, K, 32) * B;
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
    if ((long long)B * D > (1ll << 31)) return ASR_ERR_LIMIT;
    if (!w) return ASR_ERR_ARG;
    if (!B) return ASR_OK;
    if (!x || !state || !out) return ASR_ERR_ARG;
    if (dtype == ASR_F32) return conv_step_t<float>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
    if (dtype == ASR_BF16) return conv_step_t<bf16_t>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
    return conv_step_t<f16_t>(B, D, K, x, x_sb, state, w, bias, act, out, o_sb, stream);
}
