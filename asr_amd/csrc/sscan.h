// Selective state-space scan: what its forward and backward kernels share.
//   delta = softplus(dt + dt_bias)  (or dt + dt_bias),   a = exp(delta A)
//   h[s] = a h[s-1] + (delta x) B[s],   y = sum_n C[s] h[s] + D x,   out = y silu(z)  (or y)
// per row b, channel d and state n; B and C are shared by the channels of a group.
//
// A workgroup is 64 channels (one per lane, so every activation row is one coalesced access) times all states: each of its
// four waves holds SPL states per channel in registers (NB times over for more than 16 states) and walks TS frames per tile.
// What does not depend on the state (delta, delta x, gates) is formed once per (frame, channel) by the four waves together
// and handed over in LDS, B and C as broadcast reads.
#pragma once
#include "seq_common.h"
#include "../../include/asr_amd.h"      // asr_sscan_desc

#define SSCAN_TS 16          // frames of a tile; the training forward pass saves the state in front of every tile

struct SscanArgs {
    int T, B, D, N, G, dpg, tpg;     // dpg: channels of a group, tpg: 64-channel tiles of a group
    int reverse, softplus;
    int S, tpc;                      // time is cut into S chunks of tpc tiles each
    int np;                          // states, padded to what the waves hold
    int vec;                         // single frames: the state and A can be read 16 bytes at a time
    const int* lens;
    const void *x, *dt, *z, *Bm, *Cm;
    long long x_st, x_sb, dt_st, dt_sb, z_st, z_sb, b_st, b_sb, b_sg, c_st, c_sb, c_sg;
    const float *A, *Dk, *bias, *h0;
    void* out; long long o_st, o_sb;
    float *h_last, *ckpt;
    const void* dout; long long do_st, do_sb;
    const float* dh_last;
    void *dx, *ddt, *dz;
    float* dh0;
    float *c_h, *c_ds;               // per chunk: its own final state (or first adjoint), its sum of delta
    float *part_bc, *part_a, *part_d, *part_b;
};

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f

// states a wave holds per channel (SPL) and how often (NB): 4 waves * SPL * NB >= N
static inline int sscan_spl(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : 4; }
static inline int sscan_nb(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }
static inline int sscan_np(int N) { return 4 * sscan_spl(N) * sscan_nb(N); }
static inline int sscan_tiles(int T) { return (T + SSCAN_TS - 1) / SSCAN_TS; }

int sscan_chunks(int T, int B, int D, int G, int backward);
int sscan_fill(const asr_sscan_desc* d, SscanArgs* p, int backward);

// What a thread of the workgroup knows about its place.
struct Place {
    int lane, w, b, g, ct, d, len, nt, t0, t1, k;
    bool on;
};
__device__ __forceinline__ Place sscan_place(const SscanArgs& p) {
    Place q;
    q.lane = threadIdx.x & 63;
    q.w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    q.g = blockIdx.x / p.tpg;
    q.ct = blockIdx.x % p.tpg;
    q.b = blockIdx.y;
    q.k = blockIdx.z;
    const int dl = q.ct * 64 + q.lane;
    q.on = dl < p.dpg;
    q.d = q.g * p.dpg + (q.on ? dl : p.dpg - 1);
    q.len = row_len(p.lens, q.b, p.T);
    q.nt = (q.len + SSCAN_TS - 1) / SSCAN_TS;          // tiles that hold a valid frame
    q.t0 = q.k * p.tpc;
    q.t1 = min(q.t0 + p.tpc, q.nt);                     // this chunk's tiles; none if t1 <= t0
    return q;
}

// A log2(e), finite: a delta of zero (a padding frame's, or a valid one's) must leave exp(delta A) at 1 whatever the rate is.
__device__ __forceinline__ float rate2(float A) {
    const float v = A * LOG2E;
    return v < -3.0e38f ? -3.0e38f : v > 3.0e38f ? 3.0e38f : v;        // NaN stays
}

// h 2^k, a state carried over a whole chunk.  In three factors: of a state that grows (k > 0) 2^k may overflow where h 2^k does
// not, or where h is zero and stays so.  (From k = 381 on any h but zero is infinite.)
__device__ __forceinline__ float carried(float h, float k) {
    const float e = __builtin_amdgcn_exp2f(fminf(k, 381.f) * (1.f / 3.f));
    return h * e * e * e;
}

// A thread's share of a tile's rows: frames w*4 .. w*4+3 of its channel.  `base` is the row's own address (uniform), `off` the
// channel's byte offset, so an access is a scalar address plus a 32-bit lane offset.  FULL: all frames are valid.  Otherwise
// frames behind the row read its last one, and what they give is thrown away by the caller.
template <bool FULL, typename TY>
__device__ __forceinline__ void fetch_rows(TY (&o)[4], const TY* base, long long st, int s0, int len, int reverse, unsigned off) {
    const char* b = (const char*)base;
    const long long sb = st * (long long)sizeof(TY);
    if (FULL) {
        const char* r = b + (long long)(reverse ? len - 1 - s0 : s0) * sb;
        const long long step = reverse ? -sb : sb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = *(const TY*)(r + off);
            r += step;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = min(s0 + i, len - 1);
            o[i] = *(const TY*)(b + (long long)(reverse ? len - 1 - s : s) * sb + off);
        }
    }
}
// The same frames of an output: padding rows in front of p.T get zeros.
template <bool FULL, typename TY>
__device__ __forceinline__ void store_rows(TY* base, long long st, int s0, int len, int T, int reverse, unsigned off,
                                           const float (&v)[4]) {
    char* b = (char*)base;
    const long long sb = st * (long long)sizeof(TY);
    if (FULL) {
        char* r = b + (long long)(reverse ? len - 1 - s0 : s0) * sb;
        const long long step = reverse ? -sb : sb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *(TY*)(r + off) = (TY)v[i];
            r += step;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i;
            const bool ok = s < len;
            if (s < T) *(TY*)(b + (long long)((reverse && ok) ? len - 1 - s : s) * sb + off) = (TY)(ok ? v[i] : 0.f);
        }
    }
}
// Its share of B and C: TS frames x NP states, one value every 256 of them.
template <typename TY, int NP, int RB>
__device__ __forceinline__ void fetch_states(TY (&o)[RB], const TY* base, long long st, int tile, int len, int reverse, int N) {
#pragma unroll
    for (int k = 0; k < RB; ++k) {
        const int e = threadIdx.x + k * 256;
        const int s = min(tile * SSCAN_TS + min(e / NP, SSCAN_TS - 1), len - 1);
        o[k] = base[(reverse ? len - 1 - s : s) * st + min(e % NP, N - 1)];
    }
}
template <typename TY, int NP, int RB>
__device__ __forceinline__ void place_states(float* dst, const TY (&o)[RB], int tile, int len, int N) {
#pragma unroll
    for (int k = 0; k < RB; ++k) {
        const int e = threadIdx.x + k * 256;
        if (RB * 256 == SSCAN_TS * NP || e < SSCAN_TS * NP)
            dst[e] = (tile * SSCAN_TS + e / NP < len && e % NP < N) ? (float)o[k] : 0.f;
    }
}
// The kernel's arguments, read again where they are used: kept in scalar registers over the whole loop they do not fit, and
// the compiler moves them through vector registers, lane by lane.
typedef const __attribute__((address_space(4))) SscanArgs* KArgs;
__device__ __forceinline__ KArgs kargs() {
    KArgs k = (KArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return k;
}
template <bool V> struct Flag { static constexpr bool value = V; };
