#include "sscan.h"

// PRE = false: outputs (and, for training, the state in front of every tile).  PRE = true: only the state a chunk ends in
// when it starts from zero, and its sum of delta; chunk k of the main pass starts from what these give.
//
// One barrier a tile: while a tile's states are walked, the next tile's delta, delta x, B and C go into the other half of the
// LDS buffers and the tile after that is on its way from memory into registers.
//
// Bound by the vector unit: 6 issue slots per (frame, channel, state) (the exponential takes two) and 59 per (frame, channel) for
// softplus, gate, joins and addresses, 155 in all with 16 states.  Measured at T 2048, B 16, D 2048, 16 states, bf16: 326 us, 1.24
// times the 264 us of those slots at 2.4 GHz on every lane; counters say 79 % of all SIMD cycles issue a vector instruction (at the
// clock the card holds).  One row of T 16384 (24 chunks): 153 us, and 127 for the pass over chunks (slots 135 and 98).
template <typename TY, int SPL, int NB, bool PRE>
__global__ __launch_bounds__(256) void sstate_fwd_kernel(SscanArgs p) {
    constexpr int NP = 4 * SPL * NB, TS = SSCAN_TS, RB = (TS * NP + 255) / 256;
    __shared__ float2 s_du[2][TS][64];
    __shared__ __attribute__((aligned(16))) float s_B[2][TS * NP];
    __shared__ __attribute__((aligned(16))) float s_C[2][PRE ? 1 : TS * NP];
    __shared__ float s_y[2][PRE ? 1 : 4][PRE ? 1 : TS][64];
    const Place q = sscan_place(p);
    const int tid = threadIdx.x, lane = q.lane, w = q.w;
    if (PRE && q.t0 >= q.t1) return;
    const TY* px = (const TY*)p.x + q.b * p.x_sb;
    const TY* pdt = (const TY*)p.dt + q.b * p.dt_sb;
    // without a gate the input stands in for z and the gate's factor is replaced by 1: no branch in the loop
    const bool gated = p.z != nullptr, soft = p.softplus;
    const TY* pz = gated ? (const TY*)p.z + q.b * p.z_sb : px;
    const long long z_st = gated ? p.z_st : p.x_st;
    const TY* pB = (const TY*)p.Bm + q.b * p.b_sb + q.g * p.b_sg;
    const TY* pC = (const TY*)p.Cm + q.b * p.c_sb + q.g * p.c_sg;
    TY* po = (TY*)p.out + q.b * p.o_sb;
    const unsigned d = q.d;
    const float bias = p.bias ? p.bias[d] : 0.f;
    const float Dk = p.Dk ? p.Dk[d] : 0.f;
    float A2[NB][SPL], h[NB][SPL];
#pragma unroll
    for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            const int n = (m * 4 + w) * SPL + j;
            A2[m][j] = n < p.N ? rate2(p.A[(size_t)d * p.N + n]) : 0.f;
            h[m][j] = (!PRE && p.h0 && n < p.N) ? p.h0[((size_t)q.b * p.D + d) * p.N + n] : 0.f;
        }
    if (!PRE) {                       // the state this chunk starts from
        for (int j = 0; j < q.k && j * p.tpc < q.nt; ++j) {
            const float ds = p.c_ds[((size_t)j * p.B + q.b) * p.D + d];
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int i = 0; i < SPL; ++i) {
                    const int n = (m * 4 + w) * SPL + i;
                    const float hl = p.c_h[(((size_t)j * p.B + q.b) * NP + n) * p.D + d];
                    h[m][i] = carried(h[m][i], A2[m][i] * ds) + hl;
                }
        }
    }
    float dsum = 0.f;
    // on their way from memory: own frames w*4 .. w*4+3 of a tile, own part of B and C
    TY lx[4], ldt[4], lz[4], lB[RB], lC[RB];
    float rx[4], rz[4], nx[4], nz[4];               // x, z of the tile being walked and of the next
    const unsigned off = d * (unsigned)sizeof(TY);
    const auto fetch = [&](int tile, auto full) {
        constexpr bool FULL = decltype(full)::value;
        const int s0 = tile * TS + w * 4;
        fetch_rows<FULL>(lx, px, p.x_st, s0, q.len, p.reverse, off);
        fetch_rows<FULL>(ldt, pdt, p.dt_st, s0, q.len, p.reverse, off);
        if (!PRE) fetch_rows<FULL>(lz, pz, z_st, s0, q.len, p.reverse, off);
        fetch_states<TY, NP, RB>(lB, pB, p.b_st, tile, q.len, p.reverse, p.N);
        if (!PRE) fetch_states<TY, NP, RB>(lC, pC, p.c_st, tile, q.len, p.reverse, p.N);
    };
    const auto place = [&](int tile, int half, auto full) {
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ok = FULL || tile * TS + w * 4 + i < q.len;
            const float v = (float)ldt[i] + bias;
            const float sp = softplus_(v), raw = soft ? sp : v;
            const float de = ok ? raw : 0.f;
            nx[i] = ok ? (float)lx[i] : 0.f;
            if (!PRE) nz[i] = (float)lz[i];
            s_du[half][w * 4 + i][lane] = float2{de, de * nx[i]};
        }
        place_states<TY, NP, RB>(s_B[half], lB, tile, q.len, p.N);
        if (!PRE) place_states<TY, NP, RB>(s_C[half], lC, tile, q.len, p.N);
    };
    float* ck = (!PRE && p.ckpt) ? p.ckpt + (((size_t)q.t0 * p.B + q.b) * NP + w * SPL) * p.D : nullptr;
    const size_t ck_tile = (size_t)p.B * NP * p.D;
    // what a tile leaves behind: y joined, gated, stored
    const auto leave = [&](int tile, int half, auto full) {
        constexpr bool FULL = decltype(full)::value;
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = w * 4 + i;
            y[i] = ((s_y[half][0][t][lane] + s_y[half][1][t][lane]) + (s_y[half][2][t][lane] + s_y[half][3][t][lane])) + Dk * rx[i];
            y[i] *= gated ? silu_(rz[i]) : 1.0f;
        }
        if (FULL || q.on) store_rows<FULL>(po, p.o_st, tile * TS + w * 4, q.len, p.T, p.reverse, off, y);
    };
    // a tile, and behind it the tile in front (`prev`), so that its joins and stores run beside the walk.  FULL: it, the next
    // and the one after that, and the one in front, hold valid frames alone (a lane without a channel of its own does what the last
    // one with a channel does, its stores included)
    const auto walk = [&](int tile, auto full, auto prev) {
        constexpr bool FULL = decltype(full)::value;
        const int half = (tile - q.t0) & 1;
        if (!PRE && ck) {
            if (FULL || q.on)
#pragma unroll
                for (int m = 0; m < NB; ++m)
#pragma unroll
                    for (int j = 0; j < SPL; ++j)
                        *(float*)((char*)(ck + (size_t)(m * 4 * SPL + j) * p.D) + d * 4u) = h[m][j];
            ck += ck_tile;
        }
        if (!PRE && decltype(prev)::value) leave(tile - 1, half ^ 1, full);
#pragma unroll
        for (int i = 0; i < 4; ++i) { rx[i] = nx[i]; rz[i] = nz[i]; }
#pragma unroll(NB == 1 ? TS : 4)
        for (int t = 0; t < TS; ++t) {
            const float2 du = s_du[half][t][lane];
            float y = 0.f;
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int j = 0; j < SPL; ++j) {
                    const int e = t * NP + (m * 4 + w) * SPL + j;
                    h[m][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(A2[m][j] * du.x), h[m][j], du.y * s_B[half][e]);
                    if (!PRE) y = __builtin_fmaf(s_C[half][e], h[m][j], y);
                }
            if (!PRE) s_y[half][w][t][lane] = y;
            else if (w == 0) dsum += du.x;
        }
        if (FULL || tile + 1 < q.t1) {
            place(tile + 1, half ^ 1, full);
            fetch(FULL ? tile + 2 : min(tile + 2, q.t1 - 1), full);
        }
        __syncthreads();
    };
    if (q.t0 < q.t1) {
        fetch(q.t0, Flag<false>{});
        place(q.t0, 0, Flag<false>{});
        fetch(min(q.t0 + 1, q.t1 - 1), Flag<false>{});
        __syncthreads();
    }
    // (a chunk's last tiles call for the next chunk's first two: valid frames, thrown away)
    const int clear = min(q.t1, q.len / TS - 2);
    int tile = q.t0;
    if (tile < clear) walk(tile++, Flag<true>{}, Flag<false>{});
    else if (tile < q.t1) walk(tile++, Flag<false>{}, Flag<false>{});
    for (; tile < clear; ++tile) walk(tile, Flag<true>{}, Flag<true>{});
    for (; tile < q.t1; ++tile) walk(tile, Flag<false>{}, Flag<true>{});
    if (!PRE && q.t0 < q.t1) leave(q.t1 - 1, (q.t1 - 1 - q.t0) & 1, Flag<false>{});
    if (!q.on) return;
    if (PRE) {
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
            for (int j = 0; j < SPL; ++j)
                p.c_h[(((size_t)q.k * p.B + q.b) * NP + (m * 4 + w) * SPL + j) * p.D + d] = h[m][j];
        if (w == 0) p.c_ds[((size_t)q.k * p.B + q.b) * p.D + d] = dsum;
        return;
    }
    // the last valid tile's chunk (chunk 0 of an empty row) leaves the state
    const bool last = q.nt == 0 ? q.k == 0 : (q.t0 < q.nt && q.t0 + p.tpc >= q.nt);
    if (p.h_last && last) {
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
            for (int j = 0; j < SPL; ++j) {
                const int n = (m * 4 + w) * SPL + j;
                if (n < p.N) p.h_last[((size_t)q.b * p.D + d) * p.N + n] = h[m][j];
            }
    }
    const int send = min(p.T, (q.t0 + p.tpc) * TS);
    for (int s = max(q.nt, q.t0) * TS + w; s < send; s += 4) (po + (long long)s * p.o_st)[d] = (TY)0.f;   // padding
}

// One frame: thread = 4 states of a channel (one 16-byte access when N is a multiple of 4), LPC lanes per channel join y.
template <typename TY, int LPC>
__global__ __launch_bounds__(256) void sscan_step_kernel(SscanArgs p) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t ch = i / LPC;
    const int l = (int)(i % LPC), n0 = l * 4;
    if (ch >= (size_t)p.B * p.D) return;             // whole groups of LPC lanes leave together
    const int b = (int)(ch / p.D), d = (int)(ch % p.D), g = d / p.dpg;
    float de = ldf((const TY*)p.dt + b * p.dt_sb + d) + (p.bias ? p.bias[d] : 0.f);
    if (p.softplus) de = softplus_(de);
    const float x = ldf((const TY*)p.x + b * p.x_sb + d), u = de * x;
    const TY* pB = (const TY*)p.Bm + b * p.b_sb + g * p.b_sg;
    const TY* pC = (const TY*)p.Cm + b * p.c_sb + g * p.c_sg;
    float* h = p.h_last + ch * p.N;
    const float* A = p.A + (size_t)d * p.N;
    float y = 0.f;
    const int m = min(4, p.N - n0);
    if (p.vec && n0 < p.N) {
        f32x4 hv = *(f32x4*)(h + n0);
        const f32x4 av = *(const f32x4*)(A + n0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            hv[e] = __builtin_fmaf(__builtin_amdgcn_exp2f(rate2(av[e]) * de), hv[e], u * ldf(pB + n0 + e));
            y = __builtin_fmaf(ldf(pC + n0 + e), hv[e], y);
        }
        *(f32x4*)(h + n0) = hv;
    } else {
        for (int e = 0; e < m; ++e) {
            const float v = __builtin_fmaf(__builtin_amdgcn_exp2f(rate2(A[n0 + e]) * de), h[n0 + e], u * ldf(pB + n0 + e));
            h[n0 + e] = v;
            y = __builtin_fmaf(ldf(pC + n0 + e), v, y);
        }
    }
#pragma unroll
    for (int o = LPC / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
    if (l == 0) {
        if (p.Dk) y += p.Dk[d] * x;
        if (p.z) y *= silu_(ldf((const TY*)p.z + b * p.z_sb + d));
        stf((TY*)p.out + b * p.o_sb + d, y);
    }
}

// ---------------------------------------------------------------- C entries
// Chunks of time, where batch rows x channel tiles (`wgs` workgroups) leave the chip idle: a first pass over the chunks costs two
// thirds of a forward pass and 28 % of a backward one.  Measured at 1024 frames, bf16, 16 states, us:
//   workgroups        128   192   256   320   384   448   480   512   544   640   704
//   forward, one      129   130   130   164   166   167   167   167   216   218   220
//     768 / wgs        79   111   129   186   188    as one
//   backward, one     321   325   326   436   438   441   442   444   687   691   693
//     chunks          169   239   305   387   435   530   541   547   618   684   753    (2048 / wgs, from 512 on 4)
// So forward up to 256 as many as make the three workgroups of a CU.  At 256 itself that pays for f32 and for long rows alone
// (one chunk / three, us, training: T 512 f32 68.4 / 70.5, bf16 68.6 / 70.8; T 1024 142.7 / 132.3, 129.8 / 128.7; T 1207 ragged
// 165.4 / 150.2, 151.4 / 149.1; T 2262 ragged 309 / 271, 278 / 270).  Backward up to 400 four rounds of the two that a CU holds, which
// also evens out ragged rows (256 workgroups, T 1207, f32, 4 / 6 / 8 / 10 / 12 chunks: 315 / 308 / 294 / 310 / 309 us), and four chunks
// where a second round of workgroups would be nearly empty.  A single row (32 workgroups, T 16384): 8 / 16 / 24 / 32 / 64 chunks
// 453 / 310 / 277 / 287 / 286 us.  At least four tiles each.
// The rule knows the number of workgroups alone, and misses where the rest matters: ragged rows backward (480 workgroups, one chunk
// 417 us, six 386; 544 workgroups, a step 2 % slower with four than with one), short rows at 256 workgroups (above).
int sscan_chunks(int T, int B, int D, int G, int backward) {
    const long long wgs = (long long)G * ((D / G + 63) / 64) * B;
    const int nt = sscan_tiles(T);
    long long S = 1;
    if (wgs > 0 && wgs < (backward ? 401 : 257)) S = (backward ? 2048 : 768) / wgs;
    else if (backward && wgs > 512 && wgs <= 640) S = 4;
    if (S > nt / 4) S = nt / 4;
    if (S > 64) S = 64;
    return S < 1 ? 1 : (int)S;
}

int sscan_fill(const asr_sscan_desc* d, SscanArgs* p, int backward) {
    if (!d || d->dtype < ASR_F32 || d->dtype > ASR_F16) return ASR_ERR_ARG;
    if (d->T < 0 || d->B < 0 || d->D <= 0 || d->N <= 0 || d->G <= 0 || d->D % d->G) return ASR_ERR_ARG;
    if (d->N > 64 || d->B > 65535 || d->D > (1 << 20) || d->T > (1 << 24)) return ASR_ERR_LIMIT;
    if (!d->A) return ASR_ERR_ARG;
    const bool any = d->T > 0 && d->B > 0;
    if (any && (!d->x || !d->dt || !d->Bm || !d->Cm)) return ASR_ERR_ARG;
    p->T = d->T; p->B = d->B; p->D = d->D; p->N = d->N; p->G = d->G;
    p->dpg = d->D / d->G; p->tpg = (p->dpg + 63) / 64;
    p->reverse = d->reverse; p->softplus = d->softplus;
    p->S = sscan_chunks(d->T, d->B, d->D, d->G, backward);
    p->tpc = (sscan_tiles(d->T) + p->S - 1) / p->S;
    if (p->tpc < 1) p->tpc = 1;
    p->np = sscan_np(d->N);
    p->lens = d->lens;
    p->x = d->x; p->x_st = d->x_st; p->x_sb = d->x_sb;
    p->dt = d->dt; p->dt_st = d->dt_st; p->dt_sb = d->dt_sb;
    p->z = d->z; p->z_st = d->z_st; p->z_sb = d->z_sb;
    p->Bm = d->Bm; p->b_st = d->b_st; p->b_sb = d->b_sb; p->b_sg = d->b_sg;
    p->Cm = d->Cm; p->c_st = d->c_st; p->c_sb = d->c_sb; p->c_sg = d->c_sg;
    p->A = d->A; p->Dk = d->Dk; p->bias = d->dt_bias; p->h0 = d->h0;
    p->out = d->out; p->o_st = d->o_st; p->o_sb = d->o_sb;
    p->h_last = d->h_last; p->ckpt = d->ckpt;
    p->dout = d->dout; p->do_st = d->do_st; p->do_sb = d->do_sb; p->dh_last = d->dh_last;
    p->dx = d->dx; p->ddt = d->ddt; p->dz = d->dz; p->dh0 = d->dh0;
    return ASR_OK;
}

extern "C" size_t asr_sscan_ckpt_floats(int T, int B, int D, int N) {
    if (T <= 0 || B <= 0 || D <= 0 || N <= 0 || N > 64) return 0;
    return (size_t)sscan_tiles(T) * B * sscan_np(N) * D;
}

static size_t fwd_ws(int T, int B, int D, int N, int G) {
    const int S = sscan_chunks(T, B, D, G, 0);
    return S > 1 ? align256((size_t)S * B * sscan_np(N) * D * 4) + (size_t)S * B * D * 4 : 0;
}

size_t sscan_bwd_ws(int T, int B, int D, int N, int G);
extern "C" size_t asr_sscan_ws_bytes(int T, int B, int D, int N, int G, int backward) {
    if (T < 0 || B < 0 || D <= 0 || N <= 0 || N > 64 || G <= 0 || D % G) return 0;
    return backward ? sscan_bwd_ws(T, B, D, N, G) : fwd_ws(T, B, D, N, G);
}

template <typename TY, int SPL, int NB>
static void launch_fwd(const SscanArgs& p, hipStream_t stream) {
    if (p.S > 1)
        hipLaunchKernelGGL((sstate_fwd_kernel<TY, SPL, NB, true>), dim3(p.G * p.tpg, p.B, p.S - 1), dim3(256), 0, stream, p);
    hipLaunchKernelGGL((sstate_fwd_kernel<TY, SPL, NB, false>), dim3(p.G * p.tpg, p.B, p.S), dim3(256), 0, stream, p);
}
template <typename TY>
static void launch_fwd_t(const SscanArgs& p, hipStream_t stream) {
    if (p.N <= 4) launch_fwd<TY, 1, 1>(p, stream);
    else if (p.N <= 8) launch_fwd<TY, 2, 1>(p, stream);
    else if (p.N <= 16) launch_fwd<TY, 4, 1>(p, stream);
    else if (p.N <= 32) launch_fwd<TY, 4, 2>(p, stream);
    else launch_fwd<TY, 4, 4>(p, stream);
}

extern "C" int asr_sscan_fwd(const asr_sscan_desc* d, void* ws, size_t ws_bytes, hipStream_t stream) {
    SscanArgs p{};
    if (int e = sscan_fill(d, &p, 0)) return e;
    if (d->h_last && d->h_last == d->h0) return ASR_ERR_ARG;
    if (d->T > 0 && d->B > 0 && !d->out) return ASR_ERR_ARG;
    if (d->B == 0 || (d->T == 0 && !d->h_last)) return ASR_OK;
    if (p.S > 1) {
        if (!ws || ws_bytes < fwd_ws(d->T, d->B, d->D, d->N, d->G)) return ASR_ERR_WS;
        if ((uintptr_t)ws & 15) return ASR_ERR_ARG;
        p.c_h = (float*)ws;
        p.c_ds = (float*)((char*)ws + align256((size_t)p.S * p.B * p.np * p.D * 4));
    }
    if (d->dtype == ASR_F32) launch_fwd_t<float>(p, stream);
    else if (d->dtype == ASR_BF16) launch_fwd_t<bf16_t>(p, stream);
    else launch_fwd_t<f16_t>(p, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}

template <typename TY>
static void launch_step(const SscanArgs& p, hipStream_t stream) {
    const int need = (p.N + 3) / 4;
    const int lpc = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : 16;
    const dim3 grid((unsigned)(((size_t)p.B * p.D * lpc + 255) / 256));
#define STEP_(L) hipLaunchKernelGGL((sscan_step_kernel<TY, L>), grid, dim3(256), 0, stream, p)
    switch (lpc) { case 1: STEP_(1); break; case 2: STEP_(2); break; case 4: STEP_(4); break; case 8: STEP_(8); break;
                   default: STEP_(16); }
#undef STEP_
}

extern "C" int asr_sscan_step(int dtype, int B, int D, int N, int G, float* h, const void* x, long long x_sb, const void* dt,
                              long long dt_sb, const float* A, const void* Bm, long long b_sb, long long b_sg,
                              const void* Cm, long long c_sb, long long c_sg, const float* Dk, const void* z,
                              long long z_sb, const float* dt_bias, int softplus, void* out, long long o_sb,
                              hipStream_t stream) {
    if (dtype < ASR_F32 || dtype > ASR_F16 || B < 0 || D <= 0 || N <= 0 || G <= 0 || D % G || !A) return ASR_ERR_ARG;
    // 2^32 work items a launch: up to 16 of them a channel
    if (N > 64 || B > 65535 || D > (1 << 20) || (long long)B * D > (1ll << 27)) return ASR_ERR_LIMIT;
    if (!B) return ASR_OK;
    if (!h || !x || !dt || !Bm || !Cm || !out) return ASR_ERR_ARG;
    SscanArgs p{};
    p.vec = (N & 3) == 0 && !(((uintptr_t)h | (uintptr_t)A) & 15);
    p.B = B; p.D = D; p.N = N; p.G = G; p.dpg = D / G; p.softplus = softplus;
    p.x = x; p.x_sb = x_sb; p.dt = dt; p.dt_sb = dt_sb; p.A = A; p.Bm = Bm; p.b_sb = b_sb; p.b_sg = b_sg;
    p.Cm = Cm; p.c_sb = c_sb; p.c_sg = c_sg; p.Dk = Dk; p.z = z; p.z_sb = z_sb; p.bias = dt_bias; p.h_last = h;
    p.out = out; p.o_sb = o_sb;
    if (dtype == ASR_F32) launch_step<float>(p, stream);
    else if (dtype == ASR_BF16) launch_step<bf16_t>(p, stream);
    else launch_step<f16_t>(p, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}
