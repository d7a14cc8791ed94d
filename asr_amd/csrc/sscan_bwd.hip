// Backward pass of the selective scan.  With q = dh a h[s-1]:
//   dh[s] = C dy + a[s+1] dh[s+1],   dC = sum_d dy h,   dB = sum_d dh delta x,
//   dA = sum_s delta q,   d delta = sum_n A q + x sum_n dh B,   dx = delta sum_n dh B + D dy,   dz = dout y silu'(z)
// Tiles are walked from the last to the first.  A tile's states are formed again from the state saved in front of it and kept
// in registers (16 frames x states, with a), then the adjoint runs back over them.
//
// Bound by the vector unit: 14 issue slots per (frame, channel, state) and 4.4 for the sums over lanes, 116 per (frame, channel),
// 410 in all with 16 states.  Measured at T 2048, B 16, D 2048, 16 states, bf16: 866 us, 1.24 times the 700 us of those slots, and 31
// for the sums over workgroups; the bytes of both passes together are 230 us; counters: 80 % of all SIMD cycles issue a vector
// instruction.
#include "sscan.h"

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float half_join(float a, float b) {      // lanes 0-31: a[l] + a[l+32], lanes 32-63: the same of b
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float row_join(float a, float b) {       // even 16-lane rows: a's pair of rows, odd: b's
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
// Sums over the 64 lanes of sixteen values at once: lane l returns the sum of v[l >> 2].  Each of the first four steps joins
// two values in one register and halves the lanes that still have to be added: 35 instructions for 16 sums (96 one by one).
__device__ __forceinline__ float sum16(const float (&v)[16], int lane) {
    float w[8], x[4], y[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = half_join(v[i], v[i + 8]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = row_join(w[i], w[i + 4]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float keep = (lane & 8) ? x[i + 2] : x[i], give = (lane & 8) ? x[i] : x[i + 2];
        y[i] = keep + dpp<0x128>(give);                              // row_ror:8
    }
    const float keep = (lane & 4) ? y[1] : y[0], give = (lane & 4) ? y[0] : y[1];
    float z = keep + dpp<0x141>(give);                               // row_half_mirror
    z += dpp<0xB1>(z);                                               // quad_perm [1,0,3,2]
    return z + dpp<0x4E>(z);                                         // quad_perm [2,3,0,1]
}

// EDGE: a group's channels are no multiple of 64, so that its last workgroup has idle lanes.  (With the tests for them in every kernel
// the other sizes lose 5 %; three loops in one kernel cost them 18 %, by registers.)
// PRE: the adjoint a chunk hands to the one in front of it when nothing comes in from behind, and its sum of delta.
// Behind a tile's first adjoints, when the first of its states have left their registers, the tile in front of it is called from
// memory; it goes into the input buffers behind the tile's first barrier, beside the joins.  (Called a tile
// earlier, as the forward pass does, it costs 30 registers where they are scarcest: one wave per SIMD less, or spills; called
// half way through the adjoints the spills are 28 registers, and T 2048, B 16, D 2048, bf16 took 937 us instead of 886; one input
// buffer instead of two, 850.)
template <typename TY, int SPL, int NB, bool PRE, bool EDGE>
__global__ __launch_bounds__(256, 2) void sstate_bwd_kernel(SscanArgs p) {
    constexpr int NP = 4 * SPL * NB, TS = SSCAN_TS, RS = 8 / SPL;    // RS frames give sixteen sums
    constexpr int RB = (TS * NP + 255) / 256;
    // the main pass places a tile's inputs when all waves are through with the last one's: one buffer; PRE before that: two
    constexpr int HALVES = PRE ? 2 : 1;
    __shared__ float2 s_du[HALVES][TS][64];
    __shared__ float s_dy[HALVES][TS][64];
    __shared__ __attribute__((aligned(16))) float s_B[HALVES][PRE ? 1 : TS * NP], s_C[HALVES][TS * NP];
    __shared__ float2 s_s[PRE ? 1 : 4][PRE ? 1 : TS][64];
    __shared__ float s_y[PRE ? 1 : 4][PRE ? 1 : TS][64];
    __shared__ float s_bc[PRE ? 1 : TS * 2 * NP];
    const Place q = sscan_place(p);
    const bool on = !EDGE || q.on;
    const int tid = threadIdx.x, lane = q.lane, w = q.w;
    if (PRE && (q.k == 0 || q.t0 >= q.t1)) return;
    // without a gate x stands in for z and the gate's factors are replaced: no branch in the loop
    const bool gated = p.z != nullptr, soft = p.softplus;
    const unsigned d = q.d, off = d * (unsigned)sizeof(TY);
    const float bias = p.bias ? p.bias[d] : 0.f;
    const float Dk = p.Dk ? p.Dk[d] : 0.f;
    float A2[NB][SPL], r[NB][SPL], dA[NB][SPL];
#pragma unroll
    for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            const int n = (m * 4 + w) * SPL + j;
            A2[m][j] = n < p.N ? rate2(p.A[(size_t)d * p.N + n]) : 0.f;
            r[m][j] = (!PRE && p.dh_last && n < p.N) ? p.dh_last[((size_t)q.b * p.D + d) * p.N + n] : 0.f;
            dA[m][j] = 0.f;
        }
    const int nch = (q.nt + p.tpc - 1) / p.tpc;                       // chunks that hold a valid frame
    if (!PRE) {                                                       // the adjoint that comes in from behind
        for (int j = nch - 1; j > q.k; --j) {
            const float ds = p.c_ds[((size_t)j * p.B + q.b) * p.D + d];
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int i = 0; i < SPL; ++i) {
                    const int n = (m * 4 + w) * SPL + i;
                    const float rl = p.c_h[(((size_t)j * p.B + q.b) * NP + n) * p.D + d];
                    r[m][i] = carried(r[m][i], A2[m][i] * ds) + rl;
                }
        }
    }
    // idle lanes stand on a real channel: whatever it holds, they must give zeros to the sums dB and dC
    if (!on) {
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
            for (int j = 0; j < SPL; ++j) r[m][j] = 0.f;
    }
    float accD = 0.f, accb = 0.f, dsum = 0.f;
    TY lx[4], ldt[4], lz[4], lg[4], lB[RB], lC[RB];       // on their way from memory
    float rx[4], rs[4], rg[4], nx[4], ns[4], ng[4];       // x, d delta / d dt, dout silu'(z): of the tile walked and the next
    const auto fetch = [&](int tile, auto full) {
        constexpr bool FULL = decltype(full)::value;
        const KArgs k = kargs();
        const int s0 = tile * TS + w * 4, rev = k->reverse;
        if (!PRE) fetch_rows<FULL>(lx, (const TY*)k->x + q.b * k->x_sb, k->x_st, s0, q.len, rev, off);
        fetch_rows<FULL>(ldt, (const TY*)k->dt + q.b * k->dt_sb, k->dt_st, s0, q.len, rev, off);
        fetch_rows<FULL>(lg, (const TY*)k->dout + q.b * k->do_sb, k->do_st, s0, q.len, rev, off);
        const TY* z = (const TY*)(gated ? k->z : k->x);
        fetch_rows<FULL>(lz, z + q.b * (gated ? k->z_sb : k->x_sb), gated ? k->z_st : k->x_st, s0, q.len, rev, off);
        if (!PRE) fetch_states<TY, NP, RB>(lB, (const TY*)k->Bm + q.b * k->b_sb + q.g * k->b_sg, k->b_st, tile, q.len, rev, k->N);
        fetch_states<TY, NP, RB>(lC, (const TY*)k->Cm + q.b * k->c_sb + q.g * k->c_sg, k->c_st, tile, q.len, rev, k->N);
    };
    const auto place = [&](int tile, int half, auto full) {
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ok = FULL || tile * TS + w * 4 + i < q.len;
            const bool live = ok && on;                 // an idle lane's dy and delta x are zero: nothing of it in dB and dC
            const float v = (float)ldt[i] + bias, g = ok ? (float)lg[i] : 0.f;
            const float u = exp_neg_abs_(v), sp = softplus_from_(v, u), sv = sigmoid_from_(v, u);
            const float de = ok ? (soft ? sp : v) : 0.f;
            ns[i] = ok ? (soft ? sv : 1.f) : 0.f;
            const float z = ok ? (float)lz[i] : 0.f, sg = sigm_(z);
            const float dy = gated ? g * z * sg : g;
            ng[i] = g * dsilu_(z, sg);
            nx[i] = (PRE || !ok) ? 0.f : (float)lx[i];
            s_du[half][w * 4 + i][lane] = float2{de, live ? de * nx[i] : 0.f};
            s_dy[half][w * 4 + i][lane] = live ? dy : 0.f;
        }
        const int N = kargs()->N;
        if (!PRE) place_states<TY, NP, RB>(s_B[half], lB, tile, q.len, N);
        place_states<TY, NP, RB>(s_C[half], lC, tile, q.len, N);
    };
    // the state in front of a tile, first group of states: fetched a tile ahead
    float hn[SPL];
    const auto state = [&](int tile, int m, float (&o)[SPL]) {
        const KArgs k = kargs();
        const char* ck = (const char*)(k->ckpt + (((size_t)tile * k->B + q.b) * NP + (m * 4 + w) * SPL) * k->D);
        unsigned at = d * 4u;
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            o[j] = on ? *(const float*)(ck + at) : 0.f;
            ck += (size_t)k->D * 4;
        }
    };
    // a tile; FULL: it and the one in front of it hold valid frames alone
    const auto walk = [&](int tile, auto full) {
        constexpr bool FULL = decltype(full)::value;
        const int half = PRE ? (q.t1 - 1 - tile) & 1 : 0, sb = tile * TS;
#pragma unroll
        for (int i = 0; i < 4; ++i) { rx[i] = nx[i]; rs[i] = ns[i]; rg[i] = ng[i]; }
        if (PRE) {
            if (FULL || tile > q.t0) fetch(tile - 1, full);
#pragma unroll(NB == 1 ? TS : 4)
            for (int t = TS - 1; t >= 0; --t) {
                const float de = s_du[half][t][lane].x, dy = s_dy[half][t][lane];
#pragma unroll
                for (int m = 0; m < NB; ++m)
#pragma unroll
                    for (int j = 0; j < SPL; ++j)
                        r[m][j] = __builtin_amdgcn_exp2f(A2[m][j] * de) *
                                  __builtin_fmaf(s_C[half][t * NP + (m * 4 + w) * SPL + j], dy, r[m][j]);
                if (w == 0) dsum += de;
            }
        } else {
            // one group of states at a time: of two, the registers hold neither (r, A2 and dA of several groups lie in scratch)
#pragma unroll 1
            for (int m = 0; m < NB; ++m) {
                float a[TS][SPL], h[TS][SPL], h0[SPL], da[SPL];    // da: a tile's part of dA: no sum runs over all frames
                if (m == 0) {
#pragma unroll
                    for (int j = 0; j < SPL; ++j) h0[j] = hn[j];
                } else {
                    state(tile, m, h0);
                }
#pragma unroll
                for (int j = 0; j < SPL; ++j) da[j] = 0.f;
#pragma unroll
                for (int t = 0; t < TS; ++t) {
                    const float2 du = s_du[half][t][lane];
                    float y = 0.f;
#pragma unroll
                    for (int j = 0; j < SPL; ++j) {
                        const int e = t * NP + (m * 4 + w) * SPL + j;
                        a[t][j] = __builtin_amdgcn_exp2f(A2[m][j] * du.x);
                        h[t][j] = __builtin_fmaf(a[t][j], t ? h[t - 1][j] : h0[j], du.y * s_B[half][e]);
                        y = __builtin_fmaf(s_C[half][e], h[t][j], y);
                    }
                    if (m) s_y[w][t][lane] += y; else s_y[w][t][lane] = y;
                }
#pragma unroll
                for (int tb = TS / RS - 1; tb >= 0; --tb) {
                    float v[16];
#pragma unroll
                    for (int i = RS - 1; i >= 0; --i) {
                        const int t = tb * RS + i;
                        const float2 du = s_du[half][t][lane];
                        const float dy = s_dy[half][t][lane];
                        float s1 = 0.f, s2 = 0.f;
#pragma unroll
                        for (int j = 0; j < SPL; ++j) {
                            const int e = t * NP + (m * 4 + w) * SPL + j;
                            const float dh = __builtin_fmaf(s_C[half][e], dy, r[m][j]);
                            v[i * 2 * SPL + j] = dh * du.y;
                            v[i * 2 * SPL + SPL + j] = dy * h[t][j];
                            r[m][j] = a[t][j] * dh;
                            // padding: a is 1 and the last state and its gradient meet as they do in no valid frame
                            const float qq = (FULL || sb + t < q.len) ? r[m][j] * (t ? h[t - 1][j] : h0[j]) : 0.f;
                            s2 = __builtin_fmaf(qq, A2[m][j], s2);
                            da[j] = __builtin_fmaf(qq, du.x, da[j]);
                            s1 = __builtin_fmaf(dh, s_B[half][e], s1);
                        }
                        if (m) { s_s[w][t][lane].x += s1; s_s[w][t][lane].y += s2; }
                        else s_s[w][t][lane] = float2{s1, s2};
                    }
                    if (m == NB - 1 && tb == TS / RS - 2 && (FULL || tile > q.t0)) {
                        __builtin_amdgcn_sched_barrier(0);
                        fetch(tile - 1, full);
                        state(tile - 1, 0, hn);
                    }
                    const float z = sum16(v, lane);
                    if ((lane & 3) == 0) {
                        const int id = lane >> 2, t = tb * RS + id / (2 * SPL), c = (id / SPL) & 1, j = id % SPL;
                        s_bc[(t * 2 + c) * NP + (m * 4 + w) * SPL + j] = z;
                    }
                }
#pragma unroll
                for (int j = 0; j < SPL; ++j) dA[m][j] += da[j];
            }
        }
        if (PRE) {
            if (FULL || tile > q.t0) place(tile - 1, half ^ 1, full);
            __syncthreads();
            return;
        }
        __syncthreads();
        // the next inputs go in beside the joins below: a thread has read its own frames' delta and dy before it replaces them
        float de[4], dy[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { de[i] = s_du[half][w * 4 + i][lane].x; dy[i] = s_dy[half][w * 4 + i][lane]; }
        if (FULL || tile > q.t0) place(tile - 1, 0, full);
        const int s0 = sb + w * 4;
        float ox[4], odt[4], oz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = w * 4 + i;
            const float2 a = s_s[0][t][lane], b = s_s[1][t][lane], c = s_s[2][t][lane], e = s_s[3][t][lane];
            const float s1 = (a.x + b.x) + (c.x + e.x), s2 = (a.y + b.y) + (c.y + e.y);
            ox[i] = __builtin_fmaf(de[i], s1, Dk * dy[i]);
            odt[i] = (FULL || s0 + i < q.len) ? __builtin_fmaf(rx[i], s1, s2 * LN2) * rs[i] : 0.f;
            oz[i] = rg[i] * (((s_y[0][t][lane] + s_y[1][t][lane]) + (s_y[2][t][lane] + s_y[3][t][lane])) + Dk * rx[i]);
            accD = __builtin_fmaf(dy[i], rx[i], accD);     // frames of the padding give zeros
            accb += odt[i];
        }
        const KArgs k = kargs();
        const int T = k->T, rev = k->reverse;
        const long long ost = (long long)k->B * k->D, orow = (long long)q.b * k->D;
        if (on) {
            store_rows<FULL>((TY*)k->dx + orow, ost, s0, q.len, T, rev, off, ox);
            store_rows<FULL>((TY*)k->ddt + orow, ost, s0, q.len, T, rev, off, odt);
            if (gated) store_rows<FULL>((TY*)k->dz + orow, ost, s0, q.len, T, rev, off, oz);
        }
        char* pbc = (char*)(k->part_bc + (((size_t)(q.g * k->tpg + q.ct) * k->B + q.b) * T + sb) * (2 * NP));
        unsigned first = tid;
#pragma unroll
        for (int i = 0; i < (TS * 2 * NP + 255) / 256; ++i) {
            const unsigned e = first + i * 256;
            if ((TS * 2 * NP % 256 == 0 || e < TS * 2 * NP) && (FULL || sb + (int)(e / (2 * NP)) < q.len))
                *(float*)(pbc + e * 4u) = s_bc[e];
        }
        __syncthreads();
    };
    if (q.t0 < q.t1) {
        fetch(q.t1 - 1, Flag<false>{});
        if (!PRE) state(q.t1 - 1, 0, hn);
        place(q.t1 - 1, 0, Flag<false>{});
        __syncthreads();
    }
    int tile = q.t1 - 1;
    for (; tile >= q.t0 && (tile * TS + TS > q.len); --tile) walk(tile, Flag<false>{});
    // (a chunk's first tile calls for the one in front of it, which is thrown away)
    for (; tile >= max(q.t0, 1); --tile) walk(tile, Flag<true>{});
    for (; tile >= q.t0; --tile) walk(tile, Flag<false>{});
    if (PRE) {
        if (!on) return;
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
            for (int j = 0; j < SPL; ++j)
                p.c_h[(((size_t)q.k * p.B + q.b) * NP + (m * 4 + w) * SPL + j) * p.D + d] = r[m][j];
        if (w == 0) p.c_ds[((size_t)q.k * p.B + q.b) * p.D + d] = dsum;
        return;
    }
    // padding, the parts of the parameter gradients, the gradient of the first state
    const int send = min(p.T, (q.t0 + p.tpc) * TS);
    if (on) {
        for (int s = max(q.nt, q.t0) * TS + w; s < send; s += 4) {
            const size_t o = ((size_t)s * p.B + q.b) * p.D + d;
            stf((TY*)p.dx + o, 0.f);
            stf((TY*)p.ddt + o, 0.f);
            if (gated) stf((TY*)p.dz + o, 0.f);
        }
    }
    const size_t row = (size_t)q.k * p.B + q.b;
    if (on) {
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
            for (int j = 0; j < SPL; ++j) {
                const int n = (m * 4 + w) * SPL + j;
                if (n >= p.N) continue;
                p.part_a[(row * p.D + d) * p.N + n] = dA[m][j];
                if (p.dh0 && q.k == 0) p.dh0[((size_t)q.b * p.D + d) * p.N + n] = r[m][j];
            }
    }
    __syncthreads();
    s_dy[0][w][lane] = accD;
    s_dy[0][4 + w][lane] = accb;
    __syncthreads();
    if (w < 2 && on) {
        const float* v = &s_dy[0][w * 4][lane];
        (w ? p.part_b : p.part_d)[row * p.D + d] = (v[0] + v[64]) + (v[128] + v[192]);
    }
}

// The sums over workgroups, one launch.  Blocks [0, nbc * G): dB / dC, the parts of a group's channel tiles added in order and
// written in the activation type at the frame's place.  Behind them, 64 columns a block: dA, dD and d dt_bias, the parts of
// all rows and chunks (P of them) added by four groups of lanes and joined in order.
template <typename TY>
__global__ __launch_bounds__(256) void sscan_finish_kernel(SscanArgs p, TY* dB, TY* dC, float* dA, float* dD, float* db,
                                                           unsigned nbc, unsigned na, unsigned nd) {
    __shared__ float sm[4][64];
    unsigned blk = blockIdx.x;
    if (blk < nbc * p.G) {
        const int g = blk / nbc;
        const size_t i = (size_t)(blk % nbc) * 256 + threadIdx.x, per = (size_t)p.B * p.T * 2 * p.np;
        if (i >= per) return;
        const int n = (int)(i % p.np), c = (int)(i / p.np) & 1;
        const size_t bs = i / (2 * p.np);
        const int b = (int)(bs / p.T), s = (int)(bs % p.T);
        if (n >= p.N) return;
        const int len = row_len(p.lens, b, p.T);
        float v = 0.f;
        if (s < len) {
            const float* q = p.part_bc + (size_t)g * p.tpg * per + i;
#pragma unroll 8
            for (int k = 0; k < p.tpg; ++k) v += q[(size_t)k * per];
        }
        const long long f = (p.reverse && s < len) ? len - 1 - s : s;
        stf((c ? dC : dB) + ((f * p.B + b) * p.G + g) * p.N + n, v);
        return;
    }
    blk -= nbc * p.G;
    const float* part = p.part_a;
    float* out = dA;
    size_t n = (size_t)p.D * p.N;
    if (blk >= na) {                                  // dD's blocks, if it is wanted, then d dt_bias's
        blk -= na;
        n = p.D;
        const bool second = !dD || blk >= nd;
        if (dD && second) blk -= nd;
        part = second ? p.part_b : p.part_d;
        out = second ? db : dD;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, P = p.S * p.B;
    const size_t i = (size_t)blk * 64 + lane;
    float v = 0.f;
    if (i < n)
#pragma unroll 4
        for (int k = w; k < P; k += 4) v += part[(size_t)k * n + i];
    sm[w][lane] = v;
    __syncthreads();
    if (w == 0 && i < n) out[i] = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
}

// ---------------------------------------------------------------- C entry
struct BwdWs { size_t c_h, c_ds, bc, a, d, b, total; };
static BwdWs bwd_ws(int T, int B, int D, int N, int G) {
    const int S = sscan_chunks(T, B, D, G, 1), np = sscan_np(N), tpg = (D / G + 63) / 64;
    BwdWs o{};
    size_t at = 0;
    const auto take = [&](size_t floats) { const size_t v = at; at += align256(floats * 4); return v; };
    o.c_h = take(S > 1 ? (size_t)S * B * np * D : 0);
    o.c_ds = take(S > 1 ? (size_t)S * B * D : 0);
    o.bc = take((size_t)G * tpg * B * T * 2 * np);
    o.a = take((size_t)S * B * D * N);
    o.d = take((size_t)S * B * D);
    o.b = take((size_t)S * B * D);
    o.total = at;
    return o;
}
size_t sscan_bwd_ws(int T, int B, int D, int N, int G) { return bwd_ws(T, B, D, N, G).total; }

template <typename TY, int SPL, int NB, bool EDGE>
static void launch_bwd_e(const SscanArgs& p, hipStream_t stream) {
    const dim3 grid(p.G * p.tpg, p.B, p.S);
    if (p.S > 1) hipLaunchKernelGGL((sstate_bwd_kernel<TY, SPL, NB, true, EDGE>), grid, dim3(256), 0, stream, p);
    hipLaunchKernelGGL((sstate_bwd_kernel<TY, SPL, NB, false, EDGE>), grid, dim3(256), 0, stream, p);
}
template <typename TY, int SPL, int NB>
static void launch_bwd(const SscanArgs& p, hipStream_t stream) {
    if (p.dpg % 64) launch_bwd_e<TY, SPL, NB, true>(p, stream);
    else launch_bwd_e<TY, SPL, NB, false>(p, stream);
}
template <typename TY>
static void launch_bwd_t(const SscanArgs& p, const asr_sscan_desc* d, hipStream_t stream) {
    if (p.B == 0) {}
    else if (p.N <= 4) launch_bwd<TY, 1, 1>(p, stream);
    else if (p.N <= 8) launch_bwd<TY, 2, 1>(p, stream);
    else if (p.N <= 16) launch_bwd<TY, 4, 1>(p, stream);
    else if (p.N <= 32) launch_bwd<TY, 4, 2>(p, stream);
    else launch_bwd<TY, 4, 4>(p, stream);
    const unsigned nbc = (unsigned)(((size_t)p.B * p.T * 2 * p.np + 255) / 256), nd = (p.D + 63) / 64;
    const unsigned na = (unsigned)(((size_t)p.D * p.N + 63) / 64);
    hipLaunchKernelGGL((sscan_finish_kernel<TY>), dim3(nbc * p.G + na + (d->dD ? nd : 0) + (d->ddt_bias ? nd : 0)),
                       dim3(256), 0, stream, p, (TY*)d->dB, (TY*)d->dC, d->dA, d->dD, d->ddt_bias,
                       nbc, na, nd);
}

extern "C" int asr_sscan_bwd(const asr_sscan_desc* d, void* ws, size_t ws_bytes, hipStream_t stream) {
    SscanArgs p{};
    if (int e = sscan_fill(d, &p, 1)) return e;
    if (!d->dA || (d->z && !d->dz && d->T > 0 && d->B > 0)) return ASR_ERR_ARG;
    if (d->T > 0 && d->B > 0 && (!d->dout || !d->ckpt || !d->dx || !d->ddt || !d->dB || !d->dC)) return ASR_ERR_ARG;
    if (d->dh0 && d->dh0 == d->dh_last) return ASR_ERR_ARG;
    if ((double)d->B * d->T * 2 * p.np * d->G > 4.0e9) return ASR_ERR_LIMIT;        // one work item each, 2^32 a launch
    const BwdWs o = bwd_ws(d->T, d->B, d->D, d->N, d->G);
    if (o.total && (!ws || ws_bytes < o.total)) return ASR_ERR_WS;
    if ((uintptr_t)ws & 15) return ASR_ERR_ARG;
    char* base = (char*)ws;
    p.c_h = (float*)(base + o.c_h); p.c_ds = (float*)(base + o.c_ds); p.part_bc = (float*)(base + o.bc);
    p.part_a = (float*)(base + o.a); p.part_d = (float*)(base + o.d); p.part_b = (float*)(base + o.b);
    if (d->dtype == ASR_F32) launch_bwd_t<float>(p, d, stream);
    else if (d->dtype == ASR_BF16) launch_bwd_t<bf16_t>(p, d, stream);
    else launch_bwd_t<f16_t>(p, d, stream);
    ASR_CHECK_LAUNCH();
    return ASR_OK;
}
