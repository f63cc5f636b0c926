// A residual block's end and the next block's beginning in one pass over the rows:
//     t = post(f)      y = x + scale * gate * t      h = pre(y)
// post / pre: LayerNorm (v - mean) / sqrt(var + eps) * gain + bias, RMS norm v / sqrt(mean v^2 + eps) * gain, or absent (t = f, no h); scale:
// a number or one per column; gate: one row for every M / G consecutive rows (G = M: one for every element), or absent.  For training
// the rows of both norms before gain and bias go onto an 8-bit tape (tape8.cuh) with the factors 1 / sqrt(..): the normalised row is
// what the backward pass needs, and its values are of the order of one whatever f was (a tape of f itself would lose a small variation on a
// large mean).
//
// Backward, from gy = d y and gh = d h, v^ the taped rows, r their factors:
//     u = gh pre_gain      D = gy + r_pre (u - [mean u] - y^ mean(u y^))                     dx = D
//     v = scale gate D     u = v post_gain      df = r_post (u - [mean u] - f^ mean(u f^))   (no post: df = v)
//     d gate = scale t D summed over its rows; d scale = sum gate t D; d post_gain = sum v f^; d post_bias = sum v;
//     d pre_gain = sum gh y^; d pre_bias = sum gh                                            ([mean u]: LayerNorm only)
// All four sums over rows are linear in  S1 = sum gate D f^,  S0 = sum gate D,  P1 = sum gh y^,  P0 = sum gh  - four sums per column.
//
// Both are bound by HBM: every array is read or written once.  Measured at 262 144 x 128 fp32 with a gate for each of four runs of rows:
// with both tapes 116 - 130 us (from run to run; 4.9 TB/s in the middle), backward 111 - 120 + 9 us for the parameters' sums (4.7 TB/s); a large copy reaches 4.9.  A row belongs to a team of 16 to 512 lanes, four neighbouring columns per
// lane and slot, at most two slots: it stays in registers from its load to its last use, and the next row of the team is loaded before this
// one is worked on (the statistics are two dependent sums over the row: without rows in flight behind them the loads' latency is what
// the kernel takes).  Sums over a team are lane exchanges inside the vector unit, through LDS for a team of several waves; fp32, the
// variance around the mean.  Gradients of parameters: a lane adds its columns over the rows that its team walks, teams and workgroups are
// added in their order (the same bits every time).
#include "common.cuh"
#include "split_single.cuh"
#include "tape8.cuh"

struct NjArgs {
    const void *x, *f, *gate;            // rows of x, f (forward) or gy, gh (backward: x = gy, f = gh)
    const float *scale_v, *post_g, *post_b, *pre_g, *pre_b;
    void *y, *h;                         // outputs: y, h (forward) or df, dx (backward: y = dx, h = df)
    unsigned char *post_c, *post_e, *pre_c, *pre_e;     // tape: codes and bytes of the normalised rows
    float *post_r, *pre_r;               // [M] factors
    void* dgate;
    float* part;                         // backward: [workgroups][4][W] sums S1, S0, P1, P0
    long M, ldx, ldf, ldg, ldy, ldh;
    long rows_per_gate;                  // M / G (M without a gate)
    long groups;                         // backward: G, 1 without a gate
    int W, layer, has_post, has_pre, has_gate, tape, per_group, need_sums;
    int plain_sums;                      // backward: S0 and P0 too (somebody has a bias)
    float scale, eps;
};

// sums over a team of TL lanes: neighbours, quads, halves of 16 by lane permutes of the vector unit, then rows of 16 and halves of the wave
template <int CTRL>
__device__ __forceinline__ float nj_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int L>
__device__ __forceinline__ float nj_lanes(float v) {
    v = nj_dpp<0xB1>(v);                                                      // quad_perm 1 0 3 2
    v = nj_dpp<0x4E>(v);                                                      // quad_perm 2 3 0 1
    v = nj_dpp<0x141>(v);                                                     // row_half_mirror: the other four of eight
    v = nj_dpp<0x140>(v);                                                     // row_mirror: the other eight of sixteen
    if (L > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        const unsigned r0 = r[0], r1 = r[1];                                  // (a bit cast of r[1] itself reads r[0])
        v = __uint_as_float(r0) + __uint_as_float(r1);
    }
    if (L > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        const unsigned r0 = r[0], r1 = r[1];                                  // (a bit cast of r[1] itself reads r[0])
        v = __uint_as_float(r0) + __uint_as_float(r1);
    }
    return v;
}
struct NjRed {                           // the meeting place of a team of several waves: two sums, two places used in turn (one barrier per sum:
    float v[2][2][8];                    // between two uses of a place lies the barrier of the other)
};
template <int TL, bool BOTH>
__device__ __forceinline__ void nj_sum(float& a, float& b, NjRed& red, int& turn) {
    a = nj_lanes<(TL < 64 ? TL : 64)>(a);
    if (BOTH) b = nj_lanes<(TL < 64 ? TL : 64)>(b);
    if (TL > 64) {
        constexpr int NW = TL / 64;
        if (!(threadIdx.x & 63)) {
            red.v[turn][0][threadIdx.x % TL >> 6] = a;
            if (BOTH) red.v[turn][1][threadIdx.x % TL >> 6] = b;
        }
        wg_barrier();
        a = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) a += red.v[turn][0][w];
        if (BOTH) {
            b = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) b += red.v[turn][1][w];
        }
        turn ^= 1;
    }
}
__device__ __forceinline__ float nj_hsum(const t8_f4& v) { return (v[0] + v[1]) + (v[2] + v[3]); }
__device__ __forceinline__ float nj_dot(const t8_f4& a, const t8_f4& b) { return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]); }

// v -> (v - mean) r or v r in place; returns r.  Columns past the width hold zero before and after.
template <int TL, int VPT>
__device__ __forceinline__ float nj_norm(t8_f4 (&v)[VPT], int lane, const NjArgs& a, NjRed& red, int& turn) {
    const float inv = 1.0f / (float)a.W;
    float none = 0.f;
    if (a.layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) s += nj_hsum(v[i]);
        nj_sum<TL, false>(s, none, red, turn);
        s *= inv;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) v[i][c] = 4 * (i * TL + lane) + c < a.W ? v[i][c] - s : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) q += nj_dot(v[i], v[i]);
    nj_sum<TL, false>(q, none, red, turn);
    const float r = 1.0f / sqrtf(q * inv + a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] *= r;
    return r;
}
// u (times r) without its part along v^ (and, LayerNorm, without its mean): the gradient at a norm's input
template <int TL, int VPT>
__device__ __forceinline__ void nj_norm_bwd(t8_f4 (&u)[VPT], const t8_f4 (&vh)[VPT], float r, int lane, const NjArgs& a, NjRed& red, int& turn) {
    const float inv = 1.0f / (float)a.W;
    float s = 0.f, p = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) s += nj_hsum(u[i]), p += nj_dot(u[i], vh[i]);
    nj_sum<TL, true>(p, s, red, turn);
    p *= inv;
    s = a.layer ? s * inv : 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) u[i][c] = 4 * (i * TL + lane) + c < a.W ? ((u[i][c] - s) - vh[i][c] * p) * r : 0.f;
}
// the normalised row onto the tape
template <int TL, int VPT>
__device__ __forceinline__ void nj_tape(const t8_f4 (&v)[VPT], int lane, int blocks, long row, unsigned char* codes, unsigned char* bytes) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = 4 * (i * TL + lane);
        const unsigned byte = t8_byte<T8_SIGNED>(t8_max8(t8_top4<T8_SIGNED>(v[i])));
        if (c < 32 * blocks) {
            *reinterpret_cast<unsigned*>(codes + row * (32 * blocks) + c) = t8_code4<T8_SIGNED>(v[i], byte);
            if (!(lane & 7)) bytes[row * blocks + c / 32] = (unsigned char)byte;
        }
    }
}
// a row of parameters: fp32, zero past the width; `none` where there is none
__device__ __forceinline__ t8_f4 nj_par(const float* p, int c, int W, float none) { return p ? t8_load4(p + c, W - c) : t8_f4{none, none, none, none}; }
__device__ __forceinline__ t8_f4 nj_scale(const NjArgs& a, int c) {
    return a.scale_v ? nj_par(a.scale_v, c, a.W, 0.f) : t8_f4{a.scale, a.scale, a.scale, a.scale};
}
// four neighbouring values as they are in memory (a row in flight)
template <typename T>
using nj_raw = T __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ nj_raw<T> nj_load(const T* __restrict__ p, int n) {
    if (n >= 4) return *reinterpret_cast<const t8_v4<T>*>(p);
    nj_raw<T> v = nj_raw<T>(0);
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) v[i] = p[i];
    return v;
}
template <typename T>
__device__ __forceinline__ t8_f4 nj_f32(const nj_raw<T>& v) { return t8_f4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }

template <typename T, int TL, int VPT>
__global__ void __launch_bounds__(TL > 256 ? TL : 256) k_norm_join(const NjArgs a) {
    __shared__ NjRed red;
    constexpr int TEAMS = (TL > 256 ? TL : 256) / TL;
    const int lane = threadIdx.x % TL, W = a.W, blocks = (W + 31) / 32;
    const T *x = (const T*)a.x, *f = (const T*)a.f, *gate = (const T*)a.gate;
    T *y = (T*)a.y, *h = (T*)a.h;
    int turn = 0;
    t8_f4 sc[VPT], pg[VPT], pb[VPT], qg[VPT], qb[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = 4 * (i * TL + lane);
        sc[i] = nj_scale(a, c);
        pg[i] = nj_par(a.post_g, c, W, 1.f), pb[i] = nj_par(a.post_b, c, W, 0.f);
        qg[i] = nj_par(a.pre_g, c, W, 1.f), qb[i] = nj_par(a.pre_b, c, W, 0.f);
    }
    // the team's rows, and the gate row of each: advanced by the stride, split once into gate rows and the rest
    const long stride = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + threadIdx.x / TL;
    long g = row / a.rows_per_gate, in_g = row - g * a.rows_per_gate;
    const long dg = stride / a.rows_per_gate, din = stride - dg * a.rows_per_gate;
    nj_raw<T> nx[VPT], nf[VPT], ng[VPT];
    auto load = [&](long r, long gr) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            nf[i] = nj_load(f + r * a.ldf + c, W - c);
            if (x) nx[i] = nj_load(x + r * a.ldx + c, W - c);
            if (a.has_gate) ng[i] = nj_load(gate + gr * a.ldg + c, W - c);
        }
    };
    if (row < a.M) load(row, g);
    for (; row < a.M; row += stride) {
        t8_f4 v[VPT], s[VPT], m[VPT];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            v[i] = nj_f32<T>(nf[i]), s[i] = x ? nj_f32<T>(nx[i]) : t8_f4{0.f, 0.f, 0.f, 0.f};
            m[i] = a.has_gate ? sc[i] * nj_f32<T>(ng[i]) : sc[i];
        }
        g += dg, in_g += din;
        if (in_g >= a.rows_per_gate) in_g -= a.rows_per_gate, ++g;
        if (row + stride < a.M) load(row + stride, g);
        if (a.has_post) {
            const float rs = nj_norm<TL, VPT>(v, lane, a, red, turn);
            if (a.tape && lane == 0) a.post_r[row] = rs;
        }
        if (a.tape) nj_tape<TL, VPT>(v, lane, blocks, row, a.post_c, a.post_e);
        if (!y) continue;                                                     // (the tape is all that is wanted: magnet_norm_tape)
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            s[i] += m[i] * (v[i] * pg[i] + pb[i]);                            // (gain one, bias zero where there is none)
            t8_store4(y + row * a.ldy + c, W - c, s[i]);
        }
        if (!a.has_pre) continue;
        // (the second norm reads y before it is rounded to T)
        const float rs = nj_norm<TL, VPT>(s, lane, a, red, turn);
        if (a.tape) {
            if (lane == 0) a.pre_r[row] = rs;
            nj_tape<TL, VPT>(s, lane, blocks, row, a.pre_c, a.pre_e);
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            t8_store4(h + row * a.ldh + c, W - c, s[i] * qg[i] + qb[i]);
        }
    }
}

// Which rows a team walks, and where the sums of a gate row meet:
//   no gate:          any rows, one set of sums for the launch
//   G gate rows, few: per_group workgroups for each, their sums stay apart (S1, S0 without the gate) and meet in k_norm_join_gate
//   many (OWN):       a team takes whole gate rows one after the other - up to one for every row - and writes their gradients itself
template <typename T, int TL, int VPT, bool OWN>
__global__ void __launch_bounds__(TL > 64 ? 512 : 256) k_norm_join_bwd(const NjArgs a) {
    constexpr int NT = TL > 64 ? 512 : 256, TEAMS = NT / TL;
    __shared__ NjRed reds[TL > 64 ? TEAMS : 1];
    __shared__ __attribute__((aligned(16))) float part[TEAMS > 1 ? NT * 4 : 4];
    const int lane = threadIdx.x % TL, team = threadIdx.x / TL, W = a.W, blocks = (W + 31) / 32;
    NjRed& red = reds[TL > 64 ? team : 0];
    const T *gy = (const T*)a.x, *gh = (const T*)a.f, *gate = (const T*)a.gate;
    T *dx = (T*)a.y, *df = (T*)a.h, *dgate = (T*)a.dgate;
    int turn = 0;
    t8_f4 sc[VPT], pg[VPT], pb[VPT], qg[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = 4 * (i * TL + lane);
        sc[i] = nj_scale(a, c);
        pg[i] = nj_par(a.post_g, c, W, 1.f), qg[i] = nj_par(a.pre_g, c, W, 1.f);
        if (OWN) pb[i] = nj_par(a.post_b, c, W, 0.f);
    }
    // this team's rows: `row`, then row + step up to the gate row's last; OWN: then the gate row g + g_step
    const long me = (long)blockIdx.x * TEAMS + team, g_step = (long)gridDim.x * TEAMS;
    long g = OWN ? me : a.per_group ? blockIdx.x / a.per_group : 0;
    const long step = OWN ? 1 : (long)(a.per_group ? a.per_group : gridDim.x) * TEAMS;
    long row = g * a.rows_per_gate + (OWN ? 0 : a.per_group ? (long)(blockIdx.x % a.per_group) * TEAMS + team : me);
    long last = (g + 1) * a.rows_per_gate;
    // teams of several waves meet at the workgroup's barriers: all of them go round as often as the first one, which has the most rows (OWN: rows
    // and last move alike in all teams, past the last gate row too)
    const int lead = TL > 64 ? team : 0;
    bool more = OWN ? g - lead < a.groups : row - lead < last, on = OWN ? g < a.groups : row < last;
    nj_raw<T> ny[VPT], nh[VPT], ng[VPT];
    unsigned npc[VPT], nqc[VPT], npe[VPT], nqe[VPT];
    float npr = 1.f, nqr = 1.f;
    auto load = [&](long r, long gr) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            ny[i] = nj_load(gy + r * a.ldx + c, W - c);
            if (a.has_pre) nh[i] = nj_load(gh + r * a.ldf + c, W - c);
            if (a.has_gate) ng[i] = nj_load(gate + gr * a.ldg + c, W - c);
            npc[i] = npe[i] = nqc[i] = nqe[i] = 0u;
            if (c < W) {
                npc[i] = *reinterpret_cast<const unsigned*>(a.post_c + r * (32 * blocks) + c);
                npe[i] = a.post_e[r * blocks + c / 32];
                if (a.has_pre) {
                    nqc[i] = *reinterpret_cast<const unsigned*>(a.pre_c + r * (32 * blocks) + c);
                    nqe[i] = a.pre_e[r * blocks + c / 32];
                }
            }
        }
        if (a.has_post) npr = a.post_r[r];
        if (a.has_pre) nqr = a.pre_r[r];
    };
    t8_f4 S1[VPT], S0[VPT], P1[VPT], P0[VPT], T1[VPT], T0[VPT];               // T: of the gate row so far, without the gate
#pragma unroll
    for (int i = 0; i < VPT; ++i) S1[i] = S0[i] = P1[i] = P0[i] = T1[i] = T0[i] = t8_f4{0.f, 0.f, 0.f, 0.f};
    if (on) load(row, g);
    while (more) {
        t8_f4 D[VPT], v[VPT], gt[VPT], u[VPT], q[VPT];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            D[i] = nj_f32<T>(ny[i]);
            v[i] = t8_decode4<T8_SIGNED>(npc[i], npe[i]);
            gt[i] = a.has_gate ? nj_f32<T>(ng[i]) : t8_f4{1.f, 1.f, 1.f, 1.f};
            if (a.has_pre) u[i] = nj_f32<T>(nh[i]), q[i] = t8_decode4<T8_SIGNED>(nqc[i], nqe[i]);
        }
        const float pr = npr, qr = nqr;
        // the row after this one, on its way while this one is worked on
        const long r = row, gr = g;
        const bool here = TL > 64 ? __builtin_amdgcn_readfirstlane(on) : true;
        row += step;
        bool ends = false;
        if (OWN) {
            ends = row >= last;
            if (ends) {
                g += g_step;
                row = g * a.rows_per_gate, last = row + a.rows_per_gate;
                more = g - lead < a.groups, on = g < a.groups;
            }
        } else {
            more = row - lead < last, on = row < last;
        }
        if (on) load(row, g);
        if (a.has_pre) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                if (here) P0[i] += u[i], P1[i] += u[i] * q[i];
                u[i] *= qg[i];
            }
            nj_norm_bwd<TL, VPT>(u, q, qr, lane, a, red, turn);
#pragma unroll
            for (int i = 0; i < VPT; ++i) D[i] += u[i];
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            if (here) {
                if (dx) t8_store4(dx + r * a.ldy + c, W - c, D[i]);
                T0[i] += D[i], T1[i] += D[i] * v[i];
            }
            D[i] *= gt[i] * sc[i] * pg[i];
        }
        if (a.has_post) nj_norm_bwd<TL, VPT>(D, v, pr, lane, a, red, turn);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = 4 * (i * TL + lane);
            if (!here) break;
            t8_store4(df + r * a.ldh + c, W - c, D[i]);
            if (OWN && ends) {
                t8_store4(dgate + gr * W + c, W - c, (T1[i] * pg[i] + T0[i] * pb[i]) * sc[i]);
                S1[i] += gt[i] * T1[i], S0[i] += gt[i] * T0[i];
                T1[i] = T0[i] = t8_f4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    if (!a.need_sums) return;
    // ---- the workgroup's sums: the teams in order
    float* out = a.part + (size_t)blockIdx.x * 4 * W;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if ((q & 1) && !a.plain_sums) continue;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            t8_f4 s = q == 0 ? (OWN ? S1[i] : T1[i]) : q == 1 ? (OWN ? S0[i] : T0[i]) : q == 2 ? P1[i] : P0[i];
            const int c = 4 * (i * TL + lane);
            if (TEAMS > 1) {
                __syncthreads();
                *reinterpret_cast<t8_f4*>(&part[4 * threadIdx.x]) = s;
                __syncthreads();
                if (team == 0) {
                    s = *reinterpret_cast<const t8_f4*>(&part[4 * lane]);
                    for (int t = 1; t < TEAMS; ++t) s += *reinterpret_cast<const t8_f4*>(&part[4 * (t * TL + lane)]);
                }
            }
            if (team == 0)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (c + k < W) out[q * W + c + k] = s[k];
        }
    }
}

// sums of a column over n of the workgroups' sets (`first`, first + apart, ..), in order: a workgroup takes 32 columns, 32 slices of the sets each; the total in
// v of slice 0.  STEP 2: of S1 and P1 alone
template <int STEP>
__device__ __forceinline__ void nj_fold(const float* part, long first, int n, long apart, int W, int c, float (&v)[4], float (*s)[4][32]) {
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = 0.f;
    if (c < W)
#pragma unroll 4
        for (int w = slice; w < n; w += 32) {
            const float* p = part + (first + w * apart) * 4 * W + c;
#pragma unroll
            for (int q = 0; q < 4; q += STEP) v[q] += p[(long)q * W];
        }
#pragma unroll
    for (int q = 0; q < 4; q += STEP) s[slice][q][col] = v[q];
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int q = 0; q < 4; q += STEP) {
        v[q] = s[0][q][col];
        for (int k = 1; k < 32; ++k) v[q] += s[k][q][col];
    }
}
// one gate row (blockIdx.y): its gradient, and its workgroups' sums with the gate multiplied in, left in the first one's place
template <typename T, int STEP>
__global__ void __launch_bounds__(1024) k_norm_join_gate(const NjArgs a) {
    __shared__ float s[32][4][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), W = a.W;
    const long g = blockIdx.y;
    float v[4];
    nj_fold<STEP>(a.part, g * a.per_group, a.per_group, 1, W, c, v, s);
    if (threadIdx.x >= 32 || c >= W) return;
    const float gt = (float)((const T*)a.gate)[g * a.ldg + c], sc = a.scale_v ? a.scale_v[c] : a.scale;
    const float t = v[0] * (a.has_post ? a.post_g[c] : 1.f) + (a.post_b ? v[1] * a.post_b[c] : 0.f);
    ((T*)a.dgate)[g * W + c] = (T)(sc * t);
    float* p = a.part + g * a.per_group * 4 * W + c;
    p[0] = gt * v[0], p[W] = gt * v[1], p[2 * W] = v[2], p[3 * W] = v[3];
}
// the parameters' gradients from n sets of sums, `apart` sets from one to the next
template <int STEP>
__global__ void __launch_bounds__(1024) k_norm_join_params(const NjArgs a, int n, int apart, float* d_scale, float* d_post_g, float* d_post_b, float* d_pre_g,
                                                          float* d_pre_b) {
    __shared__ float s[32][4][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31);
    float v[4];
    nj_fold<STEP>(a.part, 0, n, apart, a.W, c, v, s);
    if (threadIdx.x >= 32 || c >= a.W) return;
    const float sc = a.scale_v ? a.scale_v[c] : a.scale;
    if (d_scale) d_scale[c] = v[0] * (a.has_post ? a.post_g[c] : 1.f) + (a.post_b ? v[1] * a.post_b[c] : 0.f);
    if (d_post_g) d_post_g[c] = sc * v[0];
    if (d_post_b) d_post_b[c] = sc * v[1];
    if (d_pre_g) d_pre_g[c] = v[2];
    if (d_pre_b) d_pre_b[c] = v[3];
}

// ---------------------------------------------------------------------------------------------------------------------------- launches
#define NJ_MAX_W 4096
// lanes of a row's team: two slots of four columns each, sixteen lanes at least (rows of 513 .. 1024 values: four waves with one slot each,
// so that a workgroup of four waves is one row's)
static int nj_team(int W) { return W <= 128 ? 16 : W <= 256 ? 32 : W <= 512 ? 64 : W <= 2048 ? 256 : 512; }
static int nj_teams(int W) { return W <= 2048 ? 256 / nj_team(W) : 1; }
// one row a team while that makes at most 1024 workgroups, then four rows a team (the parameters are loaded once for all of them): 262 144 x 128
// with tapes 166 us (one row a team 180, sixteen 174), 8190 x 2048 39 us (50, 44); at most 4096 workgroups
static long nj_grid(long M, int W) {
    const int teams = nj_teams(W);
    const long n = (M + teams - 1) / teams;
    return n < 1024 ? n : n < 4096 ? 1024 : n < 16384 ? n / 4 : 4096;
}
// backward: workgroups, and how many of them share a gate row (0: they are not bound to gate rows).  Up to 2048 gate rows get workgroups of
// their own - a set of sums each, added by a second launch; beyond that a team walks whole gate rows and no sums are kept per row.  Rows of
// 513 .. 2048 values go two at a time in a workgroup of eight waves: twice the rows in flight for the same partial sums (20 000 x 1000: 88 us, one at a
// time 102; bf16 61, 80).  What the registers hold of a CU's rows is 512 workgroups up to a width of 1024, 256 beyond (bf16 8000 x 2048: 64 us, 512
// of them 72; 8000 rows of 4096: 146, 155)
static long nj_bwd_grid(long M, int W, long G, int* per_group) {
    const int teams = W <= 512 ? nj_teams(W) : 512 / nj_team(W), most = W <= 1024 ? 512 : 256;
    *per_group = 0;
    if (G <= 0 || G > 2048 || G == M) {
        const long n = ((G > 2048 ? G : M) + teams - 1) / teams;
        return n < most ? n : most;
    }
    const long each = (M / G + teams - 1) / teams, n = G < most ? most / G : 1;
    *per_group = (int)(each < n ? each : n);
    return G * *per_group;
}
extern "C" int magnet_norm_join_bwd_workspace(long M, long W, long G, long* floats) {
    int per = 0;
    if (M < 1 || W < 1 || W > NJ_MAX_W || G < 0 || (G && M % G)) return -2;
    *floats = nj_bwd_grid(M, (int)W, G, &per) * 4 * W;
    return 0;
}

template <typename T>
static void nj_forward(const NjArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)nj_grid(a.M, a.W));
    const int W = a.W;
    if (W <= 64) k_norm_join<T, 16, 1><<<grid, 256, 0, st>>>(a);
    else if (W <= 128) k_norm_join<T, 16, 2><<<grid, 256, 0, st>>>(a);
    else if (W <= 256) k_norm_join<T, 32, 2><<<grid, 256, 0, st>>>(a);
    else if (W <= 512) k_norm_join<T, 64, 2><<<grid, 256, 0, st>>>(a);
    else if (W <= 1024) k_norm_join<T, 256, 1><<<grid, 256, 0, st>>>(a);
    else if (W <= 2048) k_norm_join<T, 256, 2><<<grid, 256, 0, st>>>(a);
    else k_norm_join<T, 512, 2><<<grid, 512, 0, st>>>(a);
}
template <typename T, bool OWN>
static void nj_backward(const NjArgs& a, dim3 grid, hipStream_t st) {
    const int W = a.W;
    if (W <= 64) k_norm_join_bwd<T, 16, 1, OWN><<<grid, 256, 0, st>>>(a);
    else if (W <= 128) k_norm_join_bwd<T, 16, 2, OWN><<<grid, 256, 0, st>>>(a);
    else if (W <= 256) k_norm_join_bwd<T, 32, 2, OWN><<<grid, 256, 0, st>>>(a);
    else if (W <= 512) k_norm_join_bwd<T, 64, 2, OWN><<<grid, 256, 0, st>>>(a);
    else if (W <= 1024) k_norm_join_bwd<T, 256, 1, OWN><<<grid, 512, 0, st>>>(a);
    else if (W <= 2048) k_norm_join_bwd<T, 256, 2, OWN><<<grid, 512, 0, st>>>(a);
    else k_norm_join_bwd<T, 512, 2, OWN><<<grid, 512, 0, st>>>(a);
}
extern "C" int magnet_norm_join(const void* x, long ldx, const void* f, long ldf, int dtype, long M, int W, int layer, float eps, const float* post_g,
                                const float* post_b, const float* pre_g, const float* pre_b, const void* gate, long ldg, long G, const float* scale_v,
                                float scale, void* y, void* h, void* post_codes, void* post_bytes, float* post_rstd, void* pre_codes, void* pre_bytes,
                                float* pre_rstd, void* stream) {
    if (M < 0 || W < 1 || W > NJ_MAX_W || ldx < W || ldf < W || (dtype != T8_F32 && dtype != T8_BF16) || (gate && (G < 1 || M % G || ldg < W))) return -2;
    if (M == 0) return 0;
    if (!y || (post_b && !post_g) || (pre_b && !pre_g) || (pre_g && !h)) return -2;
    const int tape = post_codes != nullptr;
    if (tape && (!post_bytes || (post_g && !post_rstd) || (pre_g && (!pre_codes || !pre_bytes || !pre_rstd)))) return -2;
    NjArgs a = {};
    a.x = x, a.f = f, a.gate = gate, a.scale_v = scale_v, a.post_g = post_g, a.post_b = post_b, a.pre_g = pre_g, a.pre_b = pre_b, a.y = y, a.h = h;
    a.post_c = (unsigned char*)post_codes, a.post_e = (unsigned char*)post_bytes, a.pre_c = (unsigned char*)pre_codes, a.pre_e = (unsigned char*)pre_bytes;
    a.post_r = post_rstd, a.pre_r = pre_rstd, a.M = M, a.ldx = ldx, a.ldf = ldf, a.ldg = ldg, a.ldy = W, a.ldh = W;
    a.rows_per_gate = gate ? M / G : M, a.W = W, a.layer = layer, a.has_post = post_g != nullptr, a.has_pre = pre_g != nullptr, a.has_gate = gate != nullptr;
    a.tape = tape, a.scale = scale, a.eps = eps;
    if (dtype == T8_F32) nj_forward<float>(a, (hipStream_t)stream);
    else nj_forward<__bf16>(a, (hipStream_t)stream);
    return (int)hipGetLastError();
}

extern "C" int magnet_norm_tape(const void* z, long ldz, int dtype, long M, int W, int layer, float eps, void* codes, void* bytes, float* rstd, void* stream) {
    if (M < 0 || W < 1 || W > NJ_MAX_W || ldz < W || (dtype != T8_F32 && dtype != T8_BF16)) return -2;
    if (M == 0) return 0;
    if (!codes || !bytes || !rstd) return -2;
    NjArgs a = {};
    a.f = z, a.post_c = (unsigned char*)codes, a.post_e = (unsigned char*)bytes, a.post_r = rstd, a.M = M, a.ldf = ldz, a.rows_per_gate = M, a.W = W;
    a.layer = layer, a.has_post = 1, a.tape = 1, a.eps = eps;
    if (dtype == T8_F32) nj_forward<float>(a, (hipStream_t)stream);
    else nj_forward<__bf16>(a, (hipStream_t)stream);
    return (int)hipGetLastError();
}

extern "C" int magnet_norm_join_bwd(const void* gy, long ldgy, const void* gh, long ldgh, int dtype, long M, int W, int layer, const float* post_g,
                                    const float* post_b, const float* pre_g, const float* pre_b, const void* gate, long ldg, long G, const float* scale_v,
                                    float scale, const void* post_codes, const void* post_bytes, const float* post_rstd, const void* pre_codes,
                                    const void* pre_bytes, const float* pre_rstd, void* dx, void* df, void* dgate, float* d_scale, float* d_post_g,
                                    float* d_post_b, float* d_pre_g, float* d_pre_b, float* workspace, void* stream) {
    if (M < 1 || W < 1 || W > NJ_MAX_W || ldgy < W || (dtype != T8_F32 && dtype != T8_BF16) || !df || (gate && (G < 1 || M % G || ldg < W || !dgate)))
        return -2;
    if (!post_codes || !post_bytes || (post_g && !post_rstd) || (pre_g && (!gh || ldgh < W || !pre_codes || !pre_bytes || !pre_rstd))) return -2;
    NjArgs a = {};
    a.x = gy, a.f = gh, a.gate = gate, a.scale_v = scale_v, a.post_g = post_g, a.post_b = post_b, a.pre_g = pre_g, a.pre_b = pre_b, a.y = dx, a.h = df;
    a.post_c = (unsigned char*)post_codes, a.post_e = (unsigned char*)post_bytes, a.pre_c = (unsigned char*)pre_codes, a.pre_e = (unsigned char*)pre_bytes;
    a.post_r = (float*)post_rstd, a.pre_r = (float*)pre_rstd, a.dgate = dgate, a.part = workspace;
    a.M = M, a.ldx = ldgy, a.ldf = ldgh, a.ldg = ldg, a.ldy = W, a.ldh = W, a.rows_per_gate = gate ? M / G : M, a.W = W, a.layer = layer;
    a.has_post = post_g != nullptr, a.has_pre = pre_g != nullptr, a.has_gate = gate != nullptr, a.scale = scale;
    const long grid = nj_bwd_grid(M, W, gate ? G : 0, &a.per_group);
    a.groups = gate ? G : 1;
    a.need_sums = a.per_group || d_scale || d_post_g || d_post_b || d_pre_g || d_pre_b;
    a.plain_sums = post_b || d_post_b || d_pre_b;
    hipStream_t st = (hipStream_t)stream;
    const bool own = gate && !a.per_group;
    if (dtype == T8_F32) own ? nj_backward<float, true>(a, dim3((unsigned)grid), st) : nj_backward<float, false>(a, dim3((unsigned)grid), st);
    else own ? nj_backward<__bf16, true>(a, dim3((unsigned)grid), st) : nj_backward<__bf16, false>(a, dim3((unsigned)grid), st);
    const dim3 pg((W + 31) / 32, a.per_group ? (unsigned)G : 1);
    if (a.per_group) {
        if (dtype == T8_F32) a.plain_sums ? k_norm_join_gate<float, 1><<<pg, 1024, 0, st>>>(a) : k_norm_join_gate<float, 2><<<pg, 1024, 0, st>>>(a);
        else a.plain_sums ? k_norm_join_gate<__bf16, 1><<<pg, 1024, 0, st>>>(a) : k_norm_join_gate<__bf16, 2><<<pg, 1024, 0, st>>>(a);
    }
    if (d_scale || d_post_g || d_post_b || d_pre_g || d_pre_b)
        (a.plain_sums ? k_norm_join_params<1> : k_norm_join_params<2>)<<<dim3(pg.x), 1024, 0, st>>>(a, a.per_group ? (int)G : (int)grid, a.per_group ? a.per_group : 1, d_scale, d_post_g, d_post_b, d_pre_g, d_pre_b);
    return (int)hipGetLastError();
}
