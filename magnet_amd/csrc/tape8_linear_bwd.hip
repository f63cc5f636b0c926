// One Linear walked back from an 8-bit tape of its input (tape8.cuh), in one pass over the rows:
//     x  = act(v)   v = the tape's value: the activated input itself (none, relu) or Swish's argument (swish)
//     dx [M][K] = act'(v) (dz W)        dW [N][K] (+)= dz^T x        db [N] (+)= column sums of dz
// What has to move is dz in, dx out and 33/32 bytes a value of the tape: 1156 bytes a row at N = K = 128, where fp32 activations make it
// 1536 (linear_bwd.hip).  Measured, a call: 2 097 152 rows of 128 x 128 behind a ReLU 547 us (4.4 TB/s; a large copy reaches 4.9; the kernel
// that reads fp32 activations 650 - 672), 218 453 rows of 64 x 64 37 us (30 - 32 in this kernel), 262 144 rows of 128 x 128 behind Swish
// 112 us.  Behind Swish 44 % of the SIMDs' cycles issue vector instructions and 22 % matrix ones, and a wave waits 44 % of its own: one
// workgroup a CU, whose waves all form exponentials, meet and then all multiply.  (Where two variants are compared below, both were measured
// with one scale for all rows of a workgroup: 3 % faster.)
//
// A workgroup of four or eight waves takes steps of 32 or 64 rows of one block of at most 128 x 128 of W.  dz is split once into two fp16 planes
// (h + l, 22 bits), the tape's codes need one plane - a code has 8 bits, fp16 holds code times a power of two exactly - (two behind
// Swish), and both meet as 16 x 16 x 32 matrix products through LDS:
//   dx^T = W^T dz^T   A = the wave's features of W^T, two planes kept in registers; B = rows of the dz image; products hh + hl + lh
//   dW   = dz^T x     A, B = transposed LDS reads of the two images, k = 32 of the step's rows; products (h + l) x
// The error of both is a few 2^-22 of the operands' magnitude, sums are held in fp32, and the workgroups' partial sums of dW and db are added
// in their order by a second kernel: the same bits every time.
//
// Scales.  fp16 spans 2^40; gradients (1e-7) and tapes (any byte) do not fit by themselves.  Every row of dz is staged times the power of two
// that puts its own largest value into [2^14, 2^15), and dx undoes it row by row: a row of dx is as good as its row of dz, whatever the
// others are, down to 2^-39 of the row's largest value.  dW needs all rows at one scale, so a row's codes take the difference: they are
// staged times 2^(row's exponent + block's byte - bound + 5), one bound for each 32 columns of x: where the largest product of a row
// of dz and a block lies, smaller ones lose what is under 2^-32 of it.  (Behind Swish the exponent of the value itself stands for the byte: far
// from zero on the negative side it has nothing to do with the argument's.)  A lane that meets a product above its bound raises a flag
// with its write; behind the barrier that the step has anyway all waves see it, add their sums so far to the workgroup's partial sums in
// memory and begin again under a new bound (with a few binades to spare): rare after the first step, and nobody waits for a maximum
// otherwise.  (Scaling the sums in registers instead costs a second set of them: measured as spills.)  A row's largest value is a few lane
// permutes, and the wave that stages a row of dz stages its codes too, so the exponent never waits for another wave.  W's columns
// have a scale each as well, by their largest value in the block of 128 rows: dx of one owes nothing to the others.
#include "common.cuh"
#include "split_single.cuh"
#include "tape8.cuh"

typedef _Float16 t8_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 t8_hp __attribute__((ext_vector_type(2)));
typedef short t8_s4 __attribute__((__vector_size__(4 * sizeof(short))));

struct T8LinArgs {
    const float* dz;                     // [M][ldz], this launch's N columns
    const unsigned char* codes;          // [M][ldc], ldc = 32 ceil(width / 32)
    const unsigned char* bytes;          // [M][ldc / 32]
    const float* w;                      // [N][ldw]
    float* dx;                           // [M][lddx]
    float* wpart;                        // [K blocks][gridDim.x][NP][KP] partial sums of dW
    float* bpart;                        // [gridDim.x][NP] partial sums of db
    long M, ldz, ldw, lddx;
    int N, K, ldc, exact, add_dx;        // exact: N = NP and K a multiple of KP; add_dx: dx += (a later block of N)
    int kb0;                             // the launch's first block of K
};

template <int CTRL>
__device__ __forceinline__ unsigned t8_dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
// the maxima of P values each over L = 16 or 32 neighbouring lanes: value p's comes out in the lanes whose number is p modulo P
template <int P, int L>
__device__ __forceinline__ unsigned t8_row_max(const unsigned (&m)[P], int lane) {
    static_assert(P == 2 || P == 4, "two or four values");
    const bool odd = lane & 1, two = lane & 2;
    unsigned v = max(odd ? m[1] : m[0], t8_dpp<0xB1>(odd ? m[0] : m[1]));                       // quad_perm 1 0 3 2: the neighbour hands over what it is not for
    if (P == 4) {
        const unsigned w = max(odd ? m[P - 1] : m[P - 2], t8_dpp<0xB1>(odd ? m[P - 2] : m[P - 1]));
        v = max(two ? w : v, t8_dpp<0x4E>(two ? v : w));                                      // quad_perm 2 3 0 1
    } else {
        v = max(v, t8_dpp<0x4E>(v));
    }
    v = max(v, t8_dpp<0x124>(v));                                                             // row_ror 4, 8: the other quads of sixteen lanes
    v = max(v, t8_dpp<0x128>(v));
    if (L == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        const unsigned r0 = r[0], r1 = r[1];
        v = max(r0, r1);
    }
    return v;
}
// exponent byte (1 .. 254) of a magnitude's bits; 0 for zero, subnormals and what is not finite
__device__ __forceinline__ unsigned t8_expo(float v) {
    const unsigned e = (__float_as_uint(v) >> 23) & 0xFFu;
    return e == 255u ? 0u : e;
}
__device__ __forceinline__ float t8_pow2(int biased) { return __uint_as_float((unsigned)min(max(biased, 0), 254) << 23); }
// four halfwords of a column out of a 16 x 4 tile: lane i of 16 points at row i / 4, columns 4 (i % 4) .., and gets column i
__device__ __forceinline__ t8_u2 t8_tr(const unsigned short* p) {
    return __builtin_bit_cast(t8_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) t8_s4*)(p)));
}
__device__ __forceinline__ t8_h8 t8_join(t8_u2 a, t8_u2 b) { return __builtin_bit_cast(t8_h8, t8_u4{a[0], a[1], b[0], b[1]}); }
// e^-v and s = 1 / (1 + e^-v), both finite.  Under -87, where e^-v nears the end of fp32, s is 0, and with it Swish and its derivative: what
// either still is there lies under 2^-118
__device__ __forceinline__ float t8_sigmoid(float v, float& e) {
    e = __expf(fminf(-v, 87.0f));
    return v < -87.0f ? 0.f : __builtin_amdgcn_rcpf(1.0f + e);
}
// Swish v s and its derivative s (1 + v (1 - s)) with 1 - s = e^-v s: no cancellation where s is near 1
__device__ __forceinline__ float t8_swish(float v, float& d) {
    float e;
    const float s = t8_sigmoid(v, e), y = v * s;
    d = s + y * (e * s);
    return y;
}

#define T8_WAVES(NP, KP) ((NP) == 128 && (KP) == 128 ? 8 : 4)
// rows of a step: 64 where two steps in LDS leave room for what a CU can hold in registers anyway (128 x 128: 539 us against 564 with 32 at
// 2 097 152 rows; 64 x 64: 34 against 38 at 218 453); 32 for the mixed shapes (two workgroups a CU) and behind Swish (two planes)
#define T8_ROWS(NP, KP, ACT) ((NP) == (KP) && (ACT) != ACT_SWISH ? 64 : 32)
#define T8_TILE(NP, KP, ACT) ((NP) == 128 && (KP) == 128 && (ACT) == ACT_SWISH ? 1 : 2)       // blocks of 16 features of a wave's tiles
#define T8_FOLD 8                        // steps whose products are added up in a row before they join the sums so far: a chain of additions in fp32
                                         // is off by its length (2 097 152 rows: 1.7e-6 of dW in one chain per workgroup)
// binades by which the products of dz and x may still grow before the scale has to change (behind Swish, whose values spread wider than a tape's
// bytes, and have a bit more of fp16's range, one more)
#define T8_ROOM(ACT) ((ACT) == ACT_SWISH ? 4 : 3)
template <int NP, int KP, int XPL, int R, int ACT>
struct T8Step {                          // a step of R rows in LDS; row strides of 16 halfwords more than a power of two spread the rows over the banks
    unsigned short z[2][R][NP + 16];
    unsigned short x[XPL][R][KP + 16];
    unsigned c[ACT == ACT_RELU ? R : 1][KP / 4 + 4];       // the codes (the mask of dx)
    float d[ACT == ACT_SWISH ? R : 1][KP + 4];             // Swish's derivative: formed where Swish is, from the same exponential
    int e[R];                                              // the rows' exponents: z is dz times 2^(141 - e)
};

// a value at a wave-uniform base plus the lane's offset in bytes (global_* with a scalar base: the caller hides the base behind an asm statement,
// or the compiler adds the two and keeps 64 bits per lane and access in registers)
template <typename V>
__device__ __forceinline__ V t8_at(const void* base, unsigned off) {
    return *reinterpret_cast<__attribute__((address_space(1))) const V*>((__attribute__((address_space(1))) const char*)(base) + off);
}
template <typename V>
__device__ __forceinline__ void t8_put(void* base, unsigned off, const V& v) {
    *reinterpret_cast<__attribute__((address_space(1))) V*>((__attribute__((address_space(1))) char*)(base) + off) = v;
}
#define T8_UNIFORM(p) asm volatile("" : "+s"(p))

// FULL: at least 64 rows, N and K multiples of four, one block of N.  Addresses are then a uniform base and one offset per lane, and nothing is
// loaded under a condition (the registers that bounds and addresses take are what decides between spilling and not): a lane whose
// columns do not exist loads existing ones instead - of dz times a scale of zero, of the tape into columns of dx and dW that are not
// written - and the last step takes the last R rows, those done already likewise.
// 128 x 128 has eight waves, the smaller shapes four.  A wave's tiles are near square - 32 features of x by half the rows for dx, 32 features
// of dz by 64 of x for dW - because what a tile needs from LDS is its two edges: 524 us at 2 097 152 rows, 537 with sixteen features by all
// rows for each wave.  Behind Swish, where a step has half the rows, it is the other way round: 105 us against 118 at 262 144 rows.
template <int NP, int KP, int ACT, bool FULL>
__global__ void __launch_bounds__(T8_WAVES(NP, KP) * 64, 2) k_tape8_linear_bwd(const T8LinArgs a) {
    constexpr int KIND = ACT == ACT_RELU ? T8_RELU : T8_SIGNED;
    constexpr int XPL = ACT == ACT_SWISH ? 2 : 1;                             // planes of x
    constexpr int R = T8_ROWS(NP, KP, ACT);
    typedef T8Step<NP, KP, XPL, R, ACT> Step;
    constexpr int NW = T8_WAVES(NP, KP), LANES = 64 * NW;
    // a wave stages WR neighbouring rows, of dz and of the codes
    constexpr int LPR = NP / 4, WR = R / NW, NLD = WR * LPR / 64;             // lanes per row of dz, rows (one after the other) of each such lane
    constexpr int CPT = R * KP / LANES, CPR = KP / CPT, CW = CPT / 4;        // codes per lane (8 or 16), lanes per row, words
    static_assert(WR * CPR == 64 && LPR == NLD * CPR, "LPR neighbouring lanes hold the codes of their rows of dz");
    // a wave's part: dx of NBK blocks of 16 features and 1 / RW of the rows; dW of NBN blocks of features of dz and KB of features of x
    constexpr int NBK = T8_TILE(NP, KP, ACT), NBN = NBK, NT = NP / 32;
    constexpr int KW = KP / 16 / NBK, RW = NW / KW, RBS = R / 16 / RW, RB = RBS < 2 ? RBS : 2;
    constexpr int NG = NP / 16 / NBN, XG = NW / NG, KB = KP / 16 / XG;
    constexpr int TB = KB / 2, CB = KP / 32, LB = 32 / CPT;                   // blocks of 32 columns: of the wave's dW, of all; lanes per block
    static_assert(KW * RW == NW && NG * XG == NW && RBS * 16 * RW == R, "waves tile both products");
    typedef unsigned t8_cw __attribute__((ext_vector_type(CW)));
    __shared__ __attribute__((aligned(16))) Step sb[2];
    __shared__ unsigned red[NW][CB], flag[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int k0 = (a.kb0 + blockIdx.y) * KP;
    const int kf = 16 * NBK * (wave % KW), wr = (wave / KW) * (R / RW);       // its features and rows of dx
    const int nf = 16 * NBN * (wave % NG), xf = 16 * KB * (wave / NG);        // its features of dz and of x in dW
    // ---- what this lane loads of a step
    const int zl = lane / LPR * NLD, zr = wave * WR + zl, zc = 4 * (lane % LPR);         // rows zr, zr + 1 ..
    const int cr = tid / CPR, cc = CPT * (tid % CPR);
    const bool c_on = k0 + cc < a.ldc;
    const int lb = a.ldc / 32;
    t8_f4 dv[NLD];
    t8_cw cv = t8_cw(0u);
    unsigned bv = 0;
    int shift = 0;                                                            // FULL, the last step: it takes the last R rows, this many of them done
    auto load = [&](long step) {
        if (FULL) {
            const long row = min(step * R, a.M - R);
            const int zcl = zc < a.N ? zc : 0, ccl = c_on ? cc : 0;
            const unsigned oz = ((unsigned)zl * (unsigned)a.ldz + zcl) * 4u, oc = (unsigned)cr * (unsigned)a.ldc + ccl, ob = (unsigned)cr * (unsigned)lb + ccl / 32;
            const unsigned char *bc = a.codes + row * a.ldc + k0, *bb = a.bytes + row * lb + k0 / 32;
            T8_UNIFORM(bc);
            T8_UNIFORM(bb);
#pragma unroll
            for (int i = 0; i < NLD; ++i) {
                const float* p = a.dz + (row + wave * WR + i) * a.ldz;
                T8_UNIFORM(p);
                dv[i] = t8_at<t8_v4<float>>(p, oz);
            }
            cv = t8_at<t8_cw>(bc, oc), bv = t8_at<unsigned char>(bb, ob);
            return;
        }
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const long r = step * R + zr + i;
            dv[i] = r < a.M ? t8_load4(a.dz + r * a.ldz + zc, a.N - zc) : t8_f4{0.f, 0.f, 0.f, 0.f};
        }
        const long r = step * R + cr;
        const bool on = c_on && r < a.M;
        cv = on ? *reinterpret_cast<const t8_cw*>(a.codes + r * a.ldc + k0 + cc) : t8_cw(0u);
        bv = on ? a.bytes[r * lb + (k0 + cc) / 32] : 0u;
    };
    const long nsteps = (a.M + R - 1) / R;
    long step = blockIdx.x;
    load(step);
    // ---- the wave's features of W^T: A operands (lane = feature of x, register j of k group q4 = feature 32 t + 8 q4 + j of dz)
    t8_h8 wh[NBK][NT], wl[NBK][NT];
    unsigned we[NBK];                                                         // a feature of x is staged times 2^(140 - its exponent): max |W| over dz -> [2^13, 2^14);
                                                                              // kept of features 4 q4 .. + 3 of a block, a byte each: what the lane gets of dx
    {
        auto w_at = [&](int b, int t, int j) -> float {
            const int n = 32 * t + 8 * q4 + j, k = k0 + kf + 16 * b + n16;
            if (FULL && a.exact) {
                const float* p = a.w + (32 * t + j) * a.ldw + k0 + kf + 16 * b;
                T8_UNIFORM(p);
                return t8_at<float>(p, ((unsigned)(8 * q4) * (unsigned)a.ldw + n16) * 4u);
            }
            return n < a.N && k < a.K ? a.w[n * a.ldw + k] : 0.f;
        };
        float wv[NBK][NT][8];                                                 // (the sums' registers are not in use yet)
#pragma unroll
        for (int b = 0; b < NBK; ++b)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) wv[b][t][j] = w_at(b, t, j);
#pragma unroll
        for (int b = 0; b < NBK; ++b) {
            unsigned et = 14;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) et = max(et, t8_expo(wv[b][t][j]));
            et = max(et, (unsigned)__shfl_xor((int)et, 16));
            et = max(et, (unsigned)__shfl_xor((int)et, 32));
            const float s = t8_pow2(267 - (int)et);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                t8_u4 h, l;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned hw, lw;
                    split_f16_prod(wv[b][t][2 * j], s, wv[b][t][2 * j + 1], s, hw, lw);
                    h[j] = hw, l[j] = lw;
                }
                wh[b][t] = __builtin_bit_cast(t8_h8, h), wl[b][t] = __builtin_bit_cast(t8_h8, l);
            }
            we[b] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) we[b] |= (unsigned)__shfl((int)et, 4 * q4 + i) << (8 * i);
        }
    }
    t8_f4 bsum = {0.f, 0.f, 0.f, 0.f};
    int ce = 28, tce[TB];                                                     // bounds on the products' exponents: of the lane's block of 32 columns, of the wave's dW
#pragma unroll
    for (int j = 0; j < TB; ++j) tce[j] = 28;
    // ---- the exponents of this lane's rows of dz and, the last one, of the row that its codes belong to.  0: a row of zeros (what is not finite does not
    // count); 14 at least otherwise, so that 2^(141 - e) is a number
    auto measure = [&](int (&e)[NLD + 1]) {
        // a magnitude's bits with the exponent one up in the top byte: what is not finite wraps to under the zero's 2^24
        unsigned m[NLD];
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            m[i] = 0u;
#pragma unroll
            for (int c = 0; c < 4; ++c) m[i] = max(m[i], (__float_as_uint(dv[i][c]) << 1) + (1u << 24));
        }
        const unsigned t = t8_row_max<NLD, LPR>(m, lane), x = t <= 1u << 24 ? 0u : max((t >> 24) - 1u, 14u);
        e[0] = (int)t8_dpp<0x00>(x), e[1] = (int)t8_dpp<0x55>(x);             // quad_perm 0 0 0 0, 1 1 1 1
        if (NLD == 4) e[NLD - 2] = (int)t8_dpp<0xAA>(x), e[NLD - 1] = (int)t8_dpp<0xFF>(x);
        const int p = lane / CPR % NLD;
        e[NLD] = p & 1 ? e[1] : e[0];
        if (NLD == 4) e[NLD] = p & 2 ? (p & 1 ? e[NLD - 1] : e[NLD - 2]) : e[NLD];
    };
    // ---- this lane's part of the step in its two images: of dz ..
    auto stage_z = [&](Step& B, const int (&e)[NLD + 1]) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const float G = FULL && zc >= a.N ? 0.f : __uint_as_float((unsigned)(268 - e[i]) << 23);         // 2^(141 - e); of zeros: some number
            t8_u2 h, l;
            unsigned hw, lw;
            split_f16_prod(dv[i][0], G, dv[i][1], G, hw, lw);
            h[0] = hw, l[0] = lw;
            split_f16_prod(dv[i][2], G, dv[i][3], G, hw, lw);
            h[1] = hw, l[1] = lw;
            *reinterpret_cast<t8_u2*>(&B.z[0][zr + i][zc]) = h;
            *reinterpret_cast<t8_u2*>(&B.z[1][zr + i][zc]) = l;
        }
        if (cc == 0) B.e[cr] = e[NLD];
    };
    // ---- .. and of x, under the bounds (ec: the exponent of its row of dz; of Swish: the values and derivatives)
    typedef t8_f4 Vals[ACT == ACT_SWISH ? CW : 1];
    auto stage_x = [&](Step& B, int ec, const Vals& y, const Vals& dy) {
        unsigned p[XPL][2 * CW];
        if (ACT == ACT_SWISH) {
            const float up = ec ? t8_pow2(268 + ec - ce) : 0.f;               // (a row without a gradient: nothing of it counts)
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                split_f16_prod(y[j][0], up, y[j][1], up, p[0][2 * j], p[XPL - 1][2 * j]);
                split_f16_prod(y[j][2], up, y[j][3], up, p[0][2 * j + 1], p[XPL - 1][2 * j + 1]);
                *reinterpret_cast<t8_f4*>(&B.d[cr][cc + 4 * j]) = dy[j];
            }
        } else {
            // byte c beside 0x64 is the fp16 number 1024 + c (signed: c + 128 after the sign bit is turned): times the power of two, less what it
            // is too much - one fused multiply-add for two codes, exact down to 2^-24
            const bool bad = bv == 255u;
            const int k = min((int)bv + ec - ce, 0) + 5;
            const _Float16 s = bad ? __builtin_bit_cast(_Float16, (unsigned short)0x7E00) : (_Float16)t8_pow2(k + 127);
            const _Float16 o = (KIND == T8_RELU ? (_Float16)-1024.0f : (_Float16)-1152.0f) * s;
            const t8_hp s2 = {s, s}, o2 = {o, o};
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const unsigned w = KIND == T8_RELU ? cv[j] : cv[j] ^ 0x80808080u;
                p[0][2 * j] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(t8_hp, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)), s2, o2));
                p[0][2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(t8_hp, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)), s2, o2));
            }
            // codes of smaller powers of two end among fp16's smallest numbers: each is rounded there by itself
            if (__any(k < -24 && k >= -33 && !bad)) {
                const float f = bad ? __uint_as_float(0x7FC00000u) : t8_pow2(k + 127);
#pragma unroll
                for (int j = 0; j < CW; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        p[0][2 * j + i] = __builtin_bit_cast(unsigned, t8_hp{(_Float16)(t8_q<KIND>(cv[j], 2 * i) * f), (_Float16)(t8_q<KIND>(cv[j], 2 * i + 1) * f)});
            }
        }
#pragma unroll
        for (int q = 0; q < XPL; ++q)
#pragma unroll
            for (int j = 0; j < CPT / 8; ++j)
                *reinterpret_cast<t8_u4*>(&B.x[q][cr][cc + 8 * j]) = t8_u4{p[q][4 * j], p[q][4 * j + 1], p[q][4 * j + 2], p[q][4 * j + 3]};
        if (ACT == ACT_RELU) *reinterpret_cast<t8_cw*>(&B.c[cr][cc / 4]) = cv;
    };
    float* const wout = a.wpart + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * NP * KP;
    bool first = true;
    int it = 0;
    while (step < nsteps) {              // one stretch of steps under the same bounds
        f32x4 accs[NBN][KB];                                                  // the stretch's sums: T8_FOLD steps at a time
#pragma unroll
        for (int b = 0; b < NBN; ++b)
#pragma unroll
            for (int x = 0; x < KB; ++x) accs[b][x] = f32x4{0.f, 0.f, 0.f, 0.f};
        bool fresh = true, same = true;
        while (same && step < nsteps) {
            f32x4 accw[NBN][KB];
#pragma unroll
            for (int b = 0; b < NBN; ++b)
#pragma unroll
                for (int x = 0; x < KB; ++x) accw[b][x] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < T8_FOLD && step < nsteps; ++k, step += gridDim.x, ++it, fresh = false) {
                Step& B = sb[it & 1];
                if (FULL) {
                    shift = (int)(step * R - min(step * R, a.M - R));
                    if (shift) {                                              // (the last step: rows that were done already count as zeros)
#pragma unroll
                        for (int i = 0; i < NLD; ++i)
                            if (zr + i < shift) dv[i] = t8_f4{0.f, 0.f, 0.f, 0.f};
                    }
                }
                int e[NLD + 1];
                Vals y, dy;
                measure(e);
                stage_z(B, e);
                // the exponent of the largest product of this lane's row of dz and its part of x (the values' own, or the tape's byte); 0: none
                int c = bv == 0u || bv == 255u ? 0 : (int)bv;
                if (ACT == ACT_SWISH) {
                    unsigned top = 0u;
#pragma unroll
                    for (int j = 0; j < CW; ++j) {
                        const t8_f4 v = t8_decode4<KIND>(cv[j], bv);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float d;
                            y[j][i] = t8_swish(v[i], d);
                            dy[j][i] = d;
                            top = max(top, __float_as_uint(y[j][i]) & 0x7FFFFFFFu);
                        }
                    }
                    c = top == 0u || top >= 0x7F800000u ? 0 : max((int)(top >> 23), 14);
                }
                c = c == 0 || e[NLD] == 0 ? 0 : c + e[NLD];
                // a stretch's first step is what its bounds are made of
                if (fresh) {
                    int t = c;
#pragma unroll
                    for (int o = 1; o < 64; o = 2 * o == LB ? CPR : 2 * o) t = max(t, __shfl_xor(t, o));    // (the lanes of a block of columns)
                    if (lane < CPR && !(lane % LB)) red[wave][lane / LB] = (unsigned)t;
                    wg_barrier();
                    auto bound = [&](int block, int now) {
                        int u = 0;
#pragma unroll
                        for (int w = 0; w < NW; ++w) u = max(u, (int)red[w][block]);
                        return u > now ? u + T8_ROOM(ACT) : now;
                    };
                    ce = bound(cc / 32, ce);
#pragma unroll
                    for (int j = 0; j < TB; ++j) tce[j] = __builtin_amdgcn_readfirstlane(bound(xf / 32 + j, tce[j]));
                    if (tid < 2) flag[tid] = 0u;                              // (everybody has read the flag that ended the last stretch)
                }
                stage_x(B, e[NLD], y, dy);
                if (!fresh && __any(c > ce) && lane == 0) flag[it & 1] = 1u;
                wg_barrier();
                if (!fresh && __builtin_amdgcn_readfirstlane((int)flag[it & 1])) {          // (the same for every wave)
                    same = false;
                    break;
                }
#pragma unroll
                for (int i = 0; i < NLD; ++i) bsum += dv[i];
                const long row0 = FULL ? min(step * R, a.M - R) : step * R;
                const int done = shift;
                asm volatile("" ::: "memory");
                load(min(step + (long)gridDim.x, nsteps - 1));                        // (past the last step: rows that nobody uses)
                asm volatile("" ::: "memory");
                // ---- dx^T: acc[b][rb] = features kf + 16 b .. of rows wr + 16 (rp + rb) ..
#pragma unroll
                for (int rp = 0; rp < RBS; rp += RB) {
                    f32x4 acc[NBK][RB];
#pragma unroll
                    for (int b = 0; b < NBK; ++b)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) acc[b][rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            const t8_h8 zh = *reinterpret_cast<const t8_h8*>(&B.z[0][wr + 16 * (rp + rb) + n16][32 * t + 8 * q4]);
                            const t8_h8 zl = *reinterpret_cast<const t8_h8*>(&B.z[1][wr + 16 * (rp + rb) + n16][32 * t + 8 * q4]);
#pragma unroll
                            for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl[b][t], zh, acc[b][rb], 0, 0, 0);
#pragma unroll
                            for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[b][t], zl, acc[b][rb], 0, 0, 0);
#pragma unroll
                            for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[b][t], zh, acc[b][rb], 0, 0, 0);
                        }
                    __builtin_amdgcn_sched_barrier(0);                                // (without these the reads of all parts move up and the registers run out)
                    // dx = act'(v) (dz W): lane = row n16 of the block of rows, features 4 q4 .. + 3 of the block of features
                    if (a.dx) {
                        float* const bx = a.dx + (row0 + wr + 16 * rp) * a.lddx + k0 + kf;
                        const unsigned ox = ((unsigned)n16 * (unsigned)a.lddx + 4 * q4) * 4u;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            const int lr = wr + 16 * (rp + rb) + n16;                 // row of the step
                            const int e = B.e[lr] - 281;
#pragma unroll
                            for (int b = 0; b < NBK; ++b) {
                                const int f = kf + 16 * b + 4 * q4, k = k0 + f;
                                t8_f4 v;
                                unsigned wb = we[b];
                                asm volatile("" : "+v"(wb));                          // (or the four bytes are kept apart in registers across the loop)
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_ldexpf(acc[b][rb][i], e + (int)(wb >> (8 * i) & 0xFFu));
                                if (ACT == ACT_RELU) {
                                    const unsigned w = B.c[lr][f / 4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i) v[i] = (w >> (8 * i)) & 0xFFu ? v[i] : 0.f;
                                }
                                if (ACT == ACT_SWISH) v *= *reinterpret_cast<const t8_f4*>(&B.d[lr][f]);
                                if (FULL) {
                                    float* o = bx + 16 * rb * a.lddx + 16 * b;
                                    T8_UNIFORM(o);
                                    if (lr >= done && k < a.K) t8_put<t8_v4<float>>(o, ox, v);
                                } else if (row0 + lr < a.M) {
                                    float* o = a.dx + (row0 + lr) * a.lddx + k;
                                    if (a.add_dx) v += t8_load4(o, a.K - k);
                                    t8_store4(o, a.K - k, v);
                                }
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                // ---- dW += dz^T x, 32 rows at a time (k group q4: rows 4 q4 .. + 3 and 16 + 4 q4 .. + 3 of both operands)
#pragma unroll
                for (int r32 = 0; r32 < R; r32 += 32) {
                    const int r0 = r32 + 4 * q4 + (n16 >> 2), c0 = 4 * (n16 & 3);
                    t8_h8 ah[NBN], al[NBN];
#pragma unroll
                    for (int b = 0; b < NBN; ++b) {
                        const int f = nf + 16 * b + c0;
                        ah[b] = t8_join(t8_tr(&B.z[0][r0][f]), t8_tr(&B.z[0][16 + r0][f]));
                        al[b] = t8_join(t8_tr(&B.z[1][r0][f]), t8_tr(&B.z[1][16 + r0][f]));
                    }
#pragma unroll
                    for (int x = 0; x < KB; ++x) {
                        const int f = xf + 16 * x + c0;
                        const t8_h8 xh = t8_join(t8_tr(&B.x[0][r0][f]), t8_tr(&B.x[0][16 + r0][f]));
                        if (XPL == 2) {
                            const t8_h8 xl = t8_join(t8_tr(&B.x[XPL - 1][r0][f]), t8_tr(&B.x[XPL - 1][16 + r0][f]));
#pragma unroll
                            for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[b], xl, accw[b][x], 0, 0, 0);
                        }
#pragma unroll
                        for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[b], xh, accw[b][x], 0, 0, 0);
#pragma unroll
                        for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[b], xh, accw[b][x], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NBN; ++b)
#pragma unroll
                for (int x = 0; x < KB; ++x) accs[b][x] += accw[b][x];
        }
        // ---- the stretch's part of the workgroup's sums: C/D row 4 q4 + i = feature of dz, column n16 = feature of x
        // (the base hidden: 32 addresses would be kept in registers across the loop)
        auto sums = [&](bool add) {
            const unsigned ol = ((unsigned)(4 * q4) * KP + n16) * 4u;
#pragma unroll
            for (int b = 0; b < NBN; ++b)
#pragma unroll
                for (int x = 0; x < KB; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* o = wout + (nf + 16 * b + i) * KP + xf + 16 * x;
                        T8_UNIFORM(o);
                        const float v = __builtin_amdgcn_ldexpf(accs[b][x][i], tce[x / 2] - (ACT == ACT_SWISH ? 282 : 273));
                        t8_put<float>(o, ol, add ? t8_at<float>(o, ol) + v : v);
                    }
        };
        if (first) sums(false);
        else sums(true);
        first = false;
    }
    if (a.kb0 + blockIdx.y == 0) {                                            // the lanes that hold the same columns of dz, in order
        float* s = reinterpret_cast<float*>(&sb[0]);
        wg_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) s[tid / LPR * NP + zc + i] = bsum[i];
        wg_barrier();
        if (tid < NP) {
            float t = 0.f;
            for (int r = 0; r < LANES / LPR; ++r) t += s[r * NP + tid];
            a.bpart[(size_t)blockIdx.x * NP + tid] = t;
        }
    }
}

// dW[n][k] (+)= sum over the workgroups of their partial sums, in order: a workgroup takes 64 neighbouring sums, its sixteen waves a run of the
// partials each (short chains: the reads' latency is what this kernel takes, and the sums' rounding grows with their length).  blockIdx.y = block of K of
// the launch, which begins at block kb0; one more, in the first launch: db
__global__ void __launch_bounds__(1024) k_tape8_linear_sum(const float* __restrict__ wpart, const float* __restrict__ bpart, int nwg, int NP, int KP, int N, int K,
                                                          int kb0, int kbn, float* __restrict__ dW, long lddw, float* __restrict__ db, int add) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool bias = blockIdx.y == kbn;
    const int o = blockIdx.x * 64 + lane, n_out = bias ? NP : NP * KP;
    if (blockIdx.x * 64 >= n_out) return;
    const float* p = bias ? bpart : wpart + (size_t)blockIdx.y * nwg * NP * KP;
    float t = 0.f;
    const int per = (nwg + 15) / 16, w1 = min(nwg, (wave + 1) * per);
#pragma unroll 8
    for (int w = wave * per; w < w1; ++w) t += p[(size_t)w * n_out + o];
    s[wave][lane] = t;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) t += s[w][lane];
    const int n = bias ? o : o / KP, k = bias ? 0 : (kb0 + blockIdx.y) * KP + o % KP;
    if (n >= N || k >= K) return;
    float* d = bias ? db + n : dW + n * lddw + k;
    if (bias && !db) return;
    *d = add ? *d + t : t;
}

__global__ void __launch_bounds__(256) k_tape8_fill0(float* __restrict__ p, long ld, int rows, int cols) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)rows * cols; i += (long)gridDim.x * 256) p[(i / cols) * ld + i % cols] = 0.f;
}
static unsigned t8_fill_grid(long n) { return (unsigned)(n < (1l << 28) ? (n + 255) / 256 : 1l << 20); }

#define T8_BLOCK 128
static int t8_pad(int n) { return n <= 64 ? 64 : 128; }                       // a block of at most 128 features, as 64 or 128
#define T8_KBLOCKS 32                         // blocks of K of a launch: the partial sums of more would take memory without end (200 000 columns: 13 GB)
// one workgroup a CU of eight waves, two (three) of four; fewer where K has several blocks
static int t8_lin_grid(long M, int np, int kp, int kblocks, int act) {
    const int R = T8_ROWS(np, kp, act);
    const long steps = (M + R - 1) / R, most = (np == 128 && kp == 128 ? 256 : 512) / (kblocks < 4 ? kblocks : 4);
    return (int)(steps < most ? steps : most);
}

extern "C" int magnet_tape8_linear_bwd_workspace(long M, long N, long K, long* floats) {
    if (M < 0 || N < 1 || K < 1 || N > T8_WIDEST || K > T8_WIDEST) return -2;
    const int kp = t8_pad((int)K), kb = (int)((K + kp - 1) / kp), np = t8_pad((int)N), kbn = kb < T8_KBLOCKS ? kb : T8_KBLOCKS;
    *floats = (long)t8_lin_grid(M, np, kp, kb, ACT_SWISH) * ((long)np * kp * kbn + np);     // (most workgroups: steps of 32 rows)
    return 0;
}

template <int NP, int KP, bool FULL>
static void t8_lin_launch(const T8LinArgs& a, int act, dim3 grid, hipStream_t st) {
    if (act == ACT_RELU) k_tape8_linear_bwd<NP, KP, ACT_RELU, FULL><<<grid, T8_WAVES(NP, KP) * 64, 0, st>>>(a);
    else if (act == ACT_SWISH) k_tape8_linear_bwd<NP, KP, ACT_SWISH, FULL><<<grid, T8_WAVES(NP, KP) * 64, 0, st>>>(a);
    else k_tape8_linear_bwd<NP, KP, ACT_NONE, FULL><<<grid, T8_WAVES(NP, KP) * 64, 0, st>>>(a);
}
template <bool FULL>
static void t8_lin_shape(const T8LinArgs& a, int np, int kp, int act, dim3 grid, hipStream_t st) {
    if (np == 128 && kp == 128) t8_lin_launch<128, 128, FULL>(a, act, grid, st);
    else if (np == 128) t8_lin_launch<128, 64, FULL>(a, act, grid, st);
    else if (kp == 128) t8_lin_launch<64, 128, FULL>(a, act, grid, st);
    else t8_lin_launch<64, 64, FULL>(a, act, grid, st);
}

extern "C" int magnet_tape8_linear_bwd_f32(const float* dz, long ldz, const void* codes, const void* bytes, const float* w, long ldw, long M, int N, int K,
                                           int act, float* dx, long lddx, float* dW, long lddw, float* db, int accumulate, float* workspace,
                                           void* stream) {
    if (M < 0 || N < 1 || K < 1 || ldz < N || ldw < K || lddw < K || (dx && lddx < K) || act < 0 || act > 2 || !dW || ((uintptr_t)codes & 15) || N > T8_WIDEST || K > T8_WIDEST)
        return -2;
    hipStream_t st = (hipStream_t)stream;
    if (M == 0) {
        if (!accumulate) {
            k_tape8_fill0<<<t8_fill_grid((long)N * K), 256, 0, st>>>(dW, lddw, N, K);
            if (db) k_tape8_fill0<<<t8_fill_grid(N), 256, 0, st>>>(db, N, 1, N);
        }
        return (int)hipGetLastError();
    }
    const int kp = t8_pad(K), kb = (K + kp - 1) / kp;
    const int np = t8_pad(N), wgs = t8_lin_grid(M, np, kp, kb, act);
    for (int n0 = 0; n0 < N; n0 += T8_BLOCK) {
        const int n = N - n0 < T8_BLOCK ? N - n0 : T8_BLOCK;
        T8LinArgs a;
        a.dz = dz + n0, a.codes = (const unsigned char*)codes, a.bytes = (const unsigned char*)bytes, a.w = w + n0 * ldw, a.dx = dx;
        a.wpart = workspace, a.bpart = workspace + (size_t)wgs * np * kp * (kb < T8_KBLOCKS ? kb : T8_KBLOCKS);
        a.M = M, a.ldz = ldz, a.ldw = ldw, a.lddx = lddx, a.N = n, a.K = K, a.ldc = (K + 31) / 32 * 32;
        a.exact = n == np && !(K % kp);
        a.add_dx = n0 > 0;
        // (32-bit byte offsets inside a lane's part of a step)
        const bool full = M >= 64 && N <= T8_BLOCK && !(n & 3) && !(K & 3) && ldz < (1l << 24) && lddx < (1l << 24) && ldw < (1l << 24);
        for (a.kb0 = 0; a.kb0 < kb; a.kb0 += T8_KBLOCKS) {
            const int kbn = kb - a.kb0 < T8_KBLOCKS ? kb - a.kb0 : T8_KBLOCKS;
            const dim3 grid(wgs, kbn);
            if (full) t8_lin_shape<true>(a, np, kp, act, grid, st);
            else t8_lin_shape<false>(a, np, kp, act, grid, st);
            k_tape8_linear_sum<<<dim3((np * kp + 63) / 64, kbn + (a.kb0 == 0)), 1024, 0, st>>>(a.wpart, a.bpart, wgs, np, kp, n, K, a.kb0, kbn, dW + n0 * lddw, lddw,
                                                                                            db ? db + n0 : nullptr, accumulate);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return (int)e;
        }
    }
    return 0;
}
