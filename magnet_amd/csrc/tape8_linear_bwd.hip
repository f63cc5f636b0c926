// One Linear walked back from an 8-bit tape of its input (tape8.cuh), in one pass over the rows:
//     x  = act(v)   v = the tape's value: the activated input itself (none, relu) or Swish's argument (swish)
//     dx [M][K] = act'(v) (dz W)        dW [N][K] (+)= dz^T x        db [N] (+)= column sums of dz
// What has to move is dz in, dx out and 33/32 bytes a value of the tape: 1156 bytes a row at N = K = 128, where fp32 activations make it
// 1536 (linear_bwd.hip).
//
// A workgroup of four waves takes steps of 32 rows of one block of at most 128 x 128 of W.  dz is split once into two fp16 planes
// (h + l, 22 bits), the tape's codes need one plane - a code has 8 bits, fp16 holds code times a power of two exactly - (two behind
// Swish), and both meet as 16 x 16 x 32 matrix products through LDS:
//   dx^T = W^T dz^T   A = the wave's features of W^T, two planes kept in registers; B = rows of the dz image; products hh + hl + lh
//   dW   = dz^T x     A, B = transposed LDS reads of the two images, k = the step's 32 rows; products (h + l) x
// The error of both is a few 2^-22 of the operands' magnitude, sums are held in fp32, and the workgroups' partial sums of dW and db are added
// in their order by a second kernel: the same bits every time.
//
// Scales.  fp16 spans 2^40; gradients (1e-7) and tapes (any byte) do not fit by themselves.  The workgroup keeps the largest exponent it
// has met, of dz and of the tape's bytes, and stages everything times the power of two that puts it at the top of the range; a step that
// brings a larger one scales the sums down first.  Rows 2^-30 below the largest so far start to lose bits, of a share that small of the sums.
// A wave scales its own part of W likewise.
#include "common.cuh"
#include "split_single.cuh"
#include "tape8.cuh"

typedef _Float16 t8_h8 __attribute__((ext_vector_type(8)));
typedef __fp16 t8_h2 __attribute__((ext_vector_type(2)));
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
    int N, K, ldc, zvec, xvec, add_dx;   // zvec / xvec: dz / dx in 16-byte accesses; add_dx: dx += (a later block of N)
};

// exponent byte (1 .. 254) of a magnitude's bits; 0 for zero, subnormals and what is not finite
__device__ __forceinline__ unsigned t8_expo(unsigned m) {
    const unsigned e = m >> 23;
    return e == 255u ? 0u : e;
}
__device__ __forceinline__ float t8_pow2(int biased) { return __uint_as_float((unsigned)min(max(biased, 0), 254) << 23); }
// two values as one word of each fp16 plane: h towards zero, l = what is left, to nearest
__device__ __forceinline__ void t8_split(float a, float b, unsigned& h, unsigned& l) {
    const t8_h2 hh = __builtin_amdgcn_cvt_pkrtz(a, b);
    const _Float16 la = (_Float16)(a - (float)hh[0]), lb = (_Float16)(b - (float)hh[1]);
    h = __builtin_bit_cast(unsigned, hh);
    l = (unsigned)__builtin_bit_cast(unsigned short, la) | (unsigned)__builtin_bit_cast(unsigned short, lb) << 16;
}
// four halfwords of a column out of a 16 x 4 tile: lane i of 16 points at row i / 4, columns 4 (i % 4) .., and gets column i
__device__ __forceinline__ t8_u2 t8_tr(const unsigned short* p) {
    return __builtin_bit_cast(t8_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) t8_s4*)(p)));
}
__device__ __forceinline__ t8_h8 t8_join(t8_u2 a, t8_u2 b) { return __builtin_bit_cast(t8_h8, t8_u4{a[0], a[1], b[0], b[1]}); }
// Swish and its derivative: s = sigmoid(v); v s and s (1 + v (1 - s))
__device__ __forceinline__ float t8_sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }
__device__ __forceinline__ float t8_dswish(float v) {
    const float s = t8_sigmoid(v);
    return s + v * s * t8_sigmoid(-v);   // (1 - s as a sigmoid: no cancellation where s is near 1)
}

template <int NP, int KP, int ACT>
__global__ void __launch_bounds__(256, 2) k_tape8_linear_bwd(const T8LinArgs a) {
    constexpr int KIND = ACT == ACT_RELU ? T8_RELU : T8_SIGNED;
    constexpr int XPL = ACT == ACT_SWISH ? 2 : 1;                             // planes of x
    constexpr int NST = NP + 16, KST = KP + 16, CST = KP / 4 + 4;             // row strides: halfwords, halfwords, words (bank spread)
    constexpr int LPR = NP / 4, NLD = 32 * LPR / 256;                         // lanes per row of dz, rows of dz per lane
    constexpr int CPR = KP / 16;                                              // lanes per row of codes (16 codes each)
    constexpr int NBK = KP / 64, NBN = NP / 64, NT = NP / 32, KB = KP / 16;   // a wave's blocks of 16 features of x / of dz
    __shared__ __attribute__((aligned(16))) unsigned short zi[2][32][NST];
    __shared__ __attribute__((aligned(16))) unsigned short xi[XPL][32][KST];
    __shared__ __attribute__((aligned(16))) unsigned ci[32][CST];
    __shared__ unsigned char bi[32][KP / 32];
    __shared__ unsigned red[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, q4 = lane >> 4;
    const int k0 = blockIdx.y * KP;
    // ---- the wave's features of W^T: A operands (lane = feature of x, register j of k group q4 = feature 32 t + 8 q4 + j of dz)
    t8_h8 wh[NBK][NT], wl[NBK][NT];
    float wscale;
    {
        float wv[NBK][NT][8];
        unsigned top = 0;
#pragma unroll
        for (int b = 0; b < NBK; ++b)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int n = 32 * t + 8 * q4 + j, k = k0 + 16 * (NBK * wave + b) + n16;
                    const float v = n < a.N && k < a.K ? a.w[n * a.ldw + k] : 0.f;
                    wv[b][t][j] = v;
                    top = max(top, t8_expo(__float_as_uint(v) & 0x7FFFFFFFu));
                }
#pragma unroll
        for (int o = 32; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
        const int e = max((int)top, 14);
        const float s = t8_pow2(267 - e);                                     // max |W| -> [2^13, 2^14)
        wscale = t8_pow2(e - 13);
#pragma unroll
        for (int b = 0; b < NBK; ++b)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                t8_u4 h, l;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned hw, lw;
                    t8_split(wv[b][t][2 * j] * s, wv[b][t][2 * j + 1] * s, hw, lw);
                    h[j] = hw, l[j] = lw;
                }
                wh[b][t] = __builtin_bit_cast(t8_h8, h), wl[b][t] = __builtin_bit_cast(t8_h8, l);
            }
    }
    // ---- what this lane loads of a step
    const int zr = tid / LPR, zc = 4 * (tid % LPR);
    const int cr = tid / CPR, cc = 16 * (tid % CPR);
    const bool c_on = cr < 32 && k0 + cc < a.ldc;
    const int lb = a.ldc / 32;
    t8_f4 dv[NLD];
    t8_u4 cv = {0u, 0u, 0u, 0u};
    unsigned bv = 0;
    auto load = [&](long step) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const long r = step * 32 + zr + i * (256 / LPR);
            dv[i] = r < a.M ? t8_load4(a.dz + r * a.ldz + zc, a.zvec && zc < a.N, a.N - zc) : t8_f4{0.f, 0.f, 0.f, 0.f};
        }
        const long r = step * 32 + cr;
        const bool on = c_on && r < a.M;
        cv = on ? *reinterpret_cast<const t8_u4*>(a.codes + r * a.ldc + k0 + cc) : t8_u4{0u, 0u, 0u, 0u};
        bv = on ? a.bytes[r * lb + (k0 + cc) / 32] : 0u;
    };
    f32x4 accw[NBN][KB];
#pragma unroll
    for (int b = 0; b < NBN; ++b)
#pragma unroll
        for (int x = 0; x < KB; ++x) accw[b][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    t8_f4 bsum = {0.f, 0.f, 0.f, 0.f};
    int ze = 14, xe = 8;                                                      // largest exponents so far: of dz, and the largest byte
    const long nsteps = (a.M + 31) / 32;
    long step = blockIdx.x;
    if (step < nsteps) load(step);
    for (; step < nsteps; step += gridDim.x) {
        // ---- the step's exponents
        {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < NLD; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) m = max(m, t8_expo(__float_as_uint(dv[i][c]) & 0x7FFFFFFFu));
            unsigned mx = bv == 255u ? 0u : bv;
#pragma unroll
            for (int o = 32; o; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o)), mx = max(mx, (unsigned)__shfl_xor((int)mx, o));
            if (lane == 0) red[wave] = m | mx << 8;
        }
        wg_barrier();                                                         // the exponents are there; the images have been read
        {
            unsigned m = 0, mx = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) m = max(m, red[w] & 0xFFu), mx = max(mx, red[w] >> 8);
            const int nz = max(ze, (int)m), nx = max(xe, (int)mx);
            if (nz > ze || nx > xe) {                                         // (the same in every lane of the workgroup)
                const float f = t8_pow2(127 + ze - nz) * t8_pow2(127 + xe - nx);
#pragma unroll
                for (int b = 0; b < NBN; ++b)
#pragma unroll
                    for (int x = 0; x < KB; ++x) accw[b][x] *= f;
                ze = nz, xe = nx;
            }
        }
        const float G = t8_pow2(267 - ze);                                    // largest |dz| -> [2^13, 2^14)
        // ---- the images
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            t8_u2 h, l;
            unsigned hw, lw;
            bsum += dv[i];
            t8_split(dv[i][0] * G, dv[i][1] * G, hw, lw);
            h[0] = hw, l[0] = lw;
            t8_split(dv[i][2] * G, dv[i][3] * G, hw, lw);
            h[1] = hw, l[1] = lw;
            *reinterpret_cast<t8_u2*>(&zi[0][zr + i * (256 / LPR)][zc]) = h;
            *reinterpret_cast<t8_u2*>(&zi[1][zr + i * (256 / LPR)][zc]) = l;
        }
        if (cr < 32) {
            // code * 2^(byte - xe + 7): at most 255 * 2^7; Swish of the value times the same power of two
            const float xs = bv == 255u ? t8_step(255u) : ACT == ACT_SWISH ? t8_step(bv) : t8_pow2(bv == 0u ? 0 : (int)bv - xe + 134);
            const float up = t8_pow2(261 - xe);
            unsigned p[XPL][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const unsigned w = cv[j >> 1];
                float v0 = t8_q<KIND>(w, 2 * (j & 1)) * xs, v1 = t8_q<KIND>(w, 2 * (j & 1) + 1) * xs;
                if (ACT == ACT_SWISH) {
                    v0 = v0 * t8_sigmoid(v0) * up, v1 = v1 * t8_sigmoid(v1) * up;
                    t8_split(v0, v1, p[0][j], p[XPL - 1][j]);
                } else {
                    p[0][j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(v0, v1));
                }
            }
#pragma unroll
            for (int q = 0; q < XPL; ++q) {
                *reinterpret_cast<t8_u4*>(&xi[q][cr][cc]) = t8_u4{p[q][0], p[q][1], p[q][2], p[q][3]};
                *reinterpret_cast<t8_u4*>(&xi[q][cr][cc + 8]) = t8_u4{p[q][4], p[q][5], p[q][6], p[q][7]};
            }
            if (ACT != ACT_NONE) *reinterpret_cast<t8_u4*>(&ci[cr][cc / 4]) = cv;
            if (ACT == ACT_SWISH && !(cc & 16)) bi[cr][cc / 32] = (unsigned char)bv;
        }
        const long row0 = step * 32;
        asm volatile("" ::: "memory");
        if (step + gridDim.x < nsteps) load(step + gridDim.x);
        asm volatile("" ::: "memory");
        wg_barrier();
        // ---- dx^T: acc[b][rb] = features 16 (NBK wave + b) .. of rows 16 rb ..
        f32x4 acc[NBK][2];
#pragma unroll
        for (int b = 0; b < NBK; ++b) acc[b][0] = acc[b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                const t8_h8 zh = *reinterpret_cast<const t8_h8*>(&zi[0][16 * rb + n16][32 * t + 8 * q4]);
                const t8_h8 zl = *reinterpret_cast<const t8_h8*>(&zi[1][16 * rb + n16][32 * t + 8 * q4]);
#pragma unroll
                for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl[b][t], zh, acc[b][rb], 0, 0, 0);
#pragma unroll
                for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[b][t], zl, acc[b][rb], 0, 0, 0);
#pragma unroll
                for (int b = 0; b < NBK; ++b) acc[b][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[b][t], zh, acc[b][rb], 0, 0, 0);
            }
        // ---- dW += dz^T x over the step's rows (k group q4: rows 4 q4 .. + 3 and 16 + 4 q4 .. + 3 of both operands)
        {
            const int r0 = 4 * q4 + (n16 >> 2), c0 = 4 * (n16 & 3);
            t8_h8 ah[NBN], al[NBN];
#pragma unroll
            for (int b = 0; b < NBN; ++b) {
                const int f = 16 * (NBN * wave + b) + c0;
                ah[b] = t8_join(t8_tr(&zi[0][r0][f]), t8_tr(&zi[0][16 + r0][f]));
                al[b] = t8_join(t8_tr(&zi[1][r0][f]), t8_tr(&zi[1][16 + r0][f]));
            }
#pragma unroll
            for (int x = 0; x < KB; ++x) {
                const t8_h8 xh = t8_join(t8_tr(&xi[0][r0][16 * x + c0]), t8_tr(&xi[0][16 + r0][16 * x + c0]));
                if (XPL == 2) {
                    const t8_h8 xl = t8_join(t8_tr(&xi[XPL - 1][r0][16 * x + c0]), t8_tr(&xi[XPL - 1][16 + r0][16 * x + c0]));
#pragma unroll
                    for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[b], xl, accw[b][x], 0, 0, 0);
                }
#pragma unroll
                for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[b], xh, accw[b][x], 0, 0, 0);
#pragma unroll
                for (int b = 0; b < NBN; ++b) accw[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[b], xh, accw[b][x], 0, 0, 0);
            }
        }
        // ---- dx = act'(v) (dz W): lane = row 16 rb + n16, features 4 q4 .. + 3 of the block
        if (a.dx) {
            const float invG = t8_pow2(ze - 13);
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                const long r = row0 + 16 * rb + n16;
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const int f = 16 * (NBK * wave + b) + 4 * q4, k = k0 + f;
                    t8_f4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = acc[b][rb][i] * wscale * invG;
                    if (ACT == ACT_RELU) {
                        const unsigned w = ci[16 * rb + n16][f / 4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (w >> (8 * i)) & 0xFFu ? v[i] : 0.f;
                    }
                    if (ACT == ACT_SWISH) {
                        const t8_f4 x = t8_decode4<KIND>(ci[16 * rb + n16][f / 4], bi[16 * rb + n16][f / 32]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] *= t8_dswish(x[i]);
                    }
                    if (r < a.M) {
                        float* o = a.dx + r * a.lddx + k;
                        if (a.add_dx) v += t8_load4(o, a.xvec && k < a.K, a.K - k);
                        t8_store4(o, a.xvec && k < a.K, a.K - k, v);
                    }
                }
            }
        }
    }
    // ---- partial sums: C/D row 4 q4 + i = feature of dz, column n16 = feature of x
    float* wout = a.wpart + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * NP * KP;
    const float s0 = t8_pow2(ze - 13), s1 = t8_pow2(xe - 7);
#pragma unroll
    for (int b = 0; b < NBN; ++b)
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                wout[(16 * (NBN * wave + b) + 4 * q4 + i) * KP + 16 * x + n16] = accw[b][x][i] * s0 * s1;
    if (blockIdx.y == 0) {                                                    // the lanes that hold the same columns of dz, in order
        float* s = reinterpret_cast<float*>(&zi[0][0][0]);
        wg_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) s[zr * NP + zc + i] = bsum[i];
        wg_barrier();
        if (tid < NP) {
            float t = 0.f;
            for (int r = 0; r < 256 / LPR; ++r) t += s[r * NP + tid];
            a.bpart[(size_t)blockIdx.x * NP + tid] = t;
        }
    }
}

// dW[n][k] (+)= sum over the workgroups of their partial sums, in order: a workgroup takes 64 neighbouring sums, its four waves a quarter of the
// partials each.  blockIdx.y = block of K; the last one: db
__global__ void __launch_bounds__(256) k_tape8_linear_sum(const float* __restrict__ wpart, const float* __restrict__ bpart, int nwg, int NP, int KP, int N, int K,
                                                          float* __restrict__ dW, long lddw, float* __restrict__ db, int add) {
    __shared__ float s[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool bias = blockIdx.y == gridDim.y - 1;
    const int o = blockIdx.x * 64 + lane, n_out = bias ? NP : NP * KP;
    if (blockIdx.x * 64 >= n_out) return;
    const float* p = bias ? bpart : wpart + (size_t)blockIdx.y * nwg * NP * KP;
    float t = 0.f;
    const int per = (nwg + 3) / 4, w1 = min(nwg, (wave + 1) * per);
#pragma unroll 8
    for (int w = wave * per; w < w1; ++w) t += p[(size_t)w * n_out + o];
    s[wave][lane] = t;
    __syncthreads();
    if (wave) return;
    t = (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]);
    const int n = bias ? o : o / KP, k = bias ? 0 : blockIdx.y * KP + o % KP;
    if (n >= N || k >= K) return;
    float* d = bias ? db + n : dW + n * lddw + k;
    if (bias && !db) return;
    *d = add ? *d + t : t;
}

__global__ void __launch_bounds__(256) k_tape8_fill0(float* __restrict__ p, long ld, int rows, int cols) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < rows * cols) p[(i / cols) * ld + i % cols] = 0.f;
}

#define T8_BLOCK 128
static int t8_pad(int n) { return n <= 64 ? 64 : 128; }                       // a block of at most 128 features, as 64 or 128
static int t8_lin_grid(long M, int kblocks) {
    const long steps = (M + 31) / 32, most = 512 / (kblocks < 4 ? kblocks : 4);
    return (int)(steps < most ? steps : most);
}

extern "C" int magnet_tape8_linear_bwd_workspace(long M, int N, int K, long* floats) {
    if (M < 0 || N < 1 || K < 1) return -2;
    const int kp = t8_pad(K), kb = (K + kp - 1) / kp, np = t8_pad(N);
    *floats = (long)t8_lin_grid(M, kb) * ((long)np * kp * kb + np);
    return 0;
}

template <int NP, int KP>
static void t8_lin_launch(const T8LinArgs& a, int act, dim3 grid, hipStream_t st) {
    if (act == ACT_RELU) k_tape8_linear_bwd<NP, KP, ACT_RELU><<<grid, 256, 0, st>>>(a);
    else if (act == ACT_SWISH) k_tape8_linear_bwd<NP, KP, ACT_SWISH><<<grid, 256, 0, st>>>(a);
    else k_tape8_linear_bwd<NP, KP, ACT_NONE><<<grid, 256, 0, st>>>(a);
}

extern "C" int magnet_tape8_linear_bwd_f32(const float* dz, long ldz, const void* codes, const void* bytes, const float* w, long ldw, long M, int N, int K,
                                           int act, float* dx, long lddx, float* dW, long lddw, float* db, int accumulate, float* workspace,
                                           void* stream) {
    if (M < 0 || N < 1 || K < 1 || ldz < N || ldw < K || lddw < K || (dx && lddx < K) || act < 0 || act > 2 || !dW || ((uintptr_t)codes & 15)) return -2;
    hipStream_t st = (hipStream_t)stream;
    if (M == 0) {
        if (!accumulate) {
            k_tape8_fill0<<<(N * K + 255) / 256, 256, 0, st>>>(dW, lddw, N, K);
            if (db) k_tape8_fill0<<<(N + 255) / 256, 256, 0, st>>>(db, N, 1, N);
        }
        return (int)hipGetLastError();
    }
    const int kp = t8_pad(K), kb = (K + kp - 1) / kp;
    const dim3 grid(t8_lin_grid(M, kb), kb);
    for (int n0 = 0; n0 < N; n0 += T8_BLOCK) {
        const int n = N - n0 < T8_BLOCK ? N - n0 : T8_BLOCK, np = t8_pad(N);
        T8LinArgs a;
        a.dz = dz + n0, a.codes = (const unsigned char*)codes, a.bytes = (const unsigned char*)bytes, a.w = w + n0 * ldw, a.dx = dx;
        a.wpart = workspace, a.bpart = workspace + (size_t)grid.x * np * kp * kb;
        a.M = M, a.ldz = ldz, a.ldw = ldw, a.lddx = lddx, a.N = n, a.K = K, a.ldc = (K + 31) / 32 * 32;
        a.zvec = !(n & 3) && !(ldz & 3) && !((uintptr_t)a.dz & 15);
        a.xvec = !(K & 3) && !(lddx & 3) && !((uintptr_t)dx & 15);
        a.add_dx = n0 > 0;
        if (np == 128 && kp == 128) t8_lin_launch<128, 128>(a, act, grid, st);
        else if (np == 128) t8_lin_launch<128, 64>(a, act, grid, st);
        else if (kp == 128) t8_lin_launch<64, 128>(a, act, grid, st);
        else t8_lin_launch<64, 64>(a, act, grid, st);
        k_tape8_linear_sum<<<dim3((np * kp + 63) / 64, kb + 1), 256, 0, st>>>(a.wpart, a.bpart, grid.x, np, kp, n, K, dW + n0 * lddw, lddw, db ? db + n0 : nullptr, accumulate);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return 0;
}
