// Writing and reading the 8-bit tape (the format: tape8.cuh).
//
// Both kernels are one pass bound by HBM: a pack reads the row (4 / 2 bytes a value) and writes 33/32 bytes a value, an unpack the other
// way.  Packing, a lane takes eight neighbouring columns, four neighbouring lanes one block of 32: the block's top is two lane permutes, the
// codes leave as eight bytes per lane, a wave's stores are whole lines.  Measured at 2 097 152 x 128 fp32: pack 242 us (5.6 TB/s), unpack
// 270 us (5.0 TB/s: three quarters of it written); a large copy reaches 4.9.  A lane walks its positions by adding the grid's stride, split once into
// rows and columns: no division in the loop, and 64-bit row offsets.
#include "common.cuh"
#include "tape8.cuh"

#define T8_CPL 8                         // columns per lane of a pack
struct T8Walk {                          // position (row, group of columns) of a flat index, and the step between two visits
    long row, drow;
    int g, dg, G;
    __device__ __forceinline__ T8Walk(long i, long stride, int groups) {
        G = groups;
        row = i / groups, g = (int)(i - row * groups);
        drow = stride / groups, dg = (int)(stride - drow * groups);
    }
    __device__ __forceinline__ void next() {
        row += drow, g += dg;
        if (g >= G) g -= G, ++row;
    }
};

template <typename T, int KIND>
__global__ void __launch_bounds__(256) k_tape8_pack(const T* __restrict__ x, long ldx, long M, int W, unsigned char* __restrict__ codes,
                                                    unsigned char* __restrict__ bytes) {
    const int blocks = (W + 31) / 32;
    T8Walk at((long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, blocks * (32 / T8_CPL));
    for (; at.row < M; at.next()) {      // (the lanes of a block leave together: groups and the stride are multiples of 4)
        const int c = T8_CPL * at.g;
        t8_f4 v[T8_CPL / 4];
        unsigned top = 0;
#pragma unroll
        for (int h = 0; h < T8_CPL / 4; ++h) {
            const int ch = c + 4 * h;
            v[h] = t8_load4(x + at.row * ldx + ch, W - ch);
            top = max(top, t8_top4<KIND>(v[h]));
        }
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));      // quad_perm 1 0 3 2, 2 3 0 1
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
        const unsigned byte = t8_byte<KIND>(top);
        *reinterpret_cast<t8_u2*>(codes + at.row * (32 * blocks) + c) = t8_u2{t8_code4<KIND>(v[0], byte), t8_code4<KIND>(v[1], byte)};
        if (!(at.g & 3)) bytes[at.row * blocks + (at.g >> 2)] = (unsigned char)byte;
    }
}

// (as many columns per lane as make 16 bytes of the result: what it writes is two or four times what it reads, and a store instruction
// then covers a run of whole lines)
template <typename T, int KIND>
__global__ void __launch_bounds__(256) k_tape8_unpack(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ bytes, long M, int W,
                                                      T* __restrict__ y, long ldy) {
    constexpr int CPL = 16 / sizeof(T), LPB = 32 / CPL;                       // columns per lane, lanes per block
    const int blocks = (W + 31) / 32;
    T8Walk at((long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, blocks * LPB);
    for (; at.row < M; at.next()) {
        const int c = CPL * at.g;
        const unsigned char* p = codes + at.row * (32 * blocks) + c;
        const unsigned byte = bytes[at.row * blocks + at.g / LPB];
        T* o = y + at.row * ldy + c;
        if (CPL == 4) {
            t8_store4(o, W - c, t8_decode4<KIND>(*reinterpret_cast<const unsigned*>(p), byte));
        } else {
            typedef T t8_v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
            const t8_u2 w = *reinterpret_cast<const t8_u2*>(p);
            const t8_f4 u = t8_decode4<KIND>(w[0], byte), v = t8_decode4<KIND>(w[1], byte);
            if (c + 8 <= W) {
                *reinterpret_cast<t8_v8*>(o) = t8_v8{(T)u[0], (T)u[1], (T)u[2], (T)u[3], (T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            } else {
                t8_store4(o, W - c, u);
                t8_store4(o + 4, W - c - 4, v);
            }
        }
    }
}

// one pass of every lane (up to a grid that still counts its lanes in 32 bits): a fixed number of workgroups that walk the array was 10 %
// slower at 2 097 152 x 128
static unsigned t8_grid(long M, int W, int lanes_per_block) {
    const long n = (M * ((W + 31) / 32) * lanes_per_block + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n > (1l << 23) ? 1l << 23 : n);
}
template <typename T>
static int t8_pack_as(const void* x, long ldx, long M, int W, int kind, void* codes, void* bytes, hipStream_t st) {
    const dim3 grid(t8_grid(M, W, 32 / T8_CPL));
    if (kind == T8_RELU)
        k_tape8_pack<T, T8_RELU><<<grid, 256, 0, st>>>((const T*)x, ldx, M, W, (unsigned char*)codes, (unsigned char*)bytes);
    else
        k_tape8_pack<T, T8_SIGNED><<<grid, 256, 0, st>>>((const T*)x, ldx, M, W, (unsigned char*)codes, (unsigned char*)bytes);
    return (int)hipGetLastError();
}
template <typename T>
static int t8_unpack_as(const void* codes, const void* bytes, long M, int W, int kind, void* y, long ldy, hipStream_t st) {
    const dim3 grid(t8_grid(M, W, 32 * sizeof(T) / 16));
    if (kind == T8_RELU)
        k_tape8_unpack<T, T8_RELU><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)bytes, M, W, (T*)y, ldy);
    else
        k_tape8_unpack<T, T8_SIGNED><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)bytes, M, W, (T*)y, ldy);
    return (int)hipGetLastError();
}

extern "C" int magnet_tape8_pack(const void* x, int dtype, long ldx, long M, int W, int kind, void* codes, void* bytes, void* stream) {
    if (M < 0 || W < 1 || W > T8_WIDEST || ldx < W || kind < 0 || kind > 1 || ((uintptr_t)codes & 15)) return -2;
    if (M == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case T8_F32: return t8_pack_as<float>(x, ldx, M, W, kind, codes, bytes, st);
        case T8_BF16: return t8_pack_as<__bf16>(x, ldx, M, W, kind, codes, bytes, st);
        case T8_F16: return t8_pack_as<_Float16>(x, ldx, M, W, kind, codes, bytes, st);
    }
    return -2;
}
extern "C" int magnet_tape8_unpack(const void* codes, const void* bytes, long M, int W, int kind, void* y, int dtype, long ldy, void* stream) {
    if (M < 0 || W < 1 || W > T8_WIDEST || ldy < W || kind < 0 || kind > 1 || ((uintptr_t)codes & 15)) return -2;
    if (M == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case T8_F32: return t8_unpack_as<float>(codes, bytes, M, W, kind, y, ldy, st);
        case T8_BF16: return t8_unpack_as<__bf16>(codes, bytes, M, W, kind, y, ldy, st);
        case T8_F16: return t8_unpack_as<_Float16>(codes, bytes, M, W, kind, y, ldy, st);
    }
    return -2;
}
