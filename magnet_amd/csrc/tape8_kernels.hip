// Writing and reading the 8-bit tape (the format: tape8.cuh).
//
// Both kernels are one pass bound by HBM: a pack reads the row (4 / 2 bytes a value) and writes 33/32 bytes a value, an unpack the other
// way.  A lane takes four neighbouring columns, eight neighbouring lanes one block of 32: the block's top is three lane exchanges, the
// codes leave as one word per lane, a wave's stores are whole lines.  A lane walks its positions by adding the grid's stride, split once
// into rows and columns: no division in the loop, and 64-bit row offsets.
#include "common.cuh"
#include "tape8.cuh"

struct T8Walk {                          // position (row, group of four columns) of a flat index, and the step between two visits
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
__global__ void __launch_bounds__(256) k_tape8_pack(const T* __restrict__ x, long ldx, long M, int W, int vec, unsigned char* __restrict__ codes,
                                                    unsigned char* __restrict__ bytes) {
    const int groups = ((W + 31) / 32) * 8;
    T8Walk at((long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, groups);
    for (; at.row < M; at.next()) {      // (the eight lanes of a block leave together: groups and the stride are multiples of 8)
        const int c = 4 * at.g;
        const t8_f4 v = t8_load4(x + at.row * ldx + c, vec && c < W, W - c);
        const unsigned byte = t8_byte<KIND>(t8_max8(t8_top4<KIND>(v)));
        *reinterpret_cast<unsigned*>(codes + at.row * (4 * groups) + c) = t8_code4<KIND>(v, byte);
        if (!(at.g & 7)) bytes[at.row * (groups / 8) + (at.g >> 3)] = (unsigned char)byte;
    }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(256) k_tape8_unpack(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ bytes, long M, int W,
                                                      T* __restrict__ y, long ldy, int vec) {
    const int groups = ((W + 31) / 32) * 8;
    T8Walk at((long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, groups);
    for (; at.row < M; at.next()) {
        const int c = 4 * at.g;
        const unsigned w = *reinterpret_cast<const unsigned*>(codes + at.row * (4 * groups) + c);
        t8_store4(y + at.row * ldy + c, vec && c < W, W - c, t8_decode4<KIND>(w, bytes[at.row * (groups / 8) + (at.g >> 3)]));
    }
}

static unsigned t8_grid(long M, int W) {
    const long n = (M * (((W + 31) / 32) * 8) + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n > 8192 ? 8192 : n);
}
// four values at once: the width, the row stride and the address are multiples of four values
static int t8_vec(const void* p, long ld, int W, size_t size) { return !(W & 3) && !(ld & 3) && !((uintptr_t)p & (4 * size - 1)); }

template <typename T>
static int t8_pack_as(const void* x, long ldx, long M, int W, int kind, void* codes, void* bytes, hipStream_t st) {
    const int vec = t8_vec(x, ldx, W, sizeof(T));
    const dim3 grid(t8_grid(M, W));
    if (kind == T8_RELU)
        k_tape8_pack<T, T8_RELU><<<grid, 256, 0, st>>>((const T*)x, ldx, M, W, vec, (unsigned char*)codes, (unsigned char*)bytes);
    else
        k_tape8_pack<T, T8_SIGNED><<<grid, 256, 0, st>>>((const T*)x, ldx, M, W, vec, (unsigned char*)codes, (unsigned char*)bytes);
    return (int)hipGetLastError();
}
template <typename T>
static int t8_unpack_as(const void* codes, const void* bytes, long M, int W, int kind, void* y, long ldy, hipStream_t st) {
    const int vec = t8_vec(y, ldy, W, sizeof(T));
    const dim3 grid(t8_grid(M, W));
    if (kind == T8_RELU)
        k_tape8_unpack<T, T8_RELU><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)bytes, M, W, (T*)y, ldy, vec);
    else
        k_tape8_unpack<T, T8_SIGNED><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)bytes, M, W, (T*)y, ldy, vec);
    return (int)hipGetLastError();
}

extern "C" int magnet_tape8_pack(const void* x, int dtype, long ldx, long M, int W, int kind, void* codes, void* bytes, void* stream) {
    if (M < 0 || W < 1 || ldx < W || kind < 0 || kind > 1 || ((uintptr_t)codes & 15)) return -2;
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
    if (M < 0 || W < 1 || ldy < W || kind < 0 || kind > 1 || ((uintptr_t)codes & 15)) return -2;
    if (M == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case T8_F32: return t8_unpack_as<float>(codes, bytes, M, W, kind, y, ldy, st);
        case T8_BF16: return t8_unpack_as<__bf16>(codes, bytes, M, W, kind, y, ldy, st);
        case T8_F16: return t8_unpack_as<_Float16>(codes, bytes, M, W, kind, y, ldy, st);
    }
    return -2;
}
