// Microscaled 4-bit storage (OCP MX, FP4 elements): blocks of 32 consecutive elements of a row share one power-of-two scale,
//     e = clamp(floor(log2 max|x|) - 2, -127, 127),  byte e + 127;   code = nearest e2m1 of x / 2^e (ties to even, |.| <= 6),
// e2m1 = {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign bit.  A block that holds an infinity or a NaN gets byte 255 (the format's NaN) and
// codes 0; a block of zeros byte 0.
//
// Layout, K-blocked like the bf16 operands of ea_gemm_bf16_kblocked: codes [ceil(K/256)][rows][128 bytes] (element k of a tile in
// nibble k & 1 of byte k / 2), scales [ceil(K/256)][rows][8 bytes] with block 4 j + g of a
// tile at byte 2 g + j (the two that a lane of the product's matrix instructions needs are neighbours); elements >= K are zeros.
// A 256-deep K tile of R rows is then one contiguous run for the product's LDS-DMA, and K needs no tail code there.
//
// Both directions are HBM-bound (2 + 17/32 bytes per element, no reuse): 13312 x 3584 in 18 us either way, 3584 x 18944 in 25 us = 6.6 -
// 6.8 TB/s (a 2 GiB copy reaches 5.0; these fit the last-level cache in part).  Matrices of a few MB cost their launch.  Four rows per
// thread keep four loads in flight; K tile by K tile per workgroup, not row by row, makes the code writes 4 KiB runs.
#include "ea_common.h"

namespace {

// the 8 codes of 8 bf16 values as one dword; the scale is an exact power of two, the instruction rounds to nearest even and saturates
__device__ __forceinline__ unsigned quant8(const u16x8 v, const float scale) {
    unsigned r = 0;
    const unsigned w0 = (unsigned)v[0] | ((unsigned)v[1] << 16), w1 = (unsigned)v[2] | ((unsigned)v[3] << 16);
    const unsigned w2 = (unsigned)v[4] | ((unsigned)v[5] << 16), w3 = (unsigned)v[6] | ((unsigned)v[7] << 16);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w0), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w1), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w2), scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w3), scale, 3);
    return r;
}

__device__ __forceinline__ int scale_byte(int block) { return 2 * (block & 3) + (block >> 2); }

// Both kernels: a workgroup is one K tile of 32 rows; half a wave is one row's tile (32 lanes x 8 elements), four threads a block of
// 32, and a thread has ROWS_PER loads in flight.  Reads (writes) of 512 contiguous bytes per row, 128 x 32 contiguous code bytes;
// neighbouring workgroups are neighbouring K tiles of the same rows.  The only division is the block index's (scalar, once).
constexpr int ROWS_PER = 4, WG_ROWS = 8 * ROWS_PER;
// 16 bytes on any even address: one access on this hardware
typedef unsigned short u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// VEC: K % 8 == 0, so a thread's elements are one load, inside the row or outside it as a whole; otherwise the row's last ones are read
// (written) one by one.
// Row r of the output is row r % per of batch element r / per of x.
template <bool VEC>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const unsigned short* __restrict__ x, unsigned char* __restrict__ q,
                                                             unsigned char* __restrict__ s, int64_t rows, int K, int kt, int64_t ld, int64_t per,
                                                             int64_t batch_stride) {
    const unsigned tile = blockIdx.x % (unsigned)kt;
    const int64_t row0 = (int64_t)(blockIdx.x / (unsigned)kt) * WG_ROWS + (threadIdx.x >> 5);
    const int c = threadIdx.x & 31, k = (int)tile * 256 + c * 8;
    u16x8 v[ROWS_PER];
#pragma unroll
    for (int i = 0; i < ROWS_PER; ++i) {
        const int64_t row = row0 + 8 * i;
        v[i] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (row < rows) {
            const int64_t b = per == rows ? 0 : row / per;
            const unsigned short* src = x + b * batch_stride + (row - b * per) * ld + k;
            if (VEC ? k < K : k + 8 <= K) {
                v[i] = *reinterpret_cast<const u16x8_any*>(src);
            } else if (!VEC) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + e < K) v[i][e] = src[e];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS_PER; ++i) {
        const int64_t row = row0 + 8 * i;
        int top = 0;                                // max |x| as its bf16 bits: the order of non-negative floats, NaN above infinity
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, (int)(v[i][e] & 0x7fff));
        top = max(top, __shfl_xor(top, 1, 64));
        top = max(top, __shfl_xor(top, 2, 64));
        const int be = top >> 7;
        const int byte = be == 255 ? 255 : (be > 2 ? be - 2 : 0);
        const float scale = __uint_as_float(byte ? (unsigned)byte << 23 : 0x00400000u);
        const unsigned codes = be == 255 ? 0u : quant8(v[i], scale);
        if (row < rows) {
            const int64_t piece = (int64_t)tile * rows + row;
            *reinterpret_cast<unsigned*>(q + piece * 128 + c * 4) = codes;
            if ((c & 3) == 0) s[piece * 8 + scale_byte(c >> 2)] = (unsigned char)byte;
        }
    }
}

// code * 2^e: at most two significant bits above a power of two, exact in bf16 down to its subnormals
template <bool VEC>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ s,
                                                               unsigned short* __restrict__ y, int64_t rows, int K, int kt) {
    const unsigned tile = blockIdx.x % (unsigned)kt;
    const int64_t row0 = (int64_t)(blockIdx.x / (unsigned)kt) * WG_ROWS + (threadIdx.x >> 5);
    const int c = threadIdx.x & 31, k = (int)tile * 256 + c * 8;
    if (k >= K) return;
    unsigned codes[ROWS_PER];
    int byte[ROWS_PER];
#pragma unroll
    for (int i = 0; i < ROWS_PER; ++i) {
        const int64_t row = row0 + 8 * i, piece = (int64_t)tile * rows + (row < rows ? row : rows - 1);
        codes[i] = *reinterpret_cast<const unsigned*>(q + piece * 128 + c * 4);
        byte[i] = s[piece * 8 + scale_byte(c >> 2)];
    }
#pragma unroll
    for (int i = 0; i < ROWS_PER; ++i) {
        const int64_t row = row0 + 8 * i;
        const float scale = __uint_as_float(byte[i] == 255 ? 0x7fc00000u : byte[i] ? (unsigned)byte[i] << 23 : 0x00400000u);
        typedef unsigned u32x4_q __attribute__((ext_vector_type(4)));
        u32x4_q w;
        w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], scale, 0));
        w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], scale, 1));
        w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], scale, 2));
        w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], scale, 3));
        if (row >= rows) continue;
        unsigned short* dst = y + row * (int64_t)K + k;
        if (VEC || k + 8 <= K) {
            *reinterpret_cast<u32x4_any*>(dst) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < K) dst[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}

bool grid_of(int64_t rows, int kt, dim3& grid) {
    const int64_t n = (rows + WG_ROWS - 1) / WG_ROWS;
    if (n > 0x7fffffff / kt) return false;
    grid = dim3((unsigned)(n * kt));
    return true;
}

}  // namespace

int ea_mxfp4_quantize_launch(const unsigned short* x, unsigned char* codes, unsigned char* scales, int64_t rows, int K, int64_t ld, int64_t per,
                             int64_t batch_stride, hipStream_t st) {
    const int kt = (int)(((int64_t)K + 255) / 256);
    dim3 grid;
    if (!grid_of(rows, kt, grid)) return EA_ERR_ARG;
    if (K % 8 == 0)
        hipLaunchKernelGGL(mxfp4_quantize_kernel<true>, grid, dim3(256), 0, st, x, codes, scales, rows, K, kt, ld, per, batch_stride);
    else
        hipLaunchKernelGGL(mxfp4_quantize_kernel<false>, grid, dim3(256), 0, st, x, codes, scales, rows, K, kt, ld, per, batch_stride);
    return EA_OK;
}

extern "C" int ea_mxfp4_quantize_bf16(const ea_bf16* x, uint8_t* codes, uint8_t* scales, int64_t rows, int K, int64_t ld, void* stream) {
    EA_REQUIRE(rows >= 0 && K > 0 && ld >= K, "ea_mxfp4_quantize_bf16: bad geometry (rows %lld, K %d, row stride %lld)", (long long)rows, K, (long long)ld);
    if (rows == 0) return EA_OK;
    EA_REQUIRE(x && codes && scales, "ea_mxfp4_quantize_bf16: null tensor");
    EA_REQUIRE((((uintptr_t)codes) & 15) == 0 && (((uintptr_t)scales) & 7) == 0, "ea_mxfp4_quantize_bf16: codes 16-byte, scales 8-byte aligned");
    EA_REQUIRE(ea_mxfp4_quantize_launch(x, codes, scales, rows, K, ld, rows, 0, (hipStream_t)stream) == EA_OK,
               "ea_mxfp4_quantize_bf16: tensor too large for one launch");
    return ea_check_launch("ea_mxfp4_quantize_bf16");
}

extern "C" int ea_mxfp4_dequantize_bf16(const uint8_t* codes, const uint8_t* scales, ea_bf16* y, int64_t rows, int K, void* stream) {
    EA_REQUIRE(rows >= 0 && K > 0, "ea_mxfp4_dequantize_bf16: bad geometry (rows %lld, K %d)", (long long)rows, K);
    if (rows == 0) return EA_OK;
    EA_REQUIRE(codes && scales && y, "ea_mxfp4_dequantize_bf16: null tensor");
    EA_REQUIRE((((uintptr_t)codes | (uintptr_t)y) & 15) == 0 && (((uintptr_t)scales) & 7) == 0,
               "ea_mxfp4_dequantize_bf16: codes / y 16-byte, scales 8-byte aligned");
    const int kt = (int)(((int64_t)K + 255) / 256);
    dim3 grid;
    EA_REQUIRE(grid_of(rows, kt, grid), "ea_mxfp4_dequantize_bf16: tensor too large for one launch");
    if (K % 8 == 0)
        hipLaunchKernelGGL(mxfp4_dequantize_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, codes, scales, y, rows, K, kt);
    else
        hipLaunchKernelGGL(mxfp4_dequantize_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, codes, scales, y, rows, K, kt);
    return ea_check_launch("ea_mxfp4_dequantize_bf16");
}
