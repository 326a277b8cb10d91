// Microscaled 4-bit storage (OCP MX, FP4 elements): blocks of 32 consecutive elements of a row share one power-of-two scale,
//     e = clamp(floor(log2 max|x|) - 2, -127, 127),  byte e + 127;   code = nearest e2m1 of x / 2^e (ties to even, |.| <= 6),
// e2m1 = {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign bit.  A block that holds an infinity or a NaN gets byte 255 (the format's NaN) and
// codes 0; a block of zeros byte 0.
//
// Layout, K-blocked like the bf16 operands of ea_gemm_bf16_kblocked: codes [ceil(K/256)][rows][128 bytes] (element k of a tile in
// nibble k & 1 of byte k / 2), scales [ceil(K/256)][rows][8 bytes]; elements >= K of the last tile are zeros with their blocks' scales.
// A 256-deep K tile of R rows is then one contiguous run for the product's LDS-DMA, and K needs no tail code there.
//
// Both directions are HBM-bound (2 + 17/32 bytes per element, no reuse).
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

// One thread = 8 elements, four threads = a block, a wave = two K tiles of one row (1 KiB read, 2 x 128 B written).
// VEC: rows of x are 16-byte aligned and K % 8 == 0, so a thread's elements are one load, inside the row or outside it as a whole.
template <bool VEC>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const unsigned short* __restrict__ x, unsigned char* __restrict__ q,
                                                             unsigned char* __restrict__ s, int64_t rows, int K, int kt, int64_t ld) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per_row = kt * 32;
    const int64_t row = i / per_row;
    if (row >= rows) return;                        // per_row is a multiple of 32: the four threads of a block leave together
    const int c = (int)(i - row * per_row);         // 8-element chunk of the row
    const int k = c * 8;
    u16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    const unsigned short* src = x + row * ld + k;
    if (VEC) {
        if (k < K) v = *reinterpret_cast<const u16x8*>(src);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) v[e] = src[e];
    }
    int top = 0;                                    // max |x| as its bf16 bits: the order of non-negative floats, NaN above infinity
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, (int)(v[e] & 0x7fff));
    top = max(top, __shfl_xor(top, 1, 64));
    top = max(top, __shfl_xor(top, 2, 64));
    const int be = top >> 7;
    const int byte = be == 255 ? 255 : (be > 2 ? be - 2 : 0);
    const float scale = __uint_as_float(byte ? (unsigned)byte << 23 : 0x00400000u);
    const unsigned codes = be == 255 ? 0u : quant8(v, scale);
    const int64_t piece = (int64_t)(c >> 5) * rows + row;
    *reinterpret_cast<unsigned*>(q + piece * 128 + (c & 31) * 4) = codes;
    if ((c & 3) == 0) s[piece * 8 + ((c & 31) >> 2)] = (unsigned char)byte;
}

// code * 2^e: at most two significant bits above a power of two, exact in bf16 down to its subnormals
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ s,
                                                               unsigned short* __restrict__ y, int64_t rows, int K, int kt) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per_row = kt * 32;
    const int64_t row = i / per_row;
    if (row >= rows) return;
    const int c = (int)(i - row * per_row), k = c * 8;
    if (k >= K) return;
    const int64_t piece = (int64_t)(c >> 5) * rows + row;
    const unsigned codes = *reinterpret_cast<const unsigned*>(q + piece * 128 + (c & 31) * 4);
    const int byte = s[piece * 8 + ((c & 31) >> 2)];
    const float scale = __uint_as_float(byte == 255 ? 0x7fc00000u : byte ? (unsigned)byte << 23 : 0x00400000u);
    u16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned n = codes >> (4 * e);
        // e2m1 -> fp32 by its definition: 0 and 0.5 below the first binade, (1 + m/2) 2^(x-1) from there on
        const unsigned m = n & 7u;
        const float mag = m < 2 ? 0.5f * (float)m : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
        const float f = mag * scale;
        o[e] = (unsigned short)((__float_as_uint(f) >> 16) | ((n & 8u) << 12));
    }
    unsigned short* dst = y + row * (int64_t)K + k;
    if (K % 8 == 0) {
        *reinterpret_cast<u16x8*>(dst) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) dst[e] = o[e];
    }
}

constexpr int64_t MAX_THREADS = (int64_t)0x7fffffff * 256;   // grid limit of one launch

}  // namespace

extern "C" int ea_mxfp4_quantize_bf16(const ea_bf16* x, uint8_t* codes, uint8_t* scales, int64_t rows, int K, int64_t ld, void* stream) {
    EA_REQUIRE(rows >= 0 && K > 0 && ld >= K, "ea_mxfp4_quantize_bf16: bad geometry (rows %lld, K %d, row stride %lld)", (long long)rows, K, (long long)ld);
    if (rows == 0) return EA_OK;
    EA_REQUIRE(x && codes && scales, "ea_mxfp4_quantize_bf16: null tensor");
    EA_REQUIRE((((uintptr_t)codes) & 15) == 0 && (((uintptr_t)scales) & 7) == 0, "ea_mxfp4_quantize_bf16: codes 16-byte, scales 8-byte aligned");
    const int kt = (int)(((int64_t)K + 255) / 256);
    const int64_t n = rows * kt * 32;
    EA_REQUIRE(n <= MAX_THREADS, "ea_mxfp4_quantize_bf16: tensor too large for one launch");
    const dim3 grid((unsigned)((n + 255) / 256));
    if (K % 8 == 0 && ld % 8 == 0 && (((uintptr_t)x) & 15) == 0)
        hipLaunchKernelGGL(mxfp4_quantize_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, x, codes, scales, rows, K, kt, ld);
    else
        hipLaunchKernelGGL(mxfp4_quantize_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, x, codes, scales, rows, K, kt, ld);
    return ea_check_launch("ea_mxfp4_quantize_bf16");
}

extern "C" int ea_mxfp4_dequantize_bf16(const uint8_t* codes, const uint8_t* scales, ea_bf16* y, int64_t rows, int K, void* stream) {
    EA_REQUIRE(rows >= 0 && K > 0, "ea_mxfp4_dequantize_bf16: bad geometry (rows %lld, K %d)", (long long)rows, K);
    if (rows == 0) return EA_OK;
    EA_REQUIRE(codes && scales && y, "ea_mxfp4_dequantize_bf16: null tensor");
    EA_REQUIRE((((uintptr_t)codes | (uintptr_t)y) & 15) == 0 && (((uintptr_t)scales) & 7) == 0,
               "ea_mxfp4_dequantize_bf16: codes / y 16-byte, scales 8-byte aligned");
    const int kt = (int)(((int64_t)K + 255) / 256);
    const int64_t n = rows * kt * 32;
    EA_REQUIRE(n <= MAX_THREADS, "ea_mxfp4_dequantize_bf16: tensor too large for one launch");
    hipLaunchKernelGGL(mxfp4_dequantize_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, codes, scales, y, rows, K,
                       kt);
    return ea_check_launch("ea_mxfp4_dequantize_bf16");
}
