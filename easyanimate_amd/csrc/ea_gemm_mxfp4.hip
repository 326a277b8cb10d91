// The product over microscaled 4-bit operands (ea_mxfp4.hip):  C_b = epi(A_b . W^T + bias)  on v_mfma_scale_f32_16x16x128_f8f6f4.
// The instruction multiplies 128 e2m1 codes per row and column, each run of 32 with its operands' scales, and adds in fp32 -- exact
// products, 16 cycles like the bf16 16x16x32 one, so a 4-bit tile moves through LDS and MFMA at the pace of a bf16 tile of a quarter
// of the K.
//
// A K tile is 256 codes = 128 bytes per row = 8 blocks of 32.  Lane (r = lane & 15, g = lane >> 4) feeds blocks 2g and 2g + 1 of its
// row to the tile's two MFMAs (the order of K is free as long as both operands agree): its two scale bytes are one 16-bit load.
// C^T orientation as in ea_gemm.hip: the weight fragment is the A operand, so a lane ends with 4 consecutive columns of one row.
//
//   gemm_mxfp4_skinny   M <= 64: 16 weight rows per workgroup, the K tiles dealt to its eight waves, operands straight from memory;
//                       for M <= 16 the activations may still be bf16 (quantised on the way, same codes as ea_mxfp4_quantize_bf16)
//   gemm_mxfp4_128      128 x 128 tiles, optionally K-split over workgroups (fp32 partial tiles in the caller's workspace, joined in
//                       a fixed order by gemm_mxfp4_join)
#include "ea_common.h"

namespace {

typedef int i32x4_m __attribute__((ext_vector_type(4)));
typedef int i32x8_m __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4_m __attribute__((ext_vector_type(4)));

struct MxArgs {
    const unsigned char* A;    // codes [kt][a_rows][128], scales [kt][a_rows][8]; batch element b = rows [b M, (b + 1) M)
    const unsigned char* As;
    const unsigned short* X;   // or bf16 activations [batch][M][K] (skinny kernel)
    const unsigned char* W;    // [kt][N][128], [kt][N][8]
    const unsigned char* Ws;
    const float* bias;
    void* C;
    const unsigned short* res;
    const float* gate;
    float* part;               // [splits][batch][M][N]
    int M, N, K, kt, splits, batch;
    int64_t a_rows, ldx, xbs, ldc, cbs, ldres, rbs, gbs;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ void glds16m(const void* gptr, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gptr,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}
__device__ __forceinline__ i32x8_m widen(const i32x4_m v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
// scale byte J of each operand's 16-bit pair
template <int J>
__device__ __forceinline__ f32x4 mfma_mx(const i32x4_m w, const int sw, const i32x4_m a, const int sa, const f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w), widen(a), c, 4, 4, J, sw, J, sa);
}

// four columns n0 .. n0 + 3 of row m: bias, activation, gate + residual in fp32, one rounding
template <int EPI>
__device__ __forceinline__ void mx_epilogue4(const MxArgs& p, const int b, const int m, const int n0, f32x4 v) {
    if (p.bias) v += *reinterpret_cast<const f32x4*>(p.bias + n0);
    if (EPI == EA_EPI_BIAS_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
    }
    if (EPI == EA_EPI_BIAS_GATE_RES) {
        const f32x4 g = *reinterpret_cast<const f32x4*>(p.gate + b * p.gbs + n0);
        const u16x4_m r = *reinterpret_cast<const u16x4_m*>(p.res + b * p.rbs + (int64_t)m * p.ldres + n0);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(g[e], v[e], bf16_bits_to_f32(r[e]));
    }
    if (EPI == EA_EPI_F32_OUT) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.C) + b * p.cbs + (int64_t)m * p.ldc + n0) = v;
    } else {
        u16x4_m o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16_bits(v[e]);
        *reinterpret_cast<u16x4_m*>(reinterpret_cast<unsigned short*>(p.C) + b * p.cbs + (int64_t)m * p.ldc + n0) = o;
    }
}

// ---- skinny -----------------------------------------------------------------------------------------------------------------------
constexpr int SK_WAVES = 8;

// one block of 32 bf16 values -> its 16 code bytes and scale byte, by ea_mxfp4_quantize_bf16's rule
__device__ __forceinline__ i32x4_m quant_block(const u16x8 (&v)[4], int& byte) {
    int top = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, (int)(v[u][e] & 0x7fff));
    const int be = top >> 7;
    byte = be == 255 ? 255 : (be > 2 ? be - 2 : 0);
    const float scale = __uint_as_float(byte ? (unsigned)byte << 23 : 0x00400000u);
    i32x4_m q;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        unsigned r = 0;
        const unsigned w0 = (unsigned)v[u][0] | ((unsigned)v[u][1] << 16), w1 = (unsigned)v[u][2] | ((unsigned)v[u][3] << 16);
        const unsigned w2 = (unsigned)v[u][4] | ((unsigned)v[u][5] << 16), w3 = (unsigned)v[u][6] | ((unsigned)v[u][7] << 16);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w0), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w1), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w2), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w3), scale, 3);
        q[u] = be == 255 ? 0 : (int)r;
    }
    return q;
}

template <int EPI, int MT, bool BF16_A>
__global__ __launch_bounds__(64 * SK_WAVES) void gemm_mxfp4_skinny_kernel(MxArgs p) {
    __shared__ f32x4 red[SK_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const int b = blockIdx.y;
    const int col0 = blockIdx.x * 16;
    const int wrow = col0 + lr < p.N ? col0 + lr : p.N - 1;
    f32x4 acc[MT];
    int arow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        arow[i] = i * 16 + lr < p.M ? i * 16 + lr : p.M - 1;
    }
    const unsigned char* wq = p.W + (int64_t)wrow * 128 + g * 32;
    const unsigned char* ws = p.Ws + (int64_t)wrow * 8 + g * 2;
    for (int t = wave; t < p.kt; t += SK_WAVES) {
        const int64_t wt = (int64_t)t * p.N;
        const i32x4_m w0 = *reinterpret_cast<const i32x4_m*>(wq + wt * 128);
        const i32x4_m w1 = *reinterpret_cast<const i32x4_m*>(wq + wt * 128 + 16);
        const int sw = *reinterpret_cast<const unsigned short*>(ws + wt * 8);
        if (BF16_A) {
            const int k0 = t * 256 + g * 64;
            const unsigned short* x = p.X + b * p.xbs + (int64_t)arow[0] * p.ldx + k0;
            u16x8 v[2][4];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                v[u >> 2][u & 3] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
                if (k0 + u * 8 < p.K) v[u >> 2][u & 3] = *reinterpret_cast<const u16x8*>(x + u * 8);
            }
            int s0, s1;
            const i32x4_m a0 = quant_block(v[0], s0);
            const i32x4_m a1 = quant_block(v[1], s1);
            acc[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w0), widen(a0), acc[0], 4, 4, 0, sw, 0, s0);
            acc[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w1), widen(a1), acc[0], 4, 4, 1, sw, 0, s1);
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t piece = (int64_t)t * p.a_rows + (int64_t)b * p.M + arow[i];
                const i32x4_m a0 = *reinterpret_cast<const i32x4_m*>(p.A + piece * 128 + g * 32);
                const i32x4_m a1 = *reinterpret_cast<const i32x4_m*>(p.A + piece * 128 + g * 32 + 16);
                const int sa = *reinterpret_cast<const unsigned short*>(p.As + piece * 8 + g * 2);
                acc[i] = mfma_mx<0>(w0, sw, a0, sa, acc[i]);
                acc[i] = mfma_mx<1>(w1, sw, a1, sa, acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave < MT) {
        f32x4 v = red[0][wave][lane];
#pragma unroll
        for (int w = 1; w < SK_WAVES; ++w) v += red[w][wave][lane];       // fixed order
        const int m = wave * 16 + lr, n0 = col0 + g * 4;
        if (m < p.M && n0 < p.N) mx_epilogue4<EPI>(p, b, m, n0, v);
    }
}

// ---- 128 x 128 --------------------------------------------------------------------------------------------------------------------
// Four waves, 64 x 64 each (4 x 4 MFMA tiles), K tiles of 256 double-buffered in LDS by LDS-DMA (rows of 128 bytes, 16-byte chunks
// XOR-swizzled with row & 7: eight consecutive rows of a fragment read hit eight different 16-byte columns); one barrier per tile.
constexpr int MX_OPER = 128 * 128, MX_STAGE = 2 * MX_OPER;

template <int EPI, bool SPLIT>
__global__ __launch_bounds__(256, 2) void gemm_mxfp4_128_kernel(MxArgs p) {
    __shared__ __attribute__((aligned(16))) char smem[2 * MX_STAGE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 1, wc = wave & 1, lr = lane & 15, g = lane >> 4;
    const int tm = blockIdx.x % p.tiles_m, tn = blockIdx.x / p.tiles_m;      // neighbours share a weight tile
    const int b = blockIdx.y;
    const int row0 = tm * 128, col0 = tn * 128;
    const int t0 = SPLIT ? (int)((int64_t)p.kt * blockIdx.z / p.splits) : 0;
    const int t1 = SPLIT ? (int)((int64_t)p.kt * (blockIdx.z + 1) / p.splits) : p.kt;
    const int64_t a_tile = p.a_rows * 128, w_tile = (int64_t)p.N * 128;

    const unsigned char* asrc[4];
    const unsigned char* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (wave * 4 + i) * 8 + (lane >> 3), cs = (lane & 7) ^ (r & 7);
        const int ra = row0 + r < p.M ? row0 + r : p.M - 1, rw = col0 + r < p.N ? col0 + r : p.N - 1;
        asrc[i] = p.A + t0 * a_tile + ((int64_t)b * p.M + ra) * 128 + cs * 16;
        wsrc[i] = p.W + t0 * w_tile + (int64_t)rw * 128 + cs * 16;
    }
    const unsigned char* sap[4];
    const unsigned char* swp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ra = row0 + wr * 64 + i * 16 + lr, rw = col0 + wc * 64 + i * 16 + lr;
        sap[i] = p.As + (t0 * p.a_rows + (int64_t)b * p.M + (ra < p.M ? ra : p.M - 1)) * 8 + g * 2;
        swp[i] = p.Ws + ((int64_t)t0 * p.N + (rw < p.N ? rw : p.N - 1)) * 8 + g * 2;
    }
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    int sa[4], sw[4];
    auto issue = [&](int stage) {
        char* d = smem + stage * MX_STAGE + wave * 4096;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            glds16m(asrc[i], d + i * 1024);
            glds16m(wsrc[i], d + MX_OPER + i * 1024);
            asrc[i] += a_tile;
            wsrc[i] += w_tile;
        }
    };
    if (t0 < t1) issue(0);
    for (int t = t0; t < t1; ++t) {
        const int st = (t - t0) & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sa[i] = *reinterpret_cast<const unsigned short*>(sap[i]);
            sw[i] = *reinterpret_cast<const unsigned short*>(swp[i]);
            sap[i] += p.a_rows * 8;
            swp[i] += (int64_t)p.N * 8;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 1 < t1) issue(st ^ 1);      // its last readers are behind the barrier above
        const char* a = smem + st * MX_STAGE + (wr * 64 + lr) * 128;
        const char* w = smem + st * MX_STAGE + MX_OPER + (wc * 64 + lr) * 128;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int ch = ((2 * g + ks) ^ (lr & 7)) << 4;
            i32x4_m af[4], wf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                af[i] = *reinterpret_cast<const i32x4_m*>(a + i * 2048 + ch);
                wf[i] = *reinterpret_cast<const i32x4_m*>(w + i * 2048 + ch);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[i][j] = ks == 0 ? mfma_mx<0>(wf[j], sw[j], af[i], sa[i], acc[i][j]) : mfma_mx<1>(wf[j], sw[j], af[i], sa[i], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = row0 + wr * 64 + i * 16 + lr;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n0 = col0 + wc * 64 + j * 16 + g * 4;
            if (n0 >= p.N) continue;
            if (SPLIT)
                *reinterpret_cast<f32x4*>(p.part + (((int64_t)blockIdx.z * p.batch + b) * p.M + m) * p.N + n0) = acc[i][j];
            else
                mx_epilogue4<EPI>(p, b, m, n0, acc[i][j]);
        }
    }
}

// sum of the K splits in their order, then the epilogue: one thread per 4 columns
template <int EPI>
__global__ __launch_bounds__(256) void gemm_mxfp4_join_kernel(MxArgs p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int nv = p.N >> 2;
    const int64_t row = i / nv;
    if (row >= (int64_t)p.batch * p.M) return;
    const int n0 = (int)(i - row * nv) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const int64_t plane = (int64_t)p.batch * p.M * p.N;
    for (int s = 0; s < p.splits; ++s) v += *reinterpret_cast<const f32x4*>(p.part + s * plane + row * p.N + n0);
    mx_epilogue4<EPI>(p, (int)(row / p.M), (int)(row % p.M), n0, v);
}

// K splits of the 128 x 128 kernel: enough workgroups for the 256 CUs, at least four K tiles each
int mx_splits(int64_t tiles, int kt) {
    int s = 1;
    while (tiles * s < 256 && kt / (s * 2) >= 4 && s < 16) s *= 2;
    return s;
}

template <int EPI>
void mx_launch(MxArgs& p, hipStream_t st) {
    if (p.M <= 64) {
        const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)p.batch);
        ea_count(p.X ? "gemm_mxfp4_skinny_bf16" : "gemm_mxfp4_skinny");
        if (p.X) hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 1, true>), grid, dim3(64 * SK_WAVES), 0, st, p);
        else if (p.M <= 16) hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 1, false>), grid, dim3(64 * SK_WAVES), 0, st, p);
        else if (p.M <= 32) hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 2, false>), grid, dim3(64 * SK_WAVES), 0, st, p);
        else hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 4, false>), grid, dim3(64 * SK_WAVES), 0, st, p);
        return;
    }
    p.tiles_m = (p.M + 127) / 128;
    p.tiles_n = (p.N + 127) / 128;
    p.splits = mx_splits((int64_t)p.tiles_m * p.tiles_n * p.batch, p.kt);
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.batch, (unsigned)p.splits);
    ea_count(p.splits > 1 ? "gemm_mxfp4_128_split" : "gemm_mxfp4_128");
    if (p.splits > 1) {
        hipLaunchKernelGGL((gemm_mxfp4_128_kernel<EPI, true>), grid, dim3(256), 0, st, p);
        const int64_t n = (int64_t)p.batch * p.M * (p.N / 4);
        hipLaunchKernelGGL(gemm_mxfp4_join_kernel<EPI>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
    } else {
        hipLaunchKernelGGL((gemm_mxfp4_128_kernel<EPI, false>), grid, dim3(256), 0, st, p);
    }
}

}  // namespace

extern "C" int64_t ea_gemm_mxfp4_workspace_bytes(int batch, int M, int N, int K) {
    if (batch <= 0 || M <= 64 || N <= 0 || K <= 0) return 0;
    const int64_t tiles = (int64_t)((M + 127) / 128) * ((N + 127) / 128) * batch;
    const int s = mx_splits(tiles, (int)(((int64_t)K + 255) / 256));
    return s > 1 ? (int64_t)s * batch * M * N * 4 : 0;
}

extern "C" int ea_gemm_mxfp4(const uint8_t* A, const uint8_t* A_scales, const ea_bf16* A_bf16, const uint8_t* W, const uint8_t* W_scales,
                             const float* bias, void* C, const ea_bf16* res, const float* gate, int batch, int M, int N, int K, int64_t lda,
                             int64_t a_batch_stride, int64_t ldc, int64_t c_batch_stride, int64_t ldres, int64_t res_batch_stride,
                             int64_t gate_batch_stride, int epilogue, void* workspace, int64_t workspace_bytes, void* stream) {
    EA_REQUIRE(batch > 0 && batch <= 65535 && M >= 0 && N > 0 && K > 0, "ea_gemm_mxfp4: bad sizes (batch %d, M %d, N %d, K %d)", batch, M, N, K);
    EA_REQUIRE(N % 8 == 0 && ldc % 8 == 0 && c_batch_stride % 8 == 0, "ea_gemm_mxfp4: N (%d), ldc and c_batch_stride must be multiples of 8", N);
    EA_REQUIRE(M <= 0x7fffff00 && N <= 0x7fffff00 && (((int64_t)M + 127) / 128) * (((int64_t)N + 127) / 128) <= 0x7fffffff &&
                   (int64_t)batch * M * (N / 4) <= (int64_t)0x7fffffff * 256,
               "ea_gemm_mxfp4: product too large for one launch (M %d, N %d)", M, N);
    EA_REQUIRE(epilogue >= 0 && epilogue <= 3, "ea_gemm_mxfp4: unknown epilogue %d", epilogue);
    if (M == 0) return EA_OK;
    EA_REQUIRE(W && W_scales && C && (A_bf16 ? !A && !A_scales : A && A_scales), "ea_gemm_mxfp4: null tensor (activations come either as codes + scales or as bf16)");
    EA_REQUIRE(((uintptr_t)A | (uintptr_t)A_bf16 | (uintptr_t)W | (uintptr_t)C | (uintptr_t)bias) % 16 == 0 &&
                   ((uintptr_t)A_scales | (uintptr_t)W_scales) % 8 == 0,
               "ea_gemm_mxfp4: codes, activations, C and bias must be 16-byte, scales 8-byte aligned");
    if (A_bf16)
        EA_REQUIRE(M <= 16 && K % 8 == 0 && lda % 8 == 0 && a_batch_stride % 8 == 0, "ea_gemm_mxfp4: bf16 activations need M <= 16 and K, lda, a_batch_stride multiples of 8");
    if (epilogue == EA_EPI_BIAS_GATE_RES)
        EA_REQUIRE(res && gate && ldres % 8 == 0 && res_batch_stride % 8 == 0 && gate_batch_stride % 4 == 0 && ((uintptr_t)res | (uintptr_t)gate) % 16 == 0,
                   "ea_gemm_mxfp4: gated-residual epilogue needs aligned res and gate");
    const int64_t need = ea_gemm_mxfp4_workspace_bytes(batch, M, N, K);
    EA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
               "ea_gemm_mxfp4: needs %lld bytes of 16-byte aligned workspace (ea_gemm_mxfp4_workspace_bytes)", (long long)need);
    MxArgs p;
    p.A = A; p.As = A_scales; p.X = A_bf16; p.W = W; p.Ws = W_scales; p.bias = bias; p.C = C; p.res = res; p.gate = gate;
    p.part = reinterpret_cast<float*>(workspace);
    p.M = M; p.N = N; p.K = K; p.kt = (int)(((int64_t)K + 255) / 256); p.splits = 1; p.batch = batch;
    p.a_rows = (int64_t)batch * M; p.ldx = lda; p.xbs = a_batch_stride; p.ldc = ldc; p.cbs = c_batch_stride;
    p.ldres = ldres; p.rbs = res_batch_stride; p.gbs = gate_batch_stride; p.tiles_m = p.tiles_n = 0;
    hipStream_t st = (hipStream_t)stream;
    switch (epilogue) {
        case EA_EPI_BIAS: mx_launch<EA_EPI_BIAS>(p, st); break;
        case EA_EPI_BIAS_GELU_TANH: mx_launch<EA_EPI_BIAS_GELU_TANH>(p, st); break;
        case EA_EPI_F32_OUT: mx_launch<EA_EPI_F32_OUT>(p, st); break;
        default: mx_launch<EA_EPI_BIAS_GATE_RES>(p, st); break;
    }
    return ea_check_launch("ea_gemm_mxfp4");
}
