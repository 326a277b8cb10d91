// The product over microscaled 4-bit operands (ea_mxfp4.hip):  C_b = epi(A_b . W^T + bias)  on v_mfma_scale_f32_16x16x128_f8f6f4.
// The instruction multiplies 128 e2m1 codes per row and column, each run of 32 with its operands' scales, and adds in fp32 -- exact
// products, 16 cycles like the bf16 16x16x32 one, so a 4-bit tile moves through LDS and MFMA at the pace of a bf16 tile of a quarter
// of the K.
//
// A K tile is 256 codes = 128 bytes per row = 8 blocks of 32.  Lane (r = lane & 15, g = lane >> 4) feeds block 4 j + g of its row to
// the tile's MFMA j; the storage keeps those two scale bytes next to each other, so they are one 16-bit load.
// C^T orientation as in ea_gemm.hip: the weight fragment is the A operand, so a lane ends with 4 consecutive columns of one row.
//
//   gemm_mxfp4_skinny   few rows: 16 weight rows per workgroup, the K tiles dealt to its eight waves, operands straight from memory;
//                       for M <= 16 the activations may still be bf16 (quantised on the way, same codes as ea_mxfp4_quantize_bf16)
//   gemm_mxfp4_tile     256 x 128 .. 64 x 64 tiles through LDS, the small ones by two groups of waves, optionally K-split over workgroups
//                       (fp32 partial tiles in the caller's workspace, joined in a fixed order by gemm_mxfp4_join)
//   gemm256_mxfp4_w4    256 x 256 tiles with a hand-placed main loop (ea_gemm_mxfp4_w4.inc)
//
// What bounds it: the weight bytes for few rows (one token x 3584 x 3584: 5.3 us, x 18944 x 3584: 10), the LDS fill of a CU for tiles up to
// 128 x 128 (24 - 33 KB per K tile at 130 - 150 GB/s; 512 x 3584 x 18944 in 33 us = 2.1 PFLOP/s with its weights from memory), the matrix
// pipe at the clock that the power budget leaves for the largest (8192^3 in 219 us = 5.0 PFLOP/s; ea_gemm_bf16 691 us).
#include "ea_common.h"
#include "ea_mxfp4_rows.h"

// ea_mxfp4.hip
int ea_mxfp4_quantize_launch(const unsigned short* x, unsigned char* codes, unsigned char* scales, int64_t rows, int K, int64_t ld, int64_t per,
                             int64_t batch_stride, hipStream_t st);
// ea_gemm.hip
int ea_gemm_mxfp4_w4_launch(const unsigned char* A, const unsigned char* As, int64_t as_bytes, const unsigned char* W, const unsigned char* Ws,
                            const float* bias, void* C, const ea_bf16* res, const float* gate, int batch, int M, int N, int kt, int64_t ldc,
                            int64_t cbs, int64_t ldres, int64_t rbs, int64_t gbs, int epilogue, hipStream_t st);

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

// Buffer-addressed LDS-DMA, 16 or 4 bytes per lane from base + voff.  live = 0 is an empty resource: the request keeps its place in
// the vmcnt order but moves nothing, so that a loop's tail needs no branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, const int live) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, live ? 0x7fffffff : 0, 0x00020000);
}
__device__ __forceinline__ void bdma16(const void* base, const int live, const int voff, void* lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(base, live), (__attribute__((address_space(3))) void*)lds_wave_base, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ void bdma4(const void* base, const int live, const int voff, void* lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(base, live), (__attribute__((address_space(3))) void*)lds_wave_base, 4, voff, 0, 0, 0);
}
__device__ __forceinline__ i32x8_m widen(const i32x4_m v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
// scale byte J of each operand's 16-bit pair
template <int J>
__device__ __forceinline__ f32x4 mfma_mx(const i32x4_m w, const int sw, const i32x4_m a, const int sa, const f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w), widen(a), c, 4, 4, J, sw, J, sa);
}

// Four columns n0 .. n0 + 3 of one row: bias, activation, gate + residual in fp32, one rounding.  The vectors come in registers so that
// a tile's epilogue loads them once, in front of everything that could wait for them.
__device__ __forceinline__ f32x4 mx_bias(const MxArgs& p, const int n0) {
    return p.bias ? *reinterpret_cast<const f32x4*>(p.bias + n0) : f32x4{0.f, 0.f, 0.f, 0.f};
}
template <int EPI>
__device__ __forceinline__ f32x4 mx_gate(const MxArgs& p, const int b, const int n0) {
    return EPI == EA_EPI_BIAS_GATE_RES ? *reinterpret_cast<const f32x4*>(p.gate + b * p.gbs + n0) : f32x4{0.f, 0.f, 0.f, 0.f};
}
template <int EPI>
__device__ __forceinline__ u16x4_m mx_res(const MxArgs& p, const int b, const int m, const int n0) {
    return EPI == EA_EPI_BIAS_GATE_RES ? *reinterpret_cast<const u16x4_m*>(p.res + b * p.rbs + (int64_t)m * p.ldres + n0) : u16x4_m{0, 0, 0, 0};
}
template <int EPI>
__device__ __forceinline__ void mx_store4(const MxArgs& p, const int b, const int m, const int n0, f32x4 v, const f32x4 bias, const f32x4 gate,
                                          const u16x4_m res) {
    v += bias;
    if (EPI == EA_EPI_BIAS_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
    }
    if (EPI == EA_EPI_BIAS_GATE_RES) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(gate[e], v[e], bf16_bits_to_f32(res[e]));
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
    const unsigned char* wq = p.W + (int64_t)wrow * 128 + g * 16;
    const unsigned char* ws = p.Ws + (int64_t)wrow * 8 + g * 2;
    for (int t = wave; t < p.kt; t += SK_WAVES) {
        const int64_t wt = (int64_t)t * p.N;
        const i32x4_m w0 = *reinterpret_cast<const i32x4_m*>(wq + wt * 128);
        const i32x4_m w1 = *reinterpret_cast<const i32x4_m*>(wq + wt * 128 + 64);
        const int sw = *reinterpret_cast<const unsigned short*>(ws + wt * 8);
        if (BF16_A) {
            const int k0 = t * 256 + g * 32;
            const unsigned short* x = p.X + b * p.xbs + (int64_t)arow[0] * p.ldx + k0;
            u16x8 v[2][4];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                v[u >> 2][u & 3] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
                const int ku = (u >> 2) * 128 + (u & 3) * 8;             // blocks g and 4 + g of the tile
                if (k0 + ku < p.K) v[u >> 2][u & 3] = *reinterpret_cast<const u16x8*>(x + ku);
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
                const i32x4_m a0 = *reinterpret_cast<const i32x4_m*>(p.A + piece * 128 + g * 16);
                const i32x4_m a1 = *reinterpret_cast<const i32x4_m*>(p.A + piece * 128 + g * 16 + 64);
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
        if (m < p.M && n0 < p.N) mx_store4<EPI>(p, b, m, n0, v, mx_bias(p, n0), mx_gate<EPI>(p, b, n0), mx_res<EPI>(p, b, m, n0));
    }
}

// ---- tiles through LDS ------------------------------------------------------------------------------------------------------------
// Block b runs on XCD b % 8 (its own L2).  An XCD takes a contiguous run of tiles, M fastest, so that the M tiles of one weight tile
// meet in one L2; with many M tiles (16 weight and 16 activation tiles at a time otherwise fall out of it) runs are walked in bands of
// 8 M tiles.
__device__ __forceinline__ bool mx_tile_of_block(const MxArgs& p, int& tm, int& tn) {
    const int total = p.tiles_m * p.tiles_n, per = (total + 7) >> 3;
    const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || idx >= total) return false;
    if (p.tiles_m <= 16) {
        tm = idx % p.tiles_m;
        tn = idx / p.tiles_m;
    } else {
        const int band = idx / (8 * p.tiles_n), first = band * 8, local = idx - band * 8 * p.tiles_n;
        const int rows = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
        tm = first + local % rows;
        tn = local / rows;
    }
    return true;
}

// BM x BN tiles, WM x WN waves, NS stages of one K tile each filled by LDS-DMA up to NS - 1 tiles ahead: rows of 128 bytes with the
// 16-byte chunks XOR-swizzled by row & 7 (eight consecutive rows of a fragment read hit eight different 16-byte columns), and behind
// them the tile's scale bytes.  One barrier per tile; the wait in front of it leaves the younger tiles in flight.
//
// KG = 2: two such groups of waves, which take the K tiles in turn (each its own stages) and join their sums through LDS: where tiles are
// few, a CU's four SIMDs have two waves each to cover what a K tile's chain of LDS reads, products and barrier leaves idle (128 x 64
// tiles, 512 x 3584 x 18944: 33 against 38 us; 64 x 64, 128 x 4096 x 11008: 12.4 against 15.1; no size slower).  128 x 128 tiles get the
// same from eight waves of 32 x 64 (1024 x 4096 x 4096: 15.2 us, four waves 15.8, two groups with two stages 16.7).
template <int BM, int BN, int WM, int WN, int NS, int KG, int EPI, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN * KG, BM * BN / (WM * WN) > 4096 ? 1 : 2) void gemm_mxfp4_tile_kernel(MxArgs p) {
    constexpr int WAVES = WM * WN;
    constexpr int TI = BM / (16 * WM), TJ = BN / (16 * WN);     // 16 x 16 MFMA tiles of a wave
    constexpr int PA = BM / (8 * WAVES), PW = BN / (8 * WAVES); // 1 KiB pieces of a wave, per operand
    constexpr int SRUNS = ((BM + BN) / 32 + WAVES - 1) / WAVES; // 256-byte runs of scales of a wave
    constexpr int OPER_A = BM * 128, OPER_W = BN * 128, STAGE = OPER_A + OPER_W + SRUNS * WAVES * 256;
    constexpr int LOADS = PA + PW + SRUNS;                      // per wave and tile
    static_assert((NS - 1) * LOADS < 64, "the counted wait has six bits");
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave_all / WAVES, wave = wave_all % WAVES;
    char* const smem = smem_all + kg * (NS * STAGE);
    const int wr = wave / WN, wc = wave % WN, lr = lane & 15, g = lane >> 4;
    int tm, tn;
    if (!mx_tile_of_block(p, tm, tn)) return;
    const int b = blockIdx.y;
    const int row0 = tm * BM, col0 = tn * BN;
    const int t0 = SPLIT ? (int)((int64_t)p.kt * blockIdx.z / p.splits) : 0;
    const int t1 = SPLIT ? (int)((int64_t)p.kt * (blockIdx.z + 1) / p.splits) : p.kt;
    const int own = (t1 - t0 - kg + KG - 1) / KG;      // K tiles t0 + kg, + KG, ..: this group's; the other group's may be one more
    const int64_t a_tile = p.a_rows * 128, w_tile = (int64_t)p.N * 128;

    // byte offsets inside the tile's rows of each operand (rows past the end read the last one again)
    int av[PA], wv[PW], sv[SRUNS];
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        const int r = (wave * PA + i) * 8 + (lane >> 3), ra = row0 + r < p.M ? r : p.M - 1 - row0;
        av[i] = ra * 128 + (((lane & 7) ^ (r & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int r = (wave * PW + i) * 8 + (lane >> 3), rw = col0 + r < p.N ? r : p.N - 1 - col0;
        wv[i] = rw * 128 + (((lane & 7) ^ (r & 7)) << 4);
    }
    // scales: 32 rows (4 bytes a lane) per request; request n of a wave is run wave + WAVES n of [BM / 32 A runs | BN / 32 W runs | ..],
    // runs past the last one (their count is rounded up so that every wave has the same number in flight) fetch the last W row again
#pragma unroll
    for (int n = 0; n < SRUNS; ++n) {
        const int run = wave + WAVES * n;
        const int r = (run < BM / 32 ? run : run - BM / 32) * 32 + (lane >> 1);
        const int last = (run < BM / 32 ? p.M - row0 : p.N - col0) - 1;
        sv[n] = (r < last ? r : last) * 8 + (lane & 1) * 4;
    }
    const unsigned char* pa = p.A + (t0 + kg) * a_tile + ((int64_t)b * p.M + row0) * 128;
    const unsigned char* pw = p.W + (t0 + kg) * w_tile + (int64_t)col0 * 128;
    const unsigned char* psa = p.As + ((t0 + kg) * p.a_rows + (int64_t)b * p.M + row0) * 8;
    const unsigned char* psw = p.Ws + ((int64_t)(t0 + kg) * p.N + col0) * 8;
    f32x4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // request d of a tile's LOADS
    auto request = [&](int d, int stage, int live) {
        char* to = smem + stage * STAGE;
        if (d < PA) bdma16(pa, live, av[d < PA ? d : 0], to + (wave * PA + d) * 1024);
        else if (d < PA + PW) bdma16(pw, live, wv[d < PA + PW ? (d >= PA ? d - PA : 0) : 0], to + OPER_A + (wave * PW + d - PA) * 1024);
        else {
            const int run = wave + WAVES * (d - PA - PW);
            bdma4(run < BM / 32 ? psa : psw, live, sv[d >= PA + PW ? d - PA - PW : 0], to + OPER_A + OPER_W + run * 256);
        }
    };
    auto advance = [&]() {
        pa += KG * a_tile;
        pw += KG * w_tile;
        psa += KG * p.a_rows * 8;
        psw += KG * (int64_t)p.N * 8;
    };
    // The two MFMA halves of a K tile carry everything else between their MFMAs, one instruction at a time, so that neither the LDS
    // reads nor the requests (a burst of them holds the wave until the memory pipe has taken them) stand in front of the matrix pipe:
    //   half 0 of tile t: read half 1's fragments; the second part of tile t + NS - 1's requests
    //   wait until tile t + 1 has landed, barrier: every wave has tile t in registers, its stage is free
    //   half 1 of tile t: read half 0's fragments and the scales of tile t + 1; the first part of tile t + NS's requests, into t's stage
    constexpr int FR = TI + TJ, SLOTS = TI * TJ, LA = (LOADS + 1) / 2, LB = LOADS - LA;
    const int a_off = (wr * (BM / WM) + lr) * 128, w_off = OPER_A + (wc * (BN / WN) + lr) * 128;
    const int ch0 = (g ^ (lr & 7)) << 4, ch1 = ((4 + g) ^ (lr & 7)) << 4;
    const int sa_off = OPER_A + OPER_W + (wr * (BM / WM) + lr) * 8 + g * 2, sw_off = OPER_A + OPER_W + (BM + wc * (BN / WN) + lr) * 8 + g * 2;
    i32x4_m a0[TI], w0[TJ], a1[TI], w1[TJ];
    int sa[TI], sw[TJ], san[TI], swn[TJ];
    auto read_frag = [&](int f, const char* base, int ch, i32x4_m (&af)[TI], i32x4_m (&wf)[TJ]) {
        if (f < TJ) wf[f < TJ ? f : 0] = *reinterpret_cast<const i32x4_m*>(base + w_off + f * 2048 + ch);
        else af[f >= TJ ? f - TJ : 0] = *reinterpret_cast<const i32x4_m*>(base + a_off + (f - TJ) * 2048 + ch);
    };
    auto read_scale = [&](int f, const char* base) {
        if (f < TJ) swn[f < TJ ? f : 0] = *reinterpret_cast<const unsigned short*>(base + sw_off + f * 128);
        else san[f >= TJ ? f - TJ : 0] = *reinterpret_cast<const unsigned short*>(base + sa_off + (f - TJ) * 128);
    };
    const int n = (t1 - t0 + KG - 1) / KG;             // trips: the last of one group may be empty
#pragma unroll
    for (int t = 0; t < NS - 1; ++t) {
#pragma unroll
        for (int d = 0; d < LOADS; ++d) request(d, t, t < own);
        advance();
    }
#pragma unroll
    for (int d = 0; d < LA; ++d) request(d, NS - 1, NS - 1 < own);
    // this wave's requests of the first tile have landed, then everybody's
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * LOADS + LA) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int f = 0; f < FR; ++f) {
        read_frag(f, smem, ch0, a0, w0);
        read_scale(f, smem);
    }
    int st = 0;
    for (int t = 0; t < n; ++t) {
#pragma unroll
        for (int i = 0; i < TI; ++i) sa[i] = KG == 1 || t < own ? san[i] : 0;       // (scale bytes 0: whatever the codes, products below 2^-240)
#pragma unroll
        for (int j = 0; j < TJ; ++j) sw[j] = KG == 1 || t < own ? swn[j] : 0;
        const int prev = st == 0 ? NS - 1 : st - 1;                  // stage of tile t + NS - 1
#pragma unroll
        for (int m = 0; m < SLOTS; ++m) {
            constexpr int F0 = FR + LB;
#pragma unroll
            for (int f = 0; f < F0; ++f)
                if (f >= m * F0 / SLOTS && f < (m + 1) * F0 / SLOTS) {
                    if (f < FR) read_frag(f, smem + st * STAGE, ch1, a1, w1);
                    else request(LA + f - FR, prev, t + NS - 1 < own);
                }
            acc[m % TI][m / TI] = mfma_mx<0>(w0[m / TI], sw[m / TI], a0[m % TI], sa[m % TI], acc[m % TI][m / TI]);
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * LOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int cur = st;
        st = st + 1 == NS ? 0 : st + 1;
#pragma unroll
        for (int m = 0; m < SLOTS; ++m) {
            constexpr int F1 = 2 * FR + LA;
#pragma unroll
            for (int f = 0; f < F1; ++f)
                if (f >= m * F1 / SLOTS && f < (m + 1) * F1 / SLOTS) {      // (behind the last tile: an old stage's bytes, not used)
                    if (f < FR) read_scale(f, smem + st * STAGE);
                    else if (f < 2 * FR) read_frag(f - FR, smem + st * STAGE, ch0, a0, w0);
                    else request(f - 2 * FR, cur, t + NS < own);
                }
            acc[m % TI][m / TI] = mfma_mx<1>(w1[m / TI], sw[m / TI], a1[m % TI], sa[m % TI], acc[m % TI][m / TI]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // join: each group takes half of the tile's row blocks, the other group's sums for them come through LDS
    constexpr int TK = TI / KG;
    if (KG == 2) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (no request may land behind this)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        f32x4* const box = reinterpret_cast<f32x4*>(smem_all) + wave * (TI * TJ * 64) + lane;
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
                if (i / TK != kg) box[(i * TJ + j) * 64] = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TK; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const f32x4 mine = kg ? acc[i + (KG - 1) * TK][j] : acc[i][j];
                acc[i][j] = mine + box[((i + kg * TK) * TJ + j) * 64];
            }
    }
    const int row_out = row0 + wr * (BM / WM) + (KG == 2 ? kg * TK * 16 : 0);
    const int n00 = col0 + wc * (BN / WN) + g * 4;
    if (SPLIT) {
#pragma unroll
        for (int i = 0; i < TK; ++i) {
            const int m = row_out + i * 16 + lr;
#pragma unroll
            for (int j = 0; j < TJ; ++j)
                if (m < p.M && n00 + j * 16 < p.N)
                    *reinterpret_cast<f32x4*>(p.part + (((int64_t)blockIdx.z * p.batch + b) * p.M + m) * p.N + n00 + j * 16) = acc[i][j];
        }
        return;
    }
    f32x4 bv[TJ], gv[TJ];
    int nc[TJ];                      // columns past N and rows past M: any address inside, never stored
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
        nc[j] = n00 + j * 16 < p.N ? n00 + j * 16 : 0;
        bv[j] = mx_bias(p, nc[j]);
        gv[j] = mx_gate<EPI>(p, b, nc[j]);
    }
#pragma unroll
    for (int i = 0; i < TK; ++i) {
        const int m = row_out + i * 16 + lr, mc = m < p.M ? m : p.M - 1;
        u16x4_m rr[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) rr[j] = mx_res<EPI>(p, b, mc, nc[j]);
#pragma unroll
        for (int j = 0; j < TJ; ++j)
            if (m < p.M && n00 + j * 16 < p.N) mx_store4<EPI>(p, b, m, n00 + j * 16, acc[i][j], bv[j], gv[j], rr[j]);
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
    const int b = (int)(row / p.M), m = (int)(row % p.M);
    mx_store4<EPI>(p, b, m, n0, v, mx_bias(p, n0), mx_gate<EPI>(p, b, n0), mx_res<EPI>(p, b, m, n0));
}

// a K tile's scales of a row are 8 bytes: stored scales, copied to where the 256 x 256 kernel may read behind the last row (one more
// launch, 3 us; 8191 x 8192 x 8192 226 us, 287 on 256 x 128 tiles, which need no copy; 3999 x 8200 x 3584 102 and 97: bits that do not
// depend on how the activations came are worth that)
__global__ __launch_bounds__(256) void copy_scales_kernel(const uint64_t* __restrict__ from, uint64_t* __restrict__ to, int64_t words) {
    const int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e * 256 < words) to[i + e * 256] = from[i + e * 256];
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct MxPlan {
    int cfg, splits;                      // -1 = skinny, else the index of its tile in MX_TILES
    bool w4;                              // the 256 x 256 kernel, where the operands and the epilogue allow it
    int64_t code_bytes, scale_bytes, part_bytes;
};
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Tiles and what a K tile of one costs a CU, in microseconds, between running alone and with the whole chip busy.  A grid takes
// ceil(tiles / 256 CUs) of them per K tile; the cheapest grid is taken: 256 x 18944 x 3584 runs in 22 us on 148 of the largest tiles and
// in 28 - 36 us on the others, 512 x 3584 x 18944 in 33 us on 224 tiles of 128 x 64 and in 35 - 46 us on the others, 1024 x 4096 x 4096 in
// 15 us on 256 of 128 x 128 and in 18 - 25 us on the others, 256 x 4096 x 4096 in 7.4 us on 256 of 64 x 64 and in 9 - 17 us on the others
// (weights from memory).
struct MxTile { int bm, bn; float us; };
constexpr float MX_W4_US = 1.2f;         // 256 x 256 tiles (ea_gemm_mxfp4_w4.inc)
constexpr MxTile MX_TILES[4] = {{256, 128, 0.75f}, {128, 128, 0.52f}, {128, 64, 0.33f}, {64, 64, 0.22f}};
// The skinny kernel reads its activations straight from memory, 16 rows at a time: best up to 16 rows (3584 x 3584: 3.9 - 4.4 us against
// 7 us of the tiles; 18944 x 3584: 9.8 - 12.6 against 11.5), and up to 32 while there are few workgroups (5.5 against 7.3; 18944 x 3584
// would take 17 against 12.5).
bool mx_skinny(int M, int N) { return M <= 16 || (M <= 32 && N <= 8192); }

int64_t mx_tiles(const MxTile& t, int batch, int M, int N) { return (((int64_t)M + t.bm - 1) / t.bm) * (((int64_t)N + t.bn - 1) / t.bn) * batch; }

// from_bf16: the activations come as bf16.  vec: their rows are 16-byte aligned with K % 8 == 0 (what the skinny kernel reads)
MxPlan mx_plan(int batch, int M, int N, int K, bool from_bf16, bool vec) {
    MxPlan n = {-1, 1, false, 0, 0, 0};
    const int64_t kt = ((int64_t)K + 255) / 256;
    if (from_bf16 && !(M <= 16 && vec)) {
        n.code_bytes = kt * batch * M * 128;
        n.scale_bytes = align256(kt * batch * M * 8 + MXW4_SCALE_PAD);     // (the 256 x 256 kernel reads scales two rows at a time)
    }
    if (mx_skinny(M, N)) return n;
    double best = 0;
    for (int i = 0; i < 4; ++i) {
        const double us = (double)((mx_tiles(MX_TILES[i], batch, M, N) + 255) / 256) * MX_TILES[i].us;
        if (n.cfg < 0 || us < best) {
            n.cfg = i;
            best = us;
        }
    }
    n.w4 = (double)((mx_tiles({256, 256, 0}, batch, M, N) + 255) / 256) * MX_W4_US < best;
    // (scales that the caller stored end with their last row: an odd one needs MXW4_SCALE_PAD bytes behind it, so they are copied)
    if (n.w4 && !from_bf16 && M % 2) n.scale_bytes = align256(kt * batch * M * 8 + MXW4_SCALE_PAD);
    if (n.w4) return n;
    // few tiles and a long K: split it while a split keeps 24 K tiles (6 us; joining two splits costs about 4).  (A larger tile is only
    // chosen when there are more than 256 of the next smaller one, so more than 128 of its own.)
    const int64_t tiles = mx_tiles(MX_TILES[n.cfg], batch, M, N);
    while (n.cfg == 3 && tiles * n.splits * 2 <= 256 && kt / (n.splits * 2) >= 24 && n.splits < 16) n.splits *= 2;
    if (n.splits > 1) n.part_bytes = (int64_t)n.splits * batch * M * N * 4;
    return n;
}

template <int BM, int BN, int WM, int WN, int NS, int KG, int EPI, bool SPLIT>
int mx_launch_tile(const MxArgs& p, hipStream_t st) {
    constexpr int WAVES = WM * WN, LDS = KG * NS * ((BM + BN) * 128 + ((BM + BN) / 32 + WAVES - 1) / WAVES * WAVES * 256);
    const auto kern = gemm_mxfp4_tile_kernel<BM, BN, WM, WN, NS, KG, EPI, SPLIT>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) {
        ea_set_error("ea_gemm_mxfp4: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
        return (int)e;
    }
    const dim3 grid((unsigned)((p.tiles_m * p.tiles_n + 7) / 8 * 8), (unsigned)p.batch, (unsigned)p.splits);
    hipLaunchKernelGGL(kern, grid, dim3(64 * WAVES * KG), LDS, st, p);
    return EA_OK;
}

template <int EPI>
int mx_launch(MxArgs& p, const MxPlan& n, hipStream_t st) {
    if (n.cfg < 0) {
        const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)p.batch);
        ea_count(p.X ? "gemm_mxfp4_skinny_bf16" : "gemm_mxfp4_skinny");
        if (p.X) hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 1, true>), grid, dim3(64 * SK_WAVES), 0, st, p);
        else if (p.M <= 16) hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 1, false>), grid, dim3(64 * SK_WAVES), 0, st, p);
        else hipLaunchKernelGGL((gemm_mxfp4_skinny_kernel<EPI, 2, false>), grid, dim3(64 * SK_WAVES), 0, st, p);
        return EA_OK;
    }
    if (EPI != EA_EPI_F32_OUT && n.w4) {             // (its epilogue goes through bf16 images of the tile)
        const int64_t as_bytes = n.scale_bytes ? n.scale_bytes : p.a_rows * p.kt * 8;
        const int rc = ea_gemm_mxfp4_w4_launch(p.A, p.As, as_bytes, p.W, p.Ws, p.bias, p.C, p.res, p.gate, p.batch, p.M, p.N, p.kt, p.ldc, p.cbs, p.ldres,
                                               p.rbs, p.gbs, EPI, st);
        if (rc != EA_ERR_ARG) return rc;
    }
    p.tiles_m = (p.M + MX_TILES[n.cfg].bm - 1) / MX_TILES[n.cfg].bm;
    p.tiles_n = (p.N + MX_TILES[n.cfg].bn - 1) / MX_TILES[n.cfg].bn;
    p.splits = n.splits;
    int rc;
    const bool split = n.splits > 1;
    switch (n.cfg) {
        case 0:
            ea_count("gemm_mxfp4_256x128");
            rc = mx_launch_tile<256, 128, 4, 2, 3, 1, EPI, false>(p, st);
            break;
        case 1:
            ea_count("gemm_mxfp4_128x128");
            rc = mx_launch_tile<128, 128, 4, 2, 4, 1, EPI, false>(p, st);
            break;
        case 2:
            ea_count("gemm_mxfp4_128x64");
            rc = mx_launch_tile<128, 64, 2, 2, 3, 2, EPI, false>(p, st);
            break;
        default:
            ea_count(split ? "gemm_mxfp4_64x64_split" : "gemm_mxfp4_64x64");
            rc = split ? mx_launch_tile<64, 64, 2, 2, 4, 2, EPI, true>(p, st) : mx_launch_tile<64, 64, 2, 2, 4, 2, EPI, false>(p, st);
    }
    if (rc == EA_OK && split) {
        const int64_t t = (int64_t)p.batch * p.M * (p.N / 4);
        hipLaunchKernelGGL(gemm_mxfp4_join_kernel<EPI>, dim3((unsigned)((t + 255) / 256)), dim3(256), 0, st, p);
    }
    return rc;
}

bool mx_vec(const ea_bf16* x, int K, int64_t lda, int64_t batch_stride) {
    return K % 8 == 0 && lda % 8 == 0 && batch_stride % 8 == 0 && ((uintptr_t)x & 15) == 0;
}

}  // namespace

extern "C" int64_t ea_gemm_mxfp4_workspace_bytes(int batch, int M, int N, int K, int a_is_bf16) {
    if (batch <= 0 || M <= 0 || N <= 0 || K <= 0) return 0;
    const MxPlan n = mx_plan(batch, M, N, K, a_is_bf16 != 0, false);
    return n.code_bytes + n.scale_bytes + n.part_bytes;
}

extern "C" int ea_gemm_mxfp4(const uint8_t* A, const uint8_t* A_scales, const ea_bf16* A_bf16, const uint8_t* W, const uint8_t* W_scales,
                             const float* bias, void* C, const ea_bf16* res, const float* gate, int batch, int M, int N, int K, int64_t lda,
                             int64_t a_batch_stride, int64_t ldc, int64_t c_batch_stride, int64_t ldres, int64_t res_batch_stride,
                             int64_t gate_batch_stride, int epilogue, void* workspace, int64_t workspace_bytes, void* stream) {
    EA_REQUIRE(batch > 0 && batch <= 65535 && M >= 0 && N > 0 && K > 0, "ea_gemm_mxfp4: bad sizes (batch %d, M %d, N %d, K %d)", batch, M, N, K);
    EA_REQUIRE(N % 8 == 0 && ldc % 8 == 0 && c_batch_stride % 8 == 0, "ea_gemm_mxfp4: N (%d), ldc and c_batch_stride must be multiples of 8", N);
    EA_REQUIRE((M <= 1 || ldc >= N) && (batch == 1 || c_batch_stride >= N), "ea_gemm_mxfp4: rows of C overlap (ldc %lld, batch stride %lld)",
               (long long)ldc, (long long)c_batch_stride);
    EA_REQUIRE(M <= 0x7fffff00 && N <= 0x7fffff00 && (((int64_t)M + 63) / 64) * (((int64_t)N + 63) / 64) <= 0x7fffffff &&
                   (int64_t)batch * M * (N / 4) <= (int64_t)0x7fffffff * 256,
               "ea_gemm_mxfp4: product too large for one launch (M %d, N %d)", M, N);
    EA_REQUIRE(epilogue >= 0 && epilogue <= 3, "ea_gemm_mxfp4: unknown epilogue %d", epilogue);
    if (M == 0) return EA_OK;
    EA_REQUIRE(W && W_scales && C && (A_bf16 ? !A && !A_scales : A && A_scales), "ea_gemm_mxfp4: null tensor (activations come either as codes + scales or as bf16)");
    EA_REQUIRE(((uintptr_t)A | (uintptr_t)W | (uintptr_t)C | (uintptr_t)bias) % 16 == 0 && ((uintptr_t)A_scales | (uintptr_t)W_scales) % 8 == 0,
               "ea_gemm_mxfp4: codes, C and bias must be 16-byte, scales 8-byte aligned");
    if (A_bf16) EA_REQUIRE(lda >= 0 && a_batch_stride >= 0 && (uintptr_t)A_bf16 % 2 == 0, "ea_gemm_mxfp4: bad activation strides");
    if (epilogue == EA_EPI_BIAS_GATE_RES)
        EA_REQUIRE(res && gate && ldres % 8 == 0 && res_batch_stride % 8 == 0 && gate_batch_stride % 4 == 0 && ((uintptr_t)res | (uintptr_t)gate) % 16 == 0,
                   "ea_gemm_mxfp4: gated-residual epilogue needs aligned res and gate");
    EA_REQUIRE(C != (const void*)A && C != (const void*)A_bf16 && C != (const void*)W, "ea_gemm_mxfp4: C must not overlap the activations or the weight");
    const MxPlan n = mx_plan(batch, M, N, K, A_bf16 != nullptr, A_bf16 && mx_vec(A_bf16, K, lda, a_batch_stride));
    const int64_t need = n.code_bytes + n.scale_bytes + n.part_bytes;
    EA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
               "ea_gemm_mxfp4: needs %lld bytes of 16-byte aligned workspace (ea_gemm_mxfp4_workspace_bytes)", (long long)need);
    hipStream_t st = (hipStream_t)stream;
    unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
    MxArgs p;
    p.A = A; p.As = A_scales; p.X = A_bf16; p.W = W; p.Ws = W_scales; p.bias = bias; p.C = C; p.res = res; p.gate = gate;
    p.part = reinterpret_cast<float*>(ws + n.code_bytes + n.scale_bytes);
    p.M = M; p.N = N; p.K = K; p.kt = (int)(((int64_t)K + 255) / 256); p.splits = 1; p.batch = batch;
    p.a_rows = (int64_t)batch * M; p.ldx = lda; p.xbs = a_batch_stride; p.ldc = ldc; p.cbs = c_batch_stride;
    p.ldres = ldres; p.rbs = res_batch_stride; p.gbs = gate_batch_stride; p.tiles_m = p.tiles_n = 0;
    if (n.code_bytes) {          // stored in front of the product; otherwise the skinny kernel quantises its rows itself
        EA_REQUIRE(ea_mxfp4_quantize_launch(A_bf16, ws, ws + n.code_bytes, p.a_rows, K, lda, M, a_batch_stride, st) == EA_OK,
                   "ea_gemm_mxfp4: activations too large for one launch");
        p.A = ws;
        p.As = ws + n.code_bytes;
        p.X = nullptr;
    } else if (n.scale_bytes && epilogue != EA_EPI_F32_OUT) {      // (fp32 results do not take that kernel)
        const int64_t words = p.a_rows * p.kt;
        hipLaunchKernelGGL(copy_scales_kernel, dim3((unsigned)((words + 1023) / 1024)), dim3(256), 0, st, reinterpret_cast<const uint64_t*>(A_scales),
                           reinterpret_cast<uint64_t*>(ws), words);
        p.As = ws;
    }
    int rc;
    switch (epilogue) {
        case EA_EPI_BIAS: rc = mx_launch<EA_EPI_BIAS>(p, n, st); break;
        case EA_EPI_BIAS_GELU_TANH: rc = mx_launch<EA_EPI_BIAS_GELU_TANH>(p, n, st); break;
        case EA_EPI_F32_OUT: rc = mx_launch<EA_EPI_F32_OUT>(p, n, st); break;
        default: rc = mx_launch<EA_EPI_BIAS_GATE_RES>(p, n, st); break;
    }
    return rc != EA_OK ? rc : ea_check_launch("ea_gemm_mxfp4");
}
