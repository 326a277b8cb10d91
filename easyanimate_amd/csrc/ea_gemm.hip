// bf16 GEMM with fused epilogues for the DiT linears:  C_b = epi(A_b . W^T + bias)   (MFMA 32x32x16).
//
// Mapping to CDNA4 (see DESIGN.md "ea_gemm_bf16"):
//   * workgroup = 256 threads = 4 waves (2 x 2), block tile 128(M) x 128(N) x 64(K); wave tile 64 x 64
//     = 2 x 2 MFMA tiles; 16 v_mfma_f32_32x32x16_bf16 per wave per K-tile.
//   * both operands are K-contiguous ([M,K] activations, [N,K] nn.Linear weights), so both are staged
//     with LDS-DMA (global_load_lds_dwordx4, 1 KiB per wave instruction) into 128-byte rows; the 16-byte
//     chunk index is XOR-swizzled with ((row>>1)&7) -- applied on the per-lane SOURCE address because the
//     DMA destination is lane-linear -- which makes every ds_read_b128 fragment read conflict-free.
//   * double-buffered LDS (2 x 32 KiB), one s_barrier per K-tile, next tile's DMA in flight during the
//     MFMAs; 2 workgroups per CU hide each other's barrier.
//   * the MFMA computes C^T tiles (A-operand = W rows, B-operand = activation rows) and the W rows are
//     fed in bit-2/bit-3-swapped order, so each lane ends with 8 *contiguous* output columns per 8
//     accumulator registers: 16-byte bf16 stores, 16-byte residual loads, vector bias/gate loads.
//   * blockIdx is remapped so that the 8 XCDs (private L2s) each walk a contiguous band of M-tiles.
#include "ea_common.h"

namespace {

constexpr int BM = 128, BN = 128, BK = 64;
constexpr int TILE_BYTES = 128 * BK * 2;       // 16 KiB per operand tile
constexpr int STAGE_BYTES = 2 * TILE_BYTES;    // A + W
constexpr int GEMM_LDS = 2 * STAGE_BYTES;      // double buffer = 64 KiB

struct GemmArgs {
    const unsigned short* A;
    const unsigned short* W;
    const float* bias;
    unsigned short* C;
    const unsigned short* res;
    const float* gate;
    int M, N, K;
    int64_t lda, abs_, ldc, cbs, ldres, rbs, gbs;
    int tiles_m, tiles_n, rows_per_xcd;
    // K-blocked operands of the 256 x 256 kernel (ea_gemm_bf16_kblocked): an operand laid out [K / 64][rows][64] -- a 64-deep K
    // tile of 256 rows is ONE contiguous 32 KiB block instead of 256 pieces a row stride apart.  Row-major defaults: a_kstep =
    // w_kstep = 64 (elements to the next K tile), ldw = K, c_kstep = 0 (C row-major).
    int64_t a_kstep = 64, w_kstep = 64, ldw = 0, c_kstep = 0;
};

__device__ __forceinline__ void glds16(const void* gptr, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gptr,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

// Buffer-addressed LDS-DMA (see ea_attention.hip): 16 bytes per lane from base + voff (per lane, fixed) + soff (scalar).
__device__ __forceinline__ void bdma16g(const void* base, int extent, int voff, int soff, void* lds_wave_base) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, extent, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds_wave_base, 16, voff, soff, 0, 0);
}

// ---- fp8 weight storage (the reference's `model_cpu_offload_and_qfloat8` mode, utils/fp8_optimization.py:17-35: every
// Linear weight is kept as torch.float8_e4m3fn = OCP E4M3 and up-cast to bf16 for each call).  The W8 kernel variants read
// the fp8 bytes themselves: a weight tile row comes in through registers (16 bytes = 16 elements per load), is widened to
// bf16 -- exact: E4M3 has 3 mantissa bits, and the fp32 the converter returns is cut to its upper half -- and is written into
// the same swizzled LDS image the LDS-DMA of bf16 weights produces.  Same MFMAs on the same values: bit-identical results,
// half the weight bytes in HBM and on the L2 -> LDS path.
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void fp8x16_to_bf16x16(const u32x4 src, u32x4& lo, u32x4& hi) {
    unsigned o[8];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)src[d], false);   // bytes 0, 1
        const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)src[d], true);    // bytes 2, 3
        const float a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];   // (bit_cast of a vector element miscompiles: copy first)
        o[2 * d] = __builtin_amdgcn_perm(__float_as_uint(a1), __float_as_uint(a0), 0x07060302u);       // (hi16(a1) << 16) | hi16(a0)
        o[2 * d + 1] = __builtin_amdgcn_perm(__float_as_uint(b1), __float_as_uint(b0), 0x07060302u);
    }
    lo = u32x4{o[0], o[1], o[2], o[3]};
    hi = u32x4{o[4], o[5], o[6], o[7]};
}
// one thread's share of a W tile: row r, 32 consecutive k (bytes) = LDS chunks c0 .. c0 + 3 of that row
struct W8Lane {
    const unsigned char* src;   // this lane's 32 bytes of K tile 0
    unsigned lds[4];            // byte offsets of its four 16-byte chunks inside a W stage (swizzle applied)
    u32x4 r[2];
    __device__ __forceinline__ void load(int k_bytes) {
        r[0] = *reinterpret_cast<const u32x4*>(src + k_bytes);
        r[1] = *reinterpret_cast<const u32x4*>(src + k_bytes + 16);
    }
    __device__ __forceinline__ void store(char* w_stage) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            u32x4 lo, hi;
            fp8x16_to_bf16x16(r[u], lo, hi);
            *reinterpret_cast<u32x4*>(w_stage + lds[2 * u]) = lo;
            *reinterpret_cast<u32x4*>(w_stage + lds[2 * u + 1]) = hi;
        }
    }
};
__device__ __forceinline__ int swap23(int m) {  // swap bits 2 and 3
    return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1);
}


// ---- XCD-aware, grouped tile mapping.  Block b runs on XCD b%8 (private 4 MiB L2).  Each XCD owns a
// contiguous band of M-tile rows and walks it in groups of 8 rows x all N-tiles, column-major inside a
// group, so the workgroups resident on an XCD at any time cover an 8 x {8 (128^2 tiles) | 4 (256^2 tiles)} patch
// of tiles: per K-step they pull 8 A-tiles + a few W-tiles through that L2 instead of ~3 + 24 (round-1 PMC:
// 10-20x HBM over-fetch with the plain N-fastest order).
__device__ __forceinline__ bool tile_of_block(const GemmArgs& p, int& tm, int& tn) {
    const int vb = blockIdx.x;
    if (p.rows_per_xcd > 0) {
        const int xcd = vb & 7, idx = vb >> 3;
        const int m_lo = xcd * p.rows_per_xcd;
        int rows = p.tiles_m - m_lo;
        rows = rows < p.rows_per_xcd ? rows : p.rows_per_xcd;
        if (rows <= 0 || idx >= rows * p.tiles_n) return false;
        const int width = 8 * p.tiles_n;
        const int first = (idx / width) * 8;
        const int local = idx % width;
        const int gsz = (rows - first) < 8 ? (rows - first) : 8;
        tm = m_lo + first + local % gsz;
        tn = local / gsz;
    } else {
        tm = vb / p.tiles_n;
        tn = vb % p.tiles_n;
    }
    return true;
}

// ---- epilogue for one lane-owned strip: output row m, columns n0..n0+7 (fp32 math, one bf16 rounding)
template <int EPI>
__device__ __forceinline__ void epilogue8(const GemmArgs& p, int b, int m, int n0, float (&v)[8]) {
    if (p.bias) {
        const f32x4 b0 = *reinterpret_cast<const f32x4*>(p.bias + n0);
        const f32x4 b1 = *reinterpret_cast<const f32x4*>(p.bias + n0 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += b0[e];
            v[4 + e] += b1[e];
        }
    }
    if (EPI == EA_EPI_BIAS_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = gelu_tanh_f(v[e]);
    }
    if (EPI == EA_EPI_BIAS_GATE_RES) {
        const float* gb = p.gate + b * p.gbs;
        const f32x4 g0 = *reinterpret_cast<const f32x4*>(gb + n0);
        const f32x4 g1 = *reinterpret_cast<const f32x4*>(gb + n0 + 4);
        const u16x8 rr = *reinterpret_cast<const u16x8*>(p.res + b * p.rbs + (int64_t)m * p.ldres + n0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = bf16_bits_to_f32(rr[e]) + g0[e] * v[e];
            v[4 + e] = bf16_bits_to_f32(rr[4 + e]) + g1[e] * v[4 + e];
        }
    }
    if (EPI == EA_EPI_F32_OUT) {
        float* Cf = reinterpret_cast<float*>(p.C) + b * p.cbs + (int64_t)m * p.ldc + n0;
        f32x4 o0, o1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o0[e] = v[e];
            o1[e] = v[4 + e];
        }
        *reinterpret_cast<f32x4*>(Cf) = o0;
        *reinterpret_cast<f32x4*>(Cf + 4) = o1;
    } else {
        u16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = f32_to_bf16_bits(v[e]);
        *reinterpret_cast<u16x8*>(p.C + b * p.cbs + (int64_t)m * p.ldc + n0) = o;
    }
}

template <int EPI, bool W8>
__global__ __launch_bounds__(256, 2) void gemm_bf16_kernel(GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int hi = lane >> 5, l31 = lane & 31;

    int tm, tn;
    if (!tile_of_block(p, tm, tn)) return;
    const int b = blockIdx.y;
    const int row0 = tm * BM, col0 = tn * BN;

    const unsigned short* Ab = p.A + b * p.abs_;

    // ---- per-lane DMA source pointers (4 x 1 KiB pieces per wave per operand tile)
    const unsigned short* asrc[4];
    const unsigned short* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int L = (wave * 4 + i) * 64 + lane;
        const int r = L >> 3, c = L & 7;
        const int cs = c ^ ((r >> 1) & 7);
        int ra = row0 + r;
        ra = ra < p.M ? ra : p.M - 1;
        int rw = col0 + r;
        rw = rw < p.N ? rw : p.N - 1;
        asrc[i] = Ab + (int64_t)ra * p.lda + cs * 8;
        wsrc[i] = p.W + (int64_t)rw * p.K + cs * 8;
    }

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // fragment read offsets (bytes) inside a tile: row*128 + ((chunk ^ ((row>>1)&7)) * 16)
    int a_off[2], w_off[2], a_sw[2], w_sw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int ra = wm * 64 + i * 32 + l31;            // activation row = MFMA column
        const int rw = wn * 64 + i * 32 + swap23(l31);    // weight row, bit2/3 swapped (see header)
        a_off[i] = ra * 128;
        a_sw[i] = (ra >> 1) & 7;
        w_off[i] = rw * 128;
        w_sw[i] = (rw >> 1) & 7;
    }

    const int nk = p.K / BK;
    // W8: thread (row tid / 2, k half tid % 2) brings 32 fp8 weights per K tile through registers (see W8Lane)
    W8Lane w8;
    if (W8) {
        const int r = tid >> 1, h = tid & 1;
        int rw = col0 + r;
        rw = rw < p.N ? rw : p.N - 1;
        w8.src = reinterpret_cast<const unsigned char*>(p.W) + (int64_t)rw * p.K + h * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) w8.lds[c] = r * 128 + (((h * 4 + c) ^ ((r >> 1) & 7)) << 4);
    }
    auto issue = [&](int t, int stage) {
        char* sa = smem + stage * STAGE_BYTES + wave * 4096;
        char* sw = sa + TILE_BYTES;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            glds16(asrc[i] + t * BK, sa + i * 1024);
            if (!W8) glds16(wsrc[i] + t * BK, sw + i * 1024);
        }
        if (W8) w8.load(t * BK);
    };

    issue(0, 0);
    for (int t = 0; t < nk; ++t) {
        // W8: tile t's weights go to their stage now -- its last readers (tile t - 2) are behind the previous barrier
        if (W8) {
            w8.store(smem + (t & 1) * STAGE_BYTES + TILE_BYTES);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 1 < nk) issue(t + 1, (t + 1) & 1);
        const char* sa = smem + (t & 1) * STAGE_BYTES;
        const char* sw = sa + TILE_BYTES;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int ch = ks * 2 + hi;
            bf16x8 af[2], wf[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                af[i] = *reinterpret_cast<const bf16x8*>(sa + a_off[i] + ((ch ^ a_sw[i]) << 4));
                wf[i] = *reinterpret_cast<const bf16x8*>(sw + w_off[i] + ((ch ^ w_sw[i]) << 4));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[j], af[i], acc[i][j], 0, 0, 0);
        }
    }

    // ---- epilogue: lane owns row m, columns n0..n0+7 per (j, g)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = row0 + wm * 64 + i * 32 + l31;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int n0 = col0 + wn * 64 + j * 32 + g * 16 + hi * 8;
                if (n0 >= p.N) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][j][g * 8 + e];
                epilogue8<EPI>(p, b, m, n0, v);
            }
        }
    }
}


// =================================================================================================
// 256 x 256 x 64 "ping-pong" kernel for the large DiT linears (M >= a few thousand rows).
//
//   * workgroup = 512 threads = 8 waves as 2 (M) x 4 (N); wave tile 128 x 64 = 4 x 2 MFMA tiles (128 accumulator
//     registers); one workgroup per CU (128 KiB LDS: A and W tiles of 256 rows x 128 B, two stages each).
//   * a K-tile is four phases (one 16-deep k-step each): L-part {6 ds_read_b128 (4 A + 2 W fragments), a share of
//     the next tile's LDS-DMA} | s_barrier | M-part {8 MFMAs at s_setprio 1} | s_barrier.  The two wave groups
//     (wr = 0 / 1; each SIMD hosts one wave of either group) run staggered by one barrier, so on every SIMD one
//     wave's MFMAs cover the other wave's LDS reads and DMA issue (CDNA4 guide, T3/T4/T5).
//   * tile t+1 is DMA'd during phases 0 (A) and 1 (W) of tile t into the other stage and waited for (vmcnt(0),
//     1000-1500 cycles later) in phase 3 before that phase's first barrier; phase 3 also retires its own ds_reads
//     before that barrier, which is what frees the stage for the DMA issued two barriers later.
//   * same operand roles / row swizzles / epilogue as the 128^2 kernel (C^T tiles, swap-2/3 W rows, 16-byte stores).
#ifdef EA_GEMM_TIMESTAMPS
__device__ unsigned long long* g_gemm_ts = nullptr;   // diagnostic builds: per-workgroup s_memtime stamps
__device__ int g_gemm_stagger = 0;                    // diagnostic builds: the first workgroup of CU c starts ((c >> 3) & 3) * n * 8128 cycles late
#endif
constexpr int OPER2 = 256 * 128;   // one operand tile, 32 KiB
constexpr int GEMM2_LDS = 4 * OPER2;

template <int EPI>
__global__ __launch_bounds__(512, 2) void gemm256_bf16_kernel(GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const int hi = lane >> 5, l31 = lane & 31;

#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts0 = __builtin_readcyclecounter();
#endif
    int tm, tn;
    if (!tile_of_block(p, tm, tn)) return;
    const int b = blockIdx.y;
    const int row0 = tm * 256, col0 = tn * 256;
    const unsigned short* Ab = p.A + b * p.abs_;

    // ---- per-lane DMA sources: 4 x 1 KiB pieces per wave per operand tile (piece q = rows 8q..8q+7)
    const unsigned short* asrc[4];
    const unsigned short* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (wave * 4 + i) * 8 + (lane >> 3), c = lane & 7;
        const int cs = c ^ ((r >> 1) & 7);
        int ra = row0 + r;
        ra = ra < p.M ? ra : p.M - 1;
        int rw = col0 + r;
        rw = rw < p.N ? rw : p.N - 1;
        asrc[i] = Ab + (int64_t)ra * p.lda + cs * 8;
        wsrc[i] = p.W + (int64_t)rw * p.K + cs * 8;
    }
    char* const dma_a = smem + wave * 4096;               // + stage*OPER2 + i*1024
    char* const dma_w = smem + 2 * OPER2 + wave * 4096;

    f32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // ---- fragment addresses: row*128 + ((chunk ^ ((row>>1)&7)) << 4), chunk = 2*ks + hi
    const int a_row = wr * 128 + l31;
    const int w_row = wc * 64 + swap23(l31);
    const int a_sw = (l31 >> 1) & 7, w_sw = (swap23(l31) >> 1) & 7;
    const char* a_k[4];
    const char* w_k[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        a_k[ks] = smem + a_row * 128 + (((ks * 2 + hi) ^ a_sw) << 4);
        w_k[ks] = smem + 2 * OPER2 + w_row * 128 + (((ks * 2 + hi) ^ w_sw) << 4);
    }

    const int nk = p.K / BK;

#define EA_G2_PHASE(S, KS, HAS_NEXT)                                                                       \
    {                                                                                                      \
        bf16x8 af[4], wf[2];                                                                               \
        _Pragma("unroll") for (int j = 0; j < 2; ++j)                                                      \
            wf[j] = *reinterpret_cast<const bf16x8*>(w_k[KS] + (S) * OPER2 + j * 4096);                    \
        _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                      \
            af[i] = *reinterpret_cast<const bf16x8*>(a_k[KS] + (S) * OPER2 + i * 4096);                    \
        if ((KS) == 0 && (HAS_NEXT)) {                                                                     \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                \
                asrc[i] += BK;                                                                             \
                glds16(asrc[i], dma_a + ((S) ^ 1) * OPER2 + i * 1024);                                     \
            }                                                                                              \
        }                                                                                                  \
        if ((KS) == 1 && (HAS_NEXT)) {                                                                     \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                \
                wsrc[i] += BK;                                                                             \
                glds16(wsrc[i], dma_w + ((S) ^ 1) * OPER2 + i * 1024);                                     \
            }                                                                                              \
        }                                                                                                  \
        if ((KS) == 3) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                         \
        __builtin_amdgcn_sched_barrier(0);                                                                 \
        __builtin_amdgcn_s_barrier();                                                                      \
        __builtin_amdgcn_sched_barrier(0);                                                                 \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                 \
        __builtin_amdgcn_sched_barrier(0);                                                                 \
        __builtin_amdgcn_s_setprio(1);                                                                     \
        _Pragma("unroll") for (int j = 0; j < 2; ++j)                                                      \
            _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                  \
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[j], af[i], acc[i][j], 0, 0, 0);     \
        __builtin_amdgcn_s_setprio(0);                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                 \
        __builtin_amdgcn_s_barrier();                                                                      \
        __builtin_amdgcn_sched_barrier(0);                                                                 \
    }
#define EA_G2_TILE(S, HAS_NEXT)      \
    EA_G2_PHASE(S, 0, HAS_NEXT)      \
    EA_G2_PHASE(S, 1, HAS_NEXT)      \
    EA_G2_PHASE(S, 2, HAS_NEXT)      \
    EA_G2_PHASE(S, 3, HAS_NEXT)

    // ---- prologue: tile 0 -> stage 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        glds16(asrc[i], dma_a + i * 1024);
        glds16(wsrc[i], dma_w + i * 1024);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts1 = __builtin_readcyclecounter();
#endif
    if (wr == 1) __builtin_amdgcn_s_barrier();   // stagger: group 1 runs one barrier behind group 0
    __builtin_amdgcn_sched_barrier(0);

    for (int t = 0; t < nk; t += 2) {
        const bool n0_ = t + 1 < nk;
        EA_G2_TILE(0, n0_)
        if (n0_) {
            const bool n1_ = t + 2 < nk;
            EA_G2_TILE(1, n1_)
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (wr == 0) __builtin_amdgcn_s_barrier();   // balance the stagger
#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts2 = __builtin_readcyclecounter();
#endif
#undef EA_G2_TILE
#undef EA_G2_PHASE

    // ---- epilogue.  bf16 outputs go through LDS (free now: every wave is past its last operand read) so that HBM
    // sees whole 128-byte rows: in accumulator layout a store instruction covers 32 rows x 32 B (partial lines, and
    // for the gated-residual epilogue the same pattern on the residual loads); staged, it covers 8 rows x 128 B.
    // Each wave owns a private 16 KiB image of its 128 x 64 output tile (rows of 128 B, 16-byte chunks XOR-swizzled
    // with (row>>1)&7 like the operand tiles), so no workgroup barrier is needed.
    if (EPI == EA_EPI_F32_OUT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = row0 + wr * 128 + i * 32 + l31;
            if (m >= p.M) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int n0 = col0 + wc * 64 + j * 32 + g * 16 + hi * 8;
                    if (n0 >= p.N) continue;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[i][j][g * 8 + e];
                    epilogue8<EPI>(p, b, m, n0, v);
                }
            }
        }
        return;
    }
    char* const img = smem + wave * 16384;
    const int mrow0 = row0 + wr * 128, ncol0 = col0 + wc * 64;
    const int r8 = lane >> 3, c8 = lane & 7;
    if (EPI == EA_EPI_BIAS_GATE_RES) {
        // residual tile -> LDS image by LDS-DMA (source-side swizzle, rows clamped at the M tail)
        const unsigned short* Rb = p.res + b * p.rbs;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int r = q * 8 + r8;
            int m = mrow0 + r;
            m = m < p.M ? m : p.M - 1;
            int n = ncol0 + ((c8 ^ ((r >> 1) & 7)) << 3);
            n = n < p.N ? n : 0;                                   // N tail: any in-bounds address, never used
            glds16(Rb + (int64_t)m * p.ldres + n, img + q * 1024);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
    {
        const float* gb = EPI == EA_EPI_BIAS_GATE_RES ? p.gate + b * p.gbs : nullptr;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int ch = j * 4 + g * 2 + hi;          // 16-byte chunk of the wave's 64 columns
                const int n0 = ncol0 + ch * 8;
                f32x4 b0 = {0.f, 0.f, 0.f, 0.f}, b1 = b0, g0 = b0, g1 = b0;
                if (n0 >= p.N) continue;                           // N tail (N % 8 == 0): whole chunk outside
                if (p.bias) {
                    b0 = *reinterpret_cast<const f32x4*>(p.bias + n0);
                    b1 = *reinterpret_cast<const f32x4*>(p.bias + n0 + 4);
                }
                if (EPI == EA_EPI_BIAS_GATE_RES) {
                    g0 = *reinterpret_cast<const f32x4*>(gb + n0);
                    g1 = *reinterpret_cast<const f32x4*>(gb + n0 + 4);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 32 + l31;
                    char* cell = img + r * 128 + ((ch ^ ((r >> 1) & 7)) << 4);
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = acc[i][j][g * 8 + e] + b0[e];
                        v[4 + e] = acc[i][j][g * 8 + 4 + e] + b1[e];
                    }
                    if (EPI == EA_EPI_BIAS_GELU_TANH) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = gelu_tanh_f(v[e]);
                    }
                    if (EPI == EA_EPI_BIAS_GATE_RES) {
                        const u16x8 rr = *reinterpret_cast<const u16x8*>(cell);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] = bf16_bits_to_f32(rr[e]) + g0[e] * v[e];
                            v[4 + e] = bf16_bits_to_f32(rr[4 + e]) + g1[e] * v[4 + e];
                        }
                    }
                    u16x8 o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = f32_to_bf16_bits(v[e]);
                    *reinterpret_cast<u16x8*>(cell) = o;
                }
            }
        }
    }
    // the image is wave-private: the wave's own LDS accesses complete in order, no barrier
    unsigned short* Cb = p.C + b * p.cbs;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = q * 8 + r8;
        const int m = mrow0 + r;
        const u16x8 o = *reinterpret_cast<const u16x8*>(img + r * 128 + ((c8 ^ ((r >> 1) & 7)) << 4));
        if (m < p.M && ncol0 + c8 * 8 < p.N) *reinterpret_cast<u16x8*>(Cb + (int64_t)m * p.ldc + ncol0 + c8 * 8) = o;
    }
#ifdef EA_GEMM_TIMESTAMPS
    if (g_gemm_ts && tid == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        unsigned long long* d = g_gemm_ts + (size_t)(blockIdx.y * gridDim.x + blockIdx.x) * 5;
        d[0] = ts0; d[1] = ts1; d[2] = ts2; d[3] = __builtin_readcyclecounter();
        d[4] = 0;
    }
#endif
}

// =================================================================================================
// The same 256 x 256 x 64 ping-pong structure on v_mfma_f32_16x16x32_bf16.  Under the package power limit the 16x16x32
// shape sustains 14 % more than 32x32x16 on random operands (tools/ubench/mfma_power.hip: 2070 vs 1820 TFLOP/s with every
// SIMD issuing nothing else; both reach 2470 on zeros) -- the accumulator traffic per flop is half -- and the big GEMMs
// run power-limited.
//   * wave tile 128 (M) x 64 (N) = 8 x 4 MFMA tiles of 16 x 16 (128 accumulator registers, as before); C^T orientation:
//     the W fragment (16 n-rows x 32 k) is the A operand, the activation fragment (32 k x 16 m-columns) the B operand, so
//     a lane holds 4 consecutive n of one output row m = lane & 15.
//   * a fragment read is 16 rows x 4 chunks of 16 B (row = lane & 15, chunk = 4 * kstep + lane / 16): the LDS rows are
//     XOR-swizzled with row & 7 (eight consecutive rows hit eight different 16-byte columns); the LDS-DMA applies the
//     swizzle on the source address as before.
//   * a K-tile is four phases: (k32 step, M half).  The first phase of a step reads the four W fragments (kept for the
//     second) and four A fragments, the second four A fragments; 16 MFMAs (256 cycles) per phase as with 8 x 32x32x16.
//   * epilogue through the wave-private LDS image (8-byte writes in accumulator layout, 16-byte row-wise read-out).
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));

#define EA_G3_PHASE(S, P, HAS_NEXT, HAS_NEXT2, SWAP, W8)                                                      \
    {                                                                                                         \
        bf16x8 af[4];                                                                                         \
        if (((P) & 1) == 0) {                                                                                 \
            _Pragma("unroll") for (int j = 0; j < 4; ++j)                                                     \
                wf[j] = *reinterpret_cast<const bf16x8*>(smem + (w_k[(P) >> 1] + (S) * OPER2 + j * 2048));    \
        }                                                                                                     \
        _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                         \
            af[i] = *reinterpret_cast<const bf16x8*>(smem + (a_k[(P) >> 1] + (S) * OPER2 + (((P) & 1) * 4 + i) * 2048)); \
        if ((P) == 0 && (HAS_NEXT)) {                                                                         \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                   \
                asrc[i] += a_kst;                                                                             \
                glds16(asrc[i], dma_a + ((S) ^ 1) * OPER2 + i * 1024);                                        \
            }                                                                                                 \
        }                                                                                                     \
        if ((P) == 1 && (HAS_NEXT) && !(W8)) {                                                                \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                   \
                wsrc[i] += w_kst;                                                                             \
                glds16(wsrc[i], dma_w + ((S) ^ 1) * OPER2 + i * 1024);                                        \
            }                                                                                                 \
        }                                                                                                     \
        if ((P) == 2 && (HAS_NEXT) && (W8)) {                                                                 \
            /* fp8 weights: tile t + 1 (in registers since the previous tile) is widened and written to its   \
               stage -- phase 3 waits for these stores; then tile t + 2 is requested into the same registers  \
               and stays in flight across phase 3 (vmcnt(2): the A pieces were issued first) */              \
            w8.store(smem + 2 * OPER2 + ((S) ^ 1) * OPER2);                                                   \
            if (HAS_NEXT2) {                                                                                  \
                w8k += BK;                                                                                    \
                w8.load(w8k);                                                                                 \
            }                                                                                                 \
        }                                                                                                     \
        if ((P) == 3) {                                                                                       \
            if ((W8) && (HAS_NEXT2)) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)" ::: "memory");              \
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                                  \
        }                                                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                    \
        __builtin_amdgcn_s_barrier();                                                                         \
        __builtin_amdgcn_sched_barrier(0);                                                                    \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                    \
        __builtin_amdgcn_sched_barrier(0);                                                                    \
        __builtin_amdgcn_s_setprio(1);                                                                        \
        _Pragma("unroll") for (int j = 0; j < 4; ++j)                                                         \
            _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                     \
                acc[((P) & 1) * 4 + i][j] = (SWAP)                                                            \
                    ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[i], wf[j], acc[((P) & 1) * 4 + i][j], 0, 0, 0) \
                    : __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j], af[i], acc[((P) & 1) * 4 + i][j], 0, 0, 0); \
        __builtin_amdgcn_s_setprio(0);                                                                        \
        __builtin_amdgcn_sched_barrier(0);                                                                    \
        __builtin_amdgcn_s_barrier();                                                                         \
        __builtin_amdgcn_sched_barrier(0);                                                                    \
    }
#define EA_G3_TILE(S, HAS_NEXT, HAS_NEXT2, SWAP, W8) \
    EA_G3_PHASE(S, 0, HAS_NEXT, HAS_NEXT2, SWAP, W8) \
    EA_G3_PHASE(S, 1, HAS_NEXT, HAS_NEXT2, SWAP, W8) \
    EA_G3_PHASE(S, 2, HAS_NEXT, HAS_NEXT2, SWAP, W8) \
    EA_G3_PHASE(S, 3, HAS_NEXT, HAS_NEXT2, SWAP, W8)
// prologue DMA of tile 0, the staggered start of the two wave groups, the K loop, and the balancing barrier.
// SWAP = 1 exchanges the MFMA operand roles (activation fragment as A, weight fragment as B): the accumulator tile is
// then the transpose -- a lane holds 4 consecutive output ROWS of one column (the fused QKV kernel's V^T tiles).
// W8 = the fp8-weight variant (needs `W8Lane w8`, set up by the kernel): W tiles through registers instead of LDS-DMA.
#define EA_G3_STAMP1
#define EA_G3_MAINLOOP(SWAP, W8)                                                                \
    {                                                                                           \
        int w8k = 0;                                                                            \
        _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                         \
            glds16(asrc[i], dma_a + i * 1024);                                                  \
            if (!(W8)) glds16(wsrc[i], dma_w + i * 1024);                                       \
        }                                                                                       \
        if (W8) {   /* tile 0 to its stage; tile 1 stays in the registers until phase 2 of tile 0 */     \
            w8.load(0);                                                                         \
            w8.store(smem + 2 * OPER2);                                                         \
            if (nk > 1) {                                                                       \
                w8k = BK;                                                                       \
                w8.load(BK);                                                                    \
            }                                                                                   \
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                  \
        }                                                                                       \
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                        \
        __builtin_amdgcn_s_barrier();                                                           \
        __builtin_amdgcn_sched_barrier(0);                                                      \
        EA_G3_STAMP1                                                                            \
        if (wr == 1) __builtin_amdgcn_s_barrier(); /* stagger: group 1 runs one barrier behind group 0 */ \
        __builtin_amdgcn_sched_barrier(0);                                                      \
        for (int t = 0; t < nk; t += 2) {                                                       \
            const bool n0_ = t + 1 < nk;                                                        \
            const bool n1_ = t + 2 < nk;                                                        \
            EA_G3_TILE(0, n0_, n1_, SWAP, W8)                                                   \
            if (n0_) {                                                                          \
                const bool n2_ = t + 3 < nk;                                                    \
                EA_G3_TILE(1, n1_, n2_, SWAP, W8)                                               \
            }                                                                                   \
        }                                                                                       \
        __builtin_amdgcn_sched_barrier(0);                                                      \
        if (wr == 0) __builtin_amdgcn_s_barrier(); /* balance the stagger */                    \
    }

// ---- epilogue of ONE wave tile (128 output rows x 64 columns, acc[i][j]: MFMA tile (row block i, column block j), C^T
// orientation: a lane holds 4 consecutive columns of row lr) through the wave-private 16 KiB LDS image `img` (rows = the wave's
// 128 output rows, 128 B = its 64 columns, 16-byte chunks XOR-swizzled with (row >> 1) & 7: the layout the residual LDS-DMA and
// the read-out use).  p.c_kstep != 0 writes the tile K-blocked (one [rows][64] block of the next GEMM's A operand).
// Round 5 (profiles/r05p_gemm_anatomy_w4a_vs_w4p.jsonl: the epilogue was 11-17 % of a K = 3072 tile, most of it exposed latency): nothing in
// here waits for a global load it issued itself.  The lane's bias / gate vectors are loaded by gemm_load_bias_gate -- by the four-wave
// kernel BEFORE its main loop --, the residual rows are requested by gemm_residual_request (four-wave kernel: both halves into two
// images before the first accumulator is read out), and the image is read out in one batch before the stores go.
template <int EPI>
__device__ __forceinline__ void gemm_load_bias_gate(const GemmArgs& p, const int b, const int ncol0, const int lane, f32x4_t* const bv,
                                                    f32x4_t* const gv) {
    const int lq = lane >> 4;
    const float* gb = EPI == EA_EPI_BIAS_GATE_RES ? p.gate + b * p.gbs : nullptr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        int n0 = ncol0 + j * 16 + lq * 4;                 // this lane's 4 columns of MFMA tile column j
        n0 = n0 < p.N ? n0 : 0;                           // N tail: any in-bounds address, never used
        bv[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        gv[j] = bv[j];
        if (p.bias) bv[j] = *reinterpret_cast<const f32x4_t*>(p.bias + n0);
        if (EPI == EA_EPI_BIAS_GATE_RES) gv[j] = *reinterpret_cast<const f32x4_t*>(gb + n0);
    }
}

// residual rows of the wave tile -> image (LDS-DMA, 16 x 1 KiB); the caller waits (vmcnt) before the epilogue reads the image
__device__ __forceinline__ void gemm_residual_request(const GemmArgs& p, const int b, char* const img, const int mrow0, const int ncol0,
                                                      const int lane) {
    const int r8 = lane >> 3, c8 = lane & 7;
    const unsigned short* Rb = p.res + b * p.rbs;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = q * 8 + r8;
        int m = mrow0 + r;
        m = m < p.M ? m : p.M - 1;
        int n = ncol0 + ((c8 ^ ((r >> 1) & 7)) << 3);
        n = n < p.N ? n : 0;                                   // N tail: any in-bounds address, never used
        glds16(Rb + (int64_t)m * p.ldres + n, img + q * 1024);
    }
}

// RES_READY: the residual rows are already in the image (requested and waited for by the caller)
template <int EPI, bool RES_READY = false>
__device__ __forceinline__ void gemm_wave_epilogue(const GemmArgs& p, int b, f32x4_t (&acc)[8][4], char* const img, const int mrow0,
                                                   const int ncol0, const int lane, const f32x4_t* const bv, const f32x4_t* const gv) {
    const int lr = lane & 15, lq = lane >> 4;
    const int r8 = lane >> 3, c8 = lane & 7;
    if (EPI == EA_EPI_BIAS_GATE_RES && !RES_READY) {
        gemm_residual_request(p, b, img, mrow0, ncol0, lane);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n0 = ncol0 + j * 16 + lq * 4;          // this lane's 4 columns of MFMA tile column j
        if (n0 >= p.N) continue;                          // N tail (N % 8 == 0, lq*4 pairs stay inside a chunk of 8)
        const int ch = j * 2 + (lq >> 1);                 // 16-byte chunk of the row, 8-byte half lq & 1
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 16 + lr;
            char* cell = img + r * 128 + ((ch ^ ((r >> 1) & 7)) << 4) + (lq & 1) * 8;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] + bv[j][e];
            if (EPI == EA_EPI_BIAS_GELU_TANH) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
            }
            if (EPI == EA_EPI_BIAS_GATE_RES) {
                const u16x4 rr = *reinterpret_cast<const u16x4*>(cell);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(gv[j][e], v[e], bf16_bits_to_f32(rr[e]));
            }
            u16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16_bits(v[e]);
            *reinterpret_cast<u16x4*>(cell) = o;
        }
    }
    unsigned short* Cb = p.C + b * p.cbs;
    u16x8 o[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = q * 8 + r8;
        o[q] = *reinterpret_cast<const u16x8*>(img + r * 128 + ((c8 ^ ((r >> 1) & 7)) << 4));
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int m = mrow0 + q * 8 + r8;
        // (K-blocked C: the wave's 64 columns are one [rows][64] block of the next GEMM's A operand -- 128 rows x 128 B, contiguous)
        unsigned short* const crow = p.c_kstep ? Cb + (int64_t)(ncol0 >> 6) * p.c_kstep + (int64_t)m * 64 + c8 * 8
                                               : Cb + (int64_t)m * p.ldc + ncol0 + c8 * 8;
        // streaming stores: C is far larger than the L2 and is not read again by this kernel -- written with the default policy it
        // pushes operand tiles out of the L2 under the main loops of the other CUs (FFN-up at config 3: 1377 -> 1427 TFLOP/s,
        // out-proj 1309 -> 1347, profiles/r05q_gemm_nt_stores_ab.txt)
        if (m < p.M && ncol0 + c8 * 8 < p.N) __builtin_nontemporal_store(o[q], reinterpret_cast<u16x8*>(crow));
    }
}

template <int EPI, bool W8>
__global__ __launch_bounds__(512, 2) void gemm256_mi16_kernel(GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const int lr = lane & 15, lq = lane >> 4;
#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts0 = __builtin_readcyclecounter();
    unsigned long long ts1 = 0;
#endif

    int tm, tn;
    if (!tile_of_block(p, tm, tn)) return;
    const int b = blockIdx.y;
    const int row0 = tm * 256, col0 = tn * 256;
    const unsigned short* Ab = p.A + b * p.abs_;

    const unsigned short* asrc[4];
    const unsigned short* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (wave * 4 + i) * 8 + (lane >> 3), c = lane & 7;
        const int cs = c ^ (r & 7);
        int ra = row0 + r;
        ra = ra < p.M ? ra : p.M - 1;
        int rw = col0 + r;
        rw = rw < p.N ? rw : p.N - 1;
        asrc[i] = Ab + (int64_t)ra * p.lda + cs * 8;
        wsrc[i] = p.W + (int64_t)rw * p.ldw + cs * 8;
    }
    const int64_t a_kst = p.a_kstep, w_kst = p.w_kstep;      // elements to the next K tile (64 row-major; rows * 64 K-blocked)
    char* const dma_a = smem + wave * 4096;
    char* const dma_w = smem + 2 * OPER2 + wave * 4096;

    f32x4_t acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.f;

    // fragment byte offsets: row * 128 + ((chunk ^ (row & 7)) << 4), chunk = 4 * ks2 + lq; + 2048 per 16-row MFMA tile
    unsigned a_k[2], w_k[2];
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
        a_k[ks2] = (wr * 128 + lr) * 128 + (((ks2 * 4 + lq) ^ (lr & 7)) << 4);
        w_k[ks2] = 2 * OPER2 + (wc * 64 + lr) * 128 + (((ks2 * 4 + lq) ^ (lr & 7)) << 4);
    }
    const int nk = p.K / BK;
    bf16x8 wf[4];
    W8Lane w8;
    if (W8) {   // thread (row tid / 2, k half tid % 2): 32 fp8 weights per K tile
        const int r = tid >> 1, h = tid & 1;
        int rw = col0 + r;
        rw = rw < p.N ? rw : p.N - 1;
        w8.src = reinterpret_cast<const unsigned char*>(p.W) + (int64_t)rw * p.K + h * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) w8.lds[c] = r * 128 + (((h * 4 + c) ^ (r & 7)) << 4);
    }

#ifdef EA_GEMM_TIMESTAMPS
#undef EA_G3_STAMP1
#define EA_G3_STAMP1 ts1 = __builtin_readcyclecounter();
#endif
    EA_G3_MAINLOOP(0, W8)
#ifdef EA_GEMM_TIMESTAMPS
#undef EA_G3_STAMP1
#define EA_G3_STAMP1
    const unsigned long long ts2 = __builtin_readcyclecounter();
#endif

    // ---- epilogue through the wave-private 16 KiB image (rows = the wave's 128 output rows, 128 B = its 64 columns,
    // 16-byte chunks XOR-swizzled with (row >> 1) & 7: the layout the residual LDS-DMA and the read-out already use)
    char* const img = smem + wave * 16384;
    const int mrow0 = row0 + wr * 128, ncol0 = col0 + wc * 64;
    f32x4_t bv[4], gv[4];
    gemm_load_bias_gate<EPI>(p, b, ncol0, lane, bv, gv);       // one batch of loads, in flight under the residual request
    gemm_wave_epilogue<EPI>(p, b, acc, img, mrow0, ncol0, lane, bv, gv);
#ifdef EA_GEMM_TIMESTAMPS
    if (g_gemm_ts && tid == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        unsigned long long* d = g_gemm_ts + (size_t)(blockIdx.y * gridDim.x + blockIdx.x) * 5;
        d[0] = ts0; d[1] = ts1; d[2] = ts2; d[3] = __builtin_readcyclecounter();
        d[4] = 0;
    }
#endif
}

// =================================================================================================
// 256 x 256 x 64 tiles with FOUR waves, one per SIMD, 128 x 128 wave tiles (8 x 8 MFMA tiles of 16x16x32 = 256 accumulator
// registers = the whole AGPR file), main loop placed by hand as ONE inline-asm block (round 5; generated by
// tools/gen_gemm_w4_asm.py into ea_gemm_w4_loop.inc -- the rules of its order stand there).  The same wave shape in fenced C++ was
// 3..8 % behind the eight-wave kernel: the compiled loop carried eight conditional branches per K tile around the DMA requests and
// compiler-placed waits.  Here: no branch inside a K tile (requests past the last tile go through an empty buffer resource), one
// barrier per operand hand-over (4 per K tile), 0.25 ds_read_b128 per MFMA.  FFN-up / FFN-down / out-projection of the 12B model at
// 2 x 53248 tokens: 1423 / 1485 / 1334 TFLOP/s.
// Same LDS layout / swizzle / DMA source addressing / C^T orientation / epilogue image as gemm256_mi16_kernel: the same
// products in another summation order over k (fp32 accumulation per 32 k, as there).
#include "ea_gemm_w4_loop.inc"

template <int EPI>
__global__ __launch_bounds__(256) void gemm256_w4a_kernel(GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    const int lr = lane & 15, lq = lane >> 4;

#ifdef EA_GEMM_TIMESTAMPS
    if (g_gemm_stagger && blockIdx.x < 256 && blockIdx.y == 0) {
        const int n = ((blockIdx.x >> 3) & 3) * g_gemm_stagger;
        for (int i = 0; i < n; ++i) __builtin_amdgcn_s_sleep(127);
    }
    const unsigned long long ts0 = __builtin_readcyclecounter();
#endif
    int tm, tn;
    if (!tile_of_block(p, tm, tn)) return;
    const int b = blockIdx.y;
    const int row0 = tm * 256, col0 = tn * 256;
    const unsigned short* Ab = p.A + b * p.abs_;
    const int nk = p.K / BK;

    // DMA pieces: a K tile of an operand is 256 rows x 128 bytes = 32 pieces of 1 KiB; wave w stages pieces 8w .. 8w+7.  Buffer
    // addressing: per-lane byte offsets relative to the tile's first row (fixed for the kernel), the K tile is the scalar offset.
    int aoff[8], woff[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = (wave * 8 + i) * 8 + (lane >> 3), c = lane & 7;
        const int cs = c ^ (r & 7);
        const int ra = (row0 + r < p.M ? row0 + r : p.M - 1) - row0;
        const int rw = (col0 + r < p.N ? col0 + r : p.N - 1) - col0;
        aoff[i] = (int)((int64_t)ra * p.lda * 2) + cs * 16;
        woff[i] = (int)((int64_t)rw * p.ldw * 2) + cs * 16;
    }
    const unsigned short* Abase = Ab + (int64_t)row0 * p.lda;
    const unsigned short* Wbase = p.W + (int64_t)col0 * p.ldw;
    const int a_rows = p.M - row0 < 256 ? p.M - row0 : 256, w_rows = p.N - col0 < 256 ? p.N - col0 : 256;
    // bytes reachable from Abase / Wbase (host-checked to fit 32 bits)
    const unsigned a_ext = (unsigned)((((int64_t)nk - 1) * p.a_kstep + ((int64_t)a_rows - 1) * p.lda + BK) * 2);
    const unsigned w_ext = (unsigned)((((int64_t)nk - 1) * p.w_kstep + ((int64_t)w_rows - 1) * p.ldw + BK) * 2);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    // fragment byte addresses of k-step 0: row * 128 + ((chunk ^ (row & 7)) << 4), chunk = lq; + 2048 per 16-row MFMA tile
    const unsigned ak0 = lds0 + (wr * 128 + lr) * 128 + ((lq ^ (lr & 7)) << 4);
    const unsigned wk0 = lds0 + 2 * OPER2 + (wc * 128 + lr) * 128 + ((lq ^ (lr & 7)) << 4);
    const unsigned lds_a = __builtin_amdgcn_readfirstlane(lds0 + wave * 8192);
    const unsigned lds_w = __builtin_amdgcn_readfirstlane(lds0 + 2 * OPER2 + wave * 8192);
    const unsigned a_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)Abase);
    const unsigned a_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)Abase >> 32));
    const unsigned w_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)Wbase);
    const unsigned w_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)Wbase >> 32));
    const unsigned a_kst = __builtin_amdgcn_readfirstlane((unsigned)(p.a_kstep * 2));
    const unsigned w_kst = __builtin_amdgcn_readfirstlane((unsigned)(p.w_kstep * 2));
    const unsigned a_ext_s = __builtin_amdgcn_readfirstlane(a_ext), w_ext_s = __builtin_amdgcn_readfirstlane(w_ext);
    const unsigned nk_s = __builtin_amdgcn_readfirstlane((unsigned)nk);
    // the lane's bias / gate vectors (4 columns in each of its 8 column blocks) are fetched by the main asm itself, in front of the first
    // operand request, into registers it returns as outputs: landed long before the epilogue asks for them (EA_W4A_MAINLOOP_ASM_BG)
    const float* const bptr = p.bias ? p.bias + col0 : nullptr;
    const float* const gptr = EPI == EA_EPI_BIAS_GATE_RES ? p.gate + b * p.gbs + col0 : nullptr;
    const unsigned bg_bytes = p.N - col0 > 0 ? (unsigned)(p.N - col0) * 4u : 0u;                  // columns past N read as zeros
    const unsigned b_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)bptr);
    const unsigned b_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)bptr >> 32));
    const unsigned b_ext = __builtin_amdgcn_readfirstlane(bptr ? bg_bytes : 0u);
    const unsigned g_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)gptr);
    const unsigned g_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)gptr >> 32));
    const unsigned g_ext = __builtin_amdgcn_readfirstlane(gptr ? bg_bytes : 0u);
    const int boff = (wc * 128 + lq * 4) * 4;
    f32x4_t bias_v[8], gate_v[8];
#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts1 = __builtin_readcyclecounter();
#endif

    f32x4_t accq[64];      // the 256 accumulators a0..a255, as the main asm's outputs: live until the read-outs consume them
    asm volatile(EA_W4A_MAINLOOP_ASM_BG
                 : EA_W4A_BG_OUTPUTS(bias_v, gate_v), EA_W4A_ACC_OUTPUTS(accq)
                 : [boff] "v"(boff), [b_lo] "s"(b_lo), [b_hi] "s"(b_hi), [b_ext] "s"(b_ext), [g_lo] "s"(g_lo), [g_hi] "s"(g_hi), [g_ext] "s"(g_ext),
                   [wk0] "v"(wk0), [ak0] "v"(ak0),
                   [aoff0] "v"(aoff[0]), [aoff1] "v"(aoff[1]), [aoff2] "v"(aoff[2]), [aoff3] "v"(aoff[3]),
                   [aoff4] "v"(aoff[4]), [aoff5] "v"(aoff[5]), [aoff6] "v"(aoff[6]), [aoff7] "v"(aoff[7]),
                   [woff0] "v"(woff[0]), [woff1] "v"(woff[1]), [woff2] "v"(woff[2]), [woff3] "v"(woff[3]),
                   [woff4] "v"(woff[4]), [woff5] "v"(woff[5]), [woff6] "v"(woff[6]), [woff7] "v"(woff[7]),
                   [a_lo] "s"(a_lo), [a_hi] "s"(a_hi), [a_ext] "s"(a_ext_s), [w_lo] "s"(w_lo), [w_hi] "s"(w_hi), [w_ext] "s"(w_ext_s),
                   [a_kst] "s"(a_kst), [w_kst] "s"(w_kst), [nk] "s"(nk_s), [lds_w] "s"(lds_w), [lds_a] "s"(lds_a)
                 : EA_W4A_CLOBBERS);
#ifdef EA_GEMM_TIMESTAMPS
    const unsigned long long ts2 = __builtin_readcyclecounter();
#endif
    __builtin_amdgcn_s_barrier();   // every wave's requests have landed and its fragment reads are done: the LDS becomes the epilogue images

    // ---- epilogue: the wave's 128 x 128 tile as two 128 x 64 halves, each through its own private 16 KiB image (the four waves share
    // 128 KiB), gemm256_mi16_kernel's code.  Both halves' residual rows are requested before the first accumulator is read out and
    // waited for once, in front of the first store: no wait in here ever covers a store.
    char* const img0 = smem + wave * 32768;
    char* const img1 = img0 + 16384;
    const int mrow0 = row0 + wr * 128;
    if (EPI == EA_EPI_BIAS_GATE_RES) {
        gemm_residual_request(p, b, img0, mrow0, col0 + wc * 128, lane);
        gemm_residual_request(p, b, img1, mrow0, col0 + wc * 128 + 64, lane);
    }
    f32x4_t acc[8][4];
    EA_W4A_READ_HALF0(acc, accq)
    if (EPI == EA_EPI_BIAS_GATE_RES) {
        // vmcnt(0) as the BUILTIN, so that the compiler's own wait bookkeeping sees it (an asm wait would leave it to place its
        // own in front of the image reads -- inside the per-column branches, and again in the middle of the stores)
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __builtin_amdgcn_sched_barrier(0);
    }
    gemm_wave_epilogue<EPI, true>(p, b, acc, img0, mrow0, col0 + wc * 128, lane, bias_v, gate_v);
    EA_W4A_READ_HALF1(acc, accq)
    gemm_wave_epilogue<EPI, true>(p, b, acc, img1, mrow0, col0 + wc * 128 + 64, lane, bias_v + 4, gate_v + 4);
#ifdef EA_GEMM_TIMESTAMPS
    if (g_gemm_ts && tid == 0) {
        const unsigned long long ts3 = __builtin_readcyclecounter();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        unsigned long long* d = g_gemm_ts + (size_t)(blockIdx.y * gridDim.x + blockIdx.x) * 5;
        d[0] = ts0; d[1] = ts1; d[2] = ts2; d[3] = ts3;
        d[4] = __builtin_readcyclecounter();
    }
#endif
}

#include "ea_gemm_mxfp4_w4.inc"

// =================================================================================================
// Fused QKV projection: ONE launch computes q, k, v = Linear_{q,k,v}(x) for a token stream and finishes each
// (128 tokens x one head) wave tile in its epilogue -- bias, qk-LayerNorm(64), interleaved RoPE, softmax scale on q,
// head-major scatter of q / k rows, transposed scatter of v -- i.e. processor.py:244-285 without the [B,n,3d] QKV
// round trip through HBM (1 write + 1 read of 6d bytes per token) and with the activations read once instead of three
// times.  The weights stay three separate [d,d] checkpoint tensors: the N axis of the launch is the concatenation
// q | k | v and an N-tile picks its weight pointer (d % 256 == 0, so a tile never straddles two weights).
//   * main loop = gemm256_mi16_kernel's.  A wave tile is 128 tokens x 64 output features = exactly one head.
//   * q / k tiles: C^T orientation as before (a lane holds 4 consecutive features of one token).  The epilogue rounds
//     acc + bias to bf16 (the value the unfused path stores in the QKV buffer), reduces mean / centred variance over the
//     64 features of a token (16 in the lane, then the 4 lanes lq = 0..3 that share the token: two xor-shuffles),
//     rounds the LayerNorm output to bf16 (processor.py:255-258), rotates the interleaved pairs with the fp32 cos / sin
//     rows of the token, multiplies q by q_scale, rounds once, and leaves through the wave-private LDS image as whole
//     128-byte rows of q_out / k_out [B, H, s_pad, 64].  Same roundings, same order as ea_gemm_bf16 followed by
//     ea_qknorm_rope_bf16 (tested: V^T bit-identical, q / k within one bf16 ulp -- the statistics are summed in another order).
//   * v tiles: the MFMA operand roles are swapped (EA_G3_MAINLOOP(1)), so a lane holds 4 consecutive TOKENS of one
//     feature; the image is written transposed ([64 features][128 tokens], 16-byte chunks XOR-swizzled with
//     feature & 15) and read out as 256-byte rows of vt_out [B, H, 64, s_pad].
struct QkvArgs {
    const unsigned short* A;
    const unsigned short* W[3];
    const float* bias[3];
    unsigned short* q_out;
    unsigned short* k_out;
    unsigned short* vt_out;
    const float* nw[2];   // norm_q / norm_k weight
    const float* nb[2];   // norm_q / norm_k bias
    const float* cosT;
    const float* sinT;
    int M, K, inner, heads, seq_off, s_pad;
    int kv_off, kv_rows;   // geometry of k_out / vt_out (rows per head, first row): equal to (seq_off, s_pad) unless the caller
                           // lets K / V^T land in another buffer (sequence parallelism: the rank's slot of the exchange buffer)
    int first_part;        // the launch's N axis starts at this third (0 = q | k | v, 1 = k | v): which = first_part + tn / tiles_per_w
    int kv_gheads;         // K / V^T destination in head GROUPS (sequence parallelism exchanging one head group at a time): head h of batch b
    int64_t kv_gstride;    // lands in group h / kv_gheads at k_out + group * kv_gstride + ((b * kv_gheads + h % kv_gheads) * kv_rows ..) * 64
                           // (kv_gheads == heads, kv_gstride == 0: one [batch, heads, kv_rows, 64] buffer)
    int64_t lda, abs_;
    float eps, q_scale;
    int tiles_m, tiles_n, rows_per_xcd;
};

// ---- the per-head epilogues of the fused QKV projection (one 128-token x 64-feature accumulator tile = one head), shared by
// gemm256_qkv_kernel (eight waves: one head per wave tile) and gemm256_qkv_w4a_kernel (four waves: two heads per wave tile)
// element offset of (batch b, head) inside the K / V^T destination (see QkvArgs::kv_gheads)
__device__ __forceinline__ int64_t qkv_kv_base(const QkvArgs& q, const int b, const int head) {
    const int g = head / q.kv_gheads;
    return (int64_t)g * q.kv_gstride + ((int64_t)b * q.kv_gheads + (head - g * q.kv_gheads)) * q.kv_rows * 64;
}

__device__ __forceinline__ void qkv_epilogue_v(const QkvArgs& q, f32x4_t (&acc)[8][4], char* const img, const float* biasb, const int feat0,
                                               const int tok0, const int64_t kvbase, const int Mv, const int lane) {
#pragma clang fp contract(off)
    const int lr = lane & 15, lq = lane >> 4;
    // lane holds tokens i*16 + 4*lq + 0..3 of feature j*16 + lr  ->  image^T [feature][token]
    float bv4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bv4[j] = biasb ? biasb[feat0 + j * 16 + lr] : 0.f;      // one batch of loads: one round trip, not four
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = j * 16 + lr;
        const float bv = bv4[j];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            u16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16_bits(acc[i][j][e] + bv);
            const int ch = i * 2 + (lq >> 1);
            *reinterpret_cast<u16x4*>(img + n * 256 + ((ch ^ (n & 15)) << 4) + (lq & 1) * 8) = o;
        }
    }
    const int r4 = lane >> 4, c16 = lane & 15;
    unsigned short* dst = q.vt_out + kvbase + q.kv_off + tok0 + c16 * 8;
    const int nv = Mv - (tok0 + c16 * 8);       // valid tokens among this lane's eight (ragged last M tile: < 8)
    if (nv >= 8) {
#pragma unroll
        for (int qq = 0; qq < 16; ++qq) {
            const int n = qq * 4 + r4;
            const u16x8 o = *reinterpret_cast<const u16x8*>(img + n * 256 + ((c16 ^ (n & 15)) << 4));
            __builtin_nontemporal_store(o, reinterpret_cast<u16x8*>(dst + (int64_t)n * q.kv_rows));   // streaming, as in gemm_wave_epilogue
        }
    } else if (nv > 0) {   // the one straddling group of a row: element stores, nothing past column kv_off + M is written
        for (int qq = 0; qq < 16; ++qq) {
            const int n = qq * 4 + r4;
            const unsigned short* src = reinterpret_cast<const unsigned short*>(img + n * 256 + ((c16 ^ (n & 15)) << 4));
            for (int e = 0; e < nv; ++e) dst[(int64_t)n * q.kv_rows + e] = src[e];
        }
    }
}

__device__ __forceinline__ void qkv_epilogue_qk(const QkvArgs& q, f32x4_t (&acc)[8][4], char* const img, const float* biasb, const int feat0,
                                                const int tok0, const int64_t bh, const int64_t kvbase, const int which, const int Mv,
                                                const int lane_e) {
    // no FMA contraction in here: three kernels (eight-wave bf16 / fp8 weights, four-wave) inline this body, and the LayerNorm / RoPE
    // arithmetic has to round identically in all of them (with contraction left to the compiler a handful of q / k values per
    // million landed on neighbouring bf16 numbers -- first GPU run of the four-wave kernel)
#pragma clang fp contract(off)
    const int lr_e = lane_e & 15, lq_e = lane_e >> 4;
    // lane_e holds features j*16 + lq_e*4 + 0..3 of token i*16 + lr_e
    const float* gw = q.nw[which];
    const float* gb = q.nb[which];
    f32x4_t bias4[4], gw4[4], gb4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = j * 16 + lq_e * 4;
        f32x4_t z = {0.f, 0.f, 0.f, 0.f};
        bias4[j] = biasb ? *reinterpret_cast<const f32x4_t*>(biasb + feat0 + n) : z;
        gw4[j] = *reinterpret_cast<const f32x4_t*>(gw + n);
        gb4[j] = *reinterpret_cast<const f32x4_t*>(gb + n);
    }
    const float osc = which == 0 ? q.q_scale : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 16 + lr_e;
        f32x4_t c4[4], s4[4];
        if (q.cosT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t tr = (int64_t)(tok0 + r < Mv ? tok0 + r : Mv - 1) * 64 + j * 16 + lq_e * 4;
                c4[j] = *reinterpret_cast<const f32x4_t*>(q.cosT + tr);
                s4[j] = *reinterpret_cast<const f32x4_t*>(q.sinT + tr);
            }
        }
        float v[4][4];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[j][e] = bf16_bits_to_f32(f32_to_bf16_bits(acc[i][j][e] + bias4[j][e]));   // the stored QKV value
                s += v[j][e];
            }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        const float mean = s * (1.0f / 64.0f);
        float qd = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = v[j][e] - mean;
                qd += d * d;
            }
        qd += __shfl_xor(qd, 16, 64);
        qd += __shfl_xor(qd, 32, 64);
        const float rstd = rsqrtf(qd * (1.0f / 64.0f) + q.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[j][e] = bf16_bits_to_f32(f32_to_bf16_bits((v[j][e] - mean) * rstd * gw4[j][e] + gb4[j][e]));
            u16x4 o;
            if (q.cosT) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float x0 = v[j][e], x1 = v[j][e + 1];
                    o[e] = f32_to_bf16_bits((x0 * c4[j][e] - x1 * s4[j][e]) * osc);
                    o[e + 1] = f32_to_bf16_bits((x1 * c4[j][e + 1] + x0 * s4[j][e + 1]) * osc);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16_bits(v[j][e] * osc);
            }
            const int ch = j * 2 + (lq_e >> 1);
            *reinterpret_cast<u16x4*>(img + r * 128 + ((ch ^ ((r >> 1) & 7)) << 4) + (lq_e & 1) * 8) = o;
        }
    }
    const int r8 = lane_e >> 3, c8 = lane_e & 7;
    unsigned short* dst = (which ? q.k_out + kvbase + (int64_t)(q.kv_off + tok0) * 64
                                 : q.q_out + (bh * q.s_pad + q.seq_off + tok0) * 64) + c8 * 8;
#pragma unroll
    for (int qq = 0; qq < 16; ++qq) {
        const int r = qq * 8 + r8;
        const u16x8 o = *reinterpret_cast<const u16x8*>(img + r * 128 + ((c8 ^ ((r >> 1) & 7)) << 4));
        if (tok0 + r < Mv) __builtin_nontemporal_store(o, reinterpret_cast<u16x8*>(dst + (int64_t)r * 64));
    }
}

template <bool W8>
__global__ __launch_bounds__(512, 2) void gemm256_qkv_kernel(QkvArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const int lr = lane & 15, lq = lane >> 4;

    int tm, tn;
    {
        GemmArgs g;
        g.tiles_m = q.tiles_m; g.tiles_n = q.tiles_n; g.rows_per_xcd = q.rows_per_xcd;
        if (!tile_of_block(g, tm, tn)) return;
    }
    const int b = blockIdx.y;
    const int row0 = tm * 256;
    const int tiles_per_w = q.inner >> 8;
    const int part = __builtin_amdgcn_readfirstlane(tn / tiles_per_w);
    const int which = q.first_part + part;                                 // 0 = q, 1 = k, 2 = v
    const int col0 = (tn - part * tiles_per_w) * 256;                      // first output feature inside that weight
    const unsigned short* Ab = q.A + b * q.abs_;
    const unsigned short* Wb = which == 0 ? q.W[0] : (which == 1 ? q.W[1] : q.W[2]);
    const float* biasb = which == 0 ? q.bias[0] : (which == 1 ? q.bias[1] : q.bias[2]);

    const unsigned short* asrc[4];
    const unsigned short* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (wave * 4 + i) * 8 + (lane >> 3), c = lane & 7;
        const int cs = c ^ (r & 7);
        const int ra = row0 + r < q.M ? row0 + r : q.M - 1;       // ragged last M tile: rows past M re-read row M - 1
        asrc[i] = Ab + (int64_t)ra * q.lda + cs * 8;
        wsrc[i] = Wb + (int64_t)(col0 + r) * q.K + cs * 8;
    }
    constexpr int64_t a_kst = BK, w_kst = BK;                     // row-major operands: the next K tile is 64 elements on
    char* const dma_a = smem + wave * 4096;
    char* const dma_w = smem + 2 * OPER2 + wave * 4096;

    f32x4_t acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.f;

    unsigned a_k[2], w_k[2];
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
        a_k[ks2] = (wr * 128 + lr) * 128 + (((ks2 * 4 + lq) ^ (lr & 7)) << 4);
        w_k[ks2] = 2 * OPER2 + (wc * 64 + lr) * 128 + (((ks2 * 4 + lq) ^ (lr & 7)) << 4);
    }
    const int nk = q.K / BK;
    bf16x8 wf[4];
    W8Lane w8;
    if (W8) {   // fp8-stored weights (q.W point at bytes): thread (row tid / 2, k half tid % 2), 32 weights per K tile
        const int r = tid >> 1, h = tid & 1;
        w8.src = reinterpret_cast<const unsigned char*>(Wb) + (int64_t)(col0 + r) * q.K + h * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) w8.lds[c] = r * 128 + (((h * 4 + c) ^ (r & 7)) << 4);
    }

    char* const img = smem + wave * 16384;
    const int tok0 = row0 + wr * 128;                 // first token (row of A) of this wave tile
    const int head = (col0 >> 6) + wc;
    const int64_t bh = (int64_t)b * q.heads + head;

    if (which == 2) {
        EA_G3_MAINLOOP(1, W8)
        int Mv = q.M;                       // laundered: nothing of the ragged-tile bookkeeping is hoisted above the main loop
        asm volatile("" : "+s"(Mv));
        int lane_e;                         // the lane id again, so that no lane-derived value stays live across the main loop
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
        qkv_epilogue_v(q, acc, img, biasb, col0 + wc * 64, tok0, qkv_kv_base(q, b, head), Mv, lane_e);
        return;
    }

    EA_G3_MAINLOOP(0, W8)
    int Mv = q.M;
    asm volatile("" : "+s"(Mv));
    int lane_e;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
    qkv_epilogue_qk(q, acc, img, biasb, col0 + wc * 64, tok0, bh, qkv_kv_base(q, b, head), which, Mv, lane_e);
}

// ---- the fused QKV projection on the four-wave hand-placed main loop (gemm256_w4a_kernel's; EA_W4A_MAINLOOP_ASM_SWAP for the V tiles).
// A wave tile is 128 tokens x 128 features = TWO heads: the shared per-head epilogues (qkv_epilogue_qk / _v above, contraction-free:
// bit-identical to gemm256_qkv_kernel) are called once per accumulator half.
__global__ __launch_bounds__(256) void gemm256_qkv_w4a_kernel(QkvArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    const int lr = lane & 15, lq = lane >> 4;

    int tm, tn;
    {
        GemmArgs g;
        g.tiles_m = q.tiles_m; g.tiles_n = q.tiles_n; g.rows_per_xcd = q.rows_per_xcd;
        if (!tile_of_block(g, tm, tn)) return;
    }
    const int b = blockIdx.y;
    const int row0 = tm * 256;
    const int tiles_per_w = q.inner >> 8;
    const int part = __builtin_amdgcn_readfirstlane(tn / tiles_per_w);
    const int which = q.first_part + part;                                 // 0 = q, 1 = k, 2 = v
    const int col0 = (tn - part * tiles_per_w) * 256;                      // first output feature inside that weight
    const unsigned short* Ab = q.A + b * q.abs_;
    const unsigned short* Wb = which == 0 ? q.W[0] : (which == 1 ? q.W[1] : q.W[2]);
    const float* biasb = which == 0 ? q.bias[0] : (which == 1 ? q.bias[1] : q.bias[2]);
    const int nk = q.K / BK;

    int aoff[8], woff[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = (wave * 8 + i) * 8 + (lane >> 3), c = lane & 7;
        const int cs = c ^ (r & 7);
        const int ra = (row0 + r < q.M ? row0 + r : q.M - 1) - row0;       // ragged last M tile: rows past M re-read row M - 1
        aoff[i] = (int)((int64_t)ra * q.lda * 2) + cs * 16;
        woff[i] = r * q.K * 2 + cs * 16;
    }
    const unsigned short* Abase = Ab + (int64_t)row0 * q.lda;
    const unsigned short* Wbase = Wb + (int64_t)col0 * q.K;
    const int a_rows = q.M - row0 < 256 ? q.M - row0 : 256;
    const unsigned a_ext = (unsigned)((((int64_t)a_rows - 1) * q.lda + q.K) * 2);
    const unsigned w_ext = (unsigned)((int64_t)256 * q.K * 2);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    const unsigned ak0 = lds0 + (wr * 128 + lr) * 128 + ((lq ^ (lr & 7)) << 4);
    const unsigned wk0 = lds0 + 2 * OPER2 + (wc * 128 + lr) * 128 + ((lq ^ (lr & 7)) << 4);
    const unsigned lds_a = __builtin_amdgcn_readfirstlane(lds0 + wave * 8192);
    const unsigned lds_w = __builtin_amdgcn_readfirstlane(lds0 + 2 * OPER2 + wave * 8192);
    const unsigned a_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)Abase);
    const unsigned a_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)Abase >> 32));
    const unsigned w_lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)Wbase);
    const unsigned w_hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)Wbase >> 32));
    const unsigned kst = BK * 2;
    const unsigned a_ext_s = __builtin_amdgcn_readfirstlane(a_ext), w_ext_s = __builtin_amdgcn_readfirstlane(w_ext);
    const unsigned nk_s = __builtin_amdgcn_readfirstlane((unsigned)nk);
#define EA_W4A_OPERANDS                                                                                                         \
    [wk0] "v"(wk0), [ak0] "v"(ak0), [aoff0] "v"(aoff[0]), [aoff1] "v"(aoff[1]), [aoff2] "v"(aoff[2]), [aoff3] "v"(aoff[3]),       \
        [aoff4] "v"(aoff[4]), [aoff5] "v"(aoff[5]), [aoff6] "v"(aoff[6]), [aoff7] "v"(aoff[7]), [woff0] "v"(woff[0]),              \
        [woff1] "v"(woff[1]), [woff2] "v"(woff[2]), [woff3] "v"(woff[3]), [woff4] "v"(woff[4]), [woff5] "v"(woff[5]),              \
        [woff6] "v"(woff[6]), [woff7] "v"(woff[7]), [a_lo] "s"(a_lo), [a_hi] "s"(a_hi), [a_ext] "s"(a_ext_s), [w_lo] "s"(w_lo),    \
        [w_hi] "s"(w_hi), [w_ext] "s"(w_ext_s), [a_kst] "s"(kst), [w_kst] "s"(kst), [nk] "s"(nk_s), [lds_w] "s"(lds_w),            \
        [lds_a] "s"(lds_a)
    f32x4_t accq[64];      // the 256 accumulators a0..a255, as the main asm's outputs: live until the read-outs consume them
    if (which == 2) {
        asm volatile(EA_W4A_MAINLOOP_ASM_SWAP : EA_W4A_ACC_OUTPUTS(accq) : EA_W4A_OPERANDS : EA_W4A_CLOBBERS);
    } else {
        asm volatile(EA_W4A_MAINLOOP_ASM : EA_W4A_ACC_OUTPUTS(accq) : EA_W4A_OPERANDS : EA_W4A_CLOBBERS);
    }
#undef EA_W4A_OPERANDS
    __builtin_amdgcn_s_barrier();

    char* const img = smem + wave * 16384;
    const int tok0 = row0 + wr * 128;                 // first token (row of A) of this wave tile
    const int head0 = (col0 >> 6) + wc * 2;           // the wave tile's two heads
    int Mv = q.M;
    asm volatile("" : "+s"(Mv));
    int lane_e;                                       // the lane id again: no lane-derived value has to stay live across the main loop
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
    f32x4_t acc[8][4];
    if (which == 2) {
        EA_W4A_READ_HALF0(acc, accq)
        qkv_epilogue_v(q, acc, img, biasb, head0 * 64, tok0, qkv_kv_base(q, b, head0), Mv, lane_e);
        EA_W4A_READ_HALF1(acc, accq)
        qkv_epilogue_v(q, acc, img, biasb, head0 * 64 + 64, tok0, qkv_kv_base(q, b, head0 + 1), Mv, lane_e);
    } else {
        EA_W4A_READ_HALF0(acc, accq)
        qkv_epilogue_qk(q, acc, img, biasb, head0 * 64, tok0, (int64_t)b * q.heads + head0, qkv_kv_base(q, b, head0), which, Mv, lane_e);
        EA_W4A_READ_HALF1(acc, accq)
        qkv_epilogue_qk(q, acc, img, biasb, head0 * 64 + 64, tok0, (int64_t)b * q.heads + head0 + 1, qkv_kv_base(q, b, head0 + 1), which, Mv,
                        lane_e);
    }
}

int g_gemm_w4a = 3;     // ea_set_option("gemm_w4a", bits): 1 = ea_gemm_bf16 / _kblocked, 2 = the fused QKV projection run on the four-wave kernels with the
                        // hand-placed main loop (default 3); 0 = the eight-wave kernels (kept: fp8 weights, cross-check)
int g_gemm_mfma = 16;   // ea_set_option("gemm_mfma", 16 | 32): MFMA shape of the 256^2 kernel (32: the first version, kept as cross-check)

template <int EPI, bool W8>
int launch_gemm(const GemmArgs& p0, int batch, int tile, hipStream_t st) {
    GemmArgs p = p0;
    if (p.ldw == 0) p.ldw = p.K;
    const int bm = tile, threads = tile == 256 ? 512 : 256;
    const int lds = tile == 256 ? GEMM2_LDS : GEMM_LDS;
    p.tiles_m = (p.M + bm - 1) / bm;
    p.tiles_n = (p.N + bm - 1) / bm;
    // small problems: plain N-fastest order over all XCDs; large M: per-XCD row bands (see tile_of_block)
    p.rows_per_xcd = p.tiles_m >= 64 ? (p.tiles_m + 7) / 8 : 0;
    dim3 grid(p.rows_per_xcd ? 8 * p.rows_per_xcd * p.tiles_n : p.tiles_m * p.tiles_n, batch);
    static bool attr_done[2] = {false, false};
    if (tile == 256) {
        if (!attr_done[1]) {
            hipFuncSetAttribute((const void*)gemm256_bf16_kernel<EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            attr_done[1] = true;
        }
        if ((g_gemm_mfma == 16 || W8) && EPI != EA_EPI_F32_OUT) {
            static bool attr16_done = false;
            if (!attr16_done) {
                hipFuncSetAttribute((const void*)gemm256_mi16_kernel<EPI, W8>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                attr16_done = true;
            }
            // the four-wave hand-placed kernel addresses its operands through 32-bit buffer offsets
            const int64_t nk64 = p.K / BK;
            const bool w4a_ok = !W8 && (g_gemm_w4a & 1) && ((nk64 - 1) * p.a_kstep + 255 * p.lda + BK) * 2 < (int64_t)0xFFFFFFFF &&
                                ((nk64 - 1) * p.w_kstep + 255 * p.ldw + BK) * 2 < (int64_t)0xFFFFFFFF;
            if (w4a_ok) {
                if constexpr (!W8) {
                    static bool attrw4_done = false;
                    if (!attrw4_done) {
                        hipFuncSetAttribute((const void*)gemm256_w4a_kernel<EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                        attrw4_done = true;
                    }
                    ea_count("gemm_256_w4a");
                    hipLaunchKernelGGL((gemm256_w4a_kernel<EPI>), grid, dim3(256), lds, st, p);
                }
                return EA_OK;
            }
            ea_count(W8 ? "gemm_256_mi16_w8" : "gemm_256_mi16");
            hipLaunchKernelGGL((gemm256_mi16_kernel<EPI, W8>), grid, dim3(threads), lds, st, p);
        } else {
            ea_count("gemm_256_mi32");
            hipLaunchKernelGGL(gemm256_bf16_kernel<EPI>, grid, dim3(threads), lds, st, p);
        }
    } else {
        if (!attr_done[0]) {
            hipFuncSetAttribute((const void*)gemm_bf16_kernel<EPI, W8>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            attr_done[0] = true;
        }
        ea_count(W8 ? "gemm_128_w8" : "gemm_128");
        hipLaunchKernelGGL((gemm_bf16_kernel<EPI, W8>), grid, dim3(threads), lds, st, p);
    }
    return EA_OK;
}

int g_gemm_tile = 0;   // 0 = auto, 128 / 256 = forced (ea_set_option("gemm_tile", ...), benchmarking only)

// W8: W points at fp8 (OCP E4M3) bytes, [N, K] K-contiguous (ea_gemm_bf16_w8)
template <bool W8>
int gemm_entry(const ea_bf16* A, const void* W, const float* bias, ea_bf16* C, const ea_bf16* res, const float* gate, int batch,
               int M, int N, int K, int64_t lda, int64_t a_batch_stride, int64_t ldc, int64_t c_batch_stride, int64_t ldres,
               int64_t res_batch_stride, int64_t gate_batch_stride, int epilogue, void* stream, int layout = 0) {
    EA_REQUIRE(A && W && C, "ea_gemm_bf16: null tensor");
    EA_REQUIRE(batch > 0 && batch <= 65535 && M >= 0 && N > 0 && K > 0, "ea_gemm_bf16: bad sizes");
    EA_REQUIRE(K % BK == 0, "ea_gemm_bf16: K=%d must be a multiple of %d", K, BK);
    EA_REQUIRE(N % 8 == 0 && lda % 8 == 0 && ldc % 8 == 0, "ea_gemm_bf16: N, lda, ldc must be multiples of 8");
    EA_REQUIRE(((uintptr_t)A | (uintptr_t)W | (uintptr_t)C) % 16 == 0, "ea_gemm_bf16: pointers must be 16-byte aligned");
    EA_REQUIRE(epilogue >= 0 && epilogue <= 3, "ea_gemm_bf16: unknown epilogue %d", epilogue);
    EA_REQUIRE(!(W8 && epilogue == EA_EPI_F32_OUT), "ea_gemm_bf16_w8: no fp32-output epilogue");
    if (epilogue == EA_EPI_BIAS_GATE_RES)
        EA_REQUIRE(res && gate && ldres % 8 == 0 && ((uintptr_t)res % 16 == 0) && ((uintptr_t)gate % 16 == 0),
                   "ea_gemm_bf16: gated-residual epilogue needs aligned res and gate");
    if (bias) EA_REQUIRE((uintptr_t)bias % 16 == 0, "ea_gemm_bf16: bias must be 16-byte aligned");
    if (M == 0) return EA_OK;
    GemmArgs p;
    p.A = A; p.W = reinterpret_cast<const unsigned short*>(W); p.bias = bias; p.C = C; p.res = res; p.gate = gate;
    p.M = M; p.N = N; p.K = K;
    p.lda = lda; p.abs_ = a_batch_stride; p.ldc = ldc; p.cbs = c_batch_stride;
    p.ldres = ldres; p.rbs = res_batch_stride; p.gbs = gate_batch_stride;
    // 256^2 ping-pong kernel when there are enough 256-row tiles to fill the 256 CUs a few times over
    int tile = g_gemm_tile;
    if (tile != 128 && tile != 256)
        tile = ((int64_t)((M + 255) / 256) * ((N + 255) / 256) * batch >= 512 && N % 256 == 0) ? 256 : 128;
    if (layout) {
        // K-blocked operands (ea_gemm_bf16_kblocked): bit 0 = A is [K / 64][M][64] per batch element, bit 1 = W is [K / 64][N][64],
        // bit 2 = C is written as [N / 64][M][64] per batch element (the A operand of a following GEMM).  Served by the 256 x 256
        // 16x16x32 kernel only (its DMA rows and its epilogue's 64-column wave tiles are what the layout is made for).
        EA_REQUIRE((layout & ~7) == 0 && !W8 && epilogue != EA_EPI_F32_OUT && g_gemm_mfma == 16 && N % 256 == 0,
                   "ea_gemm_bf16_kblocked: bf16 weights, bf16 output, N a multiple of 256 (the 256 x 256 kernel)");
        tile = 256;
        if (layout & 1) { p.lda = 64; p.a_kstep = (int64_t)M * 64; }
        if (layout & 2) { p.ldw = 64; p.w_kstep = (int64_t)N * 64; }
        if (layout & 4) { p.ldc = 64; p.c_kstep = (int64_t)M * 64; }
    }
    hipStream_t st = (hipStream_t)stream;
    switch (epilogue) {
        case EA_EPI_BIAS: launch_gemm<0, W8>(p, batch, tile, st); break;
        case EA_EPI_BIAS_GELU_TANH: launch_gemm<1, W8>(p, batch, tile, st); break;
        case EA_EPI_F32_OUT: launch_gemm<3, false>(p, batch, tile, st); break;
        default: launch_gemm<2, W8>(p, batch, tile, st); break;
    }
    return ea_check_launch(W8 ? "ea_gemm_bf16_w8" : "ea_gemm_bf16");
}

}  // namespace

// ea_gemm_mxfp4.hip's large products (gemm256_mxfp4_w4_kernel): codes / scales of [batch * M, K] and [N, K], kt K tiles; as_bytes = size of
// the activation scales' buffer.  EA_ERR_ARG if an operand does not fit the kernel's 32-bit buffer offsets.
int ea_gemm_mxfp4_w4_launch(const unsigned char* A, const unsigned char* As, int64_t as_bytes, const unsigned char* W, const unsigned char* Ws,
                            const float* bias, void* C, const ea_bf16* res, const float* gate, int batch, int M, int N, int kt, int64_t ldc,
                            int64_t cbs, int64_t ldres, int64_t rbs, int64_t gbs, int epilogue, hipStream_t st) {
    const int64_t a_rows = (int64_t)batch * M, limit = 0xFFFFFFFFll;
    if (a_rows * kt * 128 >= limit || (int64_t)N * kt * 128 >= limit || as_bytes >= limit || (int64_t)kt * 64 > 0x7fffffff) return EA_ERR_ARG;
    if (a_rows < 2 || as_bytes < a_rows * kt * 8 + (M % 2 ? MXW4_SCALE_PAD : 0)) return EA_ERR_ARG;      // (what mxw4_scale_offset's pairs reach)
    GemmArgs p;
    p.A = reinterpret_cast<const unsigned short*>(A); p.W = reinterpret_cast<const unsigned short*>(W); p.bias = bias;
    p.C = reinterpret_cast<unsigned short*>(C); p.res = res; p.gate = gate;
    p.M = M; p.N = N; p.K = kt * BK;
    p.lda = 64; p.abs_ = (int64_t)M * 64; p.ldc = ldc; p.cbs = cbs; p.ldres = ldres; p.rbs = rbs; p.gbs = gbs;
    p.a_kstep = a_rows * 64; p.w_kstep = (int64_t)N * 64; p.ldw = 64;
    p.tiles_m = (M + 255) / 256;
    p.tiles_n = (N + 255) / 256;
    p.rows_per_xcd = p.tiles_m >= 64 ? (p.tiles_m + 7) / 8 : 0;
    const dim3 grid(p.rows_per_xcd ? 8 * p.rows_per_xcd * p.tiles_n : p.tiles_m * p.tiles_n, batch);
    const auto kern = epilogue == EA_EPI_BIAS ? gemm256_mxfp4_w4_kernel<EA_EPI_BIAS>
                      : epilogue == EA_EPI_BIAS_GELU_TANH ? gemm256_mxfp4_w4_kernel<EA_EPI_BIAS_GELU_TANH> : gemm256_mxfp4_w4_kernel<EA_EPI_BIAS_GATE_RES>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, MXW4_LDS);
    if (e != hipSuccess) {
        ea_set_error("ea_gemm_mxfp4: %d bytes of LDS: %s", MXW4_LDS, hipGetErrorString(e));
        return (int)e;
    }
    ea_count("gemm_mxfp4_256_w4");
    hipLaunchKernelGGL(kern, grid, dim3(256), MXW4_LDS, st, p, As, Ws, as_bytes);
    return EA_OK;
}

extern "C" int ea_gemm_bf16(const ea_bf16* A, const ea_bf16* W, const float* bias, ea_bf16* C,
                            const ea_bf16* res, const float* gate, int batch, int M, int N, int K, int64_t lda,
                            int64_t a_batch_stride, int64_t ldc, int64_t c_batch_stride, int64_t ldres,
                            int64_t res_batch_stride, int64_t gate_batch_stride, int epilogue, void* stream) {
    return gemm_entry<false>(A, W, bias, C, res, gate, batch, M, N, K, lda, a_batch_stride, ldc, c_batch_stride, ldres,
                             res_batch_stride, gate_batch_stride, epilogue, stream);
}

extern "C" int ea_gemm_bf16_kblocked(const ea_bf16* A, const ea_bf16* W, const float* bias, ea_bf16* C,
                                     const ea_bf16* res, const float* gate, int batch, int M, int N, int K,
                                     int64_t a_batch_stride, int64_t c_batch_stride, int64_t ldres, int64_t res_batch_stride,
                                     int64_t gate_batch_stride, int epilogue, int layout, void* stream) {
    // lda / ldc are used for the operands that stay row-major (contiguous rows: K and N elements)
    return gemm_entry<false>(A, W, bias, C, res, gate, batch, M, N, K, K, a_batch_stride, N, c_batch_stride, ldres,
                             res_batch_stride, gate_batch_stride, epilogue, stream, layout);
}

extern "C" int ea_gemm_bf16_w8(const ea_bf16* A, const uint8_t* W_fp8, const float* bias, ea_bf16* C,
                               const ea_bf16* res, const float* gate, int batch, int M, int N, int K, int64_t lda,
                               int64_t a_batch_stride, int64_t ldc, int64_t c_batch_stride, int64_t ldres,
                               int64_t res_batch_stride, int64_t gate_batch_stride, int epilogue, void* stream) {
    return gemm_entry<true>(A, W_fp8, bias, C, res, gate, batch, M, N, K, lda, a_batch_stride, ldc, c_batch_stride, ldres,
                            res_batch_stride, gate_batch_stride, epilogue, stream);
}


namespace {
// W8: Wq / Wk / Wv point at fp8 (OCP E4M3) bytes (ea_qkv_gemm_norm_rope_bf16_w8)
template <bool W8>
int qkv_entry(const ea_bf16* A, const void* Wq, const void* Wk, const void* Wv,
                                          const float* bq, const float* bk, const float* bv, ea_bf16* q_out,
                                          ea_bf16* k_out, ea_bf16* vt_out, const float* nq_w, const float* nq_b,
                                          const float* nk_w, const float* nk_b, const float* cos, const float* sin,
                                          int batch, int M, int heads, int K, int64_t lda, int64_t a_batch_stride,
                                          int seq_off, int s_pad, int kv_off, int kv_rows, int parts, float ln_eps, float q_scale,
                                          void* stream, int kv_group_heads = 0, int64_t kv_group_stride = 0) {
    EA_REQUIRE(A && Wq && Wk && Wv && q_out && k_out && vt_out && nq_w && nq_b && nk_w && nk_b,
               "ea_qkv_gemm_norm_rope_bf16: null tensor");
    if (kv_group_heads <= 0) { kv_group_heads = heads; kv_group_stride = 0; }
    EA_REQUIRE(heads % kv_group_heads == 0 && kv_group_stride >= 0 && kv_group_stride % 8 == 0,
               "ea_qkv_gemm_norm_rope_bf16: kv_group_heads must divide heads, kv_group_stride must be a multiple of 8 elements");
    if (kv_rows <= 0) { kv_rows = s_pad; kv_off = seq_off; }
    if (parts == 0) parts = 7;
    EA_REQUIRE(parts == 7 || parts == 1 || parts == 6, "ea_qkv_gemm_norm_rope_bf16: parts must be 7 (q|k|v), 1 (q) or 6 (k|v)");
    EA_REQUIRE(kv_off >= 0 && kv_off % 8 == 0 && kv_rows % 8 == 0 && kv_off + M <= kv_rows,
               "ea_qkv_gemm_norm_rope_bf16: kv_off / kv_rows must be multiples of 8 with kv_off + M <= kv_rows");
    EA_REQUIRE((cos == nullptr) == (sin == nullptr), "ea_qkv_gemm_norm_rope_bf16: cos and sin go together");
    EA_REQUIRE(batch > 0 && batch <= 65535 && heads > 0 && M > 0 && K > 0, "ea_qkv_gemm_norm_rope_bf16: bad sizes");
    EA_REQUIRE((heads * 64) % 256 == 0, "ea_qkv_gemm_norm_rope_bf16: heads*64 must be a multiple of 256");
    EA_REQUIRE(K % BK == 0 && lda % 8 == 0, "ea_qkv_gemm_norm_rope_bf16: K must be a multiple of 64, lda of 8");
    EA_REQUIRE(seq_off >= 0 && seq_off % 8 == 0 && s_pad % 8 == 0 && seq_off + M <= s_pad,
               "ea_qkv_gemm_norm_rope_bf16: seq_off / s_pad must be multiples of 8 with seq_off + M <= s_pad");
    EA_REQUIRE((((uintptr_t)A | (uintptr_t)Wq | (uintptr_t)Wk | (uintptr_t)Wv | (uintptr_t)q_out | (uintptr_t)k_out |
                 (uintptr_t)vt_out | (uintptr_t)bq | (uintptr_t)bk | (uintptr_t)bv | (uintptr_t)nq_w | (uintptr_t)nq_b |
                 (uintptr_t)nk_w | (uintptr_t)nk_b | (uintptr_t)cos | (uintptr_t)sin) & 15) == 0,
               "ea_qkv_gemm_norm_rope_bf16: pointers must be 16-byte aligned");
    QkvArgs q;
    q.A = A;
    q.W[0] = reinterpret_cast<const unsigned short*>(Wq);
    q.W[1] = reinterpret_cast<const unsigned short*>(Wk);
    q.W[2] = reinterpret_cast<const unsigned short*>(Wv); q.bias[0] = bq; q.bias[1] = bk; q.bias[2] = bv;
    q.q_out = q_out; q.k_out = k_out; q.vt_out = vt_out;
    q.nw[0] = nq_w; q.nb[0] = nq_b; q.nw[1] = nk_w; q.nb[1] = nk_b; q.cosT = cos; q.sinT = sin;
    q.M = M; q.K = K; q.inner = heads * 64; q.heads = heads; q.seq_off = seq_off; q.s_pad = s_pad;
    q.kv_off = kv_off; q.kv_rows = kv_rows; q.first_part = parts == 6 ? 1 : 0;
    q.kv_gheads = kv_group_heads; q.kv_gstride = kv_group_stride;
    q.lda = lda; q.abs_ = a_batch_stride; q.eps = ln_eps; q.q_scale = q_scale;
    q.tiles_m = (M + 255) / 256;      // a ragged last tile re-reads row M - 1 and stores rows < M only
    q.tiles_n = (parts == 7 ? 3 : (parts == 6 ? 2 : 1)) * q.inner / 256;
    q.rows_per_xcd = q.tiles_m >= 64 ? (q.tiles_m + 7) / 8 : 0;
    dim3 grid(q.rows_per_xcd ? 8 * q.rows_per_xcd * q.tiles_n : q.tiles_m * q.tiles_n, batch);
    static bool attr_done = false;
    if (!attr_done) {
        hipFuncSetAttribute((const void*)gemm256_qkv_kernel<W8>, hipFuncAttributeMaxDynamicSharedMemorySize, GEMM2_LDS);
        attr_done = true;
    }
    // the four-wave hand-placed main loop (32-bit buffer offsets: a 256-row tile of A / W must be reachable within 4 GiB)
    const bool qkv_w4a = !W8 && (g_gemm_w4a & 2) && (255 * lda + K) * 2 < (int64_t)0xFFFFFFFF && (int64_t)256 * K * 2 < (int64_t)0xFFFFFFFF;
    if (qkv_w4a) ea_count("gemm_qkv_fused_w4a");       // (markers first: ea_last_dispatch() stays "gemm_qkv_fused")
    if (parts != 7) ea_count(parts == 6 ? "gemm_qkv_fused_kv_part" : "gemm_qkv_fused_q_part");
    ea_count(W8 ? "gemm_qkv_fused_w8" : "gemm_qkv_fused");
    if (qkv_w4a) {
        static bool attrw4_done = false;
        if (!attrw4_done) {
            hipFuncSetAttribute((const void*)gemm256_qkv_w4a_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, GEMM2_LDS);
            attrw4_done = true;
        }
        hipLaunchKernelGGL(gemm256_qkv_w4a_kernel, grid, dim3(256), GEMM2_LDS, (hipStream_t)stream, q);
        return ea_check_launch("ea_qkv_gemm_norm_rope_bf16");
    }
    hipLaunchKernelGGL(gemm256_qkv_kernel<W8>, grid, dim3(512), GEMM2_LDS, (hipStream_t)stream, q);
    return ea_check_launch(W8 ? "ea_qkv_gemm_norm_rope_bf16_w8" : "ea_qkv_gemm_norm_rope_bf16");
}
}  // namespace

extern "C" int ea_qkv_gemm_norm_rope_bf16(const ea_bf16* A, const ea_bf16* Wq, const ea_bf16* Wk, const ea_bf16* Wv,
                                          const float* bq, const float* bk, const float* bv, ea_bf16* q_out,
                                          ea_bf16* k_out, ea_bf16* vt_out, const float* nq_w, const float* nq_b,
                                          const float* nk_w, const float* nk_b, const float* cos, const float* sin,
                                          int batch, int M, int heads, int K, int64_t lda, int64_t a_batch_stride,
                                          int seq_off, int s_pad, int kv_off, int kv_rows, int parts, float ln_eps,
                                          float q_scale, void* stream) {
    return qkv_entry<false>(A, Wq, Wk, Wv, bq, bk, bv, q_out, k_out, vt_out, nq_w, nq_b, nk_w, nk_b, cos, sin, batch, M, heads, K, lda,
                            a_batch_stride, seq_off, s_pad, kv_off, kv_rows, parts, ln_eps, q_scale, stream);
}

// K / V^T written in head groups (see QkvArgs::kv_gheads): the sequence-parallel exchange by head groups
extern "C" int ea_qkv_gemm_norm_rope_grouped_bf16(const ea_bf16* A, const ea_bf16* Wq, const ea_bf16* Wk, const ea_bf16* Wv,
                                                  const float* bq, const float* bk, const float* bv, ea_bf16* q_out,
                                                  ea_bf16* k_out, ea_bf16* vt_out, const float* nq_w, const float* nq_b,
                                                  const float* nk_w, const float* nk_b, const float* cos, const float* sin,
                                                  int batch, int M, int heads, int K, int64_t lda, int64_t a_batch_stride,
                                                  int seq_off, int s_pad, int kv_off, int kv_rows, int parts, int kv_group_heads,
                                                  int64_t kv_group_stride, float ln_eps, float q_scale, void* stream) {
    return qkv_entry<false>(A, Wq, Wk, Wv, bq, bk, bv, q_out, k_out, vt_out, nq_w, nq_b, nk_w, nk_b, cos, sin, batch, M, heads, K, lda,
                            a_batch_stride, seq_off, s_pad, kv_off, kv_rows, parts, ln_eps, q_scale, stream, kv_group_heads, kv_group_stride);
}

extern "C" int ea_qkv_gemm_norm_rope_bf16_w8(const ea_bf16* A, const uint8_t* Wq_fp8, const uint8_t* Wk_fp8, const uint8_t* Wv_fp8,
                                             const float* bq, const float* bk, const float* bv, ea_bf16* q_out,
                                             ea_bf16* k_out, ea_bf16* vt_out, const float* nq_w, const float* nq_b,
                                             const float* nk_w, const float* nk_b, const float* cos, const float* sin,
                                             int batch, int M, int heads, int K, int64_t lda, int64_t a_batch_stride,
                                             int seq_off, int s_pad, int kv_off, int kv_rows, int parts, float ln_eps,
                                             float q_scale, void* stream) {
    return qkv_entry<true>(A, Wq_fp8, Wk_fp8, Wv_fp8, bq, bk, bv, q_out, k_out, vt_out, nq_w, nq_b, nk_w, nk_b, cos, sin, batch, M, heads, K,
                           lda, a_batch_stride, seq_off, s_pad, kv_off, kv_rows, parts, ln_eps, q_scale, stream);
}

#ifdef EA_GEMM_TIMESTAMPS
extern "C" int ea_debug_gemm_timestamps(void* buf) {
    return (int)hipMemcpyToSymbol(HIP_SYMBOL(g_gemm_ts), &buf, sizeof(void*));
}
extern "C" int ea_debug_gemm_stagger(int n) {
    return (int)hipMemcpyToSymbol(HIP_SYMBOL(g_gemm_stagger), &n, sizeof(int));
}
#endif

int ea_gemm_tile_get() { return g_gemm_tile; }
int ea_gemm_tile_set(int v) {
    if (v != 0 && v != 128 && v != 256) return -1;
    g_gemm_tile = v;
    return 0;
}
int ea_gemm_w4a_get() { return g_gemm_w4a; }
int ea_gemm_w4a_set(int v) {
    if (v < 0 || v > 3) return -1;
    g_gemm_w4a = v;
    return 0;
}
int ea_gemm_mfma_get() { return g_gemm_mfma; }
int ea_gemm_mfma_set(int v) {
    if (v != 16 && v != 32) return -1;
    g_gemm_mfma = v;
    return 0;
}
