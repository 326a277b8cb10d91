// Attention of text models: softmax(f(q k^T)) v with grouped-query heads, scores capped by a tanh and / or biased by distance, and any
// combination of causal order, a prefix that every query sees, packed documents and key lengths:
//     t = scale q.k;   t = cap tanh(t / cap);   t += bias[h][clamp(j - p, -R, R) + R]        p = q_start[b] + i, the query's position
//     key j is visible to query i:  j < valid[b]  and  (not causal or j <= p or j < prefix[b])  and  kv_docs[b][j] == q_docs[b][i]
// Order, prefix and length together are ONE limit per query -- keys j < lim(i) = min(valid, max(p + 1, prefix)) -- so a partly masked
// tile costs one comparison per score, plus one when documents are packed.  A query that sees nothing yields zeros; what hidden keys
// and values hold (NaN included) does not reach the result.
//
// A "row" is a (query, head of the group) pair: the heads that share a K / V head are packed next to each other (row = query * pack +
// head), so a K / V tile serves all of them, a single new token fills a 16-row matrix tile as far as its group reaches, and a causal
// tile's diagonal is `pack` times narrower in keys.
//
// Evaluated transposed as in the other attention kernels (S^T = K Q^T, O^T = V^T P^T on v_mfma_f32_16x16x32_bf16): a lane owns one row
// and, because K rows are fed in the order 8 (r / 4) + 4 kt + r % 4, eight consecutive keys of a 32-key block = its slice of the P^T
// operand.  V stays row-major in memory and LDS; its transposed fragments come from ds_read_b64_tr_b16.  One pass with a running
// maximum that is only moved when a score exceeds it by 2^8 (P then stays below 256 -- bf16 has fp32's exponent range -- and the
// accumulators are hardly ever rescaled).  P is rounded to bf16 for its product (a relative half step of 2^-8 each): the bf16 matrix
// instructions take no more, and a second product for what the rounding cuts off would double the work of P.V.  The results' distance
// from 64 bits grows by it from 1.7e-3 (their own rounding) to 1.8 .. 2.4e-3, relative.  The row sums are those of the rounded weights,
// by one more product with ones, in fp32.
//
//   attention_text_kernel       128 or 64 rows per workgroup (four waves, 32 or 16 rows each), K / V tiles of 64 keys double-buffered in LDS by
//                               LDS-DMA; tiles that no row of the workgroup sees are skipped (64 at a time for documents)
//   attention_text_few_kernel   up to 16 rows: each of the four waves walks its own 32-key blocks, K straight into registers
//   The few rows and the 64-row tiles can split the keys over workgroups; the join kernels combine the partial results in a fixed order.
#include "ea_common.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_a __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_a __attribute__((ext_vector_type(4)));

struct TextArgs {
    const unsigned short* q;
    const unsigned short* k;
    const unsigned short* v;
    unsigned short* out;
    const float* bias;        // [Hq][2 reach + 1] or null
    const int* q_docs;        // [B][Sq] (row stride qd_ld) or null
    const int* kv_docs;       // [B][Sk]
    const int* doc_range;     // [B][key tiles][2]: least and greatest document of each 64-key tile
    const int* prefix;        // [B] or null
    const int* valid;         // [B] or null
    const int* q_start;       // [B] or null (Sk - Sq)
    float* part;              // [splits][rows][D] and, behind it, [splits][rows][2] = (running maximum, sum)
    int64_t qb, qh, qs, kb, kh, ks, vb, vh, vs, ob, os, qd_ld, kd_ld;
    int B, Hq, Hkv, Sq, Sk, group, pack, causal, reach, splits, row_tiles, key_tiles;
    float scale, cap;
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr int BIAS_PACK_MAX = 8;        // heads packed into a row tile at most (bounds the bias window: see bias_window)

// LDS-DMA requests, 16 (4) bytes per lane at byte offset voff of a resource of `extent` bytes; past its end zeros arrive.  Written in
// assembly -- they have no result register -- because the compiler, where it sees them, waits for every request in flight in front of
// each transposed LDS read.  (Its own counted waits stay right: requests that it does not count only make them wait longer.)
typedef unsigned u32x4_s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4_s resource(const void* base, const unsigned extent) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    return u32x4_s{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)),
                   (unsigned)__builtin_amdgcn_readfirstlane((int)extent), 0x00020000u};
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(size_t)(__attribute__((address_space(3))) const char*)p);
}
__device__ __forceinline__ void dma16(const u32x4_s rs, const int voff, const unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rs) : "m0", "memory");
}
// resource over `rows` rows of 2 D bytes, `step` elements apart (rows <= 0: empty)
template <int D>
__device__ __forceinline__ u32x4_s rows_resource(const unsigned short* from, const int step, const int rows) {
    return resource(from, rows > 0 ? (unsigned)(rows - 1) * (unsigned)step * 2u + 2u * D : 0u);
}
__device__ __forceinline__ void words_to_lds(const int* from, const int words, const int voff, void* lds_wave_base) {
    const u32x4_s rs = resource(from, words > 0 ? (unsigned)words * 4u : 0u);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds_address(lds_wave_base)), "v"(voff), "s"(rs)
                 : "m0", "memory");
}
// the greater value, NaN where one is (no canonicalising moves in front of it, unlike fmaxf)
__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float log2_bias(float v) {
    const float big = 3.4028234663852886e38f;
    return fabsf(v) <= big ? fminf(fmaxf(v * LOG2E, -big), big) : v;
}

// 16-byte-chunk swizzle of the LDS rows (2 D bytes each), the same for K and V: an even number, so that 32-byte pairs of chunks stay
// together.  K fragments: eight lanes read rows {0..3, 8..11} at one chunk and eight others the neighbouring chunk; V's transposed
// reads: 32-byte pieces of rows {0..3} of every eight.  Either way the pieces land in different banks.
template <int D>
__device__ __forceinline__ int swz(int row) {
    return D == 128 ? 2 * ((row & 3) | ((row >> 3) & 1) << 2) : 2 * (((row >> 1) & 1) | ((row >> 3) & 1) << 1);
}

// ---- the rows of one wave -------------------------------------------------------------------------------------------------------
template <int D, int RT>
struct Rows {
    bf16x8 q[RT][D / 32];
    int lim[RT], doc[RT];     // keys below lim (and of the row's document) are visible
    int back[RT];             // distance bias: (last query of the tile) - (this query), + the row's head's window
    int lim_lo, lim_hi;       // over the wave's rows
    int doc_lo, doc_hi;
    f32x4 o[RT][D / 16];
    float m[RT];              // the reference maximum (log2 domain)
    f32x4 l[RT];              // the sum of the weights, in every element (a product with ones)
};

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
    return v;
}
// what a batch element's masks are: position of its first query, keys that exist, keys every query sees
struct Seq {
    int64_t first;
    int keys, prefix;
};
__device__ __forceinline__ Seq seq_of(const TextArgs& p, int b) {
    Seq s;
    s.first = p.q_start ? p.q_start[b] : (int64_t)p.Sk - p.Sq;
    s.keys = p.valid && p.valid[b] < p.Sk ? p.valid[b] : p.Sk;
    s.prefix = p.prefix ? p.prefix[b] : 0;
    return s;
}
__device__ __forceinline__ int key_limit(const TextArgs& p, const Seq& s, int qi) {
    int64_t lim = s.keys;
    if (p.causal) {
        int64_t c = s.first + qi + 1;
        c = s.prefix > c ? s.prefix : c;
        lim = c < lim ? c : lim;
    }
    return lim > 0 ? (int)lim : 0;
}

// head0: first query head of the packed set; row0: first row of this wave; qlast: last query of the workgroup's tile
template <int D, int RT>
__device__ __forceinline__ void load_rows(const TextArgs& p, Rows<D, RT>& R, const Seq& seq, int b, int head0, int row0, int qlast, int win, int lane) {
    const int lr = lane & 15, lq = lane >> 4;
    R.lim_lo = 0x7fffffff;
    R.lim_hi = 0;
    R.doc_lo = 0x7fffffff;
    R.doc_hi = -0x7fffffff - 1;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = row0 + t * 16 + lr;
        int qi = row / p.pack;
        const bool live = qi < p.Sq;
        const int hg = live ? row % p.pack : p.pack - 1;
        qi = live ? qi : p.Sq - 1;                        // rows past the end repeat the last one and are not stored
        const unsigned short* src = p.q + b * p.qb + (int64_t)(head0 + hg) * p.qh + (int64_t)qi * p.qs + lq * 8;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) R.q[t][s] = *reinterpret_cast<const bf16x8*>(src + s * 32);
        R.lim[t] = key_limit(p, seq, qi);
        R.doc[t] = p.q_docs ? p.q_docs[b * p.qd_ld + qi] : 0;
        R.back[t] = hg * win + (qlast - qi);
        R.lim_lo = min(R.lim_lo, R.lim[t]);
        R.lim_hi = max(R.lim_hi, R.lim[t]);
        R.doc_lo = min(R.doc_lo, R.doc[t]);
        R.doc_hi = max(R.doc_hi, R.doc[t]);
        R.m[t] = NEG_INF;
        R.l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) R.o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    R.lim_lo = __builtin_amdgcn_readfirstlane(wave_min(R.lim_lo));
    R.lim_hi = __builtin_amdgcn_readfirstlane(wave_max(R.lim_hi));
    if (p.q_docs) {
        R.doc_lo = __builtin_amdgcn_readfirstlane(wave_min(R.doc_lo));
        R.doc_hi = __builtin_amdgcn_readfirstlane(wave_max(R.doc_hi));
    }
}

// cap tanh(t / cap) log2(e) of t = s scale.  tanh(x) = 1 - 2 / (1 + e^2x): absolute error about cap 2^-22, so for a cap that is large
// beside the scores (cap > CAP_WIDE) small x go through the odd series x - x^3/3 + 2x^5/15 - 17x^7/315 (|x| < 0.25: the next
// term is 6e-8 of x) instead.
constexpr float CAP_WIDE = 256.0f;
__device__ __forceinline__ float capped_log2(float s, float two_over, float c1, float half_over, bool wide) {
    const float e = __builtin_amdgcn_exp2f(s * two_over);
    float t = __builtin_fmaf(-2.0f * c1, __builtin_amdgcn_rcpf(e + 1.0f), c1);
    if (wide) {
        const float x = s * half_over, x2 = x * x;
        const float series = x * __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
        t = fabsf(x) < 0.25f ? c1 * series : t;
    }
    return t;
}

// K fragments of a 32-key block: A operand, key rows in the order 8 (r / 4) + 4 kt + r % 4.  V^T fragments: lane (lr, lq) of a transposed
// read gets keys 8 lq + (0..3 | 4..7) of column 16 d + lr.  `at` is the block's LDS offset (a multiple of 256); a row's swizzle does not
// reach the bits above the row, so a fragment's place is the lane's first one with the fragment's bits flipped.
template <int D>
__device__ __forceinline__ int k_lane(int lane) {
    const int row = 8 * ((lane & 15) >> 2) + (lane & 3);
    return row * (2 * D) + (((lane >> 4) ^ swz<D>(row)) << 4);
}
template <int D>
__device__ __forceinline__ int v_lane(int lane) {
    const int row = 8 * (lane >> 4) + ((lane & 15) >> 2);
    return row * (2 * D) + ((((lane & 3) >> 1) ^ swz<D>(row)) << 4) + (lane & 1) * 8;
}
template <int D>
__device__ __forceinline__ void read_k(const char* smem, int at, bf16x8 (&kf)[2][D / 32]) {       // at: + k_lane
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) kf[kt][s] = *reinterpret_cast<const bf16x8*>(smem + (at ^ (s * 64)) + kt * (8 * D));
}
template <int D>
__device__ __forceinline__ void read_v(const char* smem, int at, u32x4_a (&vf)[D / 16]) {         // at: + v_lane
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
        const char* a = smem + (at ^ (d * 32));
        const u32x2_a lo = __builtin_bit_cast(u32x2_a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a));
        const u32x2_a hi = __builtin_bit_cast(u32x2_a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 8 * D)));
        vf[d] = u32x4_a{lo[0], lo[1], hi[0], hi[1]};
    }
}

template <int D, int RT>
__device__ __forceinline__ void block_qk(const Rows<D, RT>& R, const bf16x8 (&kf)[2][D / 32], float (&s)[RT][8]) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt][ks], R.q[t][ks], a, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][kt * 4 + r] = a[r];
        }
}

// What a score still has to be multiplied with to be in the log2 domain, behind cap_and_bias.
template <bool CAP, bool BIAS>
__device__ __forceinline__ float unit_of(const TextArgs& p) { return CAP || BIAS ? 1.0f : p.scale * LOG2E; }

// Cap and bias of one 32-key block, to the log2 domain.  win0: this lane's bias window position of key 8 lq of the block.
template <int D, int RT, bool CAP, bool BIAS, bool WIDE>
__device__ __forceinline__ void cap_and_bias(const TextArgs& p, const Rows<D, RT>& R, float (&s)[RT][8], const float* win0) {
    const float c = p.scale * LOG2E;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (CAP) s[t][e] = capped_log2(s[t][e], 2.0f * c / p.cap, p.cap * LOG2E, p.scale / p.cap, WIDE);
            if (BIAS) s[t][e] = __builtin_fmaf(s[t][e], CAP ? 1.0f : c, win0[R.back[t] + e]);
        }
}
// this lane's greatest score per row, and whether one has outgrown the reference maximum
template <int D, int RT>
__device__ __forceinline__ bool block_top(const Rows<D, RT>& R, const float (&s)[RT][8], const float unit, float (&top)[RT]) {
    bool grow = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        top[t] = max2(max2(max2(s[t][0], s[t][1]), max2(s[t][2], s[t][3])), max2(max2(s[t][4], s[t][5]), max2(s[t][6], s[t][7]))) * unit;
        grow = grow | (top[t] > R.m[t] + 8.0f);
    }
    return grow;
}
template <int D, int RT>
__device__ __forceinline__ void block_grow(Rows<D, RT>& R, const float (&top)[RT]) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float n = fmaxf(top[t], __shfl_xor(top[t], 16, 64));
        n = fmaxf(n, __shfl_xor(n, 32, 64));
        n = fmaxf(n, R.m[t]);
        const float alpha = n == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(R.m[t] - n);
        R.m[t] = n;
        R.l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) R.o[t][d] *= alpha;
    }
}
template <int D, int RT>
__device__ __forceinline__ void block_weights(const Rows<D, RT>& R, const float (&s)[RT][8], const float unit, bf16x8 (&pb)[RT]) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float ref = R.m[t] == NEG_INF ? 0.0f : R.m[t];
        u32x4_a pk;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], unit, -ref));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e + 1], unit, -ref));
            const f32x2 two = {p0, p1};
            pk[e >> 1] = __builtin_bit_cast(unsigned, __builtin_convertvector(two, bf16x2));
        }
        pb[t] = __builtin_bit_cast(bf16x8, pk);
    }
}

// Scores -> weights of one 32-key block, state updated.
// masked: some pair of the block may be hidden; docs: this lane's 8 keys' documents (masked blocks of packed documents).
template <int D, int RT, bool CAP, bool BIAS>
__device__ __forceinline__ void block_softmax(const TextArgs& p, Rows<D, RT>& R, float (&s)[RT][8], bf16x8 (&pb)[RT], int key0, bool masked,
                                              const int (&docs)[8], const float* win0, int lane) {
    const int lq = lane >> 4;
    if (CAP && p.cap > CAP_WIDE) cap_and_bias<D, RT, CAP, BIAS, true>(p, R, s, win0);
    else cap_and_bias<D, RT, CAP, BIAS, false>(p, R, s, win0);
    if (masked) {
        if (p.q_docs) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[t][e] = docs[e] == R.doc[t] ? s[t][e] : NEG_INF;
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int room = R.lim[t] - key0 - 8 * lq;
#pragma unroll
            for (int e = 0; e < 8; ++e) s[t][e] = e < room ? s[t][e] : NEG_INF;
        }
    }
    float top[RT];
    const float unit = unit_of<CAP, BIAS>(p);
    if (__ballot(block_top<D, RT>(R, s, unit, top))) block_grow<D, RT>(R, top);
    block_weights<D, RT>(R, s, unit, pb);
}

// O^T += V^T P^T, and the sums of the same (rounded) weights
template <int D, int RT>
__device__ __forceinline__ void block_pv(Rows<D, RT>& R, const u32x4_a (&vf)[D / 16], const bf16x8 (&pb)[RT]) {
    const u32x4_a ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int t = 0; t < RT; ++t) R.l[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ones), pb[t], R.l[t], 0, 0, 0);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int t = 0; t < RT; ++t) R.o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vf[d]), pb[t], R.o[t][d], 0, 0, 0);
}

// Does a fragment of V hold an infinity or a NaN?  (Both halves of every word: exponent bits all set = 0x7f80 or more without the sign.)
template <int D>
__device__ __forceinline__ bool any_odd(const u32x4_a (&vf)[D / 16]) {
    typedef short s16x2_a __attribute__((ext_vector_type(2)));
    s16x2_a top = {0, 0};
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int w = 0; w < 4; ++w) top = __builtin_elementwise_max(top, __builtin_bit_cast(s16x2_a, vf[d][w] & 0x7fff7fffu));
    return __ballot(top[0] >= 0x7f80 || top[1] >= 0x7f80) != 0;
}

// Where some of the block's pairs are hidden and V holds infinities or NaN: a hidden key's weight is 0, but 0 times those is not.  They
// are taken out of V's fragments, and what they make of the rows that do see them is added here: a product of their places with the
// weights' signs (1 where a weight is not 0) counts, for every output, the infinities of either sign and the NaN among its keys.
template <int D, int RT>
__device__ __forceinline__ void take_out_odd(Rows<D, RT>& R, u32x4_a (&vf)[D / 16], const bf16x8 (&pb)[RT]) {
    u32x4_a seen[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const unsigned p = __builtin_bit_cast(u32x4_a, pb[t])[w];
            seen[t][w] = ((p & 0x7fffu) ? 0x3f80u : 0u) | ((p & 0x7fff0000u) ? 0x3f800000u : 0u);
        }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
#pragma unroll
        for (int kind = 0; kind < 3; ++kind) {          // +infinity, -infinity, NaN
            u32x4_a at;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned lo = vf[d][w] & 0xffffu, hi = vf[d][w] >> 16;
                const bool l = kind == 0 ? lo == 0x7f80u : kind == 1 ? lo == 0xff80u : (lo & 0x7fffu) > 0x7f80u;
                const bool h = kind == 0 ? hi == 0x7f80u : kind == 1 ? hi == 0xff80u : (hi & 0x7fffu) > 0x7f80u;
                at[w] = (l ? 0x3f80u : 0u) | (h ? 0x3f800000u : 0u);
            }
            const float add = kind == 0 ? -NEG_INF : kind == 1 ? NEG_INF : __builtin_nanf("");
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, at), __builtin_bit_cast(bf16x8, seen[t]),
                                                                        f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) R.o[t][d][r] += n[r] > 0.0f ? add : 0.0f;
            }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const unsigned v = vf[d][w];
            vf[d][w] = ((v & 0x7f80u) == 0x7f80u ? 0u : v & 0xffffu) | ((v & 0x7f800000u) == 0x7f800000u ? 0u : v & 0xffff0000u);
        }
    }
}

// A 64-key tile whose pairs are all visible, for waves of 16 rows: its two blocks overlapped, one block's softmax (vector pipe) between
// the other's matrix instructions (8 heads, 4096 tokens, D = 64: 78 against 86 us, causal 60 against 70; D = 128 109 against 111).  The weights are taken against the old reference maximum; a score that has outgrown it -- seldom -- sends the
// block through block_grow and has its weights taken again.
template <int NM, int NV>
__device__ __forceinline__ void interleave() {           // NV vector instructions behind each of NM matrix instructions
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, NV, 0);
    }
}
template <int D, int RT, bool CAP, bool BIAS>
__device__ __forceinline__ void open_tile(const TextArgs& p, Rows<D, RT>& R, const char* smem, int k_at, int v_at, const float* win0) {
    constexpr int NV = (CAP ? 8 : BIAS ? 5 : 4) * (D == 64 ? 2 : 1);
    const float unit = unit_of<CAP, BIAS>(p);
    bf16x8 k0[2][D / 32], k1[2][D / 32], p0[RT], p1[RT];
    u32x4_a v0[D / 16], v1[D / 16];
    float s0[RT][8], s1[RT][8], top[RT];
    read_k<D>(smem, k_at, k0);
    read_k<D>(smem, k_at + 64 * D, k1);
    __builtin_amdgcn_sched_barrier(0);
    block_qk<D, RT>(R, k0, s0);
    __builtin_amdgcn_sched_barrier(0);
    read_v<D>(smem, v_at, v0);
    read_v<D>(smem, v_at + 64 * D, v1);
    __builtin_amdgcn_sched_barrier(0);
    block_qk<D, RT>(R, k1, s1);
    cap_and_bias<D, RT, CAP, BIAS, false>(p, R, s0, win0);
    bool grow = block_top<D, RT>(R, s0, unit, top);
    block_weights<D, RT>(R, s0, unit, p0);
    interleave<RT * 2 * (D / 32), NV>();
    __builtin_amdgcn_sched_barrier(0);
    if (__ballot(grow)) {
        block_grow<D, RT>(R, top);
        block_weights<D, RT>(R, s0, unit, p0);
    }
    __builtin_amdgcn_sched_barrier(0);
    block_pv<D, RT>(R, v0, p0);
    cap_and_bias<D, RT, CAP, BIAS, false>(p, R, s1, win0 + 32);
    grow = block_top<D, RT>(R, s1, unit, top);
    block_weights<D, RT>(R, s1, unit, p1);
    interleave<RT * (D / 16 + 1), NV>();
    __builtin_amdgcn_sched_barrier(0);
    if (__ballot(grow)) {
        block_grow<D, RT>(R, top);
        block_weights<D, RT>(R, s1, unit, p1);
    }
    block_pv<D, RT>(R, v1, p1);
}

// ---- which key tiles a workgroup visits ------------------------------------------------------------------------------------------
// Tiles [lo, hi); with documents only those whose range of documents meets [dlo, dhi]: 64 tiles are looked up at once, one per lane.
struct TileWalk {
    const int* range;      // this batch element's [tiles][2], or null
    int base, hi, dlo, dhi;
    unsigned long long left;
    int blo, bhi;          // the documents of the lane's tile in the current batch of 64
    __device__ __forceinline__ void fill(int from, int lane) {
        const int t = base + lane;
        bool want = t >= from && t < hi;
        blo = dlo; bhi = dlo;
        if (range && want) {
            blo = range[2 * t];
            bhi = range[2 * t + 1];
            want = blo <= dhi && bhi >= dlo;
        }
        left = __ballot(want);
    }
    __device__ __forceinline__ void start(int lo, int hi_, int lane) {
        hi = hi_;
        base = lo;
        left = 0;
        if (lo < hi) fill(lo, lane);
    }
    // the next tile, or -1; its documents' range goes to (lo, hi_)
    __device__ __forceinline__ int next(int lane, int& lo, int& hi_) {
        while (left == 0) {
            base += 64;
            if (base >= hi) return -1;
            fill(base, lane);
        }
        const int i = __builtin_ctzll(left);
        left &= left - 1;
        lo = __builtin_amdgcn_readlane(blo, i);
        hi_ = __builtin_amdgcn_readlane(bhi, i);
        return base + i;
    }
};

// normalise and store the wave's rows, or leave its state for the join
template <int D, int RT>
__device__ __forceinline__ void store_rows(const TextArgs& p, Rows<D, RT>& R, int b, int head0, int64_t part_row0, int split, int64_t rows_all, int row0,
                                           int lane) {
    const int lr = lane & 15, lq = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = R.l[t][0];
        const int in = row0 + t * 16 + lr, qi = in / p.pack, hg = in - qi * p.pack;
        if (qi >= p.Sq) continue;
        if (RT == 2 || p.splits == 1) {                  // (the 128-row tiles are never split)
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            unsigned short* dst = p.out + b * p.ob + (int64_t)qi * p.os + (int64_t)(head0 + hg) * D + lq * 4;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                bf16x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = (bf16_t)(l == 0.0f ? 0.0f : R.o[t][d][r] * inv);
                *reinterpret_cast<bf16x4*>(dst + d * 16) = v;
            }
        } else {
            const int64_t row = (int64_t)split * rows_all + part_row0 + in;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(p.part + row * D + d * 16 + lq * 4) = R.o[t][d];
            if (lq == 0) {
                float* ml = p.part + (int64_t)p.splits * rows_all * D + row * 2;
                ml[0] = R.m[t];
                ml[1] = l;
            }
        }
    }
}

// ---- 128 or 64 rows per workgroup --------------------------------------------------------------------------------------------------
// Bound by issue slots, not by memory or the matrix pipe: for one wave of 32 rows and a 32-key block at D = 128 the matrix instructions
// take 544 clocks of about 1240, the softmax 98 vector and 74 scalar instructions; two waves of a SIMD cover each other in part (matrix
// pipe busy 44 %).  974 TFLOP/s at 28 / 4 heads, 8192 tokens, D = 128 (988 us); 844 at 32 / 32 heads, 4096 tokens (326 us; cap 369 us,
// bias 324 us); 785 at D = 64 (2 x 32 heads, 4096 tokens: 350 us), where ea_attention_fwd_bf16's loop reaches 1288 on long sequences: it
// overlaps blocks inside a wave and keeps no maximum per block, this one overlaps waves only.  At D = 64 the registers of three workgroups
// per CU are given room for: 485 against 554 us with a cap, 424 against 533 us with a bias, 621 against 724 us with both (which costs 20
// bytes of scratch).  Measured and not taken in this loop: a tile's two blocks overlapped inside a wave of 32 rows (spills at D = 128, 407
// against 364 us at D = 64; waves of 16 rows have the room), K fragments read a block ahead, and requests spread between the
// instructions (343 against 333 us).
constexpr int TKEYS = 64;
// floats per head of a tile's bias window: its 64 keys against every query of the row tile
__host__ __device__ __forceinline__ int bias_window(int trows, int pack) { return TKEYS + (trows - 1) / pack + 2; }

template <int D, int RT, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attention_text_kernel(TextArgs p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr int TROWS = 64 * RT;
    constexpr int OPER = TKEYS * 2 * D;                 // one operand tile, bytes
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, lq = lane >> 4;
    // heads vary fastest, long (late) row tiles first: workgroups of one K / V head tend to share an XCD, causal work is dealt evenly
    const int nsets = p.Hq / p.pack;                    // packed head sets per batch element
    const int set_all = blockIdx.x % (nsets * p.B), tile = p.row_tiles - 1 - blockIdx.x / (nsets * p.B);
    const int b = set_all / nsets, set = set_all % nsets;
    const int head0 = set * p.pack, hk = head0 / p.group;
    const int split = RT == 2 ? 0 : blockIdx.y, splits = RT == 2 ? 1 : p.splits;
    const int rows = p.Sq * p.pack;
    const int q_first = tile * TROWS / p.pack;
    const int q_last = min((tile * TROWS + TROWS - 1) / p.pack, p.Sq - 1);
    const int win = BIAS ? bias_window(TROWS, p.pack) : 1;

    const Seq seq = seq_of(p, b);

    // ---- the workgroup's keys: up to the greatest limit (the limit grows with the query), documents of its queries
    const int lim_all = key_limit(p, seq, q_last);
    const int nt = (lim_all + TKEYS - 1) / TKEYS;
    TileWalk walk;
    walk.range = nullptr;
    walk.dlo = walk.dhi = 0;
    if (p.q_docs) {
        int lo = 0x7fffffff, hi = -0x7fffffff - 1;
        for (int i = q_first + lane; i <= q_last; i += 64) {
            const int id = p.q_docs[b * p.qd_ld + i];
            lo = min(lo, id);
            hi = max(hi, id);
        }
        walk.dlo = __builtin_amdgcn_readfirstlane(wave_min(lo));
        walk.dhi = __builtin_amdgcn_readfirstlane(wave_max(hi));
        walk.range = p.doc_range + (int64_t)b * p.key_tiles * 2;
    }
    walk.start((int)((int64_t)nt * split / splits), (int)((int64_t)nt * (split + 1) / splits), lane);

    const unsigned short* Kh = p.k + b * p.kb + (int64_t)hk * p.kh;
    const unsigned short* Vh = p.v + b * p.vb + (int64_t)hk * p.vh;
    // a tile's requests in two parts (K, V), so that neither stands in front of much arithmetic as one burst.  A piece is 1 KiB = PER
    // rows; of the swizzle's row bits two lie inside a piece and bit 3 is the same for a piece: i / 2 (D = 128: 4 rows), i (D = 64: 8).
    constexpr int PER = 64 / (D / 8), PIECES = TKEYS / PER / 4;
    const int vr = wave * PIECES * PER + lane / (D / 8), vc = (lane % (D / 8)) ^ swz<D>(lane / (D / 8));
    const int ks2 = (int)p.ks * 2, vs2 = (int)p.vs * 2;
    const int koff = vr * ks2 + vc * 16, voff = vr * vs2 + vc * 16;
    const int flip = ((vc ^ swz<D>(8)) - vc) * 16;                 // chunk offset of a piece whose rows have bit 3 set, minus the other's
    const unsigned lds_wave = lds_address(smem) + wave * PIECES * 1024;
    const int klane = k_lane<D>(lane), vlane = v_lane<D>(lane);
    auto issue = [&](int t, int stage, int part) {
        const unsigned to = lds_wave + (stage * 2 + part) * OPER;
        const int step2 = part ? vs2 : ks2, left = p.Sk - t * TKEYS;
        const u32x4_s rs = rows_resource<D>((part ? Vh : Kh) + (int64_t)t * (TKEYS / 2) * step2, part ? (int)p.vs : (int)p.ks, left < TKEYS ? left : TKEYS);
        int off = part ? voff : koff;
        asm volatile("" : "+v"(off));             // (the pieces' offsets are made here, not kept in registers over the loop)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) dma16(rs, off + ((i * PER) & 8 ? flip : 0) + i * PER * step2, to + i * 1024);
    };
    // bias window of tile t: entry w of head g = bias at distance 64 t - position(q_last) + w, in the log2 domain.  Finite values stay
    // finite there (the lowest float times log2 e would not): rows that are biased down as a whole keep their order.  Fetched in front of
    // a tile's requests, written behind the previous tile's arithmetic.
    float* wins = reinterpret_cast<float*>(smem + 4 * OPER + 512);
    const int64_t p_last = seq.first + q_last;
    constexpr int NB = BIAS ? 3 : 1;                  // entries per thread: pack * win <= 8 * 81
    int bsrc[NB], bw[NB];
    float bv[NB];
    if (BIAS) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int at = tid + 256 * i < p.pack * win ? tid + 256 * i : p.pack * win - 1;
            const int g = at / win;
            bw[i] = at - g * win;
            bsrc[i] = (head0 + g) * (2 * p.reach + 1) + p.reach;
        }
    }
    auto fetch_bias = [&](int t) {
        const int64_t far = (int64_t)t * TKEYS - p_last;
        const int from = far < -0x40000000 ? -0x40000000 : far > 0x40000000 ? 0x40000000 : (int)far;
#pragma unroll
        for (int i = 0; i < NB; ++i)
            if (256 * i < p.pack * win) {
                int dist = from + bw[i];
                dist = dist < -p.reach ? -p.reach : dist > p.reach ? p.reach : dist;
                bv[i] = p.bias[bsrc[i] + dist];
            }
    };
    auto write_bias = [&](int stage) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
            if (tid + 256 * i < p.pack * win) wins[stage * p.pack * win + tid + 256 * i] = log2_bias(bv[i]);
    };
    int* const tile_docs = reinterpret_cast<int*>(smem + 4 * OPER);      // [2][64]: the documents of a tile's keys
    auto issue_docs = [&](int t, int stage) {
        const int left = p.Sk - t * TKEYS;
        words_to_lds(p.kv_docs + b * p.kd_ld + t * TKEYS, left < TKEYS ? left : TKEYS, lane * 4, tile_docs + stage * 64);
    };

    int dlo, dhi, nlo = 0, nhi = 0;
    int t = walk.next(lane, dlo, dhi);
    int stage = 0;
    if (t >= 0) {
        if (BIAS) fetch_bias(t);
        issue(t, 0, 0);
        issue(t, 0, 1);
        if (p.q_docs && wave == 0) issue_docs(t, 0);
        if (BIAS) write_bias(0);
    }
    Rows<D, RT> R;                                     // (behind the first tile's requests: both are under way together)
    load_rows<D, RT>(p, R, seq, b, head0, tile * TROWS + wave * 16 * RT, q_last, win, lane);
    // One loop over 32-key blocks, two to a tile (nested loops made the compiler keep a second copy of the accumulators); with 64 rows
    // a tile that is visible as a whole takes both in one trip.
    int tn = -1, blk = 0;
    bool mine = false, masked = false;
    while (t >= 0) {
        const bool first_trip = blk == 0;
        if (first_trip) {
            tn = walk.next(lane, nlo, nhi);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (tn >= 0) {
                if (BIAS) fetch_bias(tn);
                issue(tn, stage ^ 1, 0);
                if (RT == 1) issue(tn, stage ^ 1, 1);
                if (p.q_docs && wave == 0) issue_docs(tn, stage ^ 1);
            }
            const int first = t * TKEYS;
            mine = __builtin_amdgcn_readfirstlane((int)(first < R.lim_hi && (!p.q_docs || (dlo <= R.doc_hi && dhi >= R.doc_lo)))) != 0;
            masked = __builtin_amdgcn_readfirstlane((int)!(first + TKEYS <= R.lim_lo && (!p.q_docs || (dlo == dhi && R.doc_lo == R.doc_hi && dlo == R.doc_lo)))) != 0;
        }
        const int at = stage * 2 * OPER + blk * 32 * (2 * D), key0 = t * TKEYS + blk * 32;
        const float* const win0 = wins + stage * p.pack * win + blk * 32 + 8 * lq;
        if (RT == 1 && mine && !masked && !(CAP && p.cap > CAP_WIDE)) {
            open_tile<D, RT, CAP, BIAS>(p, R, smem, at + klane, at + OPER + vlane, win0);
            blk = 1;
        } else if (mine) {
            bf16x8 kf[2][D / 32], pb[RT];
            u32x4_a vf[D / 16];
            float s[RT][8];
            read_k<D>(smem, at + klane, kf);
            block_qk<D, RT>(R, kf, s);
            read_v<D>(smem, at + OPER + vlane, vf);       // in flight under the softmax
            int docs[8];
            if (masked && p.q_docs) {
#pragma unroll
                for (int e = 0; e < 8; ++e) docs[e] = tile_docs[stage * 64 + blk * 32 + 8 * lq + e];
            }
            if (D == 128) __builtin_amdgcn_s_setprio(1);  // the vector pipe first: 4096 causal tokens 167 us, 173 without, 176 the other way round (no gain at 64)
            block_softmax<D, RT, CAP, BIAS>(p, R, s, pb, key0, masked, docs, win0, lane);
            if (D == 128) __builtin_amdgcn_s_setprio(0);
            if (masked && any_odd<D>(vf)) take_out_odd<D, RT>(R, vf, pb);
            block_pv<D, RT>(R, vf, pb);
        } else {
            blk = 1;
        }
        if (RT == 2 && first_trip && tn >= 0) issue(tn, stage ^ 1, 1);
        if (blk == 1) {
            if (BIAS && tn >= 0) write_bias(stage ^ 1);
            t = tn;
            dlo = nlo;
            dhi = nhi;
            stage ^= 1;
        }
        blk ^= 1;
    }
    store_rows<D, RT>(p, R, b, head0, (int64_t)set_all * rows, split, (int64_t)p.B * nsets * rows, tile * TROWS + wave * 16 * RT, lane);
}

// ---- up to 16 rows: the keys are what is long -----------------------------------------------------------------------------------
// Wave w of split s takes the 32-key blocks w, w + 4, .. of the split's range; its K fragments come straight from memory into registers
// (a row's 2 D bytes are read whole), its V block through a private double buffer in LDS.  No barrier until the four states are joined.
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void attention_text_few_kernel(TextArgs p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr int OPER = 32 * 2 * D;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lq = lane >> 4;
    const int nsets = p.Hq / p.pack;
    const int set_all = blockIdx.x % (nsets * p.B);
    const int b = set_all / nsets, set = set_all % nsets;
    const int head0 = set * p.pack, hk = head0 / p.group;
    const int split = blockIdx.y;
    const int rows = p.Sq * p.pack;
    const int win = 31 + p.Sq;                           // bias window of a block: its 32 keys against every query
    const Seq seq = seq_of(p, b);
    const int nb = (key_limit(p, seq, p.Sq - 1) + 31) / 32;
    const int b0 = (int)((int64_t)nb * split / p.splits), b1 = (int)((int64_t)nb * (split + 1) / p.splits);

    const unsigned short* Kh = p.k + b * p.kb + (int64_t)hk * p.kh;
    const unsigned short* Vh = p.v + b * p.vb + (int64_t)hk * p.vh;
    char* const mine = smem + wave * 2 * OPER;
    float* const win_mine = reinterpret_cast<float*>(smem + 8 * OPER) + wave * p.pack * win;
    const int64_t p_last = seq.first + p.Sq - 1;
    constexpr int PER = 64 / (D / 8), PIECES = 32 / PER;
    const int vr = lane / (D / 8), vc = (lane % (D / 8)) ^ swz<D>(vr), voff = vr * (int)p.vs * 2 + vc * 16;
    const int flip = ((vc ^ swz<D>(8)) - vc) * 16;
    auto load_k = [&](int blk, bf16x8 (&kf)[2][D / 32]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            int key = blk * 32 + 8 * (lr >> 2) + 4 * kt + (lr & 3);
            key = key < p.Sk ? key : p.Sk - 1;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) kf[kt][s] = *reinterpret_cast<const bf16x8*>(Kh + (int64_t)key * p.ks + (s * 4 + lq) * 8);
        }
    };
    const unsigned lds_mine = lds_address(mine);
    const int vlane = v_lane<D>(lane);
    auto load_v = [&](int blk, int stage) {
        const int left = p.Sk - blk * 32;
        const u32x4_s rs = rows_resource<D>(Vh + (int64_t)blk * 32 * p.vs, (int)p.vs, left < 32 ? left : 32);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) dma16(rs, voff + ((i * PER) & 8 ? flip : 0) + i * PER * (int)p.vs * 2, lds_mine + stage * OPER + i * 1024);
    };
    constexpr int NB = BIAS ? 5 : 1;                     // window entries per lane: pack * win <= 8 * 31 + 16
    int bsrc[NB], bw[NB];
    float bv[NB];
    if (BIAS) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int at = lane + 64 * i < p.pack * win ? lane + 64 * i : p.pack * win - 1, g = at / win;
            bw[i] = at - g * win;
            bsrc[i] = (head0 + g) * (2 * p.reach + 1) + p.reach;
        }
    }
    int docs[8];
    // a block's requests: what is small and looked at first (bias window, documents) in front
    auto request = [&](int blk, bf16x8 (&kf)[2][D / 32], int stage) {
        if (BIAS) {
            const int64_t far = (int64_t)blk * 32 - p_last;
            const int from = far < -0x40000000 ? -0x40000000 : far > 0x40000000 ? 0x40000000 : (int)far;
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (64 * i < p.pack * win) {
                    int dist = from + bw[i];
                    dist = dist < -p.reach ? -p.reach : dist > p.reach ? p.reach : dist;
                    bv[i] = p.bias[bsrc[i] + dist];
                }
        }
        if (p.q_docs) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = blk * 32 + 8 * lq + e;
                docs[e] = p.kv_docs[b * p.kd_ld + (key < p.Sk ? key : p.Sk - 1)];
            }
        }
        load_k(blk, kf);
        load_v(blk, stage);
    };
    bf16x8 kf[2][D / 32];
    int blk = b0 + wave, stage = 0;
    if (blk < b1) request(blk, kf, 0);
    Rows<D, 1> R;                                        // (behind the first block's requests)
    load_rows<D, 1>(p, R, seq, b, head0, 0, p.Sq - 1, win, lane);
    for (; blk < b1; blk += 4, stage ^= 1) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        bf16x8 now[2][D / 32];
        int now_docs[8];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int s = 0; s < D / 32; ++s) now[kt][s] = kf[kt][s];
#pragma unroll
        for (int e = 0; e < 8; ++e) now_docs[e] = docs[e];
        if (BIAS) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (lane + 64 * i < p.pack * win) win_mine[lane + 64 * i] = log2_bias(bv[i]);
        }
        if (blk + 4 < b1) request(blk + 4, kf, stage ^ 1);
        const int key0 = blk * 32;
        const bool masked = key0 + 32 > R.lim_lo || p.q_docs;
        if (BIAS) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        float s[1][8];
        bf16x8 pb[1];
        u32x4_a vf[D / 16];
        read_v<D>(smem, wave * 2 * OPER + stage * OPER + vlane, vf);
        block_qk<D, 1>(R, now, s);
        block_softmax<D, 1, CAP, BIAS>(p, R, s, pb, key0, masked, now_docs, win_mine + 8 * lq, lane);
        if (masked && any_odd<D>(vf)) take_out_odd<D, 1>(R, vf, pb);
        block_pv<D, 1>(R, vf, pb);
    }
    // ---- join the four waves' states through LDS: wave 0 takes the others in their order
    __syncthreads();
    constexpr int NT = D / 16;
    f32x4* const ox = reinterpret_cast<f32x4*>(smem);                  // [3][NT][64]: 3 x 16 x D floats, inside the V buffers
    float* const mx = reinterpret_cast<float*>(smem + 3 * NT * 64 * 16);   // [3][2][64]
    if (wave > 0) {
#pragma unroll
        for (int d = 0; d < NT; ++d) ox[((wave - 1) * NT + d) * 64 + lane] = R.o[0][d];
        mx[(wave - 1) * 128 + lane] = R.m[0];
        mx[(wave - 1) * 128 + 64 + lane] = R.l[0][0];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
        const float m2 = mx[w * 128 + lane], l2 = mx[w * 128 + 64 + lane];
        const float n = fmaxf(R.m[0], m2), ref = n == NEG_INF ? 0.0f : n;
        const float a1 = __builtin_amdgcn_exp2f(R.m[0] - ref), a2 = __builtin_amdgcn_exp2f(m2 - ref);
        R.m[0] = n;
        R.l[0][0] = R.l[0][0] * a1 + l2 * a2;
#pragma unroll
        for (int d = 0; d < NT; ++d) R.o[0][d] = R.o[0][d] * a1 + ox[(w * NT + d) * 64 + lane] * a2;
    }
    store_rows<D, 1>(p, R, b, head0, (int64_t)set_all * rows, split, (int64_t)p.B * nsets * rows, 0, lane);
}

// ---- the splits' partial results joined, in the order of the splits: up to 12 splits D / 4 threads per row (8400 rows, 3 splits: 24 us
// with the attention, 31 with a workgroup per row), else a workgroup per row (448 rows, 64 splits: 23 us, 31 the other way)
constexpr int MAX_SPLITS = 256;
template <int D>
__device__ __forceinline__ unsigned short* out_row_of(const TextArgs& p, const int64_t row) {
    // row = ((b * sets + set) * Sq + query) * pack + head of the set
    const int64_t rows = (int64_t)p.Sq * p.pack;
    const int nsets = p.Hq / p.pack;
    const int64_t set_all = row / rows;
    const int in = (int)(row - set_all * rows), qi = in / p.pack, hg = in % p.pack;
    const int64_t b = set_all / nsets;
    return p.out + b * p.ob + (int64_t)qi * p.os + (int64_t)((int)(set_all % nsets) * p.pack + hg) * D;
}

template <int D>
__global__ __launch_bounds__(256) void attention_text_join_rows_kernel(TextArgs p) {
    const int64_t rows_all = (int64_t)p.B * p.Hq * p.Sq, row = (int64_t)blockIdx.x * (1024 / D) + threadIdx.x / (D / 4);
    if (row >= rows_all) return;
    const int d = threadIdx.x % (D / 4) * 4;
    const float* src = p.part + row * D + d;
    const float* ml = p.part + (int64_t)p.splits * rows_all * D + row * 2;
    float m = NEG_INF, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[(int64_t)s * rows_all * 2]);
    const float ref = m == NEG_INF ? 0.0f : m;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = __builtin_amdgcn_exp2f(ml[(int64_t)s * rows_all * 2] - ref);
        l += ml[(int64_t)s * rows_all * 2 + 1] * w;
        o += *reinterpret_cast<const f32x4*>(src + (int64_t)s * rows_all * D) * w;
    }
    bf16x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (bf16_t)(l == 0.0f ? 0.0f : o[r] / l);
    *reinterpret_cast<bf16x4*>(out_row_of<D>(p, row) + d) = v;
}

// The splits' weights first (one thread each), then 256 / D threads per output element, each taking every (256 / D)-th split, and their
// sums in a fixed order.
template <int D>
__global__ __launch_bounds__(256) void attention_text_join_kernel(TextArgs p) {
    constexpr int PARTS = 256 / D;
    __shared__ float wm[MAX_SPLITS], wl[MAX_SPLITS], o_part[PARTS][D];
    const int tid = threadIdx.x;
    const int64_t rows_all = (int64_t)p.B * p.Hq * p.Sq, row = blockIdx.x;
    const float* ml = p.part + (int64_t)p.splits * rows_all * D;
    if (tid < p.splits) {
        wm[tid] = ml[((int64_t)tid * rows_all + row) * 2];
        wl[tid] = ml[((int64_t)tid * rows_all + row) * 2 + 1];
    }
    __syncthreads();
    float top = NEG_INF;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, wm[s]);
    const float ref = top == NEG_INF ? 0.0f : top;
    __syncthreads();
    if (tid < p.splits) wm[tid] = __builtin_amdgcn_exp2f(wm[tid] - ref);
    __syncthreads();
    const int d = tid % D, part = tid / D;
    const float* src = p.part + row * D + d;
    float o = 0.f, l = 0.f;
#pragma unroll 8
    for (int s = part; s < p.splits; s += PARTS) o += src[(int64_t)s * rows_all * D] * wm[s];
    o_part[part][d] = o;
    for (int s = 0; s < p.splits; ++s) l += wl[s] * wm[s];
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) o += o_part[i][d];
    out_row_of<D>(p, row)[d] = f32_to_bf16_bits(l == 0.0f ? 0.0f : o / l);
}

// least and greatest document of every 64-key tile: one wave each
__global__ __launch_bounds__(64) void doc_range_kernel(const int* __restrict__ docs, int* __restrict__ range, int64_t ld, int Sk, int tiles) {
    const int t = blockIdx.x, b = blockIdx.y;
    int key = t * 64 + (int)threadIdx.x;
    key = key < Sk ? key : Sk - 1;
    const int id = docs[b * ld + key];
    const int lo = wave_min(id), hi = wave_max(id);
    if (threadIdx.x == 0) {
        range[((int64_t)b * tiles + t) * 2] = lo;
        range[((int64_t)b * tiles + t) * 2 + 1] = hi;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct Plan {
    int group, pack, few, rt, row_tiles, key_tiles, splits;
    int64_t part_bytes, range_bytes;
};

Plan plan_of(int B, int Hq, int Hkv, int Sq, int Sk, int D, int docs, int causal) {
    Plan n;
    n.group = Hq / Hkv;
    n.pack = n.group < BIAS_PACK_MAX ? n.group : BIAS_PACK_MAX;
    while (n.group % n.pack) --n.pack;                    // the largest divisor of the group up to BIAS_PACK_MAX
    const int64_t rows = (int64_t)Sq * n.pack;
    const int64_t sets = (int64_t)B * (Hq / n.pack);
    n.few = rows <= 16;
    n.key_tiles = (int)(((int64_t)Sk + TKEYS - 1) / TKEYS);
    // 64 rows per workgroup while all of those run at once (two to a CU at D = 128, three at 64: 40 heads, 1024 tokens, D = 64, 640 of
    // them: 27 against 32 us; 28 heads, 2048 tokens, D = 128: 108 us in 896 of them, 76 in 448 of 128 rows), and in causal order over 16 or
    // more key tiles, where the longest workgroup sets the time, up to 1024 of them (32 heads, 2048 tokens, D = 64: 36 against 46 us; 28
    // heads, D = 128, 896: 56 against 63; 40 heads, D = 64, 1280: 49 against 48; 128 heads, 512 tokens, D = 64: 17.7 against 16.5)
    n.rt = sets * ((rows + 127) / 128) <= (causal && n.key_tiles >= 16 ? 512 : D == 64 ? 384 : 256) ? 1 : 2;
    n.row_tiles = n.few ? 1 : (int)((rows + 64 * n.rt - 1) / (64 * n.rt));
    // Split the keys while all workgroups still run at once (two to each of 256 CUs; 256 queries of 28 heads, 8192 keys: 64 us with 4
    // splits = 448 workgroups, 84 with 5) and a split keeps what pays for the join: 512 keys (128 queries, 4096 keys: 30 us; 38 with 256
    // keys, 33 with 1024), 256 where few rows are joined.  From 192 workgroups of whole tiles on the join costs more than is gained
    // (512 x 512: 15 against 24 us).
    const int64_t wgs = sets * n.row_tiles;
    int64_t s = 512 / wgs;
    const int64_t most = ((int64_t)Sk + 255) / (n.few ? 256 : 512);
    s = s < most ? s : most;
    s = s < 1 || (!n.few && wgs >= 192) ? 1 : s > MAX_SPLITS ? MAX_SPLITS : s;
    n.splits = (int)s;
    n.part_bytes = n.splits > 1 ? n.splits * sets * rows * (D + 2) * 4 : 0;
    n.range_bytes = docs && !n.few ? (int64_t)B * n.key_tiles * 8 : 0;
    return n;
}

template <int D, bool CAP, bool BIAS>
int launch_text(const TextArgs& p, const Plan& n, hipStream_t st) {
    const int oper = (n.few ? 32 : TKEYS) * 2 * D;
    const int win = !BIAS ? 0 : n.few ? (31 + p.Sq) * p.pack * 4 : bias_window(64 * n.rt, p.pack) * p.pack * 4;
    const int64_t sets = (int64_t)p.B * (p.Hq / p.pack);
    if (n.few) {
        const int tail = 3 * 16 * D * 4 + 3 * 2 * 64 * 4;                 // the join's image
        int lds = 8 * oper + 4 * win;
        lds = lds > tail ? lds : tail;
        if (hipFuncSetAttribute((const void*)attention_text_few_kernel<D, CAP, BIAS>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
            return ea_check_launch("ea_attention_text_bf16");
        ea_count("attention_text_few");
        hipLaunchKernelGGL((attention_text_few_kernel<D, CAP, BIAS>), dim3((unsigned)sets, (unsigned)n.splits), dim3(256), lds, st, p);
    } else {
        const int lds = 4 * oper + 512 + 2 * win;
        const auto kernel = n.rt == 1 ? attention_text_kernel<D, 1, CAP, BIAS> : attention_text_kernel<D, 2, CAP, BIAS>;
        if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
            return ea_check_launch("ea_attention_text_bf16");
        ea_count(n.rt == 2 ? "attention_text" : n.splits > 1 ? "attention_text_64_split" : "attention_text_64");      // (128 rows: never split)
        hipLaunchKernelGGL(kernel, dim3((unsigned)(sets * n.row_tiles), (unsigned)n.splits), dim3(256), lds, st, p);
    }
    if (n.splits > 1) {
        const int64_t rows_all = (int64_t)p.B * p.Hq * p.Sq;
        if (n.splits <= 12)
            hipLaunchKernelGGL(attention_text_join_rows_kernel<D>, dim3((unsigned)((rows_all + 1024 / D - 1) / (1024 / D))), dim3(256), 0, st, p);
        else
            hipLaunchKernelGGL(attention_text_join_kernel<D>, dim3((unsigned)rows_all), dim3(256), 0, st, p);
    }
    return ea_check_launch("ea_attention_text_bf16");
}

template <int D>
int dispatch_text(const TextArgs& p, const Plan& n, hipStream_t st) {
    if (p.cap > 0.0f) return p.bias ? launch_text<D, true, true>(p, n, st) : launch_text<D, true, false>(p, n, st);
    return p.bias ? launch_text<D, false, true>(p, n, st) : launch_text<D, false, false>(p, n, st);
}

bool sizes_ok(int B, int Hq, int Hkv, int Sq, int Sk, int D) {
    if (!(B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Sq >= 0 && Sk >= 0 && (D == 64 || D == 128))) return false;
    // rows of a packed set stay in 32 bits, grids within a launch's limits
    return (int64_t)Sq * BIAS_PACK_MAX <= 0x7fffff00 && Sk <= 0x7fffff00 && B <= 65535 && (int64_t)B * Hq * Sq <= 0x7fffffff && (int64_t)B * Hq < (1 << 24);
}

}  // namespace

extern "C" int64_t ea_attention_text_workspace_bytes(int batch, int q_heads, int kv_heads, int q_len, int kv_len, int head_dim, int documents) {
    if (!sizes_ok(batch, q_heads, kv_heads, q_len, kv_len, head_dim) || q_len == 0 || kv_len == 0) return 0;
    const Plan n = plan_of(batch, q_heads, kv_heads, q_len, kv_len, head_dim, documents, 0);
    return n.part_bytes + n.range_bytes;
}

extern "C" int ea_attention_text_bf16(const ea_bf16* q, const ea_bf16* k, const ea_bf16* v, ea_bf16* out, const int64_t* strides, int batch,
                                      int q_heads, int kv_heads, int q_len, int kv_len, int head_dim, float scale, int causal, float cap,
                                      const float* bias, int reach, const int* q_docs, const int* kv_docs, int64_t q_docs_ld, int64_t kv_docs_ld,
                                      const int* prefix, const int* valid, const int* q_start, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    EA_REQUIRE(head_dim == 64 || head_dim == 128, "ea_attention_text_bf16: head_dim %d (64 and 128 are built)", head_dim);
    EA_REQUIRE(sizes_ok(batch, q_heads, kv_heads, q_len, kv_len, head_dim),
               "ea_attention_text_bf16: bad sizes (batch %d, heads %d / %d, queries %d, keys %d)", batch, q_heads, kv_heads, q_len, kv_len);
    EA_REQUIRE(scale > 0.0f && scale <= 1e30f, "ea_attention_text_bf16: scale must be positive and at most 1e30");
    EA_REQUIRE(cap == 0.0f || (cap >= 1e-30f && cap <= 1e30f && scale / cap <= 1e30f),
               "ea_attention_text_bf16: cap must be 0 for none, or between 1e-30 and 1e30 and at least 1e-30 of the scale");
    EA_REQUIRE(!bias || (reach >= 0 && reach <= 0x3fffffff && (2 * (int64_t)reach + 1) * q_heads <= 0x7fffffff), "ea_attention_text_bf16: bad reach %d", reach);
    EA_REQUIRE((q_docs == nullptr) == (kv_docs == nullptr), "ea_attention_text_bf16: q_docs and kv_docs come together");
    EA_REQUIRE(!prefix || causal, "ea_attention_text_bf16: a prefix needs causal order");
    if (q_len == 0) return EA_OK;
    EA_REQUIRE(kv_len > 0, "ea_attention_text_bf16: no keys");
    EA_REQUIRE(q && k && v && out && strides, "ea_attention_text_bf16: null tensor");
    EA_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0, "ea_attention_text_bf16: 16-byte alignment");
    EA_REQUIRE(out != q && out != k && out != v, "ea_attention_text_bf16: out must not overlap q, k or v");
    for (int i = 0; i < 11; ++i)
        EA_REQUIRE(strides[i] % 8 == 0 && strides[i] >= 0, "ea_attention_text_bf16: strides must be non-negative multiples of 8 elements");
    EA_REQUIRE((batch == 1 || strides[9] >= (int64_t)q_heads * head_dim) && (q_len == 1 || strides[10] >= (int64_t)q_heads * head_dim),
               "ea_attention_text_bf16: rows of out overlap (strides %lld, %lld)", (long long)strides[9], (long long)strides[10]);
    EA_REQUIRE(strides[5] < (1 << 24) && strides[8] < (1 << 24), "ea_attention_text_bf16: row strides of k and v must be below 2^24 elements");
    const Plan n = plan_of(batch, q_heads, kv_heads, q_len, kv_len, head_dim, q_docs != nullptr, causal);
    EA_REQUIRE(n.part_bytes + n.range_bytes == 0 ||
                   (workspace && workspace_bytes >= n.part_bytes + n.range_bytes && (uintptr_t)workspace % 16 == 0),
               "ea_attention_text_bf16: needs %lld bytes of 16-byte aligned workspace (ea_attention_text_workspace_bytes)",
               (long long)(n.part_bytes + n.range_bytes));
    TextArgs p;
    p.q = q; p.k = k; p.v = v; p.out = out; p.bias = bias; p.q_docs = q_docs; p.kv_docs = kv_docs; p.prefix = prefix; p.valid = valid;
    p.q_start = q_start;
    p.part = reinterpret_cast<float*>(workspace);
    int* range = reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + n.part_bytes);
    p.doc_range = range;
    p.qb = strides[0]; p.qh = strides[1]; p.qs = strides[2];
    p.kb = strides[3]; p.kh = strides[4]; p.ks = strides[5];
    p.vb = strides[6]; p.vh = strides[7]; p.vs = strides[8];
    p.ob = strides[9]; p.os = strides[10];
    p.qd_ld = q_docs_ld; p.kd_ld = kv_docs_ld;
    p.B = batch; p.Hq = q_heads; p.Hkv = kv_heads; p.Sq = q_len; p.Sk = kv_len; p.group = n.group; p.pack = n.pack;
    p.causal = causal; p.reach = reach; p.splits = n.splits; p.row_tiles = n.row_tiles; p.key_tiles = n.key_tiles;
    p.scale = scale; p.cap = cap;
    hipStream_t st = (hipStream_t)stream;
    if (n.range_bytes)
        hipLaunchKernelGGL(doc_range_kernel, dim3((unsigned)n.key_tiles, (unsigned)batch), dim3(64), 0, st, kv_docs, range, kv_docs_ld, kv_len,
                           n.key_tiles);
    return head_dim == 128 ? dispatch_text<128>(p, n, st) : dispatch_text<64>(p, n, st);
}
