// HSTU attention of the newest positions against a K/V cache held in 4 bits, in pages.
//
// All matrix work is on v_mfma_f32_16x16x32, transposed as in hstu_common.h so that the scores never leave their lanes:
//
//   S^T[pos, row] = K[pos, :] . Q[row, :]^T     A = K, B = Q (registers, loaded once)
//   O^T[d, row]  += V^T[d, pos] . P^T[pos, row] A = V^T, B = P^T (registers)
//
// Both A operands come straight from the packed rows, with no LDS between: which of its 32 depths a lane's eight slots stand for
// is free as long as A and B agree.  K: lane (m, g) holds the words NK g .. of position m, a word being the eight depths of one
// product, in the order in which unpacking yields them (pairs four columns apart: one AND-OR makes two columns).  V: lane (m, g)
// holds the same NV = dv / 16 columns of eight positions (the eight that its scores have), so one permute joins the halves of two
// positions' words and the AND-ORs then yield (position, position + 1) pairs of each column: about one instruction per value.
//
// A code c enters a product as the float OFF + c, OFF the power of two whose mantissa step is where the code's bits lie (exact).
// What OFF adds is taken out again in fp32: from S by starting the accumulator at -sum(q OFF), from O through psum, the sum of the
// rounded P as one more product sees it (a row of ones).  With step s and lowest value l of a row
//     <q, k> = s (acc) + l sum(q),     O = sum_pos (P s) (c - 7.5) + sum_pos P (l + 7.5 s),
// the first sum on the matrix cores with P s rounded to bf16, the second in fp32: around the middle code the rounding of P s weighs
// a third of what it would around the lowest value.  For fp16 results, and for few rows, P s is kept in two bf16 words (16 bits, and bf16's
// range): results are then as far from 64 bits as rounding them leaves them.  For more rows in bf16 it is one word, as in the attention on 16-bit K and V: results
// are 0.0024 of their size from 64 bits, where rounding them alone leaves 0.0017.  Two words are twice the second product's instructions there:
// 12 rows of 256 sequences of 1000 .. 8192, four heads of 128, 189 -> 202 us, 24 rows 349 -> 387, 256 rows of 32 sequences of 1280 .. 4352 92 -> 107.
#pragma once
#include "hstu_paged_rows.h"

namespace hstu {

typedef __attribute__((ext_vector_type(8))) __bf16 pa_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 pa_f16x8;
typedef __attribute__((ext_vector_type(4))) float pa_f32x4;

struct PagedAttentionParams {
    PagedCache cache;
    const char* q;
    int64_t q_rs, q_hs;
    char* out;
    const void *lengths, *targets;
    int lengths_i64, targets_i64;
    int group, delta, w, c;  // heads of q to one of the cache; max_attn_len, contextual_seq_len
    float c1, oscale;        // t = c1 <q, k> with c1 = -alpha log2(e);  out = oscale * sum t / (1 + 2^t) v
    int share;  // step kernel: waves to a run, 4 (a workgroup) or 1
    int row_blocks, splits, run, items;  // run: chunks of one of the splits, at least
    float* partial;          // [splits][batch * delta][q heads][dv], used where splits > 1
    int64_t partial_stride;
};

// What the rows of one block see, in chunks of 32 positions: those of [a0, a0 + na), then those of [b0, b0 + nb).
struct PagedSpan {
    int n, u;  // length and its part that is no target
    int a0, na, b0, nb;
    int seen;  // the first position that a row sees: pages that end in front of it need not be there
    bool bad;  // the sequence has no room in the page table
};

// Rows i0 .. i1 - 1 of the newest `delta` positions of sequence b.
__device__ __forceinline__ PagedSpan paged_span(const PagedAttentionParams& p, int b, int i0, int i1) {
    PagedSpan s;
    const int64_t n64 = index_at(p.lengths, p.lengths_i64, b), room = (int64_t)p.cache.table_columns << p.cache.page_shift;
    s.bad = n64 > room || n64 > (1 << 30);
    s.n = s.bad || n64 < 0 ? 0 : (int)n64;
    int64_t t = p.targets ? index_at(p.targets, p.targets_i64, b) : 0;
    t = t < 0 ? 0 : t > s.n ? s.n : t;
    s.u = s.n - (int)t;
    const int first = max(s.n - p.delta + i0, 0), end = s.n - p.delta + i1;  // positions of the rows
    s.a0 = s.na = s.b0 = s.nb = s.seen = 0;
    if (end <= first) return s;
    const bool contextual = first < p.c;
    const int a_end = contextual ? max(s.u, min(end, s.u)) : min(end, s.u);
    const int id = min(p.c ? first - p.c + 1 : first, p.c ? s.u - p.c + 1 : s.u);  // of the first row: the others' are not less
    const int from = p.w > 0 && !contextual && id > p.w ? max(0, id - p.w + (p.c ? p.c - 1 : 0)) : 0;
    s.seen = from;
    if (a_end > from) s.a0 = from >> 5, s.na = ((a_end + 31) >> 5) - s.a0;
    else s.seen = max(s.u, first);
    if (end > s.u) {  // targets: the positions that only they themselves see
        const int self = max(s.u, first), done = s.a0 + s.na;
        s.b0 = max(self >> 5, s.na ? done : 0);
        s.nb = max(((end + 31) >> 5) - s.b0, 0);
    }
    return s;
}

// Chunks of a run: `run`, or more where the splits would not do; an even number.
__device__ __forceinline__ int chunks_per_run(const PagedAttentionParams& p, int chunks) { return (max(p.run, (chunks + p.splits - 1) / p.splits) + 1) & ~1; }

// What one row sees: positions [lo, hi), [0, chi) and itself.
struct RowSpan {
    int lo, hi, chi, self;
    __device__ __forceinline__ bool sees(int pos) const { return ((pos >= lo) & (pos < hi)) | (pos < chi) | (pos == self); }
};

__device__ __forceinline__ RowSpan row_span(const PagedAttentionParams& p, const PagedSpan& s, int pos) {
    RowSpan r;
    if (pos < 0) {
        r.lo = r.hi = r.chi = 0, r.self = -1;
    } else if (p.c == 0) {
        const int id = min(pos, s.u);
        r.hi = id, r.chi = 0, r.self = pos;
        r.lo = p.w > 0 ? max(0, id - p.w) : 0;
    } else if (pos < p.c) {
        r.lo = 0, r.hi = s.u, r.chi = 0, r.self = pos;
    } else {
        const int id = min(pos - p.c + 1, s.u - p.c + 1);
        r.hi = id + p.c - 1, r.self = pos;
        r.chi = id > 0 && (p.w <= 0 || id <= p.w) ? p.c : 0;
        r.lo = p.w > 0 ? max(p.c, id - p.w + p.c - 1) : p.c;
        if (r.chi && r.lo <= p.c) r.lo = 0;
    }
    return r;
}

// Codes as the floats OFF + code, two to a word: column k and column k + 4 of a word of eight, k = 0 .. 3.  AND and OR are one
// instruction, which takes one scalar and no literal: mask and offset are kept in a scalar and a vector register, and their values from the
// compiler, which would make two instructions with literals of it.  (The instruction itself in an asm block is no way: a product that
// reads its result needs wait states that the compiler does not count there.)
__device__ __forceinline__ unsigned kept_scalar(unsigned x) {
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ unsigned kept_vector(unsigned x) {
    asm("" : "+v"(x));
    return x;
}
// Rows that are the same for all lanes, read at a lane's 32-bit offset: by buffer loads, which add the two themselves (with global loads the
// compiler spends two registers and two instructions on each address).  The rows end `bytes` behind the pointer.
typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
struct UniformRows {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ UniformRows(const char* rows, unsigned bytes)
        : r(__builtin_amdgcn_make_buffer_rsrc((void*)rows, 0, (int)bytes, 0x00027000)) {}
    template <class V>
    __device__ __forceinline__ V at(unsigned offset) const {
        if constexpr (sizeof(V) == 16) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, (int)offset, 0, 0));
        else if constexpr (sizeof(V) == 8) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, (int)offset, 0, 0));
        else if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(r, (int)offset, 0, 0));
        else if constexpr (sizeof(V) == 2) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b16(r, (int)offset, 0, 0));
        else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b8(r, (int)offset, 0, 0));
    }
};
struct CodesBf16 {  // 128 + code where the code lies at bit 0, 16 + code from bit 3
    unsigned mask0, bits0, mask, bits;
    __device__ __forceinline__ CodesBf16()
        : mask0(kept_scalar(0x000F000Fu)), bits0(kept_vector(0x43004300u)), mask(kept_scalar(0x00780078u)), bits(kept_vector(0x41804180u)) {}
    __device__ __forceinline__ void four(unsigned w, unsigned (&o)[4]) const {
        o[0] = (w & mask0) | bits0;
        o[1] = ((w >> 1) & mask) | bits;
        o[2] = ((w >> 5) & mask) | bits;
        o[3] = ((w >> 9) & mask) | bits;
    }
    static __device__ __forceinline__ constexpr float off(int k) { return k == 0 ? 128.f : 16.f; }
};
struct CodesF16 {  // 64 + code, the code at bit 4
    unsigned mask, bits;
    __device__ __forceinline__ CodesF16() : mask(kept_scalar(0x00F000F0u)), bits(kept_vector(0x54005400u)) {}
    __device__ __forceinline__ void four(unsigned w, unsigned (&o)[4]) const {
        o[0] = ((w << 4) & mask) | bits;
        o[1] = (w & mask) | bits;
        o[2] = ((w >> 4) & mask) | bits;
        o[3] = ((w >> 8) & mask) | bits;
    }
    static __device__ __forceinline__ constexpr float off(int) { return 64.f; }
};

struct PagedBf16 {
    typedef __bf16 elem;
    typedef CodesBf16 codes;
    static constexpr int P_WORDS = 1;
    static __device__ __forceinline__ pa_f32x4 mma(u32x4_t a, u32x4_t b, pa_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, a), __builtin_bit_cast(pa_bf16x8, b), c, 0, 0, 0);
    }
};
struct PagedF16 {
    typedef _Float16 elem;
    typedef CodesF16 codes;
    static constexpr int P_WORDS = 2;
    static __device__ __forceinline__ pa_f32x4 mma(u32x4_t a, u32x4_t b, pa_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_f16x8, a), __builtin_bit_cast(pa_f16x8, b), c, 0, 0, 0);
    }
};

// The packed rows of 32 positions as one wave holds them, and their steps and lowest values: lane (m, g) has K of positions m and
// 16 + m, V of positions 4 g + i and 16 + 4 g + i, and the pairs of the latter positions.
template <int NK, int NV>
struct PagedChunk {
    static constexpr int VW = NV == 16 ? 2 : 1;
    unsigned k[2][NK], v[8][VW];
    u32x4_t ks[2], vs[2];
    // Tile tt from `row` of the cache on.
    __device__ __forceinline__ void load(const PagedCache& c, int64_t row, int tt, int lane) {
        constexpr int KROW = 16 * NK, VROW = 8 * NV;  // bytes
        const unsigned m = lane & 15, g = lane >> 4;
        const UniformRows kr(c.k_codes + row * KROW, 16 * KROW), vr(c.v_codes + row * VROW, 16 * VROW), ksr(c.k_scales + row * 4, 64), vsr(c.v_scales + row * 4, 64);
        const unsigned k_lane = m * KROW + g * (4 * NK), v_lane = 4 * g * VROW + m * (NV / 2);
        if constexpr (NK == 1) {
            k[tt][0] = kr.template at<unsigned>(k_lane);
        } else if constexpr (NK == 2) {
            const u32x2_t a = kr.template at<u32x2_t>(k_lane);
            k[tt][0] = a.x, k[tt][1] = a.y;
        } else {
#pragma unroll
            for (int j = 0; j < NK; j += 4) {
                const u32x4_t a = kr.template at<u32x4_t>(k_lane + 4 * j);
                k[tt][j] = a.x, k[tt][j + 1] = a.y, k[tt][j + 2] = a.z, k[tt][j + 3] = a.w;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned at = v_lane + i * VROW;
            if constexpr (NV == 2) v[4 * tt + i][0] = vr.template at<unsigned char>(at);
            else if constexpr (NV == 4) v[4 * tt + i][0] = vr.template at<unsigned short>(at);
            else {
#pragma unroll
                for (int j = 0; j < VW; ++j) v[4 * tt + i][j] = vr.template at<unsigned>(at + 4 * j);
            }
        }
        ks[tt] = ksr.template at<u32x4_t>(16 * g), vs[tt] = vsr.template at<u32x4_t>(16 * g);
    }
};

// NV columns each at 4 places NV apart: to the run's partial sums, or scaled to the result.
template <class T, int NV>
__device__ __forceinline__ void store_columns(const PagedAttentionParams& p, int split, int64_t at, const float (&o)[4][NV]) {
    if (p.splits > 1) {
        float* to = p.partial + split * p.partial_stride + at;
#pragma unroll
        for (int i = 0; i < 4 * NV; i += 4) *(pa_f32x4*)(to + i) = pa_f32x4{o[i / NV][i % NV], o[(i + 1) / NV][(i + 1) % NV], o[(i + 2) / NV][(i + 2) % NV], o[(i + 3) / NV][(i + 3) % NV]};
    } else {
        typedef __attribute__((ext_vector_type(8))) T T8;
        T* to = (T*)p.out + at;
#pragma unroll
        for (int i = 0; i < 4 * NV; i += 8) {
            T8 x;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (T)(o[(i + k) / NV][(i + k) % NV] * p.oscale);
            *(T8*)(to + i) = x;
        }
    }
}

// grid: one workgroup of four waves per (head of the cache, run, sequence); its 16 MT rows are all that share a head.  The waves share out the
// chunks of the run; their sums meet in LDS.  Unpacking and silu
// take most of it, the cache's bytes not far below: 12 rows, 256 sequences of 1000 .. 8192 positions and four heads of 128 187 us (640 MB, 124 us
// of a copy), of whose 371 thousand clocks a SIMD has 173 of vector operations and 39 of products (counted): no unit is full, waves wait for
// 45 % of their time and 28 % of the room for them stands empty, most of it while the longest sequences end.  24 rows, whose registers leave room for one
// wave of a SIMD, 350 (711 thousand, 240 and 77).  Held to two waves, with 85 registers spilled, they took a seventh longer;
// heads of 64 and 128, with seven, gained: 64 sequences of 512 .. 4096 46 us by one wave, 36 by two.
template <class TT, int DK, int DV, int MT>
__global__ __launch_bounds__(256, (MT == 2 && DK + DV < 256 ? 2 : 1)) void hstu_paged_attention_kernel(const PagedAttentionParams p) {
    typedef typename TT::elem T;
    constexpr int NK = DK / 32, NV = DV / 16, KW = 4;
    __shared__ float meet[KW * NV * 4 * 64];
    const int item = blockIdx.x;
    const int hk = item % p.cache.heads, split = (item / p.cache.heads) % p.splits, b = item / (p.cache.heads * p.splits);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int rows = p.delta * p.group;
    const PagedSpan span = paged_span(p, b, 0, p.delta);
    const int chunks = span.na + span.nb, per = chunks_per_run(p, chunks);
    const int chunk_end = min((split + 1) * per, chunks);
    if (p.splits > 1 && split * per >= chunks) return;  // (the joining kernel knows)

    u32x4_t qf[MT][NK];
    float qs[MT], qo[MT];
    RowSpan see[MT];
    int64_t out_at[MT];
    int lo_max = 0, hi_min = 1 << 30;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + m;
        const int i = r / p.group, head = hk * p.group + (r - i * p.group);
        qs[mt] = qo[mt] = 0.f;
        see[mt].lo = see[mt].hi = see[mt].chi = 0, see[mt].self = -1;
        out_at[mt] = -1;
        const int64_t row = (int64_t)b * p.delta + i;
        if (r < rows) {
            see[mt] = row_span(p, span, span.n - p.delta + i);
            out_at[mt] = (row * (p.cache.heads * p.group) + head) * DV;
            lo_max = max(lo_max, see[mt].lo), hi_min = min(hi_min, see[mt].hi);
        }
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            u32x4_t x = {0, 0, 0, 0};
            if (r < rows) x = *(const u32x4_t*)(p.q + (row * p.q_rs + head * p.q_hs + 8 * (NK * g + j)) * 2);
            // columns k and k + 4 side by side, as the codes come
            qf[mt][j] = u32x4_t{__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                                __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                typedef __attribute__((ext_vector_type(2))) T T2;
                const T2 two = __builtin_bit_cast(T2, (unsigned)qf[mt][j][k]);
                const float sum = (float)two[0] + (float)two[1];
                qs[mt] += sum, qo[mt] += sum * TT::codes::off(k);
            }
        }
        qs[mt] += __shfl_xor(qs[mt], 16, 64), qo[mt] += __shfl_xor(qo[mt], 16, 64);
        qs[mt] += __shfl_xor(qs[mt], 32, 64), qo[mt] += __shfl_xor(qo[mt], 32, 64);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) lo_max = max(lo_max, __shfl_xor(lo_max, d, 64)), hi_min = min(hi_min, __shfl_xor(hi_min, d, 64));
    lo_max = __builtin_amdgcn_readfirstlane(lo_max), hi_min = __builtin_amdgcn_readfirstlane(hi_min);

    pa_f32x4 acc[MT][NV], psum[MT];
    float plo[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        psum[mt] = pa_f32x4{0, 0, 0, 0}, plo[mt] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) acc[mt][j] = pa_f32x4{0, 0, 0, 0};
    }
    const typename TT::codes k_codes;
    const CodesBf16 v_codes;
    bool bad = span.bad;

    auto chunk_at = [&](int i) { return i < span.na ? span.a0 + i : span.b0 + (i - span.na); };
    auto work = [&](const PagedChunk<NK, NV>& x, int chunk, auto masked) __attribute__((always_inline)) {
        const int pos0 = chunk * 32 + 4 * g;
        float ka[8], kb[8], va[8], vm[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            typedef __attribute__((ext_vector_type(2))) T T2;
            const T2 k2 = __builtin_bit_cast(T2, (unsigned)x.ks[e >> 2][e & 3]), v2 = __builtin_bit_cast(T2, (unsigned)x.vs[e >> 2][e & 3]);
            ka[e] = p.c1 * (float)k2[0], kb[e] = p.c1 * (float)k2[1];
            va[e] = (float)v2[0], vm[e] = (float)v2[1] + 7.5f * (float)v2[0];
        }
        u32x4_t kf[2][NK], vf[NV];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                unsigned o[4];
                k_codes.four(x.k[tt][j], o);
                kf[tt][j] = u32x4_t{o[0], o[1], o[2], o[3]};
            }
#pragma unroll
        for (int pair = 0; pair < 4; ++pair)
#pragma unroll
            for (int h = 0; h < (NV + 3) / 4; ++h) {
                unsigned two, o[4];
                if constexpr (NV <= 4) two = x.v[2 * pair][0] | (x.v[2 * pair + 1][0] << 16);
                else two = __builtin_amdgcn_perm(x.v[2 * pair + 1][h >> 1], x.v[2 * pair][h >> 1], h & 1 ? 0x07060302u : 0x05040100u);
                v_codes.four(two, o);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (4 * h + k < NV) vf[4 * h + k][pair] = o[k];
            }
        const u32x4_t ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            pa_f32x4 s[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                s[tt] = pa_f32x4{-qo[mt], -qo[mt], -qo[mt], -qo[mt]};
#pragma unroll
                for (int j = 0; j < NK; ++j) s[tt] = TT::mma(kf[tt][j], qf[mt][j], s[tt]);
            }
            float ps[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = ka[e] * s[e >> 2][e & 3] + kb[e] * qs[mt];
                const float pr = t * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t));
                ps[e] = pr * va[e];
                float lower = __builtin_fmaf(pr, vm[e], plo[mt]);
                if constexpr (decltype(masked)::value) {
                    const bool seen = see[mt].sees(pos0 + (e >> 2) * 16 + (e & 3));
                    ps[e] = seen ? ps[e] : 0.f, lower = seen ? lower : plo[mt];
                }
                plo[mt] = lower;
            }
            pa_bf16x8 high;
#pragma unroll
            for (int e = 0; e < 8; ++e) high[e] = (__bf16)ps[e];
            const u32x4_t ph = __builtin_bit_cast(u32x4_t, high);
#pragma unroll
            for (int j = 0; j < NV; ++j) acc[mt][j] = PagedBf16::mma(vf[j], ph, acc[mt][j]);
            psum[mt] = PagedBf16::mma(ones, ph, psum[mt]);
            if constexpr (TT::P_WORDS == 2) {
                pa_bf16x8 rest;
#pragma unroll
                for (int e = 0; e < 8; ++e) rest[e] = (__bf16)(ps[e] - (float)high[e]);
                const u32x4_t pl = __builtin_bit_cast(u32x4_t, rest);
#pragma unroll
                for (int j = 0; j < NV; ++j) acc[mt][j] = PagedBf16::mma(vf[j], pl, acc[mt][j]);
                psum[mt] = PagedBf16::mma(ones, pl, psum[mt]);
            }
        }
    };

    // Pages of the two tiles of 32 of this wave's chunks, KW apart from chunk i on, one to a lane; what does not exist, or lies in front of all that is seen, has the first page.  Two
    // sets: the next one has been loaded when its turn comes.
    auto pages_of = [&](int i) __attribute__((always_inline)) {
        int page = 0;
        const int ci = i + KW * (lane >> 1), pos = ci < chunk_end ? chunk_at(ci) * 32 + (lane & 1) * 16 : span.n;
        if (pos < span.n && pos + 16 > span.seen) {
            const int64_t at = index_at(p.cache.page_table, p.cache.page_table_i64, b * p.cache.table_row_stride + (pos >> p.cache.page_shift));
            if (at < 0 || at >= p.cache.pages) bad = true;
            else page = (int)at;
        }
        return page;
    };
    PagedChunk<NK, NV> now, next;
    int i = split * per + wave, k = 0, page = pages_of(i), page_next = pages_of(i + 32 * KW);
    const int in_page = (1 << p.cache.page_shift) - 1;
    auto load = [&](PagedChunk<NK, NV>& x, int i, int k) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const int64_t pg = __builtin_amdgcn_readlane(page, 2 * (k & 31) + tt);
            x.load(p.cache, ((pg * p.cache.heads + hk) << p.cache.page_shift) + ((chunk_at(i) * 32 + tt * 16) & in_page), tt, lane);
        }
    };
    // One chunk, the next one's loads on their way.  Code of their own for chunks that all rows see whole, in a loop of their own: a condition at each
    // score would stand between them, and one around them would have the sums moved where its ways meet.
    auto one = [&](auto masked) __attribute__((always_inline)) {
        if (((k + 1) & 31) == 0) page = page_next, page_next = pages_of(i + KW + 32 * KW);
        if (i + KW < chunk_end) load(next, i + KW, k + 1);
        work(now, chunk_at(i), masked);
        now = next;
        i += KW, ++k;
    };
    const int whole0 = max(((lo_max + 31) >> 5) - span.a0, 0), whole1 = min((hi_min >> 5) - span.a0, span.na);
    if (i < chunk_end) load(now, i, 0);
    while (i < chunk_end && !(i >= whole0 && i < whole1)) one(std::true_type{});
    while (i < min(chunk_end, whole1)) one(std::false_type{});
    while (i < chunk_end) one(std::true_type{});
    bad = __any(bad);

#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float lower = plo[mt];
        lower += __shfl_xor(lower, 16, 64);
        lower += __shfl_xor(lower, 32, 64);
        if (bad) lower = __builtin_nanf("");
        float o[4][NV];  // [i][j]: column NV (4 g + i) + j
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
            for (int j = 0; j < NV; ++j) o[i4][j] = acc[mt][j][i4] - (CodesBf16::off(j & 3) + 7.5f) * psum[mt][i4] + lower;
        __syncthreads();
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
            for (int j = 0; j < NV; ++j) meet[((wave * 4 + i4) * NV + j) * 64 + lane] = o[i4][j];
        __syncthreads();
        // wave i4 adds up columns NV (4 g + i4) ..
        if (out_at[mt] >= 0) {
            const int64_t at = out_at[mt] + NV * (4 * g + wave);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < KW; ++w) x += meet[((w * 4 + wave) * NV + j) * 64 + lane];
                if (p.splits > 1) p.partial[split * p.partial_stride + at + j] = x;
                else ((T*)p.out)[at + j] = (T)(x * p.oscale);
            }
        }
    }
}

// Which part of the work this workgroup takes: sequence * each + (part of the sequence).  The longest sequences first, so that the last workgroups are
// short ones; and where all of them run at once, two to a CU, the second of a CU's is as short as its first is long.  Every workgroup ranks the lengths
// for itself, in LDS (256 of them take a microsecond); more sequences than that stay in their order.
__device__ __forceinline__ int block_order(const PagedAttentionParams& p, int each, int* lengths) {
    const int batch = p.cache.batch, total = batch * each;
    int at = blockIdx.x;
    if (batch > 256 || batch < 2) return at;
    if (total <= 512 && at >= 256) at = total - 1 - (at - 256);  // (of 256 .. 511 the last first)
    const int t = threadIdx.x;
    if (t < batch) {
        const int64_t n = index_at(p.lengths, p.lengths_i64, t);
        lengths[t] = n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : (int)n;
    }
    __syncthreads();
    if (t < batch) {
        const int n = lengths[t];
        int rank = 0;
        for (int i = 0; i < batch; ++i) rank += lengths[i] > n || (lengths[i] == n && i < t);
        lengths[256 + rank] = t;
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(lengths[256 + at / each]);
    __syncthreads();
    return b * each + at % each;
}

// The same for many rows: the four waves of a workgroup take 16 MT rows each and share what unpacking yields.  A step is 32 CH positions;
// each wave unpacks its part of them -- a tile of 16 positions of K, a quarter of the columns of V -- into LDS, in the order in which the
// products' operands lie in registers (a lane's 16 bytes side by side: reads and writes without bank conflicts), and the pairs as four
// floats a position: c1 s, c1 l of K, s, l + 7.5 s of V.  Two buffers, one barrier a step; the packed rows of the next step are on their way
// while this one is worked on.  Unpacking per wave, as above, cost as much as half of the rest and the registers of a second wave.
// For 32 positions and 32 rows a wave has 204 vector operations, 152 of them for silu, its masks and roundings, and 34 products.
// 32 sequences of 1280 .. 4352 positions with 256 rows and four heads of 128 (39 GFLOP, 32 us of the matrix cores as a large library
// product uses them): 88 us, 8 of them for joining two parts of each sequence.  No unit bounds it: of the kernel's 177 thousand clocks a SIMD has 71
// of vector operations and 41 of products (counted).  A wave lives 135 of them in the mean, because parts are parts of a sequence and the longest
// sequence has the longest, so that a quarter of the waves' room stands empty; the rest is waits, for which two waves of a SIMD
// are few.  Two workgroups of a CU, out of step with each
// other, fill the gaps of one another: the same two teams of waves in one workgroup, behind one barrier, took 106 us.  Three of 64 rows and
// one chunk a step took 91: more operations, nothing gained from a third wave.
template <class TT, int DK, int DV, int MT>
__global__ __launch_bounds__(256, 2) void hstu_paged_block_kernel(const PagedAttentionParams p) {
    typedef typename TT::elem T;
    typedef __attribute__((ext_vector_type(2))) T T2;
    constexpr int NK = DK / 32, NV = DV / 16, CH = DK == 256 ? 1 : 2, TILES = 2 * CH, HALVES = (NV + 3) / 4, KB = TILES * NK, VB = CH * NV;
    constexpr int V_UNITS = CH * HALVES, ROWS = 64 * MT;
    static_assert(TILES <= 4 && V_UNITS <= 4, "one unit of K and one of V to a wave");
    __shared__ u32x4_t frags[2][(KB + VB) * 64];
    __shared__ pa_f32x4 pairs[2][4][CH * 8];  // [buffer][which][position / 4]
    const PagedCache& c = p.cache;
    const int each = c.heads * p.row_blocks * p.splits, part = block_order(p, each, (int*)&frags[0][0]);
    const int b = part / each, rest = part - b * each, hk = rest % c.heads, rb = (rest / c.heads) % p.row_blocks, split = rest / (c.heads * p.row_blocks);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int rows = p.delta * p.group, r_end = min((rb + 1) * ROWS, rows);
    const PagedSpan span = paged_span(p, b, rb * ROWS / p.group, (r_end - 1) / p.group + 1);
    const int chunks = span.na + span.nb, per = chunks_per_run(p, chunks), begin = split * per, end = min(begin + per, chunks);
    if (p.splits > 1 && begin >= chunks) return;  // (the joining kernel knows)
    auto chunk_at = [&](int i) { return i < span.na ? span.a0 + i : span.b0 + (i - span.na); };

    // ---- unpacking ----
    const typename TT::codes k_codes;
    const CodesBf16 v_codes;
    const int in_page = (1 << c.page_shift) - 1;
    const unsigned k_lane = m * (DK / 2) + g * (4 * NK);
    const int v_chunk = wave / HALVES, v_half = wave % HALVES;  // of the wave's unit of V
    const unsigned v_lane = 4 * g * (DV / 2) + m * (NV / 2) + 2 * v_half;
    bool bad = span.bad;
    unsigned raw_k[NK], raw_v[8], raw_ks = 0, raw_vs = 0;
    // Pages of the 64 tiles of 16 positions from chunk ci on, one to a lane; what does not exist, or lies in front of all that is seen, has the first page.  Two sets: the next one
    // has been loaded when its turn comes.  (A page looked up where it is needed is two loads that the wave waits for, three times a step.)
    auto pages_of = [&](int ci) __attribute__((always_inline)) {
        int page = 0;
        const int pos = ci + (lane >> 1) < end ? chunk_at(ci + (lane >> 1)) * 32 + (lane & 1) * 16 : span.n;
        if (pos < span.n && pos + 16 > span.seen) {
            const int64_t at = index_at(c.page_table, c.page_table_i64, b * c.table_row_stride + (pos >> c.page_shift));
            if (at < 0 || at >= c.pages) bad = true;
            else page = (int)at;
        }
        return page;
    };
    int page_base = begin, page = 0, page_next = 0;
    if (begin < end) page = pages_of(begin), page_next = pages_of(begin + 32);
    // Row of the cache where the 16 positions of tile tt of chunk ci lie.
    auto row_of = [&](int ci, int tt) __attribute__((always_inline)) {
        ci = min(ci, end - 1);
        const int64_t pg = __builtin_amdgcn_readlane(page, 2 * (ci - page_base) + tt);
        return ((pg * c.heads + hk) << c.page_shift) + ((chunk_at(ci) * 32 + tt * 16) & in_page);
    };
    auto load = [&](int ci) __attribute__((always_inline)) {
        if (ci >= page_base + 32) page_base += 32, page = page_next, page_next = pages_of(page_base + 32);
        if (wave < TILES) {
            const int64_t row = row_of(ci + (wave >> 1), wave & 1);
            const UniformRows k(c.k_codes + row * (DK / 2), 16 * (DK / 2));
            if constexpr (NK == 1) {
                raw_k[0] = k.at<unsigned>(k_lane);
            } else if constexpr (NK == 2) {
                const u32x2_t a = k.at<u32x2_t>(k_lane);
                raw_k[0] = a.x, raw_k[1] = a.y;
            } else {
#pragma unroll
                for (int j = 0; j < NK; j += 4) {
                    const u32x4_t a = k.at<u32x4_t>(k_lane + 4 * j);
                    raw_k[j] = a.x, raw_k[j + 1] = a.y, raw_k[j + 2] = a.z, raw_k[j + 3] = a.w;
                }
            }
            const UniformRows ks(c.k_scales + row * 4, 64), vs(c.v_scales + row * 4, 64);
            raw_ks = ks.at<unsigned>(4 * m), raw_vs = vs.at<unsigned>(4 * m);
        }
        if (wave < V_UNITS) {
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const UniformRows v(c.v_codes + row_of(ci + v_chunk, tt) * (DV / 2), 16 * (DV / 2));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (NV == 2) raw_v[4 * tt + i] = v.at<unsigned char>(v_lane + i * (DV / 2));
                    else raw_v[4 * tt + i] = v.at<unsigned short>(v_lane + i * (DV / 2));
                }
            }
        }
    };
    auto unpack = [&](int buffer) __attribute__((always_inline)) {
        if (wave < TILES) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                unsigned o[4];
                k_codes.four(raw_k[j], o);
                frags[buffer][(wave * NK + j) * 64 + lane] = u32x4_t{o[0], o[1], o[2], o[3]};
            }
            const T2 k2 = __builtin_bit_cast(T2, raw_ks), v2 = __builtin_bit_cast(T2, raw_vs);
            float* out = (float*)&pairs[buffer][0][0] + g * (CH * 32) + wave * 16 + m;  // lane (m, g) writes one of the position's four
            const float ka = p.c1 * (float)k2[0], kb = p.c1 * (float)k2[1], va = (float)v2[0], vm = (float)v2[1] + 7.5f * (float)v2[0];
            *out = g == 0 ? ka : g == 1 ? kb : g == 2 ? va : vm;
        }
        if (wave < V_UNITS) {
            u32x4_t vf[4];
#pragma unroll
            for (int pair = 0; pair < 4; ++pair) {
                unsigned o[4];
                v_codes.four(raw_v[2 * pair] | (raw_v[2 * pair + 1] << 16), o);
#pragma unroll
                for (int k = 0; k < 4; ++k) vf[k][pair] = o[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (4 * v_half + k < NV) frags[buffer][(KB + v_chunk * NV + 4 * v_half + k) * 64 + lane] = vf[k];
        }
    };

    if (begin < end) load(begin);
    // ---- rows ----
    u32x4_t qf[MT][NK];
    float qs[MT], qo[MT];
    RowSpan see[MT];
    int64_t out_at[MT];
    int any_lo = 1 << 30, any_hi = 0, any_chi = 0, self_lo = 1 << 30, self_hi = -1;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = rb * ROWS + (wave * MT + mt) * 16 + m;
        const int i = r / p.group, head = hk * p.group + (r - i * p.group);
        qs[mt] = qo[mt] = 0.f;
        see[mt].lo = see[mt].hi = see[mt].chi = 0, see[mt].self = -1;
        out_at[mt] = -1;
        const int64_t row = (int64_t)b * p.delta + i;
        if (r < rows) {
            see[mt] = row_span(p, span, span.n - p.delta + i);
            out_at[mt] = (row * (c.heads * p.group) + head) * DV;
            any_lo = min(any_lo, see[mt].lo), any_hi = max(any_hi, see[mt].hi), any_chi = max(any_chi, see[mt].chi);
            if (see[mt].self >= 0) self_lo = min(self_lo, see[mt].self), self_hi = max(self_hi, see[mt].self);
        }
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            u32x4_t x = {0, 0, 0, 0};
            if (r < rows) x = *(const u32x4_t*)(p.q + (row * p.q_rs + head * p.q_hs + 8 * (NK * g + j)) * 2);
            // columns k and k + 4 side by side, as the codes come
            qf[mt][j] = u32x4_t{__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                                __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const T2 two = __builtin_bit_cast(T2, (unsigned)qf[mt][j][k]);
                const float sum = (float)two[0] + (float)two[1];
                qs[mt] += sum, qo[mt] += sum * TT::codes::off(k);
            }
        }
        qs[mt] += __shfl_xor(qs[mt], 16, 64), qo[mt] += __shfl_xor(qo[mt], 16, 64);
        qs[mt] += __shfl_xor(qs[mt], 32, 64), qo[mt] += __shfl_xor(qo[mt], 32, 64);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        any_lo = min(any_lo, __shfl_xor(any_lo, d, 64)), any_hi = max(any_hi, __shfl_xor(any_hi, d, 64)), any_chi = max(any_chi, __shfl_xor(any_chi, d, 64));
        self_lo = min(self_lo, __shfl_xor(self_lo, d, 64)), self_hi = max(self_hi, __shfl_xor(self_hi, d, 64));
    }
    any_lo = __builtin_amdgcn_readfirstlane(any_lo), any_hi = __builtin_amdgcn_readfirstlane(any_hi), any_chi = __builtin_amdgcn_readfirstlane(any_chi);
    self_lo = __builtin_amdgcn_readfirstlane(self_lo), self_hi = __builtin_amdgcn_readfirstlane(self_hi);

    pa_f32x4 acc[MT][NV], psum[MT], start[MT];
    float plo[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        start[mt] = pa_f32x4{-qo[mt], -qo[mt], -qo[mt], -qo[mt]};  // four registers of their own, not four moves for each tile
        asm("" : "+v"(start[mt]));
        psum[mt] = pa_f32x4{0, 0, 0, 0}, plo[mt] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) acc[mt][j] = pa_f32x4{0, 0, 0, 0};
    }
    const u32x4_t ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

    auto work_masked = [&](int buffer, int cc, int chunk, auto masked) __attribute__((always_inline)) {
        const int first = chunk * 32;
        pa_f32x4 s[MT][2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                const u32x4_t kf = frags[buffer][((2 * cc + tt) * NK + j) * 64 + lane];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][tt] = TT::mma(kf, qf[mt][j], j == 0 ? start[mt] : s[mt][tt]);
            }
        }
        // (V's operands are on their way while silu is worked on)
        u32x4_t vf[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) vf[j] = frags[buffer][(KB + cc * NV + j) * 64 + lane];
        u32x4_t ph[MT], pl[MT];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const int at = cc * 8 + tt * 4 + g;
            const pa_f32x4 ka = pairs[buffer][0][at], kb = pairs[buffer][1][at], va = pairs[buffer][2][at], vm = pairs[buffer][3][at];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float ps[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = ka[e] * s[mt][tt][e] + kb[e] * qs[mt];
                    const float pr = t * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t));
                    ps[e] = pr * va[e];
                    float lower = __builtin_fmaf(pr, vm[e], plo[mt]);
                    if constexpr (decltype(masked)::value) {
                        const bool seen = see[mt].sees(first + tt * 16 + 4 * g + e);
                        ps[e] = seen ? ps[e] : 0.f, lower = seen ? lower : plo[mt];
                    }
                    plo[mt] = lower;
                }
                typedef __attribute__((ext_vector_type(4))) __bf16 b4;
                b4 high;
#pragma unroll
                for (int e = 0; e < 4; ++e) high[e] = (__bf16)ps[e];
                const u32x2_t h2 = __builtin_bit_cast(u32x2_t, high);
                ph[mt][2 * tt] = h2.x, ph[mt][2 * tt + 1] = h2.y;
                if constexpr (TT::P_WORDS == 2) {
                    b4 rest;
#pragma unroll
                    for (int e = 0; e < 4; ++e) rest[e] = (__bf16)(ps[e] - (float)high[e]);
                    const u32x2_t l2 = __builtin_bit_cast(u32x2_t, rest);
                    pl[mt][2 * tt] = l2.x, pl[mt][2 * tt + 1] = l2.y;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                acc[mt][j] = PagedBf16::mma(vf[j], ph[mt], acc[mt][j]);
                if constexpr (TT::P_WORDS == 2) acc[mt][j] = PagedBf16::mma(vf[j], pl[mt], acc[mt][j]);
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            psum[mt] = PagedBf16::mma(ones, ph[mt], psum[mt]);
            if constexpr (TT::P_WORDS == 2) psum[mt] = PagedBf16::mma(ones, pl[mt], psum[mt]);
        }
    };

    // Chunks [whole0, whole1) of the list are seen whole by every row of the block: lowest positions grow with the rows, and so do ends, but for
    // those of contextual rows, which lie behind all others'.
    const int pos0 = span.n - p.delta + rb * ROWS / p.group, pos1 = span.n - p.delta + (r_end - 1) / p.group;
    int whole0 = 0, whole1 = 0;
    if (pos0 >= 0) {
        const int lo = row_span(p, span, pos1).lo, hi = pos1 >= p.c ? row_span(p, span, max(pos0, p.c)).hi : span.u;
        whole0 = max(((lo + 31) >> 5) - span.a0, 0), whole1 = min((hi >> 5) - span.a0, span.na);
    }
    int buffer = 0;
    auto step = [&](int i, auto masked) __attribute__((always_inline)) {
        const bool more = i + CH < end;
        if (more) load(i + CH);
#pragma unroll
        for (int cc = 0; cc < CH; ++cc) {
            if constexpr (decltype(masked)::value) {
                if (i + cc < end) {
                    const int chunk = chunk_at(i + cc), first = chunk * 32;  // (not where this wave's rows see nothing of it)
                    if ((first < any_hi && first + 32 > any_lo) || first < any_chi || (first <= self_hi && first + 32 > self_lo)) work_masked(buffer, cc, chunk, masked);
                }
            } else {
                work_masked(buffer, cc, chunk_at(i + cc), masked);
            }
        }
        if (more) unpack(buffer ^ 1);
        __syncthreads();
        buffer ^= 1;
    };
    if (begin < end) unpack(0);
    __syncthreads();
    int i = begin;
    for (; i < end && !(i >= whole0 && i + CH <= whole1); i += CH) step(i, std::true_type{});
    for (; i + CH <= min(end, whole1); i += CH) step(i, std::false_type{});
    for (; i < end; i += CH) step(i, std::true_type{});

    // one wave's bad page is everyone's
    int* said = (int*)&pairs[0][0][0];
    if (threadIdx.x == 0) *said = 0;
    __syncthreads();
    if (bad) *said = 1;
    __syncthreads();
    bad = *said != 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float lower = plo[mt];
        lower += __shfl_xor(lower, 16, 64);
        lower += __shfl_xor(lower, 32, 64);
        if (bad) lower = __builtin_nanf("");
        if (out_at[mt] < 0) continue;
        float o[4][NV];
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
            for (int j = 0; j < NV; ++j) o[i4][j] = acc[mt][j][i4] - (CodesBf16::off(j & 3) + 7.5f) * psum[mt][i4] + lower;
        store_columns<T, NV>(p, split, out_at[mt] + NV * 4 * g, o);
    }
}

// The same for few rows (at most 8 of one head of the cache), where a product of 16 columns would waste most of them: F = 16 / RP chunks
// side by side.  Column n of a score tile stands for row n % RP and chunk n / RP of F: a chunk's product fills all columns, and each lane keeps
// it where the chunk is its own.  silu and what surrounds it then run once for F chunks, on full lanes, and so do the loads of the pairs
// (step, lowest value).  For the second product a chunk's own columns have the first words of P, the columns of the chunk F / 2 away the second words, the
// others zero: its sums land in columns that nothing else uses, which are added up over the chunks at the end, and two words take no more products than
// one.  (A product for each word took 308 us below, where this takes 270.)
// Waves of a SIMD: three in 168 registers each took 281 us where two in 172 took 290 (128 sequences of 4096 .. 16384 positions, eight
// heads of 128, 1.45 GB); four rows of 128 sequences of up to 8192 88 where two in 214 took 103, but of 33 of up to 2048 16.5 where two took 14.5;
// heads of 256 need the registers of one.  The cache's bytes bound it: the same sequences in runs of up to 96
// chunks take 267 us, 5.4 TB/s where a copy of 1 GiB reaches 5.2.  One short sequence is launches and loads that wait for each other: 8 us.
template <int DK, int DV>
constexpr int STEP_WAVES = DK == 256 ? 1 : DK + DV >= 128 ? 3 : 4;

template <class TT, int DK, int DV, int RP>
__global__ __launch_bounds__(256, (STEP_WAVES<DK, DV>)) void hstu_paged_step_kernel(const PagedAttentionParams p) {
    typedef typename TT::elem T;
    typedef __attribute__((ext_vector_type(2))) T T2;
    constexpr int NK = DK / 32, NV = DV / 16, F = 16 / RP, VW = NV == 16 ? 2 : 1, U = 2;
    __shared__ float meet[4 * RP * DV];
    const PagedCache& c = p.cache;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int part = p.share == 4 ? wave : 0, item = p.share == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
    const bool idle = item >= p.items;
    const int known = idle ? 0 : item;
    const int hk = known % c.heads, b = (known / c.heads) % c.batch, split = known / (c.heads * c.batch);  // whole runs first, what is left of sequences last
    const int own = n / RP, r = n % RP, rows = p.delta * p.group;
    const PagedSpan span = paged_span(p, b, 0, p.delta);
    const int chunks = span.na + span.nb, per = chunks_per_run(p, chunks);
    const bool silent = idle || (p.splits > 1 && split * per >= chunks);  // no run: the joining kernel knows
    if (silent && p.share == 4) return;
    const int run_end = min((split + 1) * per, chunks), each = (max(run_end - split * per, 0) + p.share - 1) / p.share;
    const int begin = silent ? 0 : min(split * per + part * each, run_end), end = silent ? 0 : min(begin + each, run_end);
    auto chunk_at = [&](int i) { return i < span.na ? span.a0 + i : span.b0 + (i - span.na); };

    int lo_max = 0, hi_min = 1 << 30;
    const int row_i = r / p.group, head = hk * p.group + (r - row_i * p.group);
    if (r < rows) {
        const RowSpan see = row_span(p, span, span.n - p.delta + row_i);
        lo_max = see.lo, hi_min = see.hi;
    }
    u32x4_t qf[NK];
    float qs = 0.f, qo = 0.f;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        qf[j] = u32x4_t{0, 0, 0, 0};
        if (r < rows) qf[j] = *(const u32x4_t*)(p.q + (((int64_t)b * p.delta + row_i) * p.q_rs + head * p.q_hs + 8 * (NK * g + j)) * 2);
    }
    auto prepare_q = [&]() __attribute__((always_inline)) {  // columns k and k + 4 side by side, as the codes come; their sums
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const u32x4_t x = qf[j];
            qf[j] = u32x4_t{__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                            __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const T2 two = __builtin_bit_cast(T2, (unsigned)qf[j][k]);
                const float sum = (float)two[0] + (float)two[1];
                qs += sum, qo += sum * TT::codes::off(k);
            }
        }
        qs += __shfl_xor(qs, 16, 64), qo += __shfl_xor(qo, 16, 64);
        qs += __shfl_xor(qs, 32, 64), qo += __shfl_xor(qo, 32, 64);
#pragma unroll
        for (int d = 1; d < RP; d <<= 1) lo_max = max(lo_max, __shfl_xor(lo_max, d, 64)), hi_min = min(hi_min, __shfl_xor(hi_min, d, 64));
        lo_max = __builtin_amdgcn_readfirstlane(lo_max), hi_min = __builtin_amdgcn_readfirstlane(hi_min);
    };

    const typename TT::codes k_codes;
    const CodesBf16 v_codes;
    pa_f32x4 acc[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[j] = pa_f32x4{0, 0, 0, 0};
    float psum = 0.f, plo = 0.f;
    bool bad = span.bad;
    const int in_page = (1 << c.page_shift) - 1;
    const unsigned k_lane = n * (DK / 2) + g * (4 * NK), v_lane = 4 * g * (DV / 2) + n * (NV / 2);

    // Pages of the tiles of 16 of the F chunks from s0 on, one to a lane; what does not exist, or lies in front of all that is seen, has the first page.
    auto pages_of = [&](int s0) __attribute__((always_inline)) {
        int page = 0;
        const int pos = chunk_at(min(s0 + ((lane >> 1) & (F - 1)), end - 1)) * 32 + (lane & 1) * 16;
        if (pos < span.n && pos + 16 > span.seen) {
            const int64_t at = index_at(c.page_table, c.page_table_i64, b * c.table_row_stride + (pos >> c.page_shift));
            if (at < 0 || at >= c.pages) bad = true;
            else page = (int)at;
        }
        return page;
    };
    auto row_of = [&](int page, int s0, int ci, int tt) __attribute__((always_inline)) {  // of the cache, in rows: uniform
        const int64_t pg = __builtin_amdgcn_readlane(page, 2 * ci + tt);
        return ((pg * c.heads + hk) << c.page_shift) + ((chunk_at(s0 + ci) * 32 + tt * 16) & in_page);
    };
    auto load_k = [&](unsigned (&x)[U][2][NK], int page, int s0, int c0) __attribute__((always_inline)) {
        const int nc = min(F, end - s0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const UniformRows k(c.k_codes + row_of(page, s0, min(c0 + u, nc - 1), tt) * (DK / 2), 16 * (DK / 2));
                if constexpr (NK == 1) {
                    x[u][tt][0] = k.at<unsigned>(k_lane);
                } else if constexpr (NK == 2) {
                    const u32x2_t a = k.at<u32x2_t>(k_lane);
                    x[u][tt][0] = a.x, x[u][tt][1] = a.y;
                } else {
#pragma unroll
                    for (int j = 0; j < NK; j += 4) {
                        const u32x4_t a = k.at<u32x4_t>(k_lane + 4 * j);
                        x[u][tt][j] = a.x, x[u][tt][j + 1] = a.y, x[u][tt][j + 2] = a.z, x[u][tt][j + 3] = a.w;
                    }
                }
            }
    };
    auto load_v = [&](unsigned (&x)[U][8][VW], int page, int s0, int c0) __attribute__((always_inline)) {
        const int nc = min(F, end - s0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const UniformRows v(c.v_codes + row_of(page, s0, min(c0 + u, nc - 1), tt) * (DV / 2), 16 * (DV / 2));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned at = v_lane + i * (DV / 2);
                    if constexpr (NV == 2) x[u][4 * tt + i][0] = v.at<unsigned char>(at);
                    else if constexpr (NV == 4) x[u][4 * tt + i][0] = v.at<unsigned short>(at);
                    else {
#pragma unroll
                        for (int j = 0; j < VW; ++j) x[u][4 * tt + i][j] = v.at<unsigned>(at + 4 * j);
                    }
                }
            }
    };
    // This lane's pairs: of its own chunk's positions 4 g .. and 16 + 4 g ..
    u32x4_t ks[2], vs[2];
    auto load_pairs = [&](int page, int s0) __attribute__((always_inline)) {
        const int ci = min(own, min(F, end - s0) - 1), pos = chunk_at(s0 + ci) * 32 + 4 * g;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const int64_t pg = __shfl(page, 2 * ci + tt, 64);
            const int64_t at = ((pg * c.heads + hk) << c.page_shift) + ((pos + 16 * tt) & in_page);
            ks[tt] = *(const u32x4_t*)(c.k_scales + at * 4);
            vs[tt] = *(const u32x4_t*)(c.v_scales + at * 4);
        }
    };

    // Loads run ahead of the work on what they bring: K and V two chunks, the first V before the scores, the next F chunks' pages before
    // the scores and their first K and pairs before the sums.  (With each F chunks begun from nothing a run of 257 chunks took a sixth
    // longer than one of 256.)
    unsigned k_now[U][2][NK], k_next[U][2][NK], v_now[U][8][VW], v_next[U][8][VW];
    int page = 0, page_next = 0;
    if (begin < end) {
        page = pages_of(begin);
        load_k(k_now, page, begin, 0);
        load_pairs(page, begin);
        prepare_q();
    }
    for (int s0 = begin; s0 < end; s0 += F) {
        const int nc = min(F, end - s0);
        const bool more = s0 + F < end;
        if (more) page_next = pages_of(s0 + F);
        load_v(v_now, page, s0, 0);
        pa_f32x4 s[2] = {pa_f32x4{0, 0, 0, 0}, pa_f32x4{0, 0, 0, 0}};
        auto scores = [&](const unsigned (&x)[U][2][NK], int c0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool mine = own == c0 + u;
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    pa_f32x4 t = {-qo, -qo, -qo, -qo};
#pragma unroll
                    for (int j = 0; j < NK; ++j) {
                        unsigned o[4];
                        k_codes.four(x[u][tt][j], o);
                        t = TT::mma(u32x4_t{o[0], o[1], o[2], o[3]}, qf[j], t);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[tt][i] = mine ? t[i] : s[tt][i];
                }
            }
        };
        // (chunks behind the last are the last again: their scores are masked, P of theirs is zero)
        for (int c0 = 0; c0 < nc; c0 += U) {
            load_k(k_next, page, s0, c0 + U);
            scores(k_now, c0);
            __builtin_memcpy(k_now, k_next, sizeof(k_now));
        }
        u32x4_t ph, pl;  // P s of this lane's chunk, in two words: the second in the lane half of the chunks away
        auto silu = [&](auto masked) __attribute__((always_inline)) {
            const int own_pos = chunk_at(min(s0 + own, end - 1)) * 32 + 4 * g;
            int pos = r < rows ? span.n - p.delta + row_i : -1;
            asm volatile("" : "+v"(pos));  // what the row sees is worked out where it is needed: four registers that the loads ahead have instead
            const RowSpan see = row_span(p, span, pos);
            float ps[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const T2 k2 = __builtin_bit_cast(T2, (unsigned)ks[e >> 2][e & 3]), v2 = __builtin_bit_cast(T2, (unsigned)vs[e >> 2][e & 3]);
                const float t = p.c1 * ((float)k2[0] * s[e >> 2][e & 3] + (float)k2[1] * qs);
                const float pr = t * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t));
                ps[e] = pr * (float)v2[0];
                float lower = pr * ((float)v2[1] + 7.5f * (float)v2[0]);
                if constexpr (decltype(masked)::value) {
                    const bool seen = own < nc && see.sees(own_pos + (e >> 2) * 16 + (e & 3));
                    ps[e] = seen ? ps[e] : 0.f, lower = seen ? lower : 0.f;
                }
                plo += lower;
            }
            pa_bf16x8 high, rest;
#pragma unroll
            for (int e = 0; e < 8; ++e) high[e] = (__bf16)ps[e], psum += (float)high[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) rest[e] = (__bf16)(ps[e] - (float)high[e]), psum += (float)rest[e];
            ph = __builtin_bit_cast(u32x4_t, high), pl = __builtin_bit_cast(u32x4_t, rest);
#pragma unroll
            for (int i = 0; i < 4; ++i) pl[i] = (unsigned)__builtin_amdgcn_update_dpp(0, (int)pl[i], 0x128, 0xf, 0xf, true);  // (rotated by 8 of 16 lanes)
        };
        if (nc == F && s0 + F <= span.na && chunk_at(s0) * 32 >= lo_max && chunk_at(s0 + F - 1) * 32 + 32 <= hi_min) silu(std::false_type{});
        else silu(std::true_type{});
        auto sums = [&](const unsigned (&x)[U][8][VW], int c0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                u32x4_t b;
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = own == c0 + u ? ph[i] : own == ((c0 + u) ^ (F / 2)) ? pl[i] : 0u;
#pragma unroll
                for (int h = 0; h < (NV + 3) / 4; ++h) {
                    u32x4_t vf[4];
#pragma unroll
                    for (int pair = 0; pair < 4; ++pair) {
                        unsigned two, o[4];
                        if constexpr (NV <= 4) two = x[u][2 * pair][0] | (x[u][2 * pair + 1][0] << 16);
                        else two = __builtin_amdgcn_perm(x[u][2 * pair + 1][h >> 1], x[u][2 * pair][h >> 1], h & 1 ? 0x07060302u : 0x05040100u);
                        v_codes.four(two, o);
#pragma unroll
                        for (int k = 0; k < 4; ++k) vf[k][pair] = o[k];
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (4 * h + k >= NV) break;
                        acc[4 * h + k] = PagedBf16::mma(vf[k], b, acc[4 * h + k]);
                    }
                }
            }
        };
        if (more) {
            load_k(k_now, page_next, s0 + F, 0);
            load_pairs(page_next, s0 + F);
        }
        for (int c0 = 0; c0 < nc; c0 += U) {
            load_v(v_next, page, s0, c0 + U);
            sums(v_now, c0);
            __builtin_memcpy(v_now, v_next, sizeof(v_now));
        }
        page = page_next;
    }

    // columns of one row, over the chunks; psum and plo over the positions' lanes too
    auto columns = [&](float v) __attribute__((always_inline)) {
        if constexpr (RP <= 8) v += dpp<0x128>(v);  // rotations within 16 lanes
        if constexpr (RP <= 4) v += dpp<0x124>(v);
        if constexpr (RP <= 2) v += dpp<0x122>(v);
        if constexpr (RP <= 1) v += dpp<0x121>(v);
        return v;
    };
    psum += __shfl_xor(psum, 16, 64), plo += __shfl_xor(plo, 16, 64);
    psum += __shfl_xor(psum, 32, 64), plo += __shfl_xor(plo, 32, 64);
    psum = columns(psum), plo = columns(plo);
    if (__any(bad)) plo = __builtin_nanf("");
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const float o = columns(acc[j][i4]) - (CodesBf16::off(j & 3) + 7.5f) * psum + plo;
            if (n < RP) meet[(wave * RP + n) * DV + NV * (4 * g + i4) + j] = o;
        }
    __syncthreads();
    // the sums of the waves that share a run, or each wave's own
    const int64_t row0 = (int64_t)b * p.delta;
    for (int at = p.share == 4 ? threadIdx.x : lane; at < RP * DV && !silent; at += 64 * p.share) {
        const int rr = at / DV, d = at % DV;
        if (rr >= rows) break;
        const float x = p.share == 4 ? meet[at] + meet[RP * DV + at] + meet[2 * RP * DV + at] + meet[3 * RP * DV + at] : meet[wave * RP * DV + at];
        const int64_t to = ((row0 + rr / p.group) * (c.heads * p.group) + hk * p.group + rr % p.group) * DV + d;
        if (p.splits > 1) p.partial[split * p.partial_stride + to] = x;
        else ((T*)p.out)[to] = (T)(x * p.oscale);
    }
}

// out = oscale * the sum of the runs there are: eight columns to PARTS threads, which share out the runs and add up in a fixed order.
// The loads of a thread's runs wait for nothing, and a launch bounds it: 3 to 6 us.
template <class TT, int PARTS>
__global__ __launch_bounds__(256) void hstu_paged_join_kernel(const PagedAttentionParams p, int block_rows, int64_t total8) {
    typedef typename TT::elem T;
    const int64_t thread = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int part = (int)(thread % PARTS);
    const bool there = thread / PARTS < total8;
    const int64_t at = there ? thread / PARTS : total8 - 1;
    const int heads = p.cache.heads * p.group, words = p.cache.dv >> 3;
    const int64_t row_head = at / words, row = row_head / heads;
    const int b = (int)(row / p.delta), r = (int)(row - (int64_t)b * p.delta) * p.group + (int)(row_head - row * heads) % p.group;
    const int rb = r / block_rows, r_end = min((rb + 1) * block_rows, p.delta * p.group);
    const PagedSpan span = paged_span(p, b, rb * block_rows / p.group, (r_end - 1) / p.group + 1);
    const int chunks = span.na + span.nb, per = chunks_per_run(p, chunks), runs = (chunks + per - 1) / per;
    pa_f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    const float* from = p.partial + at * 8;
    int s = part;
    for (; s + 3 * PARTS < runs; s += 4 * PARTS) {  // four loads in flight
        pa_f32x4 a[4], c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const pa_f32x4* f = (const pa_f32x4*)(from + (s + i * PARTS) * p.partial_stride);
            a[i] = f[0], c[i] = f[1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x += a[i], y += c[i];
    }
    for (; s < runs; s += PARTS) {
        const pa_f32x4* f = (const pa_f32x4*)(from + s * p.partial_stride);
        x += f[0], y += f[1];
    }
    float o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = x[i], o[4 + i] = y[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o[i] = group_sum<PARTS>(o[i]) * p.oscale;
        if (span.bad) o[i] = __builtin_nanf("");
    }
    Cols<T> out;
    out.put(o);
    if (there && part == 0) out.store((T*)p.out + at * 8);
}

}  // namespace hstu
