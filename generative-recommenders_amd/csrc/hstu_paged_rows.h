// Rows into and out of a K/V cache that holds them in 4 bits, in pages: bound by HBM bandwidth.
//
// The lanes are laid out as in hstu_norm_rope.h, eight columns to a lane, so that a lane's codes are one word of the row.  The
// extremes of a row are log2(LPV) lane exchanges.  Codes are found by a quotient that is rounded as IEEE says, so that a tie between
// two codes (K and V have 8 or 11 bits, a step too: ties do occur) falls the same way on any machine.
#pragma once
#include <type_traits>

#include "hstu_norm_rope.h"

namespace hstu {

struct PagedCache {
    char *k_codes, *v_codes;
    char *k_scales, *v_scales;
    int64_t pages;
    int heads, page_shift, dqk, dv;
    const void* page_table;
    int64_t table_row_stride;
    int table_columns, page_table_i64, batch;
};

// Where a new row belongs.
struct Placing {
    const void *start, *offsets;
    int start_i64, offsets_i64;
    int64_t rows, rows_per_sequence;  // without offsets
};

struct AppendParams {
    PagedCache cache;
    Placing place;
    const char *k, *v;
    int64_t k_rs, k_hs, v_rs, v_hs;
    const char* k_weight;
    float eps, inv_dim;
    Turn turn;
    const void* positions;
    int positions_i64, vectors_per_group;
};

struct ReadParams {
    PagedCache cache;
    Placing place;
    char *k, *v;  // dense
    int vectors_per_group;
};

// Sequence of row `row` (-1: behind the last one) and its place there.  The LPV lanes of a group search together: each round they
// look at LPV offsets, spread over what is left of them, and keep the part between two (two rounds for 256 sequences and 16 lanes,
// where one lane alone would wait for eight loads in a row).
template <int LPV>  // 4 .. 32
__device__ __forceinline__ int find_sequence(const Placing& p, int batch, int64_t row, int64_t& place) {
    if (row >= p.rows) return -1;
    int b;
    int64_t first;
    if (!p.offsets) {
        b = (int)(row / p.rows_per_sequence);
        if (b >= batch) return -1;
        first = b * p.rows_per_sequence;
    } else {
        const int me = threadIdx.x & 63, l = me % LPV, shift = me - l;
        int lo = 0, len = batch;
        while (len > 1) {
            const int step = (len + LPV - 1) / LPV, at = l * step;
            const bool below = l == 0 || (at < len && index_at(p.offsets, p.offsets_i64, lo + at) <= row);
            const uint64_t bits = (__ballot(below) >> shift) & ((1ull << LPV) - 1);
            const int passed = __builtin_ctzll(~bits);  // lanes in front of the first that is not below
            const int skip = (passed - 1) * step;
            len = min(step, len - skip);
            lo += skip;
        }
        b = lo;
        first = index_at(p.offsets, p.offsets_i64, b);
        if (row < first || row >= index_at(p.offsets, p.offsets_i64, b + 1)) return -1;
    }
    place = index_at(p.start, p.start_i64, b) + (row - first);
    return b;
}

// Number of the row (page, position in it) of head 0 that place `place` of sequence b has; -1 if it has none.  Rows of head h are
// h << page_shift further on.
__device__ __forceinline__ int64_t cache_row(const PagedCache& c, int b, int64_t place) {
    if (b < 0 || place < 0 || (place >> c.page_shift) >= c.table_columns) return -1;
    const int64_t page = index_at(c.page_table, c.page_table_i64, b * c.table_row_stride + (place >> c.page_shift));
    if (page < 0 || page >= c.pages) return -1;
    return ((page * c.heads) << c.page_shift) + (place & ((1 << c.page_shift) - 1));
}

// Smallest and largest of eight columns, NaN where one is; and over LPV lanes (numbers only).  The instructions themselves: the
// compiler puts another in front of each operand of its min and max, to quiet NaNs.
__device__ __forceinline__ void extremes(const float (&x)[8], float& lo, float& hi) {
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; i += 2) {
        const float a = x[i], b = x[i < 7 ? i + 1 : i];
        asm("v_minimum3_f32 %0, %0, %2, %3\n\tv_maximum3_f32 %1, %1, %2, %3" : "+&v"(lo), "+&v"(hi) : "v"(a), "v"(b));
    }
}
#define HSTU_EXTREMES_DPP(how)                                                                                                              \
    asm("s_nop 1\n\tv_min_f32_dpp %0, %0, %0 " how " row_mask:0xf bank_mask:0xf\n\tv_max_f32_dpp %1, %1, %1 " how " row_mask:0xf bank_mask:0xf" \
        : "+v"(lo), "+v"(hi))
template <int LPV>
__device__ __forceinline__ void group_extremes(float& lo, float& hi) {
    static_assert(LPV >= 4 && LPV <= 32, "lanes of a cache's row");
    HSTU_EXTREMES_DPP("quad_perm:[1,0,3,2]");
    HSTU_EXTREMES_DPP("quad_perm:[2,3,0,1]");
    if constexpr (LPV >= 8) HSTU_EXTREMES_DPP("row_half_mirror");
    if constexpr (LPV >= 16) HSTU_EXTREMES_DPP("row_mirror");
    if constexpr (LPV >= 32) lo = fminf(lo, __shfl_xor(lo, 16, 64)), hi = fmaxf(hi, __shfl_xor(hi, 16, 64));
}
#undef HSTU_EXTREMES_DPP

// Eight columns of each of LPV lanes to a word of codes, and the row's step and lowest value.  (Lanes behind the row's end hold other columns of it.)
// The quotient x / step is rounded as IEEE says by Markstein's correction: q = a y with y the reciprocal of b to a unit in the last
// place, then q + (a - q b) y, whose remainder is exact; three operations a column where the compiler's division takes some fourteen.
// It is exact where the quotient is a float, which a tie between two codes is.
template <class T, int LPV>
__device__ __forceinline__ unsigned to_four_bits(const float (&x)[8], unsigned& scale) {
    float lo, hi;
    extremes(x, lo, hi);
    const int me = threadIdx.x & 63;
    const uint64_t group = ((1ull << LPV) - 1) << (me - me % LPV);
    const bool nan = (__ballot(lo != lo) & group) != 0;
    group_extremes<LPV>(lo, hi);
    // (half of everything, which is exact, so that the range of a row of large values is a float)
    const float range = 0.5f * hi - 0.5f * lo, fifteenth = range * (1.f / 7.5f);
    T step_t = (T)__builtin_fmaf(__builtin_fmaf(-fifteenth, 7.5f, range), 1.f / 7.5f, fifteenth), lo_t = (T)lo;
    const float step = (float)step_t;
    if (nan || !(step - step == 0.f)) step_t = lo_t = (T)__builtin_nanf("");
    typedef __attribute__((ext_vector_type(2))) T T2;
    T2 both;
    both[0] = step_t, both[1] = lo_t;
    scale = __builtin_bit_cast(unsigned, both);
    // step and columns by a power of two that takes the step to 1/2 .. 1, or some way there from below 2^-100
    const float by = __builtin_amdgcn_ldexpf(1.f, -max(__builtin_amdgcn_frexp_expf(step), -100) - 1), from = -lo * by, b = step * by;
    const float y0 = __builtin_amdgcn_rcpf(b), y = __builtin_fmaf(__builtin_fmaf(-b, y0, 1.f), y0, y0);
    float code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = __builtin_fmaf(x[i], by, from), q = a * y;
        code[i] = __builtin_fmaf(__builtin_fmaf(-q, b, a), y, q);
    }
    // No quotient is below 0; one above 15 1/2 there is only where the step, below the type's normal numbers, has lost bits in its rounding.
    if (__ballot(step < (std::is_same<T, __bf16>::value ? 0x1p-126f : 0x1p-14f)) != 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = fminf(code[i], 15.f);
    }
    // rounded to the nearest, ties to even, into a byte each: the even columns' word, the odd ones'
    unsigned even = 0, odd = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) even = __builtin_amdgcn_cvt_pk_u8_f32(code[2 * i], i, even), odd = __builtin_amdgcn_cvt_pk_u8_f32(code[2 * i + 1], i, odd);
    return step > 0.f ? even | (odd << 4) : 0u;
}

// grid (rows / groups of a workgroup, vectors / vectors_per_group): a row's vectors count through its heads of K, then of V.
// (16 columns to a lane, which do what a row takes once in half as many lanes, came to a third fewer instructions and to the same time,
// four waves of a SIMD in 107 registers where six have 78.  So did the first loads in front of the lookups.)  Vector operations
// bound it, with the bytes close below: 256 sequences of 64 .. 1024 rows, four heads of 128, normed and turned, 97 us (337 MB, 65 us of a
// copy; the loads and stores alone 68), of whose 200 thousand clocks a SIMD has 187 of vector operations (counted); fp16 rows that are only
// turned, 146378 of eight heads, 166 again and again, 180 to 197 with their reading between (761 MB; 321 of 410).  64 single rows take 4.5 us, one launch and three loads that wait for each other.
template <class T, int LPV, int TURN>
__global__ __launch_bounds__(256) void hstu_paged_append_kernel(const AppendParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 4;
    const int l = threadIdx.x % LPV;
    const PagedCache& c = p.cache;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPV, place = 0;
    const int b = find_sequence<LPV>(p.place, c.batch, row, place);
    const int64_t to = cache_row(c, b, place);
    const bool stored = to >= 0;
    if (row >= p.place.rows) row = p.place.rows - 1;  // (loads need no condition; nothing is stored)
    const int first = blockIdx.y * p.vectors_per_group, last = min(first + p.vectors_per_group, 2 * c.heads);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int base = which ? c.heads : 0, h0 = max(first - base, 0), h1 = min(last - base, c.heads);
        if (h0 >= h1) continue;
        const int dim = which ? c.dv : c.dqk;
        const bool cols = 8 * l < dim;
        const int col0 = cols ? 8 * l : dim - 8;
        const T* x_of = (const T*)(which ? p.v : p.k) + row * (which ? p.v_rs : p.k_rs) + col0;
        const int64_t hs = which ? p.v_hs : p.k_hs, next_codes = (int64_t)(dim >> 1) << c.page_shift, next_scales = 4ll << c.page_shift;  // bytes to the next head
        char* codes_at = (which ? c.v_codes : c.k_codes) + to * (dim >> 1) + 4 * l;
        char* scales_at = (which ? c.v_scales : c.k_scales) + to * 4;
        const bool changed = !which && (TURN != TURN_NONE || p.k_weight);
        LaneTurn t;
        float w[8];
        if (changed) {
            t.lane(p.turn, col0, l);
            if (TURN != TURN_NONE && stored) t.row(p.turn, p.positions ? index_at(p.positions, p.positions_i64, row) : place, col0);
            lane_weights((const T*)p.k_weight, col0, w);
        }
        for (int h = h0; h < h1; h += AHEAD) {
            Cols<T> in[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) in[a].load(x_of + min(h + a, h1 - 1) * hs);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (h + a >= h1) break;  // (the same for the whole workgroup)
                float x[8];
                if (changed) {
                    float y[8];
                    norm_and_turn<T, LPV, TURN>(t, in[a], w, cols, p.k_weight != nullptr, dim > 64, p.inv_dim, p.eps, y);
                    Cols<T> rounded;
                    rounded.put(y);
                    rounded.get(x);
                } else {
                    in[a].get(x);
                }
                unsigned scale;
                const unsigned codes = to_four_bits<T, LPV>(x, scale);
                if (stored && cols) *(unsigned*)(codes_at + (h + a) * next_codes) = codes;
                if (stored && l == 0) *(unsigned*)(scales_at + (h + a) * next_scales) = scale;
            }
        }
    }
}

// The inverse, value = lowest + step code, rounded once.  Bytes bound it: the rows of the sequences above 69 us, 4.9 TB/s.
template <class T, int LPV>
__global__ __launch_bounds__(256) void hstu_paged_read_kernel(const ReadParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 4;
    const int l = threadIdx.x % LPV, col0 = 8 * l;
    const int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPV;
    const PagedCache& c = p.cache;
    int64_t place = 0;
    const int b = find_sequence<LPV>(p.place, c.batch, row, place);
    if (row >= p.place.rows) return;
    const int64_t from = cache_row(c, b, place);
    const int first = blockIdx.y * p.vectors_per_group, last = min(first + p.vectors_per_group, 2 * c.heads);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int base = which ? c.heads : 0, h0 = max(first - base, 0), h1 = min(last - base, c.heads);
        const int dim = which ? c.dv : c.dqk;
        if (h0 >= h1 || col0 >= dim) continue;
        const unsigned* codes_of = (const unsigned*)(which ? c.v_codes : c.k_codes);
        const unsigned* scales_of = (const unsigned*)(which ? c.v_scales : c.k_scales);
        T* out = (T*)(which ? p.v : p.k) + row * c.heads * dim + col0;
        for (int h = h0; h < h1; h += AHEAD) {
            unsigned codes[AHEAD], scale[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                codes[a] = 0;
                scale[a] = b < 0 ? 0u : ~0u;  // zero behind the last sequence; NaN, in both types, where there is no page
                if (from >= 0 && h + a < h1) {
                    const int64_t at = from + ((int64_t)(h + a) << c.page_shift);
                    codes[a] = codes_of[at * (dim >> 3) + l];
                    scale[a] = scales_of[at];
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (h + a >= h1) break;
                typedef __attribute__((ext_vector_type(2))) T T2;
                const T2 both = __builtin_bit_cast(T2, scale[a]);
                const float step = (float)both[0], lo = (float)both[1];
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(step, (float)((codes[a] >> (4 * i)) & 15), lo);
                Cols<T> o;
                o.put(x);
                o.store(out + (int64_t)(h + a) * dim);
            }
        }
    }
}

}  // namespace hstu
