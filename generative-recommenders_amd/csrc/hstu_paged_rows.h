// Rows into and out of a K/V cache that holds them in 4 bits, in pages: bound by HBM bandwidth.
//
// The lanes are laid out as in hstu_norm_rope.h, eight columns to a lane, so that a lane's codes are one word of the row.  The
// extremes of a row are log2(LPV) lane exchanges.  Codes are found by a division that is rounded as IEEE says, so that a tie between
// two codes (K and V have 8 or 11 bits, a step too: ties do occur) falls the same way on any machine.
#pragma once
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

// Eight columns (of LPV lanes' row; lanes behind the row's end have `there` false) to a word of codes, and step and lowest value.
template <class T, int LPV>
__device__ __forceinline__ unsigned to_four_bits(const float (&x)[8], bool there, unsigned& scale) {
    float lo = __builtin_inff(), hi = -__builtin_inff();
    bool odd = false;
    if (there) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
            odd |= !(x[i] - x[i] == 0.f);
        }
    }
#pragma unroll
    for (int d = LPV / 2; d >= 1; d >>= 1) lo = fminf(lo, __shfl_xor(lo, d, 64)), hi = fmaxf(hi, __shfl_xor(hi, d, 64));
    const int me = threadIdx.x & 63;
    const uint64_t group = ((1ull << LPV) - 1) << (me - me % LPV);
    // (half of everything, which is exact, so that the range of a row of large values is a float)
    const float lo2 = 0.5f * lo;
    T step_t = (T)((0.5f * hi - lo2) / 7.5f), lo_t = (T)lo;
    const float step = (float)step_t;
    if ((__ballot(odd) & group) != 0 || !(step - step == 0.f)) step_t = lo_t = (T)__builtin_nanf("");
    typedef __attribute__((ext_vector_type(2))) T T2;
    T2 both;
    both[0] = step_t, both[1] = lo_t;
    scale = __builtin_bit_cast(unsigned, both);
    unsigned codes = 0;
    if (step > 0.f) {
        const float step2 = 0.5f * step;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = fminf(fmaxf(rintf(__builtin_fmaf(x[i], 0.5f, -lo2) / step2), 0.f), 15.f);
            codes |= (unsigned)c << (4 * i);
        }
    }
    return codes;
}

// grid (rows / groups of a workgroup, vectors / vectors_per_group): a row's vectors count through its heads of K, then of V.
template <class T, int LPV>
__global__ __launch_bounds__(256) void hstu_paged_append_kernel(const AppendParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 4;
    const int l = threadIdx.x % LPV, col0 = 8 * l;
    const int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPV;
    const PagedCache& c = p.cache;
    int64_t place = 0;
    const int b = find_sequence<LPV>(p.place, c.batch, row, place);
    const int64_t to = cache_row(c, b, place);
    const bool stored = to >= 0;
    const int first = blockIdx.y * p.vectors_per_group, last = min(first + p.vectors_per_group, 2 * c.heads);
    LaneTurn t;
    t.lane(p.turn, col0);
    bool known = true;
    if (p.turn.rotary && first < c.heads && stored) known = t.row(p.turn, p.positions ? index_at(p.positions, p.positions_i64, row) : place, col0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int base = which ? c.heads : 0, h0 = max(first - base, 0), h1 = min(last - base, c.heads);
        if (h0 >= h1) continue;
        const int dim = which ? c.dv : c.dqk;
        const bool there = stored && col0 < dim;
        const T* x_of = (const T*)(which ? p.v : p.k) + row * (which ? p.v_rs : p.k_rs) + col0;
        const int64_t hs = which ? p.v_hs : p.k_hs;
        unsigned* codes_of = (unsigned*)(which ? c.v_codes : c.k_codes);
        unsigned* scales_of = (unsigned*)(which ? c.v_scales : c.k_scales);
        float w[8], wp[8];
        if (!which) lane_weights((const T*)p.k_weight, col0, col0 < dim, t, w, wp);
        for (int h = h0; h < h1; h += AHEAD) {
            Cols<T> in[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                in[a].zero();
                if (there && h + a < h1) in[a].load(x_of + (h + a) * hs);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (h + a >= h1) break;  // (the same for the whole workgroup)
                float x[8];
                in[a].get(x);
                if (!which && (p.k_weight || p.turn.rotary)) {
                    float q[8], y[8], r = 1.f;
                    in[a].from_lane(t.byte_lane).get(q);
                    if (p.k_weight) {
                        float sq = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
                        r = rsqrtf(group_sum<LPV>(sq) * p.inv_dim + p.eps);
                    }
                    if (!known) r = __builtin_nanf("");
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i], q[i] = q[i] * r * wp[i];
                    turn<false>(t, p.turn.interleaved, x, q, y);
                    Cols<T> rounded;
                    rounded.put(y);
                    rounded.get(x);
                }
                unsigned scale;
                const unsigned codes = to_four_bits<T, LPV>(x, col0 < dim, scale);
                const int64_t at = to + ((int64_t)(h + a) << c.page_shift);
                if (there) codes_of[at * (dim >> 3) + l] = codes;
                if (there && l == 0) scales_of[at] = scale;
            }
        }
    }
}

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
