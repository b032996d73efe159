// Norms of q and k for each head with the position rotation, forward and backward: row-wise work, bound by HBM bandwidth.
//
//     n = x * rsqrt(mean(x^2) + eps) * w,   y = R n       with R the rotation of the row's position (pairs of columns)
//     g = R^T dy,   dw = sum over rows and heads of g * x * r,   dx = r * (g w - x r * mean(g w x r)),   r = rsqrt(...)
//
// A vector (one row, one head) is taken by LPV = dim / 8 lanes (rounded up to a power of two, at least four), eight columns to a lane: one 16-byte
// access each way in 16 bits, and the sums over a vector are log2(LPV) lane exchanges.  The partner of a column in the half-split
// form lies rotary / 2 columns on, rotary / 16 lanes away: lanes exchange them.  A group of LPV lanes stays with one row for several heads, so that
// positions and table rows, which the heads of a row share, are read once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hstu {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

__device__ __forceinline__ int64_t index_at(const void* p, int is_i64, int64_t i) { return is_i64 ? ((const int64_t*)p)[i] : (int64_t)((const int*)p)[i]; }

// Eight columns of a row as they lie in memory, and as floats.
template <class T>
struct Cols {
    static constexpr int WORDS = sizeof(T) * 2;
    unsigned w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
        const u32x4_t* q = (const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) {
            const u32x4_t v = q[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        u32x4_t* q = (u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) q[i] = u32x4_t{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
        } else {
            typedef __attribute__((ext_vector_type(2))) T T2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T2 v = __builtin_bit_cast(T2, w[i]);
                x[2 * i] = (float)v[0], x[2 * i + 1] = (float)v[1];
            }
        }
    }
    __device__ __forceinline__ void put(const float (&x)[8]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(x[i]);
        } else {
            typedef __attribute__((ext_vector_type(2))) T T2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                T2 v;
                v[0] = (T)x[2 * i], v[1] = (T)x[2 * i + 1];
                w[i] = __builtin_bit_cast(unsigned, v);
            }
        }
    }
};

// v of another lane of 16, by the data path of the instruction that uses it (no LDS).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// op over LPV lanes, the result in each: neighbours, pairs, then halves of 8 and of 16 mirrored (their lanes agree by then).
template <int LPV, class F>
__device__ __forceinline__ float group_reduce(float v, F&& op) {
    if constexpr (LPV >= 2) v = op(v, dpp<0xB1>(v));
    if constexpr (LPV >= 4) v = op(v, dpp<0x4E>(v));
    if constexpr (LPV >= 8) v = op(v, dpp<0x141>(v));
    if constexpr (LPV >= 16) v = op(v, dpp<0x140>(v));
    if constexpr (LPV >= 32) v = op(v, __shfl_xor(v, 16, 64));
    if constexpr (LPV >= 64) v = op(v, __shfl_xor(v, 32, 64));
    return v;
}
template <int LPV>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<LPV>(v, [](float a, float b) { return a + b; });
}

struct Turn {
    const float* table;
    int64_t table_rows;
    int rotary, interleaved;
};

// How a lane's eight columns turn: y = n c + partner s for each, s with its sign.  Where nothing turns c = 1, s = 0.
struct LaneTurn {
    float c[8], s[8];
    int byte_lane;      // half-split: 4 * the partner's lane
    unsigned keep;      // all ones where the partner counts (an infinity times s = 0 is no zero)
    bool turns, first;  // whether these columns turn; half-split: whether they are in front of their partners

    // Everything that does not depend on the row.  `l`: number of the lane in its group (its columns may be another lane's, see the kernels).
    __device__ __forceinline__ void lane(const Turn& t, int col0, int l) {
        const int half = t.rotary >> 1, group = (threadIdx.x & 63) - l;
        turns = col0 < t.rotary, first = col0 < half;
        byte_lane = 4 * (group + ((turns && !t.interleaved ? (first ? col0 + half : col0 - half) : col0) >> 3));
        keep = turns ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    }
    // Cosines and sines of position `pos`; NaN, for every column, where it is not in the table.
    __device__ __forceinline__ void row(const Turn& t, int64_t pos, int col0) {
        const bool there = pos >= 0 && pos < t.table_rows;
        const float one = there ? 1.f : __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = one, s[i] = 0.f;
        if (!turns || !there) return;
        const int half = t.rotary >> 1;
        const float* cp = t.table + pos * t.rotary + (t.interleaved ? col0 >> 1 : (first ? col0 : col0 - half));
        typedef __attribute__((ext_vector_type(4))) float f4;
        if (t.interleaved) {
#pragma unroll
            for (int k = 0; k < 4; k += 4) {
                const f4 ck = *(const f4*)(cp + k), sk = *(const f4*)(cp + half + k);
#pragma unroll
                for (int i = 0; i < 4; ++i) c[2 * (k + i)] = c[2 * (k + i) + 1] = ck[i], s[2 * (k + i)] = -sk[i], s[2 * (k + i) + 1] = sk[i];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const f4 ck = *(const f4*)(cp + k), sk = *(const f4*)(cp + half + k);
#pragma unroll
                for (int i = 0; i < 4; ++i) c[k + i] = ck[i], s[k + i] = first ? -sk[i] : sk[i];
            }
        }
    }
};

// How vectors turn, as the kernels are built for it: not at all, halves or neighbouring pairs.
enum { TURN_NONE = 0, TURN_HALVES = 1, TURN_PAIRS = 2 };

// The partners of a lane's columns, zero where they do not count.
template <int TURN>
__device__ __forceinline__ void partners(const LaneTurn& t, const float (&x)[8], float (&p)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned w = TURN == TURN_PAIRS ? __float_as_uint(x[i ^ 1]) : (unsigned)__builtin_amdgcn_ds_bpermute(t.byte_lane, (int)__float_as_uint(x[i]));
        p[i] = __uint_as_float(w & t.keep);
    }
}

// The weights of a lane's columns, ones without a norm.
template <class T>
__device__ __forceinline__ void lane_weights(const T* weight, int col0, float (&w)[8]) {
    if (weight) {
        Cols<T> c;
        c.load(weight + col0);
        c.get(w);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
    }
}

// 1 / sqrt(mean of squares + eps) of a vector: squares added pairwise, in vectors of more than 64 columns (`wide`) from sums of four on, and the
// instruction's root, good to a unit in the last place, corrected once by its residual.  The order goes by the vector's width and not by the lanes
// it is given, so that K comes out the same beside any width of V.  At 16, 32, 64, 128 and 256 columns that is also, bit by bit, what PyTorch's mean
// and reciprocal root gave on this device; at 48, 80, 104 and 512 a fifth of the rows differed in the last place.
template <int LPV>
__device__ __forceinline__ float inverse_rms(const float (&x)[8], bool there, bool wide, float inv_dim, float eps) {
#pragma clang fp contract(off)
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = x[i] * x[i];
    const float sum = LPV >= 16 && wide ? (q[0] + q[1] + q[2] + q[3]) + (q[4] + q[5] + q[6] + q[7]) : ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
    const float v = group_sum<LPV>(there ? sum : 0.f) * inv_dim + eps;
    const float r = __builtin_amdgcn_rsqf(v), h = v * r, low = __builtin_fmaf(v, r, -h);
    const float fixed = __builtin_fmaf(0.5f * r, __builtin_fmaf(-low, r, __builtin_fmaf(-h, r, 1.f)), r);
    return v > 0x1p-100f && v < 0x1p100f ? fixed : r;
}

// A vector as loaded to what is rounded and stored; `there`: whether the lane's columns are the vector's (one that has none holds another's).
// The operations are rounded one by one, as the definition has them: K is rounded to its type next and then
// to codes, where a value that comes out a unit in the last place off now and then is a whole step off.  (Weights multiplied into cosines and
// sines, and sums by fused operations, gave twenty such codes in 18 million; this costs no more.)
template <class T, int LPV, int TURN>
__device__ __forceinline__ void norm_and_turn(const LaneTurn& t, const Cols<T>& in, const float (&w)[8], bool there, bool norm, bool wide, float inv_dim,
                                              float eps, float (&y)[8]) {
#pragma clang fp contract(off)
    in.get(y);
    if (norm) {
        const float r = inverse_rms<LPV>(y, there, wide, inv_dim, eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
    }
    if constexpr (TURN != TURN_NONE) {
        float p[8];
        partners<TURN>(t, y, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * t.c[i] + p[i] * t.s[i];
    }
    // What comes next rounds an fp32 number.  (The compiler may otherwise make one instruction of the last product and its conversion to fp16, which
    // rounds once where the other form of the step rounds twice: a byte or two in a million of a cache's.)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("" : "+v"(y[i]));
}

// One side (q or k) of the step.
struct NormRopeSide {
    const char* x;
    int64_t rs, hs;      // strides in elements
    char* y;             // dense [rows, heads, dim]
    const char* weight;  // or null
    int heads;
    // backward
    const char* dy;
    int64_t dy_rs, dy_hs;
    char* dx;
    int dw;              // whether the weight's gradient is wanted
};

struct NormRopeParams {
    NormRopeSide side[2];  // q, k
    const void* positions;
    int positions_i64;
    Turn turn;
    float eps, inv_dim;
    int64_t rows;
    int dim, heads_per_group;
    float* partial;  // backward: [workgroups][2][dim]
};

// grid (rows / groups of a workgroup, heads / heads_per_group): heads count through q's, then k's.  Bytes bound it: 151302 rows of eight
// heads of q and four of k, 128 columns, 160 us (930 MB, 5.8 TB/s); 32 rows 5 us, which is one launch.
template <class T, int LPV, int TURN>
__global__ __launch_bounds__(256) void hstu_norm_rope_kernel(const NormRopeParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 4;
    // Lanes without columns, and groups without a row, go along with the last of them that there are and store nothing: loads need no
    // condition then.
    const int l = threadIdx.x % LPV;
    const bool cols = 8 * l < p.dim;
    const int col0 = cols ? 8 * l : p.dim - 8;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPV;
    const bool there = cols && row < p.rows;
    if (row >= p.rows) row = p.rows - 1;
    LaneTurn t;
    t.lane(p.turn, col0, l);
    if constexpr (TURN != TURN_NONE) t.row(p.turn, index_at(p.positions, p.positions_i64, row), col0);
    const int first = blockIdx.y * p.heads_per_group, last = min(first + p.heads_per_group, p.side[0].heads + p.side[1].heads);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const NormRopeSide& s = p.side[which];
        const int base = which ? p.side[0].heads : 0;
        const int h0 = max(first - base, 0), h1 = min(last - base, s.heads);
        if (h0 >= h1) continue;
        float w[8];
        lane_weights((const T*)s.weight, col0, w);
        const T* x = (const T*)s.x + row * s.rs + col0;
        T* out = (T*)s.y + row * s.heads * p.dim + col0;
        for (int h = h0; h < h1; h += AHEAD) {
            Cols<T> in[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) in[a].load(x + (int64_t)min(h + a, h1 - 1) * s.hs);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (h + a >= h1) break;  // (the same for the whole workgroup)
                float y[8];
                norm_and_turn<T, LPV, TURN>(t, in[a], w, cols, s.weight != nullptr, true, p.inv_dim, p.eps, y);
                Cols<T> o;
                o.put(y);
                if (there) o.store(out + (h + a) * p.dim);
            }
        }
    }
}

// The same grid, but a workgroup goes on to further rows, so that the sums for the weights stay in registers: each lane adds up its
// columns, the groups of a workgroup meet in LDS, and the workgroups' sums are added by the kernel below.  151302 rows as above: 264 us
// (1.39 GB, 5.3 TB/s), and 7 for the sums.
template <class T, int LPV, int TURN>
__global__ __launch_bounds__(256) void hstu_norm_rope_bwd_kernel(const NormRopeParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 2;
    __shared__ float meet[256 * 8];
    const int l = threadIdx.x % LPV;
    const bool cols = 8 * l < p.dim;  // (as in the forward)
    const int col0 = cols ? 8 * l : p.dim - 8;
    LaneTurn t;
    t.lane(p.turn, col0, l);
    const int first = blockIdx.y * p.heads_per_group, last = min(first + p.heads_per_group, p.side[0].heads + p.side[1].heads);
    float sum[2][8];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[which][i] = 0.f;
    for (int64_t base_row = (int64_t)blockIdx.x * GROUPS; base_row < p.rows; base_row += (int64_t)gridDim.x * GROUPS) {
        int64_t row = base_row + threadIdx.x / LPV;
        const bool there = cols && row < p.rows;
        if (row >= p.rows) row = p.rows - 1;
        if constexpr (TURN != TURN_NONE) t.row(p.turn, index_at(p.positions, p.positions_i64, row), col0);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const NormRopeSide& s = p.side[which];
            const int base = which ? p.side[0].heads : 0;
            const int h0 = max(first - base, 0), h1 = min(last - base, s.heads);
            if (h0 >= h1) continue;
            float w[8];
            lane_weights((const T*)s.weight, col0, w);
            const T* x_of = (const T*)s.x + row * s.rs + col0;
            const T* dy_of = (const T*)s.dy + row * s.dy_rs + col0;
            T* dx_of = (T*)s.dx + row * s.heads * p.dim + col0;
            for (int h = h0; h < h1; h += AHEAD) {
                Cols<T> in[AHEAD], dy[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    const int64_t at = min(h + a, h1 - 1);
                    dy[a].load(dy_of + at * s.dy_hs);
                    if (s.weight) in[a].load(x_of + at * s.hs);
                }
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (h + a >= h1) break;
                    float x[8], d[8], q[8], g[8];
                    dy[a].get(d);
                    if constexpr (TURN != TURN_NONE) {
                        partners<TURN>(t, d, q);
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] = d[i] * t.c[i] - q[i] * t.s[i];  // R^T: the partner's sine is the other's with its sign changed
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] = d[i];
                    }
                    if (s.weight) {
                        in[a].get(x);
                        const float r = inverse_rms<LPV>(x, cols, true, p.inv_dim, p.eps);
                        float dot = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[i] *= r;
                            const float term = g[i] * x[i];
                            sum[which][i] += there ? term : 0.f;
                            dot += term * w[i];
                            g[i] *= w[i];
                        }
                        const float m = group_sum<LPV>(cols ? dot : 0.f) * p.inv_dim;
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] = r * (g[i] - x[i] * m);
                    }
                    Cols<T> out;
                    out.put(g);
                    if (there) out.store(dx_of + (h + a) * p.dim);
                }
            }
        }
    }
    const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (!p.side[which].dw) continue;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) meet[(threadIdx.x / LPV) * (LPV * 8) + 8 * l + i] = sum[which][i];
        __syncthreads();
        for (int col = threadIdx.x; col < p.dim; col += 256) {
            double v[4] = {0, 0, 0, 0};
#pragma unroll 4
            for (int g = 0; g < GROUPS; g += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += meet[(g + i) * (LPV * 8) + col];
            p.partial[(wg * 2 + which) * p.dim + col] = (float)((v[0] + v[1]) + (v[2] + v[3]));
        }
    }
}

// dw[col] = sum over workgroups of partial[workgroup][which][col]: 16 columns to a workgroup, as four lanes of four, and 64 parts of
// the workgroups' sums, four of them in flight.  (With 16 parts of single columns, one load in flight, 2048 sums took 53 us.)
// Here and where groups meet the additions are in 64 bits: they are few, and with all of them in 32 a gradient in fp32 of 5679 terms a column was
// more than 1.2e-7 of its size off, where it is 0.6e-7 to 0.75e-7.
template <class T>
__global__ __launch_bounds__(256) void hstu_norm_rope_dw_kernel(const float* partial, int64_t workgroups, int dim, T* dq_weight, T* dk_weight) {
    typedef __attribute__((ext_vector_type(4))) float f4;
    __shared__ double meet[64][17];
    const int c = threadIdx.x & 3, part = threadIdx.x >> 2, which = blockIdx.y;
    const int col = blockIdx.x * 16 + 4 * c;
    T* out = which ? dk_weight : dq_weight;
    if (!out) return;
    double v[4] = {0, 0, 0, 0};
    if (col < dim) {  // (a multiple of 8)
        const float* from = partial + which * dim + col;
        auto add = [&](f4 x) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += x[k];
        };
        int64_t w = part;
        for (; w + 192 < workgroups; w += 256) {
            f4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = *(const f4*)(from + (w + 64 * i) * 2 * dim);
#pragma unroll
            for (int i = 0; i < 4; ++i) add(x[i]);
        }
        for (; w < workgroups; w += 64) add(*(const f4*)(from + w * 2 * dim));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) meet[part][4 * c + i] = v[i];
    __syncthreads();
    const int one = threadIdx.x & 15, lane16 = threadIdx.x >> 4;
    double total = meet[lane16][one] + meet[lane16 + 16][one] + meet[lane16 + 32][one] + meet[lane16 + 48][one];
    __syncthreads();
    meet[lane16][one] = total;
    __syncthreads();
    if (threadIdx.x < 16 && blockIdx.x * 16 + threadIdx.x < dim) {
        total = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) total += meet[i][threadIdx.x];
        out[blockIdx.x * 16 + threadIdx.x] = (T)(float)total;
    }
}

}  // namespace hstu
