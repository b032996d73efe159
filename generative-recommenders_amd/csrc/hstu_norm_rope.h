// Norms of q and k for each head with the position rotation, forward and backward: row-wise work, bound by HBM bandwidth.
//
//     n = x * rsqrt(mean(x^2) + eps) * w,   y = R n       with R the rotation of the row's position (pairs of columns)
//     g = R^T dy,   dw = sum over rows and heads of g * x * r,   dx = r * (g w - x r * mean(g w x r)),   r = rsqrt(...)
//
// A vector (one row, one head) is taken by LPV = dim / 8 lanes (rounded up to a power of two), eight columns to a lane: one 16-byte
// access each way in 16 bits, and the sums over a vector are log2(LPV) lane exchanges.  The partner of a column in the half-split
// form lies rotary / 2 columns on, rotary / 16 lanes away: lanes exchange the columns as they were loaded (four words in 16 bits)
// and norm their partner's themselves, with its weights.  A group of LPV lanes stays with one row for several heads, so that
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
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
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
    // the same columns of lane `byte_lane / 4` of the wave
    __device__ __forceinline__ Cols from_lane(int byte_lane) const {
        Cols o;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) o.w[i] = (unsigned)__builtin_amdgcn_ds_bpermute(byte_lane, (int)w[i]);
        return o;
    }
};

template <int LPV>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = LPV / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// How a lane's eight columns turn: cosines and sines of its columns for one row, and where its partners are.
struct Turn {
    const float* table;
    int64_t table_rows;
    int rotary, interleaved;
};

struct LaneTurn {
    float c[8], s[8];  // interleaved: of the four pairs, in c[0..3], s[0..3]
    int byte_lane;     // half-split: 4 * the partner's lane
    bool turns;        // whether these columns turn
    float sign;        // half-split: y = n c + sign * partner s

    // Everything that does not depend on the row.
    __device__ __forceinline__ void lane(const Turn& t, int col0) {
        const int half = t.rotary >> 1, me = threadIdx.x & 63;
        turns = col0 < t.rotary;
        byte_lane = 4 * me;
        sign = -1.f;
        if (!t.interleaved && turns) {
            const bool first = col0 < half;
            byte_lane = 4 * (me + (first ? half >> 3 : -(half >> 3)));
            sign = first ? -1.f : 1.f;
        }
    }
    // Cosines and sines of position `pos`; false (and zeros) where it is not in the table.
    __device__ __forceinline__ bool row(const Turn& t, int64_t pos, int col0) {
        const bool there = pos >= 0 && pos < t.table_rows;
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.f;
        if (!turns || !there) return there;
        const int half = t.rotary >> 1;
        const float* cp = t.table + pos * t.rotary + (t.interleaved ? col0 >> 1 : (col0 < half ? col0 : col0 - half));
        typedef __attribute__((ext_vector_type(4))) float f4;
        const f4 c0 = *(const f4*)cp, s0 = *(const f4*)(cp + half);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = c0[i], s[i] = s0[i];
        if (!t.interleaved) {
            const f4 c1 = *(const f4*)(cp + 4), s1 = *(const f4*)(cp + half + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[4 + i] = c1[i], s[4 + i] = s1[i];
        }
        return true;
    }
};

// y = R n for a lane's columns; `p`: the partners' columns (half-split only).  BACK: R^T.
template <bool BACK>
__device__ __forceinline__ void turn(const LaneTurn& t, int interleaved, const float (&n)[8], const float (&p)[8], float (&y)[8]) {
    if (!t.turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = n[i];
    } else if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = BACK ? -t.s[i] : t.s[i];
            y[2 * i] = n[2 * i] * t.c[i] - n[2 * i + 1] * s;
            y[2 * i + 1] = n[2 * i + 1] * t.c[i] + n[2 * i] * s;
        }
    } else {
        const float sign = BACK ? -t.sign : t.sign;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = n[i] * t.c[i] + sign * (p[i] * t.s[i]);
    }
}

// The weights of a lane's columns and of their partners; ones without a norm.
template <class T>
__device__ __forceinline__ void lane_weights(const T* weight, int col0, bool there, const LaneTurn& t, float (&w)[8], float (&wp)[8]) {
    if (weight) {
        Cols<T> c;
        c.zero();
        if (there) c.load(weight + col0);
        c.get(w);
        c.from_lane(t.byte_lane).get(wp);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = wp[i] = 1.f;
    }
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

// grid (rows / groups of a workgroup, heads / heads_per_group): heads count through q's, then k's.
template <class T, int LPV>
__global__ __launch_bounds__(256) void hstu_norm_rope_kernel(const NormRopeParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 4;
    const int l = threadIdx.x % LPV, col0 = 8 * l;
    const int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPV;
    const bool there = col0 < p.dim && row < p.rows;
    LaneTurn t;
    t.lane(p.turn, col0);
    bool known = true;
    if (p.turn.rotary) {
        const int64_t pos = row < p.rows ? index_at(p.positions, p.positions_i64, row) : 0;
        known = t.row(p.turn, pos, col0);
    }
    const int first = blockIdx.y * p.heads_per_group, last = min(first + p.heads_per_group, p.side[0].heads + p.side[1].heads);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const NormRopeSide& s = p.side[which];
        const int base = which ? p.side[0].heads : 0;
        const int h0 = max(first - base, 0), h1 = min(last - base, s.heads);
        if (h0 >= h1) continue;
        float w[8], wp[8];
        lane_weights((const T*)s.weight, col0, col0 < p.dim, t, w, wp);
        for (int h = h0; h < h1; h += AHEAD) {
            Cols<T> in[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                in[a].zero();
                if (there && h + a < h1) in[a].load((const T*)s.x + row * s.rs + (int64_t)(h + a) * s.hs + col0);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (h + a >= h1) break;  // (the same for the whole workgroup)
                float x[8], q[8], y[8];
                in[a].get(x);
                in[a].from_lane(t.byte_lane).get(q);
                float r = 1.f;
                if (s.weight) {
                    float sq = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
                    r = rsqrtf(group_sum<LPV>(sq) * p.inv_dim + p.eps);
                }
                if (!known) r = __builtin_nanf("");
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i], q[i] = q[i] * r * wp[i];
                turn<false>(t, p.turn.interleaved, x, q, y);
                Cols<T> out;
                out.put(y);
                if (there) out.store((T*)s.y + (row * s.heads + h + a) * p.dim + col0);
            }
        }
    }
}

// The same grid, but a workgroup goes on to further rows, so that the sums for the weights stay in registers: each lane adds up its
// columns, the groups of a workgroup meet in LDS, and the workgroups' sums are added by the kernel below.
template <class T, int LPV>
__global__ __launch_bounds__(256) void hstu_norm_rope_bwd_kernel(const NormRopeParams p) {
    constexpr int GROUPS = 256 / LPV, AHEAD = 2;
    __shared__ float meet[256 * 8];
    const int l = threadIdx.x % LPV, col0 = 8 * l;
    const int64_t row0 = (int64_t)blockIdx.x * GROUPS;
    LaneTurn t;
    t.lane(p.turn, col0);
    const int first = blockIdx.y * p.heads_per_group, last = min(first + p.heads_per_group, p.side[0].heads + p.side[1].heads);
    float sum[2][8];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[which][i] = 0.f;
    for (int64_t base_row = row0; base_row < p.rows; base_row += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = base_row + threadIdx.x / LPV;
        const bool there = col0 < p.dim && row < p.rows;
        bool known = true;
        if (p.turn.rotary) {
            const int64_t pos = row < p.rows ? index_at(p.positions, p.positions_i64, row) : 0;
            known = t.row(p.turn, pos, col0);
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const NormRopeSide& s = p.side[which];
            const int base = which ? p.side[0].heads : 0;
            const int h0 = max(first - base, 0), h1 = min(last - base, s.heads);
            if (h0 >= h1) continue;
            float w[8];
            {
                Cols<T> c;
                c.zero();
                if (s.weight && col0 < p.dim) c.load((const T*)s.weight + col0);
                c.get(w);
            }
            for (int h = h0; h < h1; h += AHEAD) {
                Cols<T> in[AHEAD], dy[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    in[a].zero(), dy[a].zero();
                    if (there && h + a < h1) {
                        dy[a].load((const T*)s.dy + row * s.dy_rs + (int64_t)(h + a) * s.dy_hs + col0);
                        if (s.weight) in[a].load((const T*)s.x + row * s.rs + (int64_t)(h + a) * s.hs + col0);
                    }
                }
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (h + a >= h1) break;
                    float x[8], d[8], q[8], g[8];
                    dy[a].get(d);
                    dy[a].from_lane(t.byte_lane).get(q);
                    turn<true>(t, p.turn.interleaved, d, q, g);
                    if (!known) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] = there ? __builtin_nanf("") : 0.f;
                    }
                    if (s.weight) {
                        in[a].get(x);
                        float sq = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
                        const float r = rsqrtf(group_sum<LPV>(sq) * p.inv_dim + p.eps);
                        float dot = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[i] *= r;
                            sum[which][i] += g[i] * x[i];
                            g[i] *= w[i];
                            dot += g[i] * x[i];
                        }
                        const float m = group_sum<LPV>(dot) * p.inv_dim;
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] = r * (g[i] - x[i] * m);
                    }
                    Cols<T> out;
                    out.put(g);
                    if (there) out.store((T*)s.dx + (row * s.heads + h + a) * p.dim + col0);
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
        for (int i = 0; i < 8; ++i) meet[(threadIdx.x / LPV) * (LPV * 8) + col0 + i] = sum[which][i];
        __syncthreads();
        for (int col = threadIdx.x; col < p.dim; col += 256) {
            float v = 0.f;
            for (int g = 0; g < GROUPS; ++g) v += meet[g * (LPV * 8) + col];
            p.partial[(wg * 2 + which) * p.dim + col] = v;
        }
    }
}

// dw[col] = sum over workgroups of partial[workgroup][which][col]: 16 columns to a workgroup, 16 lanes to a column.
template <class T>
__global__ __launch_bounds__(256) void hstu_norm_rope_dw_kernel(const float* partial, int64_t workgroups, int dim, T* dq_weight, T* dk_weight) {
    __shared__ float meet[16][17];
    const int c = threadIdx.x & 15, part = threadIdx.x >> 4, which = blockIdx.y;
    const int col = blockIdx.x * 16 + c;
    T* out = which ? dk_weight : dq_weight;
    if (!out) return;
    float v = 0.f;
    if (col < dim)
        for (int64_t w = part; w < workgroups; w += 16) v += partial[(w * 2 + which) * dim + col];
    meet[part][c] = v;
    __syncthreads();
    if (part == 0 && col < dim) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) total += meet[i][c];
        out[col] = (T)total;
    }
}

}  // namespace hstu
