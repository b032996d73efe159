// What stands between two blocks, forward and backward: row-wise work, bound by HBM bandwidth.
//
//     n = norm(y) wp + bp,  d = keep / (1 - p) act(gate) n,  s = x + scale d,  normed = norm(s) wn + bn
//     ds = dout + N(dnormed wn, s),  dx = ds,  dd = ds scale keep / (1 - p),  dgate = dd n act'(gate),  dn = dd act(gate),  dy = N(dn wp, y)
// with N(g, v) = r (g - v^ mean(g v^)) for v^ = r v, r = 1 / sqrt(mean(v^2) + eps), and less its mean where the norm takes v's mean away.
//
// A row is taken by LPR = width / 8 lanes (rounded up to a power of two, at least 8), eight columns to a lane.  Rows of more than 512 columns lie on
// several waves, whose sums meet in LDS.  A group of lanes goes on to further rows with its parameters, and the sums for their gradients, in registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hstu_norm_rope.h"
#include "hstu_philox.h"

namespace hstu {

enum { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_SILU = 2 };
enum { P_POST_WEIGHT, P_POST_BIAS, P_SCALE, P_PRE_WEIGHT, P_PRE_BIAS, P_COUNT };

struct ResidualNormParams {
    const char *x, *y, *gate;  // gate: or null
    int64_t x_rs, y_rs, gate_rs;
    const char* param[P_COUNT];  // each or null
    char *out, *normed;          // normed: or null
    float eps, inv_width;
    int layer_norm, act;
    int64_t rows;
    int width;
    DropoutParams drop;
    // backward
    const char *dout, *dnormed;  // either or null
    int64_t dout_rs, dnormed_rs;
    char *dx, *dy, *dgate;       // each or null
    int wanted;                  // bit k: parameter k's gradient is
    float* partial;              // [workgroups][P_COUNT][width]
};

// Eight columns of a row from column `col` on.  Not ALIGNED (rows that do not lie on 16-byte boundaries, widths that are no multiple of 8): one by one,
// the last column again for those that there are not.
template <class T, bool ALIGNED>
__device__ __forceinline__ void load8(Cols<T>& c, const T* row, int col, int width) {
    if constexpr (ALIGNED) {
        c.load(row + col);
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = row[min(col + i, width - 1)];
        __builtin_memcpy(c.w, v, sizeof(v));
    }
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void store8(const float (&x)[8], T* row, int col, int width) {
    Cols<T> c;
    c.put(x);
    if constexpr (ALIGNED) {
        c.store(row + col);
    } else {
        T v[8];
        __builtin_memcpy(v, c.w, sizeof(v));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) row[col + i] = v[i];
    }
}

// Sums over the lanes of a row, in each of them.  More than one wave to a row: `meet` has two halves, which calls take in turn, so that
// one barrier between write and read is enough.
template <int LPR>
struct RowSums {
    float* meet;  // [2][waves of the workgroup][2]
    int turn, wave, first_wave;
    __device__ __forceinline__ RowSums(float* meet_) : meet(meet_), turn(0), wave(threadIdx.x / 64), first_wave(threadIdx.x / (LPR < 64 ? 64 : LPR) * (LPR < 64 ? 1 : LPR / 64)) {}
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = group_sum<(LPR < 64 ? LPR : 64)>(v[k]);
        if constexpr (LPR > 64) {
            float* here = meet + turn * 32;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < N; ++k) here[2 * wave + k] = v[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < LPR / 64; ++w) sum += here[2 * (first_wave + w) + k];
                v[k] = sum;
            }
        }
    }
};

// v to v^, and r.  `mine`: how many of the lane's columns there are (the others hold another's).
template <class SUMS>
__device__ __forceinline__ float normalise(float (&v)[8], int mine, const ResidualNormParams& p, SUMS& sums) {
    if (p.layer_norm) {
        float m[1] = {0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) m[0] += i < mine ? v[i] : 0.f;
        sums(m);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= m[0] * p.inv_width;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) q[0] += i < mine ? v[i] * v[i] : 0.f;
    sums(q);
    const float r = 1.f / sqrtf(q[0] * p.inv_width + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= r;
    return r;
}

// g to N(g, v).
template <class SUMS>
__device__ __forceinline__ void normalise_grad(float (&g)[8], const float (&unit)[8], float r, int mine, const ResidualNormParams& p, SUMS& sums) {
    float d[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) d[0] += i < mine ? g[i] * unit[i] : 0.f, d[1] += i < mine ? g[i] : 0.f;
    sums(d);
    const float along = d[0] * p.inv_width, mean = p.layer_norm ? d[1] * p.inv_width : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = r * (g[i] - unit[i] * along - mean);
}

// keep / (1 - p) of eight elements from number `at` on.
template <bool ALIGNED>
__device__ __forceinline__ void kept8(const DropoutParams& d, uint64_t at, float (&keep)[8]) {
    constexpr int GROUPS = ALIGNED ? 2 : 3;
    uint32_t w[4 * GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const PhiloxWords q = dropout_words(d, (at >> 2) + g);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * g + i] = q.w[i];
    }
    const int off = ALIGNED ? 0 : (int)(at & 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t word = w[i];
        if constexpr (!ALIGNED) word = off == 0 ? w[i] : off == 1 ? w[i + 1] : off == 2 ? w[i + 2] : w[i + 3];
        keep[i] = word >= d.thresh ? d.scale : 0.f;
    }
}

// act(gate) and its derivative.
__device__ __forceinline__ void activate(int act, float g, float& value, float& slope) {
    value = g, slope = 1.f;
    if (act == ACT_NONE) return;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * g));
    value = act == ACT_SIGMOID ? s : g * s;
    slope = act == ACT_SIGMOID ? s * (1.f - s) : s * (1.f + g * (1.f - s));
}

template <class T, int LPR, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_residual_norm_kernel(const ResidualNormParams p) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, GROUPS = THREADS / LPR;
    __shared__ float meet[64];
    RowSums<LPR> sums(meet);
    const int l = threadIdx.x % LPR;
    const bool cols = 8 * l < p.width;
    const int col = cols ? 8 * l : 0;
    const int mine = min(max(p.width - 8 * l, 0), 8);
    Cols<T> param[P_COUNT];
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k)
        if (p.param[k]) load8<T, ALIGNED>(param[k], (const T*)p.param[k], col, p.width);
    for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t at = base + threadIdx.x / LPR, row = at < p.rows ? at : p.rows - 1;
        const bool store = cols && at < p.rows;
        Cols<T> cx, cy, cg;
        load8<T, ALIGNED>(cy, (const T*)p.y + row * p.y_rs, col, p.width);
        if (p.gate) load8<T, ALIGNED>(cg, (const T*)p.gate + row * p.gate_rs, col, p.width);
        load8<T, ALIGNED>(cx, (const T*)p.x + row * p.x_rs, col, p.width);
        float v[8], w[8];
        cy.get(v);
        if (p.param[P_POST_WEIGHT]) {
            normalise(v, mine, p, sums);
            param[P_POST_WEIGHT].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= w[i];
            if (p.param[P_POST_BIAS]) {
                param[P_POST_BIAS].get(w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += w[i];
            }
        }
        if (p.gate) {
            cg.get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float value, slope;
                activate(p.act, w[i], value, slope);
                v[i] *= value;
            }
        }
        if (p.drop.thresh) {
            kept8<ALIGNED>(p.drop, (uint64_t)row * p.width + col, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i] != 0.f ? v[i] * w[i] : 0.f;
        }
        if (p.param[P_SCALE]) {
            param[P_SCALE].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= w[i];
        }
        cx.get(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += w[i];
        if (store) store8<T, ALIGNED>(v, (T*)p.out + row * p.width, col, p.width);
        if (p.param[P_PRE_WEIGHT]) {
            normalise(v, mine, p, sums);
            param[P_PRE_WEIGHT].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= w[i];
            if (p.param[P_PRE_BIAS]) {
                param[P_PRE_BIAS].get(w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += w[i];
            }
            if (store) store8<T, ALIGNED>(v, (T*)p.normed + row * p.width, col, p.width);
        }
    }
}

template <class T, int LPR, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_residual_norm_bwd_kernel(const ResidualNormParams p) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, GROUPS = THREADS / LPR;
    __shared__ float meet[64];
    __shared__ float groups[THREADS * 8];
    RowSums<LPR> sums(meet);
    const int l = threadIdx.x % LPR;
    const bool cols = 8 * l < p.width;
    const int col = cols ? 8 * l : 0;
    const int mine = min(max(p.width - 8 * l, 0), 8);
    float total[P_COUNT][8];
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) total[k][i] = 0.f;
    Cols<T> param[P_COUNT];
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k)
        if (p.param[k]) load8<T, ALIGNED>(param[k], (const T*)p.param[k], col, p.width);
    for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t at = base + threadIdx.x / LPR, row = at < p.rows ? at : p.rows - 1;
        const bool store = cols && at < p.rows;
        const float counts = at < p.rows ? 1.f : 0.f;
        Cols<T> cx, cy, cg, cd, cn;
        load8<T, ALIGNED>(cy, (const T*)p.y + row * p.y_rs, col, p.width);
        if (p.gate) load8<T, ALIGNED>(cg, (const T*)p.gate + row * p.gate_rs, col, p.width);
        load8<T, ALIGNED>(cx, (const T*)p.x + row * p.x_rs, col, p.width);
        if (p.dout) load8<T, ALIGNED>(cd, (const T*)p.dout + row * p.dout_rs, col, p.width);
        if (p.dnormed) load8<T, ALIGNED>(cn, (const T*)p.dnormed + row * p.dnormed_rs, col, p.width);
        // forward again: unit = y^, n, act(gate), its slope, keep, s
        float unit[8], n[8], value[8], slope[8], keep[8], s[8], w[8];
        float r = 1.f;
        cy.get(unit);
        if (p.param[P_POST_WEIGHT]) r = normalise(unit, mine, p, sums);
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = unit[i];
        if (p.param[P_POST_WEIGHT]) {
            param[P_POST_WEIGHT].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] *= w[i];
        }
        if (p.param[P_POST_BIAS]) {
            param[P_POST_BIAS].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] += w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) value[i] = 1.f, slope[i] = 0.f, keep[i] = 1.f;
        if (p.gate) {
            cg.get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) activate(p.act, w[i], value[i], slope[i]);
        }
        if (p.drop.thresh) kept8<ALIGNED>(p.drop, (uint64_t)row * p.width + col, keep);
        float scale[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) scale[i] = 1.f;
        if (p.param[P_SCALE]) param[P_SCALE].get(scale);
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
        if (p.dout) cd.get(d);
        if (p.dnormed) {
            cx.get(s);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += keep[i] != 0.f ? n[i] * value[i] * keep[i] * scale[i] : 0.f;
            const float rs = normalise(s, mine, p, sums);
            float g[8];
            cn.get(g);
            param[P_PRE_WEIGHT].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                total[P_PRE_WEIGHT][i] += counts != 0.f ? g[i] * s[i] : 0.f;
                total[P_PRE_BIAS][i] += counts != 0.f ? g[i] : 0.f;
                g[i] *= w[i];
            }
            normalise_grad(g, s, rs, mine, p, sums);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] += g[i];
        }
        if (p.dx && store) store8<T, ALIGNED>(d, (T*)p.dx + row * p.width, col, p.width);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            total[P_SCALE][i] += counts != 0.f && keep[i] != 0.f ? d[i] * n[i] * value[i] * keep[i] : 0.f;
            d[i] = keep[i] != 0.f ? d[i] * scale[i] * keep[i] : 0.f;
        }
        if (p.dgate && store) {
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = d[i] * n[i] * slope[i];
            store8<T, ALIGNED>(g, (T*)p.dgate + row * p.width, col, p.width);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= value[i];
        if (p.param[P_POST_WEIGHT]) {
            param[P_POST_WEIGHT].get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                total[P_POST_WEIGHT][i] += counts != 0.f ? d[i] * unit[i] : 0.f;
                total[P_POST_BIAS][i] += counts != 0.f ? d[i] : 0.f;
                d[i] *= w[i];
            }
            normalise_grad(d, unit, r, mine, p, sums);
        }
        if (p.dy && store) store8<T, ALIGNED>(d, (T*)p.dy + row * p.width, col, p.width);
    }
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k) {
        if (!(p.wanted >> k & 1)) continue;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) groups[threadIdx.x * 8 + i] = total[k][i];
        __syncthreads();
        for (int c = threadIdx.x; c < p.width; c += THREADS) {
            double v = 0;
            for (int g = 0; g < GROUPS; ++g) v += groups[g * LPR * 8 + c];
            p.partial[((int64_t)blockIdx.x * P_COUNT + k) * p.width + c] = (float)v;
        }
    }
}

// Parameter k's gradient: the sum over `workgroups` of partial[workgroup][k][column], in 64 bits.  grid (columns / 16, P_COUNT): 16 parts of 16 columns.
struct ParameterGrads {
    void* out[P_COUNT];
};
template <class T>
__global__ __launch_bounds__(256) void hstu_residual_norm_sum_kernel(const float* partial, int64_t workgroups, int width, const ParameterGrads to) {
    __shared__ double meet[16][17];
    const int k = blockIdx.y, c = threadIdx.x & 15, part = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    if (!to.out[k]) return;
    double v = 0;
    if (col < width)
        for (int64_t w = part; w < workgroups; w += 16) v += partial[(w * P_COUNT + k) * width + col];
    meet[part][c] = v;
    __syncthreads();
    if (part || col >= width) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += meet[i][c];
    ((T*)to.out[k])[col] = (T)(float)v;
}

}  // namespace hstu
