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

// The sum over a wave, the same in all lanes for the compiler to know: rows of 16 lanes, then pairs of rows and halves by the instruction's broadcasts.
__device__ __forceinline__ float wave_total(float v) {
    v = group_sum<16>(v);
    v += __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x142, 0xa, 0xf, false));
    v += __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x143, 0xc, 0xf, false));
    return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// Sums over the lanes of a row, in each of them.  More than one wave to a row: `meet` has two halves, which calls take in turn, so that
// one barrier between write and read is enough.
template <int LPR>
struct RowSums {
    float* meet;  // [2][waves of the workgroup][2]
    int turn, wave, first_wave;
    __device__ __forceinline__ RowSums(float* meet_) : meet(meet_), turn(0), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)) {
        first_wave = LPR > 64 ? wave / (LPR / 64) * (LPR / 64) : wave;
    }
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        if constexpr (LPR < 64) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = group_sum<LPR>(v[k]);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = wave_total(v[k]);
        }
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

// What of a lane's eight columns there is: all or none where rows are ALIGNED, else the first `count`.  The others hold columns that are another's.
template <bool ALIGNED>
struct Mine {
    int count;
    template <class F>
    __device__ __forceinline__ float sum(F&& term) const {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if constexpr (ALIGNED)
                v += term(i);
            else
                v += i < count ? term(i) : 0.f;
        return !ALIGNED || count ? v : 0.f;
    }
};

// v to v^, and r: the instruction's root, good to a unit in the last place, corrected once by its residual.
template <bool ALIGNED, class SUMS>
__device__ __forceinline__ float normalise(float (&v)[8], const Mine<ALIGNED>& mine, const ResidualNormParams& p, SUMS& sums) {
    if (p.layer_norm) {
        float m[1] = {mine.sum([&](int i) { return v[i]; })};
        sums(m);
        m[0] *= p.inv_width;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= m[0];
    }
    float q[1] = {mine.sum([&](int i) { return v[i] * v[i]; })};
    sums(q);
    const float x = q[0] * p.inv_width + p.eps, r0 = __builtin_amdgcn_rsqf(x), h = x * r0, low = __builtin_fmaf(x, r0, -h);
    const float fixed = __builtin_fmaf(0.5f * r0, __builtin_fmaf(-low, r0, __builtin_fmaf(-h, r0, 1.f)), r0), r = x > 0x1p-100f && x < 0x1p100f ? fixed : r0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= r;
    return r;
}

// g to N(g, v).
template <bool ALIGNED, class SUMS>
__device__ __forceinline__ void normalise_grad(float (&g)[8], const float (&unit)[8], float r, const Mine<ALIGNED>& mine, const ResidualNormParams& p, SUMS& sums) {
    if (p.layer_norm) {
        float d[2] = {mine.sum([&](int i) { return g[i] * unit[i]; }), mine.sum([&](int i) { return g[i]; })};
        sums(d);
        const float along = d[0] * p.inv_width, mean = d[1] * p.inv_width;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = r * (__builtin_fmaf(-unit[i], along, g[i]) - mean);
    } else {
        float d[1] = {mine.sum([&](int i) { return g[i] * unit[i]; })};
        sums(d);
        const float along = d[0] * p.inv_width;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = r * __builtin_fmaf(-unit[i], along, g[i]);
    }
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

// act(gate), and its derivative.
__device__ __forceinline__ void activate(int act, const float (&g)[8], float (&value)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) value[i] = g[i];
    if (act == ACT_NONE) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) value[i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * g[i]));
    if (act == ACT_SILU)
#pragma unroll
        for (int i = 0; i < 8; ++i) value[i] *= g[i];
}
__device__ __forceinline__ void activate(int act, const float (&g)[8], float (&value)[8], float (&slope)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) value[i] = g[i], slope[i] = 1.f;
    if (act == ACT_NONE) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // With s = 1 / (1 + e), 1 - s is e s to its own last places (as a difference it is 1 % off at 12 and 0 from 17.4 on), and 0 s where e is an infinity.
        const float e = __builtin_amdgcn_exp2f(-1.44269504088896340736f * g[i]);
        value[i] = __builtin_amdgcn_rcpf(1.f + e);
        slope[i] = value[i] * (fminf(e, 0x1p126f) * value[i]);
    }
    if (act == ACT_SILU)
#pragma unroll
        for (int i = 0; i < 8; ++i) slope[i] = __builtin_fmaf(g[i], slope[i], value[i]), value[i] *= g[i];
}

// A row of parameters, as it lies in memory.
template <class T, bool ALIGNED>
__device__ __forceinline__ void load_parameters(Cols<T> (&param)[P_COUNT], const ResidualNormParams& p, int col) {
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k)
        if (p.param[k]) load8<T, ALIGNED>(param[k], (const T*)p.param[k], col, p.width);
}
// v times one of them, v plus one of them: where there is one.
template <class T>
__device__ __forceinline__ void times(float (&v)[8], const Cols<T>& c, const char* there) {
    if (!there) return;
    float w[8];
    c.get(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= w[i];
}
template <class T>
__device__ __forceinline__ void plus(float (&v)[8], const Cols<T>& c, const char* there) {
    if (!there) return;
    float w[8];
    c.get(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += w[i];
}

// 151302 rows of 1024 columns, layer norms with a gate: 307 us (1.55 GB, 5.0 TB/s); 56328 of 512 with dropout 52.
template <class T, int LPR, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_residual_norm_kernel(const ResidualNormParams p) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, GROUPS = THREADS / LPR;
    __shared__ float meet[64];
    RowSums<LPR> sums(meet);
    const int l = threadIdx.x % LPR;
    const Mine<ALIGNED> mine{min(max(p.width - 8 * l, 0), 8)};
    const int col = mine.count ? 8 * l : 0;
    Cols<T> param[P_COUNT];
    load_parameters<T, ALIGNED>(param, p, col);
    for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t at = base + threadIdx.x / LPR, row = at < p.rows ? at : p.rows - 1;
        if (LPR <= 64 && at >= p.rows) break;  // (where rows meet at barriers all go along, with the last one)
        const bool store = mine.count && at < p.rows;
        Cols<T> cx, cy, cg;
        load8<T, ALIGNED>(cy, (const T*)p.y + row * p.y_rs, col, p.width);
        if (p.gate) load8<T, ALIGNED>(cg, (const T*)p.gate + row * p.gate_rs, col, p.width);
        load8<T, ALIGNED>(cx, (const T*)p.x + row * p.x_rs, col, p.width);
        float v[8], w[8];
        cy.get(v);
        if (p.param[P_POST_WEIGHT]) {
            normalise(v, mine, p, sums);
            times(v, param[P_POST_WEIGHT], p.param[P_POST_WEIGHT]);
            plus(v, param[P_POST_BIAS], p.param[P_POST_BIAS]);
        }
        if (p.gate) {
            float value[8];
            cg.get(w);
            activate(p.act, w, value);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= value[i];
        }
        if (p.drop.thresh) {
            kept8<ALIGNED>(p.drop, (uint64_t)row * p.width + col, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i] != 0.f ? v[i] * w[i] : 0.f;  // (what is dropped may be an infinity)
        }
        times(v, param[P_SCALE], p.param[P_SCALE]);
        cx.get(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += w[i];
        if (store) store8<T, ALIGNED>(v, (T*)p.out + row * p.width, col, p.width);
        if (!p.param[P_PRE_WEIGHT]) continue;
        normalise(v, mine, p, sums);
        times(v, param[P_PRE_WEIGHT], p.param[P_PRE_WEIGHT]);
        plus(v, param[P_PRE_BIAS], p.param[P_PRE_BIAS]);
        if (store) store8<T, ALIGNED>(v, (T*)p.normed + row * p.width, col, p.width);
    }
}

// Results of the forward are worked out again; a group of lanes adds up the parameters' gradients over its rows, in a workgroup the groups meet in LDS, and
// the kernel below adds the workgroups'.
template <class T, int LPR, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_residual_norm_bwd_kernel(const ResidualNormParams p) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, GROUPS = THREADS / LPR;
    __shared__ float meet[64];
    __shared__ float groups[THREADS * 8];
    RowSums<LPR> sums(meet);
    const int l = threadIdx.x % LPR;
    const Mine<ALIGNED> mine{min(max(p.width - 8 * l, 0), 8)};
    const int col = mine.count ? 8 * l : 0;
    float total[P_COUNT][8];
#pragma unroll
    for (int k = 0; k < P_COUNT; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) total[k][i] = 0.f;
    Cols<T> param[P_COUNT];
    load_parameters<T, ALIGNED>(param, p, col);
    const bool post = p.param[P_POST_WEIGHT];
    for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t at = base + threadIdx.x / LPR, row = at < p.rows ? at : p.rows - 1;
        if (LPR <= 64 && at >= p.rows) break;
        // A group behind the last row goes along with it where rows meet at barriers, and adds nothing to the parameters' gradients; the same for a wave, which
        // has one group there.
        const bool there = LPR <= 64 || __builtin_amdgcn_readfirstlane(at < p.rows), store = mine.count && there;
        Cols<T> cx, cy, cg, cd, cn;
        load8<T, ALIGNED>(cy, (const T*)p.y + row * p.y_rs, col, p.width);
        if (p.gate) load8<T, ALIGNED>(cg, (const T*)p.gate + row * p.gate_rs, col, p.width);
        load8<T, ALIGNED>(cx, (const T*)p.x + row * p.x_rs, col, p.width);
        if (p.dout) load8<T, ALIGNED>(cd, (const T*)p.dout + row * p.dout_rs, col, p.width);
        if (p.dnormed) load8<T, ALIGNED>(cn, (const T*)p.dnormed + row * p.dnormed_rs, col, p.width);
#pragma unroll
        for (int i = 0; i < Cols<T>::WORDS; ++i) cd.w[i] = p.dout ? cd.w[i] : 0;
        // forward again: unit = y^, branch = act(gate) n as dropped
        float unit[8], n[8], value[8], slope[8], keep[8], branch[8], w[8], d[8];
        float r = 1.f;
        cy.get(unit);
        if (post) r = normalise(unit, mine, p, sums);
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = unit[i];
        times(n, param[P_POST_WEIGHT], p.param[P_POST_WEIGHT]);
        plus(n, param[P_POST_BIAS], p.param[P_POST_BIAS]);
#pragma unroll
        for (int i = 0; i < 8; ++i) branch[i] = n[i];
        if (p.gate) {
            cg.get(w);
            activate(p.act, w, value, slope);
#pragma unroll
            for (int i = 0; i < 8; ++i) branch[i] *= value[i];
        }
        if (p.drop.thresh) {
            kept8<ALIGNED>(p.drop, (uint64_t)row * p.width + col, keep);
#pragma unroll
            for (int i = 0; i < 8; ++i) branch[i] = keep[i] != 0.f ? branch[i] * keep[i] : 0.f;
        }
        cd.get(d);
        if (p.dnormed) {
            float s[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = branch[i];
            times(s, param[P_SCALE], p.param[P_SCALE]);
            cx.get(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += w[i];
            const float rs = normalise(s, mine, p, sums);
            cn.get(g);
            if (there)
#pragma unroll
                for (int i = 0; i < 8; ++i) total[P_PRE_WEIGHT][i] = __builtin_fmaf(g[i], s[i], total[P_PRE_WEIGHT][i]);
            if (there && p.param[P_PRE_BIAS])
#pragma unroll
                for (int i = 0; i < 8; ++i) total[P_PRE_BIAS][i] += g[i];
            times(g, param[P_PRE_WEIGHT], p.param[P_PRE_WEIGHT]);
            normalise_grad(g, s, rs, mine, p, sums);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] += g[i];
        }
        if (p.dx && store) store8<T, ALIGNED>(d, (T*)p.dx + row * p.width, col, p.width);
        if (p.param[P_SCALE]) {
            if (there)
#pragma unroll
                for (int i = 0; i < 8; ++i) total[P_SCALE][i] = __builtin_fmaf(d[i], branch[i], total[P_SCALE][i]);
            times(d, param[P_SCALE], p.param[P_SCALE]);
        }
        if (p.drop.thresh)
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = keep[i] != 0.f ? d[i] * keep[i] : 0.f;
        if (p.gate) {
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = d[i] * n[i] * slope[i], d[i] *= value[i];
            if (p.dgate && store) store8<T, ALIGNED>(g, (T*)p.dgate + row * p.width, col, p.width);
        }
        if (post) {
            if (there)
#pragma unroll
                for (int i = 0; i < 8; ++i) total[P_POST_WEIGHT][i] = __builtin_fmaf(d[i], unit[i], total[P_POST_WEIGHT][i]);
            if (there && p.param[P_POST_BIAS])
#pragma unroll
                for (int i = 0; i < 8; ++i) total[P_POST_BIAS][i] += d[i];
            times(d, param[P_POST_WEIGHT], p.param[P_POST_WEIGHT]);
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
            p.partial[((int64_t)k * gridDim.x + blockIdx.x) * p.width + c] = (float)v;
        }
    }
}

// A parameter's gradient: the sum over `workgroups` of partial[parameter][workgroup][column], in 64 bits.  grid (columns / 16, parameters that are wanted): 16
// columns to a workgroup, 64 parts of the sums, eight of them in flight.
struct ParameterGrads {
    void* out[P_COUNT];
    int which[P_COUNT];
};
template <class T>
__global__ __launch_bounds__(1024) void hstu_residual_norm_sum_kernel(const float* partial, int64_t workgroups, int width, const ParameterGrads to) {
    __shared__ double meet[64][17];
    const int c = threadIdx.x & 15, part = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    const float* from = partial + to.which[blockIdx.y] * workgroups * width + col;
    double v = 0;
    if (col < width) {
        int64_t k = part;
        for (; k + 448 < workgroups; k += 512) {
            float x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = from[(k + 64 * q) * width];
#pragma unroll
            for (int q = 0; q < 8; ++q) v += x[q];
        }
        for (; k < workgroups; k += 64) v += from[k * width];
    }
    meet[part][c] = v;
    __syncthreads();
    if (part >= 4) return;
    v = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) v += meet[part + 4 * q][c];
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    if (part == 0 && col < width) ((T*)to.out[blockIdx.y])[col] = (T)(float)v;
}

}  // namespace hstu
