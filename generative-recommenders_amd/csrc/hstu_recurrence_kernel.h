// The gated linear recurrence over jagged sequences, forward and backward, and its step for single rows: column-wise work.
//
//     s = sigmoid(r_t), z = rate softplus(decay) s, a = exp(-z), m = sqrt(1 - a^2), u = sigmoid(i_t) x_t
//     h_t = a h_{t-1} + m u
//     G_t = dh_t + a_{t+1} G_{t+1}
//     dx = G m sigmoid(i),  di = G m u (1 - sigmoid(i)),  q = G (u a^2 s / m - a s h_{t-1}),
//     dr = rate softplus(decay) (1 - s) q,  d decay = rate sigmoid(decay) sum q,  d h_{-1} = a_0 G_0
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hstu_norm_rope.h"

namespace hstu {

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x)); }

// log(1 + exp(d)), and its derivative.
__device__ __forceinline__ float softplus_of(float d) { return fmaxf(d, 0.f) + log1pf(expf(-fabsf(d))); }

// What a row's gates make of it.  1 - a and 1 - a^2 are wanted to their own last places: a is close to one in layers that remember, and what it
// is off by counts once for each of the 1 / (1 - a) rows that h goes back over.  So for small z both come from the series of
// 1 - exp(-z) = z (1 - z/2 + z^2/6 - ...), to z^6 below 1/4 for fp32 tensors and to z^4 below 1/16 for others (off by 1.4e-7 of it at most), and from the
// instruction's exp(-z), good to a unit in the last place, above.
template <class T>
struct Gates {
    float s, a, m, si;
    __device__ __forceinline__ Gates() {}
    __device__ __forceinline__ Gates(float r, float i, float strength) {
        s = sigmoid_of(r), si = sigmoid_of(i);
        const float z = strength * s;
        const float far = __builtin_amdgcn_exp2f(-kLog2e * z);
        float series, e;
        if constexpr (sizeof(T) == 4) {
            series = __builtin_fmaf(z, -1.f / 720, 1.f / 120);
            series = __builtin_fmaf(z, series, -1.f / 24);
        } else {
            series = -1.f / 24;
        }
        series = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, series, 1.f / 6), -.5f), 1.f);
        const bool near = z < (sizeof(T) == 4 ? .25f : .0625f);
        e = near ? z * series : 1.f - far;
        a = near ? 1.f - e : far;
        m = __builtin_amdgcn_sqrtf(e * (2.f - e));
    }
};

template <class T>
__device__ __forceinline__ float decay_at(const void* decay, int f32, int col) {
    return f32 ? ((const float*)decay)[col] : (float)((const T*)decay)[col];
}

struct ScanParams {
    const char *x, *r, *i;
    int64_t x_rs, r_rs, i_rs;  // strides in elements
    char* out;
    const void* decay;
    int decay_f32;
    float rate;
    const void* offsets;
    int offsets_i64, batch;
    int64_t rows;
    int width;
    const float* initial;
    float* final_state;
    // backward
    const char* dout;
    int64_t dout_rs;
    const float* dfinal;
    char *dx, *dr, *di;
    float* dinitial;
    float* states;   // [rows, width]
    float* partial;  // [batch, width], or null
};

// Rows [first, end) of sequence b, within the tensors.
__device__ __forceinline__ void rows_of(const ScanParams& p, int b, int64_t& first, int64_t& end) {
    first = index_at(p.offsets, p.offsets_i64, b), end = index_at(p.offsets, p.offsets_i64, b + 1);
    first = first < 0 ? 0 : first > p.rows ? p.rows : first;
    end = end < first ? first : end > p.rows ? p.rows : end;
}

// A thread per column and sequence, row after row.  grid (columns / 256, batch + 1): the last y clears the rows behind the sequences.
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_kernel(const ScanParams p) {
    const int col = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (col >= p.width) return;
    T* out = (T*)p.out + col;
    int64_t first, end;
    rows_of(p, b < p.batch ? b : b - 1, first, end);
    if (b == p.batch) {
        for (int64_t t = end; t < p.rows; ++t) out[t * p.width] = (T)0.f;
        return;
    }
    const float strength = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col));
    float h = p.initial ? p.initial[(int64_t)b * p.width + col] : 0.f;
    for (int64_t t = first; t < end; ++t) {
        const Gates<T> g((float)((const T*)p.r)[t * p.r_rs + col], (float)((const T*)p.i)[t * p.i_rs + col], strength);
        h = __builtin_fmaf(g.a, h, g.m * g.si * (float)((const T*)p.x)[t * p.x_rs + col]);
        out[t * p.width] = (T)h;
    }
    if (p.final_state) p.final_state[(int64_t)b * p.width + col] = h;
}

template <class T>
__global__ __launch_bounds__(256) void hstu_scan_bwd_kernel(const ScanParams p) {
    const int col = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (col >= p.width) return;
    int64_t first, end;
    rows_of(p, b < p.batch ? b : b - 1, first, end);
    if (b == p.batch) {
        for (int64_t t = end; t < p.rows; ++t)
            for (char* d : {p.dx, p.dr, p.di})
                if (d) ((T*)d)[t * p.width + col] = (T)0.f;
        return;
    }
    const int64_t state = (int64_t)b * p.width + col;
    const float strength = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col));
    float h = p.initial ? p.initial[state] : 0.f;
    for (int64_t t = first; t < end; ++t) {  // states in front of each row
        p.states[t * p.width + col] = h;
        const Gates<T> g((float)((const T*)p.r)[t * p.r_rs + col], (float)((const T*)p.i)[t * p.i_rs + col], strength);
        h = __builtin_fmaf(g.a, h, g.m * g.si * (float)((const T*)p.x)[t * p.x_rs + col]);
    }
    float later = p.dfinal ? p.dfinal[state] : 0.f, sum = 0.f;
    for (int64_t t = end - 1; t >= first; --t) {
        const Gates<T> g((float)((const T*)p.r)[t * p.r_rs + col], (float)((const T*)p.i)[t * p.i_rs + col], strength);
        const float x = (float)((const T*)p.x)[t * p.x_rs + col], u = g.si * x, before = p.states[t * p.width + col];
        const float G = (p.dout ? (float)((const T*)p.dout)[t * p.dout_rs + col] : 0.f) + later;
        const float share = g.m > 0.f ? g.s * __builtin_amdgcn_rcpf(g.m) : 0.f;
        const float q = G * (u * g.a * g.a * share - g.a * g.s * before);
        if (p.dx) ((T*)p.dx)[t * p.width + col] = (T)(G * g.m * g.si);
        if (p.dr) ((T*)p.dr)[t * p.width + col] = (T)(strength * (1.f - g.s) * q);
        if (p.di) ((T*)p.di)[t * p.width + col] = (T)(G * g.m * u * (1.f - g.si));
        sum += q;
        later = g.a * G;
    }
    if (p.dinitial) p.dinitial[state] = later;
    if (p.partial) p.partial[state] = sum;
}

// d decay = rate sigmoid(decay) * the sum of `count` partial sums, in 64 bits.
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_decay_kernel(const float* partial, int64_t count, int width, const void* decay, int f32, float rate, void* out) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= width) return;
    double sum = 0;
    for (int64_t k = 0; k < count; ++k) sum += partial[k * width + col];
    const double d = decay_at<T>(decay, f32, col), v = rate / (1. + exp(-d)) * sum;
    if (f32)
        ((float*)out)[col] = (float)v;
    else
        ((T*)out)[col] = (T)(float)v;
}

struct StepParams {
    const char *x, *r, *i;
    int64_t x_rs, r_rs, i_rs;
    char* out;
    const void* decay;
    int decay_f32;
    float rate;
    float* states;
    int64_t state_rows, state_rs;
    const void *slots, *new_slots;
    int slots_i64, new_slots_i64;
    int64_t rows;
    int width;
};

// grid (columns / 256, rows)
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_step_kernel(const StepParams p) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    const int64_t t = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (col >= p.width || t >= p.rows) return;
    const int64_t from = p.slots ? index_at(p.slots, p.slots_i64, t) : t, to = p.new_slots ? index_at(p.new_slots, p.new_slots_i64, t) : from;
    const bool known = from >= -1 && from < p.state_rows;
    const float strength = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col));
    float h = from >= 0 && known ? p.states[from * p.state_rs + col] : 0.f;
    const Gates<T> g((float)((const T*)p.r)[t * p.r_rs + col], (float)((const T*)p.i)[t * p.i_rs + col], strength);
    h = __builtin_fmaf(g.a, h, g.m * g.si * (float)((const T*)p.x)[t * p.x_rs + col]);
    if (!known) h = __builtin_nanf("");
    ((T*)p.out)[t * p.width + col] = (T)h;
    if (known && to >= 0 && to < p.state_rows) p.states[to * p.state_rs + col] = h;
}

}  // namespace hstu
