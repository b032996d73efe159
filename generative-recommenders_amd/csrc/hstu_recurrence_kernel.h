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

#include <type_traits>

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
    float* saved;                // [rows / 64][width]: h in front of every 64th row
    int tiles, col_blocks;
    unsigned long long* words;   // [tiles][width], then [tiles / kGroup][width]: what tiles, and groups of them, make of h; 0: not there yet
    unsigned* ticket;
    int64_t clear;               // how many words, and the ticket behind them
    // backward
    const char* dout;
    int64_t dout_rs;
    const float* dfinal;
    char *dx, *dr, *di;
    float* dinitial;
    float* partial;  // [tiles][width], or null
};

// V neighbouring columns of a row, four bytes at most.
template <class T, int V>
struct Piece {
    static_assert(V * sizeof(T) <= 4, "one register");
    unsigned w;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V * sizeof(T) == 4)
            w = *(const unsigned*)p;
        else
            w = *(const uint16_t*)p;
    }
    __device__ __forceinline__ float get(int v) const {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(w);
        else
            return (float)__builtin_bit_cast(T, (uint16_t)(v ? w >> 16 : w));
    }
    __device__ __forceinline__ static void put(const float (&x)[V], T* p) {
        if constexpr (V == 1) {
            *p = (T)x[0];
        } else {
            typedef __attribute__((ext_vector_type(2))) T T2;
            T2 v;
            v[0] = (T)x[0], v[1] = (T)x[1];
            *(T2*)p = v;
        }
    }
};

// Rows behind the last sequence, or 0.
__device__ __forceinline__ int64_t rows_end(const ScanParams& p) {
    const int64_t end = index_at(p.offsets, p.offsets_i64, p.batch);
    return end < 0 ? 0 : end > p.rows ? p.rows : end;
}

// Where sequences begin and end in a tile of R rows.
template <int R>
struct TileRows {
    int begins[R], ends[R];  // the sequence whose first, whose last row it is, or -1
    int64_t first, behind;   // first row of the sequence that the tile's first row is of; the row behind the one that its last row is of
    int low;
    template <int THREADS>
    __device__ __forceinline__ void clear() {
        for (int k = threadIdx.x; k < R; k += THREADS) begins[k] = ends[k] = -1;
        if (threadIdx.x == 0) first = behind = -1, low = 0;
    }
    // After a barrier behind clear(); needs one behind it.  The sequences' offsets are narrowed down by THREADS at a time and then looked at side by
    // side, from the one that row t0 is of to those that begin behind the tile.  Where offsets are not in order every index stays in bounds and every loop
    // ends all the same.
    template <int THREADS>
    __device__ __forceinline__ void find(const ScanParams& p, int64_t t0, int64_t end) {
        int lo = 0, hi = p.batch;
        while (hi - lo >= THREADS) {
            const int step = (hi - lo + THREADS - 1) / THREADS, at = lo + (int)threadIdx.x * step;
            if (at <= hi && index_at(p.offsets, p.offsets_i64, at) <= t0) atomicMax(&low, at);
            __syncthreads();
            lo = max(lo, low), hi = min(hi, lo + step);
            __syncthreads();
        }
        for (int base = lo; base < p.batch; base += THREADS) {
            const int b = base + threadIdx.x;
            if (b < p.batch) {
                const int64_t v = index_at(p.offsets, p.offsets_i64, b), e = min(index_at(p.offsets, p.offsets_i64, b + 1), end);
                if (e > v) {
                    if (v >= t0 && v < t0 + R) begins[v - t0] = b;
                    if (e > t0 && e <= t0 + R) ends[e - 1 - t0] = b;
                    if (v <= t0 && e > t0) first = v;
                    if (v < t0 + R && e >= t0 + R) behind = e;
                }
            }
            if (base + THREADS < p.batch && index_at(p.offsets, p.offsets_i64, base + THREADS) >= t0 + R) break;  // (the same for all)
        }
    }
};

// Bit k: whether rows[k] is a sequence's; the same in all lanes.
template <int R>
__device__ __forceinline__ void marks(const int (&rows)[R], uint64_t (&bits)[R / 64]) {
#pragma unroll
    for (int k = 0; k < R / 64; ++k) bits[k] = __ballot(rows[64 * k + (threadIdx.x & 63)] >= 0);
}
template <int ROWS, int N>
__device__ __forceinline__ unsigned marks_of(const uint64_t (&bits)[N], int wave) {
    const int at = wave * ROWS;
    return (unsigned)(bits[at >> 6] >> (at & 63)) & ((1u << ROWS) - 1);
}

// ---- tiles joined along the rows ----
//
// What a run of rows makes of the h in front of it is A h + H.  Each tile works out its (A, H), puts them down as one word for each column, and takes
// up those of the tiles in front of it, back to the first of its sequence.  A word is written and read as a whole, and is never 0 once written (A's sign bit
// is set: A is not negative), so it needs no flag and no fence beside it.  Every kGroup-th tile also joins its group's words into one, so
// that a tile of a long sequence takes up tiles / kGroup + 2 kGroup words and nothing waits for more than two others one behind another.  Tiles are
// numbered by a ticket as workgroups begin: those in front have been begun and wait for no tile behind them, so each wait ends.  (The limit on it only
// keeps a broken device from hanging.)  Which words are joined in which order goes by the tile's number and its sequence's first row alone.
constexpr int kGroup = 16;

__device__ __forceinline__ void put_word(unsigned long long* at, float A, float H) {
    const unsigned long long w = (unsigned long long)__float_as_uint(H) << 32 | (__float_as_uint(A) | 0x80000000u);
    __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Joins n words, word k at at(k), into (A, H): earlier ones are applied first.
template <int V, class AT>
__device__ __forceinline__ void join_words(int from, int to, AT&& at, float (&A)[V], float (&H)[V]) {
    constexpr int AHEAD = 4;
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
    for (int k = from; k < to; k += AHEAD) {
        unsigned long long w[AHEAD][V];
        bool there = false;
        for (int tries = 0; tries < (1 << 22) && !there; ++tries) {
            if (tries) __builtin_amdgcn_s_sleep(1);
            bool mine = true;
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
#pragma unroll
                for (int v = 0; v < V; ++v) w[q][v] = __hip_atomic_load(at(min(k + q, to - 1)) + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
#pragma unroll
                for (int v = 0; v < V; ++v) mine = mine && w[q][v] != 0;
            there = __all(mine);
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (k + q >= to) break;  // (the same for the wave)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float a = __uint_as_float((unsigned)w[q][v] & 0x7fffffffu), h = there ? __uint_as_float((unsigned)(w[q][v] >> 32)) : __builtin_nanf("");
                H[v] = k + q == from ? h : __builtin_fmaf(a, H[v], h);
                A[v] = k + q == from ? a : a * A[v];
            }
        }
    }
}

// The waves of a workgroup join n words: each a part of them, in LDS the parts.  Every thread of the workgroup calls; `meet` is free before and after.
template <int V, int WAVES, class AT>
__device__ __forceinline__ void join_together(int n, AT&& at, float2 (*meet)[64 * V], int wave, float (&A)[V], float (&H)[V]) {
    const int lane = threadIdx.x & 63, per = (n + WAVES - 1) / WAVES, from = min(wave * per, n), to = min(from + per, n);
    if (from < to) {
        join_words<V>(from, to, at, A, H);
#pragma unroll
        for (int v = 0; v < V; ++v) meet[wave][lane * V + v] = float2{A[v], H[v]};
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, H[v] = 0.f;
    for (int w = 0; w * per < n; ++w)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 s = meet[w][lane * V + v];
            H[v] = w ? __builtin_fmaf(s.x, H[v], s.y) : s.y;
            A[v] = w ? s.x * A[v] : s.x;
        }
    __syncthreads();
}

// Takes up what the tiles from `from` up to `tile` make of a column's h.
template <int V, int WAVES>
__device__ __forceinline__ void join_tiles(const ScanParams& p, int from, int tile, int col, float2 (*meet)[64 * V], int wave, float (&H)[V]) {
    const unsigned long long* words = p.words + col;
    const unsigned long long* groups = words + (int64_t)p.tiles * p.width;
    const int group = tile / kGroup, whole = (from + kGroup - 1) / kGroup;  // groups [whole, group) lie behind `from`
    const int singles = whole < group ? whole * kGroup - from : tile - from, joined = whole < group ? group - whole : 0;
    const int n = singles + joined + (whole < group ? tile - group * kGroup : 0);
    float A[V];
    join_together<V, WAVES>(
        n,
        [&](int k) {
            const unsigned long long* base = k >= singles && k < singles + joined ? groups : words;
            const int64_t at = k < singles ? from + k : k < singles + joined ? whole + k - singles : group * kGroup + k - singles - joined;
            return base + at * p.width;
        },
        meet, wave, A, H);
}

// A tile's own (A, H), by its last wave to come, and its group's by the last tile of one.  Every thread calls; `meet` is free before and after.
template <int V, int WAVES>
__device__ __forceinline__ void put_tile(const ScanParams& p, int tile, int col, bool mine, bool me, const float (&A)[V], const float (&H)[V], float2 (*meet)[64 * V],
                                         int wave) {
    if (me && mine)
#pragma unroll
        for (int v = 0; v < V; ++v) put_word(p.words + (int64_t)tile * p.width + col + v, A[v], H[v]);
    if (tile % kGroup != kGroup - 1) return;
    float a[V], h[V];
    const unsigned long long* first = p.words + (int64_t)(tile - (kGroup - 1)) * p.width + col;
    join_together<V, WAVES>(kGroup - 1, [&](int k) { return first + (int64_t)k * p.width; }, meet, wave, a, h);
    if (me && mine)
#pragma unroll
        for (int v = 0; v < V; ++v) put_word(p.words + (int64_t)(p.tiles + tile / kGroup) * p.width + col + v, A[v] * a[v], __builtin_fmaf(A[v], h[v], H[v]));
}

// No word is there yet; states of sequences without rows are what they were.
__global__ __launch_bounds__(256) void hstu_scan_clear_kernel(const ScanParams p) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    for (int64_t k = at; k < p.clear; k += step) p.words[k] = 0;
    if (at == 0 && p.ticket) *p.ticket = 0;
    if (p.final_state)
        for (int64_t k = at; k < (int64_t)p.batch * p.width; k += step) p.final_state[k] = p.initial ? p.initial[k] : 0.f;
}

template <class T, int V, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 4) void hstu_scan_kernel(const ScanParams p) {
    constexpr int R = ROWS * WAVES, COLS = 64 * V;
    __shared__ TileRows<R> map;
    __shared__ float2 sums[WAVES][COLS], meet[WAVES][COLS];
    __shared__ unsigned number;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    map.template clear<64 * WAVES>();
    if (threadIdx.x == 0) number = p.words ? atomicAdd(p.ticket, 1u) : blockIdx.x;
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(number), tile = n / p.col_blocks, col0 = (n % p.col_blocks) * COLS + lane * V, col = min(col0, p.width - V);
    const bool mine = col0 < p.width;
    const int64_t t0 = (int64_t)tile * R, w0 = t0 + wave * ROWS, end = rows_end(p);
    T* out = (T*)p.out + w0 * p.width + col;
    if (t0 >= end) {  // rows behind the last sequence (no tile in front of it waits for this one)
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (mine && w0 + j < p.rows) {
                const float zero[V] = {};
                Piece<T, V>::put(zero, out + (int64_t)j * p.width);
            }
        return;
    }
    Piece<T, V> x[ROWS], r[ROWS], i[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t row = min(w0 + j, p.rows - 1);
        x[j].load((const T*)p.x + row * p.x_rs + col);
        r[j].load((const T*)p.r + row * p.r_rs + col);
        i[j].load((const T*)p.i + row * p.i_rs + col);
    }
    float strength[V], a[ROWS][V], b[ROWS][V], A[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) strength[v] = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col + v)), A[v] = 1.f, H[v] = 0.f;
    map.template find<64 * WAVES>(p, t0, end);
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gates<T> g(r[j].get(v), i[j].get(v), strength[v]);
            a[j][v] = g.a, b[j][v] = g.m * g.si * x[j].get(v);
        }
    __syncthreads();
    uint64_t bits[R / 64];
    marks(map.begins, bits);
    const unsigned begins = marks_of<ROWS>(bits, wave);
    if (begins && p.initial)
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (begins >> j & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) b[j][v] = __builtin_fmaf(a[j][v], p.initial[(int64_t)map.begins[wave * ROWS + j] * p.width + col + v], b[j][v]);
    // (a, b) row by row; a row that begins a sequence knows nothing of what is in front of it, whatever that is
    auto rows = [&](auto any, auto&& each) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            if (decltype(any)::value && begins >> j & 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) H[v] = b[j][v], A[v] = 0.f;
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) H[v] = __builtin_fmaf(a[j][v], H[v], b[j][v]), A[v] *= a[j][v];
            }
            each(j);
        }
    };
    auto nothing = [](int) {};
    if (begins)
        rows(std::true_type{}, nothing);
    else
        rows(std::false_type{}, nothing);
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane * V + v] = float2{A[v], H[v]};
    __syncthreads();
    float fA[V], fH[V];  // of the waves in front
    bool cut = false;    // whether a sequence begins in one of them
#pragma unroll
    for (int v = 0; v < V; ++v) fA[v] = 1.f, fH[v] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) {
        if (w >= wave) break;
        const bool begun = marks_of<ROWS>(bits, w) != 0;
        cut = cut || begun;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 s = sums[w][lane * V + v];
            fH[v] = begun ? s.y : __builtin_fmaf(s.x, fH[v], s.y);
            fA[v] = begun ? 0.f : s.x * fA[v];
        }
    }
    if (p.words) {
#pragma unroll
        for (int v = 0; v < V; ++v) H[v] = begins ? H[v] : __builtin_fmaf(A[v], fH[v], H[v]), A[v] = begins ? 0.f : A[v] * fA[v];
        put_tile<V, WAVES>(p, tile, col, mine, wave == WAVES - 1, A, H, meet, wave);
        const int64_t first = map.first < 0 ? 0 : map.first;
        if (first < t0) {
            join_tiles<V, WAVES>(p, (int)(first / R), tile, col, meet, wave, H);
#pragma unroll
            for (int v = 0; v < V; ++v) fH[v] = cut ? fH[v] : __builtin_fmaf(fA[v], H[v], fH[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) H[v] = fH[v];
    if (p.saved && w0 % 64 == 0 && w0 < p.rows && mine)
#pragma unroll
        for (int v = 0; v < V; ++v) p.saved[w0 / 64 * p.width + col + v] = H[v];
    auto store = [&](int j) {
        if (w0 + j < p.rows && mine) {
            float h[V];
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = w0 + j < end ? H[v] : 0.f;
            Piece<T, V>::put(h, out + (int64_t)j * p.width);
            const int b = p.final_state ? map.ends[wave * ROWS + j] : -1;
            if (b >= 0)
#pragma unroll
                for (int v = 0; v < V; ++v) p.final_state[(int64_t)b * p.width + col + v] = H[v];
        }
    };
    if (begins)
        rows(std::true_type{}, store);
    else
        rows(std::false_type{}, store);
}

// The same from the last row to the first: G is to dh what h is to b, with a row's a on the way to the row in front of it.  h in front of each row is
// worked out again from the state that the forward saved for the tile.  c = a G is what a row passes on.
template <class T, int V, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 4) void hstu_scan_bwd_kernel(const ScanParams p) {
    constexpr int R = ROWS * WAVES, COLS = 64 * V;
    static_assert(R == 64, "the forward saves h in front of every 64th row");
    __shared__ TileRows<R> map;
    __shared__ float2 sums[WAVES][COLS], meet[WAVES][COLS];
    __shared__ float back[WAVES][COLS];
    __shared__ unsigned number;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    map.template clear<64 * WAVES>();
    if (threadIdx.x == 0) number = p.words ? atomicAdd(p.ticket, 1u) : blockIdx.x;
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(number), turned = n / p.col_blocks, tile = p.tiles - 1 - turned;
    const int col0 = (n % p.col_blocks) * COLS + lane * V, col = min(col0, p.width - V);
    const bool mine = col0 < p.width;
    const int64_t t0 = (int64_t)tile * R, w0 = t0 + wave * ROWS, end = rows_end(p), out0 = w0 * p.width + col;
    auto put = [&](char* to, int j, const float (&d)[V]) {
        if (to) Piece<T, V>::put(d, (T*)to + out0 + (int64_t)j * p.width);
    };
    if (t0 >= end) {
        const float zero[V] = {};
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (mine && w0 + j < p.rows) put(p.dx, j, zero), put(p.dr, j, zero), put(p.di, j, zero);
        if (p.partial && wave == 0 && mine)
#pragma unroll
            for (int v = 0; v < V; ++v) p.partial[(int64_t)tile * p.width + col + v] = 0.f;
        return;
    }
    Piece<T, V> x[ROWS], r[ROWS], i[ROWS], d[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t row = min(w0 + j, p.rows - 1);
        x[j].load((const T*)p.x + row * p.x_rs + col);
        r[j].load((const T*)p.r + row * p.r_rs + col);
        i[j].load((const T*)p.i + row * p.i_rs + col);
        d[j].w = 0;
        if (p.dout) d[j].load((const T*)p.dout + row * p.dout_rs + col);
    }
    float strength[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) strength[v] = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col + v)), h[v] = p.saved[(int64_t)tile * p.width + col + v];
    map.template find<64 * WAVES>(p, t0, end);
    Gates<T> g[ROWS][V];
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) g[j][v] = Gates<T>(r[j].get(v), i[j].get(v), strength[v]);
    __syncthreads();
    uint64_t bits[1], end_bits[1];
    marks(map.begins, bits);
    marks(map.ends, end_bits);
    const unsigned begins = marks_of<ROWS>(bits, wave), ends = marks_of<ROWS>(end_bits, wave);
    // Waves whose rows all lie within one sequence have nothing to ask at each.
    const bool plain = !begins && !ends && w0 + ROWS <= end;
    auto either = [&](auto&& pass) {
        if (plain)
            pass(std::true_type{});
        else
            pass(std::false_type{});
    };
    auto before = [&](auto all, int j, int v, float now) {  // h in front of row j
        if (decltype(all)::value || !(begins >> j & 1)) return now;
        return p.initial ? p.initial[(int64_t)map.begins[wave * ROWS + j] * p.width + col + v] : 0.f;
    };
    auto behind = [&](auto all, int j, float now) { return decltype(all)::value || !(ends >> j & 1) ? now : 0.f; };  // c from behind row j
    float A[V], H[V], C[V], G[ROWS][V];  // G: dh as yet
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) G[j][v] = w0 + j < end ? d[j].get(v) : 0.f;
    if (p.dfinal && ends)
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (ends >> j & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) G[j][v] += p.dfinal[(int64_t)map.ends[wave * ROWS + j] * p.width + col + v];
    either([&](auto all) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A[v] = 1.f, H[v] = C[v] = 0.f;
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
                H[v] = __builtin_fmaf(g[j][v].a, before(all, j, v, H[v]), g[j][v].m * g[j][v].si * x[j].get(v));
                A[v] *= g[j][v].a;
            }
#pragma unroll
            for (int j = ROWS - 1; j >= 0; --j) C[v] = g[j][v].a * (G[j][v] + behind(all, j, C[v]));
        }
    });
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane * V + v] = float2{A[v], H[v]}, back[wave][lane * V + v] = C[v];
    __syncthreads();
    // h in front of the wave's rows
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) {
        if (w >= wave) break;
        const bool begun = marks_of<ROWS>(bits, w) != 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 s = sums[w][lane * V + v];
            h[v] = begun ? s.y : __builtin_fmaf(s.x, h[v], s.y);
        }
    }
    // c from the waves behind
    float fA[V], fC[V];
    bool cut = false;
#pragma unroll
    for (int v = 0; v < V; ++v) fA[v] = 1.f, fC[v] = 0.f;
#pragma unroll
    for (int w = WAVES - 1; w > 0; --w) {
        if (w <= wave) break;
        const bool ended = marks_of<ROWS>(end_bits, w) != 0;
        cut = cut || ended;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float by = sums[w][lane * V + v].x, c = back[w][lane * V + v];
            fC[v] = ended ? c : __builtin_fmaf(by, fC[v], c);
            fA[v] = ended ? 0.f : by * fA[v];
        }
    }
    if (p.words) {
#pragma unroll
        for (int v = 0; v < V; ++v) C[v] = ends ? C[v] : __builtin_fmaf(A[v], fC[v], C[v]), A[v] = ends ? 0.f : A[v] * fA[v];
        put_tile<V, WAVES>(p, turned, col, mine, wave == 0, A, C, meet, wave);
        if (map.behind > t0 + R) {
            join_tiles<V, WAVES>(p, p.tiles - 1 - (int)((map.behind - 1) / R), turned, col, meet, wave, C);
#pragma unroll
            for (int v = 0; v < V; ++v) fC[v] = cut ? fC[v] : __builtin_fmaf(fA[v], C[v], fC[v]);
        }
    }
    // G of every row from the last to the first, then the results along with h from the first to the last
    float sum[V] = {};
#pragma unroll
    for (int j = 0; j < ROWS; ++j) asm("" : "+v"(x[j].w));  // products with x are worked out again: kept from above they would take 32 registers that there are not
    either([&](auto all) {
        constexpr bool ALL = decltype(all)::value;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = ROWS - 1; j >= 0; --j) {
                G[j][v] += behind(all, j, fC[v]);
                fC[v] = g[j][v].a * G[j][v];
                if (!ALL && p.dinitial && mine && begins >> j & 1) p.dinitial[(int64_t)map.begins[wave * ROWS + j] * p.width + col + v] = fC[v];
            }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            float dx[V], dr[V], di[V];
            const bool there = ALL || w0 + j < end;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gates<T>& q = g[j][v];
                const float Gm = G[j][v] * q.m, u = q.si * x[j].get(v), old = before(all, j, v, h[v]);
                const float share = q.m > 0.f ? q.s * __builtin_amdgcn_rcpf(q.m) : 0.f;
                const float dq = G[j][v] * q.a * (u * q.a * share - q.s * old);
                dx[v] = there ? Gm * q.si : 0.f;
                dr[v] = there ? strength[v] * (1.f - q.s) * dq : 0.f;
                di[v] = there ? Gm * u * (1.f - q.si) : 0.f;
                sum[v] += there ? dq : 0.f;
                h[v] = __builtin_fmaf(q.a, old, q.m * u);
            }
            if (mine && (ALL || w0 + j < p.rows)) put(p.dx, j, dx), put(p.dr, j, dr), put(p.di, j, di);
        }
    });
    if (!p.partial) return;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) back[wave][lane * V + v] = sum[v];
    __syncthreads();
    if (wave == 0 && mine)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float all = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) all += back[w][lane * V + v];
            p.partial[(int64_t)tile * p.width + col + v] = all;
        }
}

// d decay = rate sigmoid(decay) * the sum of `count` partial sums, in 64 bits: 16 columns to a workgroup, 16 parts of the sums.
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_decay_kernel(const float* partial, int64_t count, int width, const void* decay, int f32, float rate, void* out) {
    __shared__ double meet[16][17];
    const int c = threadIdx.x & 15, part = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    double sum = 0;
    if (col < width) {
        int64_t k = part;
        for (; k + 48 < count; k += 64) {
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = partial[(k + 16 * q) * width + col];
#pragma unroll
            for (int q = 0; q < 4; ++q) sum += v[q];
        }
        for (; k < count; k += 16) sum += partial[k * width + col];
    }
    meet[part][c] = sum;
    __syncthreads();
    if (part || col >= width) return;
#pragma unroll
    for (int q = 1; q < 16; ++q) sum += meet[q][c];
    const double d = decay_at<T>(decay, f32, col), v = rate / (1. + exp(-d)) * sum;
    if (f32)
        ((float*)out)[col] = (float)v;
    else
        ((T*)out)[col] = (T)(float)v;
}

// Few rows to a sequence: a workgroup for each sequence and 64 columns, ROWS * WAVES rows at a time, and no word to wait for.  grid (columns / 64,
// batch + 1): the last y clears the rows behind the sequences.
template <class T, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void hstu_scan_short_kernel(const ScanParams p) {
    constexpr int R = ROWS * WAVES;
    __shared__ float2 sums[2][WAVES][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, b = blockIdx.y, col0 = blockIdx.x * 64 + lane, col = min(col0, p.width - 1);
    const bool mine = col0 < p.width;
    const int64_t last = rows_end(p);
    T* out = (T*)p.out + col;
    if (b == p.batch) {
        for (int64_t t = last + wave; t < p.rows && mine; t += WAVES) out[t * p.width] = (T)0.f;
        return;
    }
    const int64_t first = max(index_at(p.offsets, p.offsets_i64, b), (int64_t)0), end = min(index_at(p.offsets, p.offsets_i64, b + 1), last);
    const float strength = p.rate * softplus_of(decay_at<T>(p.decay, p.decay_f32, col));
    float carry = p.initial ? p.initial[(int64_t)b * p.width + col] : 0.f;
    int turn = 0;
    for (int64_t t0 = first; t0 < end; t0 += R, turn ^= 1) {
        float a[ROWS], in[ROWS], A = 1.f, H = 0.f;
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const int64_t t = t0 + wave * ROWS + j, row = min(t, end - 1);
            const Gates<T> g((float)((const T*)p.r)[row * p.r_rs + col], (float)((const T*)p.i)[row * p.i_rs + col], strength);
            const float x = (float)((const T*)p.x)[row * p.x_rs + col];
            a[j] = t < end ? g.a : 1.f, in[j] = t < end ? g.m * g.si * x : 0.f;  // rows that there are not leave h as it is
            H = __builtin_fmaf(a[j], H, in[j]), A *= a[j];
        }
        sums[turn][wave][lane] = float2{A, H};
        __syncthreads();
        float h = carry;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float2 s = sums[turn][w][lane];
            h = w == wave ? carry : h;
            carry = __builtin_fmaf(s.x, carry, s.y);
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const int64_t t = t0 + wave * ROWS + j;
            h = __builtin_fmaf(a[j], h, in[j]);
            if (t < end && mine) out[t * p.width] = (T)h;
        }
    }
    if (p.final_state && mine && wave == 0) p.final_state[(int64_t)b * p.width + col] = carry;
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
