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

// rate softplus(d) log2(e)
__device__ __forceinline__ float strength_of(float d, float rate) { return rate * (fmaxf(d, 0.f) + log1pf(expf(-fabsf(d)))) * kLog2e; }

// 1 - a = 1 - 2^-z, and a.  1 - a and 1 - a^2 are wanted to their own last places: a is close to one in layers that remember, and what it
// is off by counts once for each of the 1 / (1 - a) rows that h goes back over.  So for small z both come from the series of
// 1 - exp(-z) = z (1 - z/2 + z^2/6 - ...), to z^6 below 1/4 for fp32 tensors and to z^4 below 1/16 for others (off by 1.4e-7 of it at most), and from the
// instruction's exp(-z), good to a unit in the last place, above.  z has the log2(e) in it; the series' terms have powers of log(2) for it.
template <class T>
__device__ __forceinline__ float lost_of(float z, float& a) {
    constexpr float k1 = 0.69314718056f, k2 = -k1 * k1 / 2, k3 = k1 * k1 * k1 / 6, k4 = k2 * k2 / -6, k5 = k3 * k1 * k1 / 20, k6 = k3 * k3 / -20;
    const float far = __builtin_amdgcn_exp2f(-z);
    float series;
    if constexpr (sizeof(T) == 4)
        series = __builtin_fmaf(z, __builtin_fmaf(z, k6, k5), k4);
    else
        series = k4;
    series = z * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, series, k3), k2), k1);
    const bool near = z < (sizeof(T) == 4 ? .25f : .0625f) * kLog2e;
    a = near ? 1.f - series : far;
    return near ? series : 1.f - far;
}

// What a row's gates make of it; `strength` has the log2(e) in it.
template <class T>
struct Gates {
    float a, m, si;
    __device__ __forceinline__ Gates(float r, float i, float strength) {
        si = sigmoid_of(i);
        const float lost = lost_of<T>(strength * sigmoid_of(r), a);
        m = __builtin_amdgcn_sqrtf(lost * (2.f - lost));
    }
};

// The same for the backward, which wants 1 - s and 1 - sigmoid(i) besides, to their own last places too (as differences they are 1 % off at gates of 12 and 0
// from 17.4 on).  With s = 1 / (1 + e), 1 - s is e s; where e is an infinity that is 0 here, as is all that it is a factor of, by s.  In one register with s, the
// smaller of the two with a sign, it takes two more selections (32 long histories 857 us where this takes 852).
template <class T>
struct BackGates {
    float a, in, per, e, shut;  // in: m sigmoid(i); per: s / m^2; e: s = 1 / (1 + e); shut: 1 - sigmoid(i)
    __device__ __forceinline__ BackGates() {}
    __device__ __forceinline__ BackGates(float r, float i, float strength) {
        e = __builtin_amdgcn_exp2f(-kLog2e * r);
        const float ei = __builtin_amdgcn_exp2f(-kLog2e * i), s = __builtin_amdgcn_rcpf(1.f + e), si = __builtin_amdgcn_rcpf(1.f + ei), lost = lost_of<T>(strength * s, a),
                    m2 = lost * (2.f - lost);
        in = __builtin_amdgcn_sqrtf(m2) * si, per = m2 >= 0x1p-126f ? s * __builtin_amdgcn_rcpf(m2) : 0.f;  // (less has no reciprocal)
        shut = fminf(ei, 0x1p126f) * si;
    }
    // s and 1 - s
    __device__ __forceinline__ void halves(float& s, float& rest) const { s = __builtin_amdgcn_rcpf(1.f + e), rest = fminf(e, 0x1p126f) * s; }
};

template <class T>
__device__ __forceinline__ float decay_at(const void* decay, int f32, int col) {
    return f32 ? ((const float*)decay)[col] : (float)((const T*)decay)[col];
}

// Tiles of kTile rows: whole sequences, one or more short ones, make a segment, and a segment's rows are cut into tiles from its first on.
constexpr int kTile = 64;

// A tile: where it is and which of its segment's it is.  The backward counts a segment's tiles from its last.
struct Tile {
    int64_t first;    // row
    int64_t behind;   // the row behind its segment's last
    int segment, at;  // -1: none
    int slot;         // where its segment's places in the lists of words and saved states begin; its own are `at` further
    int in_front;     // how many tiles of its segment lie in front of it (what the forward calls `at`)
};

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
    float* saved;               // [slots][width]: h in front of each tile
    int col_blocks;
    // what the tiles share, in scratch memory
    int segments, per_segment;  // sequences to a segment; rows behind the last sequence are one more
    int slots;
    Tile* tiles;                // [slots], in the order in which they are begun
    float* strength;            // [width]: rate softplus(decay) log2(e)
    unsigned long long *sums, *groups;  // [slots][width], [slots / kGroup + 1][width]
    unsigned* states;           // [slots][width]
    unsigned* tickets;          // one for each block of columns, kTicketPitch apart
    int64_t clear;              // how many pairs of words to clear from `sums` on: all of the four above
    int backward;
    // backward
    const char* dout;
    int64_t dout_rs;
    const float* dfinal;
    char *dx, *dr, *di;
    float* dinitial;
    float* partial;  // [slots][width], or null
};

// The rows of a tensor from one on, through a buffer descriptor: a row's offset is the wave's, a column's the lane's, and the device checks their sum, so that
// what lies behind the last row's end (and what is meant for no column) is read as zero and not written at all.  Rows that there are not are read as whatever
// lies in front of that end where rows are less than a row apart; results, whose rows are not, are written for none.  A wave's sixteen rows at most.
struct RowsFrom {
    __amdgpu_buffer_rsrc_t at;
    unsigned pitch;  // bytes from row to row: at most 2^26, so that sixteen rows end below 2^31
    __device__ __forceinline__ RowsFrom(const char* base, int64_t pitch_, int64_t row, int64_t behind, unsigned bytes) : pitch((unsigned)pitch_) {
        const int64_t rows = behind - row < 16 ? behind - row : 16;
        const uint64_t first = (uint64_t)base + row * pitch_;
        const unsigned size = base && rows > 0 ? (unsigned)(rows - 1) * pitch + bytes : 0;
        at = __builtin_amdgcn_make_buffer_rsrc((void*)first, (short)0, (int)size, 0x00020000);
    }
    template <class T>
    __device__ __forceinline__ T load(int j, unsigned off) const {
        if constexpr (sizeof(T) == 4)
            return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(at, (int)off, (int)(j * pitch), 0));
        else
            return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(at, (int)off, (int)(j * pitch), 0));
    }
    // STREAM: past the caches.  The backward's three results push each other out of them: without it a training step of 48 histories took 3 % more, and 2 % with what
    // reads them next; the forward's one is better left for its reader (prefill of 96 histories and a reader 4 % more so).
    template <class T, bool STREAM = false>
    __device__ __forceinline__ void store(int j, unsigned off, float x) const {
        const T v = (T)x;
        if constexpr (sizeof(T) == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), at, (int)off, (int)(j * pitch), STREAM ? 2 : 0);
        else
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), at, (int)off, (int)(j * pitch), STREAM ? 2 : 0);
    }
};
constexpr unsigned kNowhere = 0x80000000u;  // the offset of a column that there is not, for stores: sizes and rows' offsets are below it

// Rows behind the last sequence, or 0.
__device__ __forceinline__ int64_t rows_end(const ScanParams& p) {
    const int64_t end = index_at(p.offsets, p.offsets_i64, p.batch);
    return end < 0 ? 0 : end > p.rows ? p.rows : end;
}

// The same in all lanes, for the compiler to know.
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)x));
}

// Where sequences begin and end in a tile.
struct TileRows {
    int begins[kTile], ends[kTile];  // the sequence whose first, whose last row it is, or -1
    int low;
    __device__ __forceinline__ void clear() {
        if (threadIdx.x < kTile) begins[threadIdx.x] = ends[threadIdx.x] = -1;
        if (threadIdx.x == 0) low = 0;
    }
    // After a barrier behind clear(); needs one behind it.  The segment's sequences are narrowed down by THREADS at a time and then looked at side by
    // side, from one that begins in front of the tile to those that begin behind it.  Where offsets are not in order every index stays in bounds and every
    // loop ends all the same.
    template <int THREADS>
    __device__ __forceinline__ void find(const ScanParams& p, const Tile& tile) {
        const int64_t t0 = tile.first;
        int lo = min(tile.segment * p.per_segment, p.batch), hi = min(lo + p.per_segment, p.batch);
        const int last = hi;
        while (hi - lo >= THREADS) {
            const int step = (hi - lo + THREADS - 1) / THREADS, at = lo + (int)threadIdx.x * step;
            if (at <= hi && index_at(p.offsets, p.offsets_i64, at) <= t0) atomicMax(&low, at);
            __syncthreads();
            lo = max(lo, low), hi = min(hi, lo + step);
            __syncthreads();
        }
        for (int base = lo; base < last; base += THREADS) {
            const int b = base + threadIdx.x;
            if (b < last) {
                const int64_t v = index_at(p.offsets, p.offsets_i64, b), e = min(index_at(p.offsets, p.offsets_i64, b + 1), tile.behind);
                if (e > v) {
                    if (v >= t0 && v < t0 + kTile) begins[v - t0] = b;
                    if (e > t0 && e <= t0 + kTile) ends[e - 1 - t0] = b;
                }
            }
            if (base + THREADS < last && index_at(p.offsets, p.offsets_i64, base + THREADS) >= t0 + kTile) break;  // (the same for all)
        }
    }
};

// Bit k: whether rows[k] is a sequence's; the same in all lanes.
__device__ __forceinline__ uint64_t marks(const int (&rows)[kTile]) { return __ballot(rows[threadIdx.x & 63] >= 0); }
template <int ROWS>
__device__ __forceinline__ unsigned marks_of(uint64_t bits, int wave) {
    return (unsigned)(bits >> (wave * ROWS)) & ((1u << ROWS) - 1);
}

// ---- tiles joined along the rows ----
//
// What a tile makes of the h in front of it is A h + H, or H alone where a sequence begins in it (it is cut off).  Each tile puts its (A, H) down as
// one word for each column, its sum, and the h behind it, its state, as another once it knows it: state = A (state in front) + H.  A tile that finds no
// state in front of it yet takes up sums back to one.  A word is written and read as a whole and is never 0 once written, so it needs no flag and no
// fence beside it.
//
// Tiles are begun in the order of p.tiles, all segments' first ones in front of their second ones (64 segments at a time), by tickets that a
// workgroup takes when it runs: those in front have been begun and wait for none behind them, so each wait ends.  (The limit on it only keeps a broken
// device from hanging.)  With many segments the tile in front has nearly always been done; a single long one has hundreds of its tiles under way at
// once, and for those every kGroup-th joins the sums of its kGroup into one, and its state is defined by that: A_group (state in front of the
// group) + H_group.  So every state has one definition, and results do not depend on which tile was first.
//
// What was measured, each against the rest of the kernel as it was then: what the whole call took more.  Tiles of rows regardless of sequences, each taking up all
// sums of its sequence in front of it: a third of the time went into waits (five histories of up to 16000 rows, 1024 columns).  A pass for the sums and another
// for the rows reads everything twice.  Two columns to a lane forward: 8 % (a training step of 48 histories, 512 columns) and 11 % (the five histories).  Eight
// rows to a lane forward: 5 and 24 % more than sixteen, thirty-two 3 and 8 %; backward eight 6 % (the training step).  With all workgroups at one ticket counter,
// 3400 more of them of half the rows took 61 us more (18 ns each) and without tickets nothing more, so a block of columns has a counter of its own.
constexpr int kGroup = 16, kGroupsBack = 8, kTicketPitch = 64;
constexpr unsigned kCut = 0x7f800000u;  // A's bits where there is none

__device__ __forceinline__ void put_sum(unsigned long long* at, float A, bool cut, float H) {
    const unsigned long long w = (unsigned long long)__float_as_uint(H) << 32 | ((cut ? kCut : __float_as_uint(A)) | 0x80000000u);  // (A is not negative)
    __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_state(unsigned* at, float h) {
    const unsigned w = __float_as_uint(h);
    __hip_atomic_store(at, w ? w : 0x80000000u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // (zero as the other zero)
}
template <class W>
__device__ __forceinline__ W get_word(const W* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float sum_h(unsigned long long w) { return __uint_as_float((unsigned)(w >> 32)); }
__device__ __forceinline__ float sum_a(unsigned long long w) { return __uint_as_float((unsigned)w & 0x7fffffffu); }
__device__ __forceinline__ bool is_cut(unsigned long long w) { return ((unsigned)w & 0x7fffffffu) == kCut; }
// h behind what `w` says, from h in front of it.
__device__ __forceinline__ float apply(unsigned long long w, float h) { return is_cut(w) ? sum_h(w) : __builtin_fmaf(sum_a(w), h, sum_h(w)); }

// All lanes' words, when they are there; `never` if they never are.
template <class W>
__device__ __forceinline__ W await(const W* at, W w, W never) {
    for (int tries = 0; tries < (1 << 20); ++tries) {
        if (__all(w != 0)) return w;
        __builtin_amdgcn_s_sleep(1);
        w = get_word(at);
    }
    return never;
}
constexpr unsigned kNoState = 0x7fc00000u;
constexpr unsigned long long kNoSum = (unsigned long long)kNoState << 32 | 0x80000000u | kCut;

// What the waves of a workgroup share while they go back.
template <int WAVES>
struct Back {
    unsigned long long sums[kGroup + kGroupsBack][64];
    float states[2 * WAVES][64];
    int found[2 * WAVES];  // 0 no, 1 cut off, 2 a state
};

// Goes back over `count` sums, two to a wave at a time: sum(i) is that of the i-th from here (from 1 on), state(i) the state in front of it
// (in front of here for 0; NULL: there is none).  True: h is a state, or not needed, and the `n` sums from here to it, in back.sums[row + i - 1], go on from it.
// `all`: takes every sum, and looks for no state.  Every thread of the workgroup calls.
template <int WAVES, class SUM, class STATE>
__device__ __forceinline__ bool go_back(int count, bool all, int row, SUM&& sum, STATE&& state, Back<WAVES>& back, int wave, int& n, float& h) {
    const int lane = threadIdx.x & 63;
    for (int from = 0; from <= count; from += 2 * WAVES) {
        unsigned long long s[2];
        unsigned t[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int i = min(from + 2 * wave + q, count);
            const unsigned* front = all ? nullptr : state(i);
            s[q] = i ? get_word(sum(i)) : 1, t[q] = front ? get_word(front) : 0;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int i = from + 2 * wave + q;
            if (i > count) continue;  // (the same for the wave)
            if (i) back.sums[row + i - 1][lane] = s[q] = await(sum(i), s[q], kNoSum);
            back.states[2 * wave + q][lane] = __uint_as_float(t[q]);
            const int found = __all(t[q] != 0) ? 2 : __all(i && is_cut(s[q])) ? 1 : 0;
            if (lane == 0) back.found[2 * wave + q] = found;
        }
        __syncthreads();
        for (int k = 0; k < 2 * WAVES && from + k <= count && !all; ++k) {
            const int found = back.found[k];  // (the same for all)
            if (!found) continue;
            n = from + k, h = found == 2 ? back.states[k][lane] : 0.f;
            return true;
        }
        __syncthreads();
    }
    n = count;
    return false;
}

// h in front of tile `at` of a segment whose words begin at `slot`; and where the tile is the last of a group and not cut off (`closes`), what the tiles in
// front of it in its group make of h, (A, H) or H alone (`off`), and in `base` the h in front of the group.  Every thread of the workgroup calls.
template <int WAVES>
__device__ __forceinline__ float look_back(const ScanParams& p, int slot, int at, int col, bool closes, Back<WAVES>& back, int wave, float& A, float& H, bool& off,
                                           float& base) {
    const int lane = threadIdx.x & 63, group = at / kGroup;
    const int64_t width = p.width;
    auto sum_of = [&](int i) { return p.sums + (slot + at - i) * width + col; };
    auto state_of = [&](int tile) { return tile < 0 ? nullptr : p.states + (slot + tile) * width + col; };
    int n;
    float h;
    bool known = go_back<WAVES>(at % kGroup, closes, 0, sum_of, [&](int i) { return state_of(at - i - 1); }, back, wave, n, h);
    off = false;
    if (closes) {
        A = 1.f, H = h = 0.f;
        for (int k = n - 1; k >= 0; --k) {
            const unsigned long long w = back.sums[k][lane];
            off = off || is_cut(w), H = apply(w, H), A *= sum_a(w);  // (cut off in all columns or none)
        }
        known = off;
    }
    if (!known) {  // the state behind the group in front (there is one: a segment's first tile is cut off)
        // (a segment's groups end kGroup slots from each other, and no nearer to those of the segments beside it)
        auto group_of = [&](int i) { return p.groups + (slot + (group - i) * kGroup + kGroup - 1) / kGroup * width + col; };
        const int count = min(group, kGroupsBack);
        int m;
        if (!go_back<WAVES>(count, false, kGroup, group_of, [&](int i) { return state_of((group - i) * kGroup - 1); }, back, wave, m, h)) {
            const unsigned* far = state_of((group - count) * kGroup - 1);
            h = __uint_as_float(await(far, get_word(far), kNoState));
        }
        for (int k = m - 1; k >= 0; --k) h = apply(back.sums[kGroup + k][lane], h);
    }
    base = h;
    for (int k = n - 1; k >= 0; --k) h = apply(back.sums[k][lane], h);
    return h;
}

// What a tile has to do with the others.  `me`: the wave that has its (A, H), which it puts down.  Returns the h in front of the tile, where it
// `needs` it.  Every thread of the workgroup calls.
template <int WAVES>
__device__ __forceinline__ float join_tile(const ScanParams& p, int slot, int at, int col, bool mine, bool me, bool cut, bool needs, float A, float H,
                                           Back<WAVES>& back, int wave) {
    const bool closes = at % kGroup == kGroup - 1;
    const int64_t word = (int64_t)(slot + at) * p.width + col;
    unsigned long long* group = p.groups + (int64_t)((slot + at) / kGroup) * p.width + col;
    if (me && mine) {
        put_sum(p.sums + word, A, cut, H);
        if (cut) put_state(p.states + word, H);
        if (cut && closes) put_sum(group, 0.f, true, H);
    }
    if (!needs) return 0.f;  // (needs, where it is not cut off)
    float by, from, base;
    bool off;
    const float front = look_back<WAVES>(p, slot, at, col, closes && !cut, back, wave, by, from, off, base);
    if (!me || !mine || cut) return front;
    float state = __builtin_fmaf(A, front, H);
    if (closes) {
        by *= A, from = __builtin_fmaf(A, from, H);
        put_sum(group, by, off, from);
        state = off ? from : __builtin_fmaf(by, base, from);
    }
    put_state(p.states + word, state);
    return front;
}

// Which block of columns a workgroup takes: each as often as there are tiles, and each of the eight dies, which workgroups go to in turn, all of them
// in turn (a training step of 32 long histories, 1024 columns, took 15 % more with one die always at the same part of a row).
__device__ __forceinline__ int column_block(const ScanParams& p) { return (int)((blockIdx.x + blockIdx.x / p.col_blocks) % p.col_blocks); }

// The tile that a workgroup takes up, to LDS: one thread's work, with a barrier behind it.
__device__ __forceinline__ void take_tile(const ScanParams& p, int block, Tile& tile) { tile = p.tiles[atomicAdd(p.tickets + block * kTicketPitch, 1u)]; }

// The list of 64 segments' tiles, by workgroups that share its entries out.  Segment s has the rows from F(s) up to F(s + 1): F(0) is 0, F(s) where its
// first sequence begins, or where any in front of it does if offsets are not in order; its slots begin at F(s) / kTile + s, so that nobody has to count
// the tiles in front.  Tile k of segment s comes behind all with a lower k and those of the segments in front with the same: its place is the sum of
// min(tiles, k + 1) over the segments in front and of min(tiles, k) over the others.
struct PlanPart {
    int tiles[64], before[64], slot[64];  // before: tiles of the segments in front
    int64_t first[64], behind[64];
};
__device__ __forceinline__ void plan_tiles(const ScanParams& p, int batch, int part, int parts, PlanPart& plan) {
    const int lane = threadIdx.x & 63, s0 = 64 * batch, s = s0 + lane;
    auto bound = [&](int64_t segment) {
        if (segment > p.segments) return p.rows;
        if (segment == 0) return (int64_t)0;
        const int64_t at = index_at(p.offsets, p.offsets_i64, min(segment * p.per_segment, (int64_t)p.batch));
        return at < 0 ? (int64_t)0 : at > p.rows ? p.rows : at;
    };
    if (threadIdx.x < 64) {
        int64_t first = bound(s), behind = bound(s0 + 64), top = 0;
#pragma unroll 4
        for (int k = lane; k < s0; k += 64) top = max(top, bound(k));
        if (s0)
            for (int d = 32; d; d >>= 1) top = max(top, (int64_t)__shfl_xor((long long)top, d, 64));
        first = max(first, top);
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t other = __shfl_up((long long)first, d, 64);
            if (lane >= d) first = max(first, other);
        }
        const int64_t next = __shfl_down((long long)first, 1, 64);
        behind = lane == 63 ? max(first, behind) : next;
        const int tiles = s <= p.segments ? (int)((behind - first + kTile - 1) / kTile) : 0;
        int upto = tiles;
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(upto, d, 64);
            if (lane >= d) upto += other;
        }
        plan.tiles[lane] = tiles, plan.before[lane] = upto - tiles, plan.slot[lane] = (int)(first / kTile) + s;
        plan.first[lane] = first, plan.behind[lane] = behind;
    }
    __syncthreads();
    const int base = plan.slot[0], total = plan.before[63] + plan.tiles[63];
    const int end = s0 + 64 <= p.segments ? (int)(plan.behind[63] / kTile) + s0 + 64 : p.slots;
    for (int e = part * 256 + (int)threadIdx.x; e < end - base; e += parts * 256) {
        Tile t{};
        int at = e;
        t.at = -1;  // a slot without a tile
        if (e < total) {
            int of = 0;  // the last segment with before <= e that has tiles: e is one of its
            for (int d = 32; d; d >>= 1)
                if (plan.before[of + d] <= e) of += d;
            const int k = e - plan.before[of];
            at = 0;
            for (int q = 0; q < 64; ++q) at += min(plan.tiles[q], k + (q < of ? 1 : 0));
            t.segment = s0 + of, t.at = k, t.slot = plan.slot[of], t.in_front = p.backward ? plan.tiles[of] - 1 - k : k;
            t.first = plan.first[of] + (int64_t)kTile * t.in_front, t.behind = plan.behind[of];
        }
        p.tiles[base + at] = t;
    }
}

// What the tiles find: their list, no words yet, columns' strengths, and the states of sequences without rows as they were.
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_begin_kernel(const ScanParams p) {
    __shared__ PlanPart plan;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    typedef __attribute__((ext_vector_type(4))) unsigned u4;
    for (int64_t k = at; k < p.clear; k += step) ((u4*)p.sums)[k] = u4{0, 0, 0, 0};
    for (int64_t k = at; k < p.width; k += step) p.strength[k] = strength_of(decay_at<T>(p.decay, p.decay_f32, k), p.rate);
    if (p.partial)  // (there are slots without a tile)
        for (int64_t k = at; k < (int64_t)p.slots * p.width; k += step) p.partial[k] = 0.f;
    if (p.final_state)
        for (int64_t k = at; k < (int64_t)p.batch * p.width; k += step) p.final_state[k] = p.initial ? p.initial[k] : 0.f;
    const int batches = p.segments / 64 + 1, parts = min(max((int)gridDim.x / batches, 1), 16);
    for (int q = blockIdx.x; q < batches * parts; q += gridDim.x) {
        if (q != (int)blockIdx.x) __syncthreads();
        plan_tiles(p, q % batches, q / batches, parts, plan);
    }
}

// A workgroup takes a tile of 64 columns, a lane one of them, ROWS rows to a wave.  Bytes and waits bound it: see above.
template <class T, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 6) void hstu_scan_kernel(const ScanParams p) {
    static_assert(ROWS * WAVES == kTile && ROWS <= 16, "a row for each");
    __shared__ TileRows map;
    __shared__ float2 sums[WAVES][64];
    __shared__ Back<WAVES> back;
    __shared__ Tile taken;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, block = column_block(p);
    map.clear();
    if (threadIdx.x == 0) take_tile(p, block, taken);
    __syncthreads();
    const int at = __builtin_amdgcn_readfirstlane(taken.at), slot = __builtin_amdgcn_readfirstlane(taken.slot);
    if (at < 0) return;
    const int64_t behind = uniform(taken.behind), w0 = uniform(taken.first) + wave * ROWS;
    const int col = min(block * 64 + lane, p.width - 1);  // (a lane without a column goes along with the last)
    const bool mine = block * 64 + lane < p.width;
    const unsigned bytes = p.width * (unsigned)sizeof(T), off = col * (unsigned)sizeof(T), off_out = mine ? off : kNowhere;
    const RowsFrom out(p.out, bytes, w0, behind, bytes);
    if (__builtin_amdgcn_readfirstlane(taken.segment) == p.segments) {  // rows behind the last sequence
#pragma unroll
        for (int j = 0; j < ROWS; ++j) out.store<T>(j, off_out, 0.f);
        return;
    }
    T x[ROWS], r[ROWS], i[ROWS];
    const RowsFrom x_rows(p.x, p.x_rs * sizeof(T), w0, behind, bytes), r_rows(p.r, p.r_rs * sizeof(T), w0, behind, bytes),
        i_rows(p.i, p.i_rs * sizeof(T), w0, behind, bytes);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) r[j] = r_rows.load<T>(j, off), i[j] = i_rows.load<T>(j, off), x[j] = x_rows.load<T>(j, off);
    const float strength = p.strength[col];
    map.template find<64 * WAVES>(p, taken);
    float a[ROWS], b[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const Gates<T> g((float)r[j], (float)i[j], strength);
        a[j] = g.a, b[j] = g.m * g.si * (float)x[j];
    }
    __syncthreads();
    const uint64_t bits = marks(map.begins);
    const unsigned begins = marks_of<ROWS>(bits, wave), ends = marks_of<ROWS>(marks(map.ends), wave);
    if (begins && p.initial)
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (begins >> j & 1) b[j] = __builtin_fmaf(a[j], p.initial[(int64_t)map.begins[wave * ROWS + j] * p.width + col], b[j]);
    // Row by row; a row that begins a sequence knows nothing of what is in front of it, whatever that is.
    float A = 1.f, H = 0.f;
    auto rows = [&](auto any, auto&& each) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            if (decltype(any)::value && begins >> j & 1)
                H = b[j];
            else
                H = __builtin_fmaf(a[j], H, b[j]), A *= a[j];
            each(j);
        }
    };
    auto nothing = [](int) {};
    if (begins)
        rows(std::true_type{}, nothing);
    else
        rows(std::false_type{}, nothing);
    sums[wave][lane] = float2{A, H};
    __syncthreads();
    float fA = 1.f, fH = 0.f;  // of the waves in front
    bool cut = false;          // whether a sequence begins in one of them
#pragma unroll 1  // (all parts at once would take the registers of the rows)
    for (int w = 0; w < wave; ++w) {
        const bool begun = marks_of<ROWS>(bits, w) != 0;
        const float2 s = sums[w][lane];
        cut = cut || begun;
        fH = begun ? s.y : __builtin_fmaf(s.x, fH, s.y), fA *= s.x;
    }
    const bool needs = at > 0 && !(bits & 1);
    const float front = join_tile<WAVES>(p, slot, at, col, mine, wave == WAVES - 1, at == 0 || bits, needs, A * fA, begins ? H : __builtin_fmaf(A, fH, H), back, wave);
    if (p.saved && wave == 0 && mine) p.saved[(int64_t)(slot + at) * p.width + col] = front;
    H = needs && !cut ? __builtin_fmaf(fA, front, fH) : fH;
    if (!begins && !(ends && p.final_state)) {
        rows(std::false_type{}, [&](int j) { out.store<T>(j, off_out, H); });
        return;
    }
    rows(std::true_type{}, [&](int j) {
        out.store<T>(j, off_out, H);
        if (p.final_state && mine && ends >> j & 1) p.final_state[(int64_t)map.ends[wave * ROWS + j] * p.width + col] = H;
    });
}

// The same from the last row to the first: G is to dh what h is to b, with a row's a on the way to the row in front of it.  h in front of each row is
// worked out again from the state that the forward saved for the tile.  c = a G is what a row passes on.  Three waves of a SIMD, whose registers hold a row's gates
// from the first pass to the last: with four 14 registers were kept in memory (a training step of 48 histories took 9 % more).
template <class T, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 3) void hstu_scan_bwd_kernel(const ScanParams p) {
    static_assert(ROWS * WAVES == kTile && ROWS <= 16, "a row for each");
    __shared__ TileRows map;
    __shared__ float2 sums[WAVES][64];
    __shared__ float passed[WAVES][64];
    __shared__ Back<WAVES> back;
    __shared__ Tile taken;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, block = column_block(p);
    map.clear();
    if (threadIdx.x == 0) take_tile(p, block, taken);
    __syncthreads();
    const int turned = __builtin_amdgcn_readfirstlane(taken.at), slot = __builtin_amdgcn_readfirstlane(taken.slot);
    if (turned < 0) return;
    const int64_t behind = uniform(taken.behind), w0 = uniform(taken.first) + wave * ROWS;
    const int64_t same = slot + __builtin_amdgcn_readfirstlane(taken.in_front);  // the slot that the forward had for this tile
    const int col = min(block * 64 + lane, p.width - 1);
    const bool mine = block * 64 + lane < p.width;
    const unsigned bytes = p.width * (unsigned)sizeof(T), off = col * (unsigned)sizeof(T), off_out = mine ? off : kNowhere;
    const RowsFrom dx(p.dx, bytes, w0, behind, bytes), dr(p.dr, bytes, w0, behind, bytes), di(p.di, bytes, w0, behind, bytes);  // (none: nothing is written)
    if (__builtin_amdgcn_readfirstlane(taken.segment) == p.segments) {  // rows behind the last sequence
#pragma unroll
        for (int j = 0; j < ROWS; ++j) dx.store<T>(j, off_out, 0.f), dr.store<T>(j, off_out, 0.f), di.store<T>(j, off_out, 0.f);
        return;
    }
    T x[ROWS], r[ROWS], i[ROWS], d[ROWS];
    const RowsFrom x_rows(p.x, p.x_rs * sizeof(T), w0, behind, bytes), r_rows(p.r, p.r_rs * sizeof(T), w0, behind, bytes),
        i_rows(p.i, p.i_rs * sizeof(T), w0, behind, bytes), d_rows(p.dout, p.dout_rs * sizeof(T), w0, behind, bytes);  // (no dout: zeros)
#pragma unroll
    for (int j = 0; j < ROWS; ++j) r[j] = r_rows.load<T>(j, off), i[j] = i_rows.load<T>(j, off), x[j] = x_rows.load<T>(j, off), d[j] = d_rows.load<T>(j, off);
    const float strength = p.strength[col], natural = strength * (1 / kLog2e);
    float h = p.saved[same * p.width + col];
    map.template find<64 * WAVES>(p, taken);
    BackGates<T> g[ROWS];
    float b[ROWS];  // what a row adds to h
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {  // (the compiler kept from working these out side by side or twice, which takes registers that there are not)
        g[j] = BackGates<T>((float)r[j], (float)i[j], strength);
        b[j] = g[j].in * (float)x[j];
        asm("" : "+v"(g[j].in), "+v"(g[j].e), "+v"(g[j].per), "+v"(g[j].shut), "+v"(g[j].a), "+v"(b[j]));
    }
    __syncthreads();
    const uint64_t bits = marks(map.begins), end_bits = marks(map.ends);
    const unsigned begins = marks_of<ROWS>(bits, wave), ends = marks_of<ROWS>(end_bits, wave);
    // Waves whose rows all lie within one sequence have nothing to ask at each.
    const bool plain = !begins && !ends;
    auto either = [&](auto&& pass) {
        if (plain)
            pass(std::true_type{});
        else
            pass(std::false_type{});
    };
    auto before = [&](auto all, int j, float now) {  // h in front of row j
        if (decltype(all)::value || !(begins >> j & 1)) return now;
        return p.initial ? p.initial[(int64_t)map.begins[wave * ROWS + j] * p.width + col] : 0.f;
    };
    auto from_behind = [&](auto all, int j, float now) { return decltype(all)::value || !(ends >> j & 1) ? now : 0.f; };  // c
    float A = 1.f, H = 0.f, C = 0.f, G[ROWS];  // G: dh as yet
#pragma unroll
    for (int j = 0; j < ROWS; ++j) G[j] = (float)d[j];
    if (p.dfinal && ends)
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (ends >> j & 1) G[j] += p.dfinal[(int64_t)map.ends[wave * ROWS + j] * p.width + col];
    either([&](auto all) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            H = __builtin_fmaf(g[j].a, before(all, j, H), b[j]);
            A *= g[j].a;
        }
#pragma unroll
        for (int j = ROWS - 1; j >= 0; --j) C = g[j].a * (G[j] + from_behind(all, j, C));
    });
    sums[wave][lane] = float2{A, H}, passed[wave][lane] = C;
    __syncthreads();
    // h in front of the wave's rows
#pragma unroll 1  // (all parts at once would take the registers of the rows)
    for (int w = 0; w < wave; ++w) {
        const float2 s = sums[w][lane];
        h = marks_of<ROWS>(bits, w) ? s.y : __builtin_fmaf(s.x, h, s.y);
    }
    // c from the waves behind
    float fA = 1.f, fC = 0.f;
    bool cut = false;
#pragma unroll 1
    for (int w = WAVES - 1; w > wave; --w) {
        const bool ended = marks_of<ROWS>(end_bits, w) != 0;
        const float by = sums[w][lane].x, c = passed[w][lane];
        cut = cut || ended;
        fC = ended ? c : __builtin_fmaf(by, fC, c), fA *= by;
    }
    const bool needs = turned > 0 && !(end_bits >> (kTile - 1));
    const float front = join_tile<WAVES>(p, slot, turned, col, mine, wave == 0, turned == 0 || end_bits, needs, A * fA, ends ? C : __builtin_fmaf(A, fC, C), back, wave);
    if (needs && !cut) fC = __builtin_fmaf(fA, front, fC);
    // G of every row from the last to the first, then the results along with h from the first to the last
    float sum = 0.f;
    either([&](auto all) {
        constexpr bool ALL = decltype(all)::value;
#pragma unroll
        for (int j = ROWS - 1; j >= 0; --j) {
            G[j] += from_behind(all, j, fC);
            fC = g[j].a * G[j];
            if (!ALL && p.dinitial && mine && begins >> j & 1) p.dinitial[(int64_t)map.begins[wave * ROWS + j] * p.width + col] = fC;
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const BackGates<T>& q = g[j];
            float open, rest;
            q.halves(open, rest);
            const float old = before(all, j, h), dxj = G[j] * q.in, dq = G[j] * q.a * (b[j] * q.a * q.per - open * old);
            // Rows that there are not may have come from rows that there are, where those lie less than a row apart (one row, rows that were broadcast).  A wave has
            // some beside its segment's last row, or has none that there is and is left out below.
            sum += ALL || w0 + j < behind ? dq : 0.f;
            h = __builtin_fmaf(q.a, old, b[j]);
            dx.store<T, true>(j, off_out, dxj);
            dr.store<T, true>(j, off_out, natural * rest * dq);
            di.store<T, true>(j, off_out, G[j] * b[j] * q.shut);
        }
    });
    if (!p.partial) return;
    __syncthreads();
    passed[wave][lane] = w0 < behind ? sum : 0.f;  // (h behind the last row may be no number)
    __syncthreads();
    if (wave || !mine) return;
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += passed[w][lane];
    p.partial[same * p.width + col] = total;
}

// d decay = rate sigmoid(decay) * the sum of `count` partial sums, in 64 bits: 16 columns to a workgroup, 64 parts of the sums, eight of them in flight.
template <class T>
__global__ __launch_bounds__(1024) void hstu_scan_decay_kernel(const float* partial, int64_t count, int width, const void* decay, int f32, float rate, void* out) {
    __shared__ double meet[64][17];
    const int c = threadIdx.x & 15, part = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    double sum = 0;
    if (col < width) {
        int64_t k = part;
        for (; k + 448 < count; k += 512) {
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = partial[(k + 64 * q) * width + col];
#pragma unroll
            for (int q = 0; q < 8; ++q) sum += v[q];
        }
        for (; k < count; k += 64) sum += partial[k * width + col];
    }
    meet[part][c] = sum;
    __syncthreads();
    if (part >= 4) return;
    sum = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) sum += meet[part + 4 * q][c];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (part || col >= width) return;
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
    const float strength = strength_of(decay_at<T>(p.decay, p.decay_f32, col), p.rate);
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

// grid (rows / 16, columns / 64): a wave takes 64 columns of four rows, all of whose loads go out together; the columns' strengths, 70 operations
// each, are worked out once for them (2000 rows of 1024 columns, a row to a thread: 10.8 us; so: 8.7).
constexpr int kStepRows = 4;
template <class T>
__global__ __launch_bounds__(256) void hstu_scan_step_kernel(const StepParams p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = min((int)blockIdx.y * 64 + lane, p.width - 1);
    const bool mine = (int)blockIdx.y * 64 + lane < p.width;
    const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * kStepRows;
    if (first >= p.rows) return;
    T x[kStepRows], r[kStepRows], i[kStepRows];
    float h[kStepRows];
    int64_t to[kStepRows];
    bool known[kStepRows];
#pragma unroll
    for (int j = 0; j < kStepRows; ++j) {
        const int64_t t = min(first + j, p.rows - 1), from = p.slots ? index_at(p.slots, p.slots_i64, t) : t;
        to[j] = p.new_slots ? index_at(p.new_slots, p.new_slots_i64, t) : from;
        known[j] = from >= -1 && from < p.state_rows;
        h[j] = 0.f;
        if (from >= 0 && known[j]) h[j] = p.states[from * p.state_rs + col];
        x[j] = ((const T*)p.x)[t * p.x_rs + col], r[j] = ((const T*)p.r)[t * p.r_rs + col], i[j] = ((const T*)p.i)[t * p.i_rs + col];
    }
    const float strength = strength_of(decay_at<T>(p.decay, p.decay_f32, col), p.rate);
#pragma unroll
    for (int j = 0; j < kStepRows; ++j) {
        if (first + j >= p.rows || !mine) continue;
        const Gates<T> g((float)r[j], (float)i[j], strength);
        const float now = known[j] ? __builtin_fmaf(g.a, h[j], g.m * g.si * (float)x[j]) : __builtin_nanf("");
        ((T*)p.out)[(first + j) * p.width + col] = (T)now;
        if (known[j] && to[j] >= 0 && to[j] < p.state_rows) p.states[to[j] * p.state_rs + col] = now;
    }
}

}  // namespace hstu
