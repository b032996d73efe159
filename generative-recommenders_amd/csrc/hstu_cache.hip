// C ABI of libhstu_cache.so (include/hstu_cache.h) but for the attention: checks and launches of the row-wise steps.
#include "hstu_cache.h"

#include <atomic>
#include <cstdio>
#include <cstring>

#include "hstu_hip.h"
#include "hstu_cache_host.h"

namespace {

thread_local char g_last_error[256] = "";

int lanes_of(int dim) {
    int lanes = 4;
    while (lanes * 8 < dim) lanes *= 2;
    return lanes;
}

// Rotation: 0, or the status.
int check_turn(int rotary, int interleaved, const float* table, int64_t table_rows, int dim) {
    if (rotary < 0 || rotary > dim || table_rows < 0) return HSTU_ERR_BAD_SHAPE;
    if (rotary == 0) return 0;
    if (rotary % (interleaved ? 8 : 16) != 0) return HSTU_ERR_UNSUPPORTED;
    if (!table) return HSTU_ERR_NULL_POINTER;
    return hstu_cache_aligned(table) ? 0 : HSTU_ERR_MISALIGNED;
}

bool strides_fit(int64_t rs, int64_t hs, int per16) { return rs >= 0 && hs >= 0 && rs % per16 == 0 && hs % per16 == 0; }

// Forward and backward of the step: 0, or the status; `p` without what only one of them needs.
int fill_norm_rope(const HstuNormRopeArgs* a, hstu::NormRopeParams& p) {
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (a->dtype != HSTU_BF16 && a->dtype != HSTU_FP16 && a->dtype != HSTU_FP32) return HSTU_ERR_BAD_DTYPE;
    if (a->rows < 0 || a->dim <= 0 || a->q_heads < 0 || a->k_heads < 0) return HSTU_ERR_BAD_SHAPE;
    if (a->dim % 8 != 0 || a->dim > 512) return HSTU_ERR_BAD_HEAD_DIM;
    const int rc = check_turn(a->rotary, a->interleaved, a->table, a->table_rows, a->dim);
    if (rc) return rc;
    if (a->rotary && a->rows > 0 && !a->positions) return HSTU_ERR_NULL_POINTER;
    const int per16 = a->dtype == HSTU_FP32 ? 4 : 8;
    const void* x[2] = {a->q, a->k};
    const void* weight[2] = {a->q_weight, a->k_weight};
    void* out[2] = {a->q_out, a->k_out};
    const int64_t rs[2] = {a->q_row_stride, a->k_row_stride}, hs[2] = {a->q_head_stride, a->k_head_stride};
    const int heads[2] = {a->q_heads, a->k_heads};
    p = hstu::NormRopeParams{};
    for (int i = 0; i < 2; ++i) {
        hstu::NormRopeSide& s = p.side[i];
        if (!x[i] || heads[i] == 0) continue;
        if (!strides_fit(rs[i], hs[i], per16)) return HSTU_ERR_MISALIGNED;
        if (!hstu_cache_aligned(x[i]) || !hstu_cache_aligned(weight[i]) || !hstu_cache_aligned(out[i])) return HSTU_ERR_MISALIGNED;
        s.x = (const char*)x[i], s.rs = rs[i], s.hs = hs[i], s.y = (char*)out[i], s.weight = (const char*)weight[i], s.heads = heads[i];
    }
    p.positions = a->positions, p.positions_i64 = a->positions_i64;
    p.turn = {a->table, a->table_rows, a->rotary, a->interleaved ? 1 : 0};
    p.eps = a->eps, p.inv_dim = 1.f / a->dim;
    p.rows = a->rows, p.dim = a->dim;
    return 0;
}

// How many of a row's vectors a group of lanes takes: all of them (positions and table rows are then read once) where that leaves
// workgroups enough for the chip, else fewer.
int vectors_per_group(int64_t rows, int lanes, int vectors, int64_t enough) {
    int per = vectors;
    while (per > 1 && (rows * lanes + 255) / 256 * ((vectors + per - 1) / per) < enough) per = (per + 1) / 2;
    return per;
}

int launch_status(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    hstu_cache_set_last_error(what, (int)e);
    return HSTU_ERR_LAUNCH;
}

template <class F>
int with_lanes(int lanes, F&& f) {
    switch (lanes) {
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        case 32: return f(std::integral_constant<int, 32>{});
        default: return f(std::integral_constant<int, 64>{});
    }
}

template <class F>
int with_turn(int rotary, int interleaved, F&& f) {
    if (!rotary) return f(std::integral_constant<int, hstu::TURN_NONE>{});
    return interleaved ? f(std::integral_constant<int, hstu::TURN_PAIRS>{}) : f(std::integral_constant<int, hstu::TURN_HALVES>{});
}

template <class F>
int with_type(int dtype, F&& f) {
    if (dtype == HSTU_BF16) return f((__bf16*)nullptr);
    if (dtype == HSTU_FP16) return f((_Float16*)nullptr);
    return f((float*)nullptr);
}

// Workgroups (x, y) of the backward and what a group takes.
void bwd_grid(const HstuNormRopeArgs* a, int64_t& x, int& y, int& per) {
    const int lanes = lanes_of(a->dim), heads = (a->q ? a->q_heads : 0) + (a->k ? a->k_heads : 0);
    per = vectors_per_group(a->rows, lanes, heads, 1024);
    y = per ? (heads + per - 1) / per : 1;
    x = (a->rows * lanes + 255) / 256;
    const int64_t most = 2048 / y > 0 ? 2048 / y : 1;
    if (x > most) x = most;
    if (x < 1) x = 1;
}

}  // namespace

extern "C" __attribute__((visibility("hidden"))) void hstu_cache_set_last_error(const char* what, int hip_error) {
    snprintf(g_last_error, sizeof(g_last_error), "%s: %s", what, hipGetErrorString((hipError_t)hip_error));
}

extern "C" __attribute__((visibility("hidden"))) int hstu_cache_device_is_gfx950(void) {
    static std::atomic<int> known[64];  // 0 unknown, 1 yes, 2 no; racing threads store the same value
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
    if (known[dev] == 0) {
        hipDeviceProp_t prop;
        if (hipGetDeviceProperties(&prop, dev) != hipSuccess) return 0;
        known[dev] = strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
    }
    return known[dev] == 1;
}

extern "C" __attribute__((visibility("hidden"))) int hstu_cache_fill(const HstuPagedCache* c, hstu::PagedCache& p) {
    if (!c) return HSTU_ERR_NULL_POINTER;
    if (c->dtype != HSTU_BF16 && c->dtype != HSTU_FP16) return HSTU_ERR_BAD_DTYPE;
    if (c->pages < 0 || c->heads <= 0 || c->batch < 0 || c->table_columns < 0 || c->table_row_stride < 0) return HSTU_ERR_BAD_SHAPE;
    for (int dim : {c->dqk, c->dv})
        if (dim != 32 && dim != 64 && dim != 128 && dim != 256) return HSTU_ERR_BAD_HEAD_DIM;
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0) return HSTU_ERR_UNSUPPORTED;
    if (c->pages > 0 && (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales)) return HSTU_ERR_NULL_POINTER;
    if (c->batch > 0 && c->table_columns > 0 && !c->page_table) return HSTU_ERR_NULL_POINTER;
    for (const void* ptr : {c->k_codes, c->k_scales, c->v_codes, c->v_scales})
        if (!hstu_cache_aligned(ptr)) return HSTU_ERR_MISALIGNED;
    p.k_codes = (char*)c->k_codes, p.v_codes = (char*)c->v_codes, p.k_scales = (char*)c->k_scales, p.v_scales = (char*)c->v_scales;
    p.pages = c->pages, p.heads = c->heads, p.dqk = c->dqk, p.dv = c->dv;
    p.page_shift = __builtin_ctz((unsigned)c->page_size);
    p.page_table = c->page_table, p.table_row_stride = c->table_row_stride, p.table_columns = c->table_columns;
    p.page_table_i64 = c->page_table_i64, p.batch = c->batch;
    return 0;
}

extern "C" {

int hstu_cache_version(void) { return 100; }
const char* hstu_cache_last_error(void) { return g_last_error; }

int hstu_cache_norm_rope(const HstuNormRopeArgs* a, void* stream) {
    hstu::NormRopeParams p;
    const int rc = fill_norm_rope(a, p);
    if (rc) return rc;
    const int heads = p.side[0].heads + p.side[1].heads;
    if (a->rows == 0 || heads == 0) return 0;
    for (const hstu::NormRopeSide& s : p.side)
        if (s.heads && !s.y) return HSTU_ERR_NULL_POINTER;
    const int lanes = lanes_of(a->dim);
    p.heads_per_group = vectors_per_group(a->rows, lanes, heads, 2048);
    const int64_t blocks = (a->rows * lanes + 255) / 256, chunks = (heads + p.heads_per_group - 1) / p.heads_per_group;
    if (blocks > kMaxBlocks || chunks > 65535) return HSTU_ERR_UNSUPPORTED;
    if (!hstu_cache_device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    return with_type(a->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        return with_lanes(lanes, [&](auto l) {
            return with_turn(a->rotary, a->interleaved, [&](auto turn) {
                hipLaunchKernelGGL((hstu::hstu_norm_rope_kernel<T, decltype(l)::value, decltype(turn)::value>), dim3((unsigned)blocks, (unsigned)chunks), dim3(256), 0,
                                   (hipStream_t)stream, p);
                return launch_status("norm and rotation kernel launch");
            });
        });
    });
}

size_t hstu_cache_norm_rope_bwd_workspace_bytes(const HstuNormRopeArgs* a) {
    if (!a || a->rows <= 0 || a->dim <= 0 || a->dim > 512 || (!a->q_weight && !a->k_weight)) return 0;
    int64_t x;
    int y, per;
    bwd_grid(a, x, y, per);
    return (size_t)x * y * 2 * a->dim * sizeof(float);
}

int hstu_cache_norm_rope_bwd(const HstuNormRopeArgs* a, const HstuNormRopeGrads* g, void* stream) {
    hstu::NormRopeParams p;
    const int rc = fill_norm_rope(a, p);
    if (rc) return rc;
    if (!g) return HSTU_ERR_NULL_POINTER;
    const int heads = p.side[0].heads + p.side[1].heads, per16 = a->dtype == HSTU_FP32 ? 4 : 8;
    if (a->rows == 0 || heads == 0) return HSTU_ERR_BAD_SHAPE;  // (a weight's gradient would have to be cleared: the caller's to do)
    const void* dy[2] = {g->dq_out, g->dk_out};
    void* dx[2] = {g->dq, g->dk};
    void* dw[2] = {g->dq_weight, g->dk_weight};
    const int64_t rs[2] = {g->dq_out_row_stride, g->dk_out_row_stride}, hs[2] = {g->dq_out_head_stride, g->dk_out_head_stride};
    for (int i = 0; i < 2; ++i) {
        hstu::NormRopeSide& s = p.side[i];
        if (!s.heads) continue;
        if (!dy[i] || !dx[i]) return HSTU_ERR_NULL_POINTER;
        if (!strides_fit(rs[i], hs[i], per16) || !hstu_cache_aligned(dy[i]) || !hstu_cache_aligned(dx[i])) return HSTU_ERR_MISALIGNED;
        s.dy = (const char*)dy[i], s.dy_rs = rs[i], s.dy_hs = hs[i], s.dx = (char*)dx[i];
        s.dw = dw[i] && s.weight ? 1 : 0;
    }
    const bool weights = p.side[0].dw || p.side[1].dw;
    int64_t x;
    int y;
    bwd_grid(a, x, y, p.heads_per_group);
    if (y > 65535) return HSTU_ERR_UNSUPPORTED;
    if (weights) {
        if (!g->workspace) return HSTU_ERR_NULL_POINTER;
        if (!hstu_cache_aligned(g->workspace)) return HSTU_ERR_MISALIGNED;
        if (g->workspace_bytes < (int64_t)hstu_cache_norm_rope_bwd_workspace_bytes(a)) return HSTU_ERR_BAD_SHAPE;
        p.partial = (float*)g->workspace;
    }
    if (!hstu_cache_device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    return with_type(a->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        return with_lanes(lanes_of(a->dim), [&](auto l) {
            const int status = with_turn(a->rotary, a->interleaved, [&](auto turn) {
                hipLaunchKernelGGL((hstu::hstu_norm_rope_bwd_kernel<T, decltype(l)::value, decltype(turn)::value>), dim3((unsigned)x, (unsigned)y), dim3(256), 0,
                                   (hipStream_t)stream, p);
                return launch_status("norm and rotation backward kernel launch");
            });
            if (status) return status;
            if (!weights) return 0;
            hipLaunchKernelGGL((hstu::hstu_norm_rope_dw_kernel<T>), dim3((a->dim + 15) / 16, 2), dim3(256), 0, (hipStream_t)stream, p.partial, x * y, a->dim,
                               p.side[0].dw ? (T*)g->dq_weight : nullptr, p.side[1].dw ? (T*)g->dk_weight : nullptr);
            return launch_status("norm weight gradient kernel launch");
        });
    });
}

int hstu_cache_append(const HstuPagedCache* cache, const HstuAppendArgs* a, void* stream) {
    hstu::AppendParams p{};
    int rc = hstu_cache_fill(cache, p.cache);
    if (rc) return rc;
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (a->rows < 0 || (!a->seq_offsets && (cache->batch ? a->rows % cache->batch : a->rows) != 0)) return HSTU_ERR_BAD_SHAPE;
    rc = check_turn(a->rotary, a->interleaved, a->table, a->table_rows, cache->dqk);
    if (rc) return rc;
    if (a->rows == 0 || cache->batch == 0 || cache->pages == 0) return 0;
    if (!a->k || !a->v || !a->start) return HSTU_ERR_NULL_POINTER;
    if (!strides_fit(a->k_row_stride, a->k_head_stride, 8) || !strides_fit(a->v_row_stride, a->v_head_stride, 8)) return HSTU_ERR_MISALIGNED;
    for (const void* ptr : {a->k, a->v, a->k_weight})
        if (!hstu_cache_aligned(ptr)) return HSTU_ERR_MISALIGNED;
    p.place = {a->start, a->seq_offsets, a->start_i64, a->seq_offsets_i64, a->rows, a->seq_offsets ? 0 : a->rows / cache->batch};
    p.k = (const char*)a->k, p.v = (const char*)a->v;
    p.k_rs = a->k_row_stride, p.k_hs = a->k_head_stride, p.v_rs = a->v_row_stride, p.v_hs = a->v_head_stride;
    p.k_weight = (const char*)a->k_weight, p.eps = a->eps, p.inv_dim = 1.f / cache->dqk;
    p.turn = {a->table, a->table_rows, a->rotary, a->interleaved ? 1 : 0};
    p.positions = a->positions, p.positions_i64 = a->positions_i64;
    const int lanes = lanes_of(cache->dqk > cache->dv ? cache->dqk : cache->dv), vectors = 2 * cache->heads;
    p.vectors_per_group = vectors_per_group(a->rows, lanes, vectors, 2048);
    const int64_t blocks = (a->rows * lanes + 255) / 256, chunks = (vectors + p.vectors_per_group - 1) / p.vectors_per_group;
    if (blocks > kMaxBlocks || chunks > 65535) return HSTU_ERR_UNSUPPORTED;
    if (!hstu_cache_device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    auto launch = [&](auto* t, auto l) {
        typedef std::remove_pointer_t<decltype(t)> T;
        return with_turn(a->rotary, a->interleaved, [&](auto turn) {
            hipLaunchKernelGGL((hstu::hstu_paged_append_kernel<T, decltype(l)::value, decltype(turn)::value>), dim3((unsigned)blocks, (unsigned)chunks), dim3(256), 0,
                               (hipStream_t)stream, p);
            return launch_status("cache append kernel launch");
        });
    };
    return hstu_cache_dispatch(cache->dtype, lanes, launch);
}

int hstu_cache_read(const HstuPagedCache* cache, int64_t rows, const void* start, int32_t start_i64, const void* seq_offsets, int32_t seq_offsets_i64,
                    void* k, void* v, void* stream) {
    hstu::ReadParams p{};
    const int rc = hstu_cache_fill(cache, p.cache);
    if (rc) return rc;
    if (rows < 0 || (!seq_offsets && (cache->batch ? rows % cache->batch : rows) != 0)) return HSTU_ERR_BAD_SHAPE;
    if (rows == 0 || cache->batch == 0) return 0;
    if (!k || !v || !start) return HSTU_ERR_NULL_POINTER;
    if (!hstu_cache_aligned(k) || !hstu_cache_aligned(v)) return HSTU_ERR_MISALIGNED;
    p.place = {start, seq_offsets, start_i64, seq_offsets_i64, rows, seq_offsets ? 0 : rows / cache->batch};
    p.k = (char*)k, p.v = (char*)v;
    const int lanes = lanes_of(cache->dqk > cache->dv ? cache->dqk : cache->dv), vectors = 2 * cache->heads;
    p.vectors_per_group = vectors_per_group(rows, lanes, vectors, 2048);
    const int64_t blocks = (rows * lanes + 255) / 256, chunks = (vectors + p.vectors_per_group - 1) / p.vectors_per_group;
    if (blocks > kMaxBlocks || chunks > 65535) return HSTU_ERR_UNSUPPORTED;
    if (!hstu_cache_device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    auto launch = [&](auto* t, auto l) {
        typedef std::remove_pointer_t<decltype(t)> T;
        hipLaunchKernelGGL((hstu::hstu_paged_read_kernel<T, decltype(l)::value>), dim3((unsigned)blocks, (unsigned)chunks), dim3(256), 0, (hipStream_t)stream, p);
        return launch_status("cache read kernel launch");
    };
    return hstu_cache_dispatch(cache->dtype, lanes, launch);
}

}  // extern "C"
