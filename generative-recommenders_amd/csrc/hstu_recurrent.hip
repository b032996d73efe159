// C ABI of libhstu_recurrent.so (include/hstu_recurrent.h): checks and launches.
#include "hstu_recurrent.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "hstu_hip.h"
#include "hstu_recurrence_kernel.h"
#include "hstu_residual_norm_kernel.h"

namespace {

thread_local char g_last_error[256] = "";

int launch_status(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    snprintf(g_last_error, sizeof(g_last_error), "%s: %s", what, hipGetErrorString(e));
    return HSTU_ERR_LAUNCH;
}

bool device_is_gfx950() {
    static std::atomic<int> known[64];  // 0 unknown, 1 yes, 2 no; racing threads store the same value
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
    if (known[dev] == 0) {
        hipDeviceProp_t prop;
        if (hipGetDeviceProperties(&prop, dev) != hipSuccess) return false;
        known[dev] = strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
    }
    return known[dev] == 1;
}

template <class F>
int with_type(int dtype, F&& f) {
    if (dtype == HSTU_BF16) return f((__bf16*)nullptr);
    if (dtype == HSTU_FP16) return f((_Float16*)nullptr);
    return f((float*)nullptr);
}

bool known_type(int dtype) { return dtype == HSTU_BF16 || dtype == HSTU_FP16 || dtype == HSTU_FP32; }
int bytes_of(int dtype) { return dtype == HSTU_FP32 ? 4 : 2; }
bool aligned_to(const void* ptr, int bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }

constexpr int64_t kMaxPitch = 1 << 24;  // elements from row to row in the recurrence: a wave's sixteen rows are addressed in 31 bits
constexpr int64_t kMaxBlocks = (1 << 24) - 1;  // a launch has fewer than 2^32 threads in a dimension, and these workgroups 256

// ---- the recurrence ----

// 0, or the status.  What only one direction needs is its own to check.
int check_scan(const HstuRecurrenceArgs* a) {
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (!known_type(a->dtype)) return HSTU_ERR_BAD_DTYPE;
    if (a->rows < 0 || a->width <= 0 || a->width > 65535 * 64 || a->batch <= 0 || a->batch > (1 << 30) || !(a->rate > 0.f && std::isfinite(a->rate))) return HSTU_ERR_BAD_SHAPE;
    for (int64_t rs : {a->x_row_stride, a->decay_gate_row_stride, a->input_gate_row_stride}) {
        if (rs < 0) return HSTU_ERR_BAD_SHAPE;
        if (rs > kMaxPitch) return HSTU_ERR_UNSUPPORTED;
    }
    if (!a->seq_offsets || !a->decay) return HSTU_ERR_NULL_POINTER;
    if (a->rows > 0 && (!a->x || !a->decay_gate || !a->input_gate)) return HSTU_ERR_NULL_POINTER;
    const int es = bytes_of(a->dtype);
    if (!aligned_to(a->x, es) || !aligned_to(a->decay_gate, es) || !aligned_to(a->input_gate, es) || !aligned_to(a->out, es)) return HSTU_ERR_MISALIGNED;
    if (!aligned_to(a->decay, a->decay_f32 ? 4 : es) || !aligned_to(a->initial_state, 4) || !aligned_to(a->final_state, 4) || !aligned_to(a->saved, 4))
        return HSTU_ERR_MISALIGNED;
    if (!aligned_to(a->seq_offsets, a->seq_offsets_i64 ? 8 : 4)) return HSTU_ERR_MISALIGNED;
    return 0;
}

hstu::ScanParams scan_params(const HstuRecurrenceArgs* a) {
    hstu::ScanParams p{};
    p.x = (const char*)a->x, p.r = (const char*)a->decay_gate, p.i = (const char*)a->input_gate;
    p.x_rs = a->x_row_stride, p.r_rs = a->decay_gate_row_stride, p.i_rs = a->input_gate_row_stride;
    p.decay = a->decay, p.decay_f32 = a->decay_f32, p.rate = a->rate;
    p.offsets = a->seq_offsets, p.offsets_i64 = a->seq_offsets_i64, p.batch = a->batch;
    p.rows = a->rows, p.width = a->width, p.initial = a->initial_state;
    return p;
}

constexpr int kRows = 16, kWaves = 4;           // of a tile, forward and backward
constexpr int kShortRows = 2, kShortWaves = 8;  // at a time, where sequences are short

// Few rows to a sequence, and no state to save: a workgroup for each sequence and 64 columns, in one launch.  It walks its sequence, 16 rows in 0.6 us, where tiles take two
// launches, 10 us at least, and any length side by side.  Measured so and by tiles (us, 512 columns, bf16, from states to states): 8 sequences of 16 rows 4.9 and
// 10.7, 256 of 16 rows 8.4 and 14.4; one of 64 rows 5.1 and 10.3, of 256 13.2 and 11.4, of 1024 46 and 14.  A workgroup costs 3 ns: 512 single rows, 4096 of
// them, 13.3 and 15.4, 768 single rows 18.9 and 17.3, 2000 45 and 21; 1024 and 4096 columns cross over at 4096 workgroups, too.  What a call does not say is which
// sequence is long, and 16 rows on the average and 4096 in all bound what one among single rows can cost (300 of them, one of 3797 rows: 165 and 24), not what
// sequences of one length gain (256 of 64 rows 18.7 and 26.4).
bool scan_is_short(const HstuRecurrenceArgs* a) {
    return !a->saved && a->rows <= 16 * (int64_t)a->batch + 48 && a->rows <= 4096 && (int64_t)a->batch * ((a->width + 63) / 64) <= 4096;
}

// How the tiles of a call are counted, and what they share, behind one another in the scratch memory.
struct ScanPlan {
    int64_t per_segment, segments, slots;
    size_t groups_at, states_at, tickets_at, tiles_at, strength_at, partial_at, bytes;  // (what is in front of tiles_at is cleared)
};

// A segment is a sequence, or as many as have 512 rows on the average: half a tile is lost at its end, and more tiles wait for each other where segments are longer
// (128, 256, 512, 1024 rows: a training step of 400 sequences of 20 .. 150 rows 128, 117, 113, 113 us; prefill of 96 of 20 .. 1023 rows 57.6, 57.6, 57.6, 59.2).
ScanPlan scan_plan(const HstuRecurrenceArgs* a, bool backward) {
    ScanPlan s{};
    s.per_segment = a->rows > 0 ? (512 * (int64_t)a->batch + a->rows - 1) / a->rows : a->batch;
    if (s.per_segment > a->batch) s.per_segment = a->batch;
    if (s.per_segment < 1) s.per_segment = 1;
    s.segments = (a->batch + s.per_segment - 1) / s.per_segment;
    s.slots = a->rows / hstu::kTile + s.segments + 2;
    auto up = [](size_t bytes) { return (bytes + 15) / 16 * 16; };
    s.groups_at = (size_t)s.slots * a->width * 8;
    s.states_at = s.groups_at + (size_t)(s.slots / hstu::kGroup + 1) * a->width * 8;
    s.tickets_at = s.states_at + (size_t)s.slots * a->width * 4;
    s.tiles_at = up(s.tickets_at + (size_t)(a->width + 63) / 64 * hstu::kTicketPitch * 4);
    s.strength_at = s.tiles_at + (size_t)s.slots * sizeof(hstu::Tile);
    s.partial_at = s.strength_at + (size_t)a->width * 4;
    s.bytes = s.partial_at + (backward ? (size_t)s.slots * a->width * 4 : 0);
    return s;
}

// Sets `p` for a call: 0, or the status.
int set_plan(hstu::ScanParams& p, const ScanPlan& s, bool backward, void* scratch) {
    p.col_blocks = (p.width + 63) / 64;
    if (s.slots > kMaxBlocks / p.col_blocks) return HSTU_ERR_UNSUPPORTED;
    p.segments = (int)s.segments, p.per_segment = (int)s.per_segment, p.slots = (int)s.slots, p.backward = backward;
    char* at = (char*)scratch;
    p.sums = (unsigned long long*)at, p.groups = (unsigned long long*)(at + s.groups_at), p.states = (unsigned*)(at + s.states_at);
    p.tickets = (unsigned*)(at + s.tickets_at), p.tiles = (hstu::Tile*)(at + s.tiles_at), p.strength = (float*)(at + s.strength_at);
    p.clear = (int64_t)(s.tiles_at / 16);
    return 0;
}

int launch_begin(int dtype, const hstu::ScanParams& p, hipStream_t stream) {
    const int64_t states = p.final_state ? (int64_t)p.batch * p.width : 0, most = p.clear > states ? p.clear : states, wide = (most + p.width + 1023) / 1024, planned = p.segments / 64 + 1,
                  blocks = wide < 2048 ? wide : 2048;
    return with_type(dtype, [&](auto* t) {
        hipLaunchKernelGGL((hstu::hstu_scan_begin_kernel<std::remove_pointer_t<decltype(t)>>), dim3((unsigned)(blocks > planned ? blocks : planned < 2048 ? planned : 2048)), dim3(256), 0, stream, p);
        return launch_status("recurrence beginning kernel launch");
    });
}

}  // namespace

extern "C" {

int hstu_recurrent_version(void) { return 100; }
const char* hstu_recurrent_last_error(void) { return g_last_error; }

size_t hstu_recurrent_scan_workspace_bytes(const HstuRecurrenceArgs* a) {
    if (check_scan(a) || scan_is_short(a)) return 0;
    return scan_plan(a, false).bytes;
}

size_t hstu_recurrent_scan_saved_bytes(const HstuRecurrenceArgs* a) {
    if (check_scan(a)) return 0;
    return (size_t)scan_plan(a, false).slots * a->width * sizeof(float);
}

int hstu_recurrent_scan(const HstuRecurrenceArgs* a, void* stream) {
    const int rc = check_scan(a);
    if (rc) return rc;
    if (a->rows > 0 && !a->out) return HSTU_ERR_NULL_POINTER;
    hstu::ScanParams p = scan_params(a);
    p.out = (char*)a->out, p.final_state = a->final_state, p.saved = a->saved;
    if (scan_is_short(a)) {
        if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
        return with_type(a->dtype, [&](auto* t) {
            hipLaunchKernelGGL((hstu::hstu_scan_short_kernel<std::remove_pointer_t<decltype(t)>, kShortRows, kShortWaves>), dim3((a->width + 63) / 64, a->batch + 1),
                               dim3(64 * kShortWaves), 0, (hipStream_t)stream, p);
            return launch_status("recurrence kernel launch, short sequences");
        });
    }
    const size_t need = hstu_recurrent_scan_workspace_bytes(a);
    if (!a->workspace) return HSTU_ERR_NULL_POINTER;
    if (!aligned_to(a->workspace, 16)) return HSTU_ERR_MISALIGNED;
    if (a->workspace_bytes < (int64_t)need) return HSTU_ERR_BAD_SHAPE;
    const int status = set_plan(p, scan_plan(a, false), false, a->workspace);
    if (status) return status;
    if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    const int cleared = launch_begin(a->dtype, p, (hipStream_t)stream);
    if (cleared || a->rows == 0) return cleared;
    return with_type(a->dtype, [&](auto* t) {
        hipLaunchKernelGGL((hstu::hstu_scan_kernel<std::remove_pointer_t<decltype(t)>, kRows, kWaves>), dim3((unsigned)(p.slots * p.col_blocks)), dim3(64 * kWaves), 0,
                           (hipStream_t)stream, p);
        return launch_status("recurrence kernel launch");
    });
}

size_t hstu_recurrent_scan_bwd_workspace_bytes(const HstuRecurrenceArgs* a) {
    if (check_scan(a)) return 0;
    return scan_plan(a, true).bytes;
}

int hstu_recurrent_scan_bwd(const HstuRecurrenceArgs* a, const HstuRecurrenceGrads* g, void* stream) {
    const int rc = check_scan(a);
    if (rc) return rc;
    if (!g) return HSTU_ERR_NULL_POINTER;
    if (g->d_out_row_stride < 0) return HSTU_ERR_BAD_SHAPE;
    if (g->d_out_row_stride > kMaxPitch) return HSTU_ERR_UNSUPPORTED;
    if (!g->workspace || (a->rows > 0 && !a->saved)) return HSTU_ERR_NULL_POINTER;
    const int es = bytes_of(a->dtype);
    for (const void* ptr : {g->d_out, (const void*)g->d_x, (const void*)g->d_decay_gate, (const void*)g->d_input_gate})
        if (!aligned_to(ptr, es)) return HSTU_ERR_MISALIGNED;
    if (!aligned_to(g->d_final_state, 4) || !aligned_to(g->d_initial_state, 4) || !aligned_to(g->d_decay, a->decay_f32 ? 4 : es) || !aligned_to(g->workspace, 16))
        return HSTU_ERR_MISALIGNED;
    if (g->workspace_bytes < (int64_t)hstu_recurrent_scan_bwd_workspace_bytes(a)) return HSTU_ERR_BAD_SHAPE;
    hstu::ScanParams p = scan_params(a);
    p.saved = a->saved;
    p.dout = (const char*)g->d_out, p.dout_rs = g->d_out_row_stride, p.dfinal = g->d_final_state;
    p.dx = (char*)g->d_x, p.dr = (char*)g->d_decay_gate, p.di = (char*)g->d_input_gate, p.dinitial = g->d_initial_state;
    const ScanPlan plan = scan_plan(a, true);
    const int status = set_plan(p, plan, true, g->workspace);
    if (status) return status;
    if (g->d_decay) p.partial = (float*)((char*)g->workspace + plan.partial_at);
    if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    hstu::ScanParams clear = p;
    clear.final_state = p.dinitial, clear.initial = p.dfinal;  // the gradient of a state that no row changes
    const int cleared = launch_begin(a->dtype, clear, (hipStream_t)stream);
    if (cleared) return cleared;
    return with_type(a->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        if (a->rows > 0) {
            hipLaunchKernelGGL((hstu::hstu_scan_bwd_kernel<T, kRows, kWaves>), dim3((unsigned)(p.slots * p.col_blocks)), dim3(64 * kWaves), 0, (hipStream_t)stream, p);
            const int rows = launch_status("recurrence backward kernel launch");
            if (rows) return rows;
        }
        if (!g->d_decay) return 0;
        hipLaunchKernelGGL((hstu::hstu_scan_decay_kernel<T>), dim3((a->width + 15) / 16), dim3(1024), 0, (hipStream_t)stream, p.partial, plan.slots, a->width, a->decay,
                           a->decay_f32, a->rate, g->d_decay);
        return launch_status("recurrence decay gradient kernel launch");
    });
}

int hstu_recurrent_step(const HstuRecurrenceStepArgs* a, void* stream) {
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (!known_type(a->dtype)) return HSTU_ERR_BAD_DTYPE;
    if (a->rows < 0 || a->width <= 0 || a->width > 65535 * 64 || a->state_rows < 0 || a->state_row_stride < 0 || !(a->rate > 0.f && std::isfinite(a->rate))) return HSTU_ERR_BAD_SHAPE;
    if (a->x_row_stride < 0 || a->decay_gate_row_stride < 0 || a->input_gate_row_stride < 0) return HSTU_ERR_BAD_SHAPE;
    if (a->rows == 0) return 0;
    if (!a->x || !a->decay_gate || !a->input_gate || !a->out || !a->decay || (a->state_rows > 0 && !a->states)) return HSTU_ERR_NULL_POINTER;
    const int es = bytes_of(a->dtype);
    for (const void* ptr : {a->x, a->decay_gate, a->input_gate, (const void*)a->out})
        if (!aligned_to(ptr, es)) return HSTU_ERR_MISALIGNED;
    if (!aligned_to(a->decay, a->decay_f32 ? 4 : es) || !aligned_to(a->states, 4)) return HSTU_ERR_MISALIGNED;
    if (!aligned_to(a->slots, a->slots_i64 ? 8 : 4) || !aligned_to(a->new_slots, a->new_slots_i64 ? 8 : 4)) return HSTU_ERR_MISALIGNED;
    const int64_t blocks = (a->rows + 4 * hstu::kStepRows - 1) / (4 * hstu::kStepRows);  // four waves
    if (blocks > kMaxBlocks) return HSTU_ERR_UNSUPPORTED;
    if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    hstu::StepParams p{};
    p.x = (const char*)a->x, p.r = (const char*)a->decay_gate, p.i = (const char*)a->input_gate;
    p.x_rs = a->x_row_stride, p.r_rs = a->decay_gate_row_stride, p.i_rs = a->input_gate_row_stride;
    p.out = (char*)a->out, p.decay = a->decay, p.decay_f32 = a->decay_f32, p.rate = a->rate;
    p.states = a->states, p.state_rows = a->state_rows, p.state_rs = a->state_row_stride;
    p.slots = a->slots, p.new_slots = a->new_slots, p.slots_i64 = a->slots_i64, p.new_slots_i64 = a->new_slots_i64;
    p.rows = a->rows, p.width = a->width;
    return with_type(a->dtype, [&](auto* t) {
        hipLaunchKernelGGL((hstu::hstu_scan_step_kernel<std::remove_pointer_t<decltype(t)>>), dim3((unsigned)blocks, (a->width + 63) / 64), dim3(256), 0, (hipStream_t)stream, p);
        return launch_status("recurrence step kernel launch");
    });
}

}  // extern "C"

namespace {

// ---- between two blocks ----

int residual_lanes(int width) {
    int lanes = 8;
    while (lanes * 8 < width) lanes *= 2;
    return lanes;
}
int residual_groups(int lanes) { return lanes > 256 ? 1 : 256 / lanes; }

int64_t residual_workgroups(const HstuResidualNormArgs* a, int64_t most) {
    const int groups = residual_groups(residual_lanes(a->width));
    const int64_t all = (a->rows + groups - 1) / groups;
    return all < most ? all : most;
}

// Forward and backward: 0, or the status.  `wide`: whether all that `p` points to may be read and written in 16-byte pieces.
int fill_residual(const HstuResidualNormArgs* a, hstu::ResidualNormParams& p, bool& wide) {
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (!known_type(a->dtype)) return HSTU_ERR_BAD_DTYPE;
    if (a->rows < 0 || a->width <= 0 || a->x_row_stride < 0 || a->y_row_stride < 0 || a->gate_row_stride < 0) return HSTU_ERR_BAD_SHAPE;
    if (!(a->eps >= 0.f && std::isfinite(a->eps))) return HSTU_ERR_BAD_SHAPE;
    if (a->gate_activation < 0 || a->gate_activation > 2 || !(a->dropout_ratio >= 0. && a->dropout_ratio < 1.)) return HSTU_ERR_BAD_SHAPE;
    if ((a->post_bias && !a->post_weight) || (a->pre_bias && !a->pre_weight)) return HSTU_ERR_NULL_POINTER;
    if (a->width > 8192) return HSTU_ERR_UNSUPPORTED;
    if (a->rows > 0 && (!a->x || !a->y)) return HSTU_ERR_NULL_POINTER;
    p = hstu::ResidualNormParams{};
    const int es = bytes_of(a->dtype), per16 = 16 / es;
    const void* param[hstu::P_COUNT] = {a->post_weight, a->post_bias, a->scale, a->pre_weight, a->pre_bias};
    wide = a->width % 8 == 0;
    auto take = [&](const void* ptr, int64_t rs) {
        if (ptr && (!aligned_to(ptr, 16) || rs % per16 != 0)) wide = false;
        return aligned_to(ptr, es);
    };
    if (!take(a->x, a->x_row_stride) || !take(a->y, a->y_row_stride) || !take(a->gate, a->gate_row_stride)) return HSTU_ERR_MISALIGNED;
    for (int k = 0; k < hstu::P_COUNT; ++k) {
        if (!take(param[k], 0)) return HSTU_ERR_MISALIGNED;
        p.param[k] = (const char*)param[k];
    }
    p.x = (const char*)a->x, p.y = (const char*)a->y, p.gate = (const char*)a->gate;
    p.x_rs = a->x_row_stride, p.y_rs = a->y_row_stride, p.gate_rs = a->gate_row_stride;
    p.eps = a->eps, p.inv_width = 1.f / a->width, p.layer_norm = a->layer_norm, p.act = a->gate_activation;
    p.rows = a->rows, p.width = a->width;
    p.drop.seed = a->dropout_seed, p.drop.offset = a->dropout_offset;
    p.drop.thresh = (uint32_t)(a->dropout_ratio * 4294967296.0), p.drop.scale = (float)(1. / (1. - a->dropout_ratio));
    return 0;
}

template <class F>
int with_row(int lanes, bool wide, F&& f) {
    auto sized = [&](auto l) { return wide ? f(l, std::true_type{}) : f(l, std::false_type{}); };
    switch (lanes) {
        case 8: return sized(std::integral_constant<int, 8>{});
        case 16: return sized(std::integral_constant<int, 16>{});
        case 32: return sized(std::integral_constant<int, 32>{});
        case 64: return sized(std::integral_constant<int, 64>{});
        case 128: return sized(std::integral_constant<int, 128>{});
        case 256: return sized(std::integral_constant<int, 256>{});
        case 512: return sized(std::integral_constant<int, 512>{});
        default: return sized(std::integral_constant<int, 1024>{});
    }
}

// At most so many, which go on to further rows.  Forward: nearly none do (norm of 49028 rows of 512 columns 47 us, with 4096 workgroups 49); backward: two to a
// CU, as many as there is room for, and half as many sums to add up as with 1024 (a training step of 56328 rows 150 us, 157).
constexpr int64_t kForwardWorkgroups = 16384, kBackwardWorkgroups = 512;

}  // namespace

extern "C" {

int hstu_recurrent_residual_norm(const HstuResidualNormArgs* a, void* stream) {
    hstu::ResidualNormParams p;
    bool wide;
    const int rc = fill_residual(a, p, wide);
    if (rc) return rc;
    if (a->rows == 0) return 0;
    if (!a->out || (a->pre_weight && !a->normed)) return HSTU_ERR_NULL_POINTER;
    if (!aligned_to(a->out, bytes_of(a->dtype)) || !aligned_to(a->normed, bytes_of(a->dtype))) return HSTU_ERR_MISALIGNED;
    wide = wide && aligned_to(a->out, 16) && aligned_to(a->normed, 16);
    if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    p.out = (char*)a->out, p.normed = (char*)a->normed;
    const int lanes = residual_lanes(a->width);
    const unsigned blocks = (unsigned)residual_workgroups(a, kForwardWorkgroups);
    return with_type(a->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        return with_row(lanes, wide, [&](auto l, auto w) {
            constexpr int LPR = decltype(l)::value;
            hipLaunchKernelGGL((hstu::hstu_residual_norm_kernel<T, LPR, decltype(w)::value>), dim3(blocks), dim3(LPR > 256 ? LPR : 256), 0, (hipStream_t)stream, p);
            return launch_status("residual norm kernel launch");
        });
    });
}

size_t hstu_recurrent_residual_norm_bwd_workspace_bytes(const HstuResidualNormArgs* a) {
    if (!a || a->rows <= 0 || a->width <= 0 || a->width > 8192) return 0;
    return (size_t)residual_workgroups(a, kBackwardWorkgroups) * hstu::P_COUNT * a->width * sizeof(float);
}

int hstu_recurrent_residual_norm_bwd(const HstuResidualNormArgs* a, const HstuResidualNormGrads* g, void* stream) {
    hstu::ResidualNormParams p;
    bool wide;
    const int rc = fill_residual(a, p, wide);
    if (rc) return rc;
    if (!g) return HSTU_ERR_NULL_POINTER;
    if (g->d_out_row_stride < 0 || g->d_normed_row_stride < 0) return HSTU_ERR_BAD_SHAPE;
    if (a->rows == 0) return HSTU_ERR_BAD_SHAPE;  // (the parameters' gradients would have to be cleared: the caller's to do)
    const int es = bytes_of(a->dtype), per16 = 16 / es;
    for (const void* ptr : {g->d_out, g->d_normed, (const void*)g->d_x, (const void*)g->d_y, (const void*)g->d_gate}) {
        if (!aligned_to(ptr, es)) return HSTU_ERR_MISALIGNED;
        wide = wide && aligned_to(ptr, 16);
    }
    wide = wide && g->d_out_row_stride % per16 == 0 && g->d_normed_row_stride % per16 == 0;
    p.dout = (const char*)g->d_out, p.dout_rs = g->d_out_row_stride;
    p.dnormed = a->pre_weight ? (const char*)g->d_normed : nullptr, p.dnormed_rs = g->d_normed_row_stride;
    p.dx = (char*)g->d_x, p.dy = (char*)g->d_y, p.dgate = a->gate ? (char*)g->d_gate : nullptr;
    void* to[hstu::P_COUNT] = {g->d_post_weight, g->d_post_bias, g->d_scale, g->d_pre_weight, g->d_pre_bias};
    hstu::ParameterGrads grads{};
    int wanted = 0;
    for (int k = 0; k < hstu::P_COUNT; ++k)
        if (to[k] && p.param[k]) {
            if (!aligned_to(to[k], es)) return HSTU_ERR_MISALIGNED;
            p.wanted |= 1 << k, grads.out[wanted] = to[k], grads.which[wanted++] = k;
        }
    if (p.wanted) {
        if (!g->workspace) return HSTU_ERR_NULL_POINTER;
        if (!aligned_to(g->workspace, 16)) return HSTU_ERR_MISALIGNED;
        if (g->workspace_bytes < (int64_t)hstu_recurrent_residual_norm_bwd_workspace_bytes(a)) return HSTU_ERR_BAD_SHAPE;
        p.partial = (float*)g->workspace;
    }
    if (!device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    const int lanes = residual_lanes(a->width);
    const int64_t blocks = residual_workgroups(a, kBackwardWorkgroups);
    return with_type(a->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const int status = with_row(lanes, wide, [&](auto l, auto w) {
            constexpr int LPR = decltype(l)::value;
            hipLaunchKernelGGL((hstu::hstu_residual_norm_bwd_kernel<T, LPR, decltype(w)::value>), dim3((unsigned)blocks), dim3(LPR > 256 ? LPR : 256), 0, (hipStream_t)stream, p);
            return launch_status("residual norm backward kernel launch");
        });
        if (status || !p.wanted) return status;
        hipLaunchKernelGGL((hstu::hstu_residual_norm_sum_kernel<T>), dim3((a->width + 15) / 16, wanted), dim3(1024), 0, (hipStream_t)stream, p.partial, blocks,
                           a->width, grads);
        return launch_status("residual norm parameter gradient kernel launch");
    });
}

}  // extern "C"
