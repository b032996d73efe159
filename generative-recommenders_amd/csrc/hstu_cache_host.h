// What the translation units of libhstu_cache.so share on the host.
#pragma once
#include <stdint.h>

#include <type_traits>

#include "hstu_cache.h"
#include "hstu_hip.h"
#include "hstu_paged_rows.h"

extern "C" {
void hstu_cache_set_last_error(const char* what, int hip_error);
int hstu_cache_device_is_gfx950(void);
// The cache as the kernels take it: 0, or the status its fields give.
int hstu_cache_fill(const HstuPagedCache* cache, hstu::PagedCache& p);
}

// Largest grid in x: a launch has fewer than 2^32 threads in a dimension, and a workgroup 256 (rows of 128 columns: 2^28 of them).
constexpr int64_t kMaxBlocks = (1 << 24) - 1;

inline bool hstu_cache_aligned(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

// f(type pointer, lanes of a row) for a cache's type (bf16 or fp16) and 4 to 32 lanes.
template <class F>
int hstu_cache_dispatch(int dtype, int lanes, F&& f) {
    auto sized = [&](auto* t) {
        switch (lanes) {
            case 4: return f(t, std::integral_constant<int, 4>{});
            case 8: return f(t, std::integral_constant<int, 8>{});
            case 16: return f(t, std::integral_constant<int, 16>{});
            default: return f(t, std::integral_constant<int, 32>{});
        }
    };
    return dtype == HSTU_BF16 ? sized((__bf16*)nullptr) : sized((_Float16*)nullptr);
}
