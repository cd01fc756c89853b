// paged_common.h -- what the paged-cache launchers check alike.
#pragma once
#include <climits>

#include "../../include/rocmforge_cdna4.h"

namespace rf {

inline bool page_size_ok(int n) { return n >= 8 && n <= 1024 && (n & (n - 1)) == 0; }

inline bool cache_ok(const rf_paged_cache& c) {
    if (!c.k || !c.v || c.num_kv_heads <= 0 || c.num_kv_heads > 65535 || !page_size_ok(c.page_size) ||
        c.num_pages <= 0 || (int64_t)c.num_pages * c.page_size > INT_MAX)
        return false;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return false;
    if (((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15u) != 0) return false;
    return c.page_stride > 0 && c.row_stride > 0 && c.head_stride > 0 && c.row_stride <= (1 << 26) &&
           ((c.page_stride | c.row_stride | c.head_stride) & 7) == 0;
}

}  // namespace rf
