// What the paged key/value cache's translation units share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "kernels.cuh"

namespace bd {

// Element strides of a cache [pages][page_size][kv_heads][head_dim] (the last is 1).
struct CacheStrides {
    int64_t page, slot, head;
};

inline bool page_size_ok(int p) { return p >= 8 && p <= 256 && (p & (p - 1)) == 0; }
inline int log2_of(int p) {
    int s = 0;
    while ((1 << s) < p) ++s;
    return s;
}
// Slots and key positions are 32-bit.
inline bool pool_ok(int64_t pages, int page_size) { return pages >= 1 && pages <= INT32_MAX / page_size; }
inline bool table_ok(int64_t width, int page_size) { return width >= 1 && width <= (INT32_MAX - 512) / page_size; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// 16-byte pieces start at every stride.
inline bool cache_strides(const int64_t *s, CacheStrides &out) {
    out = CacheStrides{s[0], s[1], s[2]};
    return s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && ((s[0] | s[1] | s[2]) & 7) == 0;
}

// The bytes [begin, end) that a strided tensor lies in.
struct Span {
    uintptr_t begin, end;
    bool meets(const Span &o) const { return begin < o.end && o.begin < end; }
};
inline Span span_of(const void *p, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Span{at, at + static_cast<uintptr_t>(bytes)};
}
inline Span cache_span(const void *p, const CacheStrides &s, int64_t pages, int page_size, int heads, int head_dim) {
    return span_of(p, 2 * ((pages - 1) * s.page + (page_size - 1) * s.slot + (heads - 1) * s.head + head_dim));
}

}  // namespace bd
