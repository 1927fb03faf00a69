// Shared by the clear side's kernels (rotary.hip, attend.h, weigh.hip, evict.hip): the value types, conversions, argument checks.
#pragma once
#include "common.h"

namespace pch {
namespace clear {

using bf16 = __bf16;
using f16 = _Float16;

// Whether a tensor reference can be addressed: a base where there is anything to address, strides not negative.
inline bool usable(const HeadsRef& r, int64_t tokens, int64_t heads) {
    return (tokens == 0 || heads == 0 || r.base) && r.token >= 0 && r.head >= 0;
}
// A reference with the strides of single tokens and heads, which no address is made with and which a view may leave at any
// value, as a dense tensor's.
inline HeadsRef settled(HeadsRef r, int64_t tokens, int64_t heads, int64_t dim) {
    if (tokens < 2) r.token = dim;
    if (heads < 2) r.head = dim;
    return r;
}
// Whether an output's heads lie apart (a stride of one row only matters where there is a second one).
inline bool apart(const HeadsRef& r, int64_t tokens, int64_t heads, int64_t dim) {
    if (tokens == 0 || heads == 0) return true;
    return (tokens < 2 || r.token >= dim) && (heads < 2 || r.head >= dim);
}

// A cache in pages, as the kernels take it: sequence b's key j lies in row page[j >> log] << log plus j's low bits, page =
// table + b seq, of a pool of `count` pages; a sequence has `width` pages at most.
struct PagesRef {
    const int32_t* table;
    int64_t seq;
    int32_t width, count, log;
    // the pool's row of key j, which lies on `page`; -1: on one that the pool does not have
    __device__ __forceinline__ int64_t row(int page, uint32_t j) const {
        return (uint32_t)page < (uint32_t)count ? ((int64_t)page << log) + (j & ((1u << log) - 1)) : -1;
    }
};
// the pages of a cache of `rows` rows: 0, or the error
inline int pages_of(const CacheRef& c, int64_t seqs, int64_t rows, PagesRef* p) {
    if (seqs && !c.pages) return -1;
    if (c.width < 1 || c.pages_seq < 0 || (seqs > 1 && c.pages_seq < c.width)) return -1;
    if (c.page_rows < 16 || (c.page_rows & (c.page_rows - 1))) return -2;
    int log = 4;
    while (1 << log < c.page_rows) ++log;
    const int64_t count = rows >> log;
    *p = {c.pages, c.pages_seq, c.width, (int32_t)(count > 0x7fffffff ? 0x7fffffff : count), log};
    return 0;
}

template <class T>
__device__ __forceinline__ T* at(const HeadsRef& r, int64_t t, int64_t h) {
    return (T*)r.base + t * r.token + h * r.head;
}

}  // namespace clear
}  // namespace pch
