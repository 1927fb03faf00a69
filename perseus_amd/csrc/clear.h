// Shared by the clear side's kernels (rotary.hip, attend.hip): the value types, conversions, argument checks.
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

template <class T>
__device__ __forceinline__ T* at(const HeadsRef& r, int64_t t, int64_t h) {
    return (T*)r.base + t * r.token + h * r.head;
}

}  // namespace clear
}  // namespace pch
