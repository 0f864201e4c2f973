// What the writer and the readers of the paged 8-bit cache share.
#pragma once
#include "common.cuh"
#include <algorithm>

namespace qspec {
namespace kv8 {

// log2 of a page's tokens, 0 for a size that is none
inline int page_shift(int page_tokens) { return page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : page_tokens == 128 ? 7 : 0; }

template <bool BF16> struct Elem16 { using T = __half; };
template <> struct Elem16<true> { using T = __nv_bfloat16; };

}  // namespace kv8
}  // namespace qspec
