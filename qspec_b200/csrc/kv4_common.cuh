// What the writer and the readers of the paged 4-bit cache share.
//
// Cache of a layer: codes uint8 [pages, G, P, D / 2], two to a byte, the even column in the low half, and one word of 16 bits [pages, G, P] for each row: its scale s,
// a float32 of five significant bits (exponent in the upper eight bits, mantissa in the next four), and its zero point z in the lowest four. A code c stands
// for (c - z) s.
//
// Why so: every row has its own scale and zero point, so that what a step writes leaves other rows alone. A zero point that is a whole number makes c - z one, which is
// exact in float16: sums over values carry no offset that would have to cancel at their end. A scale of five significant bits makes (c - z) s a number of
// nine, which float16 holds as well (its exponent allowing), and lets scale and zero point share a word: 66 bytes a row of 128.
#pragma once
#include "kv8_common.cuh"

namespace qspec {
namespace kv4 {

using kv8::Elem16;
using kv8::page_shift;

#ifdef __CUDACC__
__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float((w & 0xfff0u) << 15); }
#endif

}  // namespace kv4
}  // namespace qspec
