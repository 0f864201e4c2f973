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
// `unit` / v for a value's scale v >= 2^-100. (The reciprocal is that of 2^-24 v: one of less than 2^-126 would be zero.)
__device__ __forceinline__ float over_scale(float unit, float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(v * 5.9604644775390625e-8f));
  return r * (unit * 5.9604644775390625e-8f);
}
#endif

struct PromptArgs4 {
  const void* q; long long q_ts; int q_hs;
  const uint8_t *k, *v;
  const uint16_t *kw, *vw;
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep;
  int pair;                                       // 1: CTAs of the prompt form take two tiles of 128 rows
  unsigned share;                                 // rows that a quarter of the SMs have at a time
  float scale2;                                   // scale * log2(e)
  void* out; long long out_ts; int out_hs;
  unsigned give_up;                               // for tests: roles that give their first wait up (1 softmax, 2 codes, 4 products, 8 pages)
};
int launch_prompt(const PromptArgs4& a, int D, bool bf16, cudaStream_t stream);   // kv4_prompt.cu: the requests that to_prompt_form() names

}  // namespace kv4
}  // namespace qspec
