// What the writer and the readers of the paged 8-bit cache share.
#pragma once
#include "common.cuh"
#include <algorithm>

namespace qspec {
namespace kv8 {

// log2 of a page's tokens, 0 for a size that is none
inline int page_shift(int page_tokens) { return page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : page_tokens == 128 ? 7 : 0; }

#ifdef __CUDACC__
// Two codes (bytes c + 128 of w, chosen by sel) as the float16 c, exactly: a byte behind 0x64 is 1152 + c.
__device__ __forceinline__ uint32_t exact_two(uint32_t w, uint32_t sel) {
  const uint32_t m = __byte_perm(w, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
// A scale; one that is zero or next to nothing, or no number, counts as 2^-100.
__device__ __forceinline__ float positive(float x) { return x >= 7.888609052210118e-31f ? x : 7.888609052210118e-31f; }
// A factor of scores, not so small that it would make a hidden key's score (minus infinity) no number.
__device__ __forceinline__ float normal(float x) { return fmaxf(x, 1.17549435e-38f); }
#endif

struct PromptArgs {
  const void* q; long long q_ts; int q_hs;
  const signed char *k, *v;
  const float *ks, *vs;
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep, min_rows;   // min_rows: requests with fewer rows (tokens * rep) are the other kernel's
  float scale2;                                   // scale * log2(e)
  void* out; long long out_ts; int out_hs;
  unsigned give_up;                               // for tests: roles that give their first wait up (1 softmax, 2 codes, 4 products, 8 pages)
};
constexpr int PROMPT_REP = 128;                   // heads of a group that a tile takes at most
int launch_prompt(const PromptArgs& a, int D, bool bf16, cudaStream_t stream);   // kv8_prompt.cu

template <bool BF16> struct Elem16 { using T = __half; };
template <> struct Elem16<true> { using T = __nv_bfloat16; };

}  // namespace kv8
}  // namespace qspec
