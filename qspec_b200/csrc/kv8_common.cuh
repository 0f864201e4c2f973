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
// Weights 2^(score + log2 of the value scale - reference) are rounded to float16 for their product with the codes, and the denominator is the sum of the unrounded
// ones: what float16 cannot hold is lost to the one and not to the other, always to the same side, and over a long context that adds up. So weights begin at
// 2^WEIGHT_LOG2 where the reference stands, and it follows the maximum as soon as that is 2^GROWTH_LOG2 above it: the largest is at most 2^15, what is above 2^-23 of it
// is rounded by 2^-11 of itself at most, and below that a key is off by 2^-25 of 2^9 at most. (While weights began at 1, behind a key that leads in a page whose value
// scale is 64 times the others', 131,000 keys at 2^-19.1 of its weight, 19 % of all there is, came to nothing in the sum of values.) A reference that follows
// sooner costs the prompt form: 2000 tokens after 1000, with growth by 2^8 112 us, 2^6 114, 2^5 115, 2^4 117. 2^16 is infinite, and a reference has a rounding of its
// own: beyond FAR it is subtracted from the finished exponent, which was rounded like it. Sums of weights / v are kept in units of 2^WEIGHT_LOG2, so that they
// hold for every scale that positive() leaves.
constexpr float WEIGHT_LOG2 = 9.f, GROWTH_LOG2 = 6.f, WEIGHT_UNIT = 1.f / 512.f, FAR = 1048576.f;
// An infinite one is no number either: beside a hidden key's minus infinity it would be one in rows that do not see the page.
__device__ __forceinline__ float finite_scale(float x) { return x < INFINITY ? x : NAN; }
// What scores in units of 2^-24 are multiplied with, from the scale of the keys and the row's factor: these two first, since either may be as far from 1 as float32 goes and
// the other as far on the other side. Not so small that it would make a hidden key's score (minus infinity) no number.
__device__ __forceinline__ float score_factor(float scale, float row) { return fmaxf(scale * row * 16777216.f, 1.17549435e-38f); }

// Keys that are walked at most: those that a row of the table has pages for, and one that it has none for (less than what would leave an int when it is rounded up).
__device__ __forceinline__ int keys_at_most(int width, int pshift) { return (int)min(((unsigned)width << pshift) + 1u, 0x7fffff80u); }

// Which form of the attention a request goes to, from what all requests of the call ask for; both kernels work it out alike. The prompt form takes 128 rows (tokens *
// heads of a group) and a head a CTA, so that a block of keys costs it the same however few requests there are; the other one spreads any request over the GPU but
// reads the keys again for every 16 rows. A request goes to the prompt form if the call has rows for a third of the SMs, it has PROMPT_ROWS rows or more, and its way
// through its keys is no longer than what the requests of that size have to do together would take on a quarter of the SMs (a third there, too, parted requests of
// like lengths, and the two kernels run one after the other: 4 requests of 64 tokens after 4000 to 8000 keys 159 us, so 113).
// Both forms measured, 32 / 8 heads of 128, us of the prompt form (of the other):
//   1 request, 1000 keys in front of it   32 tokens 28 (19)   128: 28 (31)   256: 30 (47)   1024: 63 (196)
//   1 request, 32000 keys                 32 tokens 444 (110)   128: 444 (343)   256: 453 (671)   512: 459 (1335)
//   4 requests, 8000 keys                 17 tokens 111 (62)   48: 113 (113)   64: 113 (142)   128: 116 (269)
//   16 requests, 1000 keys                17 tokens 27 (44)   64: 43 (103)   128: 76 (193)
constexpr int PROMPT_ROWS = 65;
__device__ __forceinline__ unsigned long long prompt_work(int n, int keys, int rep, int G) {
  const unsigned long long rows = (unsigned long long)n * rep;
  return rows >= PROMPT_ROWS ? rows * G * ((keys + 127ll) / 128) : 0ull;
}
// work: of all requests; share: rows that a quarter of the SMs have at a time (0: there is no prompt form)
__device__ __forceinline__ bool to_prompt_form(int n, int keys, int rep, unsigned share, unsigned long long work) {
  return share && (unsigned long long)n * rep >= PROMPT_ROWS && (unsigned long long)((keys + 127ll) / 128) * share <= work;
}
#endif

struct PromptArgs {
  const void* q; long long q_ts; int q_hs;
  const signed char *k, *v;
  const float *ks, *vs;
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep;
  int pair;                                       // 1: CTAs of the prompt form take two tiles of 128 rows
  unsigned share;                                 // rows that a quarter of the SMs have at a time
  float scale2;                                   // scale * log2(e)
  void* out; long long out_ts; int out_hs;
  unsigned give_up;                               // for tests: roles that give their first wait up (1 softmax, 2 codes, 4 products, 8 pages)
};
constexpr int PROMPT_REP = 128;                   // heads of a group that a tile takes at most
int launch_prompt(const PromptArgs& a, int D, bool bf16, cudaStream_t stream);   // kv8_prompt.cu: the requests that to_prompt_form() names

template <bool BF16> struct Elem16 { using T = __half; };
template <> struct Elem16<true> { using T = __nv_bfloat16; };

}  // namespace kv8
}  // namespace qspec
