// Log probabilities: of each row x of logits, with the temperature T and c = log2(e) / T,
//   y_i = c (x_i - max x),   S = sum 2^y_i,   U = sum 2^y_i y_i
// the given token's log probability ln2 (y_t - log2 S), its rank 1 + #{i: x_i > x_t}, the entropy ln2 (log2 S - U / S), and the `top` largest log probabilities with their
// tokens, equal ones by the lower token.
//
// What bounds it is reading the row, once, and the exponentials. One CTA, or a cluster of up to eight, takes a row; a CTA walks its span in batches of 1024 vectors of 16 bytes, the
// next batch's loads under way. Exponents are counted from the first batch's maximum, and by a thread that sees a larger value (they are few) from that one on, its sums multiplied again: no
// exponent is above zero, the largest value's weight is 1 exactly, and a likely token's log probability is no difference of large numbers (nor above zero). Candidates for
// the best are, of the first batch, the values that reach the smallest of as many groups' maxima as are asked for, or more (at least that many do, and hardly more than some
// hundred), and later on those above the worst of the best so far, which is brought up to date whenever four (or, of up to eight, eight) times as much has been
// seen: a few at a time. Where there are more than there
// is room for (rows that rise, rows of one value), the span is looked through once for each one that is asked for. Whichever way, values are ordered together with their
// tokens as whole numbers of 64 bits, so that there is one result. Sums are made in a fixed order in float32.
// Measured: 4 rows of 128256 in float16 6.3 us, with 5 alternatives 8.3; 256 rows 21.6, with 5 26.2 (2.5 TB/s: some 11 instructions a value, issue 60 %); 1000 rows of 151643 in float32 with 20
// 118 to 125 (5 TB/s). Not taken: exponents without an end at -16384, and sums that are no number made again (a value's instruction less; 256 rows 24.4 for 21.5); three CTAs an SM (24.9).
#include "seq_common.cuh"
#include "../../include/qspec_b200_seq.h"
#include <algorithm>

namespace qspec {
namespace logprob {

constexpr int THREADS = 256, WARPS = THREADS / 32, MOST_TOP = 32, EACH = 4;   // EACH: vectors of a thread in a batch
constexpr int GROUPS = 128, GROUP = THREADS / GROUPS, HITS = 256, CANDIDATES = 512;   // groups of neighbouring threads; vectors with candidates, candidates in them
// Alternatives that are few: us taken like more of them (so), with 1, 5, 8, 9, 12, 20: 256 float16 rows of 128256 27.6 (25.0), 29.0 (27.6), 30.4 (28.9), 30.2 (29.8), 31.1 (143: more candidates
// than there is room for), 33.3 (346); 4 rows 11.0 (9.6), 11.7 (10.4), 12.0 (10.8), 12.2 (11.1), 12.5 (11.5), 13.6 (13.5); 600 float32 rows of 151643 99 (97), 101 (99), 102 (100), 103 (101), 103 (661), 105 (1573).
constexpr int FEW_TOP = 8;
typedef unsigned long long u64;

struct Args {
  const void* logits; long long stride;
  const long long* tokens;
  float *logprobs, *entropy; long long* ranks;
  float* top_logprobs; long long* top_tokens;
  int V, span, top;                               // span: values of a CTA
  float c;
};
struct Partial {                                  // of a span: what its exponents are counted from, sums, values above the given token's, how many of the best there are
  float ref, S, U;
  int above, best;
};

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T lowest();   // minus infinity
template <> __device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ u64 add2(u64 a, u64 b) { u64 r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ u64 mul2(u64 a, u64 b) { u64 r; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }

// A vector's values: the largest (no number if one is none), all of them, how many are above another.
template <typename T> struct Lanes;
template <> struct Lanes<float> {
  static __device__ __forceinline__ float largest(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ void values(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  // how many are above `given`, of up to EACH vectors, in pairs of their own
  typedef u64 Count;
  static __device__ __forceinline__ Count none() { return 0ull; }
  static __device__ __forceinline__ void above(Count& n, const uint4& w, float given) {
    auto one = [&](uint32_t x) { return __uint_as_float(x) > given ? 1.f : 0.f; };
    n = add2(n, add2(pack_f2(one(w.x), one(w.y)), pack_f2(one(w.z), one(w.w))));
  }
  static __device__ __forceinline__ int total(const Count& n) { const float2 f = unpack_f2(n); return (int)(f.x + f.y); }
};
#define QSPEC_LANES16(T, T2, SUFFIX, UNPACK, FROM)                                                                                                               \
  template <> struct Lanes<T> {                                                                                                                                  \
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN." SUFFIX " %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b)); return r; } \
    static __device__ __forceinline__ float largest(const uint4& w) {                                                                                            \
      const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));                                                                                                   \
      const T2 h = *reinterpret_cast<const T2*>(&m);                                                                                                             \
      return max_nan(value(h.x), value(h.y));                                                                                                                    \
    }                                                                                                                                                            \
    static __device__ __forceinline__ void values(const uint4& w, float (&x)[8]) { UNPACK(w, x); }                                                                \
    typedef T2 Count;                                                                                                                                            \
    static __device__ __forceinline__ Count none() { return FROM(0.f); }                                                                                         \
    static __device__ __forceinline__ void above(Count& n, const uint4& w, float given) {   /* (given is one of the row's values; sums to 4 EACH: exact) */      \
      const T2 g = FROM(given);                                                                                                                                  \
      const T2* h = reinterpret_cast<const T2*>(&w);                                                                                                             \
      n = __hadd2(n, __hadd2(__hadd2(__hgt2(h[0], g), __hgt2(h[1], g)), __hadd2(__hgt2(h[2], g), __hgt2(h[3], g))));                                             \
    }                                                                                                                                                            \
    static __device__ __forceinline__ int total(const Count& n) { return (int)(value(n.x) + value(n.y)); }                                                       \
  };
QSPEC_LANES16(__half, __half2, "f16x2", unpack_h8, __float2half2_rn)
QSPEC_LANES16(__nv_bfloat16, __nv_bfloat162, "bf16x2", unpack_b8, __float2bfloat162_rn)
#undef QSPEC_LANES16

// Larger values first, no numbers before all, equal ones by the lower index; never 0, nor all ones (which best_below() begins with).
constexpr uint32_t NO_NUMBER = 0xfffffffeu;       // (infinity is 0xff800000)
__device__ __forceinline__ u64 key_of(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.f);              // (-0 is 0)
  const uint32_t v = x != x ? NO_NUMBER : u & 0x80000000u ? ~u : u | 0x80000000u;
  return (u64)v << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(u64 key) {
  const uint32_t v = (uint32_t)(key >> 32);
  return v == NO_NUMBER ? NAN : __uint_as_float(v & 0x80000000u ? v ^ 0x80000000u : ~v);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(uint32_t)key; }

// Floats as numbers in their order.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// A value that as many of the groups' maxima reach as are asked for (n <= GROUPS), or some more: the n-th largest, but for the lower half of its bits. Every warp finds it for itself.
__device__ __forceinline__ float nth_largest(const float* s_group, int n) {
  static_assert(GROUPS == 128, "four a lane");
  const float4 x = reinterpret_cast<const float4*>(s_group)[threadIdx.x & 31];
  if (n <= FEW_TOP) {                                       // of 32 groups, one after the other (16 steps of bisection take 1000 cycles, one of these 40)
    uint32_t most = ordered(max_nan(max_nan(x.x, x.y), max_nan(x.z, x.w))), t = 0;
    for (int i = 0; i < n; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, most);
      if (!m) break;                                        // (equal ones go together)
      t = m;
      if (most == m) most = 0;
    }
    return __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
  }
  const uint32_t k[4] = {ordered(x.x) >> 16, ordered(x.y) >> 16, ordered(x.z) >> 16, ordered(x.w) >> 16};
  uint32_t t = 0;
#pragma unroll 1
  for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
    const uint32_t y = t | bit;
    if (__reduce_add_sync(0xffffffffu, (k[0] >= y) + (k[1] >= y) + (k[2] >= y) + (k[3] >= y)) >= n) t = y;
  }
  const uint32_t u = t << 16;
  return t <= 0x7fu ? -INFINITY : __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);   // (0x7f: minus infinity and what is next to it)
}

// The vector at value `first` of the span's n, which may lie over its ends.
template <typename T>
__device__ __noinline__ uint4 edge(const T* from, int n, int first) {
  constexpr int E = Vec<T>::N;
  uint4 w;
  if (first >= 0 && first + E <= n) {
    w = __ldg(reinterpret_cast<const uint4*>(from + first));
  } else {
    T* const x = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = first + e >= 0 && first + e < n ? from[first + e] : lowest<T>();
  }
  return w;
}

// The largest key below `before` of this thread's vectors; 0: there is none.
template <typename T>
__device__ __noinline__ u64 best_below(const T* from, int n, int shift, int lo, u64 before) {
  constexpr int E = Vec<T>::N;
  u64 most = 0;
#pragma unroll 1
  for (int first = (int)threadIdx.x * E - shift; first < n; first += THREADS * E) {
    const uint4 w = edge<T>(from, n, first);
    const T* const x = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = first + e;
      const u64 key = key_of(value(x[e]), lo + i);
      if (i >= 0 && i < n && key < before && key > most) most = key;
    }
  }
  return most;
}

template <typename T, int CLUSTER>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const Args a) {
  constexpr int E = Vec<T>::N;
  using L = Lanes<T>;
  __shared__ Partial s_part;
  __shared__ u64 s_best[MOST_TOP], s_key[CANDIDATES], s_most[WARPS];
  __shared__ uint4 s_hit[HITS];
  __shared__ __align__(16) float s_group[GROUPS];
  __shared__ float s_ref[WARPS], s_sum[2][WARPS];
  __shared__ int s_above[WARPS], s_where[HITS], s_hits[2], s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  if (tid == 0) s_hits[0] = s_hits[1] = s_count = 0;
  pdl_enter();
  const T* const x_row = (const T*)a.logits + (size_t)row * a.stride;
  const int lo = min(rank * a.span, a.V), n = min(a.span, a.V - lo);
  const T* const from = x_row + lo;
  // Vectors lie on 16-byte boundaries, the first and the last may lie over the span's ends: what stands there is minus infinity instead.
  const int shift = (int)(((uintptr_t)from & 15) / sizeof(T)), vectors = n > 0 ? (n + shift + E - 1) / E : 0;
  const uint4* const at0 = reinterpret_cast<const uint4*>(from - shift) + tid;
  const int inner0 = shift ? 1 : 0, inner1 = (n + shift) / E;   // vectors that are the span's as a whole
  constexpr int BATCH = THREADS * EACH;
  const int batches = (vectors + BATCH - 1) / BATCH;
  uint4 next[EACH];
  auto load = [&](int b) {
    const int v = b * BATCH;
    if (v >= inner0 && v + BATCH <= inner1) {               // (nearly always)
#pragma unroll
      for (int j = 0; j < EACH; ++j) next[j] = __ldg(at0 + v + j * THREADS);
    } else {
#pragma unroll
      for (int j = 0; j < EACH; ++j) next[j] = edge<T>(from, n, (v + j * THREADS + tid) * E - shift);
    }
  };
  load(0);
  const long long token = a.tokens ? a.tokens[row] : -1;
  const bool there = token >= 0 && token < a.V;
  const float given = there ? value(x_row[token]) : INFINITY;   // (nothing is above it)

  float ref = -INFINITY, reach = INFINITY;                  // what exponents are counted from; what a candidate has to reach (of the first batch) or to exceed
  bool none = true;                                         // nothing but minus infinity so far: there is nothing to count from
  float limit = -INFINITY;                                  // what a value that is looked at more closely reaches
  auto set_limit = [&]() { limit = none ? -INFINITY : fminf(reach, ref); };
  u64 S2 = 0, U2 = 0;
  // (the candidates of eight batches for FEW_TOP are few)
  int above = 0, best = 0, check = a.top > FEW_TOP ? 0 : 7, turn = 0;             // check: the batch behind which the best are brought up to date; turn: which count of hits is in use
  bool first = true, lost = false;                                        // there were more candidates than there is room for
  bool odd = false;                                         // there is something that is no number
  for (int b = 0; b < batches; ++b) {
    uint4 w[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) w[j] = next[j];
    if (b + 1 < batches) load(b + 1);
    float big[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) big[j] = L::largest(w[j]);
    if (b == 0) {
      // ---- the first batch's maximum, and what the best have to reach
      float g = max_nan(max_nan(big[0], big[1]), max_nan(big[2], big[3]));
#pragma unroll
      for (int o = 1; o < GROUP; o <<= 1) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, o));
      if (tid % GROUP == 0) s_group[tid / GROUP] = g;
      __syncthreads();
      {
        const float4 x = reinterpret_cast<const float4*>(s_group)[lane];
        ref = max_nan(max_nan(x.x, x.y), max_nan(x.z, x.w));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ref = max_nan(ref, __shfl_xor_sync(0xffffffffu, ref, o));
      if (a.top) reach = nth_largest(s_group, a.top);
      none = ref == -INFINITY;
      if (none) ref = 0.f;                                  // (weights of minus infinity are zero wherever they are counted from)
      set_limit();
    }
    const float most = max_nan(max_nan(big[0], big[1]), max_nan(big[2], big[3]));
    if (!(most < limit)) {                                  // seldom: candidates, a value above all before it, no numbers. (Code that is short, and there once: it is cold)
      odd |= most != most;
      if (none ? most > -INFINITY : most > ref) {
        const float d = fmaxf((ref - most) * a.c, -16384.f), f = none ? 0.f : ex2(d);
        const float2 S = unpack_f2(S2), U = unpack_f2(U2);
        U2 = pack_f2(fmaf(S.x, d, U.x) * f, fmaf(S.y, d, U.y) * f);
        S2 = pack_f2(S.x * f, S.y * f);
        ref = most;
        none = false;
        set_limit();
      }
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (b == 0 ? big[j] >= reach : big[j] > reach) {
          const int at = atomicAdd(&s_hits[turn], 1);             // (in any order: they are put in theirs)
          if (at < HITS) {
            s_hit[at] = w[j];
            s_where[at] = ((b * EACH + j) * THREADS + tid) * E - shift;
          }
        }
    }
    if (a.ranks) {
      typename L::Count larger = L::none();
#pragma unroll
      for (int j = 0; j < EACH; ++j) L::above(larger, w[j], given);
      above += L::total(larger);
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      float x[E];
      L::values(w[j], x);
      const u64 minus = pack_f2(-ref, -ref), c2 = pack_f2(a.c, a.c);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float2 y = unpack_f2(mul2(add2(pack_f2(x[e], x[e + 1]), minus), c2));
        y = make_float2(max_nan(y.x, -16384.f), max_nan(y.y, -16384.f));   // (a weight of zero times minus infinity is no number)
        const u64 y2 = pack_f2(y.x, y.y);
        const u64 w2 = pack_f2(ex2(y.x), ex2(y.y));
        S2 = add2(S2, w2);
        U2 = ffma2_rn(w2, y2, U2);
      }
    }
    if (a.top && (b == check || b + 1 == batches)) {
      // ---- the best so far: of those of before, which are the first keys, and of the candidates
      __syncthreads();
      // What is counted from here on is counted elsewhere, whatever this says: there is no barrier between a warp's look at it and another warp's next batch.
      const int hits = s_hits[turn];
      if (hits > HITS) lost = true;                         // (the same for all)
      if (hits && !lost) {
        for (int i = tid; i < hits * E; i += THREADS) {
          const float y = value(reinterpret_cast<const T*>(s_hit)[i]);
          const int at = s_where[i / E] + i % E;
          if ((first ? y >= reach : y > reach) && at >= 0 && at < n) {
            const int k = atomicAdd(&s_count, 1);
            if (k < CANDIDATES) s_key[k] = key_of(y, lo + at);
          }
        }
        __syncthreads();
        const int count = s_count;
        if (count <= CANDIDATES) {
          for (int i = tid; i < count; i += THREADS) {
            const u64 key = s_key[i];
            int larger = 0;
#pragma unroll 4
            for (int j = 0; j < count; ++j) larger += s_key[j] > key;
            if (larger < a.top) s_best[larger] = key;
          }
          __syncthreads();
          // (the next to look at these come behind a barrier)
          best = min(count, a.top);
          if (tid < best) s_key[tid] = s_best[tid];
          if (tid == 0) { s_count = best; s_hits[turn] = 0; }
          if (best == a.top) reach = value_of(s_best[best - 1]);
        } else {
          lost = true;
        }
      }
      turn ^= 1;                                            // (the other count is zero: nothing has been counted there since it was set to that, a barrier ago)
      if (lost) reach = INFINITY;                           // all of them are looked for at the end
      first = false;
      check = (a.top > FEW_TOP ? 4 : 8) * (b + 1) - 1;
      set_limit();
    }
  }
  // ---- the threads' sums together
  float m = none ? -INFINITY : ref;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s_ref[warp] = m;
  odd = __syncthreads_or(odd);
  m = s_ref[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) m = max_nan(m, s_ref[i]);
  float S, U;
  {
    const float2 s = unpack_f2(S2), u = unpack_f2(U2);
    const float d = fmaxf((ref - m) * a.c, -16384.f), f = none ? 0.f : ref == m ? 1.f : ex2(d);
    S = (s.x + s.y) * f;
    U = ref == m ? u.x + u.y : none ? 0.f : fmaf(s.x + s.y, d, u.x + u.y) * f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    S += __shfl_xor_sync(0xffffffffu, S, o);
    U += __shfl_xor_sync(0xffffffffu, U, o);
  }
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) { s_sum[0][warp] = S; s_sum[1][warp] = U; s_above[warp] = above; }
  if (a.top && (odd || lost)) {             // (the same for all: the barrier above)
    u64 mine = best_below<T>(from, n, shift, lo, ~0ull);
    for (best = 0; best < a.top; ++best) {                  // whoever had the best looks for his next
      u64 most = mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, most, o);
        most = other > most ? other : most;
      }
      if (lane == 0) s_most[warp] = most;
      __syncthreads();
      most = s_most[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) most = s_most[i] > most ? s_most[i] : most;
      __syncthreads();
      if (!most) break;
      if (mine == most) {
        s_best[best] = most;
        mine = best_below<T>(from, n, shift, lo, most);
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    Partial p{m, 0.f, 0.f, 0, best};
    for (int i = 0; i < WARPS; ++i) { p.S += s_sum[0][i]; p.U += s_sum[1][i]; p.above += s_above[i]; }
    s_part = p;
  }
  if (CLUSTER > 1) cluster_sync_all(); else __syncthreads();

  // ---- the first CTA joins the spans
  if (rank == 0) {
    Partial p[CLUSTER];
    p[0] = s_part;
    if (CLUSTER > 1) {
#pragma unroll
      for (int r = 1; r < CLUSTER; ++r) {
        const uint32_t at = mapa_shared((uint32_t)__cvta_generic_to_shared(&s_part), r);
        p[r].ref = __uint_as_float(ld_dsmem_u32(at));
        p[r].S = __uint_as_float(ld_dsmem_u32(at + 4));
        p[r].U = __uint_as_float(ld_dsmem_u32(at + 8));
        p[r].above = (int)ld_dsmem_u32(at + 12);
        p[r].best = (int)ld_dsmem_u32(at + 16);
      }
    }
    float M = -INFINITY;
#pragma unroll
    for (int r = 0; r < CLUSTER; ++r)
      if (p[r].S != 0.f) M = max_nan(M, p[r].ref);          // (a span of minus infinities counts from nowhere)
    S = U = 0.f;
    above = 0;
#pragma unroll
    for (int r = 0; r < CLUSTER; ++r) {
      above += p[r].above;
      if (p[r].S == 0.f) continue;
      const float d = fmaxf((p[r].ref - M) * a.c, -16384.f), f = p[r].ref == M ? 1.f : ex2(d);
      S = fmaf(p[r].S, f, S);
      U = fmaf(p[r].ref == M ? p[r].U : fmaf(p[r].S, d, p[r].U), f, U);
    }
    const float ln2 = 0.69314718055994531f, lse = log2f(S);
    const bool nothing = M == -INFINITY;                    // no token has any probability
    auto logprob = [&](float x) { return nothing ? -INFINITY : ((x - M) * a.c - lse) * ln2; };
    if (tid == 0) {
      if (a.logprobs) a.logprobs[row] = token < 0 ? 0.f : there ? logprob(given) : lse != lse ? NAN : -INFINITY;
      if (a.ranks) a.ranks[row] = there ? 1 + above : 0;
      if (a.entropy) a.entropy[row] = nothing ? 0.f : lse != lse ? NAN : (lse - U / S) * ln2;
    }
    if (a.top) {
      int all = 0, mine = -1;                               // of the slices' best, one behind the other: how many, and which slice's this thread's is
      int first[CLUSTER];
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r) {
        first[r] = all;
        all += p[r].best;
      }
      __syncthreads();                                      // (candidates make room)
#pragma unroll
      for (int r = 0; r < CLUSTER; ++r)
        if (tid >= first[r] && tid < first[r] + p[r].best) mine = r;
      u64 key = 0;
      if (mine >= 0) {
        int skip = tid;
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r)
          if (r == mine) skip = tid - first[r];
        if (CLUSTER > 1) {
          const uint32_t at = mapa_shared((uint32_t)__cvta_generic_to_shared(s_best + skip), mine);
          key = (u64)ld_dsmem_u32(at) | (u64)ld_dsmem_u32(at + 4) << 32;
        } else {
          key = s_best[skip];
        }
        s_key[tid] = key;
      }
      __syncthreads();
      if (mine >= 0) {
        int larger = 0;
        for (int j = 0; j < all; ++j) larger += s_key[j] > key;
        if (larger < a.top) {
          a.top_logprobs[(size_t)row * a.top + larger] = logprob(value_of(key));
          a.top_tokens[(size_t)row * a.top + larger] = index_of(key);
        }
      }
    }
  }
  if (CLUSTER > 1) cluster_sync_all();                      // the first CTA has read the others' results
}

}  // namespace logprob
}  // namespace qspec

using namespace qspec;
using namespace qspec::logprob;

extern "C" int qspec_seq_token_logprobs_max_top(void) { return MOST_TOP; }

extern "C" int qspec_seq_token_logprobs(const void* logits, long long row_stride, const long long* tokens, float* logprobs, float* entropy, long long* ranks, float* top_logprobs,
                                        long long* top_tokens, int rows, int V, int top, float temperature, int dtype, void* stream) {
  QSPEC_REQUIRE(rows >= 0 && V >= 1 && row_stride >= V, QSPEC_ERR_INVALID_ARG, "token_logprobs: rows=%d vocabulary=%d row stride=%lld", rows, V, row_stride);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16 || dtype == QSPEC_DTYPE_F32, QSPEC_ERR_UNSUPPORTED, "token_logprobs: float16, bfloat16 or float32 logits");
  QSPEC_REQUIRE(top >= 0 && top <= MOST_TOP && top <= V, QSPEC_ERR_UNSUPPORTED, "token_logprobs: the best 0 to %d of %d tokens, got %d", std::min(MOST_TOP, V), V, top);
  const float c = 1.4426950408889634f / temperature;
  QSPEC_REQUIRE(temperature > 0.f && c > 0.f && c < INFINITY, QSPEC_ERR_INVALID_ARG, "token_logprobs: the temperature must be positive and finite, got %g", (double)temperature);
  if (rows == 0) return QSPEC_OK;
  const int size = dtype == QSPEC_DTYPE_F32 ? 4 : 2;
  QSPEC_REQUIRE(logits && (!top || (top_logprobs && top_tokens)) && (tokens || (!logprobs && !ranks)), QSPEC_ERR_INVALID_ARG, "token_logprobs: null pointer");
  QSPEC_REQUIRE((uintptr_t)logits % size == 0 && ((uintptr_t)tokens & 7) == 0, QSPEC_ERR_INVALID_ARG, "token_logprobs: logits and tokens must lie on their types' boundaries");
  // CTAs of a row: two while that leaves the SMs four each at most, four while three, eight while two and a half (larger clusters find their places less well), and more than a batch
  // each. us with 1 / 2 / 4 / 8, float16, 5 alternatives, a call alone (and calls behind one another, of which the next begins while the last rows of one are looked at):
  //   128256 values   4 rows 20 / 16 / 13 / 12   45: 21 / 18 / 15 / 15   75: 22 / 18 / 17 / 25   148: 23 / 20 / 28 / 39   256: 28 / 30 / 36 (38 / 29 / 35)   330: (40 / 38 / 44)
  //   32000 values    4 rows 10 / 11 / 9   100: 12 / 13 / 11   148: 12 / 13 / 19 (12 / 12 / 18)   256: 14 / 17 / 23 (17 / 16 / 22)   400: 16 / 26 / 32 (18 / 24 / 31)
  const int sms = std::max(sm_count(), 1), batch = THREADS * EACH * 16 / size, halves[] = {8, 6, 5};
  int cluster = 1;
  for (int i = 0; i < 3 && 2ll * rows * (2 * cluster) <= (long long)halves[i] * sms && V > cluster * batch; ++i) cluster *= 2;
  const int span = ((V + cluster - 1) / cluster + 7) / 8 * 8;
  QSPEC_REQUIRE(V <= (1 << 24), QSPEC_ERR_UNSUPPORTED, "token_logprobs: a vocabulary of %d is too large", V);
  QSPEC_REQUIRE((long long)rows * cluster < (1ll << 31), QSPEC_ERR_UNSUPPORTED, "token_logprobs: %d rows are too many for one call", rows);
  const Args a{logits, row_stride, tokens, logprobs, entropy, ranks, top_logprobs, top_tokens, V, span, top, c};
  auto run = [&](auto kern) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    QSPEC_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    QSPEC_CHECK_LAUNCH(1);
    return QSPEC_OK;
  };
#define QSPEC_LOGPROB(T)                                                                                                                                         \
  (cluster == 8 ? run(token_logprobs_kernel<T, 8>) : cluster == 4 ? run(token_logprobs_kernel<T, 4>)                                                            \
                                                                  : cluster == 2 ? run(token_logprobs_kernel<T, 2>) : run(token_logprobs_kernel<T, 1>))
  return dtype == QSPEC_DTYPE_F32 ? QSPEC_LOGPROB(float) : dtype == QSPEC_DTYPE_BF16 ? QSPEC_LOGPROB(__nv_bfloat16) : QSPEC_LOGPROB(__half);
#undef QSPEC_LOGPROB
}
