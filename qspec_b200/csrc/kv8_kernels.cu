// A key/value cache in pages and in 8 bits: the page plan of a step, the writer of the cache and its inverse. The attention that reads it is in
// kv8_attention.cu.
//
// Cache of a layer: codes int8 [pages, G, P, D] (a page's rows of one head are P * D bytes in a row) and scales float32 [pages, G] for keys and for
// values; a code c stands for c * scale. P tokens a page: a power of two from 16 to 128. A slot is page * P + row.
#include "kv8_common.cuh"
#include <type_traits>

namespace qspec {
namespace kv8 {

// ---- pages and slots of a step ----------------------------------------------------------------------------------------------------
// Nothing here is of size: three prefix sums over the requests (tokens, pages wanted, pages given back), then one thread per token, per new table entry
// and per page that goes back. Every CTA makes the sums for itself (4096 requests are 48 KB of reads from L2) and takes its share of the rest, so
// that no CTA waits for another; nothing that a call reads is written by it (table entries from `held` on and list entries from n_free on mean nothing to
// the state that came in), so that the order of the CTAs does not matter and a call can be made again.
constexpr int PLAN_REQUESTS = 4096, PLAN_EACH = 4, PLAN_SMALL = 256, PLAN_LARGE = PLAN_REQUESTS / PLAN_EACH;   // requests; of a thread; threads of a CTA

struct PlanArgs {
  const int *lengths, *counts;
  int* table;
  int* free_pages;
  const int* state;
  int *q_start, *kv_len, *positions, *seq_ids, *slots, *state_out;
  int n, width, npages, pshift, ntok;
  int top;                                         // the largest power of two below n, or 1
};

// index of the last entry of the ascending s[0 .. n - 1] that is <= x (s[0] <= x)
__device__ __forceinline__ int last_at_most(const int* s, int n, int top, int x) {
  int lo = 0;
  for (int step = top; step; step >>= 1)
    if (lo + step < n && s[lo + step] <= x) lo += step;
  return lo;
}

template <int PLAN_THREADS>
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PlanArgs a) {
  constexpr int PLAN_WARPS = PLAN_THREADS / 32;
  extern __shared__ int plan_smem[];
  int* s_tok = plan_smem;                         // first token of each request, in front of it [n + 1]
  int* s_need = s_tok + a.n + 1;                  // pages asked for before it [n + 1]
  int* s_back = s_need + a.n + 1;                 // pages given back before it [n + 1]
  int* s_len = s_back + a.n + 1;                  // tokens held, or -1 for a request that has no place for its tokens [n]
  int* s_held = s_len + a.n;                      // pages held [n]
  __shared__ int s_warp[3][32], s_refused[32], s_over;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_over = a.n;
  pdl_enter();
  const int n_free = min(max(a.state[a.n], 0), a.npages);
  int cnt[PLAN_EACH], len[PLAN_EACH], held[PLAN_EACH], need[PLAN_EACH];
  int sum[3] = {0, 0, 0};
#pragma unroll
  for (int e = 0; e < PLAN_EACH; ++e) {
    const int b = tid * PLAN_EACH + e;
    cnt[e] = len[e] = held[e] = need[e] = 0;
    if (b < a.n) {
      cnt[e] = a.counts[b];
      len[e] = a.lengths[b];
      held[e] = min(max(a.state[b], 0), a.width);
      if (cnt[e] > 0) {
        const long long want = ((long long)len[e] + cnt[e] + (1 << a.pshift) - 1) >> a.pshift;
        if (len[e] >= 0 && want <= a.width) need[e] = max((int)want - held[e], 0);
      }
    }
    // (a sum of tokens that passes the tokens there are room for says no more than that: it stays there)
    sum[0] = (int)min((long long)sum[0] + max(cnt[e], 0), (long long)a.ntok + 1);
    sum[1] += need[e];
    sum[2] += cnt[e] < 0 ? held[e] : 0;
  }
  int pre[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int v = sum[q];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = q ? v + w : (int)min((long long)v + w, (long long)a.ntok + 1);
    }
    pre[q] = v;
    if (lane == 31) s_warp[q][warp] = v;
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      int v = lane < PLAN_WARPS ? s_warp[q][lane] : 0;
#pragma unroll
      for (int o = 1; o < PLAN_WARPS; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = q ? v + w : (int)min((long long)v + w, (long long)a.ntok + 1);
      }
      if (lane < PLAN_WARPS) s_warp[q][lane] = v;
    }
  }
  __syncthreads();
  int at[3];                                       // sums in front of this thread's first request
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const int before = __shfl_up_sync(0xffffffffu, pre[q], 1), prev = warp ? s_warp[q][warp - 1] : 0;
    at[q] = prev + (lane ? before : 0);
    if (q == 0) at[q] = min(at[q], a.ntok + 1);
  }
  const int have = n_free + s_warp[2][PLAN_WARPS - 1];
  int refused = 0;
#pragma unroll
  for (int e = 0; e < PLAN_EACH; ++e) {
    const int b = tid * PLAN_EACH + e;
    if (b < a.n) {
      const int first = at[0], last = (int)min((long long)first + max(cnt[e], 0), (long long)a.ntok + 1);
      const bool ends = cnt[e] < 0;
      const bool fits = cnt[e] <= 0 || (len[e] >= 0 && ((((long long)len[e] + cnt[e] + (1 << a.pshift) - 1) >> a.pshift) <= a.width) && last <= a.ntok);
      const bool granted = !ends && fits && (need[e] == 0 || at[1] + need[e] <= have);
      s_tok[b] = min(first, a.ntok);
      if (cnt[e] > 0 && first <= a.ntok && last > a.ntok) s_over = b;   // the first whose tokens there is no room for
      s_need[b] = at[1];
      s_back[b] = at[2];
      s_len[b] = granted ? len[e] : -1;
      s_held[b] = held[e];
      if (blockIdx.x == 0) {
        a.q_start[b] = min(first, a.ntok);
        a.kv_len[b] = granted ? len[e] + cnt[e] : 0;
        a.state_out[b] = ends ? 0 : granted && need[e] ? held[e] + need[e] : held[e];
        refused += !granted && !ends;
      }
      if (b == a.n - 1) {
        s_tok[a.n] = min(last, a.ntok);
        s_need[a.n] = at[1] + need[e];
        s_back[a.n] = at[2] + (ends ? held[e] : 0);
        if (blockIdx.x == 0) a.q_start[a.n] = min(last, a.ntok);
      }
      at[0] = last;
      at[1] += need[e];
      at[2] += ends ? held[e] : 0;
    }
  }
  refused = __reduce_add_sync(0xffffffffu, refused);
  if (lane == 0) s_refused[warp] = refused;
  __syncthreads();

  // pages handed out: those of the requests that were granted are the first ones asked for. (What lies behind the last sum that fits was not granted.)
  const int total = s_need[a.n];
  int taken = total;
  if (total > have) {                              // the last request whose sum still fits
    int lo = 0, hi = a.n;                          // s_need[lo] <= have
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_need[mid] <= have) lo = mid; else hi = mid;
    }
    taken = s_need[lo];
  }
  taken = min(taken, s_need[s_over]);
  const int left = have - taken;
  const int step = gridDim.x * PLAN_THREADS, first = blockIdx.x * PLAN_THREADS + tid;
  // the nth page of those that have come back, and the nth page handed out
  auto returned = [&](int nth) {
    const int b = last_at_most(s_back, a.n, a.top, nth);
    return a.table[(size_t)b * a.width + (nth - s_back[b])];
  };
  auto page = [&](int nth) {
    const int src = have - 1 - nth;
    return src < n_free ? a.free_pages[src] : returned(src - n_free);
  };
  for (int i = first; i < taken; i += step) {
    const int b = last_at_most(s_need, a.n, a.top, i);
    a.table[(size_t)b * a.width + s_held[b] + (i - s_need[b])] = page(i);
  }
  for (int i = n_free + first; i < min(left, a.npages); i += step) a.free_pages[i] = returned(i - n_free);
  const int tokens = s_tok[a.n];
  for (int t = first; t < a.ntok; t += step) {
    int pos = -1, slot = -1, req = -1;
    if (t < tokens) {
      req = last_at_most(s_tok, a.n, a.top, t);
      const int l = s_len[req], h = s_held[req];
      if (l >= 0) {
        pos = l + (t - s_tok[req]);
        const int nth = pos >> a.pshift;
        const int pg = nth < h ? a.table[(size_t)req * a.width + nth] : page(s_need[req] + nth - h);
        if ((unsigned)pg < (unsigned)a.npages) slot = (pg << a.pshift) + (pos & ((1 << a.pshift) - 1));   // (an entry that is no page: no slot)
      }
    }
    a.positions[t] = pos;
    a.seq_ids[t] = req;
    a.slots[t] = slot;
  }
  if (blockIdx.x == 0 && warp == 0) {
    const int r = __reduce_add_sync(0xffffffffu, lane < PLAN_WARPS ? s_refused[lane] : 0);
    if (lane == 0) {
      a.state_out[a.n] = left;
      a.state_out[a.n + 1] = r;
    }
  }
}

// ---- rows into pages --------------------------------------------------------------------------------------------------------------
// A run (the consecutive tokens of one page) of up to SHORT tokens is one warp's per head, for keys and values each, a longer one a CTA's (a warp for each of
// these, too: a prompt of 4200 tokens, 40 / 8 heads, without its queries 25.5 us, so 11; all by a CTA: 1024 requests of a token each 44 us, so 12). Eight lanes
// a row, four rows of a warp at a time; a lane holds sixteen of its values, eight of each half, so that it has both of every pair that the rotation turns. The page's scale is the largest |x| of all rows: those that fit into registers stay there between the maximum and the codes, others are read
// again. A decode step's call is one load, a reduction and a store long: without barriers.
// Rotation and codes are evaluated with the roundings that their formulas have (no fused multiply-adds), so that the same codes come out of every
// implementation in float32.
struct AppendArgs {
  const void* qkv; long long ld;
  const void* cos_sin; int cos_rows;
  const int *positions, *slots;
  signed char *k, *v;
  float *ks, *vs;
  void* q; long long q_ts;
  int ntok, H, G, npages, pshift, block;          // block: tokens of a CTA
  int tshift;                                     // 2^tshift: block, or the next power of two
};
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;   // 2^-60
constexpr int APPEND_WARPS = 8, SHORT = 8;        // warps of a CTA; tokens of a run up to which it is one warp's

// the slot of token t, or -1 if it has none. Runs follow from slots alone: a token whose position the table of angles does not have is a row of its page's run for which
// nothing is written. (With such a token as an end, a page had two runs in a call, each with a scale of its own to write.)
__device__ __forceinline__ int slot_of(const AppendArgs& a, int t) {
  if (t < 0 || t >= a.ntok) return -1;
  const int s = a.slots[t];
  return s >= 0 && s < (a.npages << a.pshift) ? s : -1;
}
__device__ __forceinline__ bool has_angle(const AppendArgs& a, int t) { return (unsigned)a.positions[t] < (unsigned)a.cos_rows; }

// sixteen values of a row (token t, at position pos): x[0 .. 7] from column 8 c on, x[8 .. 15] the same of the second half
template <bool BF16, int D, bool TURN>
__device__ __forceinline__ void load_row(const AppendArgs& a, int t, int pos, int col, int c, float (&x)[16]) {
  using T = typename Elem16<BF16>::T;
  const T* row = (const T*)a.qkv + (size_t)t * a.ld + col + c * 8;
  float lo[8], hi[8];
  unpack8<BF16>(*reinterpret_cast<const uint4*>(row), lo);
  unpack8<BF16>(*reinterpret_cast<const uint4*>(row + D / 2), hi);
  if (TURN) {
    const T* tab = (const T*)a.cos_sin + (size_t)pos * D + c * 8;
    float cs[8], sn[8];
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab), cs);
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab + D / 2), sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) {                           // (not by pairs: mul.rn.f32x2 in front of add.rn.f32x2 became one multiply-add)
      x[e] = __fsub_rn(__fmul_rn(lo[e], cs[e]), __fmul_rn(hi[e], sn[e]));
      x[e + 8] = __fadd_rn(__fmul_rn(hi[e], cs[e]), __fmul_rn(lo[e], sn[e]));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) { x[e] = lo[e]; x[e + 8] = hi[e]; }
  }
}

__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  const float r = rintf(__fmul_rn(x, inv));
  return (uint32_t)(x == x ? (int)fminf(fmaxf(r, -127.f), 127.f) : 0) & 0xffu;
}

__device__ __forceinline__ float finite_max(float mx, const float (&x)[16]) {   // (what is not finite does not stretch the page's scale)
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float y = fabsf(x[e]);
    mx = fmaxf(mx, y < INFINITY ? y : 0.f);
  }
  return mx;
}
// The largest |x| so far, infinite as soon as one is not finite.
__device__ __forceinline__ float largest(float mx, const float (&x)[16]) {
  float z = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    mx = fmaxf(mx, fabsf(x[e]));
    z = fmaf(x[e], 0.f, z);
  }
  return z == 0.f ? mx : INFINITY;
}
// odd: the run has values that are not finite. Where it has none, rint(x / scale) is in the last byte of x / scale + 1.5 * 2^23.
template <int D>
__device__ __forceinline__ void store_codes(signed char* row, int c, const float (&x)[16], float inv, bool odd) {
  uint32_t w[4];
  if (odd) {
    w[0] = w[1] = w[2] = w[3] = 0u;
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e >> 2] |= code_of(x[e], inv) << (8 * (e & 3));
  } else {
    auto bits = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); };
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      w[e >> 2] = __byte_perm(__byte_perm(bits(x[e]), bits(x[e + 1]), 0x0040), __byte_perm(bits(x[e + 2]), bits(x[e + 3]), 0x0040), 0x5410);
  }
  *reinterpret_cast<uint2*>(row + c * 8) = make_uint2(w[0], w[1]);
  *reinterpret_cast<uint2*>(row + c * 8 + D / 2) = make_uint2(w[2], w[3]);
}
// the page's rows before the run onto its new scale: codes i, i + step, .. of sixteen each
__device__ __forceinline__ void rescale(signed char* rows, int pieces, int i, int step, float before, float after) {
  const float f = __fdiv_rn(before, after);
  for (; i < pieces; i += step) {
    uint4* at = reinterpret_cast<uint4*>(rows) + i;
    uint4 v = *at;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t o = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) o |= ((uint32_t)(int)rintf(__fmul_rn((float)(signed char)(w[q] >> (8 * e)), f)) & 0xffu) << (8 * e);
      w[q] = o;
    }
    *at = v;
  }
}
__device__ __forceinline__ float new_scale(float mx, float before) { return fmaxf(fmaxf(__fmul_rn(mx, 1.0f / 127.0f), before), SCALE_FLOOR); }

// How many tokens the run has that begins with token t, of slot s, where `known` of them are already: asked by a whole warp.
__device__ __forceinline__ int run_of(const AppendArgs& a, int t, int s, int known) {
  const int mask = (1 << a.pshift) - 1, lane = threadIdx.x & 31, most = mask + 1 - (s & mask);
  for (int n = known; n < most; n += 32) {
    const uint32_t out = ~__ballot_sync(0xffffffffu, n + lane < most && slot_of(a, t + n + lane) == s + n + lane);
    if (out) return n + __ffs(out) - 1;
  }
  return most;
}

// A run by WARPS warps (one, or all of the CTA's): four rows (of 128) a warp at a time, the first of them held in registers between the maximum and the codes.
template <bool BF16, int D, bool TURN, int WARPS>
__device__ __forceinline__ void write_run(const AppendArgs& a, int t0, int n, int slot, int g, int col, signed char* codes, float* scales, float* s_max) {
  constexpr int LANES = D / 16, ROWS = 32 / LANES, STEP = ROWS * WARPS;   // lanes of a row, rows of a warp, rows at a time
  const int lane = threadIdx.x & 31, warp = WARPS > 1 ? threadIdx.x >> 5 : 0, c = lane % LANES, r0 = warp * ROWS + lane / LANES;
  const int page = slot >> a.pshift, first = slot & ((1 << a.pshift) - 1);
  signed char* rows = codes + (((size_t)page * a.G + g) << a.pshift) * D;
  float* scale = scales + (size_t)page * a.G + g;
  const float before = first ? *scale : 0.f;
  float x[16];                                              // the first of this lane's rows
  auto load = [&](int r) {                                  // whether there is something to write
    if (r >= n) return false;
    const int pos = a.positions[t0 + r];
    const bool there = (unsigned)pos < (unsigned)a.cos_rows;   // (not waited for by the row's loads)
    load_row<BF16, D, TURN>(a, t0 + r, there ? pos : 0, col, c, x);
    return there;
  };
  auto over_all = [&](float mx) {                           // (and everyone has read the scale)
    mx = warp_xor_max(mx);
    if (WARPS > 1) {
      __syncthreads();
      if (lane == 0) s_max[warp] = mx;
      __syncthreads();
      mx = warp_xor_max(lane < WARPS ? s_max[lane] : 0.f);
    }
    return mx;
  };
  float mx = 0.f;
  for (int r = r0 + STEP; r < n; r += STEP)
    if (load(r)) mx = largest(mx, x);
  const bool there = load(r0);
  if (there) mx = largest(mx, x);
  mx = over_all(mx);
  const bool odd = mx == INFINITY;
  if (odd) {                                                // the largest of those that are finite
    mx = 0.f;
    for (int r = r0 + STEP; r < n; r += STEP)
      if (load(r)) mx = finite_max(mx, x);
    if (load(r0)) mx = finite_max(mx, x);
    mx = over_all(mx);
  }
  __syncwarp();
  const float after = new_scale(mx, before), inv = __frcp_rn(after);
  if (there) store_codes<D>(rows + (size_t)(first + r0) * D, c, x, inv, odd);
  for (int r = r0 + STEP; r < n; r += STEP)
    if (load(r)) store_codes<D>(rows + (size_t)(first + r) * D, c, x, inv, odd);
  if (first && after > before) rescale(rows, first * (D / 16), warp * 32 + lane, WARPS * 32, before, after);
  if (warp == 0 && lane == 0 && after != before) *scale = after;
}

// 2 G CTAs per block of tokens write the runs that begin in it: of long ones each all that belongs to a head and side, by all of its warps together; of short ones
// every warp what belongs to a run, head and side, the heads of a run next to each other. The CTAs behind them turn the block's queries.
template <bool BF16, int D>
__global__ void __launch_bounds__(APPEND_WARPS * 32, 4) kv8_append_kernel(const AppendArgs a) {
  using T = typename Elem16<BF16>::T;
  constexpr int LANES = D / 16, ROWS = 32 / LANES;
  __shared__ float s_max[APPEND_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.y * a.block, t1 = min(t0 + a.block, a.ntok);
  const int units = 2 * a.G;                                // CTAs in x that write pages
  pdl_enter();
  if ((int)blockIdx.x < units) {
    // slots from the token before this CTA's first on, two a lane: which begin a run, and where runs end as far as that shows
    const int sa = slot_of(a, t0 - 1 + lane), sb = slot_of(a, t0 + 31 + lane);
    const bool turned = t0 - 1 + lane >= 0 && t0 - 1 + lane < a.ntok && has_angle(a, t0 - 1 + lane);
    const int before = __shfl_up_sync(0xffffffffu, sa, 1), mask = (1 << a.pshift) - 1;
    const bool go_on = lane > 0 && sa >= 0 && (sa & mask) && before == sa - 1;          // token t0 - 1 + lane is in the run of the one before it
    const int last = __shfl_sync(0xffffffffu, sa, 31), before_b = __shfl_up_sync(0xffffffffu, sb, 1);
    const bool go_on_b = sb >= 0 && (sb & mask) && (lane ? before_b : last) == sb - 1;
    const uint64_t in_run = ((uint64_t)__ballot_sync(0xffffffffu, go_on) | (uint64_t)__ballot_sync(0xffffffffu, go_on_b) << 32) >> 1;   // bit i: token t0 + i
    const uint32_t begin = __ballot_sync(0xffffffffu, lane > 0 && t0 - 1 + lane < t1 && sa >= 0 && !go_on) >> 1;
    const uint32_t written = __ballot_sync(0xffffffffu, turned) >> 1;   // bit i: token t0 + i has an angle
    uint64_t more = in_run >> 1;                            // bit i: the SHORT tokens behind t0 + i are in its run
#pragma unroll
    for (int o = 1; o < SHORT; o <<= 1) more &= more >> o;
    auto write = [&](int i, int n, int u, auto warps) {     // the run of n tokens that begins with token t0 + i
      constexpr int W = decltype(warps)::value;
      int t = t0 + i, s = __shfl_sync(0xffffffffu, sa, i + 1);
      const int g = u >> 1;
      if (W > 1 && t + n >= t0 + 63) n = run_of(a, t, s, n);   // (it may be longer than that)
      if (!(written >> i & 1u)) {                           // (it begins with the first token that is written)
        do { ++t; ++s; --n; } while (n && !has_angle(a, t));
        if (!n) return;
      }
      if (u & 1) write_run<BF16, D, false, W>(a, t, n, s, g, (a.H + a.G + g) * D, a.v, a.vs, s_max);
      else write_run<BF16, D, true, W>(a, t, n, s, g, (a.H + g) * D, a.k, a.ks, s_max);
    };
    auto tokens = [&](int i) { return __ffsll((long long)~(in_run >> (i + 1))); };
    for (uint32_t left = begin & (uint32_t)more; left; left &= left - 1u) {
      const int i = __ffs(left) - 1;
      write(i, tokens(i), blockIdx.x, std::integral_constant<int, APPEND_WARPS>());
    }
    const uint32_t brief = begin & ~(uint32_t)more;
    const int rank = brief >> lane & 1u ? __popc(brief & ((1u << lane) - 1u)) : -1, all = __popc(brief) * units;
    for (int id = blockIdx.x * APPEND_WARPS + warp; id < all; id += units * APPEND_WARPS) {
      const int j = id / units, i = __ffs(__ballot_sync(0xffffffffu, rank == j)) - 1;
      write(i, tokens(i), id - j * units, std::integral_constant<int, 1>());
    }
  } else {
    // LANES lanes take a token and some of its heads, two under way at a time: one look at the position and the angles for all of them (row by row, with both
    // for each, a prompt of 4200 tokens took 26.2 us, so 24.3).
    const int c = lane % LANES, group = warp * ROWS + lane / LANES, t = t0 + (group & ((1 << a.tshift) - 1)), per_cta = (APPEND_WARPS * ROWS) >> a.tshift;
    const int p = t < t1 ? a.positions[t] : -1;
    if (p < 0 || p >= a.cos_rows) return;
    const T *row = (const T*)a.qkv + (size_t)t * a.ld + c * 8, *tab = (const T*)a.cos_sin + (size_t)p * D + c * 8;
    T* const to = (T*)a.q + (size_t)t * a.q_ts + c * 8;
    float cs[8], sn[8];
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab), cs);
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab + D / 2), sn);
    const int step = ((int)gridDim.x - units) * per_cta;
    for (int h0 = ((int)blockIdx.x - units) * per_cta + (group >> a.tshift); h0 < a.H; h0 += 2 * step) {
      uint4 lo[2], hi[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int h = min(h0 + k * step, a.H - 1);
        lo[k] = *reinterpret_cast<const uint4*>(row + h * D);
        hi[k] = *reinterpret_cast<const uint4*>(row + h * D + D / 2);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int h = h0 + k * step;
        if (h >= a.H) break;
        float x[8], y[8], o[8];
        unpack8<BF16>(lo[k], x);
        unpack8<BF16>(hi[k], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __fsub_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(y[e], sn[e]));
        *reinterpret_cast<uint4*>(to + h * D) = pack8<BF16>(o);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __fadd_rn(__fmul_rn(y[e], cs[e]), __fmul_rn(x[e], sn[e]));
        *reinterpret_cast<uint4*>(to + h * D + D / 2) = pack8<BF16>(o);
      }
    }
  }
}

// ---- rows back in 16 bits: out[i, g] = codes of slot i * their page's scale, keys and values. Eight values a thread; slots that are none give zeros.
template <bool BF16>
__global__ void __launch_bounds__(256) kv8_read_kernel(const signed char* k, const signed char* v, const float* ks, const float* vs, const int* slots, void* ko, void* vo,
                                                       unsigned chunks, int G, int dshift, int npages, int pshift) {
  using T = typename Elem16<BF16>::T;
  pdl_enter();
  const signed char* codes = blockIdx.y ? v : k;
  const float* scales = blockIdx.y ? vs : ks;
  T* out = (T*)(blockIdx.y ? vo : ko);
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < chunks; i += gridDim.x * 256) {
    const unsigned c = i & ((1u << (dshift - 3)) - 1u), row = i >> (dshift - 3);
    const int g = (int)(row % (unsigned)G);
    const int s = slots[row / (unsigned)G];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (s >= 0 && s < npages << pshift) {
      const int page = s >> pshift, r = s & ((1 << pshift) - 1);
      const uint2 w = *reinterpret_cast<const uint2*>(codes + (((((size_t)page * G + g) << pshift) + r) << dshift) + c * 8);
      const float f = scales[(size_t)page * G + g];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fmul_rn((float)(signed char)((e < 4 ? w.x : w.y) >> (8 * (e & 3))), f);
    }
    *reinterpret_cast<uint4*>(out + (size_t)i * 8) = pack8<BF16>(x);
  }
}

}  // namespace kv8
}  // namespace qspec

using namespace qspec;
using namespace qspec::kv8;

extern "C" int qspec_page_plan(const int* lengths, const int* counts, int* table, int* free_pages, const int* state, int requests, int width, int npages, int page_tokens,
                               int ntok, int* q_start, int* kv_len, int* positions, int* seq_ids, int* slots, int* state_out, void* stream) {
  QSPEC_REQUIRE(lengths && counts && table && free_pages && state && q_start && kv_len && state_out && (ntok == 0 || (positions && seq_ids && slots)), QSPEC_ERR_INVALID_ARG,
                "page_plan: null pointer");
  QSPEC_REQUIRE(requests >= 1 && requests <= PLAN_REQUESTS, QSPEC_ERR_UNSUPPORTED, "page_plan: 1 to %d requests, got %d", PLAN_REQUESTS, requests);
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "page_plan: pages of 16, 32, 64 or 128 tokens, got %d", page_tokens);
  QSPEC_REQUIRE(width >= 1 && width <= (1 << 18) && npages >= 1 && (long long)npages * page_tokens < (1ll << 31) && ntok >= 0 && ntok < (1 << 30), QSPEC_ERR_INVALID_ARG,
                "page_plan: width=%d pages=%d tokens=%d", width, npages, ntok);
  int top = 1;
  while (top * 2 < requests) top *= 2;
  const PlanArgs a{lengths, counts, table, free_pages, state, q_start, kv_len, positions, seq_ids, slots, state_out, requests, width, npages, page_shift(page_tokens), ntok, top};
  const size_t smem = (5 * (size_t)requests + 3) * sizeof(int);
  const bool large = requests > PLAN_SMALL * PLAN_EACH;
  static SmemLimit limit;
  if (large) QSPEC_CUDA(limit.raise(page_plan_kernel<PLAN_LARGE>, smem));
  const int threads = large ? PLAN_LARGE : PLAN_SMALL, grid = min(max((ntok + threads - 1) / threads, 1), 2 * max(sm_count(), 1));
  QSPEC_CUDA(launch_pdl(large ? page_plan_kernel<PLAN_LARGE> : page_plan_kernel<PLAN_SMALL>, dim3(grid), dim3(threads), smem, (cudaStream_t)stream, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}

static int check_cache(const char* who, const void* k, const void* v, const float* ks, const float* vs, int npages, int G, int page_tokens, int D) {
  QSPEC_REQUIRE(k && v && ks && vs, QSPEC_ERR_INVALID_ARG, "%s: null pointer", who);
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "%s: pages of 16, 32, 64 or 128 tokens, got %d", who, page_tokens);
  QSPEC_REQUIRE(D == 64 || D == 128, QSPEC_ERR_UNSUPPORTED, "%s: heads of 64 or 128, got %d", who, D);
  QSPEC_REQUIRE(npages >= 1 && G >= 1 && G <= 1024 && (long long)npages * page_tokens < (1ll << 31), QSPEC_ERR_INVALID_ARG, "%s: pages=%d kv heads=%d", who, npages, G);
  QSPEC_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, QSPEC_ERR_INVALID_ARG, "%s: codes must begin on a 16-byte boundary", who);
  return QSPEC_OK;
}

extern "C" int qspec_kv8_append(const void* qkv, long long ld, const void* cos_sin, int cos_rows, const int* positions, const int* slots, void* k, void* v, float* ks,
                                float* vs, void* q_out, long long q_tok_stride, int ntok, int H, int G, int D, int npages, int page_tokens, int dtype, void* stream) {
  if (int rc = check_cache("kv8_append", k, v, ks, vs, npages, G, page_tokens, D)) return rc;
  if (ntok == 0) return QSPEC_OK;
  QSPEC_REQUIRE(qkv && cos_sin && positions && slots, QSPEC_ERR_INVALID_ARG, "kv8_append: null pointer");
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv8_append: float16 or bfloat16 rows");
  QSPEC_REQUIRE(ntok > 0 && ntok < (1 << 30) && H >= 1 && H <= 4096 && cos_rows >= 1, QSPEC_ERR_INVALID_ARG, "kv8_append: tokens=%d heads=%d table rows=%d", ntok, H, cos_rows);
  QSPEC_REQUIRE(ld >= (long long)(H + 2 * G) * D && ld % 8 == 0 && (!q_out || (q_tok_stride >= (long long)H * D && q_tok_stride % 8 == 0)) && ((uintptr_t)qkv & 15) == 0 &&
                    ((uintptr_t)cos_sin & 15) == 0 && ((uintptr_t)q_out & 15) == 0,
                QSPEC_ERR_INVALID_ARG, "kv8_append: rows must lie on 16-byte boundaries (ld=%lld)", ld);
  AppendArgs a{qkv, ld, cos_sin, cos_rows, positions, slots, (signed char*)k, (signed char*)v, ks, vs, q_out, q_tok_stride, ntok, H, G, npages, page_shift(page_tokens), 1, 0};
  // Small blocks put more CTAs on a call with few tokens, large ones have fewer that find nothing to begin (32 / 8 heads of 128, pages of 16, us with blocks of 8, 16
  // and 31: 64 requests of a token 3.0, 3.8, 5.9; 200 of 6 tokens 10.5, 9.1, 8.5; one prompt of 256 3.8, 4.3, 5.2; of 512 5.6, 5.2, 5.7; of 4200 35.8, 30.6, 29.1).
  a.block = ntok <= 256 ? 8 : ntok <= 1024 ? 16 : 31;       // (31: with the token before them one a lane)
  a.tshift = ntok <= 256 ? 3 : ntok <= 1024 ? 4 : 5;
  const int heads = ((APPEND_WARPS * 32 * 16 / D) >> a.tshift) * (ntok <= 256 ? 2 : 4);   // that a CTA turns of every token (that prompt with 2: 25.7, 8: 24.8)
  // (the parts of a block of tokens side by side: page writers wait, queries stream)
  const dim3 grid(2 * G + (q_out ? (H + heads - 1) / heads : 0), (ntok + a.block - 1) / a.block);
  QSPEC_REQUIRE(grid.y <= 65535, QSPEC_ERR_UNSUPPORTED, "kv8_append: %d tokens are too many for one call", ntok);
  auto kern = dtype == QSPEC_DTYPE_F16 ? (D == 128 ? kv8_append_kernel<false, 128> : kv8_append_kernel<false, 64>)
                                       : (D == 128 ? kv8_append_kernel<true, 128> : kv8_append_kernel<true, 64>);
  QSPEC_CUDA(launch_pdl(kern, grid, dim3(APPEND_WARPS * 32), 0, (cudaStream_t)stream, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}

extern "C" int qspec_kv8_read(const void* k, const void* v, const float* ks, const float* vs, const int* slots, void* k_out, void* v_out, int rows, int G, int D, int npages,
                              int page_tokens, int dtype, void* stream) {
  if (int rc = check_cache("kv8_read", k, v, ks, vs, npages, G, page_tokens, D)) return rc;
  if (rows == 0) return QSPEC_OK;
  QSPEC_REQUIRE(rows > 0 && slots && k_out && v_out, QSPEC_ERR_INVALID_ARG, "kv8_read: null pointer or rows=%d", rows);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv8_read: float16 or bfloat16 rows");
  QSPEC_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0, QSPEC_ERR_INVALID_ARG, "kv8_read: rows must lie on 16-byte boundaries");
  const long long chunks = (long long)rows * G * (D / 8);
  QSPEC_REQUIRE(chunks < (1ll << 31), QSPEC_ERR_UNSUPPORTED, "kv8_read: %d rows are too many for one call", rows);
  const int grid = (int)std::min<long long>((chunks + 255) / 256, (long long)max(sm_count(), 1) * 8);
  auto kern = dtype == QSPEC_DTYPE_F16 ? kv8_read_kernel<false> : kv8_read_kernel<true>;
  QSPEC_CUDA(launch_pdl(kern, dim3(grid, 2), dim3(256), 0, (cudaStream_t)stream, (const signed char*)k, (const signed char*)v, ks, vs, slots, k_out, v_out, (unsigned)chunks, G,
                        D == 128 ? 7 : 6, npages, page_shift(page_tokens)));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}
