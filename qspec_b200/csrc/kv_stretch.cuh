// How the attention over a paged cache is spread over the GPU, whatever the cache's format, and how its parts are joined (kv8_attention.cu, kv4_attention.cu).
//
// Work: (request, head, row tile) items of units of 32 keys, laid end to end and cut into equal stretches, one per CTA: lengths that
// differ cost nothing, one long request uses every SM. Inside a stretch unit i is warp i % WARPS's. Every warp keeps a softmax of its own (maximum, sum and
// sums of values in registers) over the units of an item that it took; they are joined through shared memory at the item's end and, where a stretch
// ends inside an item, through the workspace: the CTA that comes last adds the parts up in their order, so that results do not depend on which it is.
#pragma once
#include "kv8_common.cuh"
#include <type_traits>

namespace qspec {
namespace kv8 {

constexpr int UNIT = 32, ROWS = 16;               // keys of a unit; rows of a tile (or, where a kernel says so, eight: TR)
constexpr float NONE = -INFINITY;
template <int D, int TR = ROWS> constexpr int PART = TR * 2 + TR * D;   // floats of a part: maxima, sums, sums of values

// The step's requests, as all kernels of a call see them.
struct Step {
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep;
  unsigned share;                                // to_prompt_form()'s; 0: there is no prompt form in this call
};

#ifdef __CUDACC__
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }

// A request's part of the work.
struct Req {
  int first, n, keys, tiles, units;               // first row of q, tokens, keys, row tiles, units of an item
  __device__ __forceinline__ long long total(int G) const { return (long long)tiles * G * units; }
};
template <int TR = ROWS>
__device__ __forceinline__ Req request(const Step& a, int b, unsigned long long work) {
  Req r;
  r.first = min(max(a.q_start[b], 0), a.ntok);
  r.n = max(min(a.q_start[b + 1], a.ntok) - r.first, 0);
  r.keys = max(a.kv_len[b], 0);
  const long long rows = (long long)r.n * a.rep;
  r.tiles = to_prompt_form(r.n, r.keys, a.rep, a.share, work) ? 0 : (int)((rows + TR - 1) / TR);
  // A request without keys has a unit that shows its rows none. Behind the table's last page is nothing but a page that there is not: one unit shows that.
  r.units = max((min(r.keys, keys_at_most(a.width, a.pshift)) + UNIT - 1) / UNIT, 1);
  return r;
}

// Where a unit lies: request, head and row tile (tiles inside heads), unit of that item.
struct Place {
  int b, g, tile, u;
  Req r;
  template <int TR = ROWS>
  __device__ __forceinline__ void forward(const Step& a, unsigned long long work, int steps) {
    u += steps;
    while (b < a.nreq && u >= r.units) {
      u -= r.units;
      if (++tile < r.tiles) continue;
      tile = 0;
      if (++g < a.G) continue;
      g = 0;
      do { if (++b >= a.nreq) return; r = request<TR>(a, b, work); } while (r.tiles == 0);
    }
  }
};

// The page that lane i has of the unit at `p`: its ith, of UNIT / P (at least one); -1: one behind the last key; BROKEN: an entry that is no page of the cache.
constexpr int BROKEN = -2;
__device__ __forceinline__ int unit_page(const Step& a, const Place& p, int lane) {
  const int n = max(UNIT >> a.pshift, 1), at = ((p.u * UNIT) >> a.pshift) + lane;
  if (p.b >= a.nreq || lane >= n || (at << a.pshift) >= p.r.keys) return -1;
  const int page = at < a.width ? a.table[(size_t)p.b * a.width + at] : BROKEN;
  return (unsigned)page < (unsigned)a.npages ? page : BROKEN;
}
// A unit whose pages are known: where its codes are (bytes from the first page's, the same for keys and values; each lane its page's) and its keys.
struct Unit {
  long long at;                                   // -1: no such page
  int key0, keys;
};
// This CTA's stretch of the work, of WARPS warps, in a grid of GRID_MOST CTAs at most. All threads of the CTA call it; its barriers are the CTA's. false: there is nothing for this CTA.
template <int WARPS> struct Shared {
  long long sum[WARPS];
  int place[4], items[WARPS], ctas[6][WARPS];
  Req req;
  int last;
};
struct Stretch {
  Place cur;                                                // the segment that all warps are in: (the rest of) one item
  bool whole;                                               // every item has CTAs of its own
  int share, todo;                                          // units that a CTA of such an item takes; units of this stretch
  long long begin, per;
};
__device__ __forceinline__ long long quotient(long long a, long long b) {   // of numbers that are not negative (in 32 bits where they fit: five times as fast)
  return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
template <int WARPS, int GRID_MOST, int TR = ROWS>
__device__ __forceinline__ bool find_stretch(const Step& a, Shared<WARPS>& s, unsigned long long& work_out, Stretch& out) {
  constexpr int THREADS = WARPS * 32, MIN_UNITS = WARPS;   // units of a stretch: one for each warp
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Up to 32 requests every warp looks for itself, without barriers (16 requests of 4 tokens after 2000 keys in 4 bits 29.7 -> 28.4 us).
  const bool few = a.nreq <= 32;
  const int lookers = few ? 32 : THREADS, per_thread = (a.nreq + lookers - 1) / lookers, b0 = (few ? lane : tid) * per_thread;
  const int requests = max(min(per_thread, a.nreq - b0), 0);
  unsigned long long work = 0;                              // that requests with rows enough for the prompt form ask for
  if (a.share) {
    for (int i = 0; i < requests; ++i) {
      const Req r = request<TR>(a, b0 + i, 0);
      work += prompt_work(r.n, r.keys, a.rep, a.G);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    if (!few) {
      if (lane == 0) s.sum[warp] = (long long)work;
      __syncthreads();
      work = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) work += (unsigned long long)s.sum[w];
      __syncthreads();
    }
  }
  Req only{0, 0, 0, 0, 1};
  if (per_thread == 1 && b0 < a.nreq) only = request<TR>(a, b0, work);
  auto req = [&](int i) { return per_thread == 1 ? only : request<TR>(a, b0 + i, work); };
  long long before, total;                                  // of the requests of the threads in front of this one, and of all
  auto scan = [&](long long mine) {
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += w;
    }
    before = incl - mine;
    if (few) { total = __shfl_sync(0xffffffffu, incl, 31); return; }
    if (lane == 31) s.sum[warp] = incl;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += s.sum[w];
      total += s.sum[w];
    }
  };
  long long mine = 0;
  int items = 0;
  for (int i = 0; i < requests; ++i) {
    const Req r = req(i);
    mine += r.total(a.G);
    items = min(items + (int)min((long long)r.tiles * a.G, (long long)GRID_MOST + 1), GRID_MOST + 1);
  }
  items = __reduce_add_sync(0xffffffffu, items);
  if (!few && lane == 0) s.items[warp] = items;
  scan(mine);
  const int grid = gridDim.x;
  long long per = max(total <= 0x7fffffff ? (long long)(((int)total - 1) / grid + 1) : (total + grid - 1) / grid, (long long)MIN_UNITS);
  // A stretch may lie over the end of an item: then the CTA joins and stores twice. With few items each gets CTAs of its own, as long as that makes no
  // stretch much longer (by a quarter and eight units at most): 4 requests of 900, 32 / 8 heads, one token each 17.0 -> 12.1 us.
  bool whole = false;
  if (!few) {
    items = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) items += s.items[w];
  }
  if (items <= grid && per < (1 << 24)) {
    constexpr int TRIES = 6;                                // lengths that are looked at
    auto length = [&](int c) { const int p = (int)per; return c == 0 ? p : c == 1 ? p + 1 : c == 2 ? p + p / 32 + 1 : c == 3 ? p + p / 16 + 2 : c == 4 ? p + p / 8 + 4 : p + p / 4 + 8; };
    int n[TRIES] = {0, 0, 0, 0, 0, 0};
    for (int i = 0; i < requests; ++i) {
      const Req r = req(i);
#pragma unroll
      for (int c = 0; c < TRIES; ++c)
        n[c] = min(n[c] + (int)min((long long)r.tiles * a.G * ((r.units - 1) / length(c) + 1), (long long)GRID_MOST + 1), GRID_MOST + 1);
    }
#pragma unroll
    for (int c = 0; c < TRIES; ++c) {
      n[c] = __reduce_add_sync(0xffffffffu, n[c]);
      if (!few && lane == 0) s.ctas[c][warp] = n[c];
    }
    if (!few) __syncthreads();
    int len = 0;
#pragma unroll
    for (int c = TRIES - 1; c >= 0; --c) {
      int sum = n[c];
      if (!few) {
        sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += s.ctas[c][w];
      }
      if (sum <= grid) len = length(c);
    }
    if (len) {
      whole = true;
      per = len;
      mine = 0;                                             // CTAs of this thread's requests
      for (int i = 0; i < requests; ++i) {
        const Req r = req(i);
        mine += (long long)r.tiles * a.G * ((r.units - 1) / len + 1);
      }
      scan(mine);
    }
  }
  // (an item's units are spread evenly over its CTAs)
  const long long begin = whole ? blockIdx.x : per * blockIdx.x;
  if (begin >= total) return false;
  int place[4] = {-1, 0, 0, 1};                             // request, item of it (head * tiles + tile), CTA of the item or unit, how many of those
  Req found{0, 0, 0, 0, 1};
  if (begin >= before && begin < before + mine) {
    long long at = before;
    for (int i = 0; i < requests; ++i) {
      const Req r = req(i);
      const int each = whole ? (r.units - 1) / (int)per + 1 : r.units;
      const long long n = (long long)r.tiles * a.G * each;
      if (begin < at + n) {
        place[0] = b0 + i;
        place[1] = (int)quotient(begin - at, each);
        place[2] = (int)(begin - at - (long long)place[1] * each);
        place[3] = each;
        found = r;
        break;
      }
      at += n;
    }
  }
  if (few) {
    const int who = __ffs(__ballot_sync(0xffffffffu, place[0] >= 0)) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) place[i] = __shfl_sync(0xffffffffu, place[i], who);
    found = {__shfl_sync(0xffffffffu, found.first, who), __shfl_sync(0xffffffffu, found.n, who), __shfl_sync(0xffffffffu, found.keys, who), __shfl_sync(0xffffffffu, found.tiles, who),
             __shfl_sync(0xffffffffu, found.units, who)};
  } else {
    if (place[0] >= 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s.place[i] = place[i];
      s.req = found;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) place[i] = s.place[i];
    found = s.req;
  }
  Place cur;
  cur.b = place[0];
  cur.r = found;
  cur.g = place[1] / cur.r.tiles;
  cur.tile = place[1] - cur.g * cur.r.tiles;
  const int share = whole ? (cur.r.units - 1) / place[3] + 1 : 0;
  cur.u = whole ? min(place[2] * share, cur.r.units) : place[2];
  const int todo = whole ? min(share, cur.r.units - cur.u) : (int)(min(begin + per, total) - begin);
  work_out = work;
  out = Stretch{cur, whole, share, todo, begin, per};
  return todo > 0;                                          // (a last share of none)
}

// Where rows go, and what CTAs leave for each other.
struct Out {
  void* out; long long out_ts; int out_hs;
  int* counters; float* parts;
};
// The warps' sums of an item's segment (units cur.u .. cur.u + seg_n - 1, from the stretch's unit seg0 on) together: s_ml [warp][maximum, sum][TR], s_o
// [warp][TR][LD] sums of values, written by the warps (not by one that saw nothing); to the rows, or, of a part of an item, into the workspace.
template <bool BF16, int D, int LD, int WARPS, int TR = ROWS>
__device__ __forceinline__ void finish_segment(const Step& a, const Out& o, const Stretch& w0, const Place& cur, int seg0, int seg_n, float* s_ml, float* s_o, Shared<WARPS>& s) {
  using T = typename Elem16<BF16>::T;
  constexpr int THREADS = WARPS * 32;
  const int tid = threadIdx.x;
  __syncthreads();
  constexpr int PER_ROW = THREADS / TR < D / 4 ? THREADS / TR : D / 4, PIECES = D / 4 / PER_ROW;   // threads of a row, float4 of a thread
  static_assert(TR * PER_ROW == THREADS, "every thread has a row");
  const int jr = tid / PER_ROW, col = tid % PER_ROW;
  float mm = NONE, ll = 0.f;
  float4 oo[PIECES];
#pragma unroll
  for (int c = 0; c < PIECES; ++c) oo[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  // the warps' maxima and sums first: loads that wait for none before them
  float mw[WARPS], lw[WARPS];
#pragma unroll
  for (int w = 0; w < WARPS; ++w) { mw[w] = s_ml[(w * 2) * TR + jr]; lw[w] = s_ml[(w * 2 + 1) * TR + jr]; }
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    // (a part that saw nothing has no sums; one that saw NaN has a sum that is not zero)
    const bool none = mw[w] == NONE && lw[w] == 0.f;
    const float mn = fmaxf(mm, mw[w]), f = mm == NONE ? 0.f : exp2_fast(mm - mn), h = mw[w] == NONE ? 1.f : exp2_fast(mw[w] - mn);
    if (!none) { mm = mn; ll = ll * f + lw[w] * h; }
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const float4 p = *reinterpret_cast<const float4*>(s_o + (w * TR + jr) * LD + (col + PER_ROW * c) * 4);
      if (!none) { oo[c].x = oo[c].x * f + p.x * h; oo[c].y = oo[c].y * f + p.y * h; oo[c].z = oo[c].z * f + p.z * h; oo[c].w = oo[c].w * f + p.w * h; }
    }
  }
  auto store_piece = [&](int r, int at, const float4& p, float f) {   // columns at .. at + 3 of the tile's row r
    const int rr = cur.tile * TR + r, tok = rr / a.rep;
    uint2 w;
    if (BF16) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(p.x * f, p.y * f), y = __floats2bfloat162_rn(p.z * f, p.w * f);
      w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    } else {
      w = make_uint2(half_pair(p.x * f, p.y * f), half_pair(p.z * f, p.w * f));
    }
    *reinterpret_cast<uint2*>((T*)o.out + (size_t)(cur.r.first + tok) * o.out_ts + (size_t)(cur.g * a.rep + rr - tok * a.rep) * o.out_hs + at) = w;
  };
  const bool starts = cur.u == 0, ends = cur.u + seg_n == cur.r.units;
  if (starts && ends) {
    if (cur.tile * TR + jr < cur.r.n * a.rep) {
      const float f = ll == 0.f ? 0.f : __fdiv_rn(WEIGHT_UNIT, ll);   // (no key: zeros)
#pragma unroll
      for (int c = 0; c < PIECES; ++c) store_piece(jr, (col + PER_ROW * c) * 4, oo[c], f);
    }
  } else {
    // ---- a part of an item: into the workspace; the item's last CTA to come adds all of them up, first part first
    const long long item0 = w0.begin + seg0 - cur.u, item1 = item0 + cur.r.units;
    const int c0 = w0.whole ? (int)blockIdx.x - cur.u / w0.share : (int)quotient(item0, w0.per), c1 = w0.whole ? c0 + (cur.r.units - 1) / w0.share : (int)quotient(item1 - 1, w0.per);
    float* part = o.parts + (size_t)(2 * blockIdx.x + (starts ? 1 : 0)) * PART<D, TR>;
    if (col == 0) { part[jr] = mm; part[TR + jr] = ll; }
#pragma unroll
    for (int c = 0; c < PIECES; ++c) *reinterpret_cast<float4*>(part + 2 * TR + jr * D + (col + PER_ROW * c) * 4) = oo[c];
    __syncthreads();
    if (tid == 0) {
      __threadfence();                                    // (of what the whole CTA has stored: the barrier is in front of it)
      const int n = c1 - c0 + 1, old = atomicAdd(o.counters + c0, 1);
      s.last = old == n - 1;
      if (old == n - 1) o.counters[c0] = 0;               // for the next call
    }
    __syncthreads();
    if (s.last) {
      // All maxima and sums first (eight threads a row), which gives every part its factor, then the sums of values: loads that wait for none before them.
      __threadfence();
      const int n = c1 - c0 + 1;
      auto from = [&](int i) { return o.parts + (size_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * PART<D, TR>; };
      float* const factor = s_o;                          // [part][row]: the sums on their way between warps have been read
      mm = NONE;
      ll = 0.f;
      for (int i0 = col; i0 < n; i0 += 8 * PER_ROW) {
        float mp[8], lp[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = i0 + k * PER_ROW;
          mp[k] = i < n ? __ldcg(from(i) + jr) : NONE;
          lp[k] = i < n ? __ldcg(from(i) + TR + jr) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool none = mp[k] == NONE;                // nothing seen, or (a sum that is not zero) no number
          const float mn = fmaxf(mm, mp[k]);
          ll = (mm == NONE ? ll : ll * exp2_fast(mm - mn)) + (none ? lp[k] : lp[k] * exp2_fast(mp[k] - mn));
          mm = mn;
          if (i0 + k * PER_ROW < n) factor[(i0 + k * PER_ROW) * TR + jr] = none && lp[k] != 0.f ? INFINITY : mp[k];
        }
      }
      const float own = mm;
#pragma unroll
      for (int x = PER_ROW / 2; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
      if (own != NONE) ll *= exp2_fast(own - mm);
#pragma unroll
      for (int x = PER_ROW / 2; x > 0; x >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, x);
      for (int i = col; i < n; i += PER_ROW) {
        const float f = factor[i * TR + jr];
        factor[i * TR + jr] = f == NONE ? 0.f : f == INFINITY ? 1.f : exp2_fast(f - mm);
      }
      if (col == 0) factor[n * TR + jr] = ll == 0.f ? 0.f : __fdiv_rn(WEIGHT_UNIT, ll);   // (no key: zeros)
      __syncthreads();
      const int rows = min(cur.r.n * a.rep - cur.tile * TR, TR);
      auto add = [&](auto most) {                           // parts of which loads are under way
        constexpr int MOST = decltype(most)::value;
        for (int x = tid; x < rows * (D / 4); x += THREADS) {
          const int r = x / (D / 4), at = x % (D / 4) * 4;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int i0 = 0; i0 < n; i0 += MOST) {
            float4 v[MOST];
#pragma unroll
            for (int k = 0; k < MOST; ++k)
              v[k] = i0 + k < n ? __ldcg(reinterpret_cast<const float4*>(from(i0 + k) + 2 * TR + r * D + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < MOST; ++k) {
              const float f = i0 + k < n ? factor[(i0 + k) * TR + r] : 0.f;
              sum.x = fmaf(v[k].x, f, sum.x); sum.y = fmaf(v[k].y, f, sum.y); sum.z = fmaf(v[k].z, f, sum.z); sum.w = fmaf(v[k].w, f, sum.w);
            }
          }
          store_piece(r, at, sum, factor[n * TR + r]);
        }
      };
      if (n <= 4) add(std::integral_constant<int, 4>{}); else add(std::integral_constant<int, 32>{});
    }
  }
}
#endif

}  // namespace kv8
}  // namespace qspec
