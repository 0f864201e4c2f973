// Softmax attention over a key/value cache in pages and in 8 bits (its layout: kv8_kernels.cu). Token i of the n that request b has in the step stands at
// position kv_len[b] - n + i and sees the keys up to its own position.
//
// A row is a (token, query head of a group) pair; 16 rows of one key/value head are a tile of mma.sync.m16n8k16, so that the heads of a group and the
// tokens that verify a draft share every key that is read. What bounds it at these row counts is the cache: 2 D bytes a key and head.
//
// Work: (request, head, row tile) items of ceil(kv_len / 64) units of 64 keys, laid end to end and cut into equal stretches, one per CTA: lengths that
// differ cost nothing, one long request uses every SM. Inside a stretch unit i is warp i % 8's. Every warp keeps a softmax of its own (maximum, sum and
// sums of values in registers) over the units of an item that it took; they are joined through shared memory at the item's end and, where a stretch
// ends inside an item, through the workspace: the CTA that comes last adds the parts up in their order, so that results do not depend on which it is.
//
// Codes go from global memory into shared memory (16 bytes a lane, asynchronously, one unit of keys and one of values per warp) and from there into
// registers as the product's operands. The order of the sum over a head's dimensions is free, so that a lane's 16 bytes of a key are its operands of four products,
// and the queries are loaded in the same order; values need their bytes of two keys interleaved (one byte permutation for two).
//   keys: the byte c + 128 alone is the float16 (c + 128) 2^-24, a subnormal number, which the tensor cores take exactly: no arithmetic but the byte's
//   place. What the 128 adds to a score is the same for all keys, 128 times the row's sum, and is where the sums begin (from the other side).
//   values: the byte behind 0x64 is the float16 1152 + c, and one subtraction makes it c. (Sums over values must not carry the 128: over many keys they
//   cancel, and what the products cut off at the accumulator's last bit would be of the size of what is left.)
//
// bfloat16 queries are multiplied by a power of two per row that brings their largest value to 2^14 .. 2^15 and are float16 from there on, exactly. A key's scale
// multiplies its scores in float32. A value's scale v goes into the exponent: the weights 2^(s + log2 v - m) lie below 2^8 whatever the scales are and are
// rounded to float16 (2^-11 relative) for the product with the codes; the denominator is the sum of the unrounded weights / v.
#include "kv8_common.cuh"

namespace qspec {
namespace kv8 {

constexpr int WARPS = 8, THREADS = WARPS * 32, UNIT = 64, ROWS = 16;
constexpr int MIN_UNITS = 8;                     // of a stretch: one for each warp
constexpr int O_LD = 144;                        // floats of a row of sums on its way between warps (16 modulo 32: eight lanes' pieces in eight banks each)
constexpr float NONE = -INFINITY;

struct AttArgs {
  const void* q; long long q_ts; int q_hs;
  const signed char *k, *v;
  const float *ks, *vs;
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep, max_rows;   // max_rows: requests with more rows than that are another kernel's
  float scale2;                                  // scale * log2(e)
  void* out; long long out_ts; int out_hs;
  int* counters; float* parts;
};

template <int D> struct Smem {
  static constexpr int BUF = UNIT * D;                                  // one unit's keys or values
  static constexpr size_t RING = (size_t)WARPS * 2 * BUF;
  static constexpr size_t Q = 2 * ROWS * D * 2;
  static constexpr size_t O = (size_t)WARPS * ROWS * O_LD * 4;
  static constexpr size_t ML = (size_t)WARPS * ROWS * 2 * 4;
  static constexpr size_t TOTAL = RING + Q + O + ML;
};
template <int D> constexpr int PART = ROWS * 2 + ROWS * D;   // floats of a part: maxima, sums, sums of values

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a scale; one that is zero or next to nothing, or no number, counts as 2^-100
__device__ __forceinline__ float positive(float x) { return x >= 7.888609052210118e-31f ? x : 7.888609052210118e-31f; }
// two codes (bytes + 128, chosen by sel from w) as exact float16
__device__ __forceinline__ uint32_t codes16(uint32_t w, uint32_t sel) {
  const uint32_t m = __byte_perm(w, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));   // 1152
  return *reinterpret_cast<const uint32_t*>(&r);
}
// two codes as float16 without the subtraction: c + 128 in units of 2^-24, the smallest float16
__device__ __forceinline__ uint32_t codes_tiny(uint32_t w, uint32_t sel) { return __byte_perm(w, 0u, sel); }
__device__ __forceinline__ uint32_t half_pair(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }

// A request's part of the work.
struct Req {
  int first, n, keys, tiles, units;               // first row of q, tokens, keys, row tiles, units of an item
  __device__ __forceinline__ long long total(int G) const { return (long long)tiles * G * units; }
};
__device__ __forceinline__ Req request(const AttArgs& a, int b) {
  Req r;
  r.first = min(max(a.q_start[b], 0), a.ntok);
  r.n = max(min(a.q_start[b + 1], a.ntok) - r.first, 0);
  r.keys = max(a.kv_len[b], 0);
  const long long rows = (long long)r.n * a.rep;
  r.tiles = rows <= a.max_rows ? (int)((rows + ROWS - 1) / ROWS) : 0;
  r.units = max((r.keys + UNIT - 1) / UNIT, 1);   // a request without keys has a unit that shows its rows none
  return r;
}

// Where a unit lies: request, head and row tile (tiles inside heads), unit of that item.
struct Place {
  int b, g, tile, u;
  Req r;
  __device__ __forceinline__ void forward(const AttArgs& a, int steps) {
    u += steps;
    while (b < a.nreq && u >= r.units) {
      u -= r.units;
      if (++tile < r.tiles) continue;
      tile = 0;
      if (++g < a.G) continue;
      g = 0;
      do { if (++b >= a.nreq) return; r = request(a, b); } while (r.tiles == 0);
    }
  }
};

template <int D>
__device__ __forceinline__ uint32_t k_chunk(int row, int c) { return (uint32_t)(row * D + ((D == 128 ? c ^ ((row & 1) << 2) : c) << 4)); }
template <int D>
__device__ __forceinline__ uint32_t v_chunk(int row, int c) { return (uint32_t)(row * D + ((D == 128 ? c ^ (row & 6) : c ^ ((row >> 1) & 3)) << 4)); }

// The page that lane i has of the unit at `p`: its ith, of 64 / P (at least one); -1: one behind the last key; BROKEN: an entry that is no page of the cache.
constexpr int BROKEN = -2;
__device__ __forceinline__ int unit_page(const AttArgs& a, const Place& p, int lane) {
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
// 64 rows of keys or of values, 16 bytes a lane: 16 rows lie in one page, whatever its size, and rows of a group are at fixed distances. Rows behind the last key are
// not fetched: what the buffer holds in their place are codes like any other, and meets weights of zero.
template <int D, bool VALUES>
__device__ __forceinline__ void fetch(const AttArgs& a, const Unit& n, uint32_t dst, int lane) {
  constexpr int CH = D / 16, PER = 32 / CH;       // 16-byte pieces of a row; rows per instruction
  const int c = lane % CH, row0 = lane / CH, have = n.keys - n.key0;
  const signed char* base = (VALUES ? a.v : a.k) + c * 16;
  const int in_page = n.key0 & ((1 << a.pshift) - 1);       // (the second half of a page of 128)
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const long long at = __shfl_sync(0xffffffffu, n.at, (16 * q) >> a.pshift);
    if (at < 0) continue;
    const signed char* src = base + at + (size_t)(((in_page + 16 * q) & ((1 << a.pshift) - 1)) + row0) * D;
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const int row = q * 16 + i * PER + row0;
      if (row < have) copy16(dst + (VALUES ? v_chunk<D>(row, c) : k_chunk<D>(row, c)), src + i * PER * D);
    }
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, 1) kv8_attention_kernel(const AttArgs a) {
  using T = typename Elem16<BF16>::T;
  using S = Smem<D>;
  constexpr int KS = D / 16, NT = D / 8, CH = D / 16;       // steps of the score product, column tiles of the value product, 16-byte pieces of a key
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_sum[WARPS];
  __shared__ int s_place[3];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, qi = lane >> 2, qj = lane & 3;
  unsigned char* const s_q = smem + S::RING;
  float* const s_o = reinterpret_cast<float*>(smem + S::RING + S::Q);
  float* const s_ml = reinterpret_cast<float*>(smem + S::RING + S::Q + S::O);   // [warp][maximum, sum][16]
  const uint32_t kbuf = shared_addr(smem) + warp * 2 * S::BUF, vbuf = kbuf + S::BUF;
  pdl_enter();

  // ---- this CTA's stretch: all units, and the request that the first one lies in
  const int per_thread = (a.nreq + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int i = 0; i < per_thread; ++i) {
    const int b = tid * per_thread + i;
    if (b < a.nreq) mine += request(a, b).total(a.G);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const long long per = max((total + gridDim.x - 1) / gridDim.x, (long long)MIN_UNITS);
  const long long begin = per * blockIdx.x, end = min(begin + per, total);
  if (begin >= end) return;
  if (begin >= before && begin < before + mine) {
    long long at = before;
    for (int i = 0; i < per_thread; ++i) {
      const Req r = request(a, min(tid * per_thread + i, a.nreq - 1));
      const long long n = r.total(a.G);
      if (begin < at + n) {
        s_place[0] = tid * per_thread + i;
        s_place[1] = (int)((begin - at) / r.units);       // item of the request: head * tiles + tile
        s_place[2] = (int)((begin - at) % r.units);
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  Place cur;                                                // the segment that all warps are in: (the rest of) one item
  cur.b = s_place[0];
  cur.u = s_place[2];
  cur.r = request(a, cur.b);
  cur.g = s_place[1] / cur.r.tiles;
  cur.tile = s_place[1] - cur.g * cur.r.tiles;
  const int todo = (int)(end - begin);                      // units of this stretch

  // queries of an item, 16 rows as they lie: a thread's 16 bytes of them (rows behind the last one are zeros)
  constexpr int PIECES_Q = D / 8;
  const int qr = tid / PIECES_Q, qc = tid % PIECES_Q;
  auto load_q = [&](const Place& p) {
    const int row = p.tile * ROWS + qr, tok = row / a.rep;
    if (qr >= ROWS || tok >= p.r.n) return make_uint4(0u, 0u, 0u, 0u);
    return *reinterpret_cast<const uint4*>((const T*)a.q + (size_t)(p.r.first + tok) * a.q_ts + (size_t)(p.g * a.rep + row - tok * a.rep) * a.q_hs + qc * 8);
  };
  auto store_q = [&](const uint4& w, int buf) {
    if (qr < ROWS) *reinterpret_cast<uint4*>(s_q + (buf * ROWS + qr) * D * 2 + qc * 16) = w;
  };

  // ---- the first unit of this warp is on its way before anything else. Pages are looked up one unit ahead of the copies, so that these do not wait for them.
  int next = warp;                                          // index in the stretch of the unit that is fetched next
  Place np = cur;
  np.forward(a, warp);
  int pages = next < todo ? unit_page(a, np, lane) : -1;
  Unit unit{-1, 0, 0};                                      // the one that was fetched last, with its scales
  float pks = 0.f, pvs = 1.f;
  auto take = [&]() {                                       // the unit at np, and the pages of the one behind it
    const bool there = pages >= 0;
    const size_t block = there ? (size_t)pages * a.G + np.g : 0;
    unit.at = there ? (long long)((block << a.pshift) * D) : -1ll;
    unit.key0 = np.u * UNIT;
    unit.keys = next < todo ? np.r.keys : 0;
    pks = there ? a.ks[block] : pages == BROKEN ? NAN : 1.f;
    pvs = there ? a.vs[block] : 1.f;
    np.forward(a, WARPS);
    pages = next + WARPS < todo ? unit_page(a, np, lane) : -1;
  };
  uint4 queries = load_q(cur);
  take();
  fetch<D, false>(a, unit, kbuf, lane);
  copy_commit();
  fetch<D, true>(a, unit, vbuf, lane);
  copy_commit();
  store_q(queries, 0);
  __syncthreads();

  int seg0 = 0;                                             // index in the stretch of the segment's first unit
  for (int seg = 0; seg0 < todo; ++seg) {
    const int seg_n = min(cur.r.units - cur.u, todo - seg0);
    Place after = cur;
    after.forward(a, seg_n);
    const bool more = seg0 + seg_n < todo;
    if (more) queries = load_q(after);                      // the next segment's queries, on their way beside this one's work

    const int tile = cur.tile, g = cur.g;
    // ---- queries into registers; bfloat16 rows by a power of two each
    uint32_t qa[KS][4];
    float rowf[2];
    int limit[2];                                           // last visible position of this lane's rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const unsigned char* row = s_q + ((seg & 1) * ROWS + qi + 8 * e) * D * 2;
      uint32_t x[CH / 4][8];
#pragma unroll
      for (int h = 0; h < CH / 4; ++h) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(row + (h * 4 + qj) * 32), w1 = *reinterpret_cast<const uint4*>(row + (h * 4 + qj) * 32 + 16);
        x[h][0] = w0.x; x[h][1] = w0.y; x[h][2] = w0.z; x[h][3] = w0.w;
        x[h][4] = w1.x; x[h][5] = w1.y; x[h][6] = w1.z; x[h][7] = w1.w;
      }
      int sh = 0;
      if (BF16) {
        float mx = 0.f;
#pragma unroll
        for (int h = 0; h < CH / 4; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[h][i] << 16)), fabsf(__uint_as_float(x[h][i] & 0xffff0000u))));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^(14 - exponent of the largest), from its bits; none for a row of zeros or one that is not finite, and in float32's range at both ends
        const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
        sh = mx > 0.f && mx < INFINITY ? min(max(14 - ex, -126), 126) : 0;
        const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
        for (int h = 0; h < CH / 4; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[h][i] = half_pair(__uint_as_float(x[h][i] << 16) * up, __uint_as_float(x[h][i] & 0xffff0000u) * up);
      }
      rowf[e] = __uint_as_float((uint32_t)(127 - sh) << 23) * a.scale2;
#pragma unroll
      for (int h = 0; h < CH / 4; ++h)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          qa[h * 4 + w][e] = x[h][2 * w];
          qa[h * 4 + w][e + 2] = x[h][2 * w + 1];
        }
      const int tok = (tile * ROWS + qi + 8 * e) / a.rep;
      limit[e] = tok < cur.r.n ? min(cur.r.keys - cur.r.n + tok, cur.r.keys - 1) : -1;
    }
    const int low = cur.r.keys - cur.r.n + tile * ROWS / a.rep;   // the lowest of the tile's rows
    // What the codes' 128 adds to a row's scores, the other way round: -128 (in units of 2^-24) times the sum of the row.
    float s0[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KS; ++i) mma16816(s0, qa[i], 0x80808080u, 0x80808080u);
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m[2] = {NONE, NONE}, l[2] = {0.f, 0.f};

    while (next < seg0 + seg_n) {
      // ---- scores of 64 keys, in units of 2^-24
      const int key0 = unit.key0;
      const float cks = pks, cvs = pvs;
      copy_wait<1>();
      __syncwarp();
      float s[8][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4][CH / 4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int h = 0; h < CH / 4; ++h)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[n][h][0]), "=r"(w[n][h][1]), "=r"(w[n][h][2]), "=r"(w[n][h][3])
                         : "r"(kbuf + k_chunk<D>((half * 4 + n) * 8 + qi, h * 4 + qj)));
#pragma unroll
        for (int n = 0; n < 4; ++n) { s[half * 4 + n][0] = s0[0]; s[half * 4 + n][1] = s0[0]; s[half * 4 + n][2] = s0[2]; s[half * 4 + n][3] = s0[2]; }
#pragma unroll
        for (int h = 0; h < CH / 4; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const uint32_t u = w[n][h][i] ^ 0x80808080u;
              mma16816(s[half * 4 + n], qa[h * 4 + i], codes_tiny(u, 0x4140), codes_tiny(u, 0x4342));
            }
      }
      __syncwarp();
      // the next unit's keys take this one's place
      next += WARPS;
      take();
      fetch<D, false>(a, unit, kbuf, lane);
      copy_commit();
      // ---- weights
      // Keys that a row does not see; and of a page that there is not, or whose scale is no number, what makes the rows NaN that do see it.
      const bool odd = __any_sync(0xffffffffu, cks != cks || cvs != cvs);
      if (key0 + UNIT - 1 > low || odd) {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const int src = (8 * nt) >> a.pshift;
          const float both = __shfl_sync(0xffffffffu, cks + cvs, src);
          const bool none = both != both;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (none) s[nt][e] = NAN;
            if (key0 + nt * 8 + qj * 2 + (e & 1) > limit[e >> 1]) s[nt][e] = NONE;
          }
        }
      }
      float kf[4][2], lv[4], iv[4], mx[2] = {NONE, NONE};   // of 16 keys each: factor of the scores, log2 of the value scale and its reciprocal
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int src = (16 * q) >> a.pshift;
        const float f = positive(__shfl_sync(0xffffffffu, cks, src)) * 16777216.f, v = positive(__shfl_sync(0xffffffffu, cvs, src));
        lv[q] = __log2f(v);
        iv[q] = __fdividef(1.f, v);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kf[q][e] = f * rowf[e];
          const float top = fmaxf(fmaxf(s[2 * q][2 * e], s[2 * q][2 * e + 1]), fmaxf(s[2 * q + 1][2 * e], s[2 * q + 1][2 * e + 1]));
          mx[e] = fmaxf(mx[e], fmaf(top, kf[q][e], lv[q])); // (factors are positive: the largest score has the largest exponent)
        }
      }
      bool grown[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        // The reference follows the maximum only where it has fallen 2^8 behind: weights stay below 2^8, and sums are seldom multiplied again.
        grown[e] = mx[e] > m[e] + 8.f || (m[e] == NONE && mx[e] > NONE);
      }
      if (__any_sync(0xffffffffu, (grown[0] && m[0] != NONE) || (grown[1] && m[1] != NONE))) {
        const float f[2] = {grown[0] ? exp2_fast(m[0] - mx[0]) : 1.f, grown[1] ? exp2_fast(m[1] - mx[1]) : 1.f};
        l[0] *= f[0];
        l[1] *= f[1];
#pragma unroll
        for (int t = 0; t < NT; ++t) { o[t][0] *= f[0]; o[t][1] *= f[0]; o[t][2] *= f[1]; o[t][3] *= f[1]; }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (grown[e]) m[e] = mx[e];                         // (a row that had seen nothing has sums of zero)
      const float ref[2] = {m[0] == NONE ? 0.f : m[0], m[1] == NONE ? 0.f : m[1]};
      // Exponents are taken from the products without a rounding in between, the reference has one: beyond 2^24 that alone would be a large exponent.
      if (__any_sync(0xffffffffu, fabsf(ref[0]) > 16777216.f || fabsf(ref[1]) > 16777216.f)) {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = fmaf(s[nt][e], kf[nt >> 1][e >> 1], lv[nt >> 1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) { kf[q][0] = kf[q][1] = 1.f; lv[q] = 0.f; }
      }
      uint32_t pa[4][4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float at[2] = {lv[q] - ref[0], lv[q] - ref[1]};
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = exp2_fast(fmaf(s[2 * q + z][e], kf[q][e >> 1], at[e >> 1]));
            part[e >> 1] += w[e];
          }
          pa[q][z * 2] = half_pair(w[0], w[1]);
          pa[q][z * 2 + 1] = half_pair(w[2], w[3]);
        }
        l[0] = fmaf(part[0], iv[q], l[0]);
        l[1] = fmaf(part[1], iv[q], l[1]);
      }
      // ---- values
      copy_wait<1>();
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        constexpr int W = D / 32;                           // 32-bit words of a lane's columns of a row
        uint32_t r[4][W];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int row = q * 16 + qj * 2 + (z & 1) + (z >> 1) * 8;
          if constexpr (D == 128)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[z][0]), "=r"(r[z][1]), "=r"(r[z][W - 2]), "=r"(r[z][W - 1]) : "r"(vbuf + v_chunk<D>(row, qi)));
          else
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(r[z][0]), "=r"(r[z][1]) : "r"(vbuf + v_chunk<D>(row, qi >> 1) + (qi & 1) * 8));
#pragma unroll
          for (int w = 0; w < W; ++w) r[z][w] ^= 0x80808080u;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t x0 = __byte_perm(r[0][w], r[1][w], 0x5140), y0 = __byte_perm(r[0][w], r[1][w], 0x7362);
          const uint32_t x1 = __byte_perm(r[2][w], r[3][w], 0x5140), y1 = __byte_perm(r[2][w], r[3][w], 0x7362);
          mma16816(o[4 * w], pa[q], codes16(x0, 0x4140), codes16(x1, 0x4140));
          mma16816(o[4 * w + 1], pa[q], codes16(x0, 0x4342), codes16(x1, 0x4342));
          mma16816(o[4 * w + 2], pa[q], codes16(y0, 0x4140), codes16(y1, 0x4140));
          mma16816(o[4 * w + 3], pa[q], codes16(y0, 0x4342), codes16(y1, 0x4342));
        }
      }
      __syncwarp();
      fetch<D, true>(a, unit, vbuf, lane);
      copy_commit();
    }

    if (more) store_q(queries, (seg + 1) & 1);              // (the last that read them has passed two barriers)
    // ---- the warps' sums of this item together. Column order on the way: [half of a lane's columns][t / 4][lane of the quad][t % 4].
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (qj == 0) {
        s_ml[(warp * 2) * ROWS + qi + 8 * e] = m[e];
        s_ml[(warp * 2 + 1) * ROWS + qi + 8 * e] = l[e];
      }
      // (a warp without a unit in this segment has nothing but its maximum to tell)
      if (m[e] != NONE || l[e] != 0.f) {
        float* row = s_o + (warp * ROWS + qi + 8 * e) * O_LD + qj * 4;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int t = 0; t < NT / 4; ++t)
            *reinterpret_cast<float4*>(row + (c * (NT / 4) + t) * 16) = make_float4(o[4 * t][2 * e + c], o[4 * t + 1][2 * e + c], o[4 * t + 2][2 * e + c], o[4 * t + 3][2 * e + c]);
      }
    }
    __syncthreads();
    constexpr int PIECES = D / 64;                          // float4 of a thread: 16 threads a row
    const int jr = tid >> 4, col = tid & 15;
    float mm = NONE, ll = 0.f;
    float4 oo[PIECES];
#pragma unroll
    for (int c = 0; c < PIECES; ++c) oo[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float mw, float lw, auto&& piece) {
      // (a part that saw nothing has no sums; one that saw NaN has a sum that is not zero)
      if (mw == NONE && lw == 0.f) return;
      const float mn = fmaxf(mm, mw), f = mm == NONE ? 0.f : exp2_fast(mm - mn), h = mw == NONE ? 1.f : exp2_fast(mw - mn);
      mm = mn;
      ll = ll * f + lw * h;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        const float4 p = piece(c);
        oo[c].x = oo[c].x * f + p.x * h; oo[c].y = oo[c].y * f + p.y * h; oo[c].z = oo[c].z * f + p.z * h; oo[c].w = oo[c].w * f + p.w * h;
      }
    };
    for (int w = 0; w < WARPS; ++w)
      join(s_ml[(w * 2) * ROWS + jr], s_ml[(w * 2 + 1) * ROWS + jr], [&](int c) { return *reinterpret_cast<const float4*>(s_o + (w * ROWS + jr) * O_LD + (col + 16 * c) * 4); });
    const int rr = tile * ROWS + jr, tok = rr / a.rep;
    auto store = [&]() {
      if (tok >= cur.r.n) return;
      const float f = ll == 0.f ? 0.f : __fdiv_rn(1.f, ll);  // no key: zeros
      T* to = (T*)a.out + (size_t)(cur.r.first + tok) * a.out_ts + (size_t)(g * a.rep + rr - tok * a.rep) * a.out_hs;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        const int at = col + 16 * c, q = at >> 2, half = q / (NT / 4), t = q % (NT / 4) * 4, j = at & 3;
        const float4 p = oo[c];
        uint2 w;
        if (BF16) {
          const __nv_bfloat162 x = __floats2bfloat162_rn(p.x * f, p.y * f), y = __floats2bfloat162_rn(p.z * f, p.w * f);
          w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        } else {
          w = make_uint2(half_pair(p.x * f, p.y * f), half_pair(p.z * f, p.w * f));
        }
        *reinterpret_cast<uint2*>(to + (2 * j + half) * NT + t) = w;
      }
    };
    const bool starts = cur.u == 0, ends = cur.u + seg_n == cur.r.units;
    if (starts && ends) {
      store();
    } else {
      // ---- a part of an item: into the workspace; the item's last CTA to come adds all of them up, first part first
      const long long item0 = begin + seg0 - cur.u, item1 = item0 + cur.r.units;
      const int c0 = (int)(item0 / per), c1 = (int)((item1 - 1) / per);
      float* part = a.parts + (size_t)(2 * blockIdx.x + (starts ? 1 : 0)) * PART<D>;
      if (col == 0) { part[jr] = mm; part[ROWS + jr] = ll; }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) *reinterpret_cast<float4*>(part + 2 * ROWS + jr * D + (col + 16 * c) * 4) = oo[c];
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int n = c1 - c0 + 1, old = atomicAdd(a.counters + c0, 1);
        s_last = old == n - 1;
        if (old == n - 1) a.counters[c0] = 0;               // for the next call
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        mm = NONE;
        ll = 0.f;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) oo[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = c0; p <= c1; ++p) {
          const float* from = a.parts + (size_t)(2 * p + (p == c0 ? 1 : 0)) * PART<D>;
          join(__ldcg(from + jr), __ldcg(from + ROWS + jr), [&](int c) { return __ldcg(reinterpret_cast<const float4*>(from + 2 * ROWS + jr * D + (col + 16 * c) * 4)); });
        }
        store();
      }
    }
    cur = after;
    seg0 += seg_n;
    __syncthreads();                                        // the sums have been read, the next queries are there
  }
  copy_wait<0>();
}

}  // namespace kv8
}  // namespace qspec

using namespace qspec;
using namespace qspec::kv8;

static int att_grid() { return max(sm_count(), 1); }

extern "C" size_t qspec_kv8_attention_workspace_bytes(void) { return 4096 + (size_t)att_grid() * 2 * PART<128> * sizeof(float); }

extern "C" int qspec_kv8_attention(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const float* ks, const float* vs, const int* table,
                                   const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok, int requests, int width, int H,
                                   int G, int D, int npages, int page_tokens, int max_tokens, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  QSPEC_REQUIRE(k && v && ks && vs && table && q_start && kv_len, QSPEC_ERR_INVALID_ARG, "kv8_attention: null pointer");
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "kv8_attention: pages of 16, 32, 64 or 128 tokens, got %d", page_tokens);
  QSPEC_REQUIRE(D == 64 || D == 128, QSPEC_ERR_UNSUPPORTED, "kv8_attention: heads of 64 or 128, got %d", D);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv8_attention: float16 or bfloat16 queries");
  QSPEC_REQUIRE(G >= 1 && H >= G && H % G == 0 && H <= 4096, QSPEC_ERR_INVALID_ARG, "kv8_attention: %d query heads, %d key/value heads", H, G);
  QSPEC_REQUIRE(ntok >= 0 && ntok < (1 << 24) && requests >= 1 && width >= 1 && npages >= 1 && max_tokens >= 1 && (long long)npages * page_tokens < (1ll << 31) &&
                    (long long)width * page_tokens < (1ll << 31),
                QSPEC_ERR_INVALID_ARG, "kv8_attention: tokens=%d requests=%d width=%d pages=%d", ntok, requests, width, npages);
  if (ntok == 0) return QSPEC_OK;
  QSPEC_REQUIRE(q && out, QSPEC_ERR_INVALID_ARG, "kv8_attention: null pointer");
  auto aligned = [](const void* p, long long ts, int hs) { return ((uintptr_t)p & 15) == 0 && ts > 0 && hs > 0 && ts % 8 == 0 && hs % 8 == 0; };
  QSPEC_REQUIRE(aligned(q, q_tok_stride, q_head_stride) && aligned(out, out_tok_stride, out_head_stride) && ((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0,
                QSPEC_ERR_INVALID_ARG, "kv8_attention: rows must lie on 16-byte boundaries");
  QSPEC_REQUIRE(workspace && workspace_bytes >= qspec_kv8_attention_workspace_bytes() && ((uintptr_t)workspace & 15) == 0, QSPEC_ERR_WORKSPACE,
                "kv8_attention: %zu bytes of workspace needed, got %zu", qspec_kv8_attention_workspace_bytes(), workspace_bytes);
  const int grid = att_grid();
  QSPEC_REQUIRE(grid <= 1024, QSPEC_ERR_UNSUPPORTED, "kv8_attention: %d SMs", grid);
  AttArgs a{q, q_tok_stride, q_head_stride, (const signed char*)k, (const signed char*)v, ks, vs, table, q_start, kv_len, requests, width, npages, page_shift(page_tokens), ntok,
            G, H / G, 0x7fffffff, scale * 1.4426950408889634f, out, out_tok_stride, out_head_stride, (int*)workspace, (float*)((char*)workspace + 4096)};
  auto run = [&](auto kern, size_t smem, SmemLimit& limit) -> int {
    QSPEC_CUDA(limit.raise(kern, smem));
    QSPEC_CUDA(launch_pdl(kern, dim3(grid), dim3(THREADS), smem, (cudaStream_t)stream, a));
    QSPEC_CHECK_LAUNCH(1);
    return QSPEC_OK;
  };
  static SmemLimit limits[4];
  if (dtype == QSPEC_DTYPE_F16)
    return D == 128 ? run(kv8_attention_kernel<false, 128>, Smem<128>::TOTAL, limits[0]) : run(kv8_attention_kernel<false, 64>, Smem<64>::TOTAL, limits[1]);
  return D == 128 ? run(kv8_attention_kernel<true, 128>, Smem<128>::TOTAL, limits[2]) : run(kv8_attention_kernel<true, 64>, Smem<64>::TOTAL, limits[3]);
}
