// Softmax attention over a key/value cache in pages and in 8 bits (its layout: kv8_kernels.cu). Token i of the n that request b has in the step stands at
// position kv_len[b] - n + i and sees the keys up to its own position.
//
// A row is a (token, query head of a group) pair; 16 rows of one key/value head are a tile of mma.sync.m16n8k16, so that the heads of a group and the
// tokens that verify a draft share every key that is read. What bounds it at these row counts is the cache: 2 D bytes a key and head.
//
// Work: (request, head, row tile) items of units of 32 keys, laid end to end and cut into equal stretches, one per CTA: lengths that
// differ cost nothing, one long request uses every SM. Inside a stretch unit i is warp i % WARPS's. Every warp keeps a softmax of its own (maximum, sum and
// sums of values in registers) over the units of an item that it took; they are joined through shared memory at the item's end and, where a stretch
// ends inside an item, through the workspace: the CTA that comes last adds the parts up in their order, so that results do not depend on which it is.
//
// Codes go from global memory into shared memory (16 bytes a lane, asynchronously, one unit of keys and one of values per warp) and from there into
// registers as the products' operands.
//   keys: a byte c + 128 alone is the float16 (c + 128) 2^-24, a subnormal number, which the tensor cores take exactly: no arithmetic but the byte's
//   place. What the 128 adds to a score is the same for all keys, 128 times the row's sum, and is where the sums begin, from the other side. The order of
//   the sum over a head's dimensions is free, so that a lane's 16 bytes of a key are its operands of four products; queries lie in shared memory in that order.
//   values: the transposing load of 16 x 16 bytes gives four keys of a column a word (the keys of the score tiles are numbered to match); the byte behind 0x64 is the
//   float16 1152 + c, and one subtraction makes it c. (Sums over values must not carry the 128: over many keys they cancel, and what the
//   products cut off would be of the size of what is left.)
//
// bfloat16 queries are multiplied by a power of two per row that brings their largest value to 2^14 .. 2^15 and are float16 from there on, exactly. A key's scale
// multiplies its scores in float32. A value's scale v goes into the exponent: the weights 2^(9 + s + log2 v - m) lie below 2^15 whatever the scales are and are
// rounded to float16 for the product with the codes (by 2^-11 of themselves at most, or by 2^-34 of the largest: kv8_common.cuh); the denominator is the sum of the
// unrounded weights / v.
#include "kv8_common.cuh"

namespace qspec {
namespace kv8 {

constexpr int WARPS = 4, THREADS = WARPS * 32, UNIT = 32, ROWS = 16;
constexpr int MIN_UNITS = WARPS;                 // of a stretch: one for each warp
constexpr int CTAS = 3;                          // of an SM: while one waits at a barrier the others compute
constexpr int GRID_MOST = 480;                   // CTAs
constexpr float NONE = -INFINITY;

struct AttArgs {
  const void* q; long long q_ts; int q_hs;
  const signed char *k, *v;
  const float *ks, *vs;
  const int *table, *q_start, *kv_len;
  int nreq, width, npages, pshift, ntok, G, rep;
  unsigned share;                                // to_prompt_form()'s; 0: there is no prompt form in this call
  float scale2;                                  // scale * log2(e)
  void* out; long long out_ts; int out_hs;
  int* counters; float* parts;
};

template <int D> struct Smem {
  static constexpr int BUF = UNIT * D;                                  // one unit's keys or values
  static constexpr size_t RING = (size_t)WARPS * 2 * BUF;
  static constexpr size_t Q = ROWS * D * 2;
  static constexpr int LD = D + 8;                                      // floats of a row of sums on its way between warps (8 modulo 32: no bank conflicts)
  static constexpr size_t SUMS = (size_t)WARPS * ROWS * LD * 4, FACTORS = (size_t)(GRID_MOST + 1) * ROWS * 4;
  static constexpr size_t O = SUMS > FACTORS ? SUMS : FACTORS;          // sums on their way between warps, or a factor for every part of an item
  static constexpr size_t ML = (size_t)WARPS * ROWS * 2 * 4;
  static constexpr size_t F = ROWS * 4;                             // factors of the rows' scores
  static constexpr size_t TOTAL = RING + Q + O + ML + F;
};
template <int D> constexpr int PART = ROWS * 2 + ROWS * D;   // floats of a part: maxima, sums, sums of values

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
// d = a b + c
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// two 16 x 16 blocks of bytes, columns first: word 2 m + h of a lane has rows 4 j .. 4 j + 3 (j = lane % 4) of column lane / 4 + 8 h of block m
__device__ __forceinline__ void load_columns(uint32_t (&w)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
// The first two / the last two of four codes (bytes c + 128) as float16: a byte alone is (c + 128) 2^-24, a subnormal number.
__device__ __forceinline__ uint32_t first_two(uint32_t w) { return __byte_perm(w, 0u, 0x4140); }
__device__ __forceinline__ uint32_t last_two(uint32_t w) { return __byte_perm(w, 0u, 0x4342); }
constexpr uint32_t MINUS_128 = 0x80808080u;      // two of -128 2^-24: what the codes' 128 adds up to, the other way round

// A request's part of the work.
struct Req {
  int first, n, keys, tiles, units;               // first row of q, tokens, keys, row tiles, units of an item
  __device__ __forceinline__ long long total(int G) const { return (long long)tiles * G * units; }
};
__device__ __forceinline__ Req request(const AttArgs& a, int b, unsigned long long work) {
  Req r;
  r.first = min(max(a.q_start[b], 0), a.ntok);
  r.n = max(min(a.q_start[b + 1], a.ntok) - r.first, 0);
  r.keys = max(a.kv_len[b], 0);
  const long long rows = (long long)r.n * a.rep;
  r.tiles = to_prompt_form(r.n, r.keys, a.rep, a.share, work) ? 0 : (int)((rows + ROWS - 1) / ROWS);
  // A request without keys has a unit that shows its rows none. Behind the table's last page is nothing but a page that there is not: one unit shows that.
  r.units = max((min(r.keys, keys_at_most(a.width, a.pshift)) + UNIT - 1) / UNIT, 1);
  return r;
}

// Where a unit lies: request, head and row tile (tiles inside heads), unit of that item.
struct Place {
  int b, g, tile, u;
  Req r;
  __device__ __forceinline__ void forward(const AttArgs& a, unsigned long long work, int steps) {
    u += steps;
    while (b < a.nreq && u >= r.units) {
      u -= r.units;
      if (++tile < r.tiles) continue;
      tile = 0;
      if (++g < a.G) continue;
      g = 0;
      do { if (++b >= a.nreq) return; r = request(a, b, work); } while (r.tiles == 0);
    }
  }
};

// Where the 16 bytes c of a row lie in a buffer, so that neither copies nor reads of eight rows meet in a bank.
template <int D>
__device__ __forceinline__ uint32_t k_chunk(int row, int c) { return (uint32_t)(row * D + ((D == 128 ? c ^ ((row & 1) << 2) : c) << 4)); }
template <int D>
__device__ __forceinline__ uint32_t v_chunk(int row, int c) { return (uint32_t)(row * D + ((D == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4)); }

// The page that lane i has of the unit at `p`: its ith, of UNIT / P (at least one); -1: one behind the last key; BROKEN: an entry that is no page of the cache.
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
// UNIT rows of keys or of values, 16 bytes a lane: 16 rows lie in one page, whatever its size, and rows of a group are at fixed distances. Rows behind the last key are
// not fetched: what the buffer holds in their place are codes like any other, and meets weights of zero.
template <int D, bool VALUES>
__device__ __forceinline__ void fetch(const AttArgs& a, const Unit& n, uint32_t dst, int lane) {
  constexpr int CH = D / 16, PER = 32 / CH;       // 16-byte pieces of a row; rows per instruction
  const int c = lane % CH, row0 = lane / CH, have = n.keys - n.key0;
  const signed char* base = (VALUES ? a.v : a.k) + (row0 * D + c * 16);
  auto rows = [&](int q, const signed char* src, bool all) {  // rows 16 q .. 16 q + 15
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const int row = q * 16 + i * PER + row0;
      if (all || row < have) copy16(dst + (VALUES ? v_chunk<D>(row, c) : k_chunk<D>(row, c)), src + i * PER * D);
    }
  };
  if (a.pshift >= 5 && have >= UNIT) {            // (one page; larger ones are several units)
    const long long at = __shfl_sync(0xffffffffu, n.at, 0);
    if (at < 0) return;
    const signed char* src = base + at + (size_t)(n.key0 & ((1 << a.pshift) - 1)) * D;
#pragma unroll
    for (int q = 0; q < UNIT / 16; ++q) rows(q, src + 16 * q * D, true);
  } else {
#pragma unroll
    for (int q = 0; q < UNIT / 16; ++q) {
      const long long at = __shfl_sync(0xffffffffu, n.at, (16 * q) >> a.pshift);
      if (at >= 0) rows(q, base + at + (size_t)((n.key0 + 16 * q) & ((1 << a.pshift) - 1)) * D, false);
    }
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, CTAS) kv8_attention_kernel(const AttArgs a) {
  using T = typename Elem16<BF16>::T;
  using S = Smem<D>;
  constexpr int NT = D / 8, CH = D / 16, KT = UNIT / 8, QT = UNIT / 16;   // column tiles of the value product, 16-byte pieces of a key (steps of the score product), key tiles
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_sum[WARPS];
  __shared__ int s_place[4], s_items[WARPS], s_ctas[6][WARPS];
  __shared__ Req s_req;
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, qi = lane >> 2, qj = lane & 3;
  unsigned char* const s_q = smem + S::RING;
  float* const s_o = reinterpret_cast<float*>(smem + S::RING + S::Q);
  float* const s_ml = reinterpret_cast<float*>(smem + S::RING + S::Q + S::O);   // [warp][maximum, sum][16]
  float* const s_f = reinterpret_cast<float*>(smem + S::RING + S::Q + S::O + S::ML);   // [16]
  const uint32_t kbuf = shared_addr(smem) + warp * 2 * S::BUF, vbuf = kbuf + S::BUF;
  pdl_enter();

  // ---- this CTA's stretch
  const int per_thread = (a.nreq + THREADS - 1) / THREADS, b0 = tid * per_thread;
  const int requests = max(min(per_thread, a.nreq - b0), 0);
  unsigned long long work = 0;                              // that requests with rows enough for the prompt form ask for
  if (a.share) {
    for (int i = 0; i < requests; ++i) {
      const Req r = request(a, b0 + i, 0);
      work += prompt_work(r.n, r.keys, a.rep, a.G);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    if (lane == 0) s_sum[warp] = (long long)work;
    __syncthreads();
    work = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) work += (unsigned long long)s_sum[w];
    __syncthreads();
  }
  Req only{0, 0, 0, 0, 1};
  if (per_thread == 1 && b0 < a.nreq) only = request(a, b0, work);
  auto req = [&](int i) { return per_thread == 1 ? only : request(a, b0 + i, work); };
  long long before, total;                                  // of the requests of the threads in front of this one, and of all
  auto scan = [&](long long mine) {
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += w;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
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
  if (lane == 0) s_items[warp] = items;
  scan(mine);
  const int grid = gridDim.x;
  long long per = max(total <= 0x7fffffff ? (long long)(((int)total - 1) / grid + 1) : (total + grid - 1) / grid, (long long)MIN_UNITS);
  // A stretch may lie over the end of an item: then the CTA joins and stores twice. With few items each gets CTAs of its own, as long as that makes no
  // stretch much longer (by a quarter and eight units at most): 4 requests of 900, 32 / 8 heads, one token each 17.0 -> 12.1 us.
  bool whole = false;
  items = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) items += s_items[w];
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
      if (lane == 0) s_ctas[c][warp] = n[c];
    }
    __syncthreads();
    int len = 0;
#pragma unroll
    for (int c = TRIES - 1; c >= 0; --c) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += s_ctas[c][w];
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
  if (begin >= total) return;
  if (begin >= before && begin < before + mine) {
    long long at = before;
    for (int i = 0; i < requests; ++i) {
      const Req r = req(i);
      const int each = whole ? (r.units - 1) / (int)per + 1 : r.units;   // of an item: CTAs, or units
      const long long n = (long long)r.tiles * a.G * each;
      if (begin < at + n) {
        s_place[0] = b0 + i;
        s_place[1] = (int)((begin - at) / each);            // item of the request: head * tiles + tile
        s_place[2] = (int)((begin - at) % each);
        s_place[3] = each;
        s_req = r;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  Place cur;                                                // the segment that all warps are in: (the rest of) one item
  cur.b = s_place[0];
  cur.r = s_req;
  cur.g = s_place[1] / cur.r.tiles;
  cur.tile = s_place[1] - cur.g * cur.r.tiles;
  const int share = whole ? (cur.r.units - 1) / s_place[3] + 1 : 0;
  cur.u = whole ? min(s_place[2] * share, cur.r.units) : s_place[2];
  const int todo = whole ? min(share, cur.r.units - cur.u) : (int)(min(begin + per, total) - begin);   // units of this stretch
  if (todo <= 0) return;                                    // (a last share of none)

  // Queries of an item: a thread's pieces of 8 values (rows behind the last one are zeros), then float16 in the order in which the product takes them: word
  // (step, lane, register) of the operand. Step 4 h + w of lane (row % 8, j) has columns 16 (4 h + j) + 4 w .. + 3.
  constexpr int IN_ROW = D / 8, PIECES_Q = ROWS * IN_ROW / THREADS, QROWS = THREADS / IN_ROW;
  const int qr = tid / IN_ROW, qc = tid % IN_ROW;
  uint4 queries[PIECES_Q];
  auto load_q = [&](const Place& p) {
#pragma unroll
    for (int i = 0; i < PIECES_Q; ++i) {
      const int row = p.tile * ROWS + qr + i * QROWS, tok = row / a.rep;
      queries[i] = make_uint4(0u, 0u, 0u, 0u);
      if (tok < p.r.n)
        queries[i] = *reinterpret_cast<const uint4*>((const T*)a.q + (size_t)(p.r.first + tok) * a.q_ts + (size_t)(p.g * a.rep + row - tok * a.rep) * a.q_hs + qc * 8);
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int i = 0; i < PIECES_Q; ++i) {
      const int row = qr + i * QROWS;
      uint32_t x[4] = {queries[i].x, queries[i].y, queries[i].z, queries[i].w};
      int sh = 0;
      if (BF16) {
        float mx = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
#pragma unroll
        for (int o = IN_ROW / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        // 2^(14 - exponent of the largest), from its bits; none for a row of zeros or one that is not finite, and in float32's range at both ends
        const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
        sh = mx > 0.f && mx < INFINITY ? min(max(14 - ex, -126), 126) : 0;
        const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = half_pair(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
      }
      if (qc == 0) s_f[row] = __uint_as_float((uint32_t)(127 - sh) << 23) * a.scale2;
      uint32_t* to = reinterpret_cast<uint32_t*>(s_q) + ((qc >> 3) * 4 + (qc & 1) * 2) * 128 + ((row & 7) * 4 + ((qc >> 1) & 3)) * 4 + (row >> 3);
      to[0] = x[0];
      to[2] = x[1];
      to[128] = x[2];
      to[130] = x[3];
    }
  };

  // ---- the first unit of this warp is on its way before anything else. Pages are looked up one unit ahead of the copies, so that these do not wait for them.
  int next = warp;                                          // index in the stretch of the unit that is fetched next
  Place np = cur;
  np.forward(a, work, warp);
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
    np.forward(a, work, WARPS);
    pages = next + WARPS < todo ? unit_page(a, np, lane) : -1;
  };
  load_q(cur);
  take();
  fetch<D, false>(a, unit, kbuf, lane);
  copy_commit();
  fetch<D, true>(a, unit, vbuf, lane);
  copy_commit();
  store_q();
  __syncthreads();

  int seg0 = 0;                                             // index in the stretch of the segment's first unit
  while (seg0 < todo) {
    const int seg_n = min(cur.r.units - cur.u, todo - seg0);
    const int tile = cur.tile, g = cur.g;
    const uint32_t frag = shared_addr(s_q) + lane * 16;
    auto query = [&](uint32_t (&x)[4], int step) {
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(frag + step * 512));
    };
    const float rowf[2] = {s_f[qi], s_f[qi + 8]};
    int limit[2];                                           // last visible position of this lane's rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = (tile * ROWS + qi + 8 * e) / a.rep;
      limit[e] = tok < cur.r.n ? min(cur.r.keys - cur.r.n + tok, cur.r.keys - 1) : -1;
    }
    const int low = cur.r.keys - cur.r.n + tile * ROWS / a.rep;   // the lowest of the tile's rows
    // What the codes' 128 adds to a row's scores, the other way round: -128 (in units of 2^-24) times the sum of the row.
    float s0[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      uint32_t x[4];
      query(x, i);
      mma16816(s0, x, MINUS_128, MINUS_128, s0);
    }
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m[2] = {NONE, NONE}, l[2] = {0.f, 0.f};

    while (next < seg0 + seg_n) {
      // ---- scores of the unit's keys, in units of 2^-24
      const int key0 = unit.key0;
      const float cks = pks, cvs = pvs;
      copy_wait<1>();
      __syncwarp();
      float s[KT][4];
#pragma unroll
      for (int h = 0; h < CH / 4; ++h) {
        uint32_t w[KT][4];
#pragma unroll
        for (int n = 0; n < KT; ++n)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[n][0]), "=r"(w[n][1]), "=r"(w[n][2]), "=r"(w[n][3])
                       : "r"(kbuf + k_chunk<D>((n >> 1) * 16 + (n & 1) * 2 + (qi >> 1) * 4 + (qi & 1), h * 4 + qj)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
          query(x, h * 4 + i);
#pragma unroll
          for (int n = 0; n < KT; ++n) {
            const uint32_t u = w[n][i] ^ 0x80808080u;
            if (h == 0 && i == 0) mma16816(s[n], x, first_two(u), last_two(u), s0);
            else mma16816(s[n], x, first_two(u), last_two(u), s[n]);
          }
        }
      }
      __syncwarp();
      // the next unit's keys take this one's place
      next += WARPS;
      take();
      fetch<D, false>(a, unit, kbuf, lane);
      copy_commit();
      // ---- weights
      // Keys that a row does not see; and of a page that there is not, or whose scale is infinite or no number, what makes the rows NaN that do see it.
      const float both = cks + cvs;
      const bool odd = __any_sync(0xffffffffu, !(both < INFINITY));
      if (key0 + UNIT - 1 > low || odd) {
#pragma unroll
        for (int nt = 0; nt < KT; ++nt) {
          const int src = (16 * (nt >> 1)) >> a.pshift;
          const bool none = !(__shfl_sync(0xffffffffu, both, src) < INFINITY);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (none) s[nt][e] = NAN;
            if (key0 + (nt >> 1) * 16 + qj * 4 + (nt & 1) * 2 + (e & 1) > limit[e >> 1]) s[nt][e] = NONE;
          }
        }
      }
      float kf[QT][2], lv[QT], iv[QT], mx[2] = {NONE, NONE};   // of 16 keys each: factor of the scores, log2 of the value scale and its reciprocal
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const int src = (16 * q) >> a.pshift;
        const float f = positive(__shfl_sync(0xffffffffu, cks, src)), v = fminf(positive(__shfl_sync(0xffffffffu, cvs, src)), 8.507059e37f);
        // (2^126, not infinite: beside a hidden key's minus infinity that would be no number)
        lv[q] = __log2f(v);
        iv[q] = __fdividef(WEIGHT_UNIT, v);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kf[q][e] = score_factor(f, rowf[e]);
          const float top = fmaxf(fmaxf(s[2 * q][2 * e], s[2 * q][2 * e + 1]), fmaxf(s[2 * q + 1][2 * e], s[2 * q + 1][2 * e + 1]));
          mx[e] = fmaxf(mx[e], fmaf(top, kf[q][e], lv[q])); // (factors are positive: the largest score has the largest exponent)
        }
      }
      bool grown[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        // The reference follows the maximum only where it has fallen behind: sums are seldom multiplied again.
        grown[e] = mx[e] > m[e] + GROWTH_LOG2 || (m[e] == NONE && mx[e] > NONE);
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
      const float ref[2] = {m[0] == NONE ? 0.f : m[0] - WEIGHT_LOG2, m[1] == NONE ? 0.f : m[1] - WEIGHT_LOG2};
      // Exponents are taken from the products without a rounding in between, the reference has one: far from zero that alone would be a large exponent.
      const bool far = __any_sync(0xffffffffu, fabsf(ref[0]) > FAR || fabsf(ref[1]) > FAR);
      if (far) {
#pragma unroll
        for (int nt = 0; nt < KT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = fmaf(s[nt][e], kf[nt >> 1][e >> 1], lv[nt >> 1]) - (m[e >> 1] == NONE ? 0.f : m[e >> 1]);
#pragma unroll
        for (int q = 0; q < QT; ++q) kf[q][0] = kf[q][1] = 1.f;
      }
      uint32_t pa[QT][4];
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const float at[2] = {far ? WEIGHT_LOG2 : lv[q] - ref[0], far ? WEIGHT_LOG2 : lv[q] - ref[1]};
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
      for (int c = 0; c < CH; c += 2)                       // 32 columns at a time
#pragma unroll
        for (int q = 0; q < QT; ++q) {
          uint32_t w[4];
          load_columns(w, vbuf + v_chunk<D>(q * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t u = w[t] ^ 0x80808080u;
            mma16816(o[2 * c + t], pa[q], exact_two(u, 0x4140), exact_two(u, 0x4342), o[2 * c + t]);
          }
        }
      __syncwarp();
      fetch<D, true>(a, unit, vbuf, lane);
      copy_commit();
    }

    Place after = cur;
    after.forward(a, work, seg_n);
    const bool more = seg0 + seg_n < todo;
    if (more) load_q(after);                                // the next segment's queries, on their way while sums are joined
    // ---- the warps' sums of this item together
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
        float* row = s_o + (warp * ROWS + qi + 8 * e) * S::LD + qj * 2;
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<float2*>(row + 8 * t) = make_float2(o[t][2 * e], o[t][2 * e + 1]);
      }
    }
    __syncthreads();
    constexpr int PER_ROW = THREADS / ROWS, PIECES = D / 4 / PER_ROW;   // threads of a row, float4 of a thread
    const int jr = tid / PER_ROW, col = tid % PER_ROW;
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
      join(s_ml[(w * 2) * ROWS + jr], s_ml[(w * 2 + 1) * ROWS + jr], [&](int c) { return *reinterpret_cast<const float4*>(s_o + (w * ROWS + jr) * S::LD + (col + PER_ROW * c) * 4); });
    auto store_piece = [&](int r, int at, const float4& p, float f) {   // columns at .. at + 3 of the tile's row r
      const int rr = tile * ROWS + r, tok = rr / a.rep;
      uint2 w;
      if (BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(p.x * f, p.y * f), y = __floats2bfloat162_rn(p.z * f, p.w * f);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
      } else {
        w = make_uint2(half_pair(p.x * f, p.y * f), half_pair(p.z * f, p.w * f));
      }
      *reinterpret_cast<uint2*>((T*)a.out + (size_t)(cur.r.first + tok) * a.out_ts + (size_t)(g * a.rep + rr - tok * a.rep) * a.out_hs + at) = w;
    };
    const bool starts = cur.u == 0, ends = cur.u + seg_n == cur.r.units;
    if (starts && ends) {
      if (tile * ROWS + jr < cur.r.n * a.rep) {
        const float f = ll == 0.f ? 0.f : __fdiv_rn(WEIGHT_UNIT, ll);   // (no key: zeros)
#pragma unroll
        for (int c = 0; c < PIECES; ++c) store_piece(jr, (col + PER_ROW * c) * 4, oo[c], f);
      }
    } else {
      // ---- a part of an item: into the workspace; the item's last CTA to come adds all of them up, first part first
      const long long item0 = begin + seg0 - cur.u, item1 = item0 + cur.r.units;
      const int c0 = whole ? (int)blockIdx.x - cur.u / share : (int)(item0 / per), c1 = whole ? c0 + (cur.r.units - 1) / share : (int)((item1 - 1) / per);
      float* part = a.parts + (size_t)(2 * blockIdx.x + (starts ? 1 : 0)) * PART<D>;
      if (col == 0) { part[jr] = mm; part[ROWS + jr] = ll; }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) *reinterpret_cast<float4*>(part + 2 * ROWS + jr * D + (col + PER_ROW * c) * 4) = oo[c];
      __syncthreads();
      if (tid == 0) {
        __threadfence();                                    // (of what the whole CTA has stored: the barrier is in front of it)
        const int n = c1 - c0 + 1, old = atomicAdd(a.counters + c0, 1);
        s_last = old == n - 1;
        if (old == n - 1) a.counters[c0] = 0;               // for the next call
      }
      __syncthreads();
      if (s_last) {
        // All maxima and sums first (eight threads a row), which gives every part its factor, then the sums of values: loads that wait for none before them.
        __threadfence();
        const int n = c1 - c0 + 1;
        auto from = [&](int i) { return a.parts + (size_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * PART<D>; };
        float* const factor = s_o;                          // [part][row]: the sums on their way between warps have been read
        mm = NONE;
        ll = 0.f;
        for (int i0 = col; i0 < n; i0 += 8 * PER_ROW) {
          float mp[8], lp[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int i = i0 + k * PER_ROW;
            mp[k] = i < n ? __ldcg(from(i) + jr) : NONE;
            lp[k] = i < n ? __ldcg(from(i) + ROWS + jr) : 0.f;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool none = mp[k] == NONE;                // nothing seen, or (a sum that is not zero) no number
            const float mn = fmaxf(mm, mp[k]);
            ll = (mm == NONE ? ll : ll * exp2_fast(mm - mn)) + (none ? lp[k] : lp[k] * exp2_fast(mp[k] - mn));
            mm = mn;
            if (i0 + k * PER_ROW < n) factor[(i0 + k * PER_ROW) * ROWS + jr] = none && lp[k] != 0.f ? INFINITY : mp[k];
          }
        }
        const float own = mm;
#pragma unroll
        for (int x = PER_ROW / 2; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
        if (own != NONE) ll *= exp2_fast(own - mm);
#pragma unroll
        for (int x = PER_ROW / 2; x > 0; x >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, x);
        for (int i = col; i < n; i += PER_ROW) {
          const float f = factor[i * ROWS + jr];
          factor[i * ROWS + jr] = f == NONE ? 0.f : f == INFINITY ? 1.f : exp2_fast(f - mm);
        }
        if (col == 0) factor[n * ROWS + jr] = ll == 0.f ? 0.f : __fdiv_rn(WEIGHT_UNIT, ll);   // (no key: zeros)
        __syncthreads();
        const int rows = min(cur.r.n * a.rep - tile * ROWS, ROWS);
        for (int x = tid; x < rows * (D / 4); x += THREADS) {
          const int r = x / (D / 4), at = x % (D / 4) * 4;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int i0 = 0; i0 < n; i0 += 32) {
            float4 v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k)
              v[k] = i0 + k < n ? __ldcg(reinterpret_cast<const float4*>(from(i0 + k) + 2 * ROWS + r * D + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float f = i0 + k < n ? factor[(i0 + k) * ROWS + r] : 0.f;
              sum.x = fmaf(v[k].x, f, sum.x); sum.y = fmaf(v[k].y, f, sum.y); sum.z = fmaf(v[k].z, f, sum.z); sum.w = fmaf(v[k].w, f, sum.w);
            }
          }
          store_piece(r, at, sum, factor[n * ROWS + r]);
        }
      }
    }
    if (more) store_q();                                    // (all have passed the barrier behind their last use of this item's)
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

static int att_grid() { return max(sm_count(), 1) * CTAS; }

extern "C" size_t qspec_kv8_attention_workspace_bytes(void) { return 4096 + (size_t)att_grid() * 2 * PART<128> * sizeof(float); }

static int attention(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const float* ks, const float* vs, const int* table, const int* q_start,
                     const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok, int requests, int width, int H, int G, int D, int npages,
                     int page_tokens, int max_tokens, float scale, int dtype, void* workspace, size_t workspace_bytes, bool always, unsigned give_up, void* stream) {
  QSPEC_REQUIRE(k && v && ks && vs && table && q_start && kv_len, QSPEC_ERR_INVALID_ARG, "kv8_attention: null pointer");
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "kv8_attention: pages of 16, 32, 64 or 128 tokens, got %d", page_tokens);
  QSPEC_REQUIRE(D == 64 || D == 128, QSPEC_ERR_UNSUPPORTED, "kv8_attention: heads of 64 or 128, got %d", D);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv8_attention: float16 or bfloat16 queries");
  QSPEC_REQUIRE(G >= 1 && H >= G && H % G == 0 && H <= 4096, QSPEC_ERR_INVALID_ARG, "kv8_attention: %d query heads, %d key/value heads", H, G);
  QSPEC_REQUIRE(scale > 0.f && scale < INFINITY, QSPEC_ERR_INVALID_ARG, "kv8_attention: scale must be positive and finite, got %g", (double)scale);
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
  QSPEC_REQUIRE(grid <= GRID_MOST, QSPEC_ERR_UNSUPPORTED, "kv8_attention: %d SMs", sm_count());
  // Requests with many rows may go to the prompt form (to_prompt_form()), in a launch of its own in front; none do if the call's rows are too few for a third of
  // the SMs (always: for tests).
  const int rep = H / G;
  const bool prompts = rep <= PROMPT_REP && (long long)max_tokens * rep >= PROMPT_ROWS && (always || (long long)ntok * H >= std::max(sm_count() / 3, 1) * 128ll);
  const unsigned share = always ? 1u : std::max(sm_count() / 4, 1) * 128u;
  if (prompts) {
    // Two tiles a CTA where the rows are more than the SMs take at once with one, by a quarter: it is 2350 cycles a tile and block of keys instead of 2850 to 3400,
    // with half as many CTAs. us of pairs (of single tiles), 32 / 8 heads, after 1000 tokens: 512 tokens 50 (36), 900: 60 (63), 2000: 113 (140); 16 requests
    // of 64: 43 (51).
    const int pair = always ? give_up >> 4 & 1 : (long long)ntok * H > 160ll * sm_count();
    const PromptArgs pa{q, q_tok_stride, q_head_stride, (const signed char*)k, (const signed char*)v, ks, vs, table, q_start, kv_len, requests, width, npages,
                        page_shift(page_tokens), ntok, G, rep, pair, share, scale * 1.4426950408889634f, out, out_tok_stride, out_head_stride, give_up};
    if (const int rc = launch_prompt(pa, D, dtype == QSPEC_DTYPE_BF16, (cudaStream_t)stream)) return rc;
  }
  AttArgs a{q, q_tok_stride, q_head_stride, (const signed char*)k, (const signed char*)v, ks, vs, table, q_start, kv_len, requests, width, npages, page_shift(page_tokens), ntok,
            G, rep, prompts ? share : 0u, scale * 1.4426950408889634f, out, out_tok_stride, out_head_stride, (int*)workspace, (float*)((char*)workspace + 4096)};
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

extern "C" int qspec_kv8_attention(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const float* ks, const float* vs, const int* table,
                                   const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok, int requests, int width, int H,
                                   int G, int D, int npages, int page_tokens, int max_tokens, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(q, q_tok_stride, q_head_stride, k, v, ks, vs, table, q_start, kv_len, out, out_tok_stride, out_head_stride, ntok, requests, width, H, G, D, npages, page_tokens,
                   max_tokens, scale, dtype, workspace, workspace_bytes, false, 0, stream);
}
extern "C" int qspec_debug_kv8_attention_give_up(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const float* ks, const float* vs,
                                                 const int* table, const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok,
                                                 int requests, int width, int H, int G, int D, int npages, int page_tokens, int max_tokens, float scale, int dtype,
                                                 void* workspace, size_t workspace_bytes, unsigned give_up, void* stream) {
  return attention(q, q_tok_stride, q_head_stride, k, v, ks, vs, table, q_start, kv_len, out, out_tok_stride, out_head_stride, ntok, requests, width, H, G, D, npages, page_tokens,
                   max_tokens, scale, dtype, workspace, workspace_bytes, true, give_up, stream);
}
