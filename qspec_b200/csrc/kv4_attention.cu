// Softmax attention over a key/value cache in pages and in 4 bits (its layout and numbers: kv4_common.cuh). Token i of the n that request b has in the step stands at
// position kv_len[b] - n + i and sees the keys up to its own position.
//
// A row is a (token, query head of a group) pair; 16 rows of one key/value head are a tile of mma.sync.m16n8k16, so that the heads of a group and the
// tokens that verify a draft share every key that is read. What bounds it at these row counts is the cache: D + 4 bytes a key and head. How the work is spread over
// the GPU, and the parts joined: kv_stretch.cuh.
//
// Codes and words go from global memory into shared memory (16 bytes a lane, asynchronously, two units of 32 keys a warp under way) and from there into registers as the
// products' operands:
//   keys: a code c alone is the float16 c 2^-24, a subnormal number, which the tensor cores take exactly; one in the upper half of a byte is 16 c 2^-24, and meets a query
//   that has been divided by 16. One instruction makes two codes an operand. What the zero point takes from a score, z times the row's sum, is taken out in float32. The order of
//   the sum over a head's columns is free, so that a lane's words of a key are its operands as they lie; queries lie in shared memory in that order.
//   values: the transposing load of 16 x 16 bytes gives four keys of a column of bytes a word (the keys of the score tiles are numbered to match); a code behind 0x64 is the
//   float16 1024 + c, or 1024 + 16 c in the upper half, and one addition or multiply-add makes it c - z. (Sums over values must not carry an offset: over many
//   keys it cancels, and what the products cut off would be of the size of what is left.)
//
// Queries are multiplied by a power of two per row that brings their largest value to 2^14 .. 2^15 and are float16 from there on, exactly (what is below 2^-38 of the
// largest may lose bits). A key's scale multiplies its scores in float32. A value's scale v goes into the exponent: the weights 2^(9 + s + log2 v - m) lie below 2^15
// whatever the scales are and are rounded to float16 for the product with the codes (by 2^-11 of themselves at most, or by 2^-34 of the largest: kv8_common.cuh); the denominator
// is the sum of the unrounded weights / v.
#include "kv4_common.cuh"
#include "kv_stretch.cuh"

namespace qspec {
namespace kv4 {
using namespace kv8;

struct AttArgs : Step, Out {
  const void* q; long long q_ts; int q_hs;
  const uint8_t *k, *v;
  const uint16_t *kw, *vw;
  float scale2;                                  // scale * log2(e)
};

template <int D> struct Smem {
  static constexpr int ROW = D / 2, CODES = UNIT * ROW, STAGES = 2;
  static constexpr int WORDS = 2 * CODES, STAGE = WORDS + 2 * UNIT * 2;   // keys, values, words of either
  static constexpr int FACTORS = 16 * 16 * 2 + 8 * 16;                    // what the words of a unit's keys come to, in the order of the products
  static constexpr int WARP = STAGES * STAGE + FACTORS;
  static constexpr size_t RING = (size_t)WARPS * WARP;
  static constexpr size_t Q = ROWS * D * 2;
  static constexpr int LD = D + 8;                                      // floats of a row of sums on its way between warps
  static constexpr size_t SUMS = (size_t)WARPS * ROWS * LD * 4, PARTS = (size_t)(GRID_MOST + 1) * ROWS * 4;
  static constexpr size_t O = SUMS > PARTS ? SUMS : PARTS;              // sums on their way between warps, or a factor for every part of an item
  static constexpr size_t ML = (size_t)WARPS * ROWS * 2 * 4;
  static constexpr size_t F = ROWS * 4;                                 // the rows' powers of two
  static constexpr size_t TOTAL = RING + Q + O + ML + F;
  static_assert(STAGE % 16 == 0 && WARP % 16 == 0, "16-byte boundaries");
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two 16 x 16 blocks of bytes, columns first: word 2 m + h of a lane has rows 4 j .. 4 j + 3 (j = lane % 4) of column lane / 4 + 8 h of block m
__device__ __forceinline__ void load_columns(uint32_t (&w)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) { uint32_t x; asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(x) : "r"(addr) : "memory"); return x; }
__device__ __forceinline__ uint32_t lds16(uint32_t addr) { uint16_t x; asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(x) : "r"(addr) : "memory"); return x; }
__device__ __forceinline__ void lds128(uint32_t (&x)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds64(uint32_t (&x)[2], uint32_t addr) { asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(x[0]), "=r"(x[1]) : "r"(addr) : "memory"); }
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t x) { asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(addr), "r"(x) : "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t x) { asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(addr), "h"((uint16_t)x) : "memory"); }
__device__ __forceinline__ uint64_t two(float a, float b) { return pack_f2(a, b); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint32_t half_add(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_bits(float x) { return __half_as_ushort(__float2half_rn(x)); }

// Where the 16 bytes c of a row lie in a buffer, so that neither copies nor reads of eight rows meet in a bank (a row is half a line of banks, or a quarter).
template <int D> __device__ __forceinline__ uint32_t k_row(int row) {   // of eight lanes four read a row and four the row two behind it
  return (uint32_t)(D == 128 ? row * 64 ^ (row >> 1 & 1) << 6 : row * 32 ^ (row >> 2 & 1) << 5);
}
template <int D> __device__ __forceinline__ uint32_t v_chunk(int row, int c) {
  return (uint32_t)(D == 128 ? row * 64 + c * 16 ^ (row >> 1 & 3) << 4 : row * 32 + c * 16 ^ (row >> 2 & 1) << 4);
}

// A unit's codes and words: 16 rows lie in one page, whatever its size. Rows behind the last key are not fetched: what the buffer holds in their place is never used but as codes, which
// are codes like any other and meet weights of zero.
template <int D>
__device__ __forceinline__ void fetch(const AttArgs& a, const Unit& n, uint32_t dst, int lane) {
  using S = Smem<D>;
  constexpr int CH = D / 32, PER = 32 / CH;       // 16-byte pieces of a row; rows per instruction
  const int c = lane % CH, row0 = lane / CH, have = n.keys - n.key0;
#pragma unroll
  for (int q = 0; q < UNIT / 16; ++q) {
    const long long at = __shfl_sync(0xffffffffu, n.at, (16 * q) >> a.pshift);
    if (at < 0 || 16 * q >= have) continue;
    const size_t first = (size_t)at + ((n.key0 + 16 * q) & ((1 << a.pshift) - 1));   // row of the cache
    const uint8_t *ks = a.k + (first + row0) * S::ROW + c * 16, *vs = a.v + (first + row0) * S::ROW + c * 16;
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const int row = 16 * q + i * PER + row0;
      if (row < have) {
        copy16(dst + k_row<D>(row) + c * 16, ks + i * PER * S::ROW);
        copy16(dst + S::CODES + v_chunk<D>(row, c), vs + i * PER * S::ROW);
      }
    }
    if (lane < 4) copy16(dst + S::WORDS + (lane >> 1) * UNIT * 2 + q * 32 + (lane & 1) * 16, (lane >> 1 ? a.vw : a.kw) + first + (lane & 1) * 8);
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, CTAS) kv4_attention_kernel(const AttArgs a) {
  using T = typename Elem16<BF16>::T;
  using S = Smem<D>;
  constexpr int NT = D / 8, W = D / 32, KT = UNIT / 8, QT = UNIT / 16;   // column tiles of the value product, words that a lane has of a key, key tiles
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared s_sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, qi = lane >> 2, qj = lane & 3;
  unsigned char* const s_q = smem + S::RING;
  float* const s_o = reinterpret_cast<float*>(smem + S::RING + S::Q);
  float* const s_ml = reinterpret_cast<float*>(smem + S::RING + S::Q + S::O);   // [warp][maximum, sum][16]
  float* const s_f = reinterpret_cast<float*>(smem + S::RING + S::Q + S::O + S::ML);   // [16]
  const uint32_t ring = shared_addr(smem) + warp * S::WARP, factors = ring + S::STAGES * S::STAGE;
  pdl_enter();

  unsigned long long work;
  Stretch stretch;
  if (!find_stretch(a, s_sh, work, stretch)) return;
  Place cur = stretch.cur;                                  // the segment that all warps are in: (the rest of) one item
  const int todo = stretch.todo;

  // Queries of an item: a thread's pieces of 8 values (rows behind the last one are zeros), then float16 in the order in which the products take them: word (step, lane,
  // register) of the operand. A lane's word i of a key has columns 8 (W j + i) .. + 7; step 2 i takes the first and the second of each four of them, step 2 i + 1 the
  // third and the fourth.
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
      float x[8], mx = 0.f;
      unpack8<BF16>(queries[i], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
      for (int o = IN_ROW / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // 2^(14 - exponent of the largest), from its bits, in float32's range at both ends; none for a row of zeros or one that is not finite
      const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
      const bool some = mx > 0.f && mx < INFINITY;
      const int sh = some ? min(max(14 - ex, -126), 126) : 0;
      const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= e & 1 ? up * 0.0625f : up;
      if (qc == 0) s_f[row] = __uint_as_float((uint32_t)(some ? 127 - sh : 1) << 23);   // (those have no say in the tile's largest)
      uint32_t* to = reinterpret_cast<uint32_t*>(s_q) + (qc % W) * 2 * 128 + ((row & 7) * 4 + qc / W) * 4 + (row >> 3);
      to[0] = half_pair(x[0], x[4]);
      to[2] = half_pair(x[1], x[5]);
      to[128] = half_pair(x[2], x[6]);
      to[130] = half_pair(x[3], x[7]);
    }
  };

  // ---- the first units of this warp are on their way before anything else. Pages are looked up one unit ahead of the copies, so that these do not wait for them.
  int next = warp;                                          // index in the stretch of the unit that is fetched next
  Place np = cur;
  np.forward(a, work, warp);
  int pages = next < todo ? unit_page(a, np, lane) : -1;
  auto take = [&]() {                                       // the unit at np, and the pages of the one behind it
    Unit unit;
    unit.at = pages >= 0 ? (long long)(((size_t)pages * a.G + np.g) << a.pshift) : -1ll;
    unit.key0 = np.u * UNIT;
    unit.keys = next < todo ? np.r.keys : 0;
    np.forward(a, work, WARPS);
    next += WARPS;
    pages = next < todo ? unit_page(a, np, lane) : -1;
    return unit;
  };
  load_q(cur);
  Unit unit0 = take();
  fetch<D>(a, unit0, ring, lane);
  copy_commit();
  Unit unit1 = take();
  fetch<D>(a, unit1, ring + S::STAGE, lane);
  copy_commit();
  store_q();
  __syncthreads();

  int seg0 = 0;                                             // index in the stretch of the segment's first unit
  int here = warp;                                          // index of the unit that is in the ring's next stage
  uint32_t stage = 0;
  while (seg0 < todo) {
    const int seg_n = min(cur.r.units - cur.u, todo - seg0);
    const int tile = cur.tile;
    const uint32_t frag = shared_addr(s_q) + lane * 16;
    auto query = [&](uint32_t (&x)[4], int step) { lds128(x, frag + step * 512); };
    // The rows' powers of two: the tile's largest goes into the keys' factors, what a row is below it (at most 1) stays the row's.
    float big = s_f[0];
#pragma unroll
    for (int r = 1; r < ROWS; ++r) big = fmaxf(big, s_f[r]);
    const float own[2] = {s_f[qi] / big, s_f[qi + 8] / big}, factor = big * a.scale2;
    int limit[2];                                           // last visible position of this lane's rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = (tile * ROWS + qi + 8 * e) / a.rep;
      limit[e] = tok < cur.r.n ? min(cur.r.keys - cur.r.n + tok, cur.r.keys - 1) : -1;
    }
    const int low = cur.r.keys - cur.r.n + tile * ROWS / a.rep;   // the lowest of the tile's rows
    // the rows' sums, in units of 2^-24 like the scores
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) {
      uint32_t x[4];
      query(x, i);
      mma16816(sums, x, 0x00010001u, 0x00100010u);
    }
    const uint64_t sum2[2] = {two(sums[0], sums[0]), two(sums[2], sums[2])}, own2[2] = {two(own[0], own[0]), two(own[1], own[1])};
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m[2] = {NONE, NONE};
    uint64_t l2[2] = {0ull, 0ull};

    while (here < seg0 + seg_n) {
      const uint32_t buf = ring + stage * S::STAGE;
      const int key0 = unit0.key0, have = unit0.keys - key0;
      copy_wait<1>();
      __syncwarp();
      // ---- a lane a key: what its words come to. Key 16 q + 4 j + 2 b + z is column 2 j + b of score tile 2 q + z.
      {
        const int q = lane >> 4, j = lane >> 2 & 3, b = lane >> 1 & 1, z = lane & 1;
        const bool broken = __shfl_sync(0xffffffffu, unit0.at, (16 * q) >> a.pshift) < 0;
        const uint32_t kw = lds16(buf + S::WORDS + lane * 2), vw = lds16(buf + S::WORDS + UNIT * 2 + lane * 2);
        const float ks = word_scale(kw), vs = word_scale(vw);
        float f = fmaxf(positive(ks) * factor, 1.17549435e-38f) * 16777216.f, v = positive(vs);
        if (broken || !(ks < INFINITY) || !(vs < INFINITY)) { f = NAN; v = 1.f; }   // rows that see it are no numbers
        if (lane >= have) { f = 0.f; v = 1.f; }
        const uint32_t at = factors + ((q * 2 + z) * 4 + j) * 16 + b * 4;
        sts32(at, __float_as_uint(f));
        sts32(at + 8, __float_as_uint(-(float)(kw & 15u)));
        sts32(at + 256, __float_as_uint(__log2f(v)));
        sts32(at + 264, __float_as_uint(__fdividef(WEIGHT_UNIT, v)));
        const uint32_t zat = factors + 512 + (q * 4 + j) * 16 + z * 4 + b * 2;
        const float zero = (float)(vw & 15u);
        sts16(zat, half_bits(-1024.f - zero));
        sts16(zat + 8, half_bits(-64.f - zero));
      }
      // ---- scores of the unit's keys, in units of 2^-24
      float s[KT][4];
      {
        uint32_t w[KT][W];
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          const uint32_t at = buf + k_row<D>((n >> 1) * 16 + (n & 1) + (qi >> 1) * 4 + (qi & 1) * 2) + qj * (W * 4);
          if constexpr (W == 4) lds128(w[n], at); else lds64(w[n], at);
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint32_t x[4], y[4];
          query(x, 2 * i);
          query(y, 2 * i + 1);
#pragma unroll
          for (int n = 0; n < KT; ++n) mma16816(s[n], x, w[n][i] & 0x000f000fu, w[n][i] & 0x00f000f0u);
#pragma unroll
          for (int n = 0; n < KT; ++n) mma16816(s[n], y, w[n][i] >> 8 & 0x000f000fu, w[n][i] >> 8 & 0x00f000f0u);
        }
      }
      __syncwarp();                                         // (the factors are there)
      // ---- exponents
      uint64_t iv2[KT];
      float mx[2] = {NONE, NONE};
#pragma unroll
      for (int n = 0; n < KT; ++n) {
        uint32_t x[4], y[4];
        const uint32_t at = factors + (n * 4 + qj) * 16;
        lds128(x, at);
        lds128(y, at + 256);
        const uint64_t f = two(__uint_as_float(x[0]), __uint_as_float(x[1])), zero = two(__uint_as_float(x[2]), __uint_as_float(x[3])), lv = two(__uint_as_float(y[0]), __uint_as_float(y[1]));
        iv2[n] = two(__uint_as_float(y[2]), __uint_as_float(y[3]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint64_t score = ffma2_rn(zero, sum2[e], two(s[n][2 * e], s[n][2 * e + 1]));
          const float2 r = unpack_f2(ffma2_rn(score, mul2(f, own2[e]), lv));
          s[n][2 * e] = r.x;
          s[n][2 * e + 1] = r.y;
        }
      }
      if (key0 + UNIT - 1 > low) {                          // keys that a row does not see
#pragma unroll
        for (int n = 0; n < KT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + (n >> 1) * 16 + qj * 4 + (e & 1) * 2 + (n & 1) > limit[e >> 1]) s[n][e] = NONE;
      }
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) mx[e] = fmaxf(fmaxf(mx[e], s[n][2 * e]), s[n][2 * e + 1]);
      // The reference follows the maximum only where it has fallen behind: sums are seldom multiplied again.
      if (__any_sync(0xffffffffu, mx[0] > m[0] + GROWTH_LOG2 || mx[1] > m[1] + GROWTH_LOG2 || (m[0] == NONE && mx[0] > NONE) || (m[1] == NONE && mx[1] > NONE))) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
          const bool grown = mx[e] > m[e] + GROWTH_LOG2 || (m[e] == NONE && mx[e] > NONE);
          f[e] = grown && m[e] != NONE ? exp2_fast(m[e] - mx[e]) : 1.f;   // (a row that had seen nothing has sums of zero)
          if (grown) m[e] = mx[e];
          l2[e] = mul2(l2[e], two(f[e], f[e]));
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) { o[t][0] *= f[0]; o[t][1] *= f[0]; o[t][2] *= f[1]; o[t][3] *= f[1]; }
      }
      // ---- weights
      uint32_t pa[QT][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ref = m[e] == NONE ? 0.f : WEIGHT_LOG2 - m[e];
        const uint64_t ref2 = two(ref, ref);
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          const float2 x = unpack_f2(add2(two(s[n][2 * e], s[n][2 * e + 1]), ref2));
          const float w0 = exp2_fast(x.x), w1 = exp2_fast(x.y);
          l2[e] = ffma2_rn(two(w0, w1), iv2[n], l2[e]);
          pa[n >> 1][(n & 1) * 2 + e] = half_pair(w0, w1);
        }
      }
      // ---- values
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        uint32_t zero[4];
        lds128(zero, factors + 512 + (q * 4 + qj) * 16);
#pragma unroll
        for (int c = 0; c < W; c += 2) {                    // 64 columns at a time
          uint32_t w[4];
          load_columns(w, buf + S::CODES + v_chunk<D>(q * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t u = w[t], v = w[t] >> 8;
            mma16816(o[4 * c + 2 * t], pa[q], half_add((u & 0x000f000fu) | 0x64006400u, zero[0]), half_add((v & 0x000f000fu) | 0x64006400u, zero[1]));
            mma16816(o[4 * c + 2 * t + 1], pa[q], half_fma((u & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, zero[2]),
                     half_fma((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, zero[3]));   // (times 1 / 16)
          }
        }
      }
      __syncwarp();                                         // the unit behind the next takes this one's place
      unit0 = unit1;
      unit1 = take();
      fetch<D>(a, unit1, buf, lane);
      copy_commit();
      here += WARPS;
      stage ^= 1u;
    }

    Place after = cur;
    after.forward(a, work, seg_n);
    const bool more = seg0 + seg_n < todo;
    if (more) load_q(after);                                // the next segment's queries, on their way while sums are joined
    // ---- the warps' sums of this item together
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 both = unpack_f2(l2[e]);
      float l = both.x + both.y;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (qj == 0) {
        s_ml[(warp * 2) * ROWS + qi + 8 * e] = m[e];
        s_ml[(warp * 2 + 1) * ROWS + qi + 8 * e] = l;
      }
      // (a warp without a unit in this segment has nothing but its maximum to tell)
      if (m[e] != NONE || l != 0.f) {
        float* row = s_o + (warp * ROWS + qi + 8 * e) * S::LD + qj * 4;   // (bytes 2 j and 2 j + 1 of eight: four columns)
#pragma unroll
        for (int t = 0; t < NT; t += 2) *reinterpret_cast<float4*>(row + 8 * t) = make_float4(o[t][2 * e], o[t + 1][2 * e], o[t][2 * e + 1], o[t + 1][2 * e + 1]);
      }
    }
    finish_segment<BF16, D, S::LD>(a, a, stretch, cur, seg0, seg_n, s_ml, s_o, s_sh);
    if (more) store_q();                                    // (all have passed the barrier behind their last use of this item's)
    cur = after;
    seg0 += seg_n;
    __syncthreads();                                        // the sums have been read, the next queries are there
  }
  copy_wait<0>();
}

}  // namespace kv4
}  // namespace qspec

using namespace qspec;
using namespace qspec::kv4;

static int att_grid() { return max(sm_count(), 1) * CTAS; }

extern "C" size_t qspec_kv4_attention_workspace_bytes(void) { return 4096 + (size_t)att_grid() * 2 * PART<128> * sizeof(float); }

static int attention(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const void* k_word, const void* v_word, const int* table,
                     const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok, int requests, int width, int H, int G, int D, int npages,
                     int page_tokens, int max_tokens, float scale, int dtype, void* workspace, size_t workspace_bytes, bool always, unsigned give_up, void* stream) {
  QSPEC_REQUIRE(k && v && k_word && v_word && table && q_start && kv_len, QSPEC_ERR_INVALID_ARG, "kv4_attention: null pointer");
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "kv4_attention: pages of 16, 32, 64 or 128 tokens, got %d", page_tokens);
  QSPEC_REQUIRE(D == 64 || D == 128, QSPEC_ERR_UNSUPPORTED, "kv4_attention: heads of 64 or 128, got %d", D);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv4_attention: float16 or bfloat16 queries");
  QSPEC_REQUIRE(G >= 1 && H >= G && H % G == 0 && H <= 4096, QSPEC_ERR_INVALID_ARG, "kv4_attention: %d query heads, %d key/value heads", H, G);
  QSPEC_REQUIRE(scale > 0.f && scale < INFINITY, QSPEC_ERR_INVALID_ARG, "kv4_attention: scale must be positive and finite, got %g", (double)scale);
  QSPEC_REQUIRE(ntok >= 0 && ntok < (1 << 24) && requests >= 1 && width >= 1 && npages >= 1 && max_tokens >= 1 && (long long)npages * page_tokens < (1ll << 31) &&
                    (long long)width * page_tokens < (1ll << 31),
                QSPEC_ERR_INVALID_ARG, "kv4_attention: tokens=%d requests=%d width=%d pages=%d", ntok, requests, width, npages);
  if (ntok == 0) return QSPEC_OK;
  QSPEC_REQUIRE(q && out, QSPEC_ERR_INVALID_ARG, "kv4_attention: null pointer");
  auto aligned = [](const void* p, long long ts, int hs) { return ((uintptr_t)p & 15) == 0 && ts > 0 && hs > 0 && ts % 8 == 0 && hs % 8 == 0; };
  QSPEC_REQUIRE(aligned(q, q_tok_stride, q_head_stride) && aligned(out, out_tok_stride, out_head_stride) &&
                    (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_word | (uintptr_t)v_word) & 15) == 0,
                QSPEC_ERR_INVALID_ARG, "kv4_attention: rows must lie on 16-byte boundaries");
  QSPEC_REQUIRE(workspace && workspace_bytes >= qspec_kv4_attention_workspace_bytes() && ((uintptr_t)workspace & 15) == 0, QSPEC_ERR_WORKSPACE,
                "kv4_attention: %zu bytes of workspace needed, got %zu", qspec_kv4_attention_workspace_bytes(), workspace_bytes);
  const int grid = att_grid();
  QSPEC_REQUIRE(grid <= GRID_MOST, QSPEC_ERR_UNSUPPORTED, "kv4_attention: %d SMs", sm_count());
  // Requests with many rows may go to the prompt form (to_prompt_form()), in a launch of its own in front; none do if the call's rows are too few for a third of
  // the SMs (always: for tests).
  const int rep = H / G;
  const bool prompts = rep <= PROMPT_REP && (long long)max_tokens * rep >= PROMPT_ROWS && (always || (long long)ntok * H >= std::max(sm_count() / 3, 1) * 128ll);
  const unsigned share = always ? 1u : std::max(sm_count() / 4, 1) * 128u;
  if (prompts) {
    // Two tiles a CTA where the rows are more than the SMs take at once with one, by a quarter.
    const int pair = always ? give_up >> 4 & 1 : (long long)ntok * H > 160ll * sm_count();
    const PromptArgs4 pa{q, q_tok_stride, q_head_stride, (const uint8_t*)k, (const uint8_t*)v, (const uint16_t*)k_word, (const uint16_t*)v_word, table, q_start, kv_len, requests, width,
                         npages, page_shift(page_tokens), ntok, G, rep, pair, share, scale * 1.4426950408889634f, out, out_tok_stride, out_head_stride, give_up};
    if (const int rc = launch_prompt(pa, D, dtype == QSPEC_DTYPE_BF16, (cudaStream_t)stream)) return rc;
  }
  const AttArgs a{{table, q_start, kv_len, requests, width, npages, page_shift(page_tokens), ntok, G, rep, prompts ? share : 0u},
                  {out, out_tok_stride, out_head_stride, (int*)workspace, (float*)((char*)workspace + 4096)}, q, q_tok_stride, q_head_stride, (const uint8_t*)k, (const uint8_t*)v,
                  (const uint16_t*)k_word, (const uint16_t*)v_word, scale * 1.4426950408889634f};
  auto run = [&](auto kern, size_t smem, SmemLimit& limit) -> int {
    QSPEC_CUDA(limit.raise(kern, smem));
    QSPEC_CUDA(launch_pdl(kern, dim3(grid), dim3(THREADS), smem, (cudaStream_t)stream, a));
    QSPEC_CHECK_LAUNCH(1);
    return QSPEC_OK;
  };
  static SmemLimit limits[4];
  if (dtype == QSPEC_DTYPE_F16)
    return D == 128 ? run(kv4_attention_kernel<false, 128>, Smem<128>::TOTAL, limits[0]) : run(kv4_attention_kernel<false, 64>, Smem<64>::TOTAL, limits[1]);
  return D == 128 ? run(kv4_attention_kernel<true, 128>, Smem<128>::TOTAL, limits[2]) : run(kv4_attention_kernel<true, 64>, Smem<64>::TOTAL, limits[3]);
}

extern "C" int qspec_kv4_attention(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const void* k_word, const void* v_word, const int* table,
                                   const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok, int requests, int width, int H,
                                   int G, int D, int npages, int page_tokens, int max_tokens, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(q, q_tok_stride, q_head_stride, k, v, k_word, v_word, table, q_start, kv_len, out, out_tok_stride, out_head_stride, ntok, requests, width, H, G, D, npages,
                   page_tokens, max_tokens, scale, dtype, workspace, workspace_bytes, false, 0, stream);
}
extern "C" int qspec_debug_kv4_attention_give_up(const void* q, long long q_tok_stride, int q_head_stride, const void* k, const void* v, const void* k_word, const void* v_word,
                                                 const int* table, const int* q_start, const int* kv_len, void* out, long long out_tok_stride, int out_head_stride, int ntok,
                                                 int requests, int width, int H, int G, int D, int npages, int page_tokens, int max_tokens, float scale, int dtype,
                                                 void* workspace, size_t workspace_bytes, unsigned give_up, void* stream) {
  return attention(q, q_tok_stride, q_head_stride, k, v, k_word, v_word, table, q_start, kv_len, out, out_tok_stride, out_head_stride, ntok, requests, width, H, G, D, npages,
                   page_tokens, max_tokens, scale, dtype, workspace, workspace_bytes, true, give_up, stream);
}
