// Softmax attention over a key/value cache in pages and in 4 bits (its layout and numbers: kv4_common.cuh). Token i of the n that request b has in the step stands at
// position kv_len[b] - n + i and sees the keys up to its own position.
//
// A row is a (token, query head of a group) pair; 16 rows of one key/value head (or 8) are a tile of mma.sync.m16n8k16, so that the heads of a group and the
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
// Queries are multiplied by a power of two per row that brings their largest value to 2^14 .. 2^15 and are float16 from there on, exactly (but for the last bits of what is below 2^-24
// of the largest, and all of what is below 2^-34: odd columns are divided by 16). A key's scale multiplies its scores in float32. A value's scale v goes into the exponent: the weights 2^(9 + s + log2 v - m) lie below 2^15
// whatever the scales are and are rounded to float16 for the product with the codes (by 2^-11 of themselves at most, or by 2^-34 of the largest: kv8_common.cuh); the denominator
// is the sum of the unrounded weights / v.
//
// Measured: 64 requests of 4 tokens after some 3000 keys each, 32 / 8 heads of 128, 76 us, 2.7 TB/s of codes and words; one token after 131071 keys, 64 / 8 heads, 45 us, 3.1 TB/s; 4 requests of a
// token after some 680 keys 12 us, which is launches and a chain of loads. At this many rows not the bytes bound it (two fifths of the time) but instructions: a unit of 32 keys takes a
// warp some 650, of which 64 are products and 250 make codes operands; the tensor cores are busy 38 % of a long walk, the units of integer arithmetic 45 %.
#include "kv4_common.cuh"
#include "kv_stretch.cuh"

namespace qspec {
namespace kv4 {
using namespace kv8;

// Tiles of sixteen rows (tokens x heads of a group), or of eight where no request has more: then codes are the products' first operand, rows the second, of eight columns, and half
// of the products, exponentials and sums' registers go. us of eight (of sixteen), 32 / 8 heads of 128, one token a request: 64 requests after 3000 keys 58 (76), after 700: 22 (34);
// 256 after 1000: 86 (106); 4 after 676: 11.7 (12.8); one of 2 after 20000: 21 (24); one after 131071, 64 / 8 heads: 46 (57).
// CTAs of an SM (while one waits at a barrier the others compute): three of four warps; four, for tiles of eight, where requests x heads of keys are more than three CTAs an SM, so that each
// may still have CTAs of its own. us with three (with four), a token each: 16 requests after 3000 keys 25 (26), 32: 40 (38), 48: 45 (52), 64: 62 (58), after 700 keys 30 (22); one after
// 131071 46 (52). Heads of 64, where four a SM spill 372 bytes, the same: 32 / 8 heads, 16 requests after 3000 keys 17.5 (19.5), 32: 23.7 (25.9), 64: 40.4 (39.9), 128: 68.4 (65.9), 64 after 700: 23.0 (15.9), 256 after
// 1000: 65.6 (58.9), one after 60000 23.0 (29.7); 64 / 16 heads, 16 after 3000 26.8 (26.2), 32: 40.6 (38.7), 128: 121 (113), 256 after 1000: 112 (103). Two of eight warps: 66, 32, 52; five of four: 67, 26, 58. Tiles of sixteen, 64 requests of 4 tokens after 3000, after 748 keys, one of 4 after 20000: two of eight warps 86, 40, 27; three of
// four 77, 32, 27; four of four 78, 28, 36.
constexpr int WARPS = 4, THREADS = WARPS * 32, SMS_MOST = 160, CTAS_MOST = 4;

struct AttArgs : Step, Out {
  const void* q; long long q_ts; int q_hs;
  const uint8_t *k, *v;
  const uint16_t *kw, *vw;
  float scale2;                                  // scale * log2(e)
};

template <int D, int TR> struct Smem {
  static constexpr int ROW = D / 2, CODES = UNIT * ROW, STAGES = 2;
  static constexpr int WORDS = 2 * CODES, STAGE = WORDS + 2 * UNIT * 2;   // keys, values, words of either
  static constexpr int FACTORS = 16 * 16 * 2 + 8 * 16;                    // what the words of a unit's keys come to, in the order of the products
  static constexpr int WARP = STAGES * STAGE + FACTORS;
  static constexpr int LD = D + 8;                                      // floats of a row of sums on its way between warps
  // units, or (at a segment's end) sums on their way between warps, or a factor for every part of an item
  static constexpr size_t RING = (size_t)WARPS * WARP, SUMS = (size_t)WARPS * TR * LD * 4, PARTS = (size_t)(SMS_MOST * CTAS_MOST + 1) * TR * 4;
  static constexpr size_t ROOM = RING > SUMS ? (RING > PARTS ? RING : PARTS) : SUMS > PARTS ? SUMS : PARTS;
  static constexpr size_t Q = TR * D * 2;
  static constexpr size_t ML = (size_t)WARPS * TR * 2 * 4;
  static constexpr size_t F = TR * 4;                                 // the rows' powers of two
  static constexpr size_t TOTAL = ROOM + Q + ML + F;
  static_assert(STAGE % 16 == 0 && WARP % 16 == 0 && ROOM % 16 == 0, "16-byte boundaries");
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// (x & mask) | magic in one instruction, which two constants would make two: they are kept in registers.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) { uint32_t r; asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(r) : "r"(x), "r"(mask), "r"(magic)); return r; }
// an 8 x 8 matrix of 16-bit values, two of a row a lane, columns for rows
__device__ __forceinline__ uint32_t turned(uint32_t x) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x)); return r; }
__device__ __forceinline__ uint32_t held(uint32_t x) { uint32_t r; asm volatile("mov.b32 %0, %1;\n" : "=r"(r) : "r"(x)); return r; }

// Where the 16 bytes c of a row lie in a buffer, so that neither copies nor reads of eight rows meet in a bank (a row is half a line of banks, or a quarter).
template <int D> __device__ __forceinline__ uint32_t k_row(int row) {   // of eight lanes four read a row and four the row two behind it
  return (uint32_t)(D == 128 ? row * 64 ^ (row >> 1 & 1) << 6 : row * 32 ^ (row >> 2 & 1) << 5);
}
template <int D> __device__ __forceinline__ uint32_t v_chunk(int row, int c) {
  return (uint32_t)(D == 128 ? row * 64 + c * 16 ^ (row >> 1 & 3) << 4 : row * 32 + c * 16 ^ (row >> 2 & 1) << 4);
}

// A unit's codes and words that lie in two pages, or are fewer than UNIT: 16 rows at a time. Rows behind the last key are not fetched: what the buffer holds in their place is never used
// but as codes, which are codes like any other and meet weights of zero.
template <int D>
__device__ __noinline__ void fetch_parts(const uint8_t* k, const uint8_t* v, const uint16_t* kw, const uint16_t* vw, int pshift, long long row, int have, uint32_t dst) {
  using S = Smem<D, ROWS>;
  constexpr int CH = D / 32, PER = 32 / CH;       // 16-byte pieces of a row; rows per instruction
  const int lane = threadIdx.x & 31, c = lane % CH, row0 = lane / CH;
#pragma unroll 1
  for (int q = 0; q < UNIT / 16; ++q) {
    const long long at = __shfl_sync(0xffffffffu, row, q);
    if (at < 0 || 16 * q >= have) continue;
    const size_t first = (size_t)at + (pshift >= 5 ? 16 * q : 0);
#pragma unroll 1
    for (int r = row0; r < 16; r += PER)
      if (16 * q + r < have) {
        copy16(dst + k_row<D>(16 * q + r) + c * 16, k + (first + r) * S::ROW + c * 16);
        copy16(dst + S::CODES + v_chunk<D>(16 * q + r, c), v + (first + r) * S::ROW + c * 16);
      }
    if (lane < 4) copy16(dst + S::WORDS + (lane >> 1) * UNIT * 2 + q * 32 + (lane & 1) * 16, (lane >> 1 ? vw : kw) + first + (lane & 1) * 8);
  }
}

template <bool BF16, int D, int TR, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) kv4_attention_kernel(const AttArgs a) {
  using T = typename Elem16<BF16>::T;
  using S = Smem<D, TR>;
  constexpr bool FEW = TR == 8;
  constexpr int NT = D / (FEW ? 16 : 8), W = D / 32, KT = UNIT / 8, QT = UNIT / 16;   // column tiles of the value product, words that a lane has of a key, key tiles
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared<WARPS> s_sh;
  __shared__ Stretch s_stretch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, qi = lane >> 2, qj = lane & 3;
  unsigned char* const s_q = smem + S::ROOM;
  float* const s_o = reinterpret_cast<float*>(smem);
  float* const s_ml = reinterpret_cast<float*>(smem + S::ROOM + S::Q);   // [warp][maximum, sum][TR]
  float* const s_f = reinterpret_cast<float*>(smem + S::ROOM + S::Q + S::ML);   // [TR]
  const uint32_t ring = shared_addr(smem) + warp * S::WARP, factors = ring + S::STAGES * S::STAGE;
  pdl_enter();

  // The stretch stays in shared memory (its place is that of the segment that all warps are in: the rest of one item): registers are what there is least of.
  unsigned long long work;
  {
    Stretch stretch;
    if (!find_stretch<WARPS, SMS_MOST * CTAS, TR>(a, s_sh, work, stretch)) return;
    if (tid == 0) s_stretch = stretch;
  }

  // Queries of an item: a thread's pieces of 8 values (rows behind the last one are zeros), then float16 in the order in which the products take them: word (step, lane,
  // register) of the operand. A lane's word i of a key has columns 8 (W j + i) .. + 7; step 2 i takes the first and the second of each four of them, step 2 i + 1 the
  // third and the fourth.
  constexpr int IN_ROW = D / 8;
  constexpr int AT_ONCE = THREADS / IN_ROW, PIECES = (TR + AT_ONCE - 1) / AT_ONCE;   // rows; pieces of a thread
  const int qr = tid / IN_ROW, qc = tid % IN_ROW;
  auto load_q = [&](const Place& p, uint4 (&pieces)[PIECES]) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int r = qr + i * AT_ONCE, row = p.tile * TR + r, tok = row / a.rep;
      pieces[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < TR && tok < p.r.n)
        pieces[i] = *reinterpret_cast<const uint4*>((const T*)a.q + (size_t)(p.r.first + tok) * a.q_ts + (size_t)(p.g * a.rep + row - tok * a.rep) * a.q_hs + qc * 8);
    }
  };
  auto store_q = [&](const uint4& piece, int r) {
    float x[8], mx = 0.f;
    unpack8<BF16>(piece, x);
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
    if (r >= TR) return;
    if (qc == 0) s_f[r] = __uint_as_float((uint32_t)(some ? 127 - sh : 1) << 23);   // (those have no say in the tile's largest)
    constexpr int STEP = 8 * TR, REG = TR / 8;              // words of a step; from a register of a row to the row's next
    uint32_t* to = reinterpret_cast<uint32_t*>(s_q) + (qc % W) * 2 * STEP + ((r & 7) * 4 + qc / W) * 2 * REG + (r >> 3);
    to[0] = half_pair(x[0], x[4]);
    to[REG] = half_pair(x[1], x[5]);
    to[STEP] = half_pair(x[2], x[6]);
    to[STEP + REG] = half_pair(x[3], x[7]);
  };

  // ---- a segment's units: warp w's are w, w + WARPS, .., two of them under way. Pages are looked up two units ahead of the copies, so that these do not wait for them: a unit lies in one
  // page, or (of 16 tokens) in two, of which odd lanes have the second.
  const int mask = (1 << a.pshift) - 1, second = a.pshift == 4 ? lane & 1 : 0;
  const int* table;                                         // the segment's request's
  int g = 0, keys = 0, next = 0, end = 0;                   // its head and keys; the unit that is fetched next, the end of the segment's units
  auto look = [&](int unit) {
    if (unit >= end) return -1;
    const int at = (unit * UNIT >> a.pshift) + second;
    if ((at << a.pshift) >= keys || at >= a.width) return -1;
    const int page = table[at];
    return (unsigned)page < (unsigned)a.npages ? page : -1;
  };
  int pages, then;                                          // of the next unit, of the one behind it
  struct Unit4 {
    bool there;                                             // this lane's page
    int key0;                                               // first key
  };
  // a lane's places in a unit that lies in one page: 512 bytes of codes an instruction, of which its 16 are always in the same place of their rows
  const uint32_t kdst = k_row<D>(lane / (D / 32)) + lane % (D / 32) * 16, vdst = v_chunk<D>(lane / (D / 32), lane % (D / 32));
  const uint32_t wdst = S::WORDS + (lane & 7) * 16;
  auto take = [&](uint32_t dst) {                           // the next unit, and the pages of the one two behind it
    Unit4 unit;
    unit.there = pages >= 0;
    unit.key0 = next * UNIT;
    const int have = next < end ? keys - unit.key0 : 0;
    const long long row = unit.there ? (long long)((((size_t)pages * a.G + g) << a.pshift) + (unit.key0 & mask)) : -1ll;
    if (a.pshift >= 5 && have >= UNIT) {                    // (the same for all lanes)
      if (unit.there) {
        const long long off = row * S::ROW + lane * 16;
        const uint8_t *ks = a.k + off, *vs = a.v + off;
#pragma unroll
        for (int i = 0; i < S::CODES / 512; ++i) {
          // (what a row's number shifts its pieces by repeats after eight rows)
          copy16(dst + kdst + i * 512, ks + i * 512);
          copy16(dst + S::CODES + vdst + i * 512, vs + i * 512);
        }
        if (lane < 8) copy16(dst + wdst, (lane & 4 ? a.vw : a.kw) + row + (lane & 3) * 8);
      }
    } else {
      fetch_parts<D>(a.k, a.v, a.kw, a.vw, a.pshift, row, have, dst);
    }
    copy_commit();
    next += WARPS;
    pages = then;
    then = look(next + WARPS);
    return unit;
  };

  const uint32_t low4 = held(0x000f000fu), high4 = held(0x00f000f0u), magic = held(0x64006400u);
  // where this lane's key leaves what it comes to
  const uint32_t words = ring + S::WORDS + lane * 2;
  const uint32_t mine = FEW ? factors + (((lane >> 4) * 2 + (lane & 1)) * 8 + (lane >> 1 & 7)) * 16 : factors + (((lane >> 4) * 2 + (lane & 1)) * 4 + (lane >> 2 & 3)) * 16 + (lane >> 1 & 1) * 4;
  const uint32_t zeros = factors + 512 + ((lane >> 4) * 4 + (lane >> 2 & 3)) * 16 + (lane & 1) * 4 + (lane >> 1 & 1) * 2;
  int seg0 = 0;                                             // index in the stretch of the segment's first unit
  __syncthreads();
  for (;;) {
    const Place cur = s_stretch.cur;
    const int seg_n = min(cur.r.units - cur.u, s_stretch.todo - seg0);
    const int tile = cur.tile;
    table = a.table + (size_t)cur.b * a.width;
    g = cur.g;
    keys = cur.r.keys;
    next = cur.u + warp;
    end = cur.u + seg_n;
    pages = look(next);
    then = look(next + WARPS);
    uint4 pieces[PIECES];
    load_q(cur, pieces);
    Unit4 unit0 = take(ring), unit1 = take(ring + S::STAGE);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) store_q(pieces[i], qr + i * AT_ONCE);
    __syncthreads();
    uint32_t stage = 0;
    const uint32_t frag = shared_addr(s_q) + lane * TR;
    auto query = [&](uint32_t (&x)[TR / 4], int step) { if constexpr (FEW) lds64(x, frag + step * 256); else lds128(x, frag + step * 512); };
    // The rows' powers of two: the tile's largest goes into the keys' factors, what a row is below it (at most 1) stays the row's,
    // with the scores' unit: scores times that first, so that neither leaves float32 where the whole does not.
    float big = s_f[0];
#pragma unroll
    for (int r = 1; r < TR; ++r) big = fmaxf(big, s_f[r]);
    const int row0 = FEW ? 2 * qj : qi, row1 = FEW ? 2 * qj + 1 : qi + 8;   // this lane's rows of the tile
    const float own[2] = {s_f[row0] / big * 16777216.f, s_f[row1] / big * 16777216.f}, factor = big * a.scale2;
    int limit[2];                                           // last visible position of this lane's rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = (tile * TR + (e ? row1 : row0)) / a.rep;
      limit[e] = tok < cur.r.n ? min(cur.r.keys - cur.r.n + tok, cur.r.keys - 1) : -1;
    }
    const int low = cur.r.keys - cur.r.n + tile * TR / a.rep;   // the lowest of the tile's rows
    // the rows' sums, in units of 2^-24 like the scores
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t qf[FEW ? 2 * W : 1][2];                        // (eight rows' queries stay in registers)
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) {
      if constexpr (FEW) {
        const uint32_t ones[4] = {0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u};
        query(qf[i], i);
        mma16816(sums, ones, qf[i][0], qf[i][1]);
      } else {
        uint32_t x[4];
        query(x, i);
        mma16816(sums, x, 0x00010001u, 0x00100010u);
      }
    }
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m[2] = {NONE, NONE};                              // what exponents are counted from
    uint64_t l2[2] = {0ull, 0ull};                          // sums of weights / v

    for (int here = cur.u + warp; here < end; here += WARPS) {
      const uint32_t buf = ring + stage * S::STAGE;
      const int key0 = unit0.key0;
      copy_wait<1>();
      __syncwarp();
      // ---- a lane a key: what its words come to. Key 16 q + 4 j + 2 b + z is column 2 j + b of score tile 2 q + z.
      {
        const bool broken = !(__ballot_sync(0xffffffffu, unit0.there) >> (lane >> 4) & 1u);
        const uint32_t kw = lds16(words + stage * S::STAGE), vw = lds16(words + stage * S::STAGE + UNIT * 2);
        const bool bad = broken || kw >= 0xff00u || vw >= 0xff00u;   // (exponent 255: infinite, or no number)
        float f = fminf(word_scale(kw) * factor, 3.402823466e38f), v = fmaxf(word_scale(vw), 7.888609052210118e-31f);   // (a score of nothing stays that)
        if (bad) { f = NAN; v = 1.f; }                      // rows that see it are no numbers
        if (key0 + lane >= keys) f = 0.f;
        const uint32_t x[4] = {__float_as_uint(f), __float_as_uint(__uint_as_float(0xcb000000u | (kw & 15u)) + 8388608.f) /* - z */, __float_as_uint(__log2f(v)),
                               __float_as_uint(over_scale(WEIGHT_UNIT, v))};
        if constexpr (FEW) {
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(mine), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
        } else {
          sts32(mine, x[0]);
          sts32(mine + 8, x[1]);
          sts32(mine + 256, x[2]);
          sts32(mine + 264, x[3]);
        }
        sts16(zeros, 0xe400u + (vw & 15u));                 // -1024 - z
        sts16(zeros + 8, 0xd400u + ((vw & 15u) << 4));      // -64 - z
      }
      // ---- scores of the unit's keys, in units of 2^-24
      float s[FEW ? QT : KT][4];                            // few rows: of 16 keys, [key 2 j + b and the next][this lane's rows]
      {
        uint32_t w[KT][W];
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          const uint32_t at = buf + k_row<D>((n >> 1) * 16 + (n & 1) + (qi >> 1) * 4 + (qi & 1) * 2) + qj * (W * 4);
          if constexpr (W == 4) lds128(w[n], at); else lds64(w[n], at);
        }
        if constexpr (FEW) {
#pragma unroll
          for (int i = 0; i < W; ++i)
#pragma unroll
            for (int q = 0; q < QT; ++q) {
              const uint32_t u = w[2 * q][i], v = w[2 * q + 1][i];
              const uint32_t x[4] = {u & 0x000f000fu, v & 0x000f000fu, u & 0x00f000f0u, v & 0x00f000f0u};
              const uint32_t y[4] = {u >> 8 & 0x000f000fu, v >> 8 & 0x000f000fu, u >> 8 & 0x00f000f0u, v >> 8 & 0x00f000f0u};
              if (i == 0) mma16816_first(s[q], x, qf[0][0], qf[0][1]); else mma16816(s[q], x, qf[2 * i][0], qf[2 * i][1]);
              mma16816(s[q], y, qf[2 * i + 1][0], qf[2 * i + 1][1]);
            }
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) {
            uint32_t x[4], y[4];
            query(x, 2 * i);
            query(y, 2 * i + 1);
#pragma unroll
            for (int n = 0; n < KT; ++n) {
              if (i == 0) mma16816_first(s[n], x, w[n][i] & 0x000f000fu, w[n][i] & 0x00f000f0u);
              else mma16816(s[n], x, w[n][i] & 0x000f000fu, w[n][i] & 0x00f000f0u);
            }
#pragma unroll
            for (int n = 0; n < KT; ++n) mma16816(s[n], y, w[n][i] >> 8 & 0x000f000fu, w[n][i] >> 8 & 0x00f000f0u);
          }
        }
      }
      __syncwarp();                                         // (the factors are there)
      // ---- exponents
      float mx[2] = {NONE, NONE};
      uint64_t iv2[FEW ? KT : 1];                           // unit / v of this lane's keys, twice
      if constexpr (FEW) {
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          uint32_t x[4];
          lds128(x, factors + (n * 8 + qi) * 16);
          const float f = __uint_as_float(x[0]), zero = __uint_as_float(x[1]), lv = __uint_as_float(x[2]), iv = __uint_as_float(x[3]);
          float* const y = s[n >> 1] + (n & 1) * 2;
          const uint64_t score = ffma2_rn(two(zero, zero), two(sums[0], sums[1]), two(y[0], y[1]));
          const float2 r = unpack_f2(ffma2_rn(mul2(score, two(own[0], own[1])), two(f, f), two(lv, lv)));
          y[0] = r.x;
          y[1] = r.y;
          iv2[n] = two(iv, iv);
        }
        if (key0 + UNIT - 1 > low) {                        // keys that a row does not see
#pragma unroll
          for (int n = 0; n < KT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key0 + (n >> 1) * 16 + (qi >> 1) * 4 + (qi & 1) * 2 + (n & 1) > limit[e]) s[n >> 1][(n & 1) * 2 + e] = NONE;
        }
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) mx[e] = fmaxf(fmaxf(mx[e], s[q][e]), s[q][2 + e]);
      } else {
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          uint32_t x[4], y[2];
          const uint32_t at = factors + (n * 4 + qj) * 16;
          lds128(x, at);
          lds64(y, at + 256);
          const uint64_t f = two(__uint_as_float(x[0]), __uint_as_float(x[1])), zero = two(__uint_as_float(x[2]), __uint_as_float(x[3])), lv = two(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint64_t score = ffma2_rn(zero, two(sums[2 * e], sums[2 * e]), two(s[n][2 * e], s[n][2 * e + 1]));
            const float2 r = unpack_f2(ffma2_rn(mul2(score, two(own[e], own[e])), f, lv));
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
      }
      // The reference follows the maximum only where that is 2^TOP_LOG2 and more above it: sums are seldom multiplied again. It is WEIGHT_LOG2 below the maximum, rounded up: far from zero
      // that is less, and weights that are counted from what it is, and the comparison with their own difference, stay finite.
      constexpr float TOP_LOG2 = WEIGHT_LOG2 + GROWTH_LOG2;
      if (__any_sync(0xffffffffu, mx[0] - m[0] > TOP_LOG2 || mx[1] - m[1] > TOP_LOG2)) {   // (of a row that had seen nothing: infinite, or nothing again and no number)
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = FEW ? 4 : 1; x < (FEW ? 32 : 4); x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
          const bool grown = mx[e] - m[e] > TOP_LOG2;
          const float to = __fadd_ru(mx[e], -WEIGHT_LOG2);
          f[e] = grown && m[e] != NONE ? exp2_fast(m[e] - to) : 1.f;   // (a row that had seen nothing has sums of zero)
          if (grown) m[e] = to;
          if (!FEW) l2[e] = mul2(l2[e], two(f[e], f[e]));
        }
        if (FEW) l2[0] = mul2(l2[0], two(f[0], f[1]));
#pragma unroll
        for (int t = 0; t < NT; ++t) { o[t][0] *= f[0]; o[t][1] *= f[FEW]; o[t][2] *= f[!FEW]; o[t][3] *= f[1]; }
      }
      // ---- weights
      uint32_t pa[QT][TR / 4];
      const float ref[2] = {m[0] == NONE ? 0.f : -m[0], m[1] == NONE ? 0.f : -m[1]};
      if constexpr (FEW) {
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          const float* const y = s[n >> 1] + (n & 1) * 2;
          const float2 x = unpack_f2(add2(two(y[0], y[1]), two(ref[0], ref[1])));
          const float w0 = exp2_fast(x.x), w1 = exp2_fast(x.y);
          l2[0] = ffma2_rn(two(w0, w1), iv2[n], l2[0]);
          pa[n >> 1][n & 1] = turned(half_pair(w0, w1));    // (a lane has two rows of a key; the product takes two keys of a row)
        }
      } else {
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          uint32_t y[2];
          lds64(y, factors + (n * 4 + qj) * 16 + 264);
          const uint64_t iv = two(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 x = unpack_f2(add2(two(s[n][2 * e], s[n][2 * e + 1]), two(ref[e], ref[e])));
            const float w0 = exp2_fast(x.x), w1 = exp2_fast(x.y);
            l2[e] = ffma2_rn(two(w0, w1), iv, l2[e]);
            pa[n >> 1][(n & 1) * 2 + e] = half_pair(w0, w1);
          }
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
          if constexpr (FEW) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t u0 = w[2 * t], v0 = u0 >> 8, u1 = w[2 * t + 1], v1 = u1 >> 8;
              const uint32_t x[4] = {half_add(and_or(u0, low4, magic), zero[0]), half_add(and_or(u1, low4, magic), zero[0]), half_add(and_or(v0, low4, magic), zero[1]),
                                     half_add(and_or(v1, low4, magic), zero[1])};
              mma16816(o[2 * (c + t)], x, pa[q][0], pa[q][1]);
              const uint32_t y[4] = {half_fma(and_or(u0, high4, magic), 0x2c002c00u, zero[2]), half_fma(and_or(u1, high4, magic), 0x2c002c00u, zero[2]),
                                     half_fma(and_or(v0, high4, magic), 0x2c002c00u, zero[3]), half_fma(and_or(v1, high4, magic), 0x2c002c00u, zero[3])};   // (times 1 / 16)
              mma16816(o[2 * (c + t) + 1], y, pa[q][0], pa[q][1]);
            }
          } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint32_t u = w[t], v = w[t] >> 8;
              mma16816(o[4 * c + 2 * t], pa[q], half_add(and_or(u, low4, magic), zero[0]), half_add(and_or(v, low4, magic), zero[1]));
              mma16816(o[4 * c + 2 * t + 1], pa[q], half_fma(and_or(u, high4, magic), 0x2c002c00u, zero[2]),
                       half_fma(and_or(v, high4, magic), 0x2c002c00u, zero[3]));   // (times 1 / 16)
            }
          }
        }
      }
      __syncwarp();                                         // the unit behind the next takes this one's place
      unit0 = unit1;
      unit1 = take(buf);
      stage ^= 1u;
    }
    copy_wait<0>();
    __syncthreads();                                        // (sums take the units' place)

    // ---- the warps' sums of this item together
    const float2 l0 = unpack_f2(l2[0]), l1 = unpack_f2(l2[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = FEW ? (e ? l0.y : l0.x) : e ? l1.x + l1.y : l0.x + l0.y;
#pragma unroll
      for (int x = FEW ? 4 : 1; x < (FEW ? 32 : 4); x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      const int r = e ? row1 : row0;
      if ((FEW ? qi : qj) == 0) {
        s_ml[(warp * 2) * TR + r] = m[e];
        s_ml[(warp * 2 + 1) * TR + r] = l;
      }
      // (a warp without a unit in this segment has nothing but its maximum to tell)
      if (m[e] != NONE || l != 0.f) {
        float* row = s_o + (warp * TR + r) * S::LD + (FEW ? qi * 2 : qj * 4);
        if constexpr (FEW) {                                // (bytes j and j + 8 of sixteen: two columns each)
#pragma unroll
          for (int t = 0; t < NT; t += 2) {
            *reinterpret_cast<float2*>(row + 16 * t) = make_float2(o[t][e], o[t + 1][e]);
            *reinterpret_cast<float2*>(row + 16 * t + 16) = make_float2(o[t][2 + e], o[t + 1][2 + e]);
          }
        } else {                                            // (bytes 2 j and 2 j + 1 of eight: four columns)
#pragma unroll
          for (int t = 0; t < NT; t += 2) *reinterpret_cast<float4*>(row + 8 * t) = make_float4(o[t][2 * e], o[t + 1][2 * e], o[t][2 * e + 1], o[t + 1][2 * e + 1]);
        }
      }
    }
    finish_segment<BF16, D, S::LD, WARPS, TR>(a, a, s_stretch, s_stretch.cur, seg0, seg_n, s_ml, s_o, s_sh);
    seg0 += seg_n;
    if (seg0 >= s_stretch.todo) break;
    __syncthreads();                                        // the sums have been read, and so has the segment's place
    if (tid == 0) s_stretch.cur.forward<TR>(a, work, seg_n);
    __syncthreads();
  }
}

}  // namespace kv4
}  // namespace qspec

using namespace qspec;
using namespace qspec::kv4;


extern "C" size_t qspec_kv4_attention_workspace_bytes(void) { return 4096 + (size_t)std::max(sm_count(), 1) * std::max(CTAS_MOST * PART<128, 8>, 3 * PART<128>) * 2 * sizeof(float); }

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
  QSPEC_REQUIRE(sm_count() <= SMS_MOST, QSPEC_ERR_UNSUPPORTED, "kv4_attention: %d SMs", sm_count());
  // Requests with many rows may go to the prompt form (to_prompt_form()), in a launch of its own in front; none do if the call's rows are too few for a third of
  // the SMs (always: for tests). Both forms measured, 32 / 8 heads of 128, us of the prompt form (of the other):
  //   1 request, 1000 keys in front of it   32 tokens 37 (19)   128: 37 (23)   160: 38 (39)   256: 38 (51)   1024: 71 (204)
  //   1 request, 32000 keys                 128 tokens 493 (345)   256: 499 (610)   512: 588 (1195)
  //   4 requests, 8000 keys                 17 tokens 139 (73)   48: 143 (145)   64: 151 (180)   128: 168 (333)
  //   16 requests, 1000 keys                17 tokens 37 (54)   64: 50 (138)   128: 88 (258)
  const int rep = H / G;
  const bool prompts = rep <= PROMPT_REP && (long long)max_tokens * rep >= PROMPT_ROWS && (always || (long long)ntok * H >= std::max(sm_count() / 3, 1) * 128ll);
  const unsigned share = always ? 1u : std::max(sm_count() / 4, 1) * 128u;
  if (prompts) {
    // Two tiles a CTA where one would not do for all rows at once. us with one (two), a request of n tokens, 32 / 8 heads of 128: 300 after 1000 39 (53), 500: 44 (57),
    // 600: 64 (58), 1000: 81 (71), 1500: 124 (101); 700 after 100 39 (42); 660 after 8000 280 (223)
    const int pair = always ? give_up >> 4 & 1 : ((long long)ntok * rep + 127) / 128 * G > sm_count();
    const PromptArgs4 pa{q, q_tok_stride, q_head_stride, (const uint8_t*)k, (const uint8_t*)v, (const uint16_t*)k_word, (const uint16_t*)v_word, table, q_start, kv_len, requests, width,
                         npages, page_shift(page_tokens), ntok, G, rep, pair, share, scale * 1.4426950408889634f, out, out_tok_stride, out_head_stride, give_up};
    if (const int rc = launch_prompt(pa, D, dtype == QSPEC_DTYPE_BF16, (cudaStream_t)stream)) return rc;
  }
  const AttArgs a{{table, q_start, kv_len, requests, width, npages, page_shift(page_tokens), ntok, G, rep, prompts ? share : 0u},
                  {out, out_tok_stride, out_head_stride, (int*)workspace, (float*)((char*)workspace + 4096)}, q, q_tok_stride, q_head_stride, (const uint8_t*)k, (const uint8_t*)v,
                  (const uint16_t*)k_word, (const uint16_t*)v_word, scale * 1.4426950408889634f};
  auto run = [&](auto kern, int ctas, size_t smem, SmemLimit& limit) -> int {
    QSPEC_CUDA(limit.raise(kern, smem));
    QSPEC_CUDA(launch_pdl(kern, dim3(std::max(sm_count(), 1) * ctas), dim3(THREADS), smem, (cudaStream_t)stream, a));
    QSPEC_CHECK_LAUNCH(1);
    return QSPEC_OK;
  };
  static SmemLimit limits[12];
  const bool few = (long long)max_tokens * rep <= 8, many = (long long)requests * G > 3ll * sm_count();
#define QSPEC_KV4_ATTENTION(BF, D, I)                                                                                                   \
  (!few   ? run(kv4_attention_kernel<BF, D, 16, 3>, 3, Smem<D, 16>::TOTAL, limits[I])                                                   \
   : many ? run(kv4_attention_kernel<BF, D, 8, 4>, 4, Smem<D, 8>::TOTAL, limits[4 + I])                                                 \
          : run(kv4_attention_kernel<BF, D, 8, 3>, 3, Smem<D, 8>::TOTAL, limits[8 + I]))
  if (dtype == QSPEC_DTYPE_F16) return D == 128 ? QSPEC_KV4_ATTENTION(false, 128, 0) : QSPEC_KV4_ATTENTION(false, 64, 1);
  return D == 128 ? QSPEC_KV4_ATTENTION(true, 128, 2) : QSPEC_KV4_ATTENTION(true, 64, 3);
#undef QSPEC_KV4_ATTENTION
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
