// Softmax attention of prompt portions over the paged 4-bit cache, on the fifth-generation tensor cores (kv4_common.cuh has the layout and the numbers, kv4_attention.cu the form for
// requests with few tokens).
//
// One CTA = one or two tiles of 128 rows of one request and key/value head; a row is a (token, query head of the group) pair. Keys are walked in blocks of 128 by two
// streams with a softmax and a sum of values of their own, so that one's products run under the other's softmax. Two tiles have a stream each, and every
// block's codes are made ready once for both; a single tile's streams take the blocks in turn and are joined at the end.
//   * pages: one warp looks the block's pages and words up (8 a lane) and leaves where the codes are, the words, and the largest exponent of the keys' scales and of the values'.
//   * codes: four warps bring a block's keys and values from global memory, make them float16 and store them as the tensor cores want them: the cache is read once, in 4
//     bits, and is never anywhere in 16. A code in the upper bits of the mantissa behind an exponent of 4 is 16 + c; (16 + c) s - (16 + z) s is one multiply-add of two
//     values, and exact: s has five bits, 16 + z has five, (c - z) s nine. s is the row's scale over the block's largest power of two, times 2^10: exact
//     down to 2^-30 of the largest. Where a block's keys' scales are further apart, or its values' more than 2^8 (of keys that a row does not see, or that count for nothing, it must not
//     notice that), s is 2^10, and the softmax takes each key's scales from shared memory (wide_block()). Eight codes of a word come out as 0 4 1 5 2 6 3 7: the order of the sum over a head's columns is free (queries are put in the same), and
//     columns of the result are put right on their way out.
//   * S = Q K^T, accumulator [128 x 128] float32 in tensor memory, one for each stream.
//   * products: a thread a stream issues them: scores once the keys are there and the stream's product before them is over (its weights lie where the scores go), the product of
//     values once half of the weights are there, then of the other half. (One thread for both was at work the whole time: six steps of some 900 cycles a pair of blocks,
//     for a look at a barrier takes 100 among warps that multiply and store.)
//   * softmax: thread = row, four warps a stream. The first half of a row's scores stays in registers between the maximum and the weights; the second half is read twice.
//     The block's power of two of the keys multiplies the scores, that of the values goes into the exponent; weights go back over the scores as float16 (off by 2^-11 of
//     themselves or by 2^-34 of the largest, as in kv4_attention.cu, or 2^-26 next to value scales that are 2^8 apart; the result is rounded to 16 bits as well).
//   * O += P V: weights from tensor memory, values from shared memory as they lie in the cache (operand "MN-major").
// Tensor memory: S | S | O | O = 512 columns. O is multiplied again only where a row's maximum grew by more than 2^6.
// What bounds it: 2000 tokens after 1000, 32 / 8 heads of 128, 116 to 118 us, 560 TFLOP/s of products (34 % of a large library product's rate). A pair of blocks takes some 5500
// cycles; its products are 2050 (64 each), the exponentials 2050 of a scheduler's special function unit, and both streams wait for one another's: the scores of a block take
// 800 to 1200 cycles, the softmax 2300 alone and 3400 beside the other's, the sum of values 800. Measured and not taken (us): two accumulators of 64 keys each for a stream, scores a turn
// ahead (151: a product of 64 columns takes as long as one of 128); one thread for both streams' products (119); the streams' exponentials in turn (120), or the second stream
// half a turn late (122: they fall into step again); 32 scores at a time, read again for the weights (118); the steps of the codes rolled into one piece of code (160). A CTA has
// 13 000 cycles to its first weights (its place 2 900, tensor memory 800, queries 6 000, the first scores 2 400) and 6 000 behind its last; here 108 SMs have two CTAs, 40 have one. (Queries put in
// order by whoever brought them, and rows out by 32 columns: 1 500 cycles less, and no time.)
//
// Every wait is bounded; a CTA whose wait runs out waits (again with a limit) for its products under way, fills its rows with NaN, counts itself
// (qspec_attn_tile_timeouts) and frees its tensor memory.
#include "kv4_common.cuh"
#include "attn_tile.cuh"

namespace qspec {
namespace kv4 {
namespace prompt {
using namespace atile;
using namespace kv8;

constexpr int SOFTMAX = 8, CONVERT = 4;                   // warps
constexpr int W_MMA = 0, W_PAGES = 2, W_CONVERT = 3, W_SOFTMAX = W_CONVERT + CONVERT, NWARPS = W_SOFTMAX + SOFTMAX, NTHREADS = NWARPS * 32;
constexpr int FACS = 4;                                   // blocks whose pages and factors are kept
constexpr float NONE = -INFINITY;

using Args = PromptArgs4;

template <int D> struct Sizes {
  static constexpr int PART = 128 * 128;                  // 128 rows x 64 elements
  static constexpr int OP = D / 64 * PART;                // an operand: 128 rows x D
  static constexpr int STAGES = 2;                        // of keys and of values
  static constexpr size_t USED = (size_t)OP * (2 + 2 * STAGES) + 1024;
  static constexpr size_t SMEM = USED > 120 * 1024 ? USED : 120 * 1024;   // one CTA an SM: each takes all of the tensor memory
  static_assert(SOFTMAX * 32 * (D + 16) <= 3 * OP, "rows on their way out, over queries and keys");
};
template <int D> constexpr uint32_t IDESC_S = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
template <int D> constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);

struct alignas(16) Block {                                            // what the other roles have to know of a block
  uint16_t kw[128], vw[128];                              // words of its keys; a key that makes rows no numbers has the scale NaN in kw and zero in vw
  long long at[8];                                        // of each 16 of its keys: the row of the cache where their codes begin, -1: nowhere
  int ke, ve;                                             // the largest exponent (of float32, biased) of the keys' scales, of the values'
  alignas(16) float k;                                    // for the softmax, 16 bytes together: the keys' power of two / 2^TOP, log2 of the values' / 2^TOP, and what weights are divided by that with
  float lv, iv;
  int wide;                                               // scales so far apart that codes stand in the operands without them; then, of each key:
  float ks[128], lvs[128], ivs[128];                      // its scale / 2^TOP (no number: rows that see it are none either), log2 of its value's / 2^TOP, and what weights are divided by that with
};
static_assert(offsetof(Block, wide) == offsetof(Block, k) + 12 && offsetof(Block, k) % 16 == 0, "read as a float4");
// How far apart exponents of a block's scales may be. Keys': what is exact beside each other in an operand (five bits from 2^TOP down to float16's last, 2^-24). Values': their largest goes into the
// exponents of all of the block's weights, and the reference with it; where a key that counts for nothing has it, later blocks' weights are that much closer to float16's end (2^-26 of the largest at 8).
constexpr int APART_K = 30, APART_V = 8;
constexpr int TOP = 10;                                   // scales over the block's largest power of two, times 2^TOP
constexpr uint32_t NO_KEY = 0xffffu, NO_VALUE = 0u;       // words of a key that makes the rows that see it no numbers

__device__ __forceinline__ void ld16(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr));
}
// Behind wait_ld(): nothing that is done with these registers is moved in front of it.
__device__ __forceinline__ void landed32(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) landed8(r + i * 8);
}

// A row's scores of a block whose scales are too far apart for the operands: made exponents, each by its own key's scales, and put back where they were. Gives the sum of weights / v, with
// the reference that the row will have (m: that it has), of the block's keys up to `limit`. (Out of line: it is
// seldom called. With every block like that 2000 tokens after 1000 take 212 us, so 118.)
__device__ __noinline__ float wide_block(uint32_t st, const Block& f, float rowf, float m, int limit) {
  float mn = NONE;
#pragma unroll 1
  for (int c0 = 0; c0 < 128; c0 += 32) {
    uint32_t x[32];
    ld32(st + c0, x);
    wait_ld();
    landed32(x);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float k = f.ks[c0 + j] * rowf, y = fmaf(__uint_as_float(x[j]), k < 1.17549435e-38f ? 1.17549435e-38f : k > 3.402823466e38f ? 3.402823466e38f : k, f.lvs[c0 + j]);
      if (c0 + j <= limit) mn = fmaxf(mn, y);
      x[j] = __float_as_uint(y);
    }
    st16(st + c0, x);
    st16(st + c0 + 16, x + 16);
  }
  wait_st();
  const float top = mn - m > GROWTH_LOG2 ? mn : m, mu = top == NONE ? 0.f : top;
  float sum = 0.f;
#pragma unroll 1
  for (int c0 = 0; c0 < 128; c0 += 32) {
    uint32_t x[32];
    ld32(st + c0, x);
    wait_ld();
    landed32(x);
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c0 + j <= limit) sum = fmaf(ex2(__uint_as_float(x[j]) - mu + WEIGHT_LOG2), f.ivs[c0 + j], sum);
  }
  return sum;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(NTHREADS, 1) kv4_prompt_kernel(const Args a) {
  using T = typename Elem16<BF16>::T;
  using Z = Sizes<D>;
  constexpr int OP = Z::OP, PARTB = Z::PART, STAGES = Z::STAGES, COLS = D / 2;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ __align__(8) uint64_t b_kfull[STAGES], b_kempty[STAGES], b_vfull[STAGES], b_vempty[STAGES], b_fac[FACS], b_facfree[FACS], b_q, b_s[2], b_p[2][2], b_o[2], b_end[2], b_join;
  __shared__ Block s_block[FACS];
  __shared__ float s_ml[2][2][128], s_rowf[256];
  __shared__ unsigned long long s_work[NWARPS];
  __shared__ int s_sum[NWARPS], s_at[5];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_fail;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rep = a.rep, tok = 128 / rep, span = tok << a.pair, g = blockIdx.x, rep_inv = 65536 / rep + 1;   // tokens of 128 rows, and of a CTA
  auto token_of = [&](int r) { return r * rep_inv >> 16; };   // r / rep, r < 256, rep <= 128
  if (tid == 0) {
    s_fail = 0;
    s_at[0] = -1;
    for (int i = 0; i < STAGES; ++i) {
      bar_init(smem_addr(&b_kfull[i]), CONVERT);
      bar_init(smem_addr(&b_vfull[i]), CONVERT);
    }
    for (int i = 0; i < FACS; ++i) bar_init(smem_addr(&b_fac[i]), 1);
    for (int i = 0; i < 2; ++i) { bar_init(smem_addr(&b_s[i]), 1); bar_init(smem_addr(&b_p[i][0]), 4); bar_init(smem_addr(&b_p[i][1]), 4); bar_init(smem_addr(&b_o[i]), 1); bar_init(smem_addr(&b_end[i]), 1); }
    bar_init(smem_addr(&b_q), SOFTMAX);
    bar_init(smem_addr(&b_join), SOFTMAX);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
  unsigned char* const gbase = raw + (base - smem_addr(raw));
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // ---- this CTA's request and tile: tiles of all requests in a row, the last one of a request (with the longest way) first. Up to 32 requests every warp looks for
  // itself, without barriers.
  const bool few = a.nreq <= 32;
  const int lookers = few ? 32 : NTHREADS, per_thread = (a.nreq + lookers - 1) / lookers, b0 = (few ? lane : tid) * per_thread, requests = max(min(per_thread, a.nreq - b0), 0);
  auto load = [&](int b, int& n, int& keys) {
    n = max(min(a.q_start[b + 1], a.ntok) - min(max(a.q_start[b], 0), a.ntok), 0);
    keys = max(a.kv_len[b], 0);
  };
  int n1 = 0, keys1 = 0;
  unsigned long long work = 0;
  for (int i = 0; i < requests; ++i) {
    load(b0 + i, n1, keys1);
    work += prompt_work(n1, keys1, rep, a.G);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
  if (!few) {
    if (lane == 0) s_work[warp] = work;
    __syncthreads();
    work = 0;
#pragma unroll
    for (int w = 0; w < NWARPS; ++w) work += s_work[w];
  }
  auto tiles_of = [&](int b) {
    if (per_thread > 1) load(b, n1, keys1);
    return to_prompt_form(n1, keys1, rep, a.share, work) ? (n1 + span - 1) / span : 0;
  };
  const int most = keys_at_most(a.width, a.pshift);
  int mine = 0;
  for (int i = 0; i < requests; ++i) mine += tiles_of(b0 + i);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  int before = incl - mine;
  if (!few) {
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NWARPS; ++w)
      if (w < warp) before += s_sum[w];
  }
  int req = -1, tile = 0, first = 0, n_new = 0, keys = 0;
  if ((int)blockIdx.y >= before && (int)blockIdx.y < before + mine) {
    int at = before;
    for (int i = 0; i < requests; ++i) {
      const int n = tiles_of(b0 + i);
      if ((int)blockIdx.y < at + n) {
        req = b0 + i;
        tile = n - 1 - ((int)blockIdx.y - at);
        first = min(max(a.q_start[req], 0), a.ntok);
        n_new = n1;
        keys = keys1;
        break;
      }
      at += n;
    }
  }
  if (few) {
    const unsigned found = __ballot_sync(0xffffffffu, req >= 0);
    if (!found) return;
    const int who = __ffs(found) - 1;
    req = __shfl_sync(0xffffffffu, req, who);
    tile = __shfl_sync(0xffffffffu, tile, who);
    first = __shfl_sync(0xffffffffu, first, who);
    n_new = __shfl_sync(0xffffffffu, n_new, who);
    keys = __shfl_sync(0xffffffffu, keys, who);
  } else {
    if (req >= 0) { s_at[0] = req; s_at[1] = tile; s_at[2] = first; s_at[3] = n_new; s_at[4] = keys; }
    __syncthreads();
    if (s_at[0] < 0) return;
    req = s_at[0]; tile = s_at[1]; first = s_at[2]; n_new = s_at[3]; keys = s_at[4];
  }
  const int t0 = tile * span, n2 = min(span, n_new - t0);   // this CTA's tokens
  const int pos0 = keys - n_new + t0;                     // position of the first
  const bool both = n2 > tok;                             // two tiles of rows, a stream each
  const int reach = min(keys, most);
  auto blocks_of = [&](int tokens) { const int seen = min(pos0 + tokens, reach); return seen > 0 ? (seen + 127) / 128 : 0; };
  const int blocks = blocks_of(n2);                       // keys that any row sees
  const int turns0 = both ? blocks_of(tok) : (blocks + 1) >> 1, turns1 = both ? blocks : blocks >> 1;   // blocks of the streams
  if (tid == 0) {
    for (int i = 0; i < FACS; ++i) bar_init(smem_addr(&b_facfree[i]), (both ? SOFTMAX : SOFTMAX / 2) + CONVERT);
    for (int i = 0; i < STAGES; ++i) { bar_init(smem_addr(&b_kempty[i]), both ? 2 : 1); bar_init(smem_addr(&b_vempty[i]), both ? 2 : 1); }   // (each stream's products)
  }
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&s_tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (tensor memory is held)
  const uint32_t kbuf = base + 2 * OP, vbuf = kbuf + STAGES * OP;

  if (warp == W_PAGES) {
    // ---- pages and words of the blocks, ahead of all others: lane i has 8 of a block's keys (i < 16: words of keys, else of values), the next block's pages on their way
    bool ok = !(a.give_up & 8u);
    if (!ok) s_fail = 1;
    const int part = (lane & 15) * 8, side = lane >> 4;
    auto page_of = [&](int n) {                             // -1: none
      const int key = n * 128 + part, at = key >> a.pshift;
      if (n >= blocks || key >= keys) return -1;
      const int page = at < a.width ? a.table[(size_t)req * a.width + at] : -1;
      return (unsigned)page < (unsigned)a.npages ? page : -1;
    };
    int page = page_of(0);
#pragma unroll 1
    for (int n = 0; ok && n < blocks; ++n) {
      const int slot = n % FACS, key = n * 128 + part;
      const bool there = page >= 0;
      const long long row = there ? (long long)((((size_t)page * a.G + g) << a.pshift) + (key & ((1 << a.pshift) - 1))) : -1ll;
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (there) w = __ldg(reinterpret_cast<const uint4*>((side ? a.vw : a.kw) + row));
      page = page_of(n + 1);
      // scales that are infinite or no number: exponent 255. (Rows behind the last key have neither say nor sight.)
      uint32_t x[4] = {w.x, w.y, w.z, w.w};
      const int have = min(max(keys - key, 0), 8);
      uint32_t most = 0u, least = 0x00ff00ffu;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most = __vmaxu2(most, x[e] >> 8 & 0x00ff00ffu);
        least = __vminu2(least, x[e] >> 8 & 0x00ff00ffu);
      }
      most = max(most & 0xffffu, most >> 16);
      least = min(least & 0xffffu, least >> 16);
      if (!__all_sync(0xffffffffu, there && have == 8 && most < 255u)) {   // (seldom: one by one)
        uint32_t bad = 0u;
        most = 0u;
        least = 255u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t ex = (x[e >> 1] >> (e & 1 ? 24 : 8)) & 0xffu;
          if (there && e < have) {
            if (ex == 255u) {
              bad |= 1u << e;
            } else {
              most = max(most, ex);
              least = min(least, ex);
            }
          }
        }
        if (!there) bad = (1u << have) - 1u;                // (a page that there is not)
        bad |= __shfl_xor_sync(0xffffffffu, bad, 16);       // of the key's word, or of the value's
        const uint32_t no = side ? NO_VALUE : NO_KEY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (bad >> (2 * e) & 1u) x[e] = (x[e] & 0xffff0000u) | no;
          if (bad >> (2 * e + 1) & 1u) x[e] = (x[e] & 0xffffu) | no << 16;
          if (2 * e >= have) x[e] = 0u;                     // (values that are no numbers would make a weight of zero one)
          else if (2 * e + 1 >= have) x[e] &= 0xffffu;
        }
      }
      uint32_t ends = (255u - max(least, 27u)) << 16 | max(most, 27u);   // (the larger of either half; 27: 2^-100, and what is below that)
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) ends = __vmaxu2(ends, __shfl_xor_sync(0xffffffffu, ends, o));
      most = ends & 0xffffu;
      const bool wide = __any_sync(0xffffffffu, (int)(most + (ends >> 16)) > 255 + (side ? APART_V : APART_K));
      // (what the others wait for begins here: nothing is left but stores)
      if (n >= FACS) ok = bar_wait(smem_addr(&b_facfree[slot]), (uint32_t)((n / FACS) - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      Block& f = s_block[slot];
      *reinterpret_cast<uint4*>((side ? f.vw : f.kw) + part) = make_uint4(x[0], x[1], x[2], x[3]);
      if (!side && !(lane & 1)) f.at[lane >> 1] = row;
      if (lane == 0) {
        f.ke = (int)most;
        f.k = __uint_as_float((uint32_t)min(max((int)most - TOP, 1), 254) << 23);
        f.wide = wide;
      }
      if (lane == 16) {
        f.ve = (int)most;
        f.lv = wide ? 0.f : (float)((int)most - 127 - TOP);
        f.iv = wide ? 0.f : __uint_as_float((uint32_t)min(max(127 + 127 + TOP - (int)most, 1), 254) << 23) * WEIGHT_UNIT;
      }
      if (__builtin_expect(wide, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float scale = word_scale(x[e >> 1] >> (e & 1 ? 16 : 0));
          if (side) {
            const float v = fmaxf(scale, 7.888609052210118e-31f);
            f.lvs[part + e] = __log2f(v) - TOP;
            f.ivs[part + e] = over_scale(WEIGHT_UNIT * (1 << TOP), v);
          } else {
            f.ks[part + e] = scale * (1.f / (1 << TOP));
          }
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(smem_addr(&b_fac[slot]));
    }
  } else if (warp < W_PAGES) {
    if (elect()) {
      const int z = warp - W_MMA, turns = z ? turns1 : turns0;
      bool ok = !(a.give_up & 4u);
      if (!ok) s_fail = 1;
      if (turns) ok = ok && bar_wait(smem_addr(&b_q), 0, &s_fail);
      const uint64_t qd = desc_k(base + (both ? z * OP : 0));
      const uint32_t s = tmem + z * 128, o = tmem + 256 + z * D;
#pragma unroll 1
      for (int j = 0; ok && j < turns; ++j) {
        const int n = both ? j : 2 * j + z, stage = n % STAGES;
        const uint32_t round = (uint32_t)(n / STAGES) & 1u, turn = (uint32_t)j & 1u;
        const bool last = both && z && n >= turns0;         // tile 0 does not see this block: tile 1 says for both that it is done with it
        ok = bar_wait(smem_addr(&b_kfull[stage]), round, &s_fail) && (!j || bar_wait(smem_addr(&b_o[z]), turn ^ 1u, &s_fail));   // (these scores take the columns of the weights before)
        if (!ok) break;
        fence_after();
        const uint64_t kd = desc_k(kbuf + stage * OP);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const uint32_t step = (uint32_t)((d >> 2) * (PARTB >> 4) + (d & 3) * 2);
          mma_ss(s, qd + step, kd + step, IDESC_S<D>, d ? 1u : 0u);
        }
        commit(smem_addr(&b_s[z]));
        commit(smem_addr(&b_kempty[stage]));
        if (last) commit(smem_addr(&b_kempty[stage]));
        ok = bar_wait(smem_addr(&b_vfull[stage]), round, &s_fail);
        if (!ok) break;
        const uint64_t vd = desc_mn(vbuf + stage * OP);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                       // 64 keys each
          ok = ok && bar_wait(smem_addr(&b_p[z][h]), turn, &s_fail);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int d = 0; d < 4; ++d) mma_ts(o, s + h * 32 + d * 8, vd + (h * 4 + d) * (2048 >> 4), IDESC_O<D>, (j || h || d) ? 1u : 0u);
        }
        if (!ok) break;
        commit(smem_addr(&b_o[z]));
        commit(smem_addr(&b_vempty[stage]));
        if (last) commit(smem_addr(&b_vempty[stage]));
      }
      // every product is over before the CTA leaves, those of a turn that was given up, too
      commit(smem_addr(&b_end[z]));
      bar_drain(smem_addr(&b_end[z]), 0);
    }
    __syncwarp();
  } else if (warp < W_SOFTMAX) {
    // ---- codes: 16 bytes (32 of them) a lane
    constexpr int ROWS = CONVERT * 32 / (D / 32), STEPS = 128 / ROWS;   // rows at a time, times
    const int ct = tid - W_CONVERT * 32;
    // (eight lanes take two pieces of four rows, so that their stores meet in no bank)
    const int c = D == 128 ? (ct >> 3 & 1) * 2 + (ct & 1) : ct & 1, row0 = D == 128 ? (ct >> 4) * 4 + (ct >> 1 & 3) : ct >> 1;
    const uint32_t part = (uint32_t)(c >> 1) * PARTB;
    uint4 here[STEPS], next[STEPS];
    auto load = [&](int t) {                                // side t % 2 (keys, values) of block t / 2
      const Block& f = s_block[(t >> 1) % FACS];
      const uint8_t* codes = (t & 1 ? a.v : a.k) + c * 16;
      const int have = keys - (t >> 1) * 128;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int row = i * ROWS + row0;
        const long long at = f.at[row >> 4];
        next[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < have && at >= 0) next[i] = __ldg(reinterpret_cast<const uint4*>(codes + (at + (row & 15)) * (D / 2)));
      }
    };
    auto store = [&](const uint4 (&w)[STEPS], uint32_t dst, const uint16_t* words, int ex, bool wide) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int row = i * ROWS + row0;
        const uint32_t word = words[row];
        const float s = wide ? (float)(1 << TOP) : word_scale(word) * __uint_as_float((uint32_t)min(max(127 + 127 + TOP - ex, 1), 254) << 23);   // (over the block's largest power of two)
        const __half2 scale = __float2half2_rn(s), zero = __float2half2_rn(-(16.f + (float)(word & 15u)) * s);
        const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        const uint32_t at = dst + part + row * 128;
        auto two = [&](uint32_t y) {
          y = (y & 0x03c003c0u) | 0x4c004c00u;
          const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&y), scale, zero);
          return *reinterpret_cast<const uint32_t*>(&r);
        };
#pragma unroll
        for (int e = 0; e < 4; ++e)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(at + ((((c & 1) * 4 + e) ^ (row & 7)) << 4)), "r"(two(x[e] << 6)), "r"(two(x[e] << 2)),
                       "r"(two(x[e] >> 2)), "r"(two(x[e] >> 6)) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
    };
    bool ok = !(a.give_up & 2u);
    if (!ok) s_fail = 1;
    auto look = [&](int n) {
      ok = ok && bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
    };
    if (blocks && ok) look(0);
    if (blocks && ok) load(0);
#pragma unroll 1
    for (int t = 0; ok && t < 2 * blocks; ++t) {            // (one piece of code for keys and values)
      const int n = t >> 1, stage = n % STAGES, side = t & 1;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) here[i] = next[i];
      if (t + 1 < 2 * blocks) {
        if (side) look(n + 1);
        if (!ok) break;
        load(t + 1);
      }
      if (n >= STAGES) ok = bar_wait(smem_addr(side ? &b_vempty[stage] : &b_kempty[stage]), (uint32_t)(n / STAGES - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const Block& f = s_block[n % FACS];
      store(here, (side ? vbuf : kbuf) + stage * OP, side ? f.vw : f.kw, side ? f.ve : f.ke, f.wide);
      if (lane == 0) {
        bar_arrive(smem_addr(side ? &b_vfull[stage] : &b_kfull[stage]));
        if (side) bar_arrive(smem_addr(&b_facfree[n % FACS]));
      }
    }
  } else {
    // ---- queries: as they are, 16 bytes a thread at a time; then a thread a row: bfloat16 rows times a power of two each, and the sums. (Loops that are
    // not unrolled: every CTA comes here once, and had to wait for the instructions.)
    constexpr int IN_ROW = D / 8;
    const int tiles = both ? 2 : 1, wi = warp - W_SOFTMAX, ti = tid - W_SOFTMAX * 32;
#pragma unroll 4
    for (int i = ti; i < tiles * 128 * IN_ROW; i += SOFTMAX * 32) {
      const int c = i % IN_ROW, row = i / IN_ROW, r = row & 127, tl = (row >> 7) * tok + token_of(r);
      const uint32_t to = base + (row >> 7) * OP + (c >> 3) * PARTB + r * 128 + (((c & 7) ^ (r & 7)) << 4);
      if (tl < n2 && r < tok * rep)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to),
                     "l"((const T*)a.q + (size_t)(first + t0 + tl) * a.q_ts + (size_t)(g * rep + r - token_of(r) * rep) * a.q_hs + c * 8) : "memory");
      else
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(to), "r"(0u) : "memory");
    }
    auto ready = [&] {                                    // for the products
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(smem_addr(&b_q));
    };
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;\n" ::: "memory");
    asm volatile("bar.sync 1, %0;\n" ::"n"(SOFTMAX * 32) : "memory");   // (behind nothing that may be given up)
    if (ti < tiles * 128) {
      const int r = ti & 127;
      unsigned char* const row = gbase + (ti >> 7) * OP + r * 128;
      auto piece = [&](int c) { return reinterpret_cast<uint4*>(row + (c >> 3) * PARTB + (((c & 7) ^ (r & 7)) << 4)); };
      int sh = 0;
      if (BF16) {
        float mx = 0.f;
#pragma unroll 1
        for (int c = 0; c < IN_ROW; ++c) {
          const uint4 w = *piece(c);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
        }
        const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
        sh = mx > 0.f && mx < INFINITY ? min(max(14 - ex, -126), 126) : 0;
      }
      const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll 2
      for (int c = 0; c < IN_ROW; ++c) {
        const uint4 w = *piece(c);
        uint32_t x[4] = {w.x, w.y, w.z, w.w};
        if (BF16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = half_pair(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
        }
        // in the order in which codes come out of a word: 0 4 1 5 2 6 3 7
        *piece(c) = make_uint4(__byte_perm(x[0], x[2], 0x5410), __byte_perm(x[0], x[2], 0x7632), __byte_perm(x[1], x[3], 0x5410), __byte_perm(x[1], x[3], 0x7632));
      }
      s_rowf[ti] = __uint_as_float((uint32_t)(127 - sh) << 23) * a.scale2;
    }
    ready();
    asm volatile("bar.sync 1, %0;\n" ::"n"(SOFTMAX * 32) : "memory");   // (the factors of the rows)
    // ---- softmax: thread = row r of stream z
    const int z = wi >> 2, r = (warp & 3) * 32 + lane, turns = z ? turns1 : turns0, zrow = both ? z * 128 : 0, ztok = both ? z * tok : 0;
    const int tl = ztok + token_of(r);
    const bool row_in = r < tok * rep && tl < n2;
    const int limit = row_in ? min(pos0 + tl, keys - 1) : -1;   // last visible position
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t st = tmem + lanes + z * 128, ot = tmem + lanes + 256 + z * D;
    bool ok = !(a.give_up & 1u);
    if (!ok) s_fail = 1;
    const float rowf = s_rowf[zrow + r];
    float m = NONE, l = 0.f;
    for (int i = 0; ok && i < turns; ++i) {
      const int n = both ? i : 2 * i + z, j0 = n * 128;
      const uint32_t turn = (uint32_t)i & 1u;
      const bool plain = __all_sync(0xffffffffu, !row_in || j0 + 127 <= limit);   // (rows that stand for no token are never stored)
      ok = bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail);
      const Block& f = s_block[n % FACS];
      const float4 factors = *reinterpret_cast<const float4*>(&f.k);
      const bool wide = __float_as_int(factors.w);
      ok = ok && bar_wait(smem_addr(&b_s[z]), turn, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      uint32_t x[64];
      auto hide = [&](uint32_t* y, int count, int c0) {     // what a row does not see
#pragma unroll
        for (int j = 0; j < count; ++j)
          if (j0 + c0 + j > limit) y[j] = 0xff800000u;
      };
      auto largest = [&](const uint32_t* y, float mx) {
        float t = __uint_as_float(y[0]);
#pragma unroll
        for (int j = 1; j < 31; j += 4) {                   // (three operands: one instruction)
          mx = fmaxf(fmaxf(mx, __uint_as_float(y[j])), __uint_as_float(y[j + 1]));
          if (j + 3 < 32) t = fmaxf(fmaxf(t, __uint_as_float(y[j + 2])), __uint_as_float(y[j + 3]));
        }
        return fmaxf(fmaxf(mx, t), __uint_as_float(y[31]));
      };
      float own = 0.f;
      if (__builtin_expect(wide, 0)) own = wide_block(st, f, rowf, m, limit - j0);
      // ---- the largest exponent: of the second half, whose scores are read again, and the first, whose scores stay
      float mn = NONE;
      auto load = [&](int c0) {
        ld32(st + c0, x);
        ld32(st + c0 + 32, x + 32);
        wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) landed8(x + 8 * j);
        if (!plain) hide(x, 64, c0);
      };
#pragma unroll 1
      for (int c0 = 64; c0 >= 0; c0 -= 64) {
        load(c0);
        mn = largest(x, mn);
        mn = largest(x + 32, mn);
      }
      // The block's powers of two: what scores are multiplied with (not so small that it would make a hidden key's minus infinity no number, nor so large that it would make a score of nothing one), what exponents begin with
      const float k = wide ? 1.f : fminf(fmaxf(rowf * factors.x, 1.17549435e-38f), 3.402823466e38f), lv = factors.y, iv = factors.z;
      mn = fmaf(mn, k, lv);                                 // (minus infinity stays that)
      const bool grown = mn - m > GROWTH_LOG2;              // (of a row that had seen nothing: infinite, or nothing again and no number; far from zero m + 6 is more than that)
      if (__any_sync(0xffffffffu, grown)) {
        const float up = grown ? ex2(m - mn) : 1.f;         // 0 for a row that had seen nothing; other rows of the warp keep theirs
        l *= up;
        if (i && __any_sync(0xffffffffu, grown && m != NONE)) {   // (the scores are there: the stream's product before them is over)
#pragma unroll 1
          for (int q = 0; q < D / 16; ++q) {
            uint32_t o[16];
            ld16(ot + q * 16, o);
            wait_ld();
            landed8(o);
            landed8(o + 8);
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * up);
            st16(ot + q * 16, o);
          }
        }
        if (grown) m = mn;
      }
      const float mu = m == NONE ? 0.f : m;
      // Exponents are taken from the products without a rounding in between, the reference and what it is joined with have one: far from zero that alone would be a
      // large exponent.
      const bool far = __any_sync(0xffffffffu, fabsf(mu) > FAR);
      const float k1 = far ? 1.f : k, at1 = far ? WEIGHT_LOG2 : lv - (mu - WEIGHT_LOG2);
      const uint64_t k2 = pair(__float_as_uint(k1), __float_as_uint(k1)), at2 = pair(__float_as_uint(at1), __float_as_uint(at1));
      uint64_t sum[2] = {0ull, 0ull};
      // ---- weights, 64 at a time
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (h) load(64);
        if (far) {
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] = __float_as_uint(fmaf(__uint_as_float(x[j]), k, lv) - mu);
          if (!plain) hide(x, 64, h * 64);                  // (scores that a row does not see may have been infinite)
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            uint32_t p0, p1;
            unpair(fma2(pair(x[c * 32 + 2 * j], x[c * 32 + 2 * j + 1]), k2, at2), p0, p1);
            p0 = __float_as_uint(ex2(__uint_as_float(p0)));
            p1 = __float_as_uint(ex2(__uint_as_float(p1)));
            sum[j & 1] = add2(sum[j & 1], pair(p0, p1));
            p[j] = half_pair(__uint_as_float(p0), __uint_as_float(p1));
          }
          st16(st + h * 32 + c * 16, p);                    // (over scores that have been read)
        }
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(smem_addr(&b_p[z][h]));
      }
      if (lane == 0) bar_arrive(smem_addr(&b_facfree[n % FACS]));
      uint32_t a0, a1;
      unpair(add2(sum[0], sum[1]), a0, a1);
      l = fmaf(__uint_as_float(a0) + __uint_as_float(a1), iv, l) + own;
    }
    if (both && z == 0)                                   // (blocks that tile 1 alone sees)
      for (int n = turns; ok && n < blocks; ++n) {
        ok = __all_sync(0xffffffffu, bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail));
        if (ok && lane == 0) bar_arrive(smem_addr(&b_facfree[n % FACS]));
      }
    // ---- out, through shared memory, 16 bytes a lane. A single tile's streams together: maxima and sums through shared memory; stream z takes half z of the
    // columns, of both sums. Of a pair either takes both halves of its own.
    constexpr int LD = COLS * 2 + 16, LANES = COLS / 8;   // bytes of half a row (and 16: no bank conflicts), lanes that take it
    unsigned char* const rows = gbase + wi * 32 * LD;   // (queries and keys are done with)
    s_ml[z][0][r] = m;
    s_ml[z][1][r] = l;
    __syncwarp();
    if (lane == 0) bar_arrive(smem_addr(&b_join));
    // the last product of either stream, and everyone's maxima
    if (ok) {
      ok = bar_wait(smem_addr(&b_join), 0, &s_fail);
      if (turns0) ok = ok && bar_wait(smem_addr(&b_o[0]), (uint32_t)(turns0 - 1) & 1u, &s_fail);
      if (turns1) ok = ok && bar_wait(smem_addr(&b_o[1]), (uint32_t)(turns1 - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
    }
    fence_after();
    if (ok) {
      const int other = both ? z : 1 - z;
      float f[2], sum = 0.f;                              // of this stream and the other one
      const float top = fmaxf(m, s_ml[other][0][r]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mi = i ? s_ml[other][0][r] : m, li = i ? s_ml[other][1][r] : l;
        f[i] = mi == NONE ? (li == 0.f ? 0.f : 1.f) : ex2(mi - top);   // nothing seen, or no number
        if (i && both) f[i] = 0.f;
        sum += li * f[i];                                 // (one that is no number shows whatever its part is)
      }
      const float d = sum != 0.f ? __fdiv_rn(WEIGHT_UNIT, sum) : limit < 0 ? 0.f : NAN;  // (no key: zeros; keys that all have minus infinity, of a query that is infinite: no numbers, like any other such)
      const bool one = turns > 0, two = !both && __any_sync(0xffffffffu, f[1] != 0.f) && (z ? turns0 : turns1) > 0;
      const uint32_t stored = __ballot_sync(0xffffffffu, row_in);
      for (int half = both ? 0 : z; half <= (both ? 1 : z); ++half) {
#pragma unroll 1
        for (int q = 0; q < COLS / 16; ++q) {
          uint32_t o0[16], o1[16];
          if (one) ld16(tmem + lanes + 256 + z * D + half * COLS + q * 16, o0);
          if (two) ld16(tmem + lanes + 256 + other * D + half * COLS + q * 16, o1);
          wait_ld();
          landed8(o0); landed8(o0 + 8);
          landed8(o1); landed8(o1 + 8);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x0 = one && f[0] != 0.f ? __uint_as_float(o0[x * 8 + e]) * f[0] : 0.f, x1 = two && f[1] != 0.f ? __uint_as_float(o1[x * 8 + e]) * f[1] : 0.f;
              v[e & 1 ? 4 + (e >> 1) : e >> 1] = (x0 + x1) * d;   // (columns come as 0 4 1 5 2 6 3 7)
            }
            *reinterpret_cast<uint4*>(rows + lane * LD + q * 32 + x * 16) = pack8<BF16>(v);
          }
        }
        __syncwarp();
        const int pc = lane % LANES;
#pragma unroll 2
        for (int rr = lane / LANES; rr < 32; rr += 32 / LANES) {
          const int r2 = (warp & 3) * 32 + rr, t2 = token_of(r2);
          if (stored >> rr & 1u)
            *reinterpret_cast<uint4*>((T*)a.out + (size_t)(first + t0 + ztok + t2) * a.out_ts + (size_t)(g * rep + r2 - t2 * rep) * a.out_hs + half * COLS + pc * 8) =
                *reinterpret_cast<const uint4*>(rows + rr * LD + pc * 16);
        }
        __syncwarp();
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (s_fail) {                                           // (written before the barrier: uniform)
    if (tid == 0) atomicAdd(&attn_tile_timeouts, 1u);
    for (int i = tid; i < n2 * rep * (D / 8); i += NTHREADS) {
      const int row = i / (D / 8), tl = row / rep;
      *reinterpret_cast<uint4*>((T*)a.out + (size_t)(first + t0 + tl) * a.out_ts + (size_t)(g * rep + row - tl * rep) * a.out_hs + i % (D / 8) * 8) =
          make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    }
  }
}

template <bool BF16, int D>
int launch(const Args& a, cudaStream_t stream) {
  static SmemLimit limit;
  auto kern = kv4_prompt_kernel<BF16, D>;
  QSPEC_CUDA(limit.raise(kern, Sizes<D>::SMEM));
  // tiles of all requests at most: full ones, and one more for each request that is large enough
  const int per = (128 / a.rep) << a.pair;
  const long long tiles = a.ntok / per + std::min<long long>(a.nreq, (long long)a.ntok * a.rep / PROMPT_ROWS + 1);
  QSPEC_REQUIRE(tiles <= 65535, QSPEC_ERR_UNSUPPORTED, "kv4_attention: %d tokens are too many for one call", a.ntok);
  QSPEC_CUDA(launch_pdl(kern, dim3(a.G, (unsigned)tiles), dim3(NTHREADS), Sizes<D>::SMEM, stream, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}

}  // namespace prompt

int launch_prompt(const PromptArgs4& a, int D, bool bf16, cudaStream_t stream) {
  return bf16 ? (D == 128 ? prompt::launch<true, 128>(a, stream) : prompt::launch<true, 64>(a, stream))
              : (D == 128 ? prompt::launch<false, 128>(a, stream) : prompt::launch<false, 64>(a, stream));
}
}  // namespace kv4

// CTAs of the form above that gave a wait up since the library was loaded on the current device; -1: not readable. Synchronises.
int kv4_timeouts() {
  unsigned n = 0;
  return cudaMemcpyFromSymbol(&n, atile::attn_tile_timeouts, sizeof(n)) == cudaSuccess ? (int)(n & 0x1fffffffu) : -1;
}
}  // namespace qspec
