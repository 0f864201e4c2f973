// Softmax attention of prompt portions over the paged 8-bit cache, on the fifth-generation tensor cores (kv8_attention.cu has the layout, and the form for requests
// with few tokens).
//
// One CTA = one or two tiles of 128 rows of one request and key/value head; a row is a (token, query head of the group) pair. Keys are walked in blocks of 128 by two
// streams with a softmax and a sum of values of their own, so that one's products run under the other's softmax. Two tiles have a stream each, and every
// block's codes are made ready once for both; a single tile's streams take the blocks in turn and are joined at the end.
//   * pages: one warp looks the block's pages and scales up and leaves where the codes are and what their products are multiplied with.
//   * codes: four warps bring a block's keys and values from global memory, make them float16 and store them as the tensor cores want them: the cache
//     is read once, in 8 bits, and is never anywhere in 16. Keys are (c + 128) 2^-24, the subnormal number that a byte is by itself; what the 128 adds
//     to a row's scores is taken out where they enter the exponent. Values are c exactly: a byte behind 0x64 is 1152 + c, less 1152.
//   * S = Q K^T, accumulator [128 x 128] float32 in tensor memory, one for each stream.
//   * softmax: thread = row, four warps a stream. Scores are read twice, for the maximum and for the weights (that keeps 128 of them out of the registers).
//     Weights go back over the scores as float16 (off by 2^-11 of themselves or by 2^-34 of the largest, as in kv8_attention.cu; the result is rounded to 16 bits as well).
//   * O += P V: weights from tensor memory, values from shared memory as they lie in the cache (operand "MN-major").
// Tensor memory: S | S | O | O = 512 columns. Scales and the exponent that takes the value scale in: as in kv8_attention.cu. O is multiplied again only
// where a row's maximum grew by more than 2^6.
// What a block of 128 x 128 (head 128) asks of an SM: 1024 cycles of the tensor cores, 1024 of the exponentials (16 a cycle), and of the schedulers 720 by the softmax
// and 400 by the codes (200 of two tiles). It takes 2350 cycles of two tiles (2850 to 3400 of one): what bounds it is a stream's way from scores to the next scores,
// 4700 cycles, of which the softmax is 3000 (a warp's 32 exponentials and what belongs to them 570) and the products with their waits 1700; start and end of a CTA are
// another 16000. Prompt of 2000 tokens after 1000, 32 / 8 heads, float16: 112 us, 586 TFLOP/s. Measured and not taken: sixteen softmax warps, two for
// a row, 125 us (their common maximum and their waits cost more than they save); a warp for each stream's products 128 us (the streams fall into step);
// scores read one chunk ahead 137 us (the copies between registers).
//
// Every wait is bounded; a CTA whose wait runs out waits (again with a limit) for its products under way, fills its rows with NaN, counts itself
// (qspec_attn_tile_timeouts) and frees its tensor memory.
#include "kv8_common.cuh"
#include "attn_tile.cuh"

namespace qspec {
namespace kv8 {
namespace prompt {
using namespace atile;

constexpr int SOFTMAX = 8, CONVERT = 4;                   // warps
constexpr int W_CONVERT = SOFTMAX, W_MMA = W_CONVERT + CONVERT, W_PAGES = W_MMA + 1, NWARPS = W_PAGES + 1, NTHREADS = NWARPS * 32;
constexpr int FACS = 4;                                   // blocks whose pages and factors are kept
constexpr float NONE = -INFINITY;

using Args = PromptArgs;

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

struct alignas(16) Block {                                            // what the other roles have to know of a block: of each 16 of its keys
  long long at[8];                                        // where their codes begin, -1: nowhere
  float kf[8], lv[8], iv[8];                              // scale of the keys; log2 of the values' scale, and its reciprocal
  unsigned bad;                                           // bit q: a page that there is not, or a scale that is no number
};

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

template <bool BF16, int D>
__global__ void __launch_bounds__(NTHREADS, 1) kv8_prompt_kernel(const Args a) {
  using T = typename Elem16<BF16>::T;
  using Z = Sizes<D>;
  constexpr int OP = Z::OP, PARTB = Z::PART, STAGES = Z::STAGES, COLS = D / 2;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ __align__(8) uint64_t b_kfull[STAGES], b_kempty[STAGES], b_vfull[STAGES], b_vempty[STAGES], b_fac[FACS], b_facfree[FACS], b_q, b_s[2], b_p[2][2], b_o[2], b_join;
  __shared__ Block s_block[FACS];
  __shared__ float s_ml[2][2][128], s_rowf[256], s_sum128[256];
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
      bar_init(smem_addr(&b_kfull[i]), CONVERT); bar_init(smem_addr(&b_kempty[i]), 1);
      bar_init(smem_addr(&b_vfull[i]), CONVERT); bar_init(smem_addr(&b_vempty[i]), 1);
    }
    for (int i = 0; i < FACS; ++i) bar_init(smem_addr(&b_fac[i]), 1);
    for (int i = 0; i < 2; ++i) { bar_init(smem_addr(&b_s[i]), 1); bar_init(smem_addr(&b_p[i][0]), 4); bar_init(smem_addr(&b_p[i][1]), 4); bar_init(smem_addr(&b_o[i]), 1); }
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
  if (tid == 0)
    for (int i = 0; i < FACS; ++i) bar_init(smem_addr(&b_facfree[i]), (both ? SOFTMAX : SOFTMAX / 2) + CONVERT);
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
    // ---- pages and factors of the blocks, ahead of all others
    bool ok = !(a.give_up & 8u);
    if (!ok) s_fail = 1;
    for (int n = 0; ok && n < blocks; ++n) {
      const int slot = n % FACS;
      if (n >= FACS) ok = bar_wait(smem_addr(&b_facfree[slot]), (uint32_t)((n / FACS) - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int key = n * 128 + lane * 16, at = key >> a.pshift;
      bool bad = false;
      long long codes = -1;
      float k = 0.f, v = 1.f;                             // (of keys that there are not: a factor that is next to nothing)
      if (lane < 8 && key < keys) {
        const int page = at < a.width ? a.table[(size_t)req * a.width + at] : -1;
        bad = (unsigned)page >= (unsigned)a.npages;
        if (!bad) {
          const size_t block = (size_t)page * a.G + g;
          codes = (long long)(((block << a.pshift) + (key & ((1 << a.pshift) - 1))) * D);
          k = finite_scale(a.ks[block]);
          v = finite_scale(a.vs[block]);
          bad = k != k || v != v;
        }
      }
      const unsigned mask = __ballot_sync(0xffffffffu, bad);
      if (lane < 8) {
        s_block[slot].at[lane] = codes;
        v = positive(v);
        s_block[slot].kf[lane] = positive(k);
        s_block[slot].lv[lane] = __log2f(v);
        s_block[slot].iv[lane] = __fdividef(WEIGHT_UNIT, v);
        if (lane == 0) s_block[slot].bad = mask;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(smem_addr(&b_fac[slot]));
    }
  } else if (warp == W_MMA) {
    if (elect()) {
      bool ok = !(a.give_up & 4u);
      if (!ok) s_fail = 1;
      int done0 = 0, done1 = 0;                           // value products that have been issued
      // Step k: stream k % 2's turn k / 2. Pairs of tiles take every block in turn, a single tile's streams every other one.
      const int steps = both ? 2 * blocks : blocks;
      auto scores = [&](int k) -> bool {
        const int z = k & 1, i = k >> 1, n = both ? i : k;
        if (i >= (z ? turns1 : turns0)) return true;
        if (!bar_wait(smem_addr(&b_kfull[n % STAGES]), (uint32_t)(n / STAGES) & 1u, &s_fail)) return false;
        // these scores take the columns of the weights of the turn before: its product must be over
        if (i && !bar_wait(smem_addr(&b_o[z]), (uint32_t)(i - 1) & 1u, &s_fail)) return false;
        fence_after();
        const uint64_t qd = desc_k(base + (both ? z * OP : 0)), kd = desc_k(kbuf + (n % STAGES) * OP);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const uint32_t step = (uint32_t)((d >> 2) * (PARTB >> 4) + (d & 3) * 2);
          mma_ss(tmem + z * 128, qd + step, kd + step, IDESC_S<D>, d ? 1u : 0u);
        }
        commit(smem_addr(&b_s[z]));
        if (!both || z) commit(smem_addr(&b_kempty[n % STAGES]));   // (tile 1 sees every block that tile 0 sees)
        return true;
      };
      ok = ok && (steps == 0 || (bar_wait(smem_addr(&b_q), 0, &s_fail) && scores(0) && (steps == 1 || scores(1))));
      for (int k = 0; ok && k < steps; ++k) {
        const int z = k & 1, i = k >> 1, n = both ? i : k;
        if (i >= (z ? turns1 : turns0)) continue;
        ok = bar_wait(smem_addr(&b_vfull[n % STAGES]), (uint32_t)(n / STAGES) & 1u, &s_fail);
        const uint64_t vd = desc_mn(vbuf + (n % STAGES) * OP);
        const uint32_t p = tmem + z * 128, o = tmem + 256 + z * D;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                     // 64 keys each
          ok = ok && bar_wait(smem_addr(&b_p[z][h]), (uint32_t)i & 1u, &s_fail);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int d = 0; d < 4; ++d) mma_ts(o, p + h * 32 + d * 8, vd + (h * 4 + d) * (2048 >> 4), IDESC_O<D>, (i || h || d) ? 1u : 0u);
        }
        if (!ok) break;
        commit(smem_addr(&b_o[z]));
        if (!both || z) commit(smem_addr(&b_vempty[n % STAGES]));
        (z ? done1 : done0) = i + 1;
        ok = k + 2 >= steps || scores(k + 2);
      }
      // every product of either stream is over before the CTA leaves, those of a turn that was given up, too
      if (done0) bar_drain(smem_addr(&b_o[0]), (uint32_t)(done0 - 1) & 1u);
      if (done1) bar_drain(smem_addr(&b_o[1]), (uint32_t)(done1 - 1) & 1u);
      if (!ok) {
        commit(smem_addr(&b_o[0]));
        bar_drain(smem_addr(&b_o[0]), (uint32_t)done0 & 1u);
      }
    }
    __syncwarp();
  } else if (warp >= W_CONVERT) {
    // ---- codes: 16 bytes a lane, 16 rows (one page's) at a time
    constexpr int CH = D / 16, ROWS = CONVERT * 32 / CH, STEPS = 128 / ROWS;   // pieces of a row, rows at a time, times
    const int ct = tid - W_CONVERT * 32;
    // (eight lanes take four pieces of two rows, so that their stores meet in no bank)
    const int c = D == 128 ? (ct >> 3 & 1) * 4 + (ct & 3) : ct & 3, row0 = D == 128 ? (ct >> 4) * 2 + (ct >> 2 & 1) : ct >> 2;
    const uint32_t part = (uint32_t)(c >> 2) * PARTB;
    uint4 kw[STEPS], vw[STEPS];
    auto load = [&](uint4 (&w)[STEPS], const signed char* codes, int n) {
      const Block& f = s_block[n % FACS];
      const int have = keys - n * 128;
      const signed char* from = codes + (row0 & 15) * D + c * 16;
      long long at[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) at[i] = f.at[(i * ROWS + row0) >> 4];
      if (have >= 128 && !f.bad) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(from + at[i]));
      } else {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          w[i] = make_uint4(0u, 0u, 0u, 0u);
          if (i * ROWS + row0 < have && at[i] >= 0) w[i] = __ldg(reinterpret_cast<const uint4*>(from + at[i]));
        }
      }
    };
    auto store = [&](const uint4 (&w)[STEPS], uint32_t dst, const bool values) {
      auto first_two = [&](uint32_t x) { return values ? exact_two(x, 0x4140) : __byte_perm(x, 0u, 0x4140); };
      auto last_two = [&](uint32_t x) { return values ? exact_two(x, 0x4342) : __byte_perm(x, 0u, 0x4342); };
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int row = i * ROWS + row0;
        const uint32_t x[4] = {w[i].x ^ 0x80808080u, w[i].y ^ 0x80808080u, w[i].z ^ 0x80808080u, w[i].w ^ 0x80808080u};
        const uint32_t at = dst + part + row * 128;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(at + ((((c & 3) * 2 + e) ^ (row0 & 7)) << 4)), "r"(first_two(x[2 * e])), "r"(last_two(x[2 * e])),
                       "r"(first_two(x[2 * e + 1])), "r"(last_two(x[2 * e + 1])) : "memory");
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
    if (blocks && ok) load(kw, a.k, 0);
    for (int n = 0; ok && n < blocks; ++n) {
      load(vw, a.v, n);
      if (n >= STAGES) ok = bar_wait(smem_addr(&b_kempty[n % STAGES]), (uint32_t)(n / STAGES - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      store(kw, kbuf + (n % STAGES) * OP, false);
      if (lane == 0) {
        bar_arrive(smem_addr(&b_kfull[n % STAGES]));
        bar_arrive(smem_addr(&b_facfree[n % FACS]));
      }
      if (n + 1 < blocks) {
        look(n + 1);
        if (!ok) break;
        load(kw, a.k, n + 1);
      }
      if (n >= STAGES) ok = bar_wait(smem_addr(&b_vempty[n % STAGES]), (uint32_t)(n / STAGES - 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      store(vw, vbuf + (n % STAGES) * OP, true);
      if (lane == 0) bar_arrive(smem_addr(&b_vfull[n % STAGES]));
    }
  } else {
    // ---- queries: as they are, 16 bytes a thread at a time; then a thread a row: bfloat16 rows times a power of two each, and the sums. (Loops that are
    // not unrolled: every CTA comes here once, and had to wait for the instructions.)
    constexpr int IN_ROW = D / 8;
    const int tiles = both ? 2 : 1;
#pragma unroll 4
    for (int i = tid; i < tiles * 128 * IN_ROW; i += SOFTMAX * 32) {
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
    if (!BF16) ready();                                   // (as they are)
    asm volatile("bar.sync 1, %0;\n" ::"n"(SOFTMAX * 32) : "memory");   // (behind nothing that may be given up)
    if (tid < tiles * 128) {
      const int r = tid & 127;
      unsigned char* const row = gbase + (tid >> 7) * OP + r * 128;
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
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int c = 0; c < IN_ROW; ++c) {
        const uint4 w = *piece(c);
        uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (BF16) x[e] = half_pair(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[e]));
          sums[e] += y.x + y.y;
        }
        if (BF16) *piece(c) = make_uint4(x[0], x[1], x[2], x[3]);
      }
      s_rowf[tid] = __uint_as_float((uint32_t)(127 - sh) << 23) * a.scale2;
      s_sum128[tid] = ((sums[0] + sums[1]) + (sums[2] + sums[3])) * (128.f / 16777216.f);
    }
    if (BF16) ready();
    asm volatile("bar.sync 1, %0;\n" ::"n"(SOFTMAX * 32) : "memory");   // (the factors of the rows)
    // ---- softmax: thread = row r of stream z
    const int z = warp >> 2, r = (warp & 3) * 32 + lane, turns = z ? turns1 : turns0, zrow = both ? z * 128 : 0, ztok = both ? z * tok : 0;
    const int tl = ztok + token_of(r);
    const bool row_in = r < tok * rep && tl < n2;
    const int limit = row_in ? min(pos0 + tl, keys - 1) : -1;   // last visible position
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t st = tmem + lanes + z * 128, ot = tmem + lanes + 256 + z * D;
    bool ok = !(a.give_up & 1u);
    if (!ok) s_fail = 1;
    const float rowf = limit < 0 ? 0.f : s_rowf[zrow + r], sum128 = limit < 0 ? 0.f : s_sum128[zrow + r];   // (a row that sees nothing has zeros, whatever its query is)
    float m = NONE, l = 0.f;
    for (int i = 0; ok && i < turns; ++i) {
      const int n = both ? i : 2 * i + z;
      const uint32_t turn = (uint32_t)i & 1u;
      const int j0 = n * 128;
      const bool plain = __all_sync(0xffffffffu, !row_in || j0 + 127 <= limit);   // (rows that stand for no token are never stored)
      ok = bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail) && bar_wait(smem_addr(&b_s[z]), turn, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const Block& f = s_block[n % FACS];
      const unsigned bad = f.bad;
      const bool odd = !plain || bad;
      // Loops over 32 columns (the weights' over 64), not over all: three kinds of warps run at once, and with the block's 128 columns laid out in a row they waited for
      // their instructions more than for anything else (4.2 of 12 cycles an instruction; with one tile a CTA the prompt above took 207 us, so 137).
      // What a row does not see, and of a page that there is not, or whose scale is no number, what makes the rows NaN that do see it:
      auto hide = [&](uint32_t (&x)[32], int c0) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (bad >> (c0 / 16 + j / 16) & 1u) x[j] = 0x7fffffffu;
          if (j0 + c0 + j > limit) x[j] = 0xff800000u;
        }
      };
      // ---- the largest exponent; and the largest that is taken from a score
      float mn = NONE, taken = 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t x[32];
        ld32(st + c0, x);
        const float2 kf = *reinterpret_cast<const float2*>(&f.kf[c0 / 16]), lv = *reinterpret_cast<const float2*>(&f.lv[c0 / 16]);
        wait_ld();
        landed32(x);
        if (odd) hide(x, c0);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float t[2] = {__uint_as_float(x[q * 16]), __uint_as_float(x[q * 16 + 1])};
#pragma unroll
          for (int j = 2; j < 16; j += 4) {               // (three operands: one instruction)
            t[0] = fmaxf(fmaxf(t[0], __uint_as_float(x[q * 16 + j])), __uint_as_float(x[q * 16 + j + 1]));
            if (j + 2 < 16) t[1] = fmaxf(fmaxf(t[1], __uint_as_float(x[q * 16 + j + 2])), __uint_as_float(x[q * 16 + j + 3]));
          }
          const float k = score_factor(q ? kf.y : kf.x, rowf);
          const float at = fmaf(-sum128, k, q ? lv.y : lv.x);
          mn = fmaxf(mn, fmaf(fmaxf(t[0], t[1]), k, at));
          taken = fmaxf(taken, fabsf(at));
        }
      }
      const bool grown = mn - m > GROWTH_LOG2;              // (of a row that had seen nothing: infinite, or nothing again and no number; far from zero m + 6 is more than that)
      const float up = grown ? ex2(m - mn) : 1.f;         // 0 for a row that had seen nothing; other rows of the warp keep theirs
      l *= up;
      if (i && __any_sync(0xffffffffu, grown && m != NONE)) {   // (the scores are there: the stream's product before them is over)
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          ld32(ot + q * 32, o);
          wait_ld();
          landed32(o);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * up);
          st16(ot + q * 32, o);
          st16(ot + q * 32 + 16, o + 16);
        }
      }
      if (grown) m = mn;
      const float mu = m == NONE ? 0.f : m;
      // Exponents are taken from the products without a rounding in between, the reference and what it is joined with have one: far from zero that alone would be a
      // large exponent.
      const bool far = __any_sync(0xffffffffu, fmaxf(fabsf(mu), taken) > FAR);
      const float ref = (far ? 0.f : mu) - WEIGHT_LOG2;
      // ---- weights
#pragma unroll 2
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t x[32], p[16];
        ld32(st + c0, x);
        const float2 kf = *reinterpret_cast<const float2*>(&f.kf[c0 / 16]), lv = *reinterpret_cast<const float2*>(&f.lv[c0 / 16]), iv = *reinterpret_cast<const float2*>(&f.iv[c0 / 16]);
        float k[2] = {score_factor(kf.x, rowf), score_factor(kf.y, rowf)}, at[2] = {fmaf(-sum128, k[0], lv.x), fmaf(-sum128, k[1], lv.y)};
        wait_ld();
        landed32(x);
        if (far) {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(fmaf(__uint_as_float(x[j]), k[j / 16], at[j / 16]) - mu);
          k[0] = k[1] = 1.f;
          at[0] = at[1] = 0.f;
        }
        if (odd) hide(x, c0);                             // (behind that: a page that a row does not see may have factors that are infinite with this row's)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint64_t k2 = pair(__float_as_uint(k[q]), __float_as_uint(k[q])), at2 = pair(__float_as_uint(at[q] - ref), __float_as_uint(at[q] - ref));
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t p0, p1;
            unpair(fma2(pair(x[q * 16 + 2 * j], x[q * 16 + 2 * j + 1]), k2, at2), p0, p1);
            p0 = __float_as_uint(ex2(__uint_as_float(p0)));
            p1 = __float_as_uint(ex2(__uint_as_float(p1)));
            sum[j & 1] = add2(sum[j & 1], pair(p0, p1));
            p[q * 8 + j] = half_pair(__uint_as_float(p0), __uint_as_float(p1));
          }
          uint32_t a0, a1;
          unpair(add2(sum[0], sum[1]), a0, a1);
          l = fmaf(__uint_as_float(a0) + __uint_as_float(a1), q ? iv.y : iv.x, l);
        }
        st16(st + c0 / 2, p);                             // (over scores that have been read)
        if (c0 & 32) {                                    // 64 keys' weights are there
          wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(smem_addr(&b_p[z][c0 >> 6]));
        }
      }
      if (lane == 0) bar_arrive(smem_addr(&b_facfree[n % FACS]));
    }
    if (both && z == 0)                                   // (blocks that tile 1 alone sees)
      for (int n = turns; ok && n < blocks; ++n) {
        ok = __all_sync(0xffffffffu, bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail));
        if (ok && lane == 0) bar_arrive(smem_addr(&b_facfree[n % FACS]));
      }
    // ---- out, through shared memory, 16 bytes a lane. A single tile's streams together: maxima and sums through shared memory; stream z takes half z of the
    // columns, of both sums. Of a pair either takes both halves of its own.
    constexpr int LD = COLS * 2 + 16, LANES = COLS / 8;   // bytes of half a row (and 16: no bank conflicts), lanes that take it
    unsigned char* const rows = gbase + warp * 32 * LD;   // (queries and keys are done with)
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
              v[e] = (x0 + x1) * d;
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
  auto kern = kv8_prompt_kernel<BF16, D>;
  QSPEC_CUDA(limit.raise(kern, Sizes<D>::SMEM));
  // tiles of all requests at most: full ones, and one more for each request that is large enough
  const int per = (128 / a.rep) << a.pair;
  const long long tiles = a.ntok / per + std::min<long long>(a.nreq, (long long)a.ntok * a.rep / PROMPT_ROWS + 1);
  QSPEC_REQUIRE(tiles <= 65535, QSPEC_ERR_UNSUPPORTED, "kv8_attention: %d tokens are too many for one call", a.ntok);
  QSPEC_CUDA(launch_pdl(kern, dim3(a.G, (unsigned)tiles), dim3(NTHREADS), Sizes<D>::SMEM, stream, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}

}  // namespace prompt

int launch_prompt(const PromptArgs& a, int D, bool bf16, cudaStream_t stream) {
  return bf16 ? (D == 128 ? prompt::launch<true, 128>(a, stream) : prompt::launch<true, 64>(a, stream))
              : (D == 128 ? prompt::launch<false, 128>(a, stream) : prompt::launch<false, 64>(a, stream));
}
}  // namespace kv8

// CTAs of the form above that gave a wait up since the library was loaded on the current device; -1: not readable. Synchronises.
int kv8_timeouts() {
  unsigned n = 0;
  return cudaMemcpyFromSymbol(&n, atile::attn_tile_timeouts, sizeof(n)) == cudaSuccess ? (int)(n & 0x1fffffffu) : -1;
}
}  // namespace qspec
