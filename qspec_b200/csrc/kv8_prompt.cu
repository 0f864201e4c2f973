// Softmax attention of prompt portions over the paged 8-bit cache, on the fifth-generation tensor cores (kv8_attention.cu has the layout, and the form for requests
// with few tokens).
//
// One CTA = 128 rows of one request and key/value head; a row is a (token, query head of the group) pair. Keys are walked in blocks of 128, which belong
// alternately to two streams with a softmax and a sum of values of their own (joined at the end), so that one's products run under the other's softmax:
//   * pages: one warp looks the block's pages and scales up and leaves where the codes are and what their products are multiplied with.
//   * codes: four warps bring a block's keys and values from global memory, make them float16 and store them as the tensor cores want them: the cache
//     is read once, in 8 bits, and is never anywhere in 16. Keys are (c + 128) 2^-24, the subnormal number that a byte is by itself; what the 128 adds
//     to a row's scores is taken out where they enter the exponent. Values are c exactly: a byte behind 0x64 is 1152 + c, less 1152.
//   * S = Q K^T, accumulator [128 x 128] float32 in tensor memory, one for each stream.
//   * softmax: thread = row, four warps a stream. Scores are read twice, for the maximum and for the weights (that keeps 128 of them out of the registers).
//     Weights go back over the scores as float16 (2^-11 relative; the result is rounded to 16 bits as well).
//   * O += P V: weights from tensor memory, values from shared memory as they lie in the cache (operand "MN-major").
// Tensor memory: S | S | O | O = 512 columns. Scales and the exponent that takes the value scale in: as in kv8_attention.cu. O is multiplied again only
// where a row's maximum grew by more than 2^8.
// Bound by the tensor cores (1024 cycles a block of 128 x 128, head 128) and the exponentials (16 a cycle: 1024) at once, and nearly by the schedulers:
// the conversion is 1600 warp instructions beside 2600 of the softmax.
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
  static constexpr size_t USED = (size_t)OP * (1 + 2 * STAGES) + 1024;
  static constexpr size_t SMEM = USED > 120 * 1024 ? USED : 120 * 1024;   // one CTA an SM: each takes all of the tensor memory
  static constexpr int LD = D / 2 + 4;                    // floats of a row's half on its way out
  static_assert(8 * 32 * LD * 4 <= 3 * OP, "rows on their way out, over queries and keys");
};
template <int D> constexpr uint32_t IDESC_S = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
template <int D> constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);

struct alignas(16) Block {                                            // what the other roles have to know of a block: of each 16 of its keys
  long long at[8];                                        // where their codes begin, -1: nowhere
  float kf[8], lv[8], iv[8];                              // scale of the keys; log2 of the values' scale, and its reciprocal
  unsigned bad;                                           // bit q: a page that there is not, or a scale that is no number
};

__device__ __forceinline__ void st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7]) : "memory");
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
  __shared__ float s_ml[2][2][128], s_rowf[128], s_sum128[128];
  __shared__ unsigned long long s_work[NWARPS];
  __shared__ int s_sum[NWARPS], s_at[3];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_fail;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rep = a.rep, tok = 128 / rep, g = blockIdx.x;
  if (tid == 0) {
    s_fail = 0;
    s_at[0] = -1;
    for (int i = 0; i < STAGES; ++i) {
      bar_init(smem_addr(&b_kfull[i]), CONVERT); bar_init(smem_addr(&b_kempty[i]), 1);
      bar_init(smem_addr(&b_vfull[i]), CONVERT); bar_init(smem_addr(&b_vempty[i]), 1);
    }
    for (int i = 0; i < FACS; ++i) { bar_init(smem_addr(&b_fac[i]), 1); bar_init(smem_addr(&b_facfree[i]), SOFTMAX / 2 + CONVERT); }
    for (int i = 0; i < 2; ++i) { bar_init(smem_addr(&b_s[i]), 1); bar_init(smem_addr(&b_p[i][0]), 4); bar_init(smem_addr(&b_p[i][1]), 4); bar_init(smem_addr(&b_o[i]), 1); }
    bar_init(smem_addr(&b_q), SOFTMAX);
    bar_init(smem_addr(&b_join), SOFTMAX);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
  unsigned char* const gbase = raw + (base - smem_addr(raw));
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // ---- this CTA's request and tile: tiles of all requests in a row, the last one of a request (with the longest way) first
  const int per_thread = (a.nreq + NTHREADS - 1) / NTHREADS, b0 = tid * per_thread, requests = max(min(per_thread, a.nreq - b0), 0);
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
  if (lane == 0) s_work[warp] = work;
  __syncthreads();
  work = 0;
#pragma unroll
  for (int w = 0; w < NWARPS; ++w) work += s_work[w];
  auto tiles_of = [&](int b) {
    if (per_thread > 1) load(b, n1, keys1);
    return to_prompt_form(n1, keys1, rep, a.share, work) ? (n1 + tok - 1) / tok : 0;
  };
  int mine = 0;
  for (int i = 0; i < requests; ++i) mine += tiles_of(b0 + i);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  int before = incl - mine;
  for (int w = 0; w < warp; ++w) before += s_sum[w];
  if ((int)blockIdx.y >= before && (int)blockIdx.y < before + mine) {
    int at = before;
    for (int i = 0; i < requests; ++i) {
      const int n = tiles_of(b0 + i);
      if ((int)blockIdx.y < at + n) {
        s_at[0] = b0 + i;
        s_at[1] = n - 1 - ((int)blockIdx.y - at);
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  if (s_at[0] < 0) return;
  const int req = s_at[0], tile = s_at[1];
  const int first = min(max(a.q_start[req], 0), a.ntok), n_new = max(min(a.q_start[req + 1], a.ntok) - first, 0), keys = max(a.kv_len[req], 0);
  const int t0 = tile * tok, n2 = min(tok, n_new - t0);   // this tile's tokens
  const int pos0 = keys - n_new + t0;                     // position of the first
  const int seen = min(pos0 + n2, keys), blocks = seen > 0 ? (seen + 127) / 128 : 0;   // keys that any row sees
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&s_tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (tensor memory is held)
  const uint32_t kbuf = base + OP, vbuf = kbuf + STAGES * OP;

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
      float k = 1.f, v = 1.f;
      if (lane < 8 && key < keys) {
        const int page = at < a.width ? a.table[(size_t)req * a.width + at] : -1;
        bad = (unsigned)page >= (unsigned)a.npages;
        if (!bad) {
          const size_t block = (size_t)page * a.G + g;
          codes = (long long)(((block << a.pshift) + (key & ((1 << a.pshift) - 1))) * D);
          k = a.ks[block];
          v = a.vs[block];
          bad = k != k || v != v;
        }
      }
      const unsigned mask = __ballot_sync(0xffffffffu, bad);
      if (lane < 8) {
        s_block[slot].at[lane] = codes;
        v = positive(v);
        s_block[slot].kf[lane] = positive(k);
        s_block[slot].lv[lane] = __log2f(v);
        s_block[slot].iv[lane] = __fdividef(1.f, v);
        if (lane == 0) s_block[slot].bad = mask;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(smem_addr(&b_fac[slot]));
    }
  } else if (warp == W_MMA) {
    if (elect()) {
      const uint64_t qd = desc_k(base);
      bool ok = !(a.give_up & 4u);
      if (!ok) s_fail = 1;
      int products = 0;                                   // value products that have been issued, block by block
      auto scores = [&](int n) -> bool {
        if (!bar_wait(smem_addr(&b_kfull[n % STAGES]), (uint32_t)(n / STAGES) & 1u, &s_fail)) return false;
        // these scores take the columns of the weights of block n - 2: their product must be over
        if (n >= 2 && !bar_wait(smem_addr(&b_o[n & 1]), (uint32_t)((n >> 1) - 1) & 1u, &s_fail)) return false;
        fence_after();
        const uint64_t kd = desc_k(kbuf + (n % STAGES) * OP);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t step = (uint32_t)((i >> 2) * (PARTB >> 4) + (i & 3) * 2);
          mma_ss(tmem + (n & 1) * 128, qd + step, kd + step, IDESC_S<D>, i ? 1u : 0u);
        }
        commit(smem_addr(&b_s[n & 1]));
        commit(smem_addr(&b_kempty[n % STAGES]));
        return true;
      };
      ok = ok && (blocks == 0 || (bar_wait(smem_addr(&b_q), 0, &s_fail) && scores(0) && (blocks == 1 || scores(1))));
      for (int n = 0; ok && n < blocks; ++n) {
        if (!bar_wait(smem_addr(&b_vfull[n % STAGES]), (uint32_t)(n / STAGES) & 1u, &s_fail)) break;
        const uint64_t vd = desc_mn(vbuf + (n % STAGES) * OP);
        const uint32_t p = tmem + (n & 1) * 128, o = tmem + 256 + (n & 1) * D;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                     // 64 keys each
          ok = ok && bar_wait(smem_addr(&b_p[n & 1][h]), (uint32_t)(n >> 1) & 1u, &s_fail);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i) mma_ts(o, p + h * 32 + i * 8, vd + (h * 4 + i) * (2048 >> 4), IDESC_O<D>, (n > 1 || h || i) ? 1u : 0u);
        }
        if (!ok) break;
        commit(smem_addr(&b_o[n & 1]));
        commit(smem_addr(&b_vempty[n % STAGES]));
        products = n + 1;
        if (n + 2 < blocks && !scores(n + 2)) break;
      }
      if (products < blocks) {                            // given up: what was issued so far
        commit(smem_addr(&b_o[products & 1]));
        products += 1;
      }
      // every product of either stream is over before the CTA leaves
      for (int n = max(products - 2, 0); n < products; ++n) bar_drain(smem_addr(&b_o[n & 1]), (uint32_t)(n >> 1) & 1u);
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
    // ---- queries: 16 bytes a thread at a time, bfloat16 rows by a power of two each
    constexpr int IN_ROW = D / 8, QROWS = SOFTMAX * 32 / IN_ROW;
    {
      const int c = tid % IN_ROW;
      uint4 w[128 / QROWS];
#pragma unroll
      for (int i = 0; i < 128 / QROWS; ++i) {
        const int r = i * QROWS + tid / IN_ROW, tl = r / rep;
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        if (tl < n2 && r < tok * rep)
          w[i] = *reinterpret_cast<const uint4*>((const T*)a.q + (size_t)(first + t0 + tl) * a.q_ts + (size_t)(g * rep + r - tl * rep) * a.q_hs + c * 8);
      }
#pragma unroll
      for (int i = 0; i < 128 / QROWS; ++i) {
        const int r = i * QROWS + tid / IN_ROW;
        uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        int sh = 0;
        if (BF16) {
          float mx = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
#pragma unroll
          for (int o = IN_ROW / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
          sh = mx > 0.f && mx < INFINITY ? min(max(14 - ex, -126), 126) : 0;
          const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = half_pair(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
        }
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[e]));
          sum += y.x + y.y;
        }
#pragma unroll
        for (int o = IN_ROW / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (c == 0) {
          s_rowf[r] = __uint_as_float((uint32_t)(127 - sh) << 23) * a.scale2 * 16777216.f;   // (scores come in units of 2^-24)
          s_sum128[r] = sum * (128.f / 16777216.f);
        }
        *reinterpret_cast<uint4*>(gbase + (c >> 3) * PARTB + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(smem_addr(&b_q));
    }
    // ---- softmax: thread = row r of the blocks of stream z
    const int z = warp >> 2, r = (warp & 3) * 32 + lane;
    const int tl = r / rep;
    const bool row_in = r < tok * rep && tl < n2;
    const int limit = row_in ? min(pos0 + tl, keys - 1) : -1;   // last visible position
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t st = tmem + lanes + z * 128, ot = tmem + lanes + 256 + z * D;
    bool ok = !(a.give_up & 1u);
    if (!ok) s_fail = 1;
    ok = ok && bar_wait(smem_addr(&b_q), 0, &s_fail);     // (the factors of the rows)
    ok = __all_sync(0xffffffffu, ok);
    const float rowf = s_rowf[r], sum128 = s_sum128[r];
    float m = NONE, l = 0.f;
    int n = z;
    for (; ok && n < blocks; n += 2) {
      const uint32_t turn = (uint32_t)(n >> 1) & 1u;
      const int j0 = n * 128;
      const bool plain = __all_sync(0xffffffffu, !row_in || j0 + 127 <= limit);   // (rows that stand for no token are never stored)
      ok = bar_wait(smem_addr(&b_fac[n % FACS]), (uint32_t)(n / FACS) & 1u, &s_fail) && bar_wait(smem_addr(&b_s[z]), turn, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const Block& f = s_block[n % FACS];
      const unsigned bad = f.bad;
      const bool odd = !plain || bad;
      // Loops over 32 columns, not unrolled: three kinds of warps run at once, and with the block's 128 columns laid out in a row they waited for their
      // instructions more than for anything else (4.2 of 12 cycles an instruction; prompt of 2000 after 1000, 32 / 8 heads 207 us, so 137).
      // What a row does not see, and of a page that there is not, or whose scale is no number, what makes the rows NaN that do see it:
      auto hide = [&](uint32_t (&x)[32], int c0) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (bad >> (c0 / 16 + j / 16) & 1u) x[j] = 0x7fffffffu;
          if (j0 + c0 + j > limit) x[j] = 0xff800000u;
        }
      };
      // ---- the largest exponent
      float mn = NONE;
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
          const float k = normal((q ? kf.y : kf.x) * rowf);
          mn = fmaxf(mn, fmaf(fmaxf(t[0], t[1]), k, fmaf(-sum128, k, q ? lv.y : lv.x)));
        }
      }
      const bool grown = mn > m + RESCALE_LOG2 || (m == NONE && mn > m);
      const float up = grown ? ex2(m - mn) : 1.f;         // 0 for a row that had seen nothing; other rows of the warp keep theirs
      l *= up;
      if (n > 1 && __any_sync(0xffffffffu, grown && m != NONE)) {   // (the scores are there: the stream's product before them is over)
#pragma unroll 1
        for (int q = 0; q < D / 8; ++q) {
          uint32_t o[8];
          ld8(ot + q * 8, o);
          wait_ld();
          landed8(o);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * up);
          st8(ot + q * 8, o);
        }
      }
      if (grown) m = mn;
      const float mu = m == NONE ? 0.f : m;
      // Exponents are taken from the products without a rounding in between, the reference has one: beyond 2^24 that alone would be a large exponent.
      const bool far = __any_sync(0xffffffffu, fabsf(mu) > 16777216.f);
      // ---- weights
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t x[32], p[16];
        ld32(st + c0, x);
        const float2 kf = *reinterpret_cast<const float2*>(&f.kf[c0 / 16]), lv = *reinterpret_cast<const float2*>(&f.lv[c0 / 16]), iv = *reinterpret_cast<const float2*>(&f.iv[c0 / 16]);
        float k[2] = {normal(kf.x * rowf), normal(kf.y * rowf)}, at[2] = {fmaf(-sum128, k[0], lv.x), fmaf(-sum128, k[1], lv.y)};
        wait_ld();
        landed32(x);
        if (odd) hide(x, c0);
        if (far) {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(fmaf(__uint_as_float(x[j]), k[j / 16], at[j / 16]));
          k[0] = k[1] = 1.f;
          at[0] = at[1] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint64_t k2 = pair(__float_as_uint(k[q]), __float_as_uint(k[q])), at2 = pair(__float_as_uint(at[q] - mu), __float_as_uint(at[q] - mu));
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
    // ---- the streams together: maxima and sums through shared memory; stream z takes half z of the columns, of both sums. Rows leave through shared memory,
    // 16 bytes a lane.
    constexpr int LD = Z::LD, LANES = COLS / 8, AT_ONCE = 32 / LANES;
    float* const rows = reinterpret_cast<float*>(gbase) + warp * 32 * LD;   // (queries and keys are done with)
    s_ml[z][0][r] = m;
    s_ml[z][1][r] = l;
    __syncwarp();
    if (lane == 0) bar_arrive(smem_addr(&b_join));
    // the last product of either stream, and everyone's maxima
    if (ok) {
      ok = bar_wait(smem_addr(&b_join), 0, &s_fail);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (blocks > i) ok = ok && bar_wait(smem_addr(&b_o[i]), (uint32_t)((blocks - 1 - i) >> 1) & 1u, &s_fail);
      ok = __all_sync(0xffffffffu, ok);
    }
    fence_after();
    if (ok) {
      float f[2], sum = 0.f;
      const float m0 = s_ml[0][0][r], m1 = s_ml[1][0][r], top = fmaxf(m0, m1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mi = i ? m1 : m0, li = s_ml[i][1][r];
        f[i] = mi == NONE ? (li == 0.f ? 0.f : 1.f) : ex2(mi - top);   // nothing seen, or no number
        sum += li * f[i];
      }
      const float d = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);          // (no key: zeros)
      const bool two = __any_sync(0xffffffffu, f[1] != 0.f) && blocks > 1;
#pragma unroll 1
      for (int q = 0; q < COLS / 8; ++q) {
        uint32_t o0[8], o1[8];
        if (blocks > 0) ld8(tmem + lanes + 256 + z * COLS + q * 8, o0);
        if (blocks > 1) ld8(tmem + lanes + 256 + D + z * COLS + q * 8, o1);
        wait_ld();
        landed8(o0);
        landed8(o1);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x0 = f[0] == 0.f ? 0.f : __uint_as_float(o0[e]) * f[0], x1 = two && f[1] != 0.f ? __uint_as_float(o1[e]) * f[1] : 0.f;
          v[e] = (x0 + x1) * d;
        }
        *reinterpret_cast<float4*>(rows + lane * LD + q * 8) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(rows + lane * LD + q * 8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      const uint32_t stored = __ballot_sync(0xffffffffu, row_in);
      __syncwarp();
      const int pc = lane % LANES;
#pragma unroll 1
      for (int k = 0; k < 32 / AT_ONCE; ++k) {
        const int rr = lane / LANES + AT_ONCE * k, r2 = (warp & 3) * 32 + rr, t2 = r2 / rep;
        if (!(stored >> rr & 1u)) continue;
        const float4 x = *reinterpret_cast<const float4*>(rows + rr * LD + pc * 8), y = *reinterpret_cast<const float4*>(rows + rr * LD + pc * 8 + 4);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        *reinterpret_cast<uint4*>((T*)a.out + (size_t)(first + t0 + t2) * a.out_ts + (size_t)(g * rep + r2 - t2 * rep) * a.out_hs + z * COLS + pc * 8) = pack8<BF16>(v);
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
  const int per = 128 / a.rep;
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
