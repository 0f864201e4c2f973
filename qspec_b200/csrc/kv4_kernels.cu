// A key/value cache in pages and in 4 bits: its writer, and rows back in 16 bits. Layout and number format: kv4_common.cuh; pages and slots of a step: kv8_kernels.cu; the
// attention that reads it: kv4_attention.cu.
#include "kv4_common.cuh"

namespace qspec {
namespace kv4 {

// ---- rows into pages --------------------------------------------------------------------------------------------------------------
// y = the rotation of x (neox pairs; queries and keys), then, if `hadamard`, y H / sqrt(D) with the Hadamard matrix of D (which leaves every product of a query and a key as it
// is, and spreads a channel that is large in all keys over a row's columns). Of a row of keys or values, in float32:
//   hi = max(largest, 0), lo = min(smallest, 0)   of the values that are finite; beyond 2^126 they count as 2^126
//   s = max((hi - lo) * (1 / 15), 2^-60), rounded to five significant bits, halves up;   z = rint(-lo / s);   c = clamp(rint(x / s) + z, 0, 15)
// All with the roundings that the formulas have (no fused multiply-adds, quotients by s correctly rounded, a product with 1 / 15 as float32 has it, which is a little more: halves stay
// halves or above), so that the same codes come out of every implementation of them in float32 (one that divides by 15 instead gives another scale to one row in a million): scales of
// five bits and values of eight or eleven make quotients that lie halfway between two codes common.
//
// D / 16 lanes take a row; a lane holds sixteen of its values, eight of each half, so that it has both of every pair that the rotation turns, and the butterflies of the
// Hadamard matrix need another lane for D / 16 of D's strides only. What bounds it: bytes, of a prompt (queries come and go in 16 bits); a launch and a chain of loads, of a step.
struct AppendArgs {
  const void* qkv; long long ld;
  const void* cos_sin; int cos_rows;
  const int *positions, *slots;
  uint8_t *k, *v;
  uint16_t *kw, *vw;
  void* q; long long q_ts;
  int ntok, H, G, npages, pshift, rows;           // rows of a token: keys, values, and queries if they are wanted
  int warps, steps;                               // warps of a token, rows of a warp in steps
};
constexpr int APPEND_WARPS = 8;
constexpr float SCALE_FLOOR = 8.673617379884035e-19f, MOST = 8.507059173023462e37f;   // 2^-60, 2^126

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b)); return r; }

// sums and differences of all strides from 1 to D / 2, x[0 .. 7] the columns 8 c .., x[8 .. 15] the same of the second half; then / sqrt(D)
template <int D>
__device__ __forceinline__ void butterflies(float (&x)[16], int c, uint32_t group) {
#pragma unroll
  for (int s = 1; s < 8; s <<= 1)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(i & s)) {
        const float a = x[i], b = x[i + s];
        x[i] = __fadd_rn(a, b);
        x[i + s] = __fsub_rn(a, b);
      }
#pragma unroll
  for (int o = 1; o < D / 16; o <<= 1) {
    const float sign = c & o ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __fmaf_rn(x[i], sign, __shfl_xor_sync(group, x[i], o));   // (exact products: a sum's one rounding)
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i], b = x[i + 8];
    constexpr float f = D == 128 ? 0.08838834764831845f : 0.125f;
    x[i] = __fmul_rn(__fadd_rn(a, b), f);
    x[i + 8] = __fmul_rn(__fsub_rn(a, b), f);
  }
}

// A warp takes `steps` times ROWS rows of a token, the next ones on their way: one look at the position and the angles for all of them. (Steps of two rows a lane, of which a warp took
// no others, 37 us for a prompt of 4200 tokens, 40 / 8 heads; these 25; two steps ahead, and three CTAs an SM, 31.)
template <bool BF16, int D, bool HADAMARD>
__global__ void __launch_bounds__(APPEND_WARPS * 32, 4) kv4_append_kernel(const AppendArgs a) {
  using T = typename Elem16<BF16>::T;
  constexpr int LANES = D / 16, ROWS = 32 / LANES;          // lanes of a row, rows of a warp at a time
  const int lane = threadIdx.x & 31, c = lane % LANES, row0 = lane / LANES;
  const uint32_t group = LANES == 8 ? 0xffu << (lane & 24) : 0xfu << (lane & 28);
  const unsigned id = blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
  const int t = (int)(id / (unsigned)a.warps), r0 = (int)(id % (unsigned)a.warps) * a.steps * ROWS + row0, end = min(r0 - row0 + a.steps * ROWS, a.rows);
  pdl_enter();
  if (t >= a.ntok) return;
  const int pos = a.positions[t], slot = a.slots[t];
  // rows of a token, in this order: keys, values, queries; they lie as queries, keys, values
  const T* const from = (const T*)a.qkv + (size_t)t * a.ld + c * 8;
  uint4 lo, hi;
  auto load = [&](int r) {
    if (r >= end) return;
    const T* row = from + (r < 2 * a.G ? a.H + r : r - 2 * a.G) * D;
    lo = __ldg(reinterpret_cast<const uint4*>(row));
    hi = __ldg(reinterpret_cast<const uint4*>(row + D / 2));
  };
  load(r0);
  if ((unsigned)pos >= (unsigned)a.cos_rows) return;
  const bool kept = slot >= 0 && slot < a.npages << a.pshift;
  float cs[8], sn[8];
  {
    const T* tab = (const T*)a.cos_sin + (size_t)pos * D + c * 8;
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab), cs);
    unpack8<BF16>(*reinterpret_cast<const uint4*>(tab + D / 2), sn);
  }
  auto row = [&](int r, const uint4& lo_r, const uint4& hi_r) {
    if (r >= end || (r < 2 * a.G && !kept)) return;         // (the same for all lanes of a row)
    float x[16];
    {
      float l[8], h[8];
      unpack8<BF16>(lo_r, l);
      unpack8<BF16>(hi_r, h);
      if (r < a.G || r >= 2 * a.G) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __fsub_rn(__fmul_rn(l[e], cs[e]), __fmul_rn(h[e], sn[e]));
          x[e + 8] = __fadd_rn(__fmul_rn(h[e], cs[e]), __fmul_rn(l[e], sn[e]));
        }
        if (HADAMARD) butterflies<D>(x, c, group);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = l[e]; x[e + 8] = h[e]; }
      }
    }
    if (r >= 2 * a.G) {
      T* to = (T*)a.q + (size_t)t * a.q_ts + (r - 2 * a.G) * D + c * 8;
      *reinterpret_cast<uint4*>(to) = pack8<BF16>(*reinterpret_cast<const float(*)[8]>(&x[0]));
      *reinterpret_cast<uint4*>(to + D / 2) = pack8<BF16>(*reinterpret_cast<const float(*)[8]>(&x[8]));
      return;
    }
    float top = x[0], low = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) { top = max_nan(top, x[e]); low = min_nan(low, x[e]); }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      top = max_nan(top, __shfl_xor_sync(group, top, o));
      low = min_nan(low, __shfl_xor_sync(group, low, o));
    }
    const bool odd = !(top <= MOST && low >= -MOST);
    if (odd) {                                              // what is not finite does not stretch the scale: infinities have the last codes, what is no number counts as zero
      top = low = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool finite = fabsf(x[e]) < INFINITY;
        x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -MOST), MOST) : 0.f;
        if (finite) { top = fmaxf(top, x[e]); low = fminf(low, x[e]); }
      }
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(group, top, o));
        low = fminf(low, __shfl_xor_sync(group, low, o));
      }
    }
    top = fmaxf(top, 0.f);
    low = fminf(low, 0.f);
    const uint32_t bits = (__float_as_uint(fmaxf(__fmul_rn(__fsub_rn(top, low), 1.f / 15.f), SCALE_FLOOR)) + (1u << 18)) >> 19;
    const float s = __uint_as_float(bits << 19), inv = __frcp_rn(s);
    const int zero = (int)fminf(rintf(__fdiv_rn(-low, s)), 15.f);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float quotient;
      if (odd) {
        quotient = fminf(fmaxf(__fdiv_rn(x[e], s), -16.f), 16.f);
      } else {
        // x / s, correctly rounded: from the correctly rounded reciprocal by one residual (Markstein 1990). |x / s| < 16.
        const float near = __fmul_rn(x[e], inv);
        quotient = __fmaf_rn(__fmaf_rn(-near, s, x[e]), inv, near);
      }
      const int k = (int)(__float_as_uint(__fadd_rn(quotient, 12582912.f)) - 0x4b400000u) + zero;   // rint(quotient): in the last bits of quotient + 1.5 2^23
      w[e >> 3] |= (uint32_t)min(max(k, 0), 15) << (4 * (e & 7));
    }
    const int g = r < a.G ? r : r - a.G;
    const size_t at = ((((size_t)(slot >> a.pshift) * a.G + g) << a.pshift) + (slot & ((1 << a.pshift) - 1)));
    uint8_t* to = (r < a.G ? a.k : a.v) + at * (D / 2) + c * 4;
    *reinterpret_cast<uint32_t*>(to) = w[0];
    *reinterpret_cast<uint32_t*>(to + D / 4) = w[1];
    if (c == 0) (r < a.G ? a.kw : a.vw)[at] = (uint16_t)(bits << 4 | (uint32_t)zero);
  };
#pragma unroll 1
  for (int r = r0; r - row0 < end; r += ROWS) {
    const uint4 l = lo, h = hi;
    load(r + ROWS);
    row(r, l, h);
  }
}

// ---- rows back in 16 bits: out[i, g] = the values of slot i, keys and values. Sixteen values a thread; slots that are none give zeros.
template <bool BF16>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* k, const uint8_t* v, const uint16_t* kw, const uint16_t* vw, const int* slots, void* ko, void* vo, unsigned chunks,
                                                       int G, int dshift, int npages, int pshift) {
  using T = typename Elem16<BF16>::T;
  pdl_enter();
  const uint8_t* codes = blockIdx.y ? v : k;
  const uint16_t* words = blockIdx.y ? vw : kw;
  T* out = (T*)(blockIdx.y ? vo : ko);
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < chunks; i += gridDim.x * 256) {
    const unsigned c = i & ((1u << (dshift - 4)) - 1u), row = i >> (dshift - 4);
    const int s = slots[row / (unsigned)G];
    uint2 w = make_uint2(0u, 0u);
    uint32_t word = 0u;
    if (s >= 0 && s < npages << pshift) {
      const size_t at = (((size_t)(s >> pshift) * G + row % (unsigned)G) << pshift) + (s & ((1 << pshift) - 1));
      w = *reinterpret_cast<const uint2*>(codes + (at << (dshift - 1)) + c * 8);
      word = words[at];
    }
    const float f = word_scale(word), zero = 8388608.f + (float)(word & 15u);
    uint4* to = reinterpret_cast<uint4*>(out + (size_t)i * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__uint_as_float(0x4b000000u | ((h ? w.y : w.x) >> (4 * e) & 15u)) - zero, f);   // (2^23 + c) - (2^23 + z)
      to[h] = pack8<BF16>(x);
    }
  }
}

}  // namespace kv4
}  // namespace qspec

using namespace qspec;
using namespace qspec::kv4;

static int check_cache(const char* who, const void* k, const void* v, const void* kw, const void* vw, int npages, int G, int page_tokens, int D) {
  QSPEC_REQUIRE(k && v && kw && vw, QSPEC_ERR_INVALID_ARG, "%s: null pointer", who);
  QSPEC_REQUIRE(page_shift(page_tokens) > 0, QSPEC_ERR_UNSUPPORTED, "%s: pages of 16, 32, 64 or 128 tokens, got %d", who, page_tokens);
  QSPEC_REQUIRE(D == 64 || D == 128, QSPEC_ERR_UNSUPPORTED, "%s: heads of 64 or 128, got %d", who, D);
  QSPEC_REQUIRE(npages >= 1 && G >= 1 && G <= 1024 && (long long)npages * page_tokens < (1ll << 31), QSPEC_ERR_INVALID_ARG, "%s: pages=%d kv heads=%d", who, npages, G);
  QSPEC_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)kw | (uintptr_t)vw) & 15) == 0, QSPEC_ERR_INVALID_ARG, "%s: codes and their words must begin on a 16-byte boundary", who);
  return QSPEC_OK;
}

extern "C" int qspec_kv4_append(const void* qkv, long long ld, const void* cos_sin, int cos_rows, const int* positions, const int* slots, void* k, void* v, void* k_word, void* v_word,
                                void* q_out, long long q_tok_stride, int ntok, int H, int G, int D, int npages, int page_tokens, int hadamard, int dtype, void* stream) {
  if (int rc = check_cache("kv4_append", k, v, k_word, v_word, npages, G, page_tokens, D)) return rc;
  if (ntok == 0) return QSPEC_OK;
  QSPEC_REQUIRE(qkv && cos_sin && positions && slots, QSPEC_ERR_INVALID_ARG, "kv4_append: null pointer");
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv4_append: float16 or bfloat16 rows");
  QSPEC_REQUIRE(ntok > 0 && ntok < (1 << 24) && H >= 1 && H <= 4096 && cos_rows >= 1, QSPEC_ERR_INVALID_ARG, "kv4_append: tokens=%d heads=%d table rows=%d", ntok, H, cos_rows);
  QSPEC_REQUIRE(ld >= (long long)(H + 2 * G) * D && ld % 8 == 0 && (!q_out || (q_tok_stride >= (long long)H * D && q_tok_stride % 8 == 0)) && ((uintptr_t)qkv & 15) == 0 &&
                    ((uintptr_t)cos_sin & 15) == 0 && ((uintptr_t)q_out & 15) == 0,
                QSPEC_ERR_INVALID_ARG, "kv4_append: rows must lie on 16-byte boundaries (ld=%lld)", ld);
  AppendArgs a{qkv, ld, cos_sin, cos_rows, positions, slots, (uint8_t*)k, (uint8_t*)v, (uint16_t*)k_word, (uint16_t*)v_word, q_out, q_tok_stride, ntok, H, G, npages,
               page_shift(page_tokens), 2 * G + (q_out ? H : 0), 0, 0};
  // Steps of a warp: as few as make warps that the SMs all hold at once (warps that come later begin a chain of loads of their own). us of the kernel, 40 / 8 heads of 128, one step (as few as that), without
  // the Hadamard matrix: 256 tokens 4.9 (4.8), 512: 7.4 (6.5), 700: 8.6 (7.5), 1000: 10.8 (9.5), 1500: 14.7 (10.9), 2000: 18.3 (13.1), 4200: 35.2 (24.7), 8000: 62.3 (43.7); with it 512: 9.3 (8.5), 1000: 13.9
  // (12.4), 4200: 44.8 (34.4). (With warps for twice the SMs' places allowed before there are two steps, 512 tokens took 7.3.)
  const int rows = D == 128 ? 4 : 8, most = (a.rows + rows - 1) / rows;
  const long long at_once = std::max(32ll * std::max(sm_count(), 1) / ntok, 1ll);   // warps of a token
  a.steps = (int)((most + at_once - 1) / at_once);
  a.warps = (most + a.steps - 1) / a.steps;
  const long long warps = (long long)ntok * a.warps;
  QSPEC_REQUIRE(warps < (1ll << 31), QSPEC_ERR_UNSUPPORTED, "kv4_append: %d tokens are too many for one call", ntok);
#define QSPEC_KV4_APPEND(BF) (D == 128 ? (hadamard ? kv4_append_kernel<BF, 128, true> : kv4_append_kernel<BF, 128, false>) : hadamard ? kv4_append_kernel<BF, 64, true> : kv4_append_kernel<BF, 64, false>)
  auto kern = dtype == QSPEC_DTYPE_F16 ? QSPEC_KV4_APPEND(false) : QSPEC_KV4_APPEND(true);
#undef QSPEC_KV4_APPEND
  QSPEC_CUDA(launch_pdl(kern, dim3((unsigned)((warps + APPEND_WARPS - 1) / APPEND_WARPS)), dim3(APPEND_WARPS * 32), 0, (cudaStream_t)stream, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}

extern "C" int qspec_kv4_read(const void* k, const void* v, const void* k_word, const void* v_word, const int* slots, void* k_out, void* v_out, int rows, int G, int D, int npages,
                              int page_tokens, int dtype, void* stream) {
  if (int rc = check_cache("kv4_read", k, v, k_word, v_word, npages, G, page_tokens, D)) return rc;
  if (rows == 0) return QSPEC_OK;
  QSPEC_REQUIRE(rows > 0 && slots && k_out && v_out, QSPEC_ERR_INVALID_ARG, "kv4_read: null pointer or rows=%d", rows);
  QSPEC_REQUIRE(dtype == QSPEC_DTYPE_F16 || dtype == QSPEC_DTYPE_BF16, QSPEC_ERR_UNSUPPORTED, "kv4_read: float16 or bfloat16 rows");
  QSPEC_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0, QSPEC_ERR_INVALID_ARG, "kv4_read: rows must lie on 16-byte boundaries");
  const long long chunks = (long long)rows * G * (D / 16);
  QSPEC_REQUIRE(chunks < (1ll << 30), QSPEC_ERR_UNSUPPORTED, "kv4_read: %d rows are too many for one call", rows);
  const int grid = (int)std::min<long long>((chunks + 255) / 256, (long long)max(sm_count(), 1) * 8);
  auto kern = dtype == QSPEC_DTYPE_F16 ? kv4_read_kernel<false> : kv4_read_kernel<true>;
  QSPEC_CUDA(launch_pdl(kern, dim3(grid, 2), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)k, (const uint8_t*)v, (const uint16_t*)k_word, (const uint16_t*)v_word, slots, k_out,
                        v_out, (unsigned)chunks, G, D == 128 ? 7 : 6, npages, page_shift(page_tokens)));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}
