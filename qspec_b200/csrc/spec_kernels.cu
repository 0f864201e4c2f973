// Verification of drafted tokens with given random numbers, and sampling from a row of probabilities (its case of no drafts).
//
// Request b has k drafts d_i, drawn from q_i, and the target's probabilities p_0 .. p_k. Draft i is taken if u_i q_i(d_i) < p_i(d_i) and all before it
// were: with probability min(1, p / q). Behind the taken ones comes one token more, by inversion: at the first place that was refused from what the
// target has over the draft, max(p - q, 0); from p where every draft was taken, or where that difference is zero everywhere. It is the
// first token whose running sum is above u * (sum of all). Tokens are then distributed as the target's own.
//
// Products, differences and sums are those of 64-bit numbers: the first two are exact, and with 150,000 terms a running sum in 32 bits would
// move the borders between tokens by as much as small tokens are wide. That also makes the result one that every implementation finds.
//
// One cluster of CTAs per request; what bounds it is reading two rows of V float32. A warp takes tiles of 1024 values, all of whose loads are on their way
// before the first is used, and keeps each tile's sum; the CTAs exchange their totals through distributed shared memory; the one in whose stretch the border
// lies looks for the tile, reads it again and finds the token in it. Sums are made in a fixed order, so that no atomics and no order of CTAs enter.
#include "common.cuh"

namespace qspec {
namespace spec {

constexpr int THREADS = 256, WARPS = THREADS / 32, PARTS = 8, PART = 128, TILE = PARTS * PART, MAX_DRAFTS = 31;   // a part: four values a lane
constexpr int MAX_TILES = 1024;                   // of a CTA's stretch

struct Args {
  const long long* drafted;
  const float *draft, *target, *uniform;
  const int* counts;
  long long d_ss, d_ps, t_ss, t_ps;               // strides of a request and of a place
  long long *tokens, *emitted;
  int k, V, span;                                 // values of a CTA's stretch (a multiple of TILE)
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// the sum over the lanes in front of this one
__device__ __forceinline__ double warp_before(double v, int lane) {
  double incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  const double w = __shfl_up_sync(0xffffffffu, incl, 1);
  return lane ? w : 0.0;
}
// What is left to draw from. A token one of whose two probabilities is no number has nothing.
__device__ __forceinline__ double rest_of(float p, float q) {
  return p > q ? (double)p - (double)q : 0.0;
}

template <int CLUSTER, bool VEC>
__global__ void __launch_bounds__(THREADS, CLUSTER == 8 ? 4 : 3) verify_drafts_kernel(const Args a) {
  static_assert(PARTS == WARPS, "a part of a tile for each warp");
  __shared__ double s_tile[MAX_TILES], s_total[2];          // of this CTA's stretch: sums of tiles; of max(p - q, 0) and of p
  __shared__ double s_part[PARTS], s_upto;
  __shared__ int s_at;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  pdl_enter();

  // ---- how many drafts are taken (every warp for itself)
  const int k = a.counts ? min(max(a.counts[b], 0), a.k) : a.k;
  bool refused = true;
  if (lane < a.k) {
    const long long d = a.drafted[(size_t)b * a.k + lane];
    if (d >= 0 && d < a.V) {
      const float q = a.draft[b * a.d_ss + lane * a.d_ps + d], p = a.target[b * a.t_ss + lane * a.t_ps + d];
      refused = !((double)a.uniform[(size_t)b * (a.k + 1) + lane] * (double)q < (double)p);
    }
  }
  const uint32_t no = __ballot_sync(0xffffffffu, refused && lane < k);
  const int taken = no ? __ffs(no) - 1 : k;
  const float* p = a.target + b * a.t_ss + taken * a.t_ps;
  bool differ = taken < k;                                  // draw from max(p - q, 0)
  const float* q = differ ? a.draft + b * a.d_ss + taken * a.d_ps : p;
  const int lo = min(rank * a.span, a.V), hi = min(lo + a.span, a.V), tiles = (hi - lo + TILE - 1) / TILE;

  auto four = [&](const float* row, int at) -> float4 {     // values at .. at + 3 of a row, zeros behind the stretch
    if (VEC && at + 4 <= hi) return *reinterpret_cast<const float4*>(row + at);
    return make_float4(at < hi ? row[at] : 0.f, at + 1 < hi ? row[at + 1] : 0.f, at + 2 < hi ? row[at + 2] : 0.f, at + 3 < hi ? row[at + 3] : 0.f);
  };
  auto rest4 = [&](const float4& x, const float4& y) { return (rest_of(x.x, y.x) + rest_of(x.y, y.y)) + (rest_of(x.z, y.z) + rest_of(x.w, y.w)); };
  const float4 nothing = make_float4(0.f, 0.f, 0.f, 0.f);

  double total = 0.0, before = 0.0;
  int second = 0;
  for (int pass = 0; pass < 2; ++pass) {                    // (a second time where the difference has nothing)
    for (int t = warp; t < tiles; t += WARPS) {
      double s = 0.0;
#pragma unroll 1
      for (int i0 = 0; i0 < PARTS; i0 += 4) {               // (eight loads a lane under way; 24 warps an SM: sixteen of 16 warps took 47 us for 190 requests, these 44)
        float4 pv[4], qv[4];
        const int at = lo + t * TILE + i0 * PART + lane * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pv[i] = four(p, at + i * PART);
          qv[i] = differ ? four(q, at + i * PART) : nothing;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s += rest4(pv[i], qv[i]);
      }
      s = warp_sum(s);
      if (lane == 0) s_tile[t] = s;
    }
    __syncthreads();
    // the stretch's sum in the order of its tiles
    if (warp == 0) {
      double s = 0.0;
      const int each = (tiles + 31) / 32;
      for (int i = 0; i < each; ++i)
        if (lane * each + i < tiles) s += s_tile[lane * each + i];
      s = warp_sum(s);
      if (lane == 0) s_total[pass] = s;
    }
    if (CLUSTER > 1) cluster_sync_all(); else __syncthreads();
    total = before = 0.0;
    for (int r = 0; r < CLUSTER; ++r) {
      double s;
      if (CLUSTER > 1) {
        const uint32_t addr = mapa_shared((uint32_t)__cvta_generic_to_shared(&s_total[pass]), r);
        asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(s) : "r"(addr) : "memory");
      } else {
        s = s_total[pass];
      }
      if (r < rank) before += s;
      total += s;
    }
    if (total > 0.0 || !differ) break;
    differ = false;                                         // (uniform over the cluster)
    second = 1;
    __syncthreads();
  }
  if (CLUSTER > 1) cluster_arrive_release();                // this CTA has read the others' sums

  // ---- the token: in the CTA whose stretch holds the border. (Every CTA has the same sums of the stretches in front of it, so that exactly one has it.)
  // A random number outside [0, 1) is taken for the nearest one inside.
  const double border = (double)fminf(fmaxf(a.uniform[(size_t)b * (a.k + 1) + a.k], 0.f), 0.99999994f) * total;
  const bool mass = total > 0.0 && total < (double)INFINITY;
  const double after = before + s_total[second];
  if (mass ? before <= border && border < after : rank == 0) {   // (the same for all of the CTA)
    if (warp == 0) {                                        // the tile, and the sum in front of it
      const int each = (tiles + 31) / 32;
      double s = 0.0;
      for (int i = 0; i < each; ++i)
        if (lane * each + i < tiles) s += s_tile[lane * each + i];
      double run = before + warp_before(s, lane);           // the sum in front of this lane's tiles
      // (the sums of tiles and those of stretches are added in different orders: where the border lies within their last bits, the last tile counts)
      uint32_t at = __ballot_sync(0xffffffffu, s > 0.0 && run + s > border);
      if (!at) at = 0x80000000u >> __clz(__ballot_sync(0xffffffffu, s > 0.0) | 1u);
      if (lane == __ffs(at) - 1) {
        int tile = 0;
        double upto = run;
        for (int i = 0; i < each && lane * each + i < tiles; ++i) {
          const double x = s_tile[lane * each + i];
          if (!(x > 0.0)) continue;
          tile = lane * each + i;                           // the one that passes the border, or the last one with something
          upto = run;
          if (run + x > border) break;
          run += x;
        }
        s_at = tile;
        s_upto = upto;
      }
    }
    __syncthreads();
    // the tile's parts, one a warp; then the values of the one that has the border
    const int first = lo + s_at * TILE + warp * PART + lane * 4;
    const float4 pv = four(p, first), qv = differ ? four(q, first) : nothing;
    const double x[4] = {rest_of(pv.x, qv.x), rest_of(pv.y, qv.y), rest_of(pv.z, qv.z), rest_of(pv.w, qv.w)};
    const double s = (x[0] + x[1]) + (x[2] + x[3]), mine = warp_sum(s);
    if (lane == 0) s_part[warp] = mine;
    __syncthreads();
    double run = s_upto, upto = s_upto;
    int where = 0;
#pragma unroll 1
    for (int i = 0; i < PARTS; ++i) {
      const double y = s_part[i];
      if (!(y > 0.0)) continue;
      where = i;
      upto = run;
      if (run + y > border) break;
      run += y;
    }
    if (warp == where) {
      int token = 0;                                        // of a row without any mass
      run = upto + warp_before(s, lane);
      uint32_t at = __ballot_sync(0xffffffffu, s > 0.0 && run + s > border);
      if (!at) at = 0x80000000u >> __clz(__ballot_sync(0xffffffffu, s > 0.0) | 1u);
      if (mass && lane == __ffs(at) - 1) {
        bool over = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!over && x[e] > 0.0) {
            token = first + e;
            run += x[e];
            over = run > border;
          }
        }
      }
      token = __shfl_sync(0xffffffffu, token, __ffs(at) - 1);
      if (lane <= a.k) {
        long long* to = a.tokens + (size_t)b * (a.k + 1) + lane;
        *to = lane < taken ? a.drafted[(size_t)b * a.k + lane] : lane == taken ? (long long)token : -1ll;
      }
      if (lane == 0) a.emitted[b] = taken + 1;
    }
  }
  if (CLUSTER > 1) cluster_wait_acquire();                  // the others have read this CTA's sum
}

}  // namespace spec
}  // namespace qspec

using namespace qspec;
using namespace qspec::spec;

extern "C" int qspec_verify_drafts_max_drafts(void) { return MAX_DRAFTS; }

extern "C" int qspec_verify_drafts(const long long* drafted, const float* draft, long long draft_seq_stride, long long draft_place_stride, const float* target,
                                   long long target_seq_stride, long long target_place_stride, const float* uniform, const int* draft_counts, long long* tokens,
                                   long long* emitted, int requests, int drafts, int vocab, void* stream) {
  QSPEC_REQUIRE(requests >= 0 && drafts >= 0 && vocab >= 1, QSPEC_ERR_INVALID_ARG, "verify_drafts: requests=%d drafts=%d vocabulary=%d", requests, drafts, vocab);
  if (requests == 0) return QSPEC_OK;
  QSPEC_REQUIRE(target && uniform && tokens && emitted && (drafts == 0 || (drafted && draft)), QSPEC_ERR_INVALID_ARG, "verify_drafts: null pointer");
  QSPEC_REQUIRE(drafts <= MAX_DRAFTS, QSPEC_ERR_UNSUPPORTED, "verify_drafts: at most %d drafts, got %d", MAX_DRAFTS, drafts);
  QSPEC_REQUIRE(vocab <= 8 * MAX_TILES * TILE && requests <= (1 << 24), QSPEC_ERR_UNSUPPORTED, "verify_drafts: vocabulary of %d, %d requests", vocab, requests);
  QSPEC_REQUIRE((drafts == 0 || (draft_seq_stride >= 0 && draft_place_stride >= 0)) && target_seq_stride >= 0 && target_place_stride >= 0, QSPEC_ERR_INVALID_ARG,
                "verify_drafts: negative stride");
  Args a{drafted, draft, target, uniform, draft_counts, draft_seq_stride, draft_place_stride, target_seq_stride, target_place_stride, tokens, emitted, drafts, vocab, 0};
  const bool vec = (((uintptr_t)target | (uintptr_t)(drafts ? draft : target)) & 15) == 0 && ((target_seq_stride | target_place_stride) & 3) == 0 &&
                   (drafts == 0 || ((draft_seq_stride | draft_place_stride) & 3) == 0);
  // CTAs of a request: eight where two rounds of such clusters hold all requests (a row's way through the GPU counts), four where they fill it by themselves. Three
  // drafts, us with eight (four): vocabulary of 152064, 64 requests 13.7 (16.8), 80: 20.7 (18.0), 96: 23.6 (19.2), 128: 28.0 (32.0), 190: 41.6 (38.8), 256: 53.4 (53.0);
  // of 32000, 16: 6.2 (5.9), 64: 7.6 (7.7), 80: 10.6 (7.9), 128: 12.7 (11.0), 256: 22.6 (17.2). (128 of the larger vocabulary is the one that the rule takes the slower
  // way: 512 CTAs, three an SM, leave a second round nearly empty.) Rows that do not begin on 16 bytes are loaded value by value: of 151643, 64 requests 18.4 (152064: 13.9), 190 of five
  // drafts 48.0 (39.9). Without drafts, of 128256: 4 rows 6.6, 64 rows 11.9; 190 rows of 152064 32.1.
  const bool many = requests > sm_count() / 2 && vocab <= 4 * MAX_TILES * TILE;
  const int cluster = many ? 4 : 8;
  a.span = ((vocab + cluster - 1) / cluster + TILE - 1) / TILE * TILE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(requests * cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  auto kern = many ? (vec ? verify_drafts_kernel<4, true> : verify_drafts_kernel<4, false>) : (vec ? verify_drafts_kernel<8, true> : verify_drafts_kernel<8, false>);
  QSPEC_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  QSPEC_CHECK_LAUNCH(1);
  return QSPEC_OK;
}
