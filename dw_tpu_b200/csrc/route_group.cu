// Group-limited top-k routing: of num_groups groups of consecutive experts
// the topk_groups best stay open, and the top k experts are chosen among
// theirs. Scores and the choice bias are those of route_topk (route.cu).
//
// The order of experts and groups is that of their values in 64 bits: f32
// scores of different logits round to the same number often enough (a sigmoid
// near 1, a bias much larger than a score) that an f32 order would depend on
// the way they are computed. Without a bias the experts are ordered by their
// logits, which every scoring function preserves.
//
// One warp per token; lane l holds experts l, l + 32, ...
#include "common.cuh"

namespace dwm {
namespace route_group {

constexpr int WARPS = 4;

struct Args {
  const void* logits;
  int64_t ld;
  const float* bias;
  int t, e, top_k, groups, keep, per;
  int scoring, top2, renorm, num_valid;
  float scale;
  int32_t* ids;
  float* w32;
  uint16_t* w16;
};

// Keys that order like the values: removed (0) < NaN (1) < -inf < ... < +inf,
// -0 = +0.
__device__ __forceinline__ uint64_t key_of(double v) {
  if (isnan(v)) return 1;
  const int64_t b = __double_as_longlong(v + 0.0);
  return (uint64_t)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double value_of(uint64_t key) {
  if (key <= 1) return __longlong_as_double(0x7FF8000000000000ll);
  return __longlong_as_double((int64_t)(key >> 63 ? key ^ (1ull << 63) : ~key));
}

// The score of logit x; softmax needs the row's maximum and sum.
__device__ __forceinline__ double score(double x, int scoring, double mx, double sum) {
  if (scoring == DWM_SCORE_SOFTMAX) {
    const double d = x == mx ? 0.0 : x - mx;  // +inf logits share the weight
    return mx == -INFINITY ? 0.0 : exp(d) / sum;
  }
  if (scoring == DWM_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-x));
  return sqrt(fmax(x, 0.0) + log1p(exp(-fabs(x))));
}

template <int LD>
__device__ __forceinline__ float load_logit(const void* logits, int64_t i) {
  if constexpr (LD == DWM_BF16)
    return bf16_bits_to_f32(static_cast<const uint16_t*>(logits)[i]);
  else
    return static_cast<const float*>(logits)[i];
}

// The warp's largest key and, of the lanes that hold it, the lowest index.
__device__ __forceinline__ void warp_best(uint64_t& key, int& idx) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t k = __shfl_xor_sync(0xffffffffu, key, o);
    const int i = __shfl_xor_sync(0xffffffffu, idx, o);
    if (k > key || (k == key && i < idx)) { key = k; idx = i; }
  }
}

// Row `tok` in 64 bits: lane j < top_k returns the j-th expert and weight.
// buf: e keys of this warp's shared memory.
template <int LD>
__device__ void route_row64(const Args& a, int64_t tok, uint64_t* buf, int lane, int& id,
                            float& weight) {
  const int64_t row = tok * a.ld;
  double mx = -INFINITY, sum = 0.0;
  if (a.scoring == DWM_SCORE_SOFTMAX) {
    for (int x = lane; x < a.e; x += 32) mx = fmax(mx, (double)load_logit<LD>(a.logits, row + x));
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    for (int x = lane; x < a.e; x += 32) {
      const double v = load_logit<LD>(a.logits, row + x);
      sum += v == mx ? 1.0 : exp(v - mx);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  for (int x = lane; x < a.e; x += 32) {
    const double v = load_logit<LD>(a.logits, row + x);
    buf[x] = key_of(a.bias ? score(v, a.scoring, mx, sum) + (double)a.bias[x] : v);
  }
  __syncwarp();

  // Lane g < groups: the value of group g, then its rank among the groups.
  uint64_t gkey = 0;
  if (lane < a.groups) {
    uint64_t m1 = 0, m2 = 0;
    for (int p = 0; p < a.per; ++p) {
      const uint64_t k = buf[lane * a.per + p];
      m2 = max(m2, min(m1, k));
      m1 = max(m1, k);
    }
    gkey = m1;
    if (a.top2) {
      double v = 0.0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint64_t k = j ? m2 : m1;
        if (k == 0) break;  // groups of one expert
        const double u = value_of(k);
        v += a.bias ? u : score(u, a.scoring, mx, sum);
      }
      gkey = key_of(v);
    }
  }
  int rank = 0;
  for (int g = 0; g < a.groups; ++g) {
    const uint64_t k = __shfl_sync(0xffffffffu, gkey, g);
    rank += k > gkey || (k == gkey && g < lane);
  }
  const uint32_t open = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.keep);
  for (int x = lane; x < a.e; x += 32)
    if (!(open >> (x / a.per) & 1u)) buf[x] = 0;
  __syncwarp();

  double s = 0.0;
  id = 0;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t bk = 0;
    int bi = 0x7fffffff;
    for (int x = lane; x < a.e; x += 32) {
      const uint64_t v = buf[x];
      if (v > bk) { bk = v; bi = x; }
    }
    warp_best(bk, bi);
    if (lane == k) id = bi;
    if (lane == (bi & 31)) buf[bi] = 0;
    __syncwarp();
  }
  if (lane < a.top_k) s = score(load_logit<LD>(a.logits, row + id), a.scoring, mx, sum);
  if (a.renorm) {
    double total = 0.0;
    for (int k = 0; k < a.top_k; ++k) total += __shfl_sync(0xffffffffu, s, k);
    s = total == 0.0 ? 0.0 : s / total;
  }
  weight = (float)(s * (double)a.scale);
}

template <int LD>
__global__ void __launch_bounds__(32 * WARPS) route_grouped_kernel(const Args a) {
  extern __shared__ uint64_t keys[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * WARPS + warp;
  if (tok >= a.t) return;
  int id = 0;
  float w = 0.0f;
  if (a.num_valid < 0 || tok < a.num_valid)
    route_row64<LD>(a, tok, keys + warp * a.e, lane, id, w);
  if (lane < a.top_k) {
    a.ids[tok * a.top_k + lane] = id;
    if (a.w32) a.w32[tok * a.top_k + lane] = w;
    if (a.w16) a.w16[tok * a.top_k + lane] = (uint16_t)f32_to_bf16_bits(w);
  }
}

}  // namespace route_group
}  // namespace dwm

using namespace dwm;

extern "C" int dwm_route_grouped_topk(const void* logits, int logits_dtype, int64_t ld_logits,
                                      int t, int e, int top_k, int num_groups, int topk_groups,
                                      int scoring, int group_score, int renormalize,
                                      float routed_scale, const float* bias,
                                      int num_valid_tokens, int32_t* topk_ids,
                                      float* topk_weights_f32, void* topk_weights_bf16,
                                      void* stream) {
  DWM_CHECK_ARG(logits_dtype == DWM_BF16 || logits_dtype == DWM_F32,
                "logits dtype must be bf16 or f32");
  DWM_CHECK_ARG(t >= 0 && e >= 1 && e <= 1024, "bad shape t=%d e=%d (e in [1, 1024])", t, e);
  DWM_CHECK_ARG(num_groups >= 1 && num_groups <= 32 && e % num_groups == 0,
                "num_groups=%d must be in [1, 32] and divide e=%d", num_groups, e);
  DWM_CHECK_ARG(topk_groups >= 1 && topk_groups <= num_groups,
                "topk_groups=%d must be in [1, num_groups=%d]", topk_groups, num_groups);
  DWM_CHECK_ARG(top_k >= 1 && top_k <= 32 && top_k <= topk_groups * (e / num_groups),
                "top_k=%d must be in [1, min(32, the open groups' %d experts)]", top_k,
                topk_groups * (e / num_groups));
  DWM_CHECK_ARG(scoring == DWM_SCORE_SOFTMAX || scoring == DWM_SCORE_SIGMOID ||
                    scoring == DWM_SCORE_SQRTSOFTPLUS,
                "unknown scoring function %d", scoring);
  DWM_CHECK_ARG(group_score == DWM_GROUP_MAX || group_score == DWM_GROUP_TOP2,
                "unknown group score %d", group_score);
  DWM_CHECK_ARG(t <= 1 || ld_logits >= e, "ld_logits is shorter than a row");
  DWM_CHECK_ARG(t == 0 || (logits && topk_ids), "NULL pointer");
  if (t == 0) return DWM_OK;
  route_group::Args a;
  a.logits = logits;
  a.ld = ld_logits;
  a.bias = bias;
  a.t = t;
  a.e = e;
  a.top_k = top_k;
  a.groups = num_groups;
  a.keep = topk_groups;
  a.per = e / num_groups;
  a.scoring = scoring;
  a.top2 = group_score == DWM_GROUP_TOP2;
  a.renorm = renormalize != 0;
  a.num_valid = num_valid_tokens;
  a.scale = routed_scale;
  a.ids = topk_ids;
  a.w32 = topk_weights_f32;
  a.w16 = static_cast<uint16_t*>(topk_weights_bf16);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((t + route_group::WARPS - 1) / route_group::WARPS);
  const size_t smem = (size_t)route_group::WARPS * e * sizeof(uint64_t);  // at most 32 KB
  if (logits_dtype == DWM_BF16)
    route_group::route_grouped_kernel<DWM_BF16><<<grid, 32 * route_group::WARPS, smem, s>>>(a);
  else
    route_group::route_grouped_kernel<DWM_F32><<<grid, 32 * route_group::WARPS, smem, s>>>(a);
  return check_cuda(cudaGetLastError(), "route_grouped_topk launch");
}
