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
// A token takes 8, 16 or 32 lanes of a warp: each lane holds a run of at most 64
// experts of one group in registers, so that the scan for the largest is the
// same few instructions for the experts of 4, 2 or 1 tokens. The lanes work in
// f32 and note how far apart the values are where a choice was made: the picks
// among themselves, the last pick and all that is left, the groups at the border.
// Where two are closer than packing and f32 tell apart (a few tokens in a hundred
// for random logits), they are compared value by value, and if that leaves a
// doubt in 64 bits; a token that this does not settle, or one of whose weights
// f32 does not hold, is done again in 64 bits by the whole warp (8-12 us, which
// one token of 1024 would make the time of all). Bound: instruction issue; a
// single token takes 3.4 us of dependent instructions, 32771 tokens of 160
// experts 20.4 us where their bytes take 3.4 (in 64 bits, as f64 logits: 108).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dwm {
namespace route_group {

constexpr int WARPS = 2;

struct Args {
  const void* logits;
  int64_t ld;
  const float* bias;
  int t, e, top_k, groups, keep, per;
  int scoring, top2, renorm, num_valid;
  // 2^lpt_log lanes a token, 2^lg_log lanes a group, run experts a lane; vec:
  // every run starts on 16 bytes and is a whole number of 16-byte loads.
  int lpt_log, lg_log, run, vec;
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
__device__ __forceinline__ auto load_logit(const void* logits, int64_t i) {
  if constexpr (LD == DWM_BF16)
    return bf16_bits_to_f32(static_cast<const uint16_t*>(logits)[i]);
  else if constexpr (LD == DWM_F32)
    return static_cast<const float*>(logits)[i];
  else
    return static_cast<const double*>(logits)[i];
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

struct Pick {
  int id;
  float weight;
};

// Row `tok` in 64 bits: lane j < top_k returns the j-th expert and weight.
// buf: e keys of this warp's shared memory.
template <int LD>
__device__ __noinline__ Pick route_row64(const Args& a, int64_t tok, uint64_t* buf, int lane) {
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
  int id = 0;
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
  return {id, (float)(s * (double)a.scale)};
}

__device__ __forceinline__ void store_pick(const Args& a, int64_t tok, int k, int id,
                                           float weight) {
  const int64_t at = tok * a.top_k + k;
  a.ids[at] = id;
  if (a.w32) a.w32[at] = weight;
  if (a.w16) a.w16[at] = (uint16_t)f32_to_bf16_bits(weight);
}

// Logits of 64 bits, whose order f32 does not hold: every token as above, a warp
// each (32768 x 256 with a bias: 157 us).
__global__ void __launch_bounds__(32 * WARPS) route_grouped64_kernel(const Args a) {
  extern __shared__ uint64_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  overlap_wait();
  overlap_next();
  for (int64_t tok = (int64_t)blockIdx.x * WARPS + warp; tok < a.t;
       tok += (int64_t)gridDim.x * WARPS) {
    Pick p{0, 0.0f};
    if (a.num_valid < 0 || tok < a.num_valid)
      p = route_row64<DWM_F64>(a, tok, smem + warp * a.e, lane);
    if (lane < a.top_k) store_pick(a, tok, lane, p.id, p.weight);
  }
}

// 32-bit keys of numbers (not NaN), ordered as the 64-bit ones.
__device__ __forceinline__ uint32_t key32(float v) {
  const int b = __float_as_int(v + 0.0f);
  return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value32(uint32_t key) {
  return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}

// The f32 score; FULL: for the weights, else for the choices, with the division of
// two steps.
template <bool FULL>
__device__ __forceinline__ float score32(float x, int scoring, float mx, float inv_sum) {
  // (mx is 0 where every logit is -inf.)
  if (scoring == DWM_SCORE_SOFTMAX) return expf(x == mx ? 0.0f : x - mx) * inv_sum;
  if (scoring == DWM_SCORE_SIGMOID)
    return FULL ? 1.0f / (1.0f + expf(-x)) : __fdividef(1.0f, 1.0f + expf(-x));
  return sqrtf(fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
}

// The weight: score32 with the rounding of a softmax's exponent made good (it is as
// many units as the exponent is large).
__device__ __forceinline__ float weight32(float x, int scoring, float mx, float inv_sum) {
  const float s = score32<true>(x, scoring, mx, inv_sum);
  if (scoring != DWM_SCORE_SOFTMAX) return s;
  const float d = x - mx, t = d - x, off = (x - (d - t)) - (mx + t);  // x - mx = d + off
  return fabsf(d) < INFINITY ? fmaf(s, off, s) : s;
}
// Logits (under a softmax, to its maximum) whose scores f32 does not hold to its full
// precision, and 64 bits do.
__device__ __forceinline__ bool faint(float x, int scoring, float mx) {
  const float d = scoring == DWM_SCORE_SOFTMAX ? x - mx : x;
  return d < -80.0f && d > -1500.0f;
}

// How far apart two choices, or two sums of two, have to be for their f32 order to
// be that of 64 bits, in units u = 2^-24 of the token's largest |score| + |bias|.
// A choice is off by
//   sigmoid       10: expf 4 (2 ulp), 1 + e 1, __fdividef 4, the bias 1
//   sqrtsoftplus   7: half of (expf 4, log1pf 4, their sum 1), the root 1, the bias 1
//   softmax        7: expf 4, the exponent |d| e^-|d| < 1, the product 1, the bias 1;
//                     and all of a token's alike, by the sum over the experts, expf 4,
//                     the exponents ln 1024 (their mean size is below that), the
//                     additions in sequence and the reciprocal 1
// So two choices differ by twice the one and the other once (their difference is at
// most the larger), two sums of two by twice that and 4 for the additions. Scores
// below FLOOR are not measured by themselves: of a sqrtsoftplus down there f32 holds
// no more than 4e-23.
constexpr float UNIT = 1.0f / 16777216.0f;
constexpr float FLOOR = 1e-15f;
template <int KPL, int LPT_LOG>
__device__ __forceinline__ float margin_of(int scoring, bool sums) {
  constexpr int ADDS = KPL + LPT_LOG;  // of a lane's and of the lanes'
  constexpr int SOFTMAX = 2 * 7 + 4 + 7 + ADDS + 1, OTHER = 2 * 10;
  // (1 and 2 for the differences and margins themselves.)
  return scoring == DWM_SCORE_SOFTMAX ? (sums ? 2 * SOFTMAX + 6 : SOFTMAX + 1) * UNIT
                                      : (sums ? 2 * OTHER + 6 : OTHER + 1) * UNIT;
}
// Without a bias a sum of two scores is off relative to itself, in the same units by
// 6, of a softmax by 5 and the size of its exponent, which above FLOOR is at most 35;
// of two of them twice that, with room.
constexpr float RELATIVE = 128 * UNIT;

// Within a lane the keys are made unique: their low bits, as many as KPL places
// take, are the place in the run, the lowest place the largest. That takes up
// to 2^bits steps off the value.
template <int KPL>
struct Packed {
  using Set = std::conditional_t<KPL <= 32, uint32_t, uint64_t>;  // of places
  static constexpr uint32_t PLACES = KPL <= 32 ? 31 : 63;
  // The difference of two values that packing may hide, of the larger.
  static constexpr float HIDDEN = (KPL <= 32 ? 2.0f : 4.0f) / 262144.0f;
  static __device__ __forceinline__ float value(uint32_t key) {
    return value32(key >> 31 ? key & ~PLACES : key | PLACES);
  }
};
constexpr int DEEP = 6;  // a lane's largest that are kept sorted

// Sum or maximum over a token's lanes.
template <int LPT>
__device__ __forceinline__ float seg_sum(float v) {
#pragma unroll
  for (int o = LPT / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LPT>
__device__ __forceinline__ uint32_t seg_max(uint32_t v) {
  if (LPT == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
  for (int o = LPT / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LPT>
__device__ __forceinline__ float seg_max(float v) {
#pragma unroll
  for (int o = LPT / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The largest of the keys (below `limit`, if BELOW), descending (0: no more).
template <bool BELOW, int KPL>
__device__ __forceinline__ void largest(const uint32_t (&key)[KPL], uint32_t limit,
                                        uint32_t (&l)[DEEP]) {
#pragma unroll
  for (int j = 0; j < DEEP; ++j) l[j] = 0;
#pragma unroll
  for (int i = 0; i < KPL; ++i) {
    uint32_t k = !BELOW || key[i] < limit ? key[i] : 0u;
#pragma unroll
    for (int j = 0; j < DEEP && j <= i; ++j) {
      const uint32_t t = min(l[j], k);
      l[j] = max(l[j], k);
      k = t;
    }
  }
}

// Element s of an array in registers.
template <class T, int N>
__device__ __forceinline__ T of_slot(const T (&v)[N], int s) {
  T r = v[0];
#pragma unroll
  for (int j = 1; j < N; ++j)
    if (s == j) r = v[j];
  return r;
}

// CTAs an SM whose registers fit at once: many tokens are bound by instruction issue
// and gain from more warps (72 registers for runs of up to 24: 32771 tokens of 160
// experts 20.1 us, with 96 22.3; 96 for longer ones: 32768 of 256 27.4 us, with 128
// 29.9), few tokens by latency alone.
constexpr int resident(int kpl, int lpt_log) { return lpt_log != 3 ? 1 : kpl <= 24 ? 14 : 10; }

// KPL: places in a lane's run; WHOLE: a lane that has experts uses them all (28
// experts in runs of 4 leave one lane of eight without any); 2^LPT_LOG lanes a token.
template <int LD, int KPL, bool WHOLE, int LPT_LOG>
__global__ void __launch_bounds__(32 * WARPS, resident(KPL, LPT_LOG))
    route_grouped_kernel(const Args a) {
  using P = Packed<KPL>;
  constexpr uint32_t PLACES = P::PLACES;
  constexpr int NS = 32 >> LPT_LOG;  // picks a lane holds (top_k is at most 32)
  extern __shared__ uint64_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* buf = smem + warp * a.e;
  constexpr int lpt_log = LPT_LOG, lpt = 1 << lpt_log;
  const int sl = lane & (lpt - 1), seg = lane & ~(lpt - 1);
  const uint32_t seg_mask = (lpt == 32 ? 0xFFFFFFFFu : (1u << lpt) - 1u) << seg;
  const int g = sl >> a.lg_log, part = sl & ((1 << a.lg_log) - 1);
  const bool in_group = g < a.groups;
  // This lane's experts: places [0, count) from expert `first`.
  const int start = part * a.run;
  const int count = in_group ? max(0, min(a.run, a.per - start)) : 0;
  const int first = count > 0 ? g * a.per + start : 0;
  auto has = [&](int i) { return WHOLE ? true : i < count; };
  const bool biased = a.bias != nullptr;
  const int tpw = 32 >> lpt_log;  // tokens a warp
  const int64_t stride = (int64_t)gridDim.x * WARPS * tpw;
  overlap_wait();
  overlap_next();
  for (int64_t base = ((int64_t)blockIdx.x * WARPS + warp) * tpw; base < a.t; base += stride) {
    const int64_t tok = base + (lane >> lpt_log);
    const bool live = tok < a.t;
    const bool real = live && (a.num_valid < 0 || tok < a.num_valid);
    const int64_t row = (live ? tok : base) * a.ld;

    float v[KPL];
    if (a.vec) {
      // (count is a.run or 0, a multiple of a 16-byte load.)
      constexpr int PER = LD == DWM_BF16 ? 8 : 4;
#pragma unroll
      for (int i = 0; i < KPL; i += PER) {
        const int64_t at = row + first + (has(i) ? i : 0);
        if constexpr (LD == DWM_BF16) {
          const uint4 q = *reinterpret_cast<const uint4*>(
              static_cast<const uint16_t*>(a.logits) + at);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (i + j < KPL)
              v[i + j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        } else {
          const float4 q =
              *reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + at);
          const float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (i + j < KPL) v[i + j] = w[j];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < KPL; ++i)
        v[i] = load_logit<LD>(a.logits, row + first + (has(i) ? i : 0));
    }

    bool nan = false;
    float mx = 0.0f, inv_sum = 1.0f;
    if (a.scoring == DWM_SCORE_SOFTMAX) {
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < KPL; ++i) mx = fmaxf(mx, v[i]);  // (an absent one repeats the first)
      mx = seg_max<lpt>(count > 0 ? mx : -INFINITY);
      if (mx == -INFINITY) mx = 0.0f;
      if (biased || !a.renorm) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
          const float s = score32<true>(v[i], DWM_SCORE_SOFTMAX, mx, 1.0f);
          if (has(i)) sum += s;
        }
        sum = seg_sum<lpt>(count > 0 ? sum : 0.0f);
        inv_sum = sum > 0.0f ? 1.0f / sum : 1.0f;
      }
    }
    float size = FLOOR;  // the largest |score| + |bias|
    auto margin = [&](bool sums) { return margin_of<KPL, LPT_LOG>(a.scoring, sums) * size; };
    if (biased) {
      auto choices = [&](int scoring) {
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
          const float s = score32<false>(v[i], scoring, mx, inv_sum);
          const float b = a.bias[first + (has(i) ? i : 0)];
          size = fmaxf(size, fabsf(s) + (fabsf(b) < INFINITY ? fabsf(b) : 0.0f));
          v[i] = s + b;
        }
      };
      if (a.scoring == DWM_SCORE_SOFTMAX)
        choices(DWM_SCORE_SOFTMAX);
      else if (a.scoring == DWM_SCORE_SIGMOID)
        choices(DWM_SCORE_SIGMOID);
      else
        choices(DWM_SCORE_SQRTSOFTPLUS);
      size = seg_max<lpt>(size);
    }
    // A lane's two largest, exact; its keys.
    uint32_t key[KPL], m1 = 0, m2 = 0;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
      nan |= isnan(v[i]);
      const uint32_t k = has(i) ? key32(v[i]) : 0u;
      m2 = max(m2, min(m1, k));
      m1 = max(m1, k);
      key[i] = has(i) ? (k & ~PLACES) | (PLACES - (uint32_t)i) : 0u;
    }
    bool unsure = nan;  // not decided in f32
    uint32_t l[DEEP];
    largest<false>(key, 0u, l);
    if (count == 0) m1 = m2 = 0;
    auto expert = [&](uint32_t k) { return first + (int)(PLACES - (k & PLACES)); };

    // bf16 logits without a bias fit the keys whole; otherwise the values are
    // formed again where the keys are too coarse.
    const bool exact = LD == DWM_BF16 && !biased;
    auto choice = [&](int e) {
      const float x = load_logit<LD>(a.logits, row + e);
      return biased ? score32<false>(x, a.scoring, mx, inv_sum) + a.bias[e] : x;
    };
    auto choice64 = [&](int e) {
      const double x = load_logit<LD>(a.logits, row + e);
      return biased ? score(x, a.scoring, 0.0, 1.0) + (double)a.bias[e] : x;
    };
    // What the values of a lane's packed keys up to k are below, in 64 bits.
    auto bound = [&](uint32_t k) {
      const double x = P::value(k & ~PLACES);
      return x + (biased ? (double)margin(false) + (double)P::HIDDEN * size
                         : (double)P::HIDDEN * fabs(x));
    };
    for (int o = (1 << a.lg_log) / 2; o; o >>= 1) {
      const uint32_t n1 = __shfl_xor_sync(0xffffffffu, m1, o),
                     n2 = __shfl_xor_sync(0xffffffffu, m2, o);
      m2 = max(min(m1, n1), max(m2, n2));
      m1 = max(m1, n1);
    }
    uint32_t gkey = m1;
    if (a.top2 && m2) {
      float p = value32(m1), q = value32(m2);
      if (!biased) {
        p = score32<true>(p, a.scoring, mx, 1.0f);
        q = score32<true>(q, a.scoring, mx, 1.0f);
      }
      gkey = key32(p + q);
      unsure |= isnan(p + q);
    }
    int rank = 0;
    for (int q = 0; q < a.groups; ++q) {
      const uint32_t k = __shfl_sync(0xffffffffu, gkey, seg + (q << a.lg_log));
      rank += k > gkey || (k == gkey && q < g);
    }
    bool open = in_group && rank < a.keep;
    // In 64 bits a softmax's sum takes every expert; without a bias the order
    // does not need it.
    const bool settles = !(biased && a.scoring == DWM_SCORE_SOFTMAX);
    if (a.keep < a.groups && (biased || a.top2)) {
      const float in = value32(~seg_max<lpt>(open ? ~gkey : 0u));  // the least of the open
      const float out = value32(seg_max<lpt>(in_group && !open ? gkey : 0u));
      const bool close = biased ? !(in - out > margin(a.top2))
                                : !(in > FLOOR && in - out > RELATIVE * in);
      if (__any_sync(0xffffffffu, close && real)) {
        // The groups' values in 64 bits, from each lane's first four.
        double c[4], d1 = -INFINITY, d2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j] = count > 0 && l[j] ? choice64(expert(l[j])) : -INFINITY;
          d2 = fmax(d2, fmin(d1, c[j]));
          d1 = fmax(d1, c[j]);
        }
        // A fifth that may be one of the two largest: not settled.
        bool sure = settles && (count == 0 || !l[4] || (a.top2 ? d2 : d1) > bound(l[4]));
        for (int o = (1 << a.lg_log) / 2; o; o >>= 1) {
          const double n1 = __shfl_xor_sync(0xffffffffu, d1, o),
                       n2 = __shfl_xor_sync(0xffffffffu, d2, o);
          d2 = fmax(fmin(d1, n1), fmax(d2, n2));
          d1 = fmax(d1, n1);
        }
        double gv = d1;
        if (a.top2 && a.per > 1)
          gv = biased ? d1 + d2
                      : score(d1, a.scoring, (double)mx, 1.0) + score(d2, a.scoring, (double)mx, 1.0);
        rank = 0;
        for (int q = 0; q < a.groups; ++q) {
          const double k = __shfl_sync(0xffffffffu, gv, seg + (q << a.lg_log));
          rank += k > gv || (k == gv && q < g);
        }
        if (close) {
          open = in_group && rank < a.keep;
          unsure |= !sure;
        }
      }
    }

    // The top k, the largest of the lanes' largest each time.
    if (!open || count == 0) l[0] = 0;
    int left = open ? count : 0;  // in l or below it
    typename P::Set gone = 0;     // the places that are picked
    const int n_open = a.keep * a.per;
    uint32_t top = 0;  // the last pick's packed value
    int last_id = 0, slot_id[NS] = {};
    auto pick = [&](int k) {
      top = seg_max<lpt>(l[0] & ~PLACES);
      // Of equal ones the lowest lane's, whose experts come first.
      const uint32_t who = __ballot_sync(0xffffffffu, (l[0] & ~PLACES) == top) & seg_mask;
      const int winner = __ffs(who) - 1;
      last_id = __shfl_sync(0xffffffffu, expert(l[0]), winner);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (k == s * lpt + sl) slot_id[s] = last_id;
      uint32_t taken = 0;
      if (lane == winner) {
        taken = l[0];
        gone |= (typename P::Set)1 << (PLACES - (taken & PLACES));
#pragma unroll
        for (int j = 0; j + 1 < DEEP; ++j) l[j] = l[j + 1];
        l[DEEP - 1] = 0;
        --left;
      }
      // More than DEEP of one lane: the next ones from its keys.
      const bool empty = taken && !l[0] && left > 0;
      if (__any_sync(0xffffffffu, empty)) {
        if (empty) largest<true>(key, taken, l);
      }
    };
    // Packed values x <= last whose order packing or f32 may hide.
    auto near = [&](float last, float x) {
      return !(last - x > (biased ? margin(false) + P::HIDDEN * size
                                  : P::HIDDEN * fmaxf(fabsf(x), fabsf(last))));
    };
    // Whether the choice of expert e certainly comes before that of f, which has
    // the higher index if they tie.
    auto ahead = [&](int e, int f) {
      const float p = choice(e), q = choice(f);
      if (biased ? p - q > margin(false) : p > q) return true;
      // Equal logits and biases are a tie in 64 bits too.
      return load_logit<LD>(a.logits, row + e) == load_logit<LD>(a.logits, row + f) &&
             (!biased || a.bias[e] == a.bias[f]);
    };
    bool close = false;
    float last = 0.0f;
    int picks = a.top_k, k = 0;
    uint32_t rest = 0;  // the largest packed value that is left
    bool settling = false;
    while (true) {
      for (; k < picks; ++k) {
        const int before = last_id;
        pick(k);
        if (!exact) {
          const float x = P::value(top);
          if (k > 0 && near(last, x)) close |= k < a.top_k && !ahead(before, last_id);
          last = x;
        }
      }
      if (exact) break;
      rest = picks < n_open ? seg_max<lpt>(l[0] & ~PLACES) : 0u;
      if (settling) break;
      // What is left comes after the last pick: its largest packed value clearly, or
      // each expert by itself (of one packed value the largest need not be the first).
      const bool cut = rest && near(last, P::value(rest));
      if (__any_sync(0xffffffffu, cut && real)) {
        bool sure = true;
        if (cut && l[0] && near(last, P::value(l[0]))) {
          sure = ahead(last_id, expert(l[0]));
          // (What is near and not in the list comes after what is.)
          if (sure && left > 1 && (!l[1] || near(last, P::value(l[1]))))
            for (int i = 0; i < count; ++i)
              if (!(gone >> i & 1)) sure = sure && ahead(last_id, first + i);
        }
        close |= (__ballot_sync(0xffffffffu, !sure) & seg_mask) != 0;
      }
      settling = __any_sync(0xffffffffu, close && real);
      if (!settling) break;
      picks = min(min(a.top_k + 4, n_open), NS * lpt);
    }
    if (settling) {
      // Up to four picks more, then all of them in the order of their 64-bit
      // values; what was not picked has to be below the last that is chosen.
      const int all = picks;
      double c[NS];
      int place[NS] = {}, id[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) c[s] = s * lpt + sl < all ? choice64(slot_id[s]) : 0.0;
      double least = 0.0;  // the value at the place top_k - 1
      for (int k = 0; k < all; ++k) {
        const int of = seg + (k & (lpt - 1)), s = k >> lpt_log;
        const double v = __shfl_sync(0xffffffffu, of_slot(c, s), of);
        const int e = __shfl_sync(0xffffffffu, of_slot(slot_id, s), of);
#pragma unroll
        for (int j = 0; j < NS; ++j) place[j] += v > c[j] || (v == c[j] && e < slot_id[j]);
      }
#pragma unroll
      for (int j = 0; j < NS; ++j) id[j] = slot_id[j];
      for (int k = 0; k < all; ++k) {
        const int of = seg + (k & (lpt - 1)), s = k >> lpt_log;
        const int to = __shfl_sync(0xffffffffu, of_slot(place, s), of);
        const int e = __shfl_sync(0xffffffffu, of_slot(slot_id, s), of);
        const double v = __shfl_sync(0xffffffffu, of_slot(c, s), of);
        if (to == a.top_k - 1) least = v;
#pragma unroll
        for (int j = 0; j < NS; ++j)
          if (to == j * lpt + sl) id[j] = e;
      }
      if (close) {
        unsure |= !settles || (rest && !(least > bound(rest)));
#pragma unroll
        for (int j = 0; j < NS; ++j) slot_id[j] = id[j];
      }
    }

    // Weights: slot s of lane sl is the pick s * lpt + sl.
    float w[NS], total = 0.0f;
    bool weak = false;  // a weight that takes 64 bits
    auto weights = [&](int scoring) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        w[s] = 0.0f;
        if (s * lpt + sl < a.top_k) {
          const float x = load_logit<LD>(a.logits, row + slot_id[s]);
          w[s] = weight32(x, scoring, mx, inv_sum);
          weak |= faint(x, scoring, mx);
        }
        total += w[s];
      }
    };
    if (a.scoring == DWM_SCORE_SOFTMAX)
      weights(DWM_SCORE_SOFTMAX);
    else if (a.scoring == DWM_SCORE_SIGMOID)
      weights(DWM_SCORE_SIGMOID);
    else
      weights(DWM_SCORE_SQRTSOFTPLUS);
    if (a.renorm) total = seg_sum<lpt>(total);
    // What one lane of a token is unsure of, all are.
    const uint32_t doubts = __ballot_sync(0xffffffffu, ((unsure && in_group) || weak) && real);
    if (live && !(doubts & seg_mask)) {
      const float scale = !a.renorm ? a.scale : total == 0.0f ? 0.0f : a.scale;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int k = s * lpt + sl;
        if (k < a.top_k) {
          const float x = (a.renorm && total != 0.0f ? w[s] / total : w[s]) * scale;
          store_pick(a, tok, k, real ? slot_id[s] : 0, real ? x : 0.0f);
        }
      }
    }
    for (uint32_t again = doubts; again;) {
      const int of = (__ffs(again) - 1) >> lpt_log;
      again &= ~((lpt == 32 ? 0xFFFFFFFFu : (1u << lpt) - 1u) << (of << lpt_log));
      const Pick p = route_row64<LD>(a, base + of, buf, lane);
      if (lane < a.top_k) store_pick(a, base + of, lane, p.id, p.weight);
      __syncwarp();
    }
  }
}

int launch64(const Args& a, cudaStream_t s) {
  const unsigned grid =
      (unsigned)std::min<int64_t>(((int64_t)a.t + WARPS - 1) / WARPS, (int64_t)num_sms() * 64);
  return check_cuda(overlap_launch(route_grouped64_kernel, dim3(grid), dim3(32 * WARPS),
                                   (size_t)WARPS * a.e * sizeof(uint64_t), 1, s, a),
                    "route_grouped_topk launch");
}

template <int LD, int KPL, int LPT_LOG>
int launch(const Args& a, cudaStream_t s) {
  const int64_t tokens = (int64_t)WARPS * (32 >> LPT_LOG);  // a CTA's
  const unsigned grid =
      (unsigned)std::min<int64_t>((a.t + tokens - 1) / tokens, (int64_t)num_sms() * 64);
  const size_t smem = (size_t)WARPS * a.e * sizeof(uint64_t);  // at most 32 KB
  auto fn = a.run == KPL && a.per % a.run == 0 ? route_grouped_kernel<LD, KPL, true, LPT_LOG>
                                               : route_grouped_kernel<LD, KPL, false, LPT_LOG>;
  return check_cuda(overlap_launch(fn, dim3(grid), dim3(32 * WARPS), smem, 1, s, a),
                    "route_grouped_topk launch");
}

// Places for a lane's run: the next multiple of 4. Places that stay empty cost as much
// as the others: 32768 tokens of 160 experts in 8 groups with a bias take 25.0 us in
// 20 places, 29.7 in 24 and 34.7 in 32; of 96 experts 20.0 in 12 and 23.9 in 16.
template <int LD, int LPT_LOG>
int by_run(const Args& a, cudaStream_t s) {
  if (a.run <= 4) return launch<LD, 4, LPT_LOG>(a, s);
  if (a.run <= 8) return launch<LD, 8, LPT_LOG>(a, s);
  if (a.run <= 12) return launch<LD, 12, LPT_LOG>(a, s);
  if (a.run <= 16) return launch<LD, 16, LPT_LOG>(a, s);
  if (a.run <= 20) return launch<LD, 20, LPT_LOG>(a, s);
  if (a.run <= 24) return launch<LD, 24, LPT_LOG>(a, s);
  if (a.run <= 28) return launch<LD, 28, LPT_LOG>(a, s);
  if (a.run <= 32) return launch<LD, 32, LPT_LOG>(a, s);
  if constexpr (LPT_LOG == 5) return launch<LD, 64, LPT_LOG>(a, s);
  return set_error(DWM_ERR_UNSUPPORTED, "run=%d", a.run);  // (more lanes have fewer)
}

template <int LD>
int run(const Args& a, cudaStream_t s) {
  return a.lpt_log == 3   ? by_run<LD, 3>(a, s)
         : a.lpt_log == 4 ? by_run<LD, 4>(a, s)
                          : by_run<LD, 5>(a, s);
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
  DWM_CHECK_ARG(logits_dtype == DWM_BF16 || logits_dtype == DWM_F32 || logits_dtype == DWM_F64,
                "logits dtype must be bf16, f32 or f64");
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
  const int es = logits_dtype == DWM_F64 ? 8 : logits_dtype == DWM_F32 ? 4 : 2;
  auto misaligned = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size; };
  DWM_CHECK_ARG(!misaligned(logits, es) && !misaligned(bias, 4) && !misaligned(topk_ids, 4) &&
                    !misaligned(topk_weights_f32, 4) && !misaligned(topk_weights_bf16, 2),
                "misaligned pointer");
  // Tokens are written while others are read.
  const int64_t picks = (int64_t)t * top_k;
  const RowSpan outs[3] = {row_span(topk_ids, 1, picks, picks, 4),
                           row_span(topk_weights_f32, 1, picks, picks, 4),
                           row_span(topk_weights_bf16, 1, picks, picks, 2)};
  for (int i = 0; i < 3; ++i)
    DWM_CHECK_ARG(!rows_overlap(outs[i], row_span(logits, t, e, ld_logits, es)) &&
                      !rows_overlap(outs[i], row_span(bias, 1, e, e, 4)) &&
                      !rows_overlap(outs[i], outs[(i + 1) % 3]),
                  "an output overlaps an input or another output");
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
  if (logits_dtype == DWM_F64) return route_group::launch64(a, s);
  // Lanes: a power of two of groups, each of as many lanes as leave at most 32
  // experts a lane (64 where the warp has no more lanes); 8 a token at least, and
  // up to twelve tokens an SM the whole warp, for its shorter runs and its one
  // instruction for a maximum (256 experts: one token 3.4 us against 4.9 with 8
  // lanes, 1776 tokens 5.5 and 6.9, 2500 tokens 7.9 and 7.4, 32768 tokens 51.7 and
  // 25.6; of 160 experts 49.9 and 18.8).
  const int lanes_log = t <= 12 * (int64_t)num_sms() ? 5 : 3;
  int groups_log = 0;
  while ((1 << groups_log) < num_groups) ++groups_log;
  a.lg_log = 0;
  while (groups_log + a.lg_log < 5 &&
         ((a.per + (1 << a.lg_log) - 1) >> a.lg_log > 32 || groups_log + a.lg_log < lanes_log))
    ++a.lg_log;
  a.lpt_log = groups_log + a.lg_log;
  a.run = (a.per + (1 << a.lg_log) - 1) >> a.lg_log;
  a.vec = a.per % a.run == 0 && a.run * es % 16 == 0 && (t == 1 || ld_logits * es % 16 == 0) &&
          (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  return logits_dtype == DWM_BF16 ? route_group::run<DWM_BF16>(a, s)
                                  : route_group::run<DWM_F32>(a, s);
}
