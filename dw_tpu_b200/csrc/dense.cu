// Dense product with its epilogue: out = residual_scale * residual +
// act(x w^T + bias), bf16 operands, f32 accumulation, rounded once. The
// products around the expert layer that are not FP4: the router's logits, the
// shared expert's projections.
//
// Split kernel. The product is computed transposed: 128 rows of w are UMMA
// operand A, up to 128 rows of x are operand B, so a decode batch pays for its
// own tokens (N = 16 and up) and not for 128. The k axis is split over a
// cluster of 1, 2, 4 or 8 CTAs, which fills the GPU when w has few rows. Each
// CTA puts its f32 partial tile in its shared memory; the cluster's CTAs then
// share the tile's outputs out among them, and each adds the partials of its
// share in CTA order (over distributed shared memory), so the result depends
// on the shapes alone: no atomics, no workspace.
//
// With SwiGLU a tile is 64 gate rows and the 64 up rows of the same features,
// which meet in the partial tile.
//
// Bound: at decode the stream of w (two CTAs per SM keep ~190 KB of copies in
// flight), for small shapes the launch and one memory latency, from ~100 rows
// of x the tensor cores.
#include <algorithm>

#include "common.cuh"

namespace dwm {
namespace dense {

constexpr int BK = 64;          // k per stage: one 128-byte swizzled row
constexpr int TILE_W = 128;     // rows of w per tile
constexpr int THREADS = 256;
constexpr int A_STAGE = TILE_W * BK * 2;  // 16 KiB
constexpr int MAX_CLUSTER = 8;

struct Args {
  const void* bias;      // [n] or NULL
  const void* residual;  // [m, n_out] or NULL
  void* out;             // [m, n_out]
  int64_t ldr, ldo;
  int m, n_out, k;
  int act;
  int bias_f32, res_f32, out_f32;
  int res_vec, out_vec;  // 8 elements at a column that is a multiple of 8 are 16-byte aligned
  float limit, res_scale;
  int* status;
};

template <int BT>
struct Layout {
  static constexpr int B_STAGE = BT * BK * 2;
  static constexpr int STG = A_STAGE + B_STAGE;
  static constexpr int S = 98304 / STG;  // two CTAs per SM
  static constexpr int PARTIAL = BT * TILE_W * 4;  // f32 [BT][TILE_W] over the stages
  static constexpr int OFF_BAR = S * STG > PARTIAL ? S * STG : PARTIAL;
  static constexpr int OFF_MISC = OFF_BAR + (2 * S + 1) * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;  // slack for 1 KiB alignment
  static constexpr int TMEM_COLS = BT < 32 ? 32 : BT;
  static_assert(STG % 1024 == 0, "swizzled tiles need 1 KiB alignment");
  static_assert(S >= 2 && 2 * (ALLOC + 1024) <= 233472, "two CTAs per SM");
};

__device__ __forceinline__ float ld1(const void* p, int64_t i, int f32) {
  return f32 ? static_cast<const float*>(p)[i]
             : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

__device__ __forceinline__ float sigmoid_full(float v) { return 1.0f / (1.0f + expf(-v)); }

// The activation of one value. An f32 output takes full-precision functions,
// a bf16 one (half a step: 2^-9 of the value) the MUFU forms (~1e-6).
__device__ __forceinline__ float act1(float v, int act, int f32) {
  if (act == DWM_ACT_SILU) return v * (f32 ? sigmoid_full(v) : sigmoid_fast(v));
  if (act == DWM_ACT_GELU) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
  if (act == DWM_ACT_GELU_TANH) {
    // 0.5 (1 + tanh(u)) = sigmoid(2 u)
    const float u = 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
    return v * (f32 ? sigmoid_full(u) : sigmoid_fast(u));
  }
  return v;
}

// Outputs [col, col + 8) of row `row` from the products z (and, with SwiGLU,
// the up products u): bias, activation, residual, one rounding.
__device__ __forceinline__ void epilogue8(const Args& a, int64_t row, int col, float (&z)[8],
                                          const float (&u)[8]) {
  const bool glu = a.act == DWM_ACT_SWIGLU || a.act == DWM_ACT_SWIGLU_CLAMP;
  const bool whole = col + 8 <= a.n_out;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    float v = z[q], up = u[q];
    if (a.bias && (whole || col + q < a.n_out)) {
      v += ld1(a.bias, col + q, a.bias_f32);
      if (glu) up += ld1(a.bias, a.n_out + col + q, a.bias_f32);
    }
    if (glu) {
      if (a.act == DWM_ACT_SWIGLU_CLAMP) {
        v = fminf(v, a.limit);
        up = fminf(fmaxf(up, -a.limit), a.limit);
      }
      v = v * (a.out_f32 ? sigmoid_full(v) : sigmoid_fast(v)) * up;
    } else {
      v = act1(v, a.act, a.out_f32);
    }
    z[q] = v;
  }
  if (a.residual) {
    const int64_t at = row * a.ldr + col;
    if (whole && a.res_vec) {
      float r[8];
      if (a.res_f32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + at);
        const float4 x = p[0], y = p[1];
        r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
        r[4] = y.x; r[5] = y.y; r[6] = y.z; r[7] = y.w;
      } else {
        const uint4 x =
            *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.residual) + at);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          r[2 * q] = __uint_as_float(w[q] << 16);
          r[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = fmaf(a.res_scale, r[q], z[q]);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (col + q < a.n_out) z[q] = fmaf(a.res_scale, ld1(a.residual, at + q, a.res_f32), z[q]);
    }
  }
  const int64_t at = row * a.ldo + col;
  if (whole && a.out_vec) {
    if (a.out_f32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
      p[0] = make_float4(z[0], z[1], z[2], z[3]);
      p[1] = make_float4(z[4], z[5], z[6], z[7]);
    } else {
      uint4 o;
      o.x = f32_to_bf16_bits(z[0]) | (f32_to_bf16_bits(z[1]) << 16);
      o.y = f32_to_bf16_bits(z[2]) | (f32_to_bf16_bits(z[3]) << 16);
      o.z = f32_to_bf16_bits(z[4]) | (f32_to_bf16_bits(z[5]) << 16);
      o.w = f32_to_bf16_bits(z[6]) | (f32_to_bf16_bits(z[7]) << 16);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) = o;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (col + q < a.n_out) {
        if (a.out_f32)
          static_cast<float*>(a.out)[at + q] = z[q];
        else
          static_cast<uint16_t*>(a.out)[at + q] = (uint16_t)f32_to_bf16_bits(z[q]);
      }
  }
}

// 4 floats of another CTA's shared memory, by its shared::cluster address.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// grid (cluster, w tiles, x tiles); GLU: the tile's 128 rows of w are 64 gate
// rows and the up rows of the same features.
template <int BT, bool GLU>
__global__ void __launch_bounds__(THREADS, 2)
    dense_split_kernel(const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_x, const Args a) {
  using L = Layout<BT>;
  constexpr int S = L::S;
  constexpr int FEAT = GLU ? TILE_W / 2 : TILE_W;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = gridDim.x;
  const int rank = blockIdx.x;  // the cluster spans the grid's x axis
  const int col0 = blockIdx.y * FEAT;
  const int row0 = blockIdx.z * BT;
  const int kt = (a.k + BK - 1) / BK;
  const int k_lo = (int)((int64_t)kt * rank / split), k_hi = (int)((int64_t)kt * (rank + 1) / split);
  const int steps = k_hi - k_lo;  // at least one

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // w is read once where one tile holds all rows of x, else once a tile.
      const uint64_t pol_w = gridDim.z == 1 ? policy_evict_first() : policy_evict_last();
      const uint64_t pol_x = policy_evict_last();
      int i = 0;
      for (; i < steps; ++i) {
        const int st = i % S;
        if (!mbar_wait(&empty[st], ((i / S) & 1) ^ 1, abort_flag, a.status)) break;
        mbar_arrive_expect_tx(&full[st], L::STG);
        uint8_t* dst = smem + st * L::STG;
        const int x = (k_lo + i) * BK;
        if (GLU) {
          tma_load_2d(dst, &tm_w, &full[st], x, col0, pol_w);
          tma_load_2d(dst + A_STAGE / 2, &tm_w, &full[st], x, a.n_out + col0, pol_w);
        } else {
          tma_load_2d(dst, &tm_w, &full[st], x, col0, pol_w);
        }
        tma_load_2d(dst + A_STAGE, &tm_x, &full[st], x, row0, pol_x);
      }
      // Every copy has landed before the stages are written over, also after a
      // wait that ran out.
      for (int j = max(0, i - S); j < i; ++j)
        mbar_wait(&full[j % S], (j / S) & 1, nullptr, a.status);
    }
  } else if (warp == 1) {
    const bool issuer = elect_one();
    constexpr uint32_t idesc = idesc_bf16(TILE_W, BT, false, false);
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const int st = i % S;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (i / S) & 1, abort_flag, a.status));
      if (!ok) break;
      tc_fence_after();
      if (issuer) {
        const uint32_t base = smem_u32(smem + st * L::STG);
#pragma unroll
        for (int j = 0; j < BK / 16; ++j)
          umma_bf16(tmem, smem_desc_sw128(base + j * 32, 16, 1024),
                    smem_desc_sw128(base + A_STAGE + j * 32, 16, 1024), idesc, (i | j) != 0);
        umma_commit(&empty[st]);
      }
      __syncwarp();
    }
    if (issuer) umma_commit(done);
    __syncwarp();
  }
  // Every UMMA complete (so every copy has landed and been read): the stages
  // become the partial tile.
  __syncwarp();
  bool ok = mbar_wait(done, 0, nullptr, a.status);
  ok = __syncthreads_and(ok) != 0 && *abort_flag == 0;
  tc_fence_after();
  float* part = reinterpret_cast<float*>(smem);
  {
    // Warp w reads TMEM lanes (rows of w) 32 (w % 4) .. and one half of the
    // columns (rows of x).
    const int q = warp & 3, half = warp >> 2;
    constexpr int COLS = BT / 2 < 16 ? 16 : BT / 2;
    if (half * COLS < BT) {
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + half * COLS + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          part[(half * COLS + c + e) * TILE_W + q * 32 + lane] = __uint_as_float(r[e]);
      }
    }
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, L::TMEM_COLS);

  // This CTA's share of the tile's outputs, 8 columns a thread.
  if (ok) {
    constexpr int CH = FEAT / 8;
    const int rows = min(BT, a.m - row0);
    const int items = rows * CH;
    const int lo = (int)((int64_t)items * rank / split), hi = (int)((int64_t)items * (rank + 1) / split);
    const uint32_t base = smem_u32(part);
    for (int i = lo + (int)threadIdx.x; i < hi; i += THREADS) {
      const int t = i / CH, c = (i % CH) * 8;
      if (col0 + c >= a.n_out) continue;
      float z[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = u[e] = 0.0f;
      const uint32_t off = base + (uint32_t)((t * TILE_W + c) * 4);
      for (int p = 0; p < split; ++p) {
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(off), "r"(p));
        const float4 x = ld_cluster_f4(at), y = ld_cluster_f4(at + 16);
        z[0] += x.x; z[1] += x.y; z[2] += x.z; z[3] += x.w;
        z[4] += y.x; z[5] += y.y; z[6] += y.z; z[7] += y.w;
        if (GLU) {
          const float4 v = ld_cluster_f4(at + FEAT * 4), w = ld_cluster_f4(at + FEAT * 4 + 16);
          u[0] += v.x; u[1] += v.y; u[2] += v.z; u[3] += v.w;
          u[4] += w.x; u[5] += w.y; u[6] += w.z; u[7] += w.w;
        }
      }
      epilogue8(a, row0 + t, col0 + c, z, u);
    }
  }
  __syncwarp();
  if (split > 1) cluster_sync();  // no CTA exits while another reads its tile
}

template <int BT, bool GLU>
int launch_split(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, int split,
                 const Args& a, cudaStream_t stream) {
  using L = Layout<BT>;
  constexpr int FEAT = GLU ? TILE_W / 2 : TILE_W;
  DWM_CHECK_ARG((a.m + (int64_t)BT - 1) / BT <= 65535 && (a.n_out + (int64_t)FEAT - 1) / FEAT <= 65535,
                "m=%d rows by %d columns exceed the grid", a.m, a.n_out);
  CUtensorMap tm_w, tm_x;
  int rc = encode_tmap_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, w, (uint64_t)a.k, (uint64_t)n,
                          (uint64_t)ldw * 2, BK, FEAT, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = encode_tmap_2d(&tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, (uint64_t)a.k, (uint64_t)a.m,
                      (uint64_t)ldx * 2, BK, BT, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = set_smem_limit(reinterpret_cast<const void*>(dense_split_kernel<BT, GLU>), L::ALLOC,
                      "dense smem attribute");
  if (rc) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)split, (unsigned)((a.n_out + FEAT - 1) / FEAT),
                     (unsigned)((a.m + BT - 1) / BT));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = L::ALLOC;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, dense_split_kernel<BT, GLU>, tm_w, tm_x, a),
                    "dense_matmul launch");
}

int run(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, const Args& a,
        cudaStream_t stream) {
  const bool glu = a.act == DWM_ACT_SWIGLU || a.act == DWM_ACT_SWIGLU_CLAMP;
  const int bt = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
  const int feat = glu ? TILE_W / 2 : TILE_W;
  const int64_t tiles = (int64_t)((a.n_out + feat - 1) / feat) * ((a.m + bt - 1) / bt);
  const int kt = (a.k + BK - 1) / BK;
  // Two CTAs per SM; at least two k steps a CTA.
  int split = 1;
  while (split < MAX_CLUSTER && tiles * split * 2 <= 2 * num_sms() && kt >= 4 * split) split *= 2;
#define DWM_DENSE_SPLIT(BT)                                                     \
  return glu ? launch_split<BT, true>(x, ldx, w, ldw, n, split, a, stream)      \
             : launch_split<BT, false>(x, ldx, w, ldw, n, split, a, stream)
  if (bt == 16) DWM_DENSE_SPLIT(16);
  if (bt == 32) DWM_DENSE_SPLIT(32);
  if (bt == 64) DWM_DENSE_SPLIT(64);
  DWM_DENSE_SPLIT(128);
#undef DWM_DENSE_SPLIT
}

}  // namespace dense
}  // namespace dwm

using namespace dwm;

extern "C" int dwm_dense_matmul(const void* x, int64_t ldx, const void* w, int64_t ldw, int m,
                                int n, int k, const void* bias, int bias_dtype, int act,
                                float act_limit, const void* residual, int residual_dtype,
                                int64_t ldr, float residual_scale, void* out, int out_dtype,
                                int64_t ldo, void* stream) {
  auto is_float = [](int d) { return d == DWM_BF16 || d == DWM_F32; };
  auto addr = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool glu = act == DWM_ACT_SWIGLU || act == DWM_ACT_SWIGLU_CLAMP;
  DWM_CHECK_ARG(m >= 0 && n >= 1 && k >= 8, "bad shape m=%d n=%d k=%d", m, n, k);
  DWM_CHECK_ARG(k % 8 == 0, "k=%d must be a multiple of 8", k);
  DWM_CHECK_ARG(act >= DWM_ACT_NONE && act <= DWM_ACT_GELU_TANH, "unknown activation %d", act);
  DWM_CHECK_ARG(!glu || n % 2 == 0, "SwiGLU needs [gate | up] halves: n=%d is odd", n);
  DWM_CHECK_ARG(act != DWM_ACT_SWIGLU_CLAMP || act_limit > 0.0f, "act_limit must be positive");
  DWM_CHECK_ARG(is_float(out_dtype) && (!bias || is_float(bias_dtype)) &&
                    (!residual || is_float(residual_dtype)),
                "out, bias and residual must be bf16 or f32");
  const int n_out = glu ? n / 2 : n;
  // One row: its stride is free, and not looked at.
  if (m <= 1) { ldx = k; ldr = n_out; ldo = n_out; }
  if (n == 1) ldw = k;
  DWM_CHECK_ARG(ldx >= k && ldw >= k && ldo >= n_out && (!residual || ldr >= n_out),
                "a row stride is shorter than a row");
  DWM_CHECK_ARG(ldx % 8 == 0 && ldw % 8 == 0, "rows of x and w must start on 16 bytes "
                "(strides %lld, %lld must be multiples of 8)", (long long)ldx, (long long)ldw);
  DWM_CHECK_ARG(ldx < (1ll << 38) && ldw < (1ll << 38), "a row stride is too long");
  if (m == 0) return DWM_OK;
  DWM_CHECK_ARG(x && w && out, "NULL pointer");
  DWM_CHECK_ARG(addr(x) % 16 == 0 && addr(w) % 16 == 0, "x and w must be 16-byte aligned");
  const int oes = out_dtype == DWM_F32 ? 4 : 2, res = residual_dtype == DWM_F32 ? 4 : 2;
  const int bes = bias_dtype == DWM_F32 ? 4 : 2;
  DWM_CHECK_ARG(addr(out) % oes == 0 && (!residual || addr(residual) % res == 0) &&
                    (!bias || addr(bias) % bes == 0),
                "misaligned pointer");
  // The output may be the residual itself; any other overlap would be read
  // after it is written.
  const RowSpan o = row_span(out, m, n_out, ldo, oes);
  DWM_CHECK_ARG(!rows_overlap(o, row_span(x, m, k, ldx, 2)) &&
                    !rows_overlap(o, row_span(w, n, k, ldw, 2)) &&
                    !rows_overlap(o, row_span(bias, 1, n, n, bes)),
                "out overlaps an input");
  DWM_CHECK_ARG((residual == out && ldr == ldo && res == oes) ||
                    !rows_overlap(o, row_span(residual, m, n_out, ldr, res)),
                "out overlaps the residual without being it");
  dense::Args a;
  a.bias = bias;
  a.residual = residual;
  a.out = out;
  a.ldr = ldr;
  a.ldo = ldo;
  a.m = m;
  a.n_out = n_out;
  a.k = k;
  a.act = act;
  a.bias_f32 = bias_dtype == DWM_F32;
  a.res_f32 = residual_dtype == DWM_F32;
  a.out_f32 = out_dtype == DWM_F32;
  a.res_vec = residual && addr(residual) % 16 == 0 && ldr * res % 16 == 0;
  a.out_vec = addr(out) % 16 == 0 && ldo * oes % 16 == 0;
  a.limit = act_limit;
  a.res_scale = residual_scale;
  a.status = status_ptr();
  return dense::run(x, ldx, w, ldw, n, a, static_cast<cudaStream_t>(stream));
}
