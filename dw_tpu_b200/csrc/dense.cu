// Dense product with its epilogue: out = residual_scale * residual +
// act(x w^T + bias), bf16 operands, f32 accumulation, rounded once. The
// products around the expert layer that are not FP4: the router's logits, the
// shared expert's projections.
//
// Three kernels; run_epi chooses. Split kernel (a decode batch): the product is
// computed transposed, 128 rows of w as UMMA operand A, up to 128 rows of x as
// operand B, so a decode batch pays for its own tokens (N = 16 and up) and not for
// 128. The k axis is split over a cluster of 1, 2, 4 or 8 CTAs, which fills the GPU
// when w has few rows. Each CTA owns some of the tile's rows of x; all send it their
// f32 partials of those rows (bulk copies between the CTAs' shared memories), and it
// adds them in CTA order, so the result depends on the shapes alone: no atomics, no
// workspace.
//
// With SwiGLU a tile is 64 gate rows and the 64 up rows of the same features,
// which meet in the partial tile.
//
// Bound: a fixed part of some 5 us (set-up, the first copies, the exchange of the
// partials, the epilogue, which nothing overlaps), then the stream of w at the rate of
// the HBM: 64 x 4096 x 4096 with SwiGLU takes 10.5 us (its bytes 5.2), twice the k 5 us
// more, 64 x 4096 x 32768 48 (5.6 TB/s). One CTA per SM keeps ~190 KB of copies in flight.
#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace dwm {
namespace dense {

constexpr int BK = 64;          // k per stage: one 128-byte swizzled row
constexpr int TILE_W = 128;     // rows of w per tile
constexpr int THREADS = 256;
constexpr int A_STAGE = TILE_W * BK * 2;  // 16 KiB
constexpr int MAX_CLUSTER = 8;
// An f32 result is the sum of parts of at most this many k steps (2048 k), each an
// accumulator of its own. The tensor cores cut an accumulator off after every addition,
// always towards zero: one over 4096 k loses 4.4e-6 of the sum, over 8192 9.1e-6, where
// f32 additions with rounding lose 0.6e-6 and 1e-6; in parts 2.1e-6 at any k. (A bf16
// result rounds off 1.7e-3 and takes one accumulator. The few-rows kernel's warps have
// at most an eighth of k, and lose 0.15e-6 of 8192.)
constexpr int PART_STEPS = 32;

struct Args {
  const void* bias;      // [n] or NULL
  const void* residual;  // [m, n_out] or NULL
  void* out;             // [m, n_out]
  int64_t ldr, ldo;
  int m, n_out, k;
  int act;
  int bias_f32, res_f32, out_f32;
  // 8 elements at a column that is a multiple of 8 are 16-byte aligned
  int bias_vec, res_vec, out_vec;
  int out_wide;  // 32 bytes of a row are 32-byte aligned
  float limit, res_scale;
  // Split kernel: k steps of an accumulator, and the columns that they all take.
  int part_steps, tmem_cols;
  int* status;
};

template <int BT>
struct Layout {
  static constexpr int B_STAGE = BT * BK * 2;
  static constexpr int STG = A_STAGE + B_STAGE;
  static constexpr int S = 204800 / STG;  // 6 (BT = 128) to 11 stages
  static constexpr int PARTIAL = BT * TILE_W * 4;  // f32 [BT][TILE_W], over the stages
  static constexpr int OFF_RECV = PARTIAL;         // the other CTAs' partials of the own rows
  static constexpr int OFF_BAR = S * STG;
  static constexpr int OFF_MISC = OFF_BAR + (2 * S + 2) * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;  // slack for 1 KiB alignment
  static constexpr int MAX_PARTS = 512 / BT;  // accumulators that fit TMEM
  static_assert(STG % 1024 == 0, "swizzled tiles need 1 KiB alignment");
  static_assert(2 * PARTIAL <= S * STG && ALLOC <= 232448, "shared memory");
};

__device__ __forceinline__ float ld1(const void* p, int64_t i, int f32) {
  return f32 ? static_cast<const float*>(p)[i]
             : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// 8 neighbouring elements, 16-byte aligned.
__device__ __forceinline__ void load_8(const void* p, int64_t i, int f32, float (&v)[8]) {
  if (f32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 x = q[j];
      v[4 * j] = x.x; v[4 * j + 1] = x.y; v[4 * j + 2] = x.z; v[4 * j + 3] = x.w;
    }
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    }
  }
}

// 32 bytes, 32-byte aligned: one whole sector.
__device__ __forceinline__ void stg_256(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 8 values to `p` (bf16 or f32), 16-byte aligned; wide: 32-byte aligned.
__device__ __forceinline__ void store_8(void* p, int64_t i, int f32, bool wide,
                                        const float (&v)[8]) {
  if (f32) {
    float* at = static_cast<float*>(p) + i;
    uint32_t w[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) w[q] = __float_as_uint(v[q]);
    if (wide) {
      stg_256(at, w);
    } else {
      *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(at + 4) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]),
                   f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7]));
  }
}

__device__ __forceinline__ float sigmoid_full(float v) { return 1.0f / (1.0f + expf(-v)); }

// What a kernel's epilogue applies: nothing, a function of each element, or
// SwiGLU of two (kernels of their own: the branches of the others would cost
// the plain product its instruction cache).
constexpr int PLAIN = 0, POINT = 1, GLU = 2;

// The functions of one element. An f32 output takes full-precision functions,
// a bf16 one (half a step: 2^-8 of the value) the MUFU forms (~1e-6).
template <int ACT>
__device__ __forceinline__ float act_of(float z, int f32) {
  if (ACT == DWM_ACT_SILU) return z * (f32 ? sigmoid_full(z) : sigmoid_fast(z));
  if (ACT == DWM_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  // 0.5 (1 + tanh(u)) = sigmoid(2 u)
  const float u = 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
  return z * (f32 ? sigmoid_full(u) : sigmoid_fast(u));
}
template <int ACT, int N>
__device__ __forceinline__ void act_of_n(float (&z)[N], int f32) {
#pragma unroll
  for (int q = 0; q < N; ++q) z[q] = act_of<ACT>(z[q], f32);
}
template <int N>
__device__ __forceinline__ void point_act(float (&z)[N], int act, int f32) {
  if (act == DWM_ACT_SILU)
    act_of_n<DWM_ACT_SILU>(z, f32);
  else if (act == DWM_ACT_GELU)
    act_of_n<DWM_ACT_GELU>(z, f32);
  else
    act_of_n<DWM_ACT_GELU_TANH>(z, f32);
}
template <int EPI, int N>
__device__ __forceinline__ void activate(const Args& a, float (&z)[N], float (&u)[N]) {
  if (EPI == GLU) {
    if (a.act == DWM_ACT_SWIGLU_CLAMP) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        // (A NaN stays one.)
        z[q] = z[q] > a.limit ? a.limit : z[q];
        u[q] = u[q] > a.limit ? a.limit : u[q] < -a.limit ? -a.limit : u[q];
      }
    }
    if (a.out_f32) {
#pragma unroll
      for (int q = 0; q < N; ++q) z[q] = z[q] * sigmoid_full(z[q]) * u[q];
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) z[q] = z[q] * sigmoid_fast(z[q]) * u[q];
    }
  } else if (EPI == POINT) {
    point_act(z, a.act, a.out_f32);
  }
}

// Outputs [col, col + 8) of row `row` from the products z (and, with SwiGLU, the up
// products u): bias, activation, residual, one rounding. Rows of out start on 16 bytes
// (Args::out_vec).
template <int EPI>
__device__ __forceinline__ void epilogue(const Args& a, int64_t row, int col, float (&z)[8],
                                         float (&u)[8]) {
  const bool whole = col + 8 <= a.n_out;
  if (a.bias) {
    float b[8];
    auto bias = [&](int off) {
      if (whole && a.bias_vec) {
        load_8(a.bias, off + col, a.bias_f32, b);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) b[q] = ld1(a.bias, off + min(col + q, a.n_out - 1), a.bias_f32);
      }
    };
    bias(0);
#pragma unroll
    for (int q = 0; q < 8; ++q) z[q] += b[q];
    if (EPI == GLU) {
      bias(a.n_out);
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] += b[q];
    }
  }
  activate<EPI>(a, z, u);
  if (a.residual) {
    const int64_t at = row * a.ldr + col;
    if (whole && a.res_vec) {
      float r[8];
      load_8(a.residual, at, a.res_f32, r);
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = fmaf(a.res_scale, r[q], z[q]);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (col + q < a.n_out) z[q] = fmaf(a.res_scale, ld1(a.residual, at + q, a.res_f32), z[q]);
    }
  }
  const int64_t at = row * a.ldo + col;
  if (whole) {
    store_8(a.out, at, a.out_f32, a.out_wide != 0, z);
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

// For outputs whose rows do not start on 16 bytes: column `col` of the rows
// [row, row + n), n <= N; neighbouring threads take neighbouring columns. Eight
// rows at a time keep the loads and functions of several in flight (one at a
// time took 10 us more for 1024 x 777).
template <int EPI, int N>
__device__ __forceinline__ void epilogue_column(const Args& a, int64_t row, int n, int col,
                                                float (&z)[N], float (&u)[N]) {
  if (a.bias) {
    const float b = ld1(a.bias, col, a.bias_f32);
#pragma unroll
    for (int q = 0; q < N; ++q) z[q] += b;
    if (EPI == GLU) {
      const float c = ld1(a.bias, a.n_out + col, a.bias_f32);
#pragma unroll
      for (int q = 0; q < N; ++q) u[q] += c;
    }
  }
  activate<EPI>(a, z, u);
  if (a.residual) {
    float r[N];
    const int64_t at = row * a.ldr + col;
    if (a.res_f32) {
#pragma unroll
      for (int q = 0; q < N; ++q)
        r[q] = static_cast<const float*>(a.residual)[at + (int64_t)min(q, n - 1) * a.ldr];
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q)
        r[q] = bf16_bits_to_f32(
            static_cast<const uint16_t*>(a.residual)[at + (int64_t)min(q, n - 1) * a.ldr]);
    }
#pragma unroll
    for (int q = 0; q < N; ++q) z[q] = fmaf(a.res_scale, r[q], z[q]);
  }
  const int64_t at = row * a.ldo + col;
  if (a.out_f32) {
    float* o = static_cast<float*>(a.out) + at;
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (q < n) o[q * a.ldo] = z[q];
  } else {
    uint16_t* o = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (q < n) o[q * a.ldo] = (uint16_t)f32_to_bf16_bits(z[q]);
  }
}

// A bulk copy from this CTA's shared memory to CTA `to` of the cluster, which
// completes on that CTA's mbarrier. dst, bar: the addresses here of what they
// are there.
__device__ __forceinline__ void bulk_to_cta(uint32_t dst, uint32_t src, uint32_t bytes,
                                            uint32_t bar, int to) {
  asm volatile(
      "{\n\t.reg .b32 d, b;\n\t"
      "mapa.shared::cluster.u32 d, %0, %4;\n\t"
      "mapa.shared::cluster.u32 b, %3, %4;\n\t"
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [d], [%1], %2, [b];"
      "\n\t}" ::"r"(dst),
      "r"(src), "r"(bytes), "r"(bar), "r"(to)
      : "memory");
}

// grid (cluster, w tiles, x tiles); GLU: the tile's 128 rows of w are 64 gate
// rows and the up rows of the same features.
template <int BT, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    dense_split_kernel(const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_x, const Args a) {
  using L = Layout<BT>;
  constexpr int S = L::S;
  constexpr int FEAT = EPI == GLU ? TILE_W / 2 : TILE_W;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint64_t* received = done + 1;
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
    mbar_init(received, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  overlap_wait();
  overlap_next();

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
        if (EPI == GLU) {
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
    uint32_t acc = tmem;  // the part's accumulator
    int in = 0;           // its steps so far
    for (int i = 0; i < steps; ++i) {
      const int st = i % S;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (i / S) & 1, abort_flag, a.status));
      if (!ok) break;
      tc_fence_after();
      if (issuer) {
        const uint32_t base = smem_u32(smem + st * L::STG);
#pragma unroll
        for (int j = 0; j < BK / 16; ++j)
          umma_bf16(acc, smem_desc_sw128(base + j * 32, 16, 1024),
                    smem_desc_sw128(base + A_STAGE + j * 32, 16, 1024), idesc, (in | j) != 0);
        umma_commit(&empty[st]);
      }
      __syncwarp();
      if (++in == a.part_steps) {
        in = 0;
        acc += BT;
      }
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
  const int rows = min(BT, a.m - row0);
  const int own = BT / split;  // this CTA's rows of x: from rank * own
  const int mine = max(0, min(own, rows - rank * own));
  const uint32_t part = smem_u32(smem);
  {
    // The partial tile [row of x][row of w]. Warp w reads TMEM lanes (rows of
    // w) 32 (w % 4) .. and one half of the columns (rows of x).
    const int q = warp & 3, half = warp >> 2;
    constexpr int COLS = BT / 2 < 16 ? 16 : BT / 2;
    if (half * COLS < BT) {
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        const int t0 = half * COLS + c;
        if (t0 >= rows) break;
        uint32_t r[16];
        uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + t0;
        tmem_ld16(at, r);
        tmem_ld_wait(r);
        for (int i = a.part_steps; i < steps; i += a.part_steps) {
          uint32_t more[16];
          at += BT;
          tmem_ld16(at, more);
          tmem_ld_wait(more);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(more[e]));
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sts_u32(part + (uint32_t)(((t0 + e) * TILE_W + q * 32 + lane) * 4), r[e]);
      }
    }
  }
  tc_fence_before();
  if (split > 1) {
    fence_proxy_async_smem();  // the partials, for the bulk copies
    if (threadIdx.x == 0)
      mbar_arrive_expect_tx(received, (uint32_t)((split - 1) * mine * TILE_W * 4));
    // Every CTA of the cluster is done with its stages, where the partials of
    // the others now go.
    cluster_sync();
    if ((int)threadIdx.x < split && (int)threadIdx.x != rank) {
      const int to = threadIdx.x, n = max(0, min(own, rows - to * own));
      if (n > 0)
        bulk_to_cta(part + (uint32_t)(L::OFF_RECV + (rank - (rank > to)) * own * TILE_W * 4),
                    part + (uint32_t)(to * own * TILE_W * 4), (uint32_t)(n * TILE_W * 4),
                    smem_u32(received), to);
    }
    __syncwarp();
    ok = mbar_wait(received, 0, nullptr, a.status) && ok;
    __syncwarp();
    cluster_arrive();  // this CTA has what it waits for
  } else {
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, a.tmem_cols);

  // This CTA's rows: the partials in CTA order, 8 columns a thread.
  if (ok) {
    const int cols = min(FEAT, a.n_out - col0);
    // Where CTA p's partials of the own rows are.
    auto from = [&](int p) {
      return part + (uint32_t)((p == rank ? rank * own * TILE_W * 4
                                          : L::OFF_RECV + (p - (p > rank)) * own * TILE_W * 4));
    };
    if (a.out_vec) {
      constexpr int CH = FEAT / 8;
      for (int i = threadIdx.x; i < mine * CH; i += THREADS) {
        const int t = i / CH, c = (i % CH) * 8;
        if (c >= cols) continue;
        float z[8], u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = u[e] = 0.0f;
        auto add = [](float (&v)[8], uint32_t p) {
          const uint4 x = lds_u128(p), y = lds_u128(p + 16);
          v[0] += __uint_as_float(x.x); v[1] += __uint_as_float(x.y);
          v[2] += __uint_as_float(x.z); v[3] += __uint_as_float(x.w);
          v[4] += __uint_as_float(y.x); v[5] += __uint_as_float(y.y);
          v[6] += __uint_as_float(y.z); v[7] += __uint_as_float(y.w);
        };
        for (int p = 0; p < split; ++p) {
          const uint32_t at = from(p) + (uint32_t)((t * TILE_W + c) * 4);
          add(z, at);
          if (EPI == GLU) add(u, at + FEAT * 4);
        }
        epilogue<EPI>(a, row0 + rank * own + t, col0 + c, z, u);
      }
    } else {
      const int c = threadIdx.x % FEAT;
      if (c < cols)
        for (int t = threadIdx.x / FEAT * 8; t < mine; t += THREADS / FEAT * 8) {
          float z[8], u[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) z[q] = u[q] = 0.0f;
          for (int p = 0; p < split; ++p) {
            // (Rows past the own ones are read within the shared memory, and
            // dropped.)
            const uint32_t at = from(p) + (uint32_t)((t * TILE_W + c) * 4);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              z[q] += lds_f32(at + q * TILE_W * 4);
              if (EPI == GLU) u[q] += lds_f32(at + (q * TILE_W + FEAT) * 4);
            }
          }
          epilogue_column<EPI>(a, row0 + rank * own + t, min(8, mine - t), col0 + c, z, u);
        }
    }
  }
  // A CTA's partials may still be on their way to another one until all have
  // arrived.
  __syncwarp();
  if (split > 1) cluster_wait();
}

// Clusters of `size` CTAs, one CTA per SM, resident at once on the current
// device (asked once of each): as many as the split kernel with its largest
// shared memory allows, which the pair kernel's equals.
int resident_clusters(int size) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> cached[kMaxDevices][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int i = size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3;
  const bool keep = dev >= 0 && dev < kMaxDevices;
  if (keep) {
    const int n = cached[dev][i].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int n = num_sms() / size;
  if (size > 1) {
    using L = Layout<128>;
    auto fn = dense_split_kernel<128, PLAIN>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)size, (unsigned)std::max(1, n));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = L::ALLOC;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (set_smem_limit(reinterpret_cast<const void*>(fn), L::ALLOC, "dense smem attribute") ==
            DWM_OK &&
        cudaOccupancyMaxActiveClusters(&got, fn, &cfg) == cudaSuccess && got > 0)
      n = got;
    else
      (void)cudaGetLastError();
  }
  n = std::max(1, n);
  if (keep) cached[dev][i].store(n, std::memory_order_relaxed);
  return n;
}

template <int BT, int EPI>
int launch_split(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, int split,
                 Args a, cudaStream_t stream) {
  using L = Layout<BT>;
  const int steps = ((a.k + BK - 1) / BK + split - 1) / split;  // of a CTA, or one fewer
  a.part_steps =
      a.out_f32 ? std::max(PART_STEPS, (steps + L::MAX_PARTS - 1) / L::MAX_PARTS) : steps;
  const int parts = (steps + a.part_steps - 1) / a.part_steps;
  for (a.tmem_cols = 32; a.tmem_cols < parts * BT;) a.tmem_cols *= 2;
  constexpr int FEAT = EPI == GLU ? TILE_W / 2 : TILE_W;
  DWM_CHECK_ARG((a.m + (int64_t)BT - 1) / BT <= 65535 &&
                    (a.n_out + (int64_t)FEAT - 1) / FEAT <= 65535,
                "m=%d rows by %d columns exceed the grid", a.m, a.n_out);
  CUtensorMap tm_w, tm_x;
  int rc = encode_tmap_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, w, (uint64_t)a.k, (uint64_t)n,
                          (uint64_t)ldw * 2, BK, FEAT, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = encode_tmap_2d(&tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, (uint64_t)a.k, (uint64_t)a.m,
                      (uint64_t)ldx * 2, BK, BT, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = set_smem_limit(reinterpret_cast<const void*>(dense_split_kernel<BT, EPI>), L::ALLOC,
                      "dense smem attribute");
  if (rc) return rc;
  return check_cuda(overlap_launch(dense_split_kernel<BT, EPI>,
                                   dim3((unsigned)split, (unsigned)((a.n_out + FEAT - 1) / FEAT),
                                        (unsigned)((a.m + BT - 1) / BT)),
                                   dim3(THREADS), L::ALLOC, split, stream, tm_w, tm_x, a),
                    "dense_matmul launch");
}

// ---------------------------------------------------------------------------
// Pair kernel (prompts). Two CTAs on neighbouring SMs (cta_group::2) share a
// tile of 256 rows of x by 256 rows of w: each CTA loads its 128 rows of both
// (one box each a k step), the even one issues the 256 x 256 x 16 UMMAs, and
// each CTA's TMEM receives its 128 rows of x by all 256 columns, twice (the
// epilogue of a tile overlaps the main loop of the next). Persistent: one pair
// of SMs takes every ncl-th tile, eight rows of tiles at a time so that what
// runs together shares its operands in L2. With SwiGLU the even CTA's half of
// w's rows is the gate and the odd one's the up projection of 128 features, so
// a feature's two products are two columns of one TMEM lane.
//
// Warps 0-7 epilogue (TMEM lane quarter w % 4, half w / 4 of the columns): a row
// a lane, 32 columns at a time through swizzled shared memory and TMA, the
// residual in and the result out (16-byte accesses of a row a lane instead cost
// 32 cache lines an instruction: 1024 x 2048 x 4096 with an f32 residual took 26
// us); warp 8 TMA; warp 9 UMMA.
//
// Bound: the tensor cores: 8192 x 4096 x 4096 with SwiGLU 169-180 us (1530-1630
// TFLOP/s, by how long the power limit lets the clock stand); at one wave of tiles
// the first loads and the last epilogue, which nothing overlaps: 1024 x 2048 x 4096
// with bias and f32 residual 22.3 us, without them 17.8.
// ---------------------------------------------------------------------------
namespace pair {

constexpr int TILE = 256;      // rows of x, and of w, per tile
constexpr int HALF = 128;      // per CTA
constexpr int THREADS = 320;
constexpr int EPI_WARPS = 8, TMA_WARP = 8, MMA_WARP = 9;
constexpr int OP_STAGE = HALF * BK * 2;  // 16 KiB: one operand's k step
constexpr int STG = 2 * OP_STAGE;
constexpr int BOX = 32;                  // rows and columns of an epilogue step
constexpr int OUT_BYTES = BOX * BOX * 4;  // a warp's: one f32 step or two bf16 ones
// RES: the residual comes by TMA, into room for two f32 or four bf16 steps a
// warp, which leaves four k steps of operands instead of six.
template <bool RES>
struct Layout {
  static constexpr int S = RES ? 4 : 6;
  static constexpr int RES_BYTES = RES ? 2 * OUT_BYTES : 0;
  static constexpr int OFF_OUT = S * STG;
  static constexpr int OFF_RES = OFF_OUT + EPI_WARPS * OUT_BYTES;
  static constexpr int OFF_BAR = OFF_RES + EPI_WARPS * RES_BYTES;
  static constexpr int OFF_MISC = OFF_BAR + (2 * S + 5 + 4 * EPI_WARPS) * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;  // slack for 1 KiB alignment
  static_assert(ALLOC <= 232448, "exceeds the 227 KiB per-CTA shared memory");
};
constexpr int TMEM_COLS = 512;
constexpr int GROUP_ROWS = 8;  // rows of tiles taken together

__device__ __forceinline__ void tile_at(int idx, int mt, int nt, int& tm, int& tn) {
  const int per = GROUP_ROWS * nt, g = idx / per;
  const int rows = min(GROUP_ROWS, mt - g * GROUP_ROWS);
  const int in = idx - g * per;
  tm = g * GROUP_ROWS + in % rows;
  tn = in / rows;
}

// Byte offset of 16-byte chunk c of row r in a box of 32 rows of 32 elements, as
// TMA swizzles it: 64-byte rows (bf16) or 128-byte rows (f32).
__device__ __forceinline__ uint32_t box_at(int r, int c, int f32) {
  return f32 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4))
             : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// VEC: rows of out and of the residual start on 16 bytes; RES: there is one
// (without VEC it is read where it is added). SUMS: a sum over k is made of parts
// (PART_STEPS): one accumulator takes them, and the epilogue warps add each to the
// other one, where they find the whole sum at last. (The UMMAs wait for that once a
// part: 8192 x 8192 x 2048 f32 takes 209 us, 196 with one accumulator.)
template <int EPI, bool VEC, bool RES, bool SUMS>
__global__ void __launch_bounds__(THREADS, 1)
    dense_pair_kernel(const __grid_constant__ CUtensorMap tm_x,
                      const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_out,
                      const __grid_constant__ CUtensorMap tm_res, const Args a) {
  using L = Layout<RES>;
  constexpr int S = L::S;
  constexpr int FEAT = EPI == GLU ? HALF : TILE;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);  // even CTA: both CTAs' copies landed
  uint64_t* empty = full + S;          // each CTA: the pair's UMMAs done with the stage
  uint64_t* acc_full = empty + S;      // each CTA: accumulator complete
  uint64_t* acc_empty = acc_full + 2;  // even CTA: both CTAs drained it
  uint64_t* drain = acc_empty + 2;     // each CTA: every UMMA complete
  uint64_t* res_full = drain + 1;      // [EPI_WARPS][4]: a residual step has landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cl = (int)cluster_index(), ncl = (int)cluster_count();
  const int mt = (a.m + TILE - 1) / TILE, nt = (a.n_out + FEAT - 1) / FEAT;
  const int total = mt * nt;
  const int kt = (a.k + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * EPI_WARPS);
    }
    mbar_init(drain, 1);
    if (RES)
      for (int i = 0; i < 4 * EPI_WARPS; ++i) mbar_init(&res_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == MMA_WARP) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  // Barriers initialised and TMEM allocated in both CTAs before any
  // cross-CTA arrival.
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  overlap_wait();
  overlap_next();
  const uint32_t full_0 = mapa_shared(full, 0);
  const uint32_t acc_empty_0 = mapa_shared(acc_empty, 0);

  if (warp < EPI_WARPS) {
    const int q = warp & 3, half = warp >> 2;
    const uint32_t stage = smem_u32(smem + L::OFF_OUT + warp * OUT_BYTES);
    uint8_t* res_smem = smem + L::OFF_RES + warp * L::RES_BYTES;
    const uint32_t res_at = smem_u32(res_smem);
    const int out_step = a.out_f32 ? OUT_BYTES : OUT_BYTES / 2;  // bytes of a step
    const int res_step = a.res_f32 ? OUT_BYTES : OUT_BYTES / 2, res_ring = a.res_f32 ? 2 : 4;
    int out_buf = 0, res_buf = 0;
    uint32_t res_ph = 0;
    int slot = 0;
    uint32_t ph = 0;
    bool res_ok = true;
    for (int idx = cl; idx < total; idx += ncl) {
      int tm, tn;
      tile_at(idx, mt, nt, tm, tn);
      const int64_t row0 = (int64_t)tm * TILE + rank * HALF + q * 32;
      const int col0 = tn * FEAT + half * (FEAT / 2);
      const int valid = (int)min((int64_t)32, a.m - row0);  // rows, maybe none
      // Steps of 32 output columns, of two blocks of 16.
      const int cols = valid <= 0 ? 0 : min(FEAT / 2, a.n_out - col0);
      const int steps = (cols + BOX - 1) / BOX, blocks = (cols + 15) / 16;
      auto fetch_res = [&](int i) {  // lane 0: step i into the ring's place for it
        const int at = (res_buf + i) % res_ring;
        uint64_t* bar = &res_full[warp * 4 + at];
        mbar_arrive_expect_tx(bar, (uint32_t)res_step);
        tma_load_2d(res_smem + at * res_step, &tm_res, bar, col0 + i * BOX, (int)row0,
                    policy_evict_first());
      };
      if (RES && lane == 0) {
        for (int i = 0; i < min(steps, res_ring); ++i) fetch_res(i);
        for (int i = res_ring; i < steps; ++i)
          tma_prefetch_2d(&tm_res, col0 + i * BOX, (int)row0);
      }
      // Bias of four of the warp's columns (SwiGLU: of the gate's in the first
      // 16 lanes, of the up projection's in the others).
      float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (VEC && a.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = min(col0 + (EPI == GLU ? lane & 15 : lane) * 4 + j, a.n_out - 1);
          bias[j] = ld1(a.bias, c + (EPI == GLU && lane >= 16 ? a.n_out : 0), a.bias_f32);
        }
      }
      // The residual's copies in flight, of `left` steps, land before the exit.
      auto land = [&](int left) {
        if (RES && lane == 0)
          for (int i = 0; i < min(left, res_ring); ++i) {
            const int at = (res_buf + i) % res_ring;
            mbar_wait(&res_full[warp * 4 + at], (res_ph >> at) & 1u, nullptr, a.status);
          }
      };
      if (!__all_sync(0xffffffffu, mbar_wait<64>(&acc_full[slot], ph, abort_flag, a.status))) {
        land(steps);
        break;
      }
      tc_fence_after();
      uint32_t acc =
          tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(slot * TILE + half * (FEAT / 2));
      uint32_t r0[16], r1[16];
      if (SUMS) {
        bool whole = true;
        for (int k0 = 0;;) {
          for (int c = 0; c < blocks * 16; c += 16)
#pragma unroll
            for (int up = 0; up < (EPI == GLU ? 2 : 1); ++up) {
              const uint32_t at = acc + (uint32_t)(c + up * HALF);
              tmem_ld16(at, r0);
              if (k0 > 0) tmem_ld16(at + TILE, r1);
              tmem_ld_wait(r0);
              if (k0 > 0) {
                tmem_ld_wait(r1);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  r0[j] = __float_as_uint(__uint_as_float(r0[j]) + __uint_as_float(r1[j]));
              }
              tmem_st16(at + TILE, r0);
            }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(acc_empty_0);
          ph ^= 1;
          k0 += PART_STEPS;
          if (k0 >= kt) break;
          if (!__all_sync(0xffffffffu, mbar_wait<64>(&acc_full[0], ph, abort_flag, a.status))) {
            whole = false;
            break;
          }
          tc_fence_after();
        }
        if (!whole) {
          land(steps);
          break;
        }
        acc += TILE;
      }
      auto fetch = [&](int c) {
        tmem_ld16(acc + c, r0);
        if (EPI == GLU) tmem_ld16(acc + c + HALF, r1);
      };
      if (blocks > 0) fetch(0);
      for (int b = 0; b < blocks; ++b) {
        const int c = b * 16;
        tmem_ld_wait(r0);
        if (EPI == GLU) tmem_ld_wait(r1);
        if (VEC) {
          float z[16], u[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            z[j] = __uint_as_float(r0[j]);
            u[j] = EPI == GLU ? __uint_as_float(r1[j]) : 0.0f;
          }
          if (b + 1 < blocks) fetch(c + 16);
          if (a.bias) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              z[j] += __shfl_sync(0xffffffffu, bias[j & 3], (c + j) >> 2);
              if (EPI == GLU) u[j] += __shfl_sync(0xffffffffu, bias[j & 3], 16 + ((c + j) >> 2));
            }
          }
          activate<EPI>(a, z, u);
          if (RES) {
            if ((b & 1) == 0 &&
                !__all_sync(0xffffffffu, mbar_wait(&res_full[warp * 4 + res_buf],
                                                   (res_ph >> res_buf) & 1u, abort_flag,
                                                   a.status))) {
              land(steps - (b >> 1));
              res_ok = false;
              break;
            }
            const uint32_t from = res_at + (uint32_t)(res_buf * res_step);
            float r[16];
            if (a.res_f32) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint4 x = lds_u128(from + box_at(lane, (b & 1) * 4 + j, 1));
                r[4 * j] = __uint_as_float(x.x); r[4 * j + 1] = __uint_as_float(x.y);
                r[4 * j + 2] = __uint_as_float(x.z); r[4 * j + 3] = __uint_as_float(x.w);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint4 x = lds_u128(from + box_at(lane, (b & 1) * 2 + j, 0));
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  r[8 * j + 2 * e] = __uint_as_float(w[e] << 16);
                  r[8 * j + 2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = fmaf(a.res_scale, r[j], z[j]);
          }
          if ((b & 1) == 0) {
            // The store that last read this buffer is done with it.
            if (lane == 0) {
              if (a.out_f32)
                bulk_wait_read<0>();
              else
                bulk_wait_read<1>();
            }
            __syncwarp();
          }
          const uint32_t to = stage + (uint32_t)(out_buf * out_step);
          if (a.out_f32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              sts_u128(to + box_at(lane, (b & 1) * 4 + j, 1), __float_as_uint(z[4 * j]),
                       __float_as_uint(z[4 * j + 1]), __float_as_uint(z[4 * j + 2]),
                       __float_as_uint(z[4 * j + 3]));
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              sts_u128(to + box_at(lane, (b & 1) * 2 + j, 0),
                       f32x2_to_bf16x2(z[8 * j], z[8 * j + 1]),
                       f32x2_to_bf16x2(z[8 * j + 2], z[8 * j + 3]),
                       f32x2_to_bf16x2(z[8 * j + 4], z[8 * j + 5]),
                       f32x2_to_bf16x2(z[8 * j + 6], z[8 * j + 7]));
          }
          if ((b & 1) == 1 || b + 1 == blocks) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              // (Columns and rows past the end are not stored.)
              tma_store_2d(&tm_out, to, col0 + (b >> 1) * BOX, (int)row0);
              bulk_commit();
            }
            if (!a.out_f32) out_buf ^= 1;
            if (RES) {
              // Every lane has read the step: its place takes the next but few.
              res_ph ^= 1u << res_buf;
              if (lane == 0 && (b >> 1) + res_ring < steps) {
                uint64_t* bar = &res_full[warp * 4 + res_buf];
                mbar_arrive_expect_tx(bar, (uint32_t)res_step);
                tma_load_2d(res_smem + res_buf * res_step, &tm_res, bar,
                            col0 + ((b >> 1) + res_ring) * BOX, (int)row0, policy_evict_first());
              }
              if (++res_buf == res_ring) res_buf = 0;
            }
          }
        } else {
          // A column a lane, two rows of 16 at a time, by way of shared memory:
          // 16-byte blocks of a row of 32, XORed with the row against conflicts.
          auto block_at = [&](int rr, int j) {
            return stage + (uint32_t)(rr * 128 + ((j ^ (rr & 7)) << 4));
          };
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sts_u128(block_at(lane, j), r0[4 * j], r0[4 * j + 1], r0[4 * j + 2], r0[4 * j + 3]);
            if (EPI == GLU)
              sts_u128(block_at(lane, 4 + j), r1[4 * j], r1[4 * j + 1], r1[4 * j + 2],
                       r1[4 * j + 3]);
          }
          __syncwarp();
          if (b + 1 < blocks) fetch(c + 16);
          const int col = lane % 16;
          if (col0 + c + col < a.n_out)
            for (int rr = lane / 16 * 8; rr < valid; rr += 16) {
              float z[8], u[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                z[q] = lds_f32(block_at(rr + q, col / 4) + (uint32_t)(col % 4) * 4);
                if (EPI == GLU)
                  u[q] = lds_f32(block_at(rr + q, 4 + col / 4) + (uint32_t)(col % 4) * 4);
              }
              epilogue_column<EPI>(a, row0 + rr, min(8, valid - rr), col0 + c + col, z, u);
            }
          __syncwarp();
        }
      }
      if (!res_ok) break;
      if (!SUMS) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(acc_empty_0 + (uint32_t)(slot * 8));
        if (++slot == 2) { slot = 0; ph ^= 1; }
      }
    }
    if (VEC && lane == 0) bulk_wait_all();  // before this CTA's shared memory goes
  } else if (warp == TMA_WARP) {
    if (lane == 0) {
      const uint64_t pol_w = policy_evict_last(), pol_x = policy_evict_normal();
      int st = 0;
      uint32_t ph = 0, armed = 0, par = 0;
      bool ok = true;
      for (int idx = cl; idx < total && ok; idx += ncl) {
        int tm, tn;
        tile_at(idx, mt, nt, tm, tn);
        const int xrow = tm * TILE + (int)rank * HALF;
        const int wrow = EPI == GLU ? tn * FEAT + (rank ? a.n_out : 0) : tn * FEAT + (int)rank * HALF;
        for (int kk = 0; kk < kt; ++kk) {
          if (!mbar_wait(&empty[st], ph ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * STG);
          armed |= 1u << st;
          par = (par & ~(1u << st)) | (ph << st);
          const uint32_t bar = full_0 + (uint32_t)(st * 8);
          uint8_t* dst = smem + st * STG;
          tma_load_2d_pair(dst, &tm_x, bar, kk * BK, xrow, pol_x);
          tma_load_2d_pair(dst + OP_STAGE, &tm_w, bar, kk * BK, wrow, pol_w);
          if (++st == S) { st = 0; ph ^= 1; }
        }
      }
      // Every stage this warp filled is released by the pair's UMMAs (so its
      // copies have landed) before the CTA can exit.
      for (int i = 0; i < S; ++i)
        if (armed & (1u << i)) mbar_wait(&empty[i], (par >> i) & 1, nullptr, a.status);
    }
  } else {
    if (rank == 0) {
      const bool issuer = elect_one();
      constexpr uint32_t idesc = idesc_bf16(TILE, TILE, false, false);
      int st = 0, slot = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      const int part = SUMS ? PART_STEPS : kt;  // k steps of an accumulator
      for (int idx = cl; idx < total && ok; idx += ncl) {
        for (int k0 = 0; k0 < kt && ok; k0 += part) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&acc_empty[slot], acc_ph ^ 1, abort_flag, a.status));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(slot * TILE);
          const int k1 = min(kt, k0 + part);
          for (int kk = k0; kk < k1; ++kk) {
            if (!__all_sync(0xffffffffu, mbar_wait(&full[st], ph, abort_flag, a.status))) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (issuer) {
              const uint32_t base = smem_u32(smem + st * STG);
#pragma unroll
              for (int j = 0; j < BK / 16; ++j)
                umma_pair_bf16(d, smem_desc_sw128(base + j * 32, 16, 1024),
                               smem_desc_sw128(base + OP_STAGE + j * 32, 16, 1024), idesc,
                               ((kk - k0) | j) != 0);
              umma_commit_pair(&empty[st]);
            }
            __syncwarp();
            if (++st == S) { st = 0; ph ^= 1; }
          }
          if (!ok) break;
          if (issuer) umma_commit_pair(&acc_full[slot]);
          __syncwarp();
          if (SUMS) {
            acc_ph ^= 1;  // (the other accumulator is the epilogue's)
          } else if (++slot == 2) {
            slot = 0;
            acc_ph ^= 1;
          }
        }
      }
      if (issuer) umma_commit_pair(drain);
      __syncwarp();
    }
    // Both CTAs: every UMMA (which writes both TMEMs) completes before TMEM
    // is released.
    // The odd CTA waits here from the start, so its limit grows with the tiles.
    if (lane == 0) {
      const uint64_t t0 = globaltimer_ns(), limit = kWaitLimitNs * (uint64_t)(1 + total / ncl);
      while (!mbar_try_wait(drain, 0)) {
        __nanosleep(500);
        if (globaltimer_ns() - t0 > limit) {
          report(a.status, DWM_DEV_TIMEOUT);
          break;
        }
      }
    }
  }
  // Both CTAs are done with every barrier, shared tile and TMEM column.
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
  cluster_sync();
}

template <int EPI, bool VEC, bool RES, bool SUMS>
int launch_as(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, const Args& a,
              cudaStream_t stream) {
  using L = Layout<RES>;
  constexpr int FEAT = EPI == GLU ? HALF : TILE;
  const int64_t tiles = (int64_t)((a.m + (int64_t)TILE - 1) / TILE) *
                        ((a.n_out + (int64_t)FEAT - 1) / FEAT);
  DWM_CHECK_ARG(tiles < (1ll << 30), "m=%d rows by %d columns are too many tiles", a.m, a.n_out);
  CUtensorMap tm_x, tm_w, tm_out, tm_res;
  int rc = encode_tmap_2d(&tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, (uint64_t)a.k, (uint64_t)a.m,
                          (uint64_t)ldx * 2, BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = encode_tmap_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, w, (uint64_t)a.k, (uint64_t)n,
                      (uint64_t)ldw * 2, BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  auto box_map = [&](CUtensorMap* map, const void* p, int64_t ld, int f32) {
    return encode_tmap_2d(
        map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p,
        (uint64_t)a.n_out, (uint64_t)a.m, (uint64_t)ld * (f32 ? 4 : 2), BOX, BOX,
        f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  };
  tm_out = tm_res = tm_x;  // (unused without VEC, without RES)
  if (VEC && (rc = box_map(&tm_out, a.out, a.ldo, a.out_f32))) return rc;
  if (RES && (rc = box_map(&tm_res, a.residual, a.ldr, a.res_f32))) return rc;
  auto fn = dense_pair_kernel<EPI, VEC, RES, SUMS>;
  rc = set_smem_limit(reinterpret_cast<const void*>(fn), L::ALLOC, "dense pair smem attribute");
  if (rc) return rc;
  return check_cuda(
      overlap_launch(fn,
                     dim3(2 * (unsigned)std::min<int64_t>(tiles, resident_clusters(2))),
                     dim3(THREADS), L::ALLOC, 2, stream, tm_x, tm_w, tm_out, tm_res, a),
      "dense_matmul launch");
}

template <int EPI, bool VEC, bool RES>
int launch(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, const Args& a,
           cudaStream_t stream) {
  return a.out_f32 && (a.k + BK - 1) / BK > PART_STEPS
             ? launch_as<EPI, VEC, RES, true>(x, ldx, w, ldw, n, a, stream)
             : launch_as<EPI, VEC, RES, false>(x, ldx, w, ldw, n, a, stream);
}

}  // namespace pair

// ---------------------------------------------------------------------------
// Few-rows kernel (decode steps, and small products). 16 rows of w (SwiGLU: 8
// gate rows and the 8 up rows of the same features) are operand A of
// mma.m16n8k16, up to 8 NT rows of x operand B, both straight from global memory
// into registers: lane t of a quad takes 8 consecutive k of a row in one 16-byte
// load and gives its halves to two products, which add the same k in both
// operands, in another order than they lie. A CTA's warps take every eighth of
// 64 k, the CTAs of a cluster (when w has few rows) every so many of those; the
// partial sums are added in warp and in CTA order.
//
// Bound: the stream of w, and for small w the launch and a memory latency,
// which a kernel without TMA, mbarriers and TMEM to set up gets to sooner: 1 x
// 4096 x 256 takes 2.4 us (split kernel 5.3), 1 x 4096 x 8192 13.8 (4.9 TB/s; 14.1).
// Tiles of 32 x 32 read half as much for a product: 333 x 1000 x 776 takes 5.4 us
// with them, 9.5 with 16 x 16, 8.5 with the split kernel.
// ---------------------------------------------------------------------------
namespace few {

constexpr int WARPS = 8, THREADS = 32 * WARPS;

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int EPI>
__host__ __device__ __forceinline__ int tiles(int n_out, int mt) {
  const int feat = (EPI == GLU ? 8 : 16) * mt;
  return (n_out + feat - 1) / feat;
}

// A tile: MT groups of 16 rows of w by NT groups of 8 rows of x. U: 64-k steps
// whose loads are issued together. MAX_SPLIT: the most CTAs on one tile's k. grid:
// x tiles x w tiles x split.
template <int MT, int NT, int U, int MAX_SPLIT, int EPI>
__global__ void __launch_bounds__(THREADS, 2)
    dense_few_kernel(const uint16_t* x, int64_t ldx, const uint16_t* w,
                     int64_t ldw, int split, const Args a) {
  constexpr int GROUP = EPI == GLU ? 8 : 16;  // output columns of 16 rows of w
  constexpr int FEAT = MT * GROUP;
  constexpr int ROWS = MT * 16 + 4;    // (4: apart, the quads' sums are in banks of their own)
  constexpr int SUMS = 8 * NT * ROWS;  // [row of x][row of the tile]
  __shared__ float part[WARPS][SUMS];
  __shared__ float recv[MAX_SPLIT][SUMS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % split, tile = blockIdx.x / split, nt = tiles<EPI>(a.n_out, MT);
  const int col0 = tile % nt * FEAT, row0 = tile / nt * (8 * NT);
  if (split > 1) cluster_arrive();
  // Rows past the last repeat it; their sums are not used.
  const uint16_t *wp[MT][2], *xp[NT];
#pragma unroll
  for (int g = 0; g < MT; ++g) {
    const int r0 = min(col0 + g * GROUP + gid, a.n_out - 1);
    const int r1 = EPI == GLU ? r0 + a.n_out : min(col0 + g * GROUP + gid + 8, a.n_out - 1);
    wp[g][0] = w + r0 * ldw + t * 8;
    wp[g][1] = w + r1 * ldw + t * 8;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) xp[j] = x + min(row0 + gid + 8 * j, a.m - 1) * ldx + t * 8;
  float c[MT][NT][4];
#pragma unroll
  for (int g = 0; g < MT; ++g)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[g][j][e] = 0.0f;
  // The outputs of a thread: column f of `mine` rows of the tile from `row`.
  constexpr int OUTS = 8 * NT * FEAT > THREADS ? 8 * NT * FEAT / THREADS : 1;
  const int row = threadIdx.x / FEAT * OUTS, f = threadIdx.x % FEAT;
  const int mine = col0 + f < a.n_out ? min(OUTS, min(8 * NT, a.m - row0) - row) : 0;
  overlap_wait();
  overlap_next();
  if (a.residual && rank == 0)
    for (int q = 0; q < mine; ++q) {
      const int64_t at = (row0 + row + q) * a.ldr + col0 + f;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.residual) +
                                                    at * (a.res_f32 ? 4 : 2)));
    }

  const int kt = (a.k + BK - 1) / BK, stride = split * WARPS;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int s = rank * WARPS + warp; s < kt; s += stride * U) {
    uint4 ws[U][2][MT][2], xs[U][2][NT];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t at = (int64_t)(s + i * stride) * BK + h * 32;
        const bool in = at + t * 8 < a.k;  // 8 k are all in or all out
#pragma unroll
        for (int g = 0; g < MT; ++g)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            ws[i][h][g][r] = in ? __ldcs(reinterpret_cast<const uint4*>(wp[g][r] + at)) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          xs[i][h][j] = in ? *reinterpret_cast<const uint4*>(xp[j] + at) : zero;
      }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < MT; ++g)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 &p = ws[i][h][g][0], &q = ws[i][h][g][1], &v = xs[i][h][j];
            mma(c[g][j], p.x, q.x, p.y, q.y, v.x, v.y);
            mma(c[g][j], p.z, q.z, p.w, q.w, v.z, v.w);
          }
  }
#pragma unroll
  for (int g = 0; g < MT; ++g)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[warp][(8 * j + 2 * t + (e & 1)) * ROWS + g * 16 + gid + 8 * (e >> 1)] = c[g][j][e];
  __syncthreads();
  if (split > 1) {
    cluster_wait();  // the cluster's first CTA is there
    for (int i = threadIdx.x; i < SUMS; i += THREADS) {
      float v = 0.0f;
#pragma unroll
      for (int p = 0; p < WARPS; ++p) v += part[p][i];
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(&recv[rank][i], 0)), "f"(v)
                   : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  }
  if (mine <= 0) return;
  float z[OUTS], u[OUTS];
#pragma unroll
  for (int q = 0; q < OUTS; ++q) {
    const int at = (row + q) * ROWS + f / GROUP * 16 + f % GROUP;
    z[q] = u[q] = 0.0f;
    if (split == 1) {
#pragma unroll
      for (int p = 0; p < WARPS; ++p) {
        z[q] += part[p][at];
        if (EPI == GLU) u[q] += part[p][at + 8];
      }
    } else {
      for (int p = 0; p < split; ++p) {
        z[q] += recv[p][at];
        if (EPI == GLU) u[q] += recv[p][at + 8];
      }
    }
  }
  epilogue_column<EPI, OUTS>(a, row0 + row, mine, col0 + f, z, u);
}

// How many CTAs share a tile's k, and what the kernel takes, in us.
struct Plan {
  int64_t ctas;
  int split;
  float us;
};
template <int EPI>
Plan plan(const Args& a, int mt, int nt, int max_split, float hbm) {
  // Twice the CTAs on the k axis as long as all run at once and every warp keeps
  // two steps (1 x 4096 x 256: 3.2 us unsplit, 2.4 over four; 1 x 2048 x 4096: 3.7
  // unsplit, 6.7 over two).
  const int64_t nb = ((int64_t)a.m + 8 * nt - 1) / (8 * nt);
  const int kt = (a.k + BK - 1) / BK, sms = num_sms();
  Plan p{tiles<EPI>(a.n_out, mt) * nb, 1, 0.0f};
  while (p.split < max_split && p.ctas <= sms && kt >= 4 * p.split * WARPS) {
    p.split *= 2;
    p.ctas *= 2;
  }
  const float v = std::max(1.0f, (float)p.ctas / (float)sms), steps = (float)kt / (float)p.split;
  const float waves = (float)((p.ctas + 2 * sms - 1) / (2 * sms));
  p.us = 1.15f + (mt == 1 ? std::max(1.45f * hbm, waves * 0.042f * steps +
                                                      v * (0.46f + 0.024f * steps))
                          : std::max(2.0f * hbm, waves * 0.09f * steps +
                                                     v * (0.8f + 0.045f * steps)));
  return p;
}

template <int MT, int NT, int U, int MAX_SPLIT, int EPI>
int launch(const void* x, int64_t ldx, const void* w, int64_t ldw, const Plan& p, const Args& a,
           cudaStream_t stream) {
  return check_cuda(overlap_launch(dense_few_kernel<MT, NT, U, MAX_SPLIT, EPI>,
                                   dim3((unsigned)p.ctas), dim3(THREADS), 0, p.split, stream,
                                   static_cast<const uint16_t*>(x), ldx,
                                   static_cast<const uint16_t*>(w), ldw, p.split, a),
                    "dense_matmul launch");
}

}  // namespace few

// The kernel, and how k is split, by what they take, in us. Fitted to times of
// every kernel and split at 169 shapes, k = 64 .. 8192, n = 16 .. 8192, m = 16 ..
// 2048, bf16 out without bias and residual, one launch after another; HBM: w and x at 6.5 TB/s:
//   few, tiles of 16 x 16   1.15 + max(1.45 * HBM, waves * 0.042 * k steps of a CTA
//                                      + CTAs an SM * (0.46 + 0.024 * k steps))
//        tiles of 32 x 32   1.15 + max(2 * HBM, waves * 0.09 * k steps
//                                      + CTAs an SM * (0.8 + 0.045 * k steps))
//   split                  -0.6 + waves * (max(0.22 * k steps, 1.05 * HBM / waves)
//                                          + 2.75 + 2.5 * b (+ 0.85 + 0.8 * b split))
//   pair                    5 + waves * max(0.35 * k steps, 1.33 * HBM / waves)
// b: rows of x in a tile / 128. A wave: two CTAs per SM in the first, one CTA in the
// others: as many clusters as fit (of 8 CTAs fewer than 18, since a cluster stays
// within a GPC). The choice takes 0.5% more than the fastest on average, 25% at
// most. E.g. k = 1000, n = 776: few 2.7 us at m = 48, split 5.4; 5.4 (large tiles)
// and 8.5 at m = 333, 9.5 and 8.6 at 512. k = 2048, n = 4096: split 10.5, pair 15.4
// at m = 256; 25.3 and 17.8 at 1024.
template <int EPI>
int run_epi(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, const Args& a,
            cudaStream_t stream) {
  const int bt = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
  const int feat = EPI == GLU ? TILE_W / 2 : TILE_W, pfeat = EPI == GLU ? 128 : 256;
  const int64_t tiles = (int64_t)((a.n_out + feat - 1) / feat) * ((a.m + bt - 1) / bt);
  const int64_t ptiles = (int64_t)((a.n_out + pfeat - 1) / pfeat) * ((a.m + 255) / 256);
  const int kt = (a.k + BK - 1) / BK;
  auto waves = [](int64_t tiles, int cluster) {
    const int64_t c = resident_clusters(cluster);
    return (float)((tiles + c - 1) / c);
  };
  const float hbm = 2.0f * (float)a.k * ((float)a.m + (float)n) / 6.5e6f;
  const float b = (float)bt / 128.0f;
  int split = 1;
  float best = 0.0f;
  // (An f32 result's parts have to fit a CTA's TMEM.)
  int first = 1;
  while (a.out_f32 && first < MAX_CLUSTER && kt > first * PART_STEPS * (512 / bt)) first *= 2;
  for (int s = first; s <= MAX_CLUSTER && (s == first || kt >= 2 * s); s *= 2) {
    const float v = waves(tiles, s);
    const float t = v * (std::max(0.22f * (float)((kt + s - 1) / s), 1.05f * hbm / v) + 2.75f +
                         2.5f * b + (s > 1 ? 0.85f + 0.8f * b : 0.0f)) -
                    0.6f;
    if (s == first || t < best) {
      best = t;
      split = s;
    }
  }
  const float pv = waves(ptiles, 2);
  const float t_pair = 5.0f + pv * std::max(0.35f * (float)kt, 1.33f * hbm / pv);
  const few::Plan small = few::plan<EPI>(a, 1, a.m <= 8 ? 1 : 2, 8, hbm);
  const few::Plan large = few::plan<EPI>(a, 2, 4, 2, hbm);
  // Up to 8 rows always, of w's rows 16 at a time unless a warp has but one step of
  // many tiles (1 x 512 x 8192: 3.7 us, 2.9 with 32; 1 x 4096 x 4096: 7.1 and 11).
  if (a.m <= 8)
    return kt <= few::WARPS && large.us < small.us
               ? few::launch<2, 4, 1, 2, EPI>(x, ldx, w, ldw, large, a, stream)
               : few::launch<1, 1, 4, 8, EPI>(x, ldx, w, ldw, small, a, stream);
  if (a.m > 64) best = std::min(best, t_pair);
  const few::Plan& least = small.us < large.us ? small : large;
  if (least.us < best && least.ctas <= INT32_MAX)
    return &least == &small ? few::launch<1, 2, 2, 8, EPI>(x, ldx, w, ldw, small, a, stream)
                            : few::launch<2, 4, 1, 2, EPI>(x, ldx, w, ldw, large, a, stream);
  if (a.m > 64 && t_pair == best)
    return !a.out_vec || (a.residual && !a.res_vec)
               ? pair::launch<EPI, false, false>(x, ldx, w, ldw, n, a, stream)
           : a.residual ? pair::launch<EPI, true, true>(x, ldx, w, ldw, n, a, stream)
                        : pair::launch<EPI, true, false>(x, ldx, w, ldw, n, a, stream);
  if (bt == 16) return launch_split<16, EPI>(x, ldx, w, ldw, n, split, a, stream);
  if (bt == 32) return launch_split<32, EPI>(x, ldx, w, ldw, n, split, a, stream);
  if (bt == 64) return launch_split<64, EPI>(x, ldx, w, ldw, n, split, a, stream);
  return launch_split<128, EPI>(x, ldx, w, ldw, n, split, a, stream);
}

int run(const void* x, int64_t ldx, const void* w, int64_t ldw, int n, const Args& a,
        cudaStream_t stream) {
  if (a.act == DWM_ACT_NONE) return run_epi<PLAIN>(x, ldx, w, ldw, n, a, stream);
  if (a.act == DWM_ACT_SWIGLU || a.act == DWM_ACT_SWIGLU_CLAMP)
    return run_epi<GLU>(x, ldx, w, ldw, n, a, stream);
  return run_epi<POINT>(x, ldx, w, ldw, n, a, stream);
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
  // (Coordinates of whole tiles are 32-bit numbers.)
  DWM_CHECK_ARG(std::max({m, n, k}) <= INT32_MAX - 1024, "m=%d n=%d k=%d are too large", m, n, k);
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
  a.bias_vec = bias && addr(bias) % 16 == 0 && (!glu || (int64_t)n_out * bes % 16 == 0);
  a.res_vec = residual && addr(residual) % 16 == 0 && ldr * res % 16 == 0;
  a.out_vec = addr(out) % 16 == 0 && ldo * oes % 16 == 0;
  a.out_wide = addr(out) % 32 == 0 && ldo * oes % 32 == 0;
  a.limit = act_limit;
  a.res_scale = residual_scale;
  a.part_steps = a.tmem_cols = 0;
  a.status = status_ptr();
  return dense::run(x, ldx, w, ldw, n, a, static_cast<cudaStream_t>(stream));
}
