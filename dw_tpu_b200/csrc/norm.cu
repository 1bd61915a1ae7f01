// The norms before and after a block, with the block's gate, its scale and
// the residual's scale, in one pass over the rows:
//
//   r = residual_scale * residual + scale * gate * n2(y)     (after the block)
//   h = n1(r)                                                (before the next)
//
// n1 and n2 are RMS norms, v * rsqrt(mean(v^2) + eps) * w (+ b), or layer
// norms, the same of v - mean(v). Without y there is only h = n1(residual).
// All sums, statistics and products are f32; r and h are each rounded once,
// and h is formed from the f32 r, not from its rounding, so that the fused
// call is no less exact than f32 arithmetic throughout.
//
// Few rows (block_norm_kernel): one CTA takes one row (a warp, rows of up to 1024
// elements), every load of it issued before the first sum. Bound: the launch and
// one memory latency (4096 elements: 1 row 1.8 us, 64 rows with everything 2.7).
//
// Many rows (block_norm_stream_kernel): one CTA per SM, its groups of threads take
// rows in turn from a ring of bulk copies, the rows' vectors in shared memory.
// Bound: memory, a row of each tensor read and written once and kept in registers
// between the two norms: 8192 x 4096 bf16 with both norms and a gate by channel
// 45.8 us (5.9 TB/s; 74 with a CTA a row). Rows that do not start on 16 bytes take
// an element a load, and are bound by instruction issue: 1023 x 5003, layer norms,
// f32 residual, full gate 27.1 us (2.6 TB/s).
#include <algorithm>

#include "common.cuh"

namespace dwm {
namespace norm {

struct Args {
  const void* y;      // NULL: no block output, h = n1(residual)
  const void* res;
  const void* vec[4]; // weight and bias of n2 (inner = 0: n2 is the identity) and of n1
  const void* gate;   // of y's type
  void* r_out;        // NULL without y
  void* h_out;        // NULL: no n1
  int64_t ldy, ldres, ldg, ldr, ldh;  // row strides in elements
  int t, h;
  int inner;          // apply n2
  int layer;          // layer norm, else RMS norm
  int gate_mode;      // DWM_GATE_*
  int y_f32, res_f32, w_f32, h_f32;
  float eps, scale, res_scale;
  // Streaming kernel: a group's ring of stages, and where the residual's and
  // the full gate's rows start in a stage.
  int stages, stage_bytes, off_res, off_gate;
  // Where the vectors lie in its shared memory, a channel's gate the fifth;
  // 0 bytes apart: left in global memory.
  int vec_bytes;
  int* status;
};
constexpr int W2 = 0, B2 = 1, W1 = 2, B1 = 3, CHANNEL_GATE = 4;

// Element types known when the kernel is compiled, or when it runs.
constexpr int BF = 0, FP = 1, ANY = 2;
template <int D>
__device__ __forceinline__ bool is_f32(int runtime) {
  return D == ANY ? runtime != 0 : D == FP;
}
template <int D>
__device__ __forceinline__ int bytes_of(int runtime) {
  return is_f32<D>(runtime) ? 4 : 2;
}

// A thread's loads of a row: CPT of VEC elements, load c at column
// (i + c * threads) * VEC. VEC = 8: 16-byte loads (the host has checked the
// alignment), the threads a run-time number; VEC = 1: an element each, T threads,
// so that the offsets of a thread's loads are constants, the first sure_loads of
// them within the row for every row that the launch gives this CPT.
template <int CPT, int T>
__host__ __device__ constexpr int sure_loads() {
  return T == 512 ? (CPT > 16 ? CPT - 8 : CPT - 2) : T == 128 ? 2 : 0;
}
template <int VEC, int CPT, int T>
struct Cols {
  int h, first;
  int col[VEC == 8 ? CPT : 1];
  bool in_[VEC == 8 ? CPT : 1];

  __device__ __forceinline__ Cols(int h, int i, int threads) : h(h), first(i) {
    if constexpr (VEC == 8) {
      // Loads past the row's end read its first elements, which nothing uses.
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        col[c] = (i + c * threads) * VEC;
        in_[c] = col[c] < h;  // h is a multiple of VEC
        if (!in_[c]) col[c] = 0;
      }
    }
  }
  __device__ __forceinline__ int at(int c) const {
    return VEC == 8 ? col[c % (VEC == 8 ? CPT : 1)] : first + c * T;
  }
  __device__ __forceinline__ bool in(int c) const {
    return VEC == 8 ? in_[c % (VEC == 8 ? CPT : 1)]
                    : c < sure_loads<CPT, T>() || first + c * T < h;
  }
};

// Its elements are worked on in pairs: two neighbours of a load, or (VEC = 1)
// those of two loads. Elements past the end of the row are 0 with VEC = 1.
__host__ __device__ constexpr int pairs(int vec, int cpt) { return vec == 8 ? 4 * cpt : cpt / 2; }

// The elements as they were loaded.
template <int VEC, int CPT, int T, int D>
struct Raw {
  static constexpr int W = VEC == 1 ? 1 : D == BF ? 4 : 8;  // words per load
  static constexpr int NP = pairs(VEC, CPT);
  using C = Cols<VEC, CPT, T>;
  uint32_t u[CPT][W];

  // From global memory. One branch on the type for all loads, so that they
  // are issued together.
  __device__ __forceinline__ void load(const void* p, const C& cols, int f32) {
    if (is_f32<D>(f32)) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const uint8_t* q = static_cast<const uint8_t*>(p) + cols.at(c) * 4;
        if constexpr (VEC == 1) {
          u[c][0] = cols.in(c) ? *reinterpret_cast<const uint32_t*>(q) : 0u;
        } else {
          put(c, 0, *reinterpret_cast<const uint4*>(q));
          put(c, 4, *reinterpret_cast<const uint4*>(q + 16));
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const uint8_t* q = static_cast<const uint8_t*>(p) + cols.at(c) * 2;
        if constexpr (VEC == 1)
          u[c][0] = cols.in(c) ? *reinterpret_cast<const uint16_t*>(q) : 0u;
        else
          put(c, 0, *reinterpret_cast<const uint4*>(q));
      }
    }
  }
  // From shared memory.
  __device__ __forceinline__ void load_s(uint32_t p, const C& cols, int f32) {
    if (is_f32<D>(f32)) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const uint32_t q = p + (uint32_t)cols.at(c) * 4;
        if constexpr (VEC == 1) {
          u[c][0] = cols.in(c) ? lds_u32(q) : 0u;
        } else {
          put(c, 0, lds_u128(q));
          put(c, 4, lds_u128(q + 16));
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const uint32_t q = p + (uint32_t)cols.at(c) * 2;
        if constexpr (VEC == 1)
          u[c][0] = cols.in(c) ? lds_u16(q) : 0u;
        else
          put(c, 0, lds_u128(q));
      }
    }
  }
  __device__ __forceinline__ void put(int c, int w, const uint4& x) {
    u[c][w % W] = x.x; u[c][(w + 1) % W] = x.y; u[c][(w + 2) % W] = x.z; u[c][(w + 3) % W] = x.w;
  }
  template <bool F>
  __device__ __forceinline__ F2 at(int p) const {
    if constexpr (VEC == 1) {
      const uint32_t a = u[2 * p][0], b = u[2 * p + 1][0];
      return F ? f2(__uint_as_float(a), __uint_as_float(b))
               : f2(__uint_as_float(a << 16), __uint_as_float(b << 16));
    } else {
      const int c = p / 4, j = p % 4;
      if (F) return f2(__uint_as_float(u[c][(2 * j) % W]), __uint_as_float(u[c][(2 * j + 1) % W]));
      return f2(__uint_as_float(u[c][j] << 16), __uint_as_float(u[c][j] & 0xFFFF0000u));
    }
  }
  // v <- f(v, elements) for all pairs; again one branch on the type.
  template <class F>
  __device__ __forceinline__ void into(F2 (&v)[NP], int f32, const F& f) const {
    if (is_f32<D>(f32)) {
#pragma unroll
      for (int p = 0; p < NP; ++p) v[p] = f(v[p], at<true>(p));
    } else {
#pragma unroll
      for (int p = 0; p < NP; ++p) v[p] = f(v[p], at<false>(p));
    }
  }
};

// The pairs to their places in the row at `row`.
template <int VEC, int CPT, int T>
__device__ __forceinline__ void store(uint8_t* row, bool f32, const Cols<VEC, CPT, T>& cols,
                                      const F2 (&v)[pairs(VEC, CPT)]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if (!cols.in(c)) continue;
      float e[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) f2_split(v[4 * c + q], e[2 * q], e[2 * q + 1]);
      if (f32) {
        float4* q = reinterpret_cast<float4*>(row + cols.at(c) * 4);
        q[0] = make_float4(e[0], e[1], e[2], e[3]);
        q[1] = make_float4(e[4], e[5], e[6], e[7]);
      } else {
        *reinterpret_cast<uint4*>(row + cols.at(c) * 2) =
            make_uint4(f32x2_to_bf16x2(e[0], e[1]), f32x2_to_bf16x2(e[2], e[3]),
                       f32x2_to_bf16x2(e[4], e[5]), f32x2_to_bf16x2(e[6], e[7]));
      }
    }
  } else {
    if (f32) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        float e[2];
        f2_split(v[c / 2], e[0], e[1]);
        if (cols.in(c)) *reinterpret_cast<float*>(row + cols.at(c) * 4) = e[c % 2];
      }
    } else {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        float e[2];
        f2_split(v[c / 2], e[0], e[1]);
        if (cols.in(c))
          *reinterpret_cast<uint16_t*>(row + cols.at(c) * 2) = (uint16_t)f32_to_bf16_bits(e[c % 2]);
      }
    }
  }
}

// The threads that share a row: threads() of them (T if not 0) (whole warps), this one the
// `i`-th, barrier `bar` theirs alone. part: one slot a warp for each of a
// row's (at most four) sums, so one barrier a sum is enough; 16-byte aligned,
// the slots of absent warps zero.
template <int T>
struct Group {
  int i, run_threads, bar;
  float (*part)[32];

  __device__ __forceinline__ int threads() const { return T ? T : run_threads; }
  __device__ __forceinline__ void sync() const {
    if (threads() == 32)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads()) : "memory");
  }
  __device__ __forceinline__ void clear_parts() const {
    for (int j = i; j < 128; j += threads()) part[j / 32][j % 32] = 0.0f;
  }
  // Sum over the row's threads, in a fixed order: the same bits in all of
  // them. between() runs after the barrier (with one warp a row: none).
  template <class F>
  __device__ __forceinline__ float sum(float v, int slot, const F& between) const {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threads() == 32) {
      between();
      return v;
    }
    if ((i & 31) == 0) part[slot][i >> 5] = v;
    sync();
    between();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < threads(); w += 128) {
      const float4 p = *reinterpret_cast<const float4*>(&part[slot][w / 32]);
      s += (p.x + p.y) + (p.z + p.w);
    }
    return s;
  }
};

// u <- norm(u) * w + b over a row. read_done() runs once every thread of the
// row has all of its elements of u.
template <int VEC, int CPT, int T, int WD, class Vec, class Done>
__device__ __forceinline__ void normalise(F2 (&u)[pairs(VEC, CPT)], const Cols<VEC, CPT, T>& cols,
                                          const Args& a, const Group<T>& g, int slot, float inv_h,
                                          const Vec& vec, int weight, int bias,
                                          const Done& read_done) {
  constexpr int NP = pairs(VEC, CPT);
  auto total = [](F2 x) {
    float lo, hi;
    f2_split(x, lo, hi);
    return lo + hi;
  };
  // (VEC = 1: what is past the end is 0.)
  auto in = [&](int p) { return VEC == 1 || cols.in(p / 4); };
  if (a.layer) {
    F2 s = f2(0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (in(p)) s = f2_add(s, u[p]);
    const float mean = g.sum(total(s), slot, [] {}) * inv_h;
    const F2 minus = f2(-mean, -mean);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      u[p] = f2_add(u[p], minus);
      if (VEC == 1 && 2 * p + 1 >= sure_loads<CPT, T>()) {
        float lo, hi;
        f2_split(u[p], lo, hi);
        u[p] = f2(cols.in(2 * p) ? lo : 0.0f, cols.in(2 * p + 1) ? hi : 0.0f);
      }
    }
  }
  F2 s2 = f2(0.0f, 0.0f);
#pragma unroll
  for (int p = 0; p < NP; ++p)
    if (in(p)) s2 = f2_fma(u[p], u[p], s2);
  const float rstd = rsqrtf(g.sum(total(s2), slot + 1, read_done) * inv_h + a.eps);
  const F2 rstd2 = f2(rstd, rstd);
  vec(weight, [&](const Raw<VEC, CPT, T, WD>& w) {
    w.into(u, a.w_f32, [&](F2 v, F2 x) { return f2_mul(f2_mul(v, rstd2), x); });
  });
  if (a.vec[bias])
    vec(bias, [&](const Raw<VEC, CPT, T, WD>& b) {
      b.into(u, a.w_f32, [](F2 v, F2 x) { return f2_add(v, x); });
    });
}

// One row: both norms, gate, residual, stores. y, res, gate and vec (a weight
// or bias) are functions that hand their loaded elements on: from registers
// where the caller has loaded them ahead, or from where they lie. r_out and
// h_out point to the row. slot: of the sums of n1 (n2's have 0 and 1). read_done()
// runs once every thread has the row's elements.
template <int VEC, int CPT, int T, int YD, int RD, int WD, class Y, class Res, class Gate,
          class Vec, class Done>
__device__ __forceinline__ void do_row(const Args& a, const Group<T>& g, int slot, uint8_t* r_out,
                                       uint8_t* h_out, float inv_h,
                                       const Cols<VEC, CPT, T>& cols, float gate_tok, const Y& y,
                                       const Res& res, const Gate& gate, const Vec& vec,
                                       const Done& read_done) {
  using RawY = Raw<VEC, CPT, T, YD>;
  using RawR = Raw<VEC, CPT, T, RD>;
  F2 v[pairs(VEC, CPT)];
  if (a.y) {
    y([&](const RawY& x) { x.into(v, a.y_f32, [](F2, F2 e) { return e; }); });
    if (a.inner)
      normalise<VEC, CPT, T, WD>(v, cols, a, g, 0, inv_h, vec, W2, B2, [] {});
    if (a.gate_mode >= DWM_GATE_CHANNEL)
      gate([&](const RawY& x) { x.into(v, a.y_f32, [](F2 u, F2 e) { return f2_mul(u, e); }); });
    const F2 scale = f2(a.scale * gate_tok, a.scale * gate_tok);
    const F2 res_scale = f2(a.res_scale, a.res_scale);
    res([&](const RawR& x) {
      x.into(v, a.res_f32, [&](F2 u, F2 e) { return f2_fma(scale, u, f2_mul(res_scale, e)); });
    });
    store<VEC, CPT, T>(r_out, is_f32<RD>(a.res_f32), cols, v);
  } else {
    res([&](const RawR& x) { x.into(v, a.res_f32, [](F2, F2 e) { return e; }); });
  }
  if (a.h_out) {
    normalise<VEC, CPT, T, WD>(v, cols, a, g, slot, inv_h, vec, W1, B1, read_done);
    store<VEC, CPT, T>(h_out, a.h_f32 != 0, cols, v);
  } else {
    g.sync();
    read_done();
  }
}

template <int YD>
__device__ __forceinline__ float token_gate(const Args& a, int64_t row) {
  if (a.gate_mode != DWM_GATE_TOKEN) return 1.0f;
  return is_f32<YD>(a.y_f32)
             ? static_cast<const float*>(a.gate)[row * a.ldg]
             : bf16_bits_to_f32(static_cast<const uint16_t*>(a.gate)[row * a.ldg]);
}

__device__ __forceinline__ const uint8_t* row_ptr(const void* p, int64_t row, int64_t ld, int es) {
  return static_cast<const uint8_t*>(p) + row * ld * es;
}
__device__ __forceinline__ uint8_t* row_ptr(void* p, int64_t row, int64_t ld, int es) {
  return static_cast<uint8_t*>(p) + row * ld * es;
}

// The most threads of a CTA: those that a row of MAX_H needs, and in the
// streaming kernel 1024 (64 registers each) unless a thread has 32 elements.
template <int VEC, int CPT>
constexpr int max_threads(bool stream) {
  return VEC * CPT > 16 || !stream ? 512 : 1024;
}

// A few rows: one group a row, every load of a row issued before its first
// sum, so that a row costs one memory latency. threadIdx.y: the CTA's groups.
template <int VEC, int CPT, int T, int YD, int RD, int WD>
__global__ void __launch_bounds__(max_threads<VEC, CPT>(false)) block_norm_kernel(const Args a) {
  __shared__ __align__(16) float part[4][32];
  const Group<T> g{(int)threadIdx.x, (int)blockDim.x, 0, part};
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  overlap_wait();
  overlap_next();
  if (row >= a.t) return;  // a whole warp of a CTA with a warp a row
  const Cols<VEC, CPT, T> cols(a.h, g.i, g.threads());
  const int ye = bytes_of<YD>(a.y_f32), re = bytes_of<RD>(a.res_f32);
  const uint8_t* pg = row_ptr(a.gate, a.gate_mode == DWM_GATE_FULL ? row : 0, a.ldg, ye);
  // Up to 16 elements a thread everything is loaded ahead; the gate and the
  // weights of more would not fit the registers.
  constexpr bool AHEAD = VEC == 8 && CPT <= 2;
  Raw<VEC, CPT, T, YD> y, gate;
  Raw<VEC, CPT, T, RD> res;
  Raw<VEC, CPT, T, WD> w2, w1;
  if (a.y) y.load(row_ptr(a.y, row, a.ldy, ye), cols, a.y_f32);
  res.load(row_ptr(a.res, row, a.ldres, re), cols, a.res_f32);
  if (AHEAD) {
    if (a.inner) w2.load(a.vec[W2], cols, a.w_f32);
    if (a.gate_mode >= DWM_GATE_CHANNEL) gate.load(pg, cols, a.y_f32);
    if (a.h_out) w1.load(a.vec[W1], cols, a.w_f32);
  }
  const float tok = token_gate<YD>(a, row);
  if (g.threads() > 32) {
    g.clear_parts();
    g.sync();
  }
  do_row<VEC, CPT, T, YD, RD, WD>(
      a, g, 2, row_ptr(a.r_out, row, a.ldr, re), row_ptr(a.h_out, row, a.ldh, a.h_f32 ? 4 : 2),
      1.0f / (float)a.h, cols, tok, [&](auto f) { f(y); }, [&](auto f) { f(res); },
      [&](auto f) {
        if (!AHEAD) gate.load(pg, cols, a.y_f32);
        f(gate);
      },
      [&](int which, auto f) {
        if (AHEAD && which == W2) {
          f(w2);
        } else if (AHEAD && which == W1) {
          f(w1);
        } else {
          Raw<VEC, CPT, T, WD> x;
          x.load(a.vec[which], cols, a.w_f32);
          f(x);
        }
      },
      [] {});
}

// Many rows: one CTA an SM, its groups taking rows in turn. A group's first
// thread keeps a ring of bulk copies (cp.async.bulk) of its next rows of y,
// residual and full gate in flight, so that the memory is busy while the group
// sums and stores. The vectors that all rows share lie in shared memory (the
// ring leaves the L1 cache too small for them). A row whose bytes do not start on 16 is copied from
// the 16-byte granule it starts in to the one it ends in.
__device__ __forceinline__ uint32_t bulk_bytes(const uint8_t* p, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  return (uint32_t)(((at + bytes + 15) & ~15ull) - (at & ~15ull));
}
__device__ __forceinline__ void bulk_row(uint32_t dst, const uint8_t* p, int bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(p) & ~15ull), "r"(bulk_bytes(p, bytes)), "r"(smem_u32(bar))
      : "memory");
}

constexpr int MAX_STAGES = 8;
constexpr int MAX_GROUPS = 16;

template <int VEC, int CPT, int T, int YD, int RD, int WD>
__global__ void __launch_bounds__(max_threads<VEC, CPT>(true), 1)
    block_norm_stream_kernel(const Args a) {
  __shared__ __align__(16) float part[MAX_GROUPS][4][32];
  __shared__ uint64_t full[MAX_GROUPS][MAX_STAGES];
  __shared__ int abort_word;
  extern __shared__ __align__(16) uint8_t ring[];
  volatile int* abort_flag = &abort_word;
  const int gi = threadIdx.y, groups = blockDim.y;
  const Group<T> g{(int)threadIdx.x, (int)blockDim.x, gi, part[gi]};
  const uint32_t vectors = smem_u32(ring);
  const uint32_t stages =
      vectors + (uint32_t)(5 * a.vec_bytes + gi * a.stages * a.stage_bytes);
  if (g.i == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(&full[gi][s], 1);
    fence_mbar_init();
    *abort_flag = 0;
  }
  g.clear_parts();
  __syncthreads();
  overlap_wait();
  overlap_next();
  const Cols<VEC, CPT, T> cols(a.h, g.i, g.threads());
  const float inv_h = 1.0f / (float)a.h;
  const int64_t first = (int64_t)blockIdx.x * groups + gi, step = (int64_t)gridDim.x * groups;
  const bool full_gate = a.gate_mode == DWM_GATE_FULL;
  const int ye = bytes_of<YD>(a.y_f32), re = bytes_of<RD>(a.res_f32), he = a.h_f32 ? 4 : 2;
  auto fetch = [&](int64_t row, int s) {
    const uint8_t* py = row_ptr(a.y, row, a.ldy, ye);
    const uint8_t* pr = row_ptr(a.res, row, a.ldres, re);
    const uint8_t* pg = row_ptr(a.gate, row, a.ldg, ye);
    uint32_t bytes = bulk_bytes(pr, a.h * re);
    if (a.y) bytes += bulk_bytes(py, a.h * ye);
    if (full_gate) bytes += bulk_bytes(pg, a.h * ye);
    uint64_t* bar = &full[gi][s];
    const uint32_t dst = stages + (uint32_t)(s * a.stage_bytes);
    mbar_arrive_expect_tx(bar, bytes);
    if (a.y) bulk_row(dst, py, a.h * ye, bar);
    bulk_row(dst + a.off_res, pr, a.h * re, bar);
    if (full_gate) bulk_row(dst + a.off_gate, pg, a.h * ye, bar);
  };
  if (g.i == 0)
    for (int s = 0; s < a.stages; ++s)
      if (first + s * step < a.t) fetch(first + s * step, s);
  if (a.vec_bytes) {
    // 16 bytes a load, or an element a load where they are not aligned.
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const void* p = j < 4 ? a.vec[j] : a.gate_mode == DWM_GATE_CHANNEL ? a.gate : nullptr;
      const int es = j < 4 ? bytes_of<WD>(a.w_f32) : ye;
      if (!p) continue;
      uint8_t* dst = ring + j * a.vec_bytes;
      const int tid = gi * g.threads() + g.i, threads = groups * g.threads();
      if (VEC == 8) {
        for (int i = tid; i < a.h * es / 16; i += threads)
          reinterpret_cast<uint4*>(dst)[i] = static_cast<const uint4*>(p)[i];
      } else if (es == 4) {
        for (int i = tid; i < a.h; i += threads)
          reinterpret_cast<uint32_t*>(dst)[i] = static_cast<const uint32_t*>(p)[i];
      } else {
        for (int i = tid; i < a.h; i += threads)
          reinterpret_cast<uint16_t*>(dst)[i] = static_cast<const uint16_t*>(p)[i];
      }
    }
    __syncthreads();
  }
  int s = 0, slot = 2;
  uint32_t ph = 0;
  uint8_t* r_out = row_ptr(a.r_out, first, a.ldr, re);
  uint8_t* h_out = row_ptr(a.h_out, first, a.ldh, he);
  for (int64_t row = first; row < a.t; row += step) {
    const float tok = token_gate<YD>(a, row);
    // After a wait that ran out (reported in the status word) the rows are not
    // what they should be, but the group stays together.
    mbar_wait(&full[gi][s], ph, abort_flag, a.status);
    const uint32_t at = stages + (uint32_t)(s * a.stage_bytes);
    // Where the row's first byte sits in its first granule.
    auto lead = [&](const void* p, int64_t ld, int es) {
      return VEC == 8 ? 0u : (uint32_t)reinterpret_cast<uint64_t>(row_ptr(p, row, ld, es)) & 15u;
    };
    do_row<VEC, CPT, T, YD, RD, WD>(
        a, g, slot, r_out, h_out, inv_h, cols, tok,
        [&](auto f) {
          Raw<VEC, CPT, T, YD> x;
          x.load_s(at + lead(a.y, a.ldy, ye), cols, a.y_f32);
          f(x);
        },
        [&](auto f) {
          Raw<VEC, CPT, T, RD> x;
          x.load_s(at + a.off_res + lead(a.res, a.ldres, re), cols, a.res_f32);
          f(x);
        },
        [&](auto f) {
          if (full_gate) {
            Raw<VEC, CPT, T, YD> x;
            x.load_s(at + a.off_gate + lead(a.gate, a.ldg, ye), cols, a.y_f32);
            f(x);
          } else {
            Raw<VEC, CPT, T, YD> x;
            if (a.vec_bytes)
              x.load_s(vectors + CHANNEL_GATE * a.vec_bytes, cols, a.y_f32);
            else
              x.load(a.gate, cols, a.y_f32);
            f(x);
          }
        },
        [&](int which, auto f) {
          Raw<VEC, CPT, T, WD> x;
          if (a.vec_bytes)
            x.load_s(vectors + which * a.vec_bytes, cols, a.w_f32);
          else
            x.load(a.vec[which], cols, a.w_f32);
          f(x);
        },
        [&] {
          if (g.i == 0 && row + a.stages * step < a.t) fetch(row + a.stages * step, s);
        });
    r_out += step * a.ldr * re;
    h_out += step * a.ldh * he;
    // An RMS norm without n2 has one barrier a row: a warp that is ahead must not
    // write its next sum where another still reads this row's.
    if (!a.inner) slot ^= 2;
    if (++s == a.stages) { s = 0; ph ^= 1; }
  }
  // A copy that a wait gave up on lands before the exit.
  if (g.i == 0 && *abort_flag)
    for (int i = 0; i < a.stages; ++i) mbar_wait(&full[gi][i], ph ^ (i >= s), nullptr, a.status);
}

template <int VEC, int CPT, int T, int YD, int RD, int WD>
int launch(Args a, cudaStream_t s) {
  const int n = (a.h + VEC - 1) / VEC;  // loads a row
  // A group: as many warps as the row takes with CPT loads a thread.
  const int threads = T ? T : ((n + CPT - 1) / CPT + 31) / 32 * 32;
  const int groups = std::min(MAX_GROUPS, max_threads<VEC, CPT>(true) / threads);
  if ((int64_t)a.t > 2 * (int64_t)num_sms() * groups) {
    auto room = [&](int f32) { return (a.h * (f32 ? 4 : 2) + 15) / 16 * 16 + (VEC == 1 ? 16 : 0); };
    a.off_res = a.y ? room(a.y_f32) : 0;
    a.off_gate = a.off_res + room(a.res_f32);
    a.stage_bytes = a.off_gate + (a.gate_mode == DWM_GATE_FULL ? room(a.y_f32) : 0);
    const int budget = 208 * 1024;
    a.vec_bytes = (a.h * std::max(a.w_f32 ? 4 : 2, a.y_f32 ? 4 : 2) + 15) / 16 * 16;
    if (5 * a.vec_bytes + 2 * groups * a.stage_bytes > budget) a.vec_bytes = 0;
    const int left = budget - 5 * a.vec_bytes;
    a.stages = std::min(MAX_STAGES, left / (groups * a.stage_bytes));
    if (a.stages >= 2) {
      auto fn = block_norm_stream_kernel<VEC, CPT, T, YD, RD, WD>;
      const int rc = set_smem_limit(reinterpret_cast<const void*>(fn), budget, "norm smem attribute");
      if (rc) return rc;
      a.status = status_ptr();
      return check_cuda(
          overlap_launch(fn, dim3((unsigned)num_sms()), dim3((unsigned)threads, (unsigned)groups),
                         (size_t)5 * a.vec_bytes + (size_t)groups * a.stages * a.stage_bytes, 1, s,
                         a),
          "block_norm launch");
    }
  }
  // A warp a row, four a CTA, or a CTA a row.
  const int rows = threads == 32 ? 4 : 1;
  return check_cuda(overlap_launch(block_norm_kernel<VEC, CPT, T, YD, RD, WD>,
                                   dim3((unsigned)((a.t + rows - 1) / rows)),
                                   dim3((unsigned)threads, (unsigned)rows), 0, 1, s, a),
                    "block_norm launch");
}

template <int VEC, int YD, int RD, int WD>
int by_width(const Args& a, cudaStream_t s) {
  const int n = (a.h + VEC - 1) / VEC;
  const bool many = a.t > 2 * num_sms();
  if constexpr (VEC == 8) {
    // Few rows: a load a thread.
    if (n <= 32 || (!many && n <= 512)) return launch<8, 1, 0, YD, RD, WD>(a, s);
    if (n <= 1024) return launch<8, 2, 0, YD, RD, WD>(a, s);
    return launch<8, 4, 0, YD, RD, WD>(a, s);
  } else {
    // (sure_loads goes by these.)
    if (n <= 32 * 8) return launch<1, 8, 32, YD, RD, WD>(a, s);
    if (n <= 128 * 8) return launch<1, 8, 128, YD, RD, WD>(a, s);
    if (n <= 512 * 4) return launch<1, 4, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 6) return launch<1, 6, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 8) return launch<1, 8, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 10) return launch<1, 10, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 12) return launch<1, 12, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 14) return launch<1, 14, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 16) return launch<1, 16, 512, YD, RD, WD>(a, s);
    if (n <= 512 * 24) return launch<1, 24, 512, YD, RD, WD>(a, s);
    return launch<1, 32, 512, YD, RD, WD>(a, s);
  }
}

// Rows of at most 32 elements a thread of 512.
constexpr int MAX_H = 16384;

int run(const Args& a, bool vec, cudaStream_t s) {
  // (Types known when the kernel is compiled gained rows without VEC 1%.)
  if (!vec) return by_width<1, ANY, ANY, ANY>(a, s);
#define DWM_NORM(YD, RD, WD)                                                               \
  if ((a.y_f32 != 0) == (YD == FP) && (a.res_f32 != 0) == (RD == FP) &&                    \
      (a.w_f32 != 0) == (WD == FP))                                                        \
    return by_width<8, YD, RD, WD>(a, s);
  DWM_NORM(BF, BF, BF)
  DWM_NORM(BF, BF, FP)
  DWM_NORM(BF, FP, BF)
  DWM_NORM(BF, FP, FP)
  DWM_NORM(FP, BF, BF)
  DWM_NORM(FP, BF, FP)
  DWM_NORM(FP, FP, BF)
  DWM_NORM(FP, FP, FP)
#undef DWM_NORM
  return set_error(DWM_ERR_UNSUPPORTED, "norm dtype combination");
}

}  // namespace norm
}  // namespace dwm

using namespace dwm;

extern "C" int dwm_block_norm(const void* y, int y_dtype, int64_t ldy, const void* residual,
                              int residual_dtype, int64_t ldres, int t, int h, int kind,
                              float eps, int inner, const void* w2, const void* b2,
                              const void* gate, int gate_mode, int64_t ldg,
                              float scale, float residual_scale, const void* w1, const void* b1,
                              int w_dtype, void* r_out, int64_t ldr, void* h_out, int h_dtype,
                              int64_t ldh, void* stream) {
  auto is_float = [](int d) { return d == DWM_BF16 || d == DWM_F32; };
  auto es = [](int d) { return d == DWM_F32 ? 4 : 2; };
  DWM_CHECK_ARG(t >= 0 && h >= 1, "bad shape t=%d h=%d", t, h);
  DWM_CHECK_ARG(h <= norm::MAX_H, "h=%d exceeds %d", h, norm::MAX_H);
  DWM_CHECK_ARG(kind == DWM_NORM_RMS || kind == DWM_NORM_LAYER, "unknown norm kind %d", kind);
  DWM_CHECK_ARG(eps > 0.0f, "eps must be positive");
  DWM_CHECK_ARG(is_float(residual_dtype) && is_float(w_dtype) && is_float(h_dtype) &&
                    (!y || is_float(y_dtype)),
                "dtypes must be bf16 or f32");
  DWM_CHECK_ARG(gate_mode >= DWM_GATE_NONE && gate_mode <= DWM_GATE_FULL &&
                    (gate_mode == DWM_GATE_NONE) == (gate == nullptr),
                "bad gate mode %d", gate_mode);
  if (t == 0) return DWM_OK;
  DWM_CHECK_ARG(residual, "NULL residual");
  if (y) {
    DWM_CHECK_ARG(r_out, "NULL r_out");
    DWM_CHECK_ARG(!inner || w2, "the norm after the block needs its weight");
  } else {
    DWM_CHECK_ARG(!r_out && !gate && !inner && h_out,
                  "without y there is only h = norm(residual)");
  }
  DWM_CHECK_ARG(!h_out || w1, "the norm before the next block needs its weight");
  auto aligned = [&](const void* p, int d) { return reinterpret_cast<uintptr_t>(p) % es(d) == 0; };
  DWM_CHECK_ARG((!y || aligned(y, y_dtype)) && (!gate || aligned(gate, y_dtype)) &&
                    aligned(residual, residual_dtype) && aligned(r_out, residual_dtype) &&
                    aligned(h_out, h_dtype) && aligned(w1, w_dtype) && aligned(b1, w_dtype) &&
                    aligned(w2, w_dtype) && aligned(b2, w_dtype),
                "misaligned pointer");
  DWM_CHECK_ARG((!y || ldy >= h || t == 1) && (ldres >= h || t == 1) &&
                    (!r_out || ldr >= h || t == 1) && (!h_out || ldh >= h || t == 1) &&
                    (gate_mode != DWM_GATE_FULL || ldg >= h || t == 1) &&
                    (gate_mode != DWM_GATE_TOKEN || ldg >= 1 || t == 1),
                "a row stride is shorter than a row");
  // Every thread reads its elements of a row before it writes them, so an
  // output may be one of the row inputs in place, element for element;
  // anything else that overlaps an output is refused.
  {
    const RowSpan r = row_span(r_out, t, h, ldr, es(residual_dtype));
    const RowSpan ho = row_span(h_out, t, h, ldh, es(h_dtype));
    struct In {
      const void* p;
      int64_t ld;
      int es;
    };
    const In ins[3] = {{y, ldy, es(y_dtype)},
                       {residual, ldres, es(residual_dtype)},
                       {gate_mode == DWM_GATE_FULL ? gate : nullptr, ldg, es(y_dtype)}};
    DWM_CHECK_ARG(!rows_overlap(r, ho), "the two outputs overlap");
    for (const In& i : ins) {
      const RowSpan in = row_span(i.p, t, h, i.ld, i.es);
      const bool same_r = i.p == r_out && (i.ld == ldr || t == 1) && i.es == es(residual_dtype);
      const bool same_h = i.p == h_out && (i.ld == ldh || t == 1) && i.es == es(h_dtype);
      DWM_CHECK_ARG(same_r || !rows_overlap(in, r),
                    "r_out overlaps an input without being that input");
      DWM_CHECK_ARG(same_h || !rows_overlap(in, ho),
                    "h_out overlaps an input without being that input");
    }
    const RowSpan vecs[5] = {
        row_span(w2, 1, h, h, es(w_dtype)), row_span(b2, 1, h, h, es(w_dtype)),
        row_span(w1, 1, h, h, es(w_dtype)), row_span(b1, 1, h, h, es(w_dtype)),
        gate_mode == DWM_GATE_CHANNEL ? row_span(gate, 1, h, h, es(y_dtype))
                                      : row_span(gate_mode == DWM_GATE_TOKEN ? gate : nullptr, t,
                                                 1, ldg, es(y_dtype))};
    for (const RowSpan& v : vecs)
      DWM_CHECK_ARG(!rows_overlap(v, r) && !rows_overlap(v, ho),
                    "an output overlaps a weight or the gate");
  }
  // 16-byte loads where every row of every tensor starts on 16 bytes.
  auto rows16 = [&](const void* p, int64_t ld, int d) {
    return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (t == 1 || ld * es(d) % 16 == 0));
  };
  const bool vec = h % 8 == 0 && rows16(y, ldy, y_dtype) && rows16(residual, ldres, residual_dtype) &&
                   rows16(r_out, ldr, residual_dtype) && rows16(h_out, ldh, h_dtype) &&
                   rows16(w1, 0, w_dtype) && rows16(b1, 0, w_dtype) && rows16(w2, 0, w_dtype) &&
                   rows16(b2, 0, w_dtype) &&
                   (gate_mode < DWM_GATE_CHANNEL ||
                    rows16(gate, gate_mode == DWM_GATE_FULL ? ldg : 0, y_dtype));
  norm::Args a;
  a.y = y;
  a.res = residual;
  a.vec[norm::W2] = w2;
  a.vec[norm::B2] = b2;
  a.vec[norm::W1] = w1;
  a.vec[norm::B1] = b1;
  a.gate = gate;
  a.r_out = r_out;
  a.h_out = h_out;
  a.ldy = ldy;
  a.ldres = ldres;
  a.ldg = ldg;
  a.ldr = ldr;
  a.ldh = ldh;
  a.t = t;
  a.h = h;
  a.inner = inner != 0;
  a.layer = kind == DWM_NORM_LAYER;
  a.gate_mode = gate_mode;
  a.y_f32 = y && y_dtype == DWM_F32;
  a.res_f32 = residual_dtype == DWM_F32;
  a.w_f32 = w_dtype == DWM_F32;
  a.h_f32 = h_dtype == DWM_F32;
  a.eps = eps;
  a.scale = scale;
  a.res_scale = residual_scale;
  a.stages = a.stage_bytes = a.off_res = a.off_gate = a.vec_bytes = 0;
  a.status = nullptr;
  return norm::run(a, vec, static_cast<cudaStream_t>(stream));
}
