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
// Bound: memory. A row of each tensor is read once and written once, and
// stays in registers between the two norms. One CTA takes one row (a warp,
// rows of up to 1024 elements), each thread up to 32 of its elements.
#include "common.cuh"

namespace dwm {
namespace norm {

struct Args {
  const void* y;      // NULL: no block output, h = n1(residual)
  const void* res;
  const void* w2;     // n2's weight and bias; inner = 0: n2 is the identity
  const void* b2;
  const void* w1;     // n1's
  const void* b1;
  const void* gate;
  void* r_out;        // NULL without y
  void* h_out;        // NULL: no n1
  int64_t ldy, ldres, ldg, ldr, ldh;  // row strides in elements
  int t, h;
  int inner;          // apply n2
  int layer;          // layer norm, else RMS norm
  int gate_mode;      // DWM_GATE_*
  int w_f32, gate_f32, h_f32;
  float eps, scale, res_scale;
};

__device__ __forceinline__ float ld1(const void* p, int64_t i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i]
             : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// N consecutive elements as f32. N = 8: 16-byte loads (the caller has checked
// the alignment); N = 1: one element.
template <int N>
__device__ __forceinline__ void ld(const void* p, int64_t i, bool f32, float (&v)[N]) {
  if constexpr (N == 8) {
    if (f32) {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      const float4 a = q[0], b = q[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
      }
    }
  } else {
    v[0] = ld1(p, i, f32);
  }
}

template <int N>
__device__ __forceinline__ void st(void* p, int64_t i, bool f32, const float (&v)[N]) {
  if constexpr (N == 8) {
    if (f32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 q;
      q.x = f32_to_bf16_bits(v[0]) | (f32_to_bf16_bits(v[1]) << 16);
      q.y = f32_to_bf16_bits(v[2]) | (f32_to_bf16_bits(v[3]) << 16);
      q.z = f32_to_bf16_bits(v[4]) | (f32_to_bf16_bits(v[5]) << 16);
      q.w = f32_to_bf16_bits(v[6]) | (f32_to_bf16_bits(v[7]) << 16);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = q;
    }
  } else {
    if (f32)
      static_cast<float*>(p)[i] = v[0];
    else
      static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(v[0]);
  }
}

// Sum over the threads of one row: a warp (warps == 1), or the whole CTA by
// way of `part` (one slot a warp; summed in warp order by every thread, so
// all threads hold the same bits). Each sum of a row has a `part` of its own,
// so one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, int warps, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int w = 0; w < warps; ++w) s += part[w];
  return s;
}

// VEC elements a load (8, or 1 for rows that are not 16-byte aligned), CPT
// loads a thread: thread i of the row's TPR threads holds elements
// (i + c * TPR) * VEC + [0, VEC). YF / RF: y and the residual are f32.
template <int VEC, int CPT, bool YF, bool RF>
__global__ void __launch_bounds__(512) block_norm_kernel(const Args a) {
  __shared__ float part[4][32];
  const int tpr = blockDim.x, warps = tpr >> 5;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.t) return;  // whole warps of a one-warp-per-row CTA
  const bool layer = a.layer != 0;
  const float inv_h = 1.0f / (float)a.h;
  bool in[CPT];
  int col[CPT];
  float v[CPT][VEC], res[CPT][VEC];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    col[c] = ((int)threadIdx.x + c * tpr) * VEC;
    in[c] = col[c] < a.h;  // h is a multiple of VEC
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[c][q] = res[c][q] = 0.0f;
    if (in[c]) {
      if (a.y) ld<VEC>(a.y, row * a.ldy + col[c], YF, v[c]);
      ld<VEC>(a.res, row * a.ldres + col[c], RF, res[c]);
    }
  }

  // mean and reciprocal root of the mean square of u over the row.
  auto stats = [&](float (&u)[CPT][VEC], float* p0, float* p1, float& mean, float& rstd) {
    mean = 0.0f;
    if (layer) {
      float s = 0.0f;
#pragma unroll
      for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int q = 0; q < VEC; ++q) s += u[c][q];
      mean = row_sum(s, warps, p0) * inv_h;
    }
    float s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (in[c]) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float d = u[c][q] - mean;
          s2 = fmaf(d, d, s2);
        }
      }
    rstd = rsqrtf(row_sum(s2, warps, p1) * inv_h + a.eps);
  };

  if (a.y) {
    float mean = 0.0f, rstd = 1.0f;
    if (a.inner) stats(v, part[0], part[1], mean, rstd);
    const float tok = a.gate_mode == DWM_GATE_TOKEN ? ld1(a.gate, row * a.ldg, a.gate_f32) : 1.0f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if (!in[c]) continue;
      if (a.inner) {
        float w[VEC];
        ld<VEC>(a.w2, col[c], a.w_f32, w);
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[c][q] = (v[c][q] - mean) * rstd * w[q];
        if (a.b2) {
          ld<VEC>(a.b2, col[c], a.w_f32, w);
#pragma unroll
          for (int q = 0; q < VEC; ++q) v[c][q] += w[q];
        }
      }
      if (a.gate_mode == DWM_GATE_TOKEN) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[c][q] *= tok;
      } else if (a.gate_mode != DWM_GATE_NONE) {
        float g[VEC];
        ld<VEC>(a.gate, (a.gate_mode == DWM_GATE_FULL ? row * a.ldg : 0) + col[c], a.gate_f32, g);
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[c][q] *= g[q];
      }
#pragma unroll
      for (int q = 0; q < VEC; ++q) res[c][q] = fmaf(a.scale, v[c][q], a.res_scale * res[c][q]);
      st<VEC>(a.r_out, row * a.ldr + col[c], RF, res[c]);
    }
  }
  if (a.h_out) {
    float mean, rstd;
    stats(res, part[2], part[3], mean, rstd);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if (!in[c]) continue;
      float w[VEC];
      ld<VEC>(a.w1, col[c], a.w_f32, w);
#pragma unroll
      for (int q = 0; q < VEC; ++q) res[c][q] = (res[c][q] - mean) * rstd * w[q];
      if (a.b1) {
        ld<VEC>(a.b1, col[c], a.w_f32, w);
#pragma unroll
        for (int q = 0; q < VEC; ++q) res[c][q] += w[q];
      }
      st<VEC>(a.h_out, row * a.ldh + col[c], a.h_f32, res[c]);
    }
  }
}

template <int VEC, int CPT>
int launch(const Args& a, bool yf, bool rf, int tpr, int rows, cudaStream_t s) {
  const dim3 block((unsigned)tpr, (unsigned)rows);
  const unsigned grid = (unsigned)((a.t + rows - 1) / rows);
  if (yf)
    rf ? block_norm_kernel<VEC, CPT, true, true><<<grid, block, 0, s>>>(a)
       : block_norm_kernel<VEC, CPT, true, false><<<grid, block, 0, s>>>(a);
  else
    rf ? block_norm_kernel<VEC, CPT, false, true><<<grid, block, 0, s>>>(a)
       : block_norm_kernel<VEC, CPT, false, false><<<grid, block, 0, s>>>(a);
  return check_cuda(cudaGetLastError(), "block_norm launch");
}

// Rows of at most 32 elements a thread and 512 threads (a thread's two rows
// of f32 are 64 registers, which 1024 threads would not have).
constexpr int MAX_H = 16384;

int run(const Args& a, bool yf, bool rf, bool vec, cudaStream_t s) {
  const int n = vec ? a.h / 8 : a.h;  // loads a row
  const int max_cpt = vec ? 4 : 32;
  int tpr = 32;
  while (tpr < 512 && tpr * max_cpt < n) tpr *= 2;
  if (tpr > 32 || n > 128) {
    // A CTA a row: more threads with fewer loads each, down to two.
    while (tpr < 512 && (n + tpr - 1) / tpr > (vec ? 2 : 8)) tpr *= 2;
  }
  const int rows = tpr == 32 ? 4 : 1;
  const int cpt = (n + tpr - 1) / tpr;
  if (vec) {
    if (cpt <= 1) return launch<8, 1>(a, yf, rf, tpr, rows, s);
    if (cpt <= 2) return launch<8, 2>(a, yf, rf, tpr, rows, s);
    return launch<8, 4>(a, yf, rf, tpr, rows, s);
  }
  if (cpt <= 4) return launch<1, 4>(a, yf, rf, tpr, rows, s);
  if (cpt <= 8) return launch<1, 8>(a, yf, rf, tpr, rows, s);
  if (cpt <= 16) return launch<1, 16>(a, yf, rf, tpr, rows, s);
  return launch<1, 32>(a, yf, rf, tpr, rows, s);
}

}  // namespace norm
}  // namespace dwm

using namespace dwm;

extern "C" int dwm_block_norm(const void* y, int y_dtype, int64_t ldy, const void* residual,
                              int residual_dtype, int64_t ldres, int t, int h, int kind,
                              float eps, int inner, const void* w2, const void* b2,
                              const void* gate, int gate_dtype, int gate_mode, int64_t ldg,
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
                    (!y || is_float(y_dtype)) && (!gate || is_float(gate_dtype)),
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
                       {gate_mode == DWM_GATE_FULL ? gate : nullptr, ldg, es(gate_dtype)}};
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
        gate_mode == DWM_GATE_CHANNEL ? row_span(gate, 1, h, h, es(gate_dtype))
                                      : row_span(gate_mode == DWM_GATE_TOKEN ? gate : nullptr, t,
                                                 1, ldg, es(gate_dtype))};
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
                    rows16(gate, gate_mode == DWM_GATE_FULL ? ldg : 0, gate_dtype));
  norm::Args a;
  a.y = y;
  a.res = residual;
  a.w2 = w2;
  a.b2 = b2;
  a.w1 = w1;
  a.b1 = b1;
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
  a.w_f32 = w_dtype == DWM_F32;
  a.gate_f32 = gate_dtype == DWM_F32;
  a.h_f32 = h_dtype == DWM_F32;
  a.eps = eps;
  a.scale = scale;
  a.res_scale = residual_scale;
  return norm::run(a, y && y_dtype == DWM_F32, residual_dtype == DWM_F32, vec,
                   static_cast<cudaStream_t>(stream));
}
