// The two kernels behind the products of narrow linear layers and the line between them.
#pragma once

#include <type_traits>

#include "tgt_common.cuh"

namespace tgt {

constexpr int kMostProducts = 3;

// torch's relu and (exact) gelu and the latter's derivative; NaN stays NaN
__device__ __forceinline__ float relu(float x) { return x < 0.f ? 0.f : x; }
__device__ __forceinline__ float normal_cdf(float x) { return 0.5f * (1.f + erff(x * 0.70710678118654752440f)); }
__device__ __forceinline__ float gelu(float x) { return x * normal_cdf(x); }
__device__ __forceinline__ float gelu_slope(float x) {
  return normal_cdf(x) + x * (0.39894228040143267794f * expf(-0.5f * x * x));
}

// 1 / (1 + exp(-x)) to 2^-20, from the mathematics: exp(-y) = 2^t exp(r) with t = -y log2(e) as it rounds and r = -y - t ln(2)
// what that leaves, at most 1e-5, so exp(r) is 1 + r; then the approximate reciprocal (1 unit).  0 below -87, next to where the
// quotient leaves the normal numbers (2^-125 is lost), and for whatever a NaN makes of it.  x logistic(x) at 400,001 places from -110 to
// 110: 2^-21.3 from 64 bits at most.
__device__ __forceinline__ float logistic(float x) {
  const float y = fminf(fmaxf(x, -87.f), 87.f);
  const float t = -y * 1.44269504088896341f, r = fmaf(-t, 0.693147180559945309f, -y);
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, r, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return x < -87.f ? 0.f : s;
}
// Activations of the gated block, silu among them, and with SLOPE their derivatives (of relu zero at zero).
template <int ACT, bool SLOPE>
__device__ __forceinline__ float gate_activation(float x, float& slope) {
  if constexpr (ACT == TGT_ACT_SILU) {
    const float s = logistic(x);
    if (SLOPE) slope = s * (1.f + x * (1.f - s));
    return x * s;
  } else if constexpr (ACT == TGT_ACT_GELU) {
    if (SLOPE) slope = gelu_slope(x);
    return gelu(x);
  } else {
    if (SLOPE) slope = x <= 0.f ? 0.f : 1.f;
    return relu(x);
  }
}
// f(the activation as a constant), so that code over many values branches once
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == TGT_ACT_SILU) f(std::integral_constant<int, TGT_ACT_SILU>());
  else if (act == TGT_ACT_GELU) f(std::integral_constant<int, TGT_ACT_GELU>());
  else f(std::integral_constant<int, TGT_ACT_RELU>());
}
// act(g) u of four values
template <int ACT>
__device__ __forceinline__ float4 gated(const float4& g, const float4& u) {
  float unused;
  return make_float4(gate_activation<ACT, false>(g.x, unused) * u.x, gate_activation<ACT, false>(g.y, unused) * u.y,
                     gate_activation<ACT, false>(g.z, unused) * u.z, gate_activation<ACT, false>(g.w, unused) * u.w);
}
// and their gradients from that of the product: {dg, du}
template <int ACT>
__device__ __forceinline__ void gated_grad(const float4& d, const float4& g, const float4& u, float4& dg, float4& du) {
  float4 s;
  du.x = d.x * gate_activation<ACT, true>(g.x, s.x); du.y = d.y * gate_activation<ACT, true>(g.y, s.y);
  du.z = d.z * gate_activation<ACT, true>(g.z, s.z); du.w = d.w * gate_activation<ACT, true>(g.w, s.w);
  dg = make_float4(d.x * u.x * s.x, d.y * u.y * s.y, d.z * u.z * s.z, d.w * u.w * s.w);
}

// C_j[r][c] = f(sum_s sum_k A_s[r][k] B_sj[c][k] + bias_j[c]); one of `sources` (s) and `outputs` (j) is 1.
struct LinearRows {
  const float* a[kMostProducts];      // [rows, red]
  const float* w[kMostProducts];      // [cols, red], or [red, cols] when transposed
  const float* bias[kMostProducts];   // [cols] or null
  float* c[kMostProducts];            // [rows, cols]
  int64_t rows;
  int red, cols;
  int sources, outputs;
  bool transposed;
  bool onto;                          // c holds part of the sums already, they are added to it
  // what is done to a sum on its way out, all of it for a single output only (null / 0: nothing):
  int act;                            // TGT_ACT_*: c = act(sum + bias); pre (may be null) receives sum + bias
  float* pre;
  int gate_act;                       // c = sum * act'(at gate[r][c]); for TGT_ACT_RELU gate is the activation's result
  const float* gate;
  const float* add;                   // c = ... + add[r][c]
};

// nothing but a bias is added to the sums
inline bool is_plain(const LinearRows& p) {
  return !p.onto && p.act == TGT_ACT_NONE && p.pre == nullptr && p.gate_act == TGT_ACT_NONE && p.add == nullptr;
}

// four values of a row
__device__ __forceinline__ void finish_values(const LinearRows& p, int out, int64_t row, int col, float4 v) {
  const int64_t at = row * p.cols + col;
  if (p.onto) {
    const float4 c = *reinterpret_cast<const float4*>(p.c[out] + at);
    v.x += c.x; v.y += c.y; v.z += c.z; v.w += c.w;
  }
  if (p.bias[out] != nullptr) {
    const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias[out] + col));
    v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
  }
  if (p.pre != nullptr) *reinterpret_cast<float4*>(p.pre + at) = v;
  if (p.act == TGT_ACT_RELU) {
    v.x = relu(v.x); v.y = relu(v.y); v.z = relu(v.z); v.w = relu(v.w);
  } else if (p.act == TGT_ACT_GELU) {
    v.x = gelu(v.x); v.y = gelu(v.y); v.z = gelu(v.z); v.w = gelu(v.w);
  }
  if (p.gate_act != 0) {
    const float4 g = __ldg(reinterpret_cast<const float4*>(p.gate + at));
    if (p.gate_act == TGT_ACT_RELU) {
      v.x = g.x <= 0.f ? 0.f : v.x; v.y = g.y <= 0.f ? 0.f : v.y;
      v.z = g.z <= 0.f ? 0.f : v.z; v.w = g.w <= 0.f ? 0.f : v.w;
    } else {
      v.x *= gelu_slope(g.x); v.y *= gelu_slope(g.y); v.z *= gelu_slope(g.z); v.w *= gelu_slope(g.w);
    }
  }
  if (p.add != nullptr) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p.add + at));
    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
  }
  *reinterpret_cast<float4*>(p.c[out] + at) = v;
}

// Full fp32 FMAs on tiles of 32 rows (linear_rows.cu): sources == 1, not transposed, not onto.
int linear_few_rows(const LinearRows& p, cudaStream_t stream);

// Tiles of 128 rows x 64 columns that the tensor cores would get; with fewer, the FMA kernel's smaller tiles occupy the
// chip better (us back to back, FMA / tensor cores, 64 x 64: 4,097 rows 4.2 / 6.3, 8,192 rows 6.0 / 6.5, 16,384 rows 10.7 / 6.5;
// 64 x 128 at 8,192 rows, 128 tiles, 8.9 / 6.6).
inline bool few_rows(int64_t rows, int cols) { return (rows + 127) / 128 * ((cols + 63) / 64) < 80; }

// The gated block's products on the tensor cores with the gate in their finish (linear_mma.cu): gate = x w_gate^T, up = x w_up^T and
// h = act(gate) up; dgate and dup from dh = dy w_down.  For reductions that are one launch and rows that fill the chip.
bool gated_in_one(int64_t rows, int reduce, int tile_columns);
int linear_gated(const float* x, const float* w_gate, const float* w_up, int64_t rows, int reduce, int cols, int act, float* h,
                 float* gate, float* up, cudaStream_t stream);
int linear_gated_grad(const float* dy, const float* w_down, const float* gate, const float* up, int64_t rows, int reduce, int cols,
                      int act, float* dgate, float* dup, cudaStream_t stream);

}  // namespace tgt
