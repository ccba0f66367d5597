// The gated feed-forward block for a few rows in bf16, as serving calls it: h = act(x Wg^T) * (x Wu^T), y = h Wd^T + add.
//
// With a few rows the three weights, read once, are all that counts, and tiles of 128 rows on a handful of SMs do not read
// them fast enough.  So every 8 columns of h (16 with more rows), and every 16 of y, are a CTA's, whose warps share k: a
// lane loads 16 bytes of a weight's row at a time straight into the fragment of mma.sync (16 weight rows x 16 of k, by 8
// rows of x), several steps ahead.  Which elements of k a fragment's places hold is free as long as x is loaded the same
// way: a lane's eight consecutive elements are the places of two products.  In the first kernel the sixteen weight rows are
// 8 of Wg and the 8 of Wu for the same columns, so one lane ends up with both sums of a value of h.  The sums of the warps
// are added in their order.  The second kernel is the first's dependent: its first loads of Wd are on their way before it
// waits for h.
//
// One row, 2,048 x 5,632 x 2,048, weights not in the L2: 18 us, of which the SMs are busy 7.8 and 5.7 (46 and 23 MB, 0.9 of
// the bandwidth).  Bringing Wd into the L2 from the first kernel on made that 20.
#include "linear_rows.cuh"

namespace tgt {
namespace {

constexpr int kMostFewRows = 32;

struct FewRows {
  const __nv_bfloat16* a;        // [rows, red]
  const __nv_bfloat16* w[2];     // [cols, red]: of the gate and of the up projection, or one
  const __nv_bfloat16* add;      // [rows, cols], may be null
  __nv_bfloat16* out;            // [rows, cols]
  int rows, red, cols, act;
};

__device__ __forceinline__ void multiply_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// TILES: of 8 rows of x; SETS: of 16 weight rows; DEPTH: steps of 32 of k whose weights are on their way.  GATED: the columns'
// sums of two weights become act(.) * (.); otherwise they are columns of one weight.
template <int TILES, int SETS, int WARPS, int DEPTH, bool GATED>
__global__ void __launch_bounds__(32 * WARPS) few_rows_kernel(const FewRows p) {
  constexpr int kSetCols = GATED ? 8 : 16;
  __shared__ float s_sums[WARPS][SETS][TILES][4][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int col0 = blockIdx.x * (kSetCols * SETS);
  if (GATED) release_dependents();
  // of every set this lane's two weight rows; behind the last column any row, whose sums nobody takes
  const __nv_bfloat16 *w0[SETS], *w1[SETS];
#pragma unroll
  for (int m = 0; m < SETS; ++m) {
    const int c0 = min(col0 + m * kSetCols + g, p.cols - 1), c1 = GATED ? c0 : min(c0 + 8, p.cols - 1);
    w0[m] = p.w[0] + int64_t(c0) * p.red;
    w1[m] = p.w[GATED ? 1 : 0] + int64_t(c1) * p.red;
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float d[SETS][TILES][4];
#pragma unroll
  for (int m = 0; m < SETS; ++m)
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[m][n][i] = 0.f;
  uint4 f0[DEPTH][SETS], f1[DEPTH][SETS];
  // of k: a warp's two steps in a row are 128 bytes of a weight's row
  auto place = [&](int step) { return ((step >> 1) * WARPS + warp) * 64 + (step & 1) * 32 + 8 * t; };
  const int steps = 2 * ((p.red + WARPS * 64 - 1) / (WARPS * 64));
  auto load_weights = [&](int slot, int step) {
    const int k = place(step);
#pragma unroll
    for (int m = 0; m < SETS; ++m) {
      f0[slot][m] = k < p.red ? __ldg(reinterpret_cast<const uint4*>(w0[m] + k)) : zero;
      f1[slot][m] = k < p.red ? __ldg(reinterpret_cast<const uint4*>(w1[m] + k)) : zero;
    }
  };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) load_weights(s, s);
  if (!GATED) dependent_wait();                   // for a
  for (int first = 0; first < steps; first += DEPTH) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      const int k = place(first + s);
#pragma unroll
      for (int n = 0; n < TILES; ++n) {
        const int row = n * 8 + g;
        const uint4 x = row < p.rows && k < p.red ? __ldg(reinterpret_cast<const uint4*>(p.a + int64_t(row) * p.red + k)) : zero;
#pragma unroll
        for (int m = 0; m < SETS; ++m) {
          multiply_add(d[m][n], f0[s][m].x, f1[s][m].x, f0[s][m].y, f1[s][m].y, x.x, x.y);
          multiply_add(d[m][n], f0[s][m].z, f1[s][m].z, f0[s][m].w, f1[s][m].w, x.z, x.w);
        }
      }
      load_weights(s, first + s + DEPTH);
    }
  }
#pragma unroll
  for (int m = 0; m < SETS; ++m)
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s_sums[warp][m][n][i][lane] = d[m][n][i];
  __syncthreads();
  // d[0], d[1]: of weight row g by rows 2t, 2t + 1 of x; d[2], d[3]: of weight row g + 8
  constexpr int kValues = GATED ? 2 : 4;
  for (int v = threadIdx.x; v < SETS * TILES * kValues * 32; v += 32 * WARPS) {
    const int l = v % 32, i = v / 32 % kValues, n = v / (32 * kValues) % TILES, m = v / (32 * kValues * TILES);
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      s += s_sums[w][m][n][i][l];
      if (GATED) u += s_sums[w][m][n][i + 2][l];
    }
    const int row = n * 8 + 2 * (l % 4) + i % 2, col = col0 + m * kSetCols + l / 4 + (i / 2) * 8;
    if (row >= p.rows || col >= p.cols) continue;
    if (GATED) {
      const float a = p.act == TGT_ACT_SILU ? s / (1.f + __expf(-s)) : p.act == TGT_ACT_GELU ? gelu(s) : relu(s);
      s = a * u;
    } else if (p.add != nullptr) {
      s += __bfloat162float(p.add[int64_t(row) * p.cols + col]);
    }
    p.out[int64_t(row) * p.cols + col] = __float2bfloat16_rn(s);
  }
}

template <int TILES, int SETS, int WARPS, int DEPTH, bool GATED>
int launch(const FewRows& p, cudaStream_t stream) {
  constexpr int kCols = (GATED ? 8 : 16) * SETS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.cols + kCols - 1) / kCols);
  cfg.blockDim = dim3(32 * WARPS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  if (!GATED) {
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  TGT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, few_rows_kernel<TILES, SETS, WARPS, DEPTH, GATED>, p));
  return TGT_OK;
}
// Eight columns of h a CTA; over 8 rows, whose loads of x are as many bytes as the weights', sixteen where that leaves no SM
// without a CTA.  us, weights not in the L2, eight / sixteen: 16 rows 2,048 x 5,632 24.6 / 22.8, 4,096 x 11,008 77 / 69, 32 rows
// 768 x 2,048 10.1 / 12.2; one row 2,048 x 5,632 18.2 / 18.8 (the weights' bytes 10.7), 4,096 x 11,008 51 / 54 (42).
template <int TILES>
int launch_both(const FewRows& first, const FewRows& second, cudaStream_t stream) {
  int rc;
  if constexpr (TILES > 1)
    rc = first.cols >= 16 * sm_count() ? launch<TILES, 2, 4, 4, true>(first, stream) : launch<TILES, 1, 8, 4, true>(first, stream);
  else
    rc = launch<TILES, 1, 8, 4, true>(first, stream);
  return rc != TGT_OK ? rc : launch<TILES, 1, 16, 4, false>(second, stream);
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_gated_few_rows(const void* x, const void* w_gate, const void* w_up, const void* w_down, const void* add,
                                  int64_t rows, int in, int mid, int out, int act, void* h, void* y, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_CHECK_ARG(act == TGT_ACT_SILU || act == TGT_ACT_GELU || act == TGT_ACT_RELU, "act is none of silu, gelu and relu");
  TGT_CHECK_ARG(rows >= 0 && rows <= kMostFewRows, "rows must be 0 to %d", kMostFewRows);
  TGT_CHECK_ARG(in >= 1 && mid >= 1 && out >= 1, "widths must be positive");
  if (in % 8 != 0 || mid % 8 != 0 || out % 8 != 0 || in > 65536 || mid > 65536 || out > 65536)
    return set_error(TGT_ERR_UNSUPPORTED, "widths %d, %d and %d: multiples of 8, at most 65536", in, mid, out);
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(x && w_gate && w_up && w_down && h && y, "x, w_gate, w_up, w_down, h and y must not be null");
  TGT_CHECK_ARG(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(h),
                "tensors must be 16-byte aligned");
  using T = __nv_bfloat16;
  const FewRows first{static_cast<const T*>(x), {static_cast<const T*>(w_gate), static_cast<const T*>(w_up)}, nullptr,
                      static_cast<T*>(h), int(rows), in, mid, act};
  const FewRows second{static_cast<const T*>(h), {static_cast<const T*>(w_down), nullptr}, static_cast<const T*>(add),
                       static_cast<T*>(y), int(rows), mid, out, act};
  return rows <= 8 ? launch_both<1>(first, second, stream) : rows <= 16 ? launch_both<2>(first, second, stream)
                                                                        : launch_both<4>(first, second, stream);
}
