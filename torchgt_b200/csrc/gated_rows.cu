// The gated feed-forward block for a few rows in bf16, as serving calls it: h = act(x Wg^T) * (x Wu^T), y = h Wd^T + add.
//
// With a few rows the three weights, read once, are all that counts, and tiles of 128 rows on a handful of SMs do not read
// them fast enough.  So every 16 columns of h, and every 16 or 32 of y, are a CTA's, whose warps share k.  A lane copies 16
// bytes of a weight's row at a time, asynchronously and several steps ahead, to a place of its own in shared memory, from where
// they are a fragment of mma.sync as they lie (16 weight rows x 16 of k, by 8 rows of x).  Which elements of k a fragment's
// places hold is free as long as x is loaded the same way: a lane's eight consecutive elements are the places of two
// products.  In the first kernel the sixteen weight rows are 8 of Wg and the 8 of Wu for the same columns, so one lane ends
// up with both sums of a value of h.  The sums of the warps are added in their order.
//
// The second kernel is the first's dependent: it comes in as the first's last CTAs run, and what it has room for of Wd, up to
// 160 KB an SM, is on its way before it waits for h.  (In registers, four steps ahead, one row 2,048 x 5,632 x 2,048 took 18.5 us;
// so 15.7, with the first kernel's weights the same way, which lets more of them be under way, 14.5.)
//
// us from graphs, weights not in the L2: one row 2,048 x 5,632 x 2,048 14.5 (69 MB, 10.7 at the bandwidth), 768 x 2,048 x 768 4.5,
// 4,096 x 11,008 x 4,096 45.4 (42).  Bringing Wd into the L2 from the first kernel on did not help.
#include "linear_rows.cuh"
#include "tensor_core.cuh"

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

// The copies of a lane into a place of its own, which no other lane reads: 16 bytes, or zeros
__device__ __forceinline__ void bring(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// TILES: of 8 rows of x; SETS: of 16 weight rows; DEPTH: steps of 32 of k whose weights are on their way.  GATED: the columns'
// sums of two weights become act(.) * (.); otherwise they are columns of one weight.
template <int TILES, int SETS, int WARPS, int DEPTH, bool GATED>
__global__ void __launch_bounds__(32 * WARPS) few_rows_kernel(const FewRows p) {
  constexpr int kSetCols = GATED ? 8 : 16;
  extern __shared__ __align__(16) uint4 s_weights[];          // [DEPTH][WARPS][SETS][2][32]
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
  // of k: a warp's two steps in a row are 128 bytes of a weight's row
  auto place = [&](int step) { return ((step >> 1) * WARPS + warp) * 64 + (step & 1) * 32 + 8 * t; };
  const int steps = 2 * ((p.red + WARPS * 64 - 1) / (WARPS * 64));
  constexpr int kSlot = WARPS * SETS * 64;
  const uint4* const mine = s_weights + warp * (SETS * 64) + lane;
  const uint32_t to = tc::smem_address(mine);
  auto bring_weights = [&](int slot, int step) {
    const int k = place(step);
    const bool there = k < p.red;
    if (step < steps) {
#pragma unroll
      for (int m = 0; m < SETS; ++m) {
        bring(to + (slot * kSlot + m * 64) * 16, w0[m] + (there ? k : 0), there);
        bring(to + (slot * kSlot + m * 64 + 32) * 16, w1[m] + (there ? k : 0), there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) bring_weights(s, s);
  if (!GATED) dependent_wait();                 // for a
  constexpr int kBatch = TILES == 1 ? 6 : TILES == 2 ? 3 : 2;    // steps whose rows of a are on their way together
  for (int first = 0, slot = 0; first < steps; first += kBatch) {
    uint4 x[kBatch][TILES];
#pragma unroll
    for (int s = 0; s < kBatch; ++s)
#pragma unroll
      for (int n = 0; n < TILES; ++n) {
        const int row = n * 8 + g, k = place(first + s);
        const uint4* const from = reinterpret_cast<const uint4*>(p.a + int64_t(row) * p.red + k);
        x[s][n] = row >= p.rows || k >= p.red ? zero : GATED ? __ldg(from) : __ldcg(from);     // h is written while this kernel waits
      }
#pragma unroll
    for (int s = 0; s < kBatch; ++s) {
      if (first + s >= steps) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
#pragma unroll
      for (int m = 0; m < SETS; ++m) {
        const uint4 f0 = mine[slot * kSlot + m * 64], f1 = mine[slot * kSlot + m * 64 + 32];
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
          multiply_add(d[m][n], f0.x, f1.x, f0.y, f1.y, x[s][n].x, x[s][n].y);
          multiply_add(d[m][n], f0.z, f1.z, f0.w, f1.w, x[s][n].z, x[s][n].w);
        }
      }
      bring_weights(slot, first + s + DEPTH);
      slot = slot + 1 == DEPTH ? 0 : slot + 1;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  static_assert(DEPTH * 1024 >= TILES * 512, "the sums in the place of the weights");
  using Sums = float[SETS][TILES][4][32];
  Sums* const s_sums = reinterpret_cast<Sums*>(s_weights);
  __syncthreads();                                // every warp is through with its weights
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
      // 2^-20 + |s| 2^-23 off (the power's rounding), next to a rounding to 8 bits
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
  cfg.dynamicSmemBytes = DEPTH * WARPS * SETS * 1024;
  const int rc = allow_shared_memory<few_rows_kernel<TILES, SETS, WARPS, DEPTH, GATED>>(DEPTH * WARPS * SETS * 1024);
  if (rc != TGT_OK) return rc;
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
// us, weights not in the L2.  First kernel over 16 rows, by eight and by four warps a CTA (a CTA of eight has half of an SM's registers):
// 32 rows 4,096 x 2,048 x 512 17.2 / 23.4, 4,096 x 4,096 x 4,096 26.2 / 31.1, 2,048 x 5,632 x 2,048 25.3 / 21.8.  Second kernel, all of
// an SM's memory for one set of columns, for two, or for several CTAs: one row 2,048 x 5,632 x 2,048 10, 5 and 3 steps 15.7, 17.7, 18.3;
// 4,096 x 11,008 x 4,096 50.8, 45.4, 46.8; 512 x 2,048 x 16,384 one set 15.7, two 17.1; 32 rows 1,024 x 4,096 x 8,192 32.7, 27.0.
template <int TILES>
int launch_both(const FewRows& first, const FewRows& second, cudaStream_t stream) {
  const int rc = TILES > 2 && first.cols > 32 * sm_count() ? launch<TILES, 2, 4, 3, true>(first, stream)
                                                           : launch<TILES, 2, 8, 3, true>(first, stream);
  if (rc != TGT_OK) return rc;
  const int sets = (second.cols + 15) / 16;
  if (sets <= sm_count()) return launch<TILES, 1, 16, 10, false>(second, stream);
  if (sets <= 2 * sm_count()) return launch<TILES, 2, 16, 5, false>(second, stream);
  return TILES > 1 ? launch<TILES, 2, 16, 3, false>(second, stream) : launch<TILES, 1, 16, 4, false>(second, stream);
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
