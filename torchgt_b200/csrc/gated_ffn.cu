// Gated feed-forward block, h = act(x Wg^T) * (x Wu^T), y = h Wd^T + residual, forward and backward.
//
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//
// bf16: five products of gated_gemm.cuh.  The gate's and the up projection's columns of a tile are summed side by side, so
// the activation and their product are taken from fp32 sums before anything is rounded; dg and du leave the product that makes dh,
// dx is one sum over both, and each weight's gradient is summed over rows that all SMs share.
// fp32: the split products of linear_mma.cu, with the gate between them in kernels of their own.
#include <atomic>

#include "gated_gemm.cuh"

namespace tgt {
namespace tma {

int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int box_rows, int box_columns) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void*> entry{nullptr};
  void* f = entry.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult found;
    TGT_CHECK_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || f == nullptr)
      return set_error(TGT_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    entry.store(f, std::memory_order_release);
  }
  const cuuint64_t sizes[2] = {cuuint64_t(columns), cuuint64_t(rows)}, pitch[1] = {cuuint64_t(columns) * 2};
  const cuuint32_t box[2] = {cuuint32_t(box_columns), cuuint32_t(box_rows)}, steps[2] = {1, 1};
  auto encode = [&] {
    return reinterpret_cast<Encode>(f)(
        map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), sizes, pitch, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
        box_columns == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {      // the thread (one of autograd's, say) has made no call that binds a context yet
    const int dev = current_device();
    if (dev < 0) return TGT_ERR_CUDA;
    TGT_CHECK_CUDA(cudaSetDevice(dev));
    rc = encode();
  }
  if (rc != CUDA_SUCCESS)
    return set_error(TGT_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d for %lld rows of %lld", int(rc), (long long)rows,
                     (long long)columns);
  return TGT_OK;
}

}  // namespace tma

namespace {

using gemm::Gemm;
constexpr int kMostWidth = 65536;
constexpr int64_t kMostRows = int64_t(1) << 30;

int operand(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, bool mn_major, int tile_rows) {
  return tma::make_map(map, base, rows, columns, mn_major ? gemm::kChunk : tile_rows, 64);
}
int result(CUtensorMap* map, const void* base, int64_t rows, int64_t columns) {
  return tma::make_map(map, base, rows, columns, 32, gemm::kStoreCols);
}
int tiles_of(int64_t n, int tile) { return int((n + tile - 1) / tile); }

#define TGT_RETURN_IF(...)             \
  do {                                 \
    const int _rc = (__VA_ARGS__);     \
    if (_rc != TGT_OK) return _rc;     \
  } while (0)

template <int BN, bool A_MN, bool B_MN, gemm::Finish FINISH>
int launch(const Gemm& p, int grid, cudaStream_t stream) {
  constexpr auto kernel = gemm::gemm_kernel<BN, A_MN, B_MN, FINISH>;
  TGT_RETURN_IF(allow_shared_memory<gemm::gemm_kernel<BN, A_MN, B_MN, FINISH>>(gemm::smem_bytes(BN)));
  kernel<<<grid, gemm::kThreads, gemm::smem_bytes(BN), stream>>>(p);
  TGT_CHECK_CUDA(cudaGetLastError());
  return TGT_OK;
}

// Columns of a tile: the width whose rounds of tiles over the SMs cost least, a column of a narrower tile costing more (its
// rows are read again, and products of fewer columns do not fill the tensor cores).
int tile_columns_for(int64_t m, int columns, int narrowest) {
  int best = 256;
  double least = 0;
  for (int bn = 256; bn >= narrowest; bn /= 2) {
    const int64_t tiles = int64_t(tiles_of(m, gemm::kTileM)) * tiles_of(columns, bn);
    const int64_t rounds = (tiles + sm_count() - 1) / sm_count();
    const double cost = double(rounds) * (bn == 256 ? 256 : bn == 128 ? 140 : 84);
    if (bn == 256 || cost < least) {
      best = bn;
      least = cost;
    }
  }
  return best;
}
int grid_for(const Gemm& p) {
  const int64_t tiles = int64_t(p.m_tiles) * p.n_tiles;
  return int(tiles < sm_count() ? tiles : sm_count());
}
template <bool A_MN, bool B_MN, gemm::Finish FINISH>
int launch_any(int bn, const Gemm& p, cudaStream_t stream) {
  if (bn == 256) return launch<256, A_MN, B_MN, FINISH>(p, grid_for(p), stream);
  if (bn == 128) return launch<128, A_MN, B_MN, FINISH>(p, grid_for(p), stream);
  if constexpr (FINISH != gemm::kGated) return launch<64, A_MN, B_MN, FINISH>(p, grid_for(p), stream);
  return set_error(TGT_ERR_INVALID, "no tile of %d columns", bn);
}

// What weight_grad's parts need: tiles of 128 rows of out_features x `bn` of in_features, `ctas` shares of all their chunks.
struct PartsPlan {
  int bn, product_tiles, m_tiles, n_tiles, chunks, ctas;
  size_t bytes() const { return (size_t(m_tiles) * n_tiles + ctas) * bn * gemm::kTileM * sizeof(float); }
};
PartsPlan plan_parts(int count, int64_t rows, int out_features, int in_features) {
  PartsPlan q;
  q.bn = in_features > 128 ? 256 : in_features > 64 ? 128 : 64;
  q.product_tiles = tiles_of(out_features, gemm::kTileM);
  q.m_tiles = q.product_tiles * count;
  q.n_tiles = tiles_of(in_features, q.bn);
  q.chunks = tiles_of(rows, gemm::kChunk);
  const int64_t all = int64_t(q.m_tiles) * q.n_tiles * q.chunks;
  q.ctas = int(all < sm_count() ? all : sm_count());
  return q;
}

int check_widths(int64_t rows, int a, int b, int dtype, int act) {
  TGT_CHECK_ARG(dtype == TGT_F32 || dtype == TGT_BF16, "dtype must be TGT_F32 or TGT_BF16");
  TGT_CHECK_ARG(act == TGT_ACT_SILU || act == TGT_ACT_GELU || act == TGT_ACT_RELU, "act is none of silu, gelu and relu");
  TGT_CHECK_ARG(rows >= 0, "rows must be >= 0");
  TGT_CHECK_ARG(a >= 1 && b >= 1, "widths must be positive");
  if (dtype == TGT_BF16 && (a % 8 != 0 || b % 8 != 0 || a > kMostWidth || b > kMostWidth || rows > kMostRows))
    return set_error(TGT_ERR_UNSUPPORTED, "widths %d and %d over %lld rows: multiples of 8, at most %d, over at most 2^30 rows", a, b,
                     (long long)rows, kMostWidth);
  return TGT_OK;
}

// ---- fp32: the gate between the products -------------------------------------------------------------------------------
constexpr int kGateThreads = 256;
template <bool SLOPE>
__device__ __forceinline__ float act_f32(int act, float x, float& slope) {
  if (act == TGT_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-x));
    if (SLOPE) slope = s * (1.f + x * (1.f - s));
    return x * s;
  }
  if (act == TGT_ACT_GELU) {
    if (SLOPE) slope = gelu_slope(x);
    return gelu(x);
  }
  if (SLOPE) slope = x <= 0.f ? 0.f : 1.f;
  return relu(x);
}
__global__ void __launch_bounds__(kGateThreads) gate_kernel(const float4* gate, const float4* up, int64_t n, int act, float4* h) {
  for (int64_t i = blockIdx.x * int64_t(kGateThreads) + threadIdx.x; i < n; i += int64_t(gridDim.x) * kGateThreads) {
    const float4 g = __ldg(gate + i), u = __ldg(up + i);
    float unused;
    h[i] = make_float4(act_f32<false>(act, g.x, unused) * u.x, act_f32<false>(act, g.y, unused) * u.y,
                       act_f32<false>(act, g.z, unused) * u.z, act_f32<false>(act, g.w, unused) * u.w);
  }
}
// dgate holds dh and receives dgate
__global__ void __launch_bounds__(kGateThreads) gate_grad_kernel(const float4* gate, const float4* up, int64_t n, int act,
                                                                 float4* dgate, float4* dup) {
  for (int64_t i = blockIdx.x * int64_t(kGateThreads) + threadIdx.x; i < n; i += int64_t(gridDim.x) * kGateThreads) {
    const float4 g = __ldg(gate + i), u = __ldg(up + i), d = dgate[i];
    float4 slope, a;
    a.x = act_f32<true>(act, g.x, slope.x); a.y = act_f32<true>(act, g.y, slope.y);
    a.z = act_f32<true>(act, g.z, slope.z); a.w = act_f32<true>(act, g.w, slope.w);
    dgate[i] = make_float4(d.x * u.x * slope.x, d.y * u.y * slope.y, d.z * u.z * slope.z, d.w * u.w * slope.w);
    dup[i] = make_float4(d.x * a.x, d.y * a.y, d.z * a.z, d.w * a.w);
  }
}
int gate_grid(int64_t n) {
  const int64_t want = (n + kGateThreads - 1) / kGateThreads, most = int64_t(sm_count()) * 8;
  return int(want < most ? want : most);
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_gated_hidden(const void* x, const void* w_gate, const void* w_up, int64_t rows, int in, int mid, int act,
                                int dtype, void* h, void* gate, void* up, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, in, mid, dtype, act));
  TGT_CHECK_ARG((gate == nullptr) == (up == nullptr), "gate and up go together");
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(x && w_gate && w_up && h, "x, w_gate, w_up and h must not be null");
  TGT_CHECK_ARG(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(h) && aligned16(gate) && aligned16(up),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    TGT_CHECK_ARG(gate != nullptr, "in fp32 gate and up must not be null");
    const float* w[2] = {static_cast<const float*>(w_gate), static_cast<const float*>(w_up)};
    const float* bias[2] = {nullptr, nullptr};
    float* c[2] = {static_cast<float*>(gate), static_cast<float*>(up)};
    TGT_RETURN_IF(tgt_linear_rows_multi(static_cast<const float*>(x), w, bias, 2, rows, in, mid, TGT_ACT_NONE, nullptr, nullptr, c,
                                        stream));
    const int64_t n = rows * mid / 4;
    gate_kernel<<<gate_grid(n), kGateThreads, 0, stream>>>(static_cast<const float4*>(gate), static_cast<const float4*>(up), n, act,
                                                           static_cast<float4*>(h));
    TGT_CHECK_CUDA(cudaGetLastError());
    return TGT_OK;
  }
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  const int bn = tile_columns_for(rows, 2 * mid, 128);
  TGT_RETURN_IF(operand(&p.a[0], x, rows, in, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_gate, mid, in, false, bn / 2));
  TGT_RETURN_IF(operand(&p.b[1], w_up, mid, in, false, bn / 2));
  p.a[1] = p.a[0];
  TGT_RETURN_IF(result(&p.out[0], h, rows, mid));
  p.keep = gate != nullptr;
  if (p.keep) {
    TGT_RETURN_IF(result(&p.out[1], gate, rows, mid));
    TGT_RETURN_IF(result(&p.out[2], up, rows, mid));
  }
  p.m = rows; p.n = mid;
  p.m_tiles = tiles_of(rows, gemm::kTileM); p.n_tiles = tiles_of(mid, bn / 2);
  p.chunks = p.source_chunks = tiles_of(in, gemm::kChunk);
  p.act = act;
  return launch_any<false, false, gemm::kGated>(bn, p, stream);
}

extern "C" int tgt_gated_output(const void* h, const void* w_down, const void* add, int64_t rows, int mid, int out, int dtype,
                                void* y, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, mid, out, dtype, TGT_ACT_SILU));
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(h && w_down && y, "h, w_down and y must not be null");
  TGT_CHECK_ARG(aligned16(h) && aligned16(w_down) && aligned16(add) && aligned16(y), "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    const float *w = static_cast<const float*>(w_down), *bias = nullptr;
    float* c = static_cast<float*>(y);
    return tgt_linear_rows_multi(static_cast<const float*>(h), &w, &bias, 1, rows, mid, out, TGT_ACT_NONE, nullptr,
                                 static_cast<const float*>(add), &c, stream);
  }
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  const int bn = tile_columns_for(rows, out, 64);
  TGT_RETURN_IF(operand(&p.a[0], h, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_down, out, mid, false, bn));
  p.a[1] = p.a[0]; p.b[1] = p.b[0];
  TGT_RETURN_IF(result(&p.out[0], y, rows, out));
  p.add = static_cast<const __nv_bfloat16*>(add);
  p.m = rows; p.n = out;
  p.m_tiles = tiles_of(rows, gemm::kTileM); p.n_tiles = tiles_of(out, bn);
  p.chunks = p.source_chunks = tiles_of(mid, gemm::kChunk);
  return launch_any<false, false, gemm::kPlain>(bn, p, stream);
}

extern "C" int tgt_gated_hidden_grad(const void* dy, const void* w_down, const void* gate, const void* up, int64_t rows, int out,
                                     int mid, int act, int dtype, void* dgate, void* dup, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, out, mid, dtype, act));
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(dy && w_down && gate && up && dgate && dup, "dy, w_down, gate, up, dgate and dup must not be null");
  TGT_CHECK_ARG(aligned16(dy) && aligned16(w_down) && aligned16(gate) && aligned16(up) && aligned16(dgate) && aligned16(dup),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    TGT_RETURN_IF(tgt_linear_input_grad(static_cast<const float*>(dy), static_cast<const float*>(w_down), rows, out, mid,
                                        static_cast<float*>(dgate), stream));
    const int64_t n = rows * mid / 4;
    gate_grad_kernel<<<gate_grid(n), kGateThreads, 0, stream>>>(static_cast<const float4*>(gate), static_cast<const float4*>(up), n,
                                                                act, static_cast<float4*>(dgate), static_cast<float4*>(dup));
    TGT_CHECK_CUDA(cudaGetLastError());
    return TGT_OK;
  }
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  const int bn = tile_columns_for(rows, mid, 64);
  TGT_RETURN_IF(operand(&p.a[0], dy, rows, out, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_down, out, mid, true, bn));
  p.a[1] = p.a[0]; p.b[1] = p.b[0];
  TGT_RETURN_IF(result(&p.out[0], dgate, rows, mid));
  TGT_RETURN_IF(result(&p.out[1], dup, rows, mid));
  p.gate = static_cast<const __nv_bfloat16*>(gate); p.up = static_cast<const __nv_bfloat16*>(up);
  p.m = rows; p.n = mid;
  p.m_tiles = tiles_of(rows, gemm::kTileM); p.n_tiles = tiles_of(mid, bn);
  p.chunks = p.source_chunks = tiles_of(out, gemm::kChunk);
  p.act = act;
  return launch_any<false, true, gemm::kGatedGrad>(bn, p, stream);
}

extern "C" int tgt_gated_input_grad(const void* dgate, const void* dup, const void* w_gate, const void* w_up, int64_t rows, int mid,
                                    int in, int dtype, void* dx, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, mid, in, dtype, TGT_ACT_SILU));
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(dgate && dup && w_gate && w_up && dx, "dgate, dup, w_gate, w_up and dx must not be null");
  TGT_CHECK_ARG(aligned16(dgate) && aligned16(dup) && aligned16(w_gate) && aligned16(w_up) && aligned16(dx),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    const float* d[2] = {static_cast<const float*>(dgate), static_cast<const float*>(dup)};
    const float* w[2] = {static_cast<const float*>(w_gate), static_cast<const float*>(w_up)};
    return tgt_linear_input_grad_multi(d, w, 2, rows, mid, in, TGT_ACT_NONE, nullptr, static_cast<float*>(dx), stream);
  }
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  const int bn = tile_columns_for(rows, in, 64);
  TGT_RETURN_IF(operand(&p.a[0], dgate, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.a[1], dup, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_gate, mid, in, true, bn));
  TGT_RETURN_IF(operand(&p.b[1], w_up, mid, in, true, bn));
  TGT_RETURN_IF(result(&p.out[0], dx, rows, in));
  p.m = rows; p.n = in;
  p.m_tiles = tiles_of(rows, gemm::kTileM); p.n_tiles = tiles_of(in, bn);
  p.source_chunks = tiles_of(mid, gemm::kChunk);
  p.chunks = 2 * p.source_chunks;
  return launch_any<false, true, gemm::kPlain>(bn, p, stream);
}

extern "C" int tgt_gated_weight_grad_scratch_bytes(int count, int64_t rows, int out_features, int in_features, int dtype,
                                                   size_t* bytes) {
  using namespace tgt;
  TGT_CHECK_ARG(bytes != nullptr, "bytes is null");
  TGT_CHECK_ARG(count == 1 || count == 2, "count must be 1 or 2");
  TGT_RETURN_IF(check_widths(rows, out_features, in_features, dtype, TGT_ACT_SILU));
  if (dtype == TGT_F32) return tgt_linear_wgrad_multi_scratch_bytes(count, rows, in_features, out_features, bytes);
  *bytes = rows == 0 ? 0 : plan_parts(count, rows, out_features, in_features).bytes();
  return TGT_OK;
}

extern "C" int tgt_gated_weight_grad(const void* const* dy, const void* x, int count, int64_t rows, int out_features,
                                     int in_features, int dtype, void* const* dw, void* scratch, size_t scratch_bytes,
                                     void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_CHECK_ARG(count == 1 || count == 2, "count must be 1 or 2");
  TGT_RETURN_IF(check_widths(rows, out_features, in_features, dtype, TGT_ACT_SILU));
  TGT_CHECK_ARG(dw && dw[0] && dw[count - 1], "dw must not be null");
  if (rows == 0) {
    for (int i = 0; i < count; ++i)
      TGT_CHECK_CUDA(cudaMemsetAsync(dw[i], 0, size_t(out_features) * in_features * (dtype == TGT_F32 ? 4 : 2), stream));
    return TGT_OK;
  }
  TGT_CHECK_ARG(dy && dy[0] && dy[count - 1] && x, "dy and x must not be null");
  TGT_CHECK_ARG(aligned16(dy[0]) && aligned16(dy[count - 1]) && aligned16(x) && aligned16(dw[0]) && aligned16(dw[count - 1]) &&
                    aligned16(scratch),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    const float* d[2] = {static_cast<const float*>(dy[0]), static_cast<const float*>(dy[count - 1])};
    float* w[2] = {static_cast<float*>(dw[0]), static_cast<float*>(dw[count - 1])};
    float* bias[2] = {nullptr, nullptr};
    return tgt_linear_wgrad_multi(d, static_cast<const float*>(x), count, rows, in_features, out_features, w, bias, scratch,
                                  scratch_bytes, stream);
  }
  const PartsPlan q = plan_parts(count, rows, out_features, in_features);
  if (scratch == nullptr || scratch_bytes < q.bytes())
    return set_error(TGT_ERR_WORKSPACE, "scratch holds %zu bytes, %zu needed", scratch_bytes, q.bytes());
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  for (int i = 0; i < 2; ++i)
    TGT_RETURN_IF(operand(&p.a[i], dy[i < count ? i : 0], rows, out_features, true, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], x, rows, in_features, true, q.bn));
  p.b[1] = p.b[0];
  p.partial = static_cast<float*>(scratch);
  p.m = out_features; p.n = in_features;
  p.m_tiles = q.m_tiles; p.n_tiles = q.n_tiles; p.product_tiles = q.product_tiles;
  p.chunks = p.source_chunks = q.chunks;
  gemm::SumParts s{p.partial, {static_cast<__nv_bfloat16*>(dw[0]), static_cast<__nv_bfloat16*>(dw[count - 1])}, out_features,
                   in_features, q.m_tiles, q.n_tiles, q.product_tiles, q.chunks, q.ctas};
  const dim3 grid(unsigned(q.m_tiles) * q.n_tiles, 4 * q.bn / 64);
  if (q.bn == 256) {
    TGT_RETURN_IF((launch<256, true, true, gemm::kPartial>(p, q.ctas, stream)));
    gemm::sum_parts_kernel<256><<<grid, gemm::kSumThreads, 0, stream>>>(s);
  } else if (q.bn == 128) {
    TGT_RETURN_IF((launch<128, true, true, gemm::kPartial>(p, q.ctas, stream)));
    gemm::sum_parts_kernel<128><<<grid, gemm::kSumThreads, 0, stream>>>(s);
  } else {
    TGT_RETURN_IF((launch<64, true, true, gemm::kPartial>(p, q.ctas, stream)));
    gemm::sum_parts_kernel<64><<<grid, gemm::kSumThreads, 0, stream>>>(s);
  }
  TGT_CHECK_CUDA(cudaGetLastError());
  return TGT_OK;
}
