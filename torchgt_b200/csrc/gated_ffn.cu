// Gated feed-forward block, h = act(x Wg^T) * (x Wu^T), y = h Wd^T + residual, forward and backward.
//
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//
// bf16: five products of gated_gemm.cuh.  The gate's and the up projection's columns of a tile are summed side by side, so
// the activation and their product are taken from fp32 sums before anything is rounded; dg and du leave the product that makes dh,
// dx is one sum over both, and each weight's gradient is summed over rows that all SMs share.  What goes from one product into the
// next, h, dg and du, is rounded to bf16, the type the tensor cores take at twice the rate of any wider one: y is 1.9e-3 from 64 bits
// in the 2-norm (its own rounding alone 1.7e-3), the gradients 2.3e-3.
// fp32: the split products of linear_mma.cu with the gate in their finish, or, for reductions over several launches and few rows,
// with the gate in kernels of its own.
#include <atomic>

#include "gated_gemm.cuh"

namespace tgt {
namespace tma {

int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int box_rows) {
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
  const cuuint32_t box[2] = {64, cuuint32_t(box_rows)}, steps[2] = {1, 1};
  auto encode = [&] {
    return reinterpret_cast<Encode>(f)(
        map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), sizes, pitch, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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
  return tma::make_map(map, base, rows, columns, mn_major ? gemm::kChunk : tile_rows);
}
uint16_t* words(void* t) { return static_cast<uint16_t*>(t); }
const uint16_t* words(const void* t) { return static_cast<const uint16_t*>(t); }
int tiles_of(int64_t n, int tile) { return int((n + tile - 1) / tile); }

#define TGT_RETURN_IF(...)             \
  do {                                 \
    const int _rc = (__VA_ARGS__);     \
    if (_rc != TGT_OK) return _rc;     \
  } while (0)

// How a product is cut up: tiles of 128 rows of a CTA, or of 256 of a pair, x `bn` columns; `split` CTAs along k to one of a CTA.
struct Cut {
  bool pair;
  int bn, split;
  int rows() const { return pair ? 2 * gemm::kTileM : gemm::kTileM; }
  int b_rows() const { return pair ? bn / 2 : bn; }      // of B that one copy brings in
};

template <int BN, bool PAIR, bool A_MN, bool B_MN, gemm::Finish FINISH, int SPLIT = 1>
int launch(const Gemm& p, int walkers, cudaStream_t stream, bool chained) {
  constexpr int kSmem = gemm::smem_bytes(PAIR ? BN / 2 : BN, FINISH), kCluster = PAIR ? 2 : SPLIT;
  TGT_RETURN_IF(allow_shared_memory<gemm::gemm_kernel<BN, PAIR, A_MN, B_MN, FINISH, SPLIT>>(kSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(walkers * kCluster);
  cfg.blockDim = dim3(gemm::kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (kCluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = kCluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (chained) {               // the dependent of the kernel in front of it, one of this entry point's
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  TGT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gemm::gemm_kernel<BN, PAIR, A_MN, B_MN, FINISH, SPLIT>, p));
  return TGT_OK;
}

// Everything about how a product is done that its sizes decide.
struct Plan {
  Cut cut;
  int m_tiles, n_tiles, product_tiles, chunks, walkers, whole;
  int shared() const { return m_tiles * n_tiles - whole; }
  size_t scratch() const { return shared() == 0 ? 0 : size_t(shared() + walkers) * cut.bn * cut.rows() * sizeof(float); }
  void into(Gemm& p) const {
    p.m_tiles = m_tiles; p.n_tiles = n_tiles; p.product_tiles = product_tiles;
    p.chunks = chunks; p.whole = whole;
  }
};

constexpr Cut kCuts[] = {{true, 256, 1}, {true, 128, 1}, {false, 256, 1}, {false, 128, 1}, {false, 64, 1}};
enum Along { kWhole, kShare, kSplit };      // what may be done along k with too few tiles

// The cut, and whether the last round's tiles are shared, of the least time by what was measured: us a chunk of k, a finish of
// 256 columns, a start, and sharing.  us by pairs of 256 and 128 columns, single CTAs of 256, 128 and 64: y of 8,191 rows, 5,632 x 2,048
// 137, 153, 187, 172, 307; 333 rows, 2,048 x 768 16.6, 12.6, 16.3, 13.7, 11.8; dx of 64,000 rows, 128 x 64 12.8, 11.9, 13.3, 10.0, 8.5;
// h of 1,000 rows, 768 x 2,048, with what is kept 12.5, 14.6, 11.5, 13.0, -.  Shared or not: two weight gradients of 16,384 rows, 2,816 x
// 1,024 135 / 166 (88 tiles for 74 pairs), of 64,000 rows, 128 x 64 19 / 223; one of 16,384 rows, 1,024 x 2,816 (44 tiles) 89 / 83.  By one
// CTA a tile, 2, 4 and 8 of 64 columns: y of 40 rows, 2,048 x 768 11.0, 8.7, 7.5, 6.9; of 333 rows 11.4, 9.5; of 100 rows, 5,632 x 2,048
// 23.7, 15.6, 12.1; h of 40 rows, 768 x 2,048 6.8, 7.9, 9.0.  By one, and 2 of 128 columns: y of 333 rows, 5,632 x 2,048 25.1, 18.7; of
// 600 rows, 4,096 x 1,024 19.1, 15.5.
Plan plan_for(int products, int64_t m, int columns, int narrowest, int chunks, double finish, Along along) {
  const bool may_share = along == kShare;
  constexpr double kChunkTime[] = {0.39, 0.255, 0.42, 0.277, 0.235}, kStart[] = {1, 1, 0, 0, 0};
  Plan best{};
  double least = 0;
  for (int i = 0; i < 5; ++i) {
    Plan q;
    q.cut = kCuts[i];
    if (q.cut.bn < narrowest) continue;
    q.product_tiles = tiles_of(m, q.cut.rows());
    q.m_tiles = q.product_tiles * products;
    q.n_tiles = tiles_of(columns, q.cut.bn);
    q.chunks = chunks;
    const int64_t tiles = int64_t(q.m_tiles) * q.n_tiles, most = sm_count() / (q.cut.pair ? 2 : 1);
    const double out = finish * q.cut.bn / 256;
    for (int share = 0; share < (may_share ? 2 : 1); ++share) {
      q.whole = int(share ? tiles / most * most : tiles);
      const int64_t parts = q.shared() * int64_t(chunks);
      if (share && (parts == 0 || (q.whole > 0 && parts < most))) continue;
      q.walkers = int(share ? (q.whole > 0 || parts > most ? most : parts) : tiles < most ? tiles : most);
      const int64_t rounds = (q.whole + most - 1) / most;
      // SMs without a tile leave power to the others
      const double chunk = kChunkTime[i] * (0.8 + 0.2 * (share || rounds == 0 ? 1.0 : double(q.whole) / double(rounds * most)));
      const double round = chunks * chunk > out ? chunks * chunk : out;
      double time = kStart[i] + out + double(rounds) * round;
      // what is shared is read at other places of k by everybody; then the parts are written, read and added
      if (share) time += double(parts) / q.walkers * chunk * 1.15 + 8 + double(q.scratch()) / 2e6;
      if (least == 0 || time < least) {
        best = q;
        least = time;
      }
    }
    // Several CTAs a tile where there are SMs for them (clusters of two find all, larger ones not): what they put together, and that
    // they start and end together, in us.
    if (along != kSplit || q.cut.pair || q.cut.bn > 128) continue;
    double together = q.cut.bn == 64 ? 2.2 : 2.5;
    for (int split = 2; split <= 8 && tiles * split <= (split == 2 ? sm_count() : sm_count() * 7 / 8) && chunks >= 2 * split;
         split *= 2) {
      together += q.cut.bn == 64 ? 0.25 : 1.4;
      const double time = (chunks + split - 1) / split * kChunkTime[i] * 0.8 + together;
      if (time < least) {
        best = q;
        best.cut.split = split;
        best.whole = best.walkers = int(tiles);
        least = time;
      }
    }
  }
  return best;
}

template <int BN, bool PAIR, bool A_MN, bool B_MN, gemm::Finish FINISH>
int launch_cut(const Plan& q, Gemm& p, void* scratch, size_t scratch_bytes, cudaStream_t stream, bool chained) {
  if (q.scratch() > 0) {
    if (scratch == nullptr || scratch_bytes < q.scratch())
      return set_error(TGT_ERR_WORKSPACE, "scratch holds %zu bytes, %zu needed", scratch_bytes, q.scratch());
    TGT_CHECK_ARG(aligned16(scratch), "scratch must be 16-byte aligned");
    p.partial = static_cast<float*>(scratch);
  }
  if constexpr (!PAIR && !B_MN && BN <= 128) {
    if (q.cut.split == 2) return launch<BN, PAIR, A_MN, B_MN, FINISH, 2>(p, q.walkers, stream, chained);
    if (q.cut.split == 4) return launch<BN, PAIR, A_MN, B_MN, FINISH, 4>(p, q.walkers, stream, chained);
    if (q.cut.split == 8) return launch<BN, PAIR, A_MN, B_MN, FINISH, 8>(p, q.walkers, stream, chained);
  }
  TGT_RETURN_IF(launch<BN, PAIR, A_MN, B_MN, FINISH>(p, q.walkers, stream, chained));
  if constexpr (A_MN) {
    if (q.shared() == 0) return TGT_OK;
    const gemm::SumParts s{p.partial, {p.out[0], p.out[1]}, p.m, p.n, q.m_tiles, q.n_tiles,
                           q.product_tiles, q.whole, q.chunks, q.walkers};
    const dim3 grid(q.shared(), q.cut.rows() / 32 * BN / 64);
    if (q.walkers / q.shared() > 8) gemm::sum_parts_kernel<BN, PAIR, 4><<<grid, 1024, 0, stream>>>(s);
    else gemm::sum_parts_kernel<BN, PAIR, 1><<<grid, 256, 0, stream>>>(s);
    TGT_CHECK_CUDA(cudaGetLastError());
  }
  return TGT_OK;
}
template <bool A_MN, bool B_MN, gemm::Finish FINISH>
int launch_plan(const Plan& q, Gemm& p, void* scratch, size_t scratch_bytes, cudaStream_t stream, bool chained = false) {
  q.into(p);
  if (q.cut.pair) {
    if (q.cut.bn == 256) return launch_cut<256, true, A_MN, B_MN, FINISH>(q, p, scratch, scratch_bytes, stream, chained);
    return launch_cut<128, true, A_MN, B_MN, FINISH>(q, p, scratch, scratch_bytes, stream, chained);
  }
  if (q.cut.bn == 256) return launch_cut<256, false, A_MN, B_MN, FINISH>(q, p, scratch, scratch_bytes, stream, chained);
  if (q.cut.bn == 128) return launch_cut<128, false, A_MN, B_MN, FINISH>(q, p, scratch, scratch_bytes, stream, chained);
  if constexpr (FINISH != gemm::kGated) return launch_cut<64, false, A_MN, B_MN, FINISH>(q, p, scratch, scratch_bytes, stream, chained);
  return set_error(TGT_ERR_INVALID, "no tile of %d columns", q.cut.bn);
}

// the finishes' times of 256 columns (us)
constexpr double kPlainTime = 3, kPlusTime = 4, kGatedTime = 3, kKeptTime = 4, kGradTime = 5;
Plan weight_grad_plan(int count, int64_t rows, int out_features, int in_features) {
  return plan_for(count, out_features, in_features, 64, tiles_of(rows, gemm::kChunk), kPlainTime, kShare);
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
__global__ void __launch_bounds__(kGateThreads) gate_kernel(const float4* gate, const float4* up, int64_t n, int act, float4* h) {
  with_activation(act, [&](auto a) {
    for (int64_t i = blockIdx.x * int64_t(kGateThreads) + threadIdx.x; i < n; i += int64_t(gridDim.x) * kGateThreads)
      h[i] = gated<decltype(a)::value>(__ldg(gate + i), __ldg(up + i));
  });
}
// dgate holds dh and receives dgate
__global__ void __launch_bounds__(kGateThreads) gate_grad_kernel(const float4* gate, const float4* up, int64_t n, int act,
                                                                 float4* dgate, float4* dup) {
  with_activation(act, [&](auto a) {
    for (int64_t i = blockIdx.x * int64_t(kGateThreads) + threadIdx.x; i < n; i += int64_t(gridDim.x) * kGateThreads) {
      float4 dg, du;
      gated_grad<decltype(a)::value>(dgate[i], __ldg(gate + i), __ldg(up + i), dg, du);
      dgate[i] = dg;
      dup[i] = du;
    }
  });
}
int gate_grid(int64_t n) {
  const int64_t want = (n + kGateThreads - 1) / kGateThreads, most = int64_t(sm_count()) * 8;
  return int(want < most ? want : most);
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_gated_hidden(const void* x, const void* w_gate, const void* w_up, int64_t rows, int in, int mid, int act,
                                int dtype, void* h, void* gate, void* up, void* low, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, in, mid, dtype, act));
  TGT_CHECK_ARG((gate == nullptr) == (up == nullptr) && (dtype == TGT_F32 || (gate == nullptr) == (low == nullptr)),
                "gate, up and in bf16 low go together");
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(x && w_gate && w_up && h, "x, w_gate, w_up and h must not be null");
  TGT_CHECK_ARG(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(h) && aligned16(gate) && aligned16(up) &&
                    aligned16(low),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    TGT_CHECK_ARG(gate != nullptr, "in fp32 gate and up must not be null");
    if (in > 1024 || mid > 1024 || in % 4 != 0 || mid % 4 != 0)
      return set_error(TGT_ERR_UNSUPPORTED, "in=%d mid=%d: both must be multiples of 4, at most 1024", in, mid);
    const float* w[2] = {static_cast<const float*>(w_gate), static_cast<const float*>(w_up)};
    const float* bias[2] = {nullptr, nullptr};
    float* c[2] = {static_cast<float*>(gate), static_cast<float*>(up)};
    if (gated_in_one(rows, in, 2 * mid))
      return linear_gated(static_cast<const float*>(x), w[0], w[1], rows, in, mid, act, static_cast<float*>(h), c[0], c[1], stream);
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
  const Plan q = plan_for(1, rows, 2 * mid, 128, tiles_of(in, gemm::kChunk), gate != nullptr ? kKeptTime : kGatedTime, kSplit);
  TGT_RETURN_IF(operand(&p.a[0], x, rows, in, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_gate, mid, in, false, q.cut.bn / 2));
  TGT_RETURN_IF(operand(&p.b[1], w_up, mid, in, false, q.cut.bn / 2));
  p.a[1] = p.a[0];
  p.out[0] = words(h);
  p.keep = gate != nullptr;
  p.out[1] = words(gate); p.out[2] = words(up); p.out[3] = words(low);
  p.m = int(rows); p.n = mid;
  p.source_chunks = q.chunks;
  p.act = act;
  return launch_plan<false, false, gemm::kGated>(q, p, nullptr, 0, stream);
}

namespace tgt {
namespace {

int gated_output(const void* h, const void* w_down, const void* add, int64_t rows, int mid, int out, int dtype, void* y,
                 cudaStream_t stream, bool chained) {
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
  const Plan q = plan_for(1, rows, out, 64, tiles_of(mid, gemm::kChunk), add != nullptr ? kPlusTime : kPlainTime, kSplit);
  TGT_RETURN_IF(operand(&p.a[0], h, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_down, out, mid, false, q.cut.b_rows()));
  p.a[1] = p.a[0]; p.b[1] = p.b[0];
  p.out[0] = words(y);
  p.read[0] = words(add);
  p.m = int(rows); p.n = out;
  p.source_chunks = q.chunks;
  return add != nullptr ? launch_plan<false, false, gemm::kPlus>(q, p, nullptr, 0, stream, chained)
                        : launch_plan<false, false, gemm::kPlain>(q, p, nullptr, 0, stream, chained);
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_gated_output(const void* h, const void* w_down, const void* add, int64_t rows, int mid, int out, int dtype,
                                void* y, void* stream) {
  return tgt::gated_output(h, w_down, add, rows, mid, out, dtype, y, static_cast<cudaStream_t>(stream), false);
}

extern "C" int tgt_gated_block(const void* x, const void* w_gate, const void* w_up, const void* w_down, const void* add, int64_t rows,
                               int in, int mid, int out, int act, int dtype, void* h, void* gate, void* up, void* low, void* y,
                               void* stream) {
  const int rc = tgt_gated_hidden(x, w_gate, w_up, rows, in, mid, act, dtype, h, gate, up, low, stream);
  return rc != TGT_OK ? rc : tgt::gated_output(h, w_down, add, rows, mid, out, dtype, y, static_cast<cudaStream_t>(stream), true);
}

extern "C" int tgt_gated_hidden_grad(const void* dy, const void* w_down, const void* gate, const void* up, const void* low,
                                     int64_t rows, int out, int mid, int act, int dtype, void* dgate, void* dup, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_RETURN_IF(check_widths(rows, out, mid, dtype, act));
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(dy && w_down && gate && up && (low || dtype == TGT_F32) && dgate && dup,
                "dy, w_down, gate, up, low, dgate and dup must not be null");
  TGT_CHECK_ARG(aligned16(dy) && aligned16(w_down) && aligned16(gate) && aligned16(up) && aligned16(low) && aligned16(dgate) &&
                    aligned16(dup),
                "tensors must be 16-byte aligned");
  if (dtype == TGT_F32) {
    if (out > 1024 || mid > 1024 || out % 4 != 0 || mid % 4 != 0)
      return set_error(TGT_ERR_UNSUPPORTED, "out=%d mid=%d: both must be multiples of 4, at most 1024", out, mid);
    if (gated_in_one(rows, out, mid))
      return linear_gated_grad(static_cast<const float*>(dy), static_cast<const float*>(w_down), static_cast<const float*>(gate),
                               static_cast<const float*>(up), rows, out, mid, act, static_cast<float*>(dgate), static_cast<float*>(dup),
                               stream);
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
  const Plan q = plan_for(1, rows, mid, 64, tiles_of(out, gemm::kChunk), kGradTime, kWhole);
  TGT_RETURN_IF(operand(&p.a[0], dy, rows, out, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_down, out, mid, true, q.cut.b_rows()));
  p.a[1] = p.a[0]; p.b[1] = p.b[0];
  p.out[0] = words(dgate);
  p.out[1] = words(dup);
  p.read[0] = words(gate); p.read[1] = words(up); p.read[2] = words(low);
  p.m = int(rows); p.n = mid;
  p.source_chunks = q.chunks;
  p.act = act;
  return launch_plan<false, true, gemm::kGatedGrad>(q, p, nullptr, 0, stream);
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
  const Plan q = plan_for(1, rows, in, 64, 2 * tiles_of(mid, gemm::kChunk), kPlainTime, kWhole);
  TGT_RETURN_IF(operand(&p.a[0], dgate, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.a[1], dup, rows, mid, false, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], w_gate, mid, in, true, q.cut.b_rows()));
  TGT_RETURN_IF(operand(&p.b[1], w_up, mid, in, true, q.cut.b_rows()));
  p.out[0] = words(dx);
  p.m = int(rows); p.n = in;
  p.source_chunks = q.chunks / 2;
  return launch_plan<false, true, gemm::kPlain>(q, p, nullptr, 0, stream);
}

extern "C" int tgt_gated_weight_grad_scratch_bytes(int count, int64_t rows, int out_features, int in_features, int dtype,
                                                   size_t* bytes) {
  using namespace tgt;
  TGT_CHECK_ARG(bytes != nullptr, "bytes is null");
  TGT_CHECK_ARG(count == 1 || count == 2, "count must be 1 or 2");
  TGT_RETURN_IF(check_widths(rows, out_features, in_features, dtype, TGT_ACT_SILU));
  if (dtype == TGT_F32) return tgt_linear_wgrad_multi_scratch_bytes(count, rows, in_features, out_features, bytes);
  *bytes = rows == 0 ? 0 : weight_grad_plan(count, rows, out_features, in_features).scratch();
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
  const Plan q = weight_grad_plan(count, rows, out_features, in_features);
  Gemm p{};
  TGT_RETURN_IF(expired_wait_word(&p.expired));
  for (int i = 0; i < 2; ++i)
    TGT_RETURN_IF(operand(&p.a[i], dy[i < count ? i : 0], rows, out_features, true, gemm::kTileM));
  TGT_RETURN_IF(operand(&p.b[0], x, rows, in_features, true, q.cut.b_rows()));
  p.b[1] = p.b[0];
  p.out[0] = words(dw[0]); p.out[1] = words(dw[count - 1]);
  p.m = out_features; p.n = in_features;
  p.source_chunks = q.chunks;
  return launch_plan<true, true, gemm::kPlain>(q, p, scratch, scratch_bytes, stream);
}
