// Learned relative position bias of the attention's edges: the bias that tgt_sparse_attn_fwd takes per edge and head, from a
// table with a row per bucket of the distance between the edge's ends, and the gradient of the table.
//
//   offset = position[source] - position[destination];  bias[e] = table[bucket(offset)];  dtable[b] = sum of dbias[e] of b's edges
//
// A bucket is the number of borders that the distance reaches (both ways: the second half of the table is for sources
// behind the destination).  Borders are whole numbers made by the caller, so no logarithm decides on which side of one a distance
// lies.
// Forward: a warp takes 32 edges, a lane finds one edge's bucket, then the warp writes the 32 rows of bias as one run.
// Backward: a warp adds the rows of dbias to sums of its own in shared memory, one per bucket and lane: lanes are (edge of a
// group, head), so no two of them share a word or a bank, and what a hub's bucket costs is what any costs.  The sums
// of a CTA's warps and then of the CTAs are added in a fixed order: no atomics, the same bits every time.  Both directions are bound by the
// ids and the rows of bias; the forward keeps the buckets, 2 bytes an edge in the place of the 16 of two ids.
// The sums are fp32, a lane's own of up to some thousand terms: 1.2e-7 to 2.5e-7 from 64 bits in the 2-norm over all list lengths.
// us, 18.2 M edges x 8 heads, 870,001 positions: forward 217 (910 MB; without positions 146: two random reads an edge are requests of
// their own and keep the way to the L2 busy in 86 % of the cycles), backward 130 (issue slots 75 % busy, DRAM 56 %) and 9 for the
// last sums (620 MB); 526,450 edges 8.5, 8.4 and 4.5.
#include "tgt_common.cuh"

namespace tgt {
namespace {

constexpr int kMostBuckets = 512, kMostHeads = 256;
constexpr int kBiasThreads = 256;
constexpr int bias_threads(bool shared) { return shared ? 1024 : kBiasThreads; }
constexpr uint16_t kNoBucket = 0xffff;      // of an edge with an id outside the positions

struct BiasFwd {
  const void* source;          // ids
  const void* destination;
  const void* positions;       // may be null: the ids themselves
  int64_t n_positions, n_edges;
  const float* table;
  float* bias;
  uint16_t* buckets;           // may be null
  int heads, behind;           // behind: the first bucket of sources behind the destination, or 0
  int n_borders, search;       // search: the largest power of two up to n_borders, 0 without any
  unsigned share;              // 2^22 / pieces of a row, rounded up
  int32_t borders[kMostBuckets];
};

template <typename Id, typename Pos>
__device__ __forceinline__ int bucket_of(const BiasFwd& p, const int32_t* borders, int64_t e) {
  int64_t s = __ldcs(static_cast<const Id*>(p.source) + e), d = __ldcs(static_cast<const Id*>(p.destination) + e);
  if (p.positions != nullptr) {
    if (s < 0 || s >= p.n_positions || d < 0 || d >= p.n_positions) return kNoBucket;
    s = __ldg(static_cast<const Pos*>(p.positions) + s);
    d = __ldg(static_cast<const Pos*>(p.positions) + d);
  }
  // the difference of any two positions fits 64 bits without a sign
  const uint64_t far = s > d ? (p.behind > 0 ? uint64_t(s) - uint64_t(d) : 0) : uint64_t(d) - uint64_t(s);
  const int32_t distance = far > 0x7fffffffu ? 0x7fffffff : int32_t(far);
  int n = 0;
  for (int step = p.search; step > 0; step >>= 1)
    if (n + step <= p.n_borders && borders[n + step - 1] <= distance) n += step;
  return n + (s > d ? p.behind : 0);
}

// SHARED: 4, 8 or 16 heads, and the table lies in shared memory, a row as the eight pieces of 16 bytes that the lanes of a
// transaction take, each from banks of its own: its one, two or four pieces again and again.
template <typename Id, typename Pos, int VEC, bool SHARED>
__global__ void __launch_bounds__(bias_threads(SHARED), 2048 / bias_threads(SHARED)) position_bias_kernel(const __grid_constant__ BiasFwd p) {
  constexpr int kThreads = bias_threads(SHARED);
  __shared__ int32_t s_borders[kMostBuckets];
  extern __shared__ __align__(16) float4 s_table[];          // SHARED: [buckets][8]
  const int lane = threadIdx.x % 32, pieces = p.heads / VEC;
  for (int i = threadIdx.x; i < p.n_borders; i += kThreads) s_borders[i] = p.borders[i];
  if constexpr (SHARED) {
    const int buckets = (p.n_borders + 1) * (p.behind > 0 ? 2 : 1);
    for (int i = threadIdx.x; i < buckets * 8; i += kThreads)
      s_table[i] = __ldg(reinterpret_cast<const float4*>(p.table) + i / 8 * pieces + i % 8 % pieces);
  }
  __syncthreads();
  const int64_t warps = int64_t(gridDim.x) * (kThreads / 32);
  for (int64_t e0 = (int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32) * 32; e0 < p.n_edges; e0 += warps * 32) {
    const int64_t e = e0 + lane;
    int bucket = kNoBucket;
    if (e < p.n_edges) {
      bucket = bucket_of<Id, Pos>(p, s_borders, e);
      if (p.buckets != nullptr) p.buckets[e] = uint16_t(bucket);
    }
    const int live = int(min(p.n_edges - e0, int64_t(32))) * pieces;
    float* const out = p.bias + e0 * p.heads;
    for (int i = 0; i < pieces; ++i) {
      const int piece = i * 32 + lane;
      const int of = int((unsigned(piece) * p.share) >> 22);
      const int b = __shfl_sync(0xffffffffu, bucket, of);
      if (piece >= live) continue;
      const float nan = __int_as_float(0x7fffffff);
      if constexpr (VEC == 4) {
        float4 v = make_float4(nan, nan, nan, nan);
        if (b != kNoBucket)
          v = SHARED ? s_table[b * 8 + lane % 8] : __ldg(reinterpret_cast<const float4*>(p.table) + b * pieces + (piece - of * pieces));
        __stcs(reinterpret_cast<float4*>(out) + piece, v);
      } else {
        out[piece] = b != kNoBucket ? __ldg(p.table + b * pieces + (piece - of * pieces)) : nan;
      }
    }
  }
}

struct BiasBwd {
  const float* dbias;
  const uint16_t* buckets;
  float* partial;              // [gridDim.x][n_buckets][heads]
  int64_t n_edges;
  int n_buckets, heads;
};

struct TableSum {
  const float* partial;        // [ctas][values]
  float* dtable;
  int ctas, values;
};

// HP: heads of a warp, a power of two; blockIdx.y picks which
template <int HP>
__global__ void __launch_bounds__(kBiasThreads) position_bias_grad_kernel(const BiasBwd p) {
  extern __shared__ float s_sums[];                          // [warps][n_buckets][32]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  float* const sums = s_sums + warp * p.n_buckets * 32;
  for (int b = 0; b < p.n_buckets; ++b) sums[b * 32 + lane] = 0.f;
  constexpr int kSlots = 32 / HP;                            // edges of a group
  const int slot = lane / HP, h0 = blockIdx.y * 32, h = h0 + lane % HP;
  const bool has_head = h < p.heads;
  // A batch is eight groups; the next one's rows are on their way while this one's are added, whose sums in shared memory wait
  // for one another (as far as the compiler can know).
  constexpr int kBatch = 8, kEdges = kBatch * kSlots, kWords = kEdges > 32 ? kEdges / 32 : 1;
  const int64_t step = int64_t(gridDim.x) * warps * kEdges;
  int64_t e0 = (int64_t(blockIdx.x) * warps + warp) * kEdges;
  float next[kBatch];
  int next_bucket[kWords];
  auto load = [&]() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int64_t e = e0 + 32 * k + lane;
      next_bucket[k] = e < p.n_edges && 32 * k + lane < kEdges ? __ldcs(p.buckets + e) : kNoBucket;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t e = e0 + i * kSlots + slot;
      next[i] = has_head && e < p.n_edges ? __ldcs(p.dbias + e * p.heads + h) : 0.f;
    }
  };
  load();
  while (e0 < p.n_edges) {
    float v[kBatch];
    int bucket[kWords];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = next[i];
#pragma unroll
    for (int k = 0; k < kWords; ++k) bucket[k] = next_bucket[k];
    e0 += step;
    load();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int b = __shfl_sync(0xffffffffu, bucket[i * kSlots / 32], i * kSlots % 32 + slot);
      if (b != kNoBucket) sums[b * 32 + lane] += v[i];
    }
  }
  release_dependents();
  __syncthreads();
  for (int i = threadIdx.x; i < p.n_buckets * HP; i += blockDim.x) {
    const int b = i / HP, head = i % HP;
    if (h0 + head >= p.heads) continue;
    float s = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int k = 0; k < kSlots; ++k) s += s_sums[(w * p.n_buckets + b) * 32 + k * HP + head];
    p.partial[(int64_t(blockIdx.x) * p.n_buckets + b) * p.heads + h0 + head] = s;
  }
}

// A block adds 32 values of the CTAs' sums: 32 warps, eight in flight each.
constexpr int kTableThreads = 1024;
__global__ void __launch_bounds__(kTableThreads) position_bias_table_kernel(const TableSum p) {
  __shared__ float s_part[32][33];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = blockIdx.x * 32 + lane;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = 0.f;
  dependent_wait();
  if (i < p.values)
    for (int c = warp; c < p.ctas; c += 32 * 8)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + 32 * j < p.ctas) s[j] += __ldcg(p.partial + int64_t(c + 32 * j) * p.values + i);
  s_part[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  float v = s_part[lane][warp];                   // of value `warp` of the block, the sums of warp `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0 && blockIdx.x * 32 + warp < p.values) p.dtable[blockIdx.x * 32 + warp] = v;
}

struct GradPlan {
  int hp, warps, smem, ctas;
};
constexpr int kMostSmem = 200 * 1024;
GradPlan plan_grad(int64_t n_edges, int n_buckets, int heads) {
  GradPlan g;
  g.hp = 1;
  while (g.hp < 32 && g.hp < heads) g.hp *= 2;
  const int per_warp = n_buckets * 128;
  g.warps = kMostSmem / per_warp;
  g.warps = g.warps > kBiasThreads / 32 ? kBiasThreads / 32 : g.warps;
  g.smem = g.warps * per_warp;
  int resident = kMostSmem / g.smem;
  resident = resident > 6 ? 6 : resident;
  // a CTA clears and adds up its sums: at least eight steps a warp before there is a second
  const int64_t batch = 8 * (32 / g.hp), steps = (n_edges + batch - 1) / batch, want = (steps + 8 * g.warps - 1) / (8 * g.warps);
  const int64_t most = int64_t(sm_count()) * resident;
  g.ctas = int(want < 1 ? 1 : want > most ? most : want);
  return g;
}

template <int HP>
int launch_grad(const BiasBwd& p, const GradPlan& g, cudaStream_t stream) {
  const int rc = allow_shared_memory<position_bias_grad_kernel<HP>>(kMostSmem);
  if (rc != TGT_OK) return rc;
  position_bias_grad_kernel<HP><<<dim3(g.ctas, (p.heads + 31) / 32), g.warps * 32, g.smem, stream>>>(p);
  TGT_CHECK_CUDA(cudaGetLastError());
  return TGT_OK;
}

int check_sizes(int64_t n_edges, int n_buckets, int heads) {
  TGT_CHECK_ARG(n_edges >= 0, "n_edges must be >= 0");
  TGT_CHECK_ARG(n_buckets >= 1 && heads >= 1, "the table must have a bucket and a head");
  if (n_buckets > kMostBuckets || heads > kMostHeads)
    return set_error(TGT_ERR_UNSUPPORTED, "%d buckets of %d heads: at most %d of %d", n_buckets, heads, kMostBuckets, kMostHeads);
  return TGT_OK;
}

// The table in the L1 / in shared memory, where many edges pay for large CTAs and for laying it out, us: 18.2 M edges, 8 heads 230 / 217;
// 4 M, 64,000 positions, 4 heads 46.7 / 45.5, 8 51.9 / 48.6, 16 66 / 62, 32 98 / 105; 1.2 M, 8 heads 17.3 / 16.3; 526,450 9.5 / 9.9; 45,056
// 3.4 / 4.2.  (The next edges' ids asked for a turn ahead: 217 -> 211 with positions, without 146 -> 156.)
constexpr int kSharedBuckets = 128;
template <typename Id, typename Pos>
int launch_forward(const BiasFwd& p, cudaStream_t stream) {
  const bool wide = p.heads % 4 == 0 && aligned16(p.table) && aligned16(p.bias);
  const int buckets = (p.n_borders + 1) * (p.behind > 0 ? 2 : 1);
  const bool shared = wide && 16 % p.heads == 0 && buckets <= kSharedBuckets && p.n_edges >= int64_t(8192) * sm_count();
  const int threads = bias_threads(shared);
  const int64_t want = (p.n_edges + threads - 1) / threads, most = int64_t(sm_count()) * (2048 / threads);
  const unsigned grid = unsigned(want < most ? want : most);
  if (shared) position_bias_kernel<Id, Pos, 4, true><<<grid, threads, buckets * 128, stream>>>(p);
  else if (wide) position_bias_kernel<Id, Pos, 4, false><<<grid, threads, 0, stream>>>(p);
  else position_bias_kernel<Id, Pos, 1, false><<<grid, threads, 0, stream>>>(p);
  TGT_CHECK_CUDA(cudaGetLastError());
  return TGT_OK;
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_edge_position_bias(const void* edge_index, int64_t n_edges, int wide_ids, const void* positions,
                                      int64_t n_positions, int wide_positions, const int32_t* borders, int n_borders,
                                      int both_ways, const float* table, int heads, float* bias, uint16_t* buckets,
                                      void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  TGT_CHECK_ARG(n_borders >= 0 && n_borders < kMostBuckets, "n_borders must be 0 to %d", kMostBuckets - 1);
  const int rc = check_sizes(n_edges, (n_borders + 1) * (both_ways ? 2 : 1), heads);
  if (rc != TGT_OK) return rc;
  TGT_CHECK_ARG(n_borders == 0 || borders != nullptr, "borders is null");
  for (int i = 0; i < n_borders; ++i)
    TGT_CHECK_ARG(borders[i] >= (i > 0 ? borders[i - 1] : 1), "borders must be positive and in order");
  TGT_CHECK_ARG(positions == nullptr || n_positions >= 0, "n_positions must be >= 0");
  if (n_edges == 0) return TGT_OK;
  TGT_CHECK_ARG(edge_index && table && bias, "edge_index, table and bias must not be null");
  BiasFwd p{};
  p.source = edge_index;
  p.destination = static_cast<const char*>(edge_index) + n_edges * (wide_ids ? 8 : 4);
  p.positions = positions;
  p.n_positions = n_positions; p.n_edges = n_edges;
  p.table = table; p.bias = bias; p.buckets = buckets;
  p.heads = heads;
  p.behind = both_ways ? n_borders + 1 : 0;
  p.n_borders = n_borders;
  p.search = n_borders > 0 ? 1 : 0;
  while (2 * p.search <= n_borders && p.search > 0) p.search *= 2;
  const int pieces = heads % 4 == 0 && aligned16(table) && aligned16(bias) ? heads / 4 : heads;
  p.share = ((1u << 22) + pieces - 1) / pieces;
  for (int i = 0; i < n_borders; ++i) p.borders[i] = borders[i];
  if (wide_ids)
    return wide_positions ? launch_forward<int64_t, int64_t>(p, stream) : launch_forward<int64_t, int32_t>(p, stream);
  return wide_positions ? launch_forward<int32_t, int64_t>(p, stream) : launch_forward<int32_t, int32_t>(p, stream);
}

extern "C" int tgt_edge_position_bias_grad_scratch_bytes(int64_t n_edges, int n_buckets, int heads, size_t* bytes) {
  using namespace tgt;
  TGT_CHECK_ARG(bytes != nullptr, "bytes is null");
  const int rc = check_sizes(n_edges, n_buckets, heads);
  if (rc != TGT_OK) return rc;
  *bytes = size_t(plan_grad(n_edges, n_buckets, heads).ctas) * n_buckets * heads * sizeof(float);
  return TGT_OK;
}

extern "C" int tgt_edge_position_bias_grad(const float* dbias, const uint16_t* buckets, int64_t n_edges, int n_buckets, int heads,
                                           float* dtable, void* scratch, size_t scratch_bytes, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_sizes(n_edges, n_buckets, heads);
  if (rc != TGT_OK) return rc;
  TGT_CHECK_ARG(dtable != nullptr, "dtable must not be null");
  const int values = n_buckets * heads;
  if (n_edges == 0) {
    TGT_CHECK_CUDA(cudaMemsetAsync(dtable, 0, size_t(values) * sizeof(float), stream));
    return TGT_OK;
  }
  TGT_CHECK_ARG(dbias && buckets, "dbias and buckets must not be null");
  const GradPlan g = plan_grad(n_edges, n_buckets, heads);
  const size_t need = size_t(g.ctas) * values * sizeof(float);
  if (scratch == nullptr || scratch_bytes < need)
    return set_error(TGT_ERR_WORKSPACE, "scratch holds %zu bytes, %zu needed", scratch_bytes, need);
  const BiasBwd p{dbias, buckets, static_cast<float*>(scratch), n_edges, n_buckets, heads};
  switch (g.hp) {
    case 1: rc = launch_grad<1>(p, g, stream); break;
    case 2: rc = launch_grad<2>(p, g, stream); break;
    case 4: rc = launch_grad<4>(p, g, stream); break;
    case 8: rc = launch_grad<8>(p, g, stream); break;
    case 16: rc = launch_grad<16>(p, g, stream); break;
    default: rc = launch_grad<32>(p, g, stream); break;
  }
  if (rc != TGT_OK) return rc;
  const TableSum sum{p.partial, dtable, g.ctas, values};
  TGT_CHECK_CUDA(launch_chained(position_bias_table_kernel, dim3((values + 31) / 32), kTableThreads, stream, kLinkStitch, sum));
  return TGT_OK;
}
