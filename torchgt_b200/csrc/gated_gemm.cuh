// bf16 products with fp32 sums for the gated feed-forward block (gated_ffn.cu): one kernel whose operands lie either way
// round and whose finish is one of four.
//
//   D[m][n] = sum over k of A[m][k] B[n][k]
//
// A CTA takes tiles of 128 x BN.  One warp brings the operands in by TMA, 64 of k at a time, into a ring of stages; one
// issues tcgen05.mma on them, four a stage; eight finish the tile before from the other half of the tensor memory: 32 rows
// and half of the columns each, 32 columns at a time, through a small buffer of shared memory per warp from which TMA stores
// whole 64-byte rows.  An operand is `k`-major (rows of k, as x and the forward's weights) or `mn`-major (rows of m or n: what the
// gradients read without a transposed copy).
#pragma once

#include "linear_rows.cuh"
#include "tma.cuh"

namespace tgt {
namespace gemm {

constexpr int kTileM = 128, kChunk = 64;          // rows of a tile; of k, a stage
constexpr int kFinishWarps = 8, kThreads = 32 * (kFinishWarps + 2);
constexpr int kBytesA = kTileM * kChunk * 2;
constexpr int kStoreCols = 32, kStoreBytes = 32 * kStoreCols * 2;    // of a warp's buffers, two each

enum Finish {
  kPlain,        // out[0] = D + add
  kGated,        // columns are BN / 2 of the gate and BN / 2 of the up projection: out[0] = act(gate) up, out[1] = gate, out[2] = up
  kGatedGrad,    // D is dh: out[0] = dgate, out[1] = dup, from gate and up
  kPartial,      // fp32 sums of a part of k -> partial
};

struct Gemm {
  CUtensorMap a[2], b[2];      // kGated: b of the gate and of the up projection; kPartial: a of two products of one b; else sources
  CUtensorMap out[3];
  const __nv_bfloat16* add;    // kPlain; may be null
  const __nv_bfloat16* gate;   // kGatedGrad
  const __nv_bfloat16* up;
  float* partial;              // kPartial: [grid + tiles][BN][kTileM]
  int64_t m;
  int n;                       // columns of out (kGated: of each of the two)
  int m_tiles, n_tiles;        // kPartial with two products: m_tiles of both
  int chunks;                  // of k, over all sources
  int source_chunks;           // of the first source
  int product_tiles;           // kPartial: m_tiles of one product
  int act;
  bool keep;                   // kGated: out[1] and out[2] are wanted
  int* expired;                // expired_wait_word
};

__host__ __device__ constexpr int stages_of(int bn) { return bn == 256 ? 4 : bn == 128 ? 6 : 8; }
__host__ __device__ constexpr int stage_bytes(int bn) { return kBytesA + bn * kChunk * 2; }
constexpr int smem_bytes(int bn) {   // with room to start on 1,024 bytes
  return 1024 + stages_of(bn) * stage_bytes(bn) + kFinishWarps * 2 * kStoreBytes + (2 * stages_of(bn) + 5) * 8 + 16;
}
static_assert(smem_bytes(256) <= 227 * 1024 && smem_bytes(128) <= 227 * 1024 && smem_bytes(64) <= 227 * 1024, "one CTA per SM");

// The tiles, or with kPartial the parts of tiles, of a CTA, in the order all its warps take them.
template <bool PARTS>
struct Work {
  int64_t at, end;
  int chunks, tile, k0, k1;
  __device__ __forceinline__ explicit Work(const Gemm& p) : chunks(p.chunks) {
    const int64_t tiles = int64_t(p.m_tiles) * p.n_tiles;
    if (PARTS) {
      at = tiles * chunks * blockIdx.x / gridDim.x;
      end = tiles * chunks * (blockIdx.x + 1) / gridDim.x;
    } else {
      at = blockIdx.x;
      end = tiles;
    }
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    if (PARTS) {
      tile = int(at / chunks);
      k0 = int(at - int64_t(tile) * chunks);
      k1 = int(min(int64_t(chunks), k0 + end - at));
      at += k1 - k0;
    } else {
      tile = int(at);
      k0 = 0;
      k1 = chunks;
      at += gridDim.x;
    }
    return true;
  }
};
// Bands of eight row tiles, column by column: what CTAs work on at one time shares its rows and columns in the L2.
__device__ __forceinline__ void place(int m_tiles, int n_tiles, int tile, int& m_tile, int& n_tile) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * n_tiles), in_band = tile - band * kBand * n_tiles;
  const int rows = min(kBand, m_tiles - band * kBand);
  n_tile = in_band / rows;
  m_tile = band * kBand + in_band - n_tile * rows;
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// act(x), and with SLOPE its derivative.  The results are rounded to 8 bits: the fast exponential and quotient are 2^-20 off.
template <bool SLOPE>
__device__ __forceinline__ float activate(int act, float x, float& slope) {
  if (act == TGT_ACT_SILU) {
    const float s = sigmoid(x);
    if (SLOPE) slope = s * (1.f + x * (1.f - s));
    return x * s;
  }
  if (act == TGT_ACT_GELU) {
    const float cdf = normal_cdf(x);
    if (SLOPE) slope = cdf + x * (0.39894228040143267794f * __expf(-0.5f * x * x));
    return x * cdf;
  }
  if (SLOPE) slope = x <= 0.f ? 0.f : 1.f;
  return relu(x);
}

template <int BN, bool A_MN, bool B_MN, Finish FINISH>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Gemm p) {
  constexpr int kStages = stages_of(BN), kStage = stage_bytes(BN);
  constexpr bool kParts = FINISH == kPartial;
  extern __shared__ uint8_t s_raw[];
  const uint32_t s_ring = (tc::smem_address(s_raw) + 1023) & ~1023u;
  uint8_t* const s_rest = s_raw + (s_ring - tc::smem_address(s_raw)) + kStages * kStage;
  uint64_t* const s_full = reinterpret_cast<uint64_t*>(s_rest + kFinishWarps * 2 * kStoreBytes);
  uint64_t* const s_empty = s_full + kStages;
  uint64_t* const s_sums = s_empty + kStages;            // two: the sums of a half are complete
  uint64_t* const s_taken = s_sums + 2;                  // two: the sums of a half have been read
  uint64_t* const s_drained = s_taken + 2;
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_drained + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (warp == kFinishWarps && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      tma::prefetch(&p.a[i]);
      tma::prefetch(&p.b[i]);
    }
    for (int i = 0; i < kStages; ++i) {
      tma::barrier_init(s_full + i, 1);
      tma::barrier_init(s_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      tma::barrier_init(s_sums + i, 1);
      tma::barrier_init(s_taken + i, kFinishWarps);
    }
    tma::barrier_init(s_drained, 1);
    tma::barriers_ready();
  }
  if (warp == kFinishWarps + 1) tc::allocate<2 * BN>(s_tmem);
  tc::fence_before_barrier();
  __syncthreads();
  tc::fence_after_barrier();
  const uint32_t tmem = *s_tmem;
  Work<kParts> work(p);

  if (warp == kFinishWarps) {
    // ---- operands in ----
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;                                // an empty ring's stages count as taken
      bool ok = true;
      while (ok && work.next()) {
        int m_tile, n_tile, from_a = 0;
        place(p.m_tiles, p.n_tiles, work.tile, m_tile, n_tile);
        if (FINISH == kPartial && m_tile >= p.product_tiles) {
          m_tile -= p.product_tiles;
          from_a = 1;
        }
        const int m0 = m_tile * kTileM, n0 = n_tile * (FINISH == kGated ? BN / 2 : BN);
        for (int chunk = work.k0; chunk < work.k1; ++chunk) {
          if (!(ok = tc::wait(s_empty + stage, phase))) break;
          tma::arrive_expecting(s_full + stage, kStage);
          const bool second = !kParts && chunk >= p.source_chunks;
          const CUtensorMap* a = &p.a[kParts ? from_a : int(second)];
          const CUtensorMap* b = &p.b[FINISH == kGated || kParts ? 0 : int(second)];
          const int k = (second ? chunk - p.source_chunks : chunk) * kChunk;
          const uint32_t to_a = s_ring + stage * kStage, to_b = to_a + kBytesA;
          if constexpr (A_MN) {
#pragma unroll
            for (int i = 0; i < kTileM / 64; ++i) tma::load(to_a + i * 8192, a, m0 + i * 64, k, s_full + stage);
          } else {
            tma::load(to_a, a, k, m0, s_full + stage);
          }
          if constexpr (FINISH == kGated) {
            tma::load(to_b, b, k, n0, s_full + stage);
            tma::load(to_b + BN / 2 * kChunk * 2, &p.b[1], k, n0, s_full + stage);
          } else if constexpr (B_MN) {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) tma::load(to_b + i * 8192, b, n0 + i * 64, k, s_full + stage);
          } else {
            tma::load(to_b, b, k, n0, s_full + stage);
          }
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
      if (!ok) tc::report_expired_wait(p.expired);
      // no copy into this CTA's shared memory may be under way when it ends: the last turn of every stage
      for (int i = 0; i < kStages; ++i) tc::wait(s_full + i, i < stage ? phase ^ 1 : phase);
    }
  } else if (warp == kFinishWarps + 1) {
    // ---- products ----
    if (lane == 0) {
      constexpr uint32_t instr = tc::instruction(kTileM, BN, A_MN, B_MN);
      int stage = 0, half = 0;
      uint32_t phase = 0, taken[2] = {1, 1};
      bool ok = true;
      while (ok && work.next()) {
        if (!(ok = tc::wait(s_taken + half, taken[half]))) break;
        taken[half] ^= 1;
        tc::fence_after_barrier();
        for (int chunk = work.k0; chunk < work.k1; ++chunk) {
          if (!(ok = tc::wait(s_full + stage, phase))) break;
          tc::fence_after_barrier();
          const uint32_t a = s_ring + stage * kStage, b = a + kBytesA;
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k) {
            const uint64_t da = A_MN ? tc::mn_major(a + 2048 * k, 8192) : tc::k_major(a + 32 * k);
            const uint64_t db = B_MN ? tc::mn_major(b + 2048 * k, 8192) : tc::k_major(b + 32 * k);
            tc::multiply(tmem + half * BN, da, db, instr, chunk > work.k0 || k > 0);
          }
          tc::commit(s_empty + stage);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        tc::commit(s_sums + half);
        half ^= 1;
      }
      if (!ok) {
        tc::report_expired_wait(p.expired);
        tc::commit(s_drained);                           // products that still run write to the memory given back
        tc::wait(s_drained, 0);
      }
    }
  } else {
    // ---- sums out ----
    const int rows0 = warp % 4 * 32, side = warp / 4;
    const uint32_t s_store = tc::smem_address(s_rest) + warp * 2 * kStoreBytes;
    constexpr int kCols = FINISH == kGated ? BN / 2 : BN;                // columns of out in a tile
    int buffer = 0, half = 0;
    uint32_t complete[2] = {0, 0};
    bool ok = true;
    // 32 values of the calling thread's row -> out
    auto put = [&](const CUtensorMap* map, const float (&v)[32], int row, int col) {
      if (lane == 0) tma::groups_read<1>();              // the buffer's last store
      __syncwarp();
      const uint32_t to = s_store + buffer * kStoreBytes + lane * 64;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = to + ((i ^ (lane >> 1)) & 3) * 16;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(f32_to_bf16x2(v[8 * i], v[8 * i + 1])),
                     "r"(f32_to_bf16x2(v[8 * i + 2], v[8 * i + 3])), "r"(f32_to_bf16x2(v[8 * i + 4], v[8 * i + 5])),
                     "r"(f32_to_bf16x2(v[8 * i + 6], v[8 * i + 7]))
                     : "memory");
      }
      tc::publish_operands();
      __syncwarp();
      if (lane == 0) {
        if (row < p.m && col < p.n) tma::store(map, s_store + buffer * kStoreBytes, col, row);
        tma::end_group();
      }
      buffer ^= 1;
    };
    auto sums = [&](uint32_t at, float (&v)[32]) {
      uint32_t r[2][16];
      tc::read16(at, r[0]);
      tc::read16(at + 16, r[1]);
      tc::reads_done();
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = ok ? __uint_as_float(r[i / 16][i % 16]) : __int_as_float(0x7fffffff);
    };
    // 32 columns of a row of a matrix like out
    auto fetch = [&](const __nv_bfloat16* from, int64_t row, int col, uint4 (&v)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = row < p.m && col + 8 * i < p.n ? __ldg(reinterpret_cast<const uint4*>(from + row * p.n + col) + i)
                                              : make_uint4(0u, 0u, 0u, 0u);
    };
    auto widen8 = [](const uint4& w, float* f) {
      bf16x2_to_f32(w.x, f[0], f[1]); bf16x2_to_f32(w.y, f[2], f[3]);
      bf16x2_to_f32(w.z, f[4], f[5]); bf16x2_to_f32(w.w, f[6], f[7]);
    };
    while (work.next()) {
      int m_tile, n_tile;
      place(p.m_tiles, p.n_tiles, work.tile, m_tile, n_tile);
      const int row0 = m_tile * kTileM + rows0, col0 = n_tile * kCols + side * (kCols / 2);
      const int64_t row = row0 + lane;
      const uint32_t from = tmem + half * BN + (uint32_t(rows0) << 16) + side * (kCols / 2);
      if (ok && !(ok = tc::wait(s_sums + half, complete[half])) && lane == 0) tc::report_expired_wait(p.expired);
      ok = __all_sync(~0u, ok);
      complete[half] ^= 1;
      tc::fence_after_barrier();
#pragma unroll 1
      for (int j = 0; j < kCols / 2; j += 32) {
        const int col = col0 + j;
        float v[32];
        sums(from + j, v);
        if constexpr (FINISH == kPlain) {
          if (p.add != nullptr) {
            uint4 w[4];
            fetch(p.add, row, col, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float f[8];
              widen8(w[i], f);
#pragma unroll
              for (int x = 0; x < 8; ++x) v[8 * i + x] += f[x];
            }
          }
          put(&p.out[0], v, row0, col);
        } else if constexpr (FINISH == kGated) {
          float u[32];
          sums(from + BN / 2 + j, u);
          if (p.keep) {
            put(&p.out[1], v, row0, col);
            put(&p.out[2], u, row0, col);
          }
          float unused;
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = activate<false>(p.act, v[i], unused) * u[i];
          put(&p.out[0], v, row0, col);
        } else if constexpr (FINISH == kGatedGrad) {
          uint4 g[4], u[4];
          fetch(p.gate, row, col, g);
          fetch(p.up, row, col, u);
          float dg[32];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float gf[8], uf[8];
            widen8(g[i], gf);
            widen8(u[i], uf);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              float slope;
              const float a = activate<true>(p.act, gf[x], slope), dh = v[8 * i + x];
              dg[8 * i + x] = dh * uf[x] * slope;
              v[8 * i + x] = dh * a;
            }
          }
          put(&p.out[0], dg, row0, col);
          put(&p.out[1], v, row0, col);
        } else {
          // a column of 32 rows at a time: 128 bytes
          float* to = p.partial + (int64_t(blockIdx.x) + work.tile) * (BN * kTileM) + (side * (kCols / 2) + j) * kTileM + rows0 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) to[i * kTileM] = v[i];
        }
      }
      tc::fence_before_barrier();
      __syncwarp();
      if (lane == 0) tma::arrive(s_taken + half);
      half ^= 1;
    }
    if (lane == 0) tma::groups_done();
  }
  __syncwarp();
  tc::fence_before_barrier();
  __syncthreads();
  if (warp == kFinishWarps + 1) tc::release<2 * BN>(tmem);
}

// kPartial's results of a tile added in the order of k and rounded: out[which][m][n].  A block takes 32 rows x 64 columns.
struct SumParts {
  const float* partial;
  __nv_bfloat16* out[2];
  int64_t m;                 // of one product
  int n, m_tiles, n_tiles, product_tiles, chunks, ctas;
};
constexpr int kSumThreads = 256;
template <int BN>
__global__ void __launch_bounds__(kSumThreads) sum_parts_kernel(const SumParts p) {
  __shared__ float s_block[64][33];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tile = blockIdx.x, r0 = blockIdx.y % 4 * 32, c0 = blockIdx.y / 4 * 64;
  const int64_t all = int64_t(p.m_tiles) * p.n_tiles * p.chunks, begin = int64_t(tile) * p.chunks, end = begin + p.chunks;
  int m_tile, n_tile;
  place(p.m_tiles, p.n_tiles, tile, m_tile, n_tile);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  // the CTA that had the tile's first chunk, and those after it
  for (int64_t cta = ((begin + 1) * p.ctas - 1) / all; cta < p.ctas && all * cta / p.ctas < end; ++cta) {
    const float* from = p.partial + (cta + tile) * (BN * kTileM) + (c0 + warp * 8) * kTileM + r0 + lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += __ldg(from + i * kTileM);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_block[warp * 8 + i][lane] = s[i];
  __syncthreads();
  const int which = m_tile >= p.product_tiles;
  const int64_t row = int64_t(m_tile - which * p.product_tiles) * kTileM + r0 + threadIdx.x / 8;
  const int c = threadIdx.x % 8 * 8, col = n_tile * BN + c0 + c;
  if (row >= p.m || col >= p.n) return;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s_block[c + i][threadIdx.x / 8];
  Lane<__nv_bfloat16, 16>::store(p.out[which] + row * p.n + col, v);
}

}  // namespace gemm
}  // namespace tgt
