// bf16 products with fp32 sums for the gated feed-forward block (gated_ffn.cu): one kernel whose operands lie either way
// round and whose finish is one of four.  Of weight gradients, which are long sums for few results, the last tiles, those
// that do not fill all SMs, are shared out along k: their parts go to scratch and a second kernel adds them.
//
//   D[m][n] = sum over k of A[m][k] B[n][k]
//
// A CTA takes tiles of 128 x BN; or several (SPLIT) take one between them, each a part of k, and each finishes a part of
// the rows from all their sums, which they read from one another's shared memory; or two CTAs (PAIR) take tiles of 256 x BN
// together: each has 128 rows of A and of the sums and brings in half of B's rows, and the first issues the products for
// both, so a tile costs a third less of what the L2 hands out.  One warp brings the operands in by TMA, 64 of k at a time, into a ring of stages; one issues tcgen05.mma on them,
// four a stage; eight finish the tile before from the other half of the tensor memory: 32 rows and half of the columns
// each, 32 columns at a time.  A lane reads a row of the sums; what is read and written of global memory goes by four lanes
// to 64 bytes of a row, and 4 KB of shared memory per warp stand between the two.  An operand is `k`-major (rows of k, as x
// and the forward's weights) or `mn`-major (rows of m or n: what the gradients read without a transposed copy).
//
// TFLOP/s at 1.4 to 1.9 GHz (library's product in brackets where there is one): y of 18,944 rows 4,096 x 2,048 1,555
// (1,580); of 8,191 rows 5,632 x 2,048, 3.5 rounds of tiles in 4, 1,391 (1,540); h of 8,191 rows 2,048 x 5,632 1,540, with
// what is kept 16,384 rows 1,024 x 2,816 1,170 (370 MB out); dgate and dup 800 (460 MB in and out); dx 1,400; the weights'
// gradients 1,380.  What bounds them, 16,384 rows 1,024 x 2,816: the tensor pipe is active in 85 % of the cycles of dWg and dWu, 77 of
// dx, 67 of h with what is kept (shared memory's pipe 52 %, 315 MB out), and under a long run there is the power cap; in dgate and
// dup 43, with DRAM at 54 % and shared memory's pipe at 44: there the eight finishing warps, on 37 % of the issue slots, wait for
// what they read.
#pragma once

#include "linear_rows.cuh"
#include "tma.cuh"

namespace tgt {
namespace gemm {

constexpr int kTileM = 128, kChunk = 64;          // rows of a tile; of k, a stage
constexpr int kFinishWarps = 8, kThreads = 32 * (kFinishWarps + 2);
constexpr int kBytesA = kTileM * kChunk * 2;
constexpr int kBlockBytes = 4096;                 // of a warp: 32 rows of 32 sums, or two of 32 results

enum Finish {
  kPlain,        // out[0] = D
  kPlus,         // out[0] = D + add
  kGated,        // columns are BN / 2 of the gate and BN / 2 of the up projection: out[0] = act(gate) up, out[1..3] = both, kept
  kGatedGrad,    // D is dh: out[0] = dgate, out[1] = dup, from the two as they were kept
};

struct Gemm {
  // of two sources (k one after the other), or a of two products of one b, or (kGated) b of the two projections
  CUtensorMap a[2], b[2];
  uint16_t* out[4];            // [m][n]; of two products out[0] and out[1]
  const uint16_t* read[3];     // kPlus: add; kGatedGrad: the three that were kept
  float* partial;              // [walkers + tiles that are shared][CTAs of a tile][BN][kTileM]
  int m;
  int n;                       // columns of out (kGated: of each of the two)
  int m_tiles, n_tiles;        // m_tiles of all products
  int whole;                   // tiles that are not shared, the first (all but of weight gradients)
  int chunks;                  // of k, over all sources
  int source_chunks;           // of the first source
  int product_tiles;           // m_tiles of one product
  int act;
  bool keep;                   // kGated: out[1..3] are wanted
  int* expired;                // expired_wait_word
};

// What a CTA keeps in shared memory: stages of 64 of k of its rows of A and `rows` of B, then per finishing warp the block
// above and 2 KB of what the finish reads of every matrix, then the barriers.
__host__ __device__ constexpr int read_by(Finish f) { return f == kGatedGrad ? 3 : f == kPlus ? 1 : 0; }
__host__ __device__ constexpr int stage_bytes(int rows) { return kBytesA + rows * kChunk * 2; }
__host__ __device__ constexpr int warp_bytes(Finish f) { return kBlockBytes + read_by(f) * 2048; }
__host__ __device__ constexpr int stages_of(int rows, Finish f) {
  const int fit = (227 * 1024 - 1024 - 256 - kFinishWarps * warp_bytes(f)) / stage_bytes(rows);
  return fit < 8 ? fit : 8;
}
constexpr int smem_bytes(int rows, Finish f) {   // with room to start on 1,024 bytes
  return 1024 + stages_of(rows, f) * stage_bytes(rows) + kFinishWarps * warp_bytes(f) + (2 * stages_of(rows, f) + 5) * 8 + 16;
}
static_assert(smem_bytes(256, kGatedGrad) <= 227 * 1024 && smem_bytes(256, kPlain) <= 227 * 1024 && smem_bytes(64, kPlain) <= 227 * 1024,
              "one CTA per SM");

// ---- what one CTA or a pair does with the tensor cores -------------------------------------------------------------
template <bool PAIR, int COLS>
__device__ __forceinline__ void allocate(uint32_t* slot) {       // by one warp, of each CTA of a pair
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_address(slot)), "n"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    tc::allocate<COLS>(slot);
  }
}
template <bool PAIR, int COLS>
__device__ __forceinline__ void release(uint32_t address) {      // by the warps that allocated
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "n"(COLS));
  else tc::release<COLS>(address);
}
template <bool PAIR>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"(uint32_t(add)) : "memory");
  } else {
    tc::multiply(d, a, b, instr, add);
  }
}
// bar, of both CTAs of a pair, completes a phase when all products this thread has issued are done
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     tc::smem_address(bar)),
                 "h"(uint16_t(3))
                 : "memory");
  } else {
    tc::commit(bar);
  }
}
// address of the first CTA's copy of something in shared memory
template <bool PAIR>
__device__ __forceinline__ uint32_t first_ctas(uint32_t address) {
  if constexpr (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(address) : "r"(address));
  return address;
}
__device__ __forceinline__ void cluster_barrier() {              // every thread of all CTAs, a warp together
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 16 bytes of shared memory of CTA `cta` of the cluster, at the place that `address` is in this one's
__device__ __forceinline__ float4 load_of(uint32_t address, int cta) {
  float4 v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address), "r"(cta) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t word_of(uint32_t address, int cta) {
  uint32_t v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
               : "=r"(v) : "r"(address), "r"(cta) : "memory");
  return v;
}
template <bool PAIR>
__device__ __forceinline__ void load(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (PAIR) {      // the bytes count at the first CTA's barrier
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            to),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    tma::load(to, map, x, y, bar);
  }
}

// The tiles of a walker (a CTA, or a pair of them), in the order all its warps take them: whole ones round by round, then its
// share of the chunks of the others, which is a part of a tile or of several.  With SPLIT the CTA's part of the one tile of its cluster.
template <int SPLIT>
struct Work {
  int64_t at, end;             // of the shared chunks
  int next_tile, whole, step, chunks, tile, k0, k1;
  __device__ __forceinline__ Work(const Gemm& p, int walker, int walkers)
      : next_tile(walker), whole(p.whole), step(walkers), chunks(p.chunks) {
    const int64_t shared = (int64_t(p.m_tiles) * p.n_tiles - p.whole) * chunks;
    at = shared * walker / walkers;
    end = shared * (walker + 1) / walkers;
  }
  __device__ __forceinline__ bool next() {
    if (next_tile < whole) {
      tile = next_tile;
      next_tile += step;
      k0 = SPLIT == 1 ? 0 : int(int64_t(chunks) * (blockIdx.x % SPLIT) / SPLIT);
      k1 = SPLIT == 1 ? chunks : int(int64_t(chunks) * (blockIdx.x % SPLIT + 1) / SPLIT);
      return true;
    }
    if (at >= end) return false;
    const int of = int(at / chunks);
    tile = whole + of;
    k0 = int(at - int64_t(of) * chunks);
    k1 = int(min(int64_t(chunks), k0 + end - at));
    at += k1 - k0;
    return true;
  }
  __device__ __forceinline__ bool part() const { return tile >= whole; }
};
// Bands of eight row tiles, column by column: what CTAs work on at one time shares its rows and columns in the L2.
__device__ __forceinline__ void place(int m_tiles, int n_tiles, int tile, int& m_tile, int& n_tile) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * n_tiles), in_band = tile - band * kBand * n_tiles;
  const int rows = min(kBand, m_tiles - band * kBand);
  n_tile = in_band / rows;
  m_tile = band * kBand + in_band - n_tile * rows;
}

// 1 / (1 + exp(-x)): 0 and 1 at the ends of the range, NaN stays
__device__ __forceinline__ float sigmoid(float x) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
// act(x), and with SLOPE its derivative.  The results are rounded to 8 bits: the fast exponential and quotient are 2^-20 off, and by
// the rounding of the power |x| 2^-23 more (2^-17 at -64).
template <int ACT, bool SLOPE>
__device__ __forceinline__ float activate(float x, float& slope) {
  if constexpr (ACT == TGT_ACT_SILU) {
    const float s = sigmoid(x);
    if (SLOPE) slope = s * (1.f + x * (1.f - s));
    return x * s;
  } else if constexpr (ACT == TGT_ACT_GELU) {
    const float cdf = normal_cdf(x);
    if (SLOPE) slope = cdf + x * (0.39894228040143267794f * __expf(-0.5f * x * x));
    return x * cdf;
  } else {
    if (SLOPE) slope = x <= 0.f ? 0.f : 1.f;
    return relu(x);
  }
}
// How the two projections are kept for the gradients: the upper 16 bits of each fp32 sum, and the 8 bits below those of
// both in a third word.  Their rounding would be in every gradient, next to the roundings of dgate, dup and the result that
// cannot be avoided: kept in bf16 dx, dWg and dWu are 3.1e-3 from 64 bits (2-norm), with the 8 bits 2.3e-3, rounding the
// results alone 1.7e-3.
__device__ __forceinline__ uint32_t upper_pair(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ uint32_t lower_pair(float g0, float u0, float g1, float u1) {
  return __byte_perm(__byte_perm(__float_as_uint(g0), __float_as_uint(u0), 0x0051),
                     __byte_perm(__float_as_uint(g1), __float_as_uint(u1), 0x0051), 0x5410);
}
// the gate's (which 0) or the up projection's (1) value i of a pair; the last byte, of which nothing is known, is the one before
// it again
__device__ __forceinline__ float whole(uint32_t upper, uint32_t lower, int i, int which) {
  return __uint_as_float(__byte_perm(lower, upper, i == 0 ? (which == 0 ? 0x5400 : 0x5411) : (which == 0 ? 0x7622 : 0x7633)));
}

template <int BN, bool PAIR, bool A_MN, bool B_MN, Finish FINISH, int SPLIT = 1>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Gemm p) {
  constexpr int kRowsB = PAIR ? BN / 2 : BN, kStages = stages_of(kRowsB, FINISH), kStage = stage_bytes(kRowsB);
  constexpr int kCtas = PAIR ? 2 : 1, kTileRows = kTileM * kCtas;
  static_assert(SPLIT == 1 || (!PAIR && FINISH != kGatedGrad && kStages * kStage >= kTileM * BN * 4), "sums in the place of the ring");
  constexpr bool kShares = A_MN && FINISH == kPlain;     // weight gradients: few tiles, long sums
  extern __shared__ uint8_t s_raw[];
  const uint32_t s_ring = (tc::smem_address(s_raw) + 1023) & ~1023u;
  uint8_t* const s_rest = s_raw + (s_ring - tc::smem_address(s_raw)) + kStages * kStage;
  uint64_t* const s_full = reinterpret_cast<uint64_t*>(s_rest + kFinishWarps * warp_bytes(FINISH));   // of a pair the first CTA's
  uint64_t* const s_empty = s_full + kStages;
  uint64_t* const s_sums = s_empty + kStages;            // two: the sums of a half are complete
  uint64_t* const s_taken = s_sums + 2;                  // two: the sums of a half have been read; of a pair the first CTA's
  uint64_t* const s_drained = s_taken + 2;
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_drained + 1);     // and, next to it, whether a wait of a split tile ran out
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR ? blockIdx.x % 2 : 0;            // in the pair: clusters of two along x
  const int walker = blockIdx.x / (kCtas * SPLIT);

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
      tma::barrier_init(s_taken + i, kFinishWarps * kCtas);
    }
    tma::barrier_init(s_drained, 1);
    s_tmem[1] = 0u;
    tma::barriers_ready();
  }
  __syncwarp();
  if (FINISH == kGated) release_dependents();            // the product of h, if it was launched so
  if (warp == kFinishWarps + 1) allocate<PAIR, 2 * BN>(s_tmem);
  tc::fence_before_barrier();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();
  tc::fence_after_barrier();
  const uint32_t tmem = *s_tmem;
  dependent_wait();                                      // for h; before any wait here that has a limit
  Work<SPLIT> work(p, walker, gridDim.x / (kCtas * SPLIT));

  // The two warps that feed the tensor cores go through their loops together and elect a lane where something is issued: in code that a
  // lane runs alone the compiler cannot keep what an instruction takes in uniform registers (tiles of 128 x 128 and 128 x 64
  // took 0.33 us for 64 of k whatever their operands, 8,191 rows of 5,632 x 2,048 205 and 366 us).
  if (warp == kFinishWarps) {
    // ---- operands in ----
    int stage = 0;
    uint32_t phase = 1;                                  // an empty ring's stages count as taken
    const uint32_t full = first_ctas<PAIR>(tc::smem_address(s_full));
    bool ok = true;
    while (ok && work.next()) {
      int m_tile, n_tile;
      place(p.m_tiles, p.n_tiles, work.tile, m_tile, n_tile);
      const bool other = m_tile >= p.product_tiles;      // of two products
      if (other) m_tile -= p.product_tiles;
      const int m0 = m_tile * kTileRows + rank * kTileM;
      const int n0 = FINISH == kGated ? n_tile * (BN / 2) : n_tile * BN + rank * kRowsB;
      for (int chunk = work.k0; chunk < work.k1; ++chunk) {
        if (!(ok = tma::wait(s_empty + stage, phase))) break;
        if (tc::elect()) {
          if (rank == 0) tma::arrive_expecting(s_full + stage, kCtas * kStage);
          const uint32_t bar = full + stage * 8;
          const bool second = chunk >= p.source_chunks;
          const CUtensorMap* a = &p.a[second || other];
          const CUtensorMap* b = &p.b[FINISH == kGated ? rank : int(second)];
          const int k = (second ? chunk - p.source_chunks : chunk) * kChunk;
          const uint32_t to_a = s_ring + stage * kStage, to_b = to_a + kBytesA;
          if constexpr (A_MN) {
#pragma unroll
            for (int i = 0; i < kTileM / 64; ++i) load<PAIR>(to_a + i * 8192, a, m0 + i * 64, k, bar);
          } else {
            load<PAIR>(to_a, a, k, m0, bar);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int i = 0; i < kRowsB / 64; ++i) load<PAIR>(to_b + i * 8192, b, n0 + i * 64, k, bar);
          } else {
            load<PAIR>(to_b, b, k, n0, bar);
            if constexpr (FINISH == kGated && !PAIR) load<PAIR>(to_b + BN / 2 * kChunk * 2, &p.b[1], k, n0, bar);
          }
        }
        __syncwarp();
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
    if (!ok && lane == 0) tc::report_expired_wait(p.expired);
    // no copy into shared memory may be under way when the CTAs end: the last turn of every stage
    if (rank == 0)
      for (int i = 0; i < kStages; ++i) tc::wait(s_full + i, i < stage ? phase ^ 1 : phase);
  } else if (warp == kFinishWarps + 1) {
    // ---- products ----
    if (rank == 0) {
      constexpr uint32_t instr = tc::instruction(kTileRows, BN, A_MN, B_MN);
      int stage = 0, half = 0;
      uint32_t phase = 0, taken = 1;                     // of the half: both change together
      bool ok = true;
      while (ok && work.next()) {
        if (!(ok = tma::wait(s_taken + half, taken))) break;
        tc::fence_after_barrier();
        for (int chunk = work.k0; chunk < work.k1; ++chunk) {
          if (!(ok = tma::wait(s_full + stage, phase))) break;
          tc::fence_after_barrier();
          const uint32_t a = s_ring + stage * kStage, b = a + kBytesA;
          if (tc::elect()) {
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k) {
              const uint64_t da = A_MN ? tc::mn_major(a + 2048 * k, 8192) : tc::k_major(a + 32 * k);
              const uint64_t db = B_MN ? tc::mn_major(b + 2048 * k, 8192) : tc::k_major(b + 32 * k);
              multiply<PAIR>(tmem + half * BN, da, db, instr, chunk > work.k0 || k > 0);
            }
            commit<PAIR>(s_empty + stage);
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        if (tc::elect()) commit<PAIR>(s_sums + half);
        __syncwarp();
        if (half == 1) taken ^= 1;
        half ^= 1;
      }
      if (!ok) {
        if (lane == 0) tc::report_expired_wait(p.expired);
        if (tc::elect()) commit<PAIR>(s_drained);       // products that still run write to the memory given back
        __syncwarp();
        tc::wait(s_drained, 0);
      }
    }
  } else {
    // ---- sums out ----
    const int rows0 = warp % 4 * 32, side = warp / 4;
    uint8_t* const s_block = s_rest + warp * warp_bytes(FINISH);
    constexpr int kCols = FINISH == kGated ? BN / 2 : BN;                // columns of out in a tile
    int buffer = 0, half = 0;
    uint32_t complete = 0;                               // of the half: both change together
    bool ok = true;
    // In the pass over global memory a lane has four pieces of 8 columns: piece `piece` of rows `first`, first + 8, ...
    const int first = lane / 4, piece = lane % 4;
    // 32 rows of 32 results, a lane's row by four words a time -> out
    auto put = [&](uint16_t* to, int row0, int col0, auto&& word) {
      uint8_t* const into = s_block + buffer * (kBlockBytes / 2);        // read two turns ago, by all lanes before the last
      buffer ^= 1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(into + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16) =
            make_uint4(word(8 * i), word(8 * i + 2), word(8 * i + 4), word(8 * i + 6));
      __syncwarp();
      const int col = col0 + 8 * piece;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = first + 8 * i;
        const uint4 v = *reinterpret_cast<const uint4*>(into + r * 64 + ((piece ^ (r >> 1)) & 3) * 16);
        if (row0 + r < p.m && col < p.n) *reinterpret_cast<uint4*>(to + (row0 + r) * int64_t(p.n) + col) = v;
      }
    };
    // 32 rows of 32 sums by rows in, by pieces out
    auto turn = [&](const float (&v)[32]) {
      __syncwarp();                                      // the sums before these have been read
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<float4*>(s_block + lane * 128 + ((i ^ lane) & 7) * 16) =
            make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      __syncwarp();
    };
    auto turned = [&](int r, float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(s_block + r * 128 + (((2 * piece + i) ^ r) & 7) * 16);
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
    };
    auto sums = [&](uint32_t at, float (&v)[32]) {
      uint32_t r[2][16];
      __syncwarp();                                      // lanes without a row or a column have left the stores before this
      tc::read16(at, r[0]);
      tc::read16(at + 16, r[1]);
      tc::reads_done();
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i / 16][i % 16]);
      if (!ok) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7fffffff);
      }
    };
    // What the finish reads of global memory comes by asynchronous copies into places of the lane's own, a piece of 8 columns
    // of every matrix at a time: as soon as a piece has been read its place is filled with the piece of the next 32 columns, or of
    // the next tile.  (As loads into registers they were waited for a piece at a time: dgate and dup of 16,384 x 2,816 152 us.)
    constexpr int kRead = SPLIT == 1 ? read_by(FINISH) : 0;
    const uint32_t s_read = tc::smem_address(s_block + kBlockBytes + lane * 16);
    auto fetch = [&](int i, int row0, int col0) {
      const int r = row0 + first + 8 * i, col = col0 + 8 * piece;
      const bool there = r < p.m && col < p.n;
      const int64_t at = there ? r * int64_t(p.n) + col : 0;
#pragma unroll
      for (int k = 0; k < kRead; ++k)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s_read + (k * 4 + i) * 512), "l"(p.read[k] + at),
                     "r"(there ? 16 : 0)
                     : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto fetched = [&](int i, uint4 (&v)[kRead > 0 ? kRead : 1]) {
      asm volatile("cp.async.wait_group 3;" ::: "memory");           // but the last three: the oldest of four
#pragma unroll
      for (int k = 0; k < kRead; ++k) v[k] = *reinterpret_cast<const uint4*>(s_block + kBlockBytes + lane * 16 + (k * 4 + i) * 512);
    };
    Work<SPLIT> ahead = work;                           // a step in front of `work`: what is fetched
    int ahead_row = 0, ahead_col = 0, ahead_j = kCols;
    auto advance = [&]() {
      ahead_j += 64;
      if (ahead_j >= kCols) {
        ahead_j = side * 32;
        int m_tile, n_tile;
        if (ahead.next()) {
          place(p.m_tiles, p.n_tiles, ahead.tile, m_tile, n_tile);
          ahead_row = m_tile * kTileRows + rank * kTileM + rows0;
          ahead_col = n_tile * kCols;
        } else {
          ahead_row = p.m;                               // nothing is read: zeros
        }
      }
    };
    if constexpr (kRead > 0) {
      advance();
      for (int i = 0; i < 4; ++i) fetch(i, ahead_row, ahead_col + ahead_j);
    }
    while (work.next()) {
      int m_tile, n_tile;
      place(p.m_tiles, p.n_tiles, work.tile, m_tile, n_tile);
      const bool other = FINISH == kPlain && m_tile >= p.product_tiles;
      if (other) m_tile -= p.product_tiles;
      const int row0 = m_tile * kTileRows + rank * kTileM + rows0, col0 = n_tile * kCols;
      const uint32_t from = tmem + half * BN + (uint32_t(rows0) << 16);
      if (ok && !(ok = tc::wait(s_sums + half, complete)) && lane == 0) tc::report_expired_wait(p.expired);
      ok = __all_sync(~0u, ok);
      tc::fence_after_barrier();
      if constexpr (SPLIT > 1) {
        // in the place of the ring, which has been used up: rows of BN sums, their 16-byte pieces in an order by row
#pragma unroll 1
        for (int j = side * 32; j < BN; j += 64) {
          float v[32];
          sums(from + j, v);
          uint8_t* const to = s_raw + (s_ring - tc::smem_address(s_raw)) + (rows0 + lane) * (BN * 4);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(to + ((j / 4 + i) ^ (lane & 7)) * 16) =
                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        if (!ok && lane == 0) s_tmem[1] = 1u;            // copies that come late may write there still
      }
#pragma unroll 1
      for (int j = SPLIT == 1 ? side * 32 : kCols; j < kCols; j += 64) {
        const int col = col0 + j;
        float v[32];
        sums(from + j, v);
        if constexpr (kRead > 0) advance();
        if (kShares && work.part()) {
          // a column of 32 rows at a time: 128 bytes
          float* to = p.partial + ((int64_t(walker) + work.tile - p.whole) * kCtas + rank) * (BN * kTileM) + j * kTileM + rows0 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) to[i * kTileM] = v[i];
          continue;
        }
        if constexpr (FINISH == kPlain) {
          put(p.out[other], row0, col, [&](int i) { return f32_to_bf16x2(v[i], v[i + 1]); });
        } else if constexpr (FINISH == kPlus) {
          turn(v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = first + 8 * i;
            float d[8], f[8];
            uint4 add[1];
            fetched(i, add);
            fetch(i, ahead_row, ahead_col + ahead_j);
            turned(r, d);
            Lane<__nv_bfloat16, 16>::unpack(add[0], f);
#pragma unroll
            for (int x = 0; x < 8; ++x) d[x] += f[x];
            if (row0 + r < p.m && col + 8 * piece < p.n)
              *reinterpret_cast<uint4*>(p.out[0] + (row0 + r) * int64_t(p.n) + col + 8 * piece) =
                  make_uint4(f32_to_bf16x2(d[0], d[1]), f32_to_bf16x2(d[2], d[3]), f32_to_bf16x2(d[4], d[5]),
                             f32_to_bf16x2(d[6], d[7]));
          }
        } else if constexpr (FINISH == kGated) {
          float u[32];
          sums(from + BN / 2 + j, u);
          if (p.keep) {
            put(p.out[1], row0, col, [&](int i) { return upper_pair(v[i], v[i + 1]); });
            put(p.out[2], row0, col, [&](int i) { return upper_pair(u[i], u[i + 1]); });
            put(p.out[3], row0, col, [&](int i) { return lower_pair(v[i], u[i], v[i + 1], u[i + 1]); });
          }
          with_activation(p.act, [&](auto act) {
            float unused;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = activate<decltype(act)::value, false>(v[i], unused) * u[i];
          });
          put(p.out[0], row0, col, [&](int i) { return f32_to_bf16x2(v[i], v[i + 1]); });
        } else if constexpr (FINISH == kGatedGrad) {
          turn(v);
          with_activation(p.act, [&](auto act) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = first + 8 * i;
              float dh[8];
              uint4 kept[3];
              fetched(i, kept);
              fetch(i, ahead_row, ahead_col + ahead_j);
              turned(r, dh);
              const uint32_t g[4] = {kept[0].x, kept[0].y, kept[0].z, kept[0].w}, u[4] = {kept[1].x, kept[1].y, kept[1].z, kept[1].w},
                             low[4] = {kept[2].x, kept[2].y, kept[2].z, kept[2].w};
              uint32_t dg[4], du[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                float a[2], b[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  float slope;
                  const float f = activate<decltype(act)::value, true>(whole(g[x], low[x], y, 0), slope), d = dh[2 * x + y];
                  a[y] = d * whole(u[x], low[x], y, 1) * slope;
                  b[y] = d * f;
                }
                dg[x] = f32_to_bf16x2(a[0], a[1]);
                du[x] = f32_to_bf16x2(b[0], b[1]);
              }
              if (row0 + r < p.m && col + 8 * piece < p.n) {
                const int64_t at = (row0 + r) * int64_t(p.n) + col + 8 * piece;
                *reinterpret_cast<uint4*>(p.out[0] + at) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
                *reinterpret_cast<uint4*>(p.out[1] + at) = make_uint4(du[0], du[1], du[2], du[3]);
              }
            }
          });
        }
      }
      tc::fence_before_barrier();
      __syncwarp();
      if (lane == 0) tma::arrive<PAIR>(first_ctas<PAIR>(tc::smem_address(s_taken + half)));
      if (half == 1) complete ^= 1;
      half ^= 1;
    }
    if constexpr (kRead > 0) asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  tc::fence_before_barrier();
  __syncthreads();
  if constexpr (SPLIT > 1) {
    cluster_barrier();                                   // all parts' sums are in place
    constexpr int kCols = FINISH == kGated ? BN / 2 : BN, kPieces = kCols / 8, kRows = kTileM / SPLIT;
    int m_tile, n_tile;
    place(p.m_tiles, p.n_tiles, walker, m_tile, n_tile);
    bool failed = false;
#pragma unroll
    for (int k = 0; k < SPLIT; ++k) failed |= word_of(tc::smem_address(s_tmem + 1), k) != 0u;
    // 8 columns from `column` on of row r of the tile, summed over the parts in their order
    auto all_parts = [&](int r, int column, float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
      for (int k = 0; k < SPLIT; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 f = load_of(s_ring + r * (BN * 4) + ((column / 4 + i) ^ (r & 7)) * 16, k);
          v[4 * i] += f.x; v[4 * i + 1] += f.y; v[4 * i + 2] += f.z; v[4 * i + 3] += f.w;
        }
      if (failed) v[0] = v[1] = v[2] = v[3] = v[4] = v[5] = v[6] = v[7] = __int_as_float(0x7fffffff);
    };
    for (int t = threadIdx.x; t < kRows * kPieces; t += kThreads) {
      const int r = blockIdx.x % SPLIT * kRows + t / kPieces, c = t % kPieces * 8;
      const int64_t row = int64_t(m_tile) * kTileM + r;
      const int col = n_tile * kCols + c;
      if (row >= p.m || col >= p.n) continue;
      const int64_t at = row * p.n + col;
      float v[8];
      all_parts(r, c, v);
      auto store = [&](uint16_t* to, auto&& word) { *reinterpret_cast<uint4*>(to + at) = make_uint4(word(0), word(2), word(4), word(6)); };
      if constexpr (FINISH == kGated) {
        float u[8];
        all_parts(r, BN / 2 + c, u);
        if (p.keep) {
          store(p.out[1], [&](int i) { return upper_pair(v[i], v[i + 1]); });
          store(p.out[2], [&](int i) { return upper_pair(u[i], u[i + 1]); });
          store(p.out[3], [&](int i) { return lower_pair(v[i], u[i], v[i + 1], u[i + 1]); });
        }
        with_activation(p.act, [&](auto act) {
          float unused;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = activate<decltype(act)::value, false>(v[i], unused) * u[i];
        });
      } else if constexpr (FINISH == kPlus) {
        float f[8];
        Lane<__nv_bfloat16, 16>::load(reinterpret_cast<const __nv_bfloat16*>(p.read[0]) + at, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += f[i];
      }
      store(p.out[0], [&](int i) { return f32_to_bf16x2(v[i], v[i + 1]); });
    }
    __syncwarp();                                        // of lanes that left the loop apart: a barrier takes whole warps
    cluster_barrier();                                   // nobody reads another's sums any more
  }
  if constexpr (PAIR) cluster_barrier();                 // neither uses the other's shared or tensor memory any more
  if (warp == kFinishWarps + 1) release<PAIR, 2 * BN>(tmem);
}

// The parts of a shared tile added in the order of k and rounded: out[product][m][n].  A block takes 32
// rows x 64 columns; its warps take 8 columns each, in SLICES slices of the parts where there are many.
struct SumParts {
  const float* partial;
  uint16_t* out[2];
  int m, n, m_tiles, n_tiles, product_tiles, whole, chunks, walkers;
};
template <int BN, bool PAIR, int SLICES>
__global__ void __launch_bounds__(256 * SLICES) sum_parts_kernel(const SumParts p) {
  constexpr int kCtas = PAIR ? 2 : 1, kTileRows = kTileM * kCtas, kTogether = 4;
  __shared__ float s_block[SLICES][64][33];
  const int warp = threadIdx.x / 32 % 8, slice = threadIdx.x / 256, lane = threadIdx.x % 32;
  const int shared_tile = blockIdx.x, r0 = blockIdx.y % (kTileRows / 32) * 32, c0 = blockIdx.y / (kTileRows / 32) * 64;
  const int64_t all = (int64_t(p.m_tiles) * p.n_tiles - p.whole) * p.chunks;
  const int64_t begin = int64_t(shared_tile) * p.chunks, end = begin + p.chunks;
  // the walker that had the tile's first chunk, and the one behind its last
  const int64_t w0 = ((begin + 1) * p.walkers - 1) / all, w1 = (end * p.walkers - 1) / all + 1;
  const int64_t from_w = w0 + (w1 - w0) * slice / SLICES, to_w = w0 + (w1 - w0) * (slice + 1) / SLICES;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  for (int64_t w = from_w; w < to_w; w += kTogether) {
    float v[kTogether][8];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const float* from = p.partial + ((w + k + shared_tile) * kCtas + r0 / kTileM) * (BN * kTileM) + (c0 + warp * 8) * kTileM +
                          r0 % kTileM + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = w + k < to_w ? __ldg(from + i * kTileM) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[k][i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_block[slice][warp * 8 + i][lane] = s[i];
  __syncthreads();
  if (slice > 0) return;
  int m_tile, n_tile;
  place(p.m_tiles, p.n_tiles, p.whole + shared_tile, m_tile, n_tile);
  const bool other = m_tile >= p.product_tiles;
  const int64_t row = int64_t(m_tile - (other ? p.product_tiles : 0)) * kTileRows + r0 + threadIdx.x / 8;
  const int c = threadIdx.x % 8 * 8, col = n_tile * BN + c0 + c;
  if (row >= p.m || col >= p.n) return;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) v[i] += s_block[k][c + i][threadIdx.x / 8];
  }
  Lane<__nv_bfloat16, 16>::store(reinterpret_cast<__nv_bfloat16*>(p.out[other]) + row * p.n + col, v);
}

}  // namespace gemm
}  // namespace tgt
