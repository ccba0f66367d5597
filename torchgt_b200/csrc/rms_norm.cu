// Root-mean-square norm of rows, with the residual addition in front of it, forward and backward, and with its result in 8 bits.
//
//   v = x + residual,  rstd = 1 / sqrt(mean(v^2) + eps),  y = v rstd w,  sum = v
//   g = dy w,  u = v rstd:   dx = rstd (g - u mean(g u)) + dsum,  dw = sum over rows of dy u
//   8 bits:  scale = max(max |y| / 448, 2^-126),  values = e4m3(y (1 / scale)), 1 / scale rounded: a division less per value
//
// All of it in fp32, rounded once where it is stored; y comes from v before v is rounded for the residual stream.  In bf16 the
// forward can leave the next 8 bits of v beside the rounded sum for the backward: with the sum alone its rounding is in dw next
// to dw's own (2.4e-3 from 64 bits in the 2-norm, with them 1.7e-3), for an eighth more bytes.
// What is read and written bounds it: x and the residual in, y and the sum out; dy, the residual stream's gradient and the sum
// in, dx out.  A row is held in registers between its sums and its results: by a group of 8 to 32 lanes, or by a CTA where it
// is longer than a warp should hold, the next row on its way meanwhile.  Rows that are a whole number of 16-byte pieces from
// 16-byte boundaries on move in such pieces, all others value by value.  The weight's gradient is summed per thread over the rows it
// walks, then over a CTA's groups and over the CTAs in a fixed order: no atomics, the same bits every time.
// us (a copy's rate would be): bf16 with a residual, 16,384 x 2,048 forward with the kept bits 46 (47), backward 59 (47); 16,384 x
// 5,120 to e4m3 96 (91); fp32 64,001 x 64 9.8 (10.1) and 11.3 (10.1, in part from the L2).
#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "tgt_common.cuh"

namespace tgt {
namespace {

constexpr int kMostHidden = 16384;
constexpr int kGroupThreads = 256;      // of a CTA whose rows belong to groups of lanes

// ---- pieces of a row -------------------------------------------------------------------------------------------------
template <typename T, int VEC>
struct Piece {                          // a 16-byte piece as it is in memory
  static_assert(VEC * sizeof(T) == 16, "16 bytes");
  typename Lane<T, 16>::Raw raw;
  __device__ __forceinline__ void load(const T* row, int piece) { raw = Lane<T, 16>::raw_at(row, unsigned(piece)); }
  __device__ __forceinline__ void clear() { raw = Lane<T, 16>::raw_zero(); }
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const { Lane<T, 16>::unpack(raw, f); }
  __device__ __forceinline__ static void store(T* row, int piece, const float (&f)[VEC]) {
    Lane<T, 16>::store_at(row, unsigned(piece), f);
  }
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
struct Piece<T, 1> {                    // one value
  T raw;
  __device__ __forceinline__ void load(const T* row, int piece) { raw = row[piece]; }
  __device__ __forceinline__ void clear() { raw = T(0.f); }
  __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = widen(raw); }
  __device__ __forceinline__ static void store(T* row, int piece, const float (&f)[1]) { row[piece] = T(f[0]); }
};

// What a bf16 sum's rounding took from it, in steps of 2^-8 of its last place: the bits of v are (sum << 16) + (rest << 8),
// rounded.  (The end of the range of a byte is a step nearer than it should be.)
__device__ __forceinline__ int rest_of(float v) {
  const int32_t bits = __float_as_int(v), sum = int32_t(__bfloat16_as_ushort(__float2bfloat16_rn(v))) << 16;
  return min(max((bits - sum + 128) >> 8, -128), 127);
}
__device__ __forceinline__ float with_rest(float sum, int rest) { return __int_as_float(__float_as_int(sum) + rest * 256); }
template <int VEC>
__device__ __forceinline__ void store_rest(int8_t* row, int piece, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= uint32_t(rest_of(v[i]) & 0xff) << (8 * (i % 4));
    reinterpret_cast<uint2*>(row)[piece] = make_uint2(w[0], w[1]);
  } else {
    row[piece] = int8_t(rest_of(v[0]));
  }
}
template <int VEC>
struct Rest {                           // of a piece, as it is in memory
  uint2 raw;
  __device__ __forceinline__ void load(const int8_t* row, int piece) {
    if constexpr (VEC == 8) raw = __ldg(reinterpret_cast<const uint2*>(row) + piece);
    else raw.x = uint32_t(int32_t(row[piece]));
  }
  __device__ __forceinline__ void clear() { raw = make_uint2(0u, 0u); }
  __device__ __forceinline__ int at(int i) const { return int(int8_t((i < 4 ? raw.x : raw.y) >> (8 * (i % 4)))); }
};

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {   // +-448 where a value is larger, NaN stays NaN
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int piece, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    row[piece] = uint8_t(__nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3));
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = e4m3x2(f[4 * i], f[4 * i + 1]) | uint32_t(e4m3x2(f[4 * i + 2], f[4 * i + 3])) << 16;
    if constexpr (VEC == 4) reinterpret_cast<uint32_t*>(row)[piece] = w[0];
    else reinterpret_cast<uint2*>(row)[piece] = make_uint2(w[0], w[1]);
  }
}

// ---- sums over the threads of a row: LPR lanes of a warp, or (LPR == 0) the CTA ------------------------------------------
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct LargestBits {   // of non-negative values as whole numbers: NaN is above infinity, so it is not lost
  __device__ __forceinline__ float operator()(float a, float b) const {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
  }
};
// `turn` changes with every sum: a sum's words are not written again before all have passed the barrier of the next.
constexpr int kPartWords = 64;
template <int LPR, class Op>
__device__ __forceinline__ float over_row(float x, float* s_part, int& turn, Op op) {
#pragma unroll
  for (int o = (LPR == 0 ? 32 : LPR) / 2; o > 0; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
  if constexpr (LPR == 0) {
    const int warps = blockDim.x / 32;
    s_part += turn;
    turn ^= 32;
    if (threadIdx.x % 32 == 0) s_part[threadIdx.x / 32] = x;
    __syncthreads();
    x = s_part[0];
    for (int w = 1; w < warps; ++w) x = op(x, s_part[w]);
  }
  return x;
}

// Which rows and which of their pieces a thread has: row first_row + row_of_cta, then rows_at_once further on, while first_row,
// which all threads of the CTA have in common, is a row; pieces first, first + step, ...
template <int LPR>
struct Place {
  int64_t first_row, rows_at_once;
  int row_of_cta, first, step;
  __device__ __forceinline__ Place() {
    constexpr int kRows = LPR == 0 ? 1 : kGroupThreads / (LPR == 0 ? 1 : LPR);
    first_row = int64_t(blockIdx.x) * kRows;
    rows_at_once = int64_t(gridDim.x) * kRows;
    row_of_cta = LPR == 0 ? 0 : threadIdx.x / (LPR == 0 ? 1 : LPR);
    first = LPR == 0 ? threadIdx.x : threadIdx.x % (LPR == 0 ? 1 : LPR);
    step = LPR == 0 ? blockDim.x : LPR;
  }
};
// Whether a thread has registers for the next row while it works on one: 32-bit words of a matrix that it holds
constexpr bool row_ahead(int pieces, int vec, size_t value, int most) { return pieces * (vec == 1 ? 1 : int(vec * value / 4)) <= most; }
constexpr int most_threads(int lpr, int vec) { return lpr != 0 ? kGroupThreads : vec == 1 ? 1024 : 512; }

// ---- forward ---------------------------------------------------------------------------------------------------------
template <typename T>
struct RmsFwd {
  const T* x;
  const T* residual;   // may be null
  const T* weight;
  T* sum;              // may be null
  int8_t* rest;        // may be null (bf16)
  T* y;                // or, in 8 bits, values and scales
  uint8_t* values;
  float* scales;
  float* rstd;         // may be null
  int64_t rows;
  int hidden;
  float eps;
};

template <typename T, int VEC, int LPR, int PIECES, bool E4M3>
__global__ void __launch_bounds__(most_threads(LPR, VEC)) rms_norm_fwd_kernel(const RmsFwd<T> p) {
  __shared__ float s_part[kPartWords];
  int turn = 0;
  const Place<LPR> at;
  const int pieces = p.hidden / VEC;
  const float inv_hidden = 1.f / float(p.hidden);
  Piece<T, VEC> next[PIECES], next_res[PIECES];              // the next row, on its way
  auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
      if (r < p.rows && c < pieces) {
        next[j].load(p.x + r * p.hidden, c);
        if (p.residual != nullptr) next_res[j].load(p.residual + r * p.hidden, c);
      } else {
        next[j].clear();
      }
    }
  };
  constexpr bool kAhead = row_ahead(PIECES, VEC, sizeof(T), 16);
  if (kAhead) load(at.first_row + at.row_of_cta);
  for (int64_t r0 = at.first_row; r0 < p.rows; r0 += at.rows_at_once) {
    const int64_t r = r0 + at.row_of_cta;
    const bool live = r < p.rows;
    Piece<T, VEC> x[PIECES], res[PIECES];
    if (!kAhead) load(r);
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      x[j] = next[j];
      res[j] = next_res[j];
    }
    if (kAhead) load(r + at.rows_at_once);
    float v[PIECES][VEC], squares = 0.f;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
      x[j].unpack(v[j]);
      if (p.residual != nullptr && live && c < pieces) {
        float f[VEC];
        res[j].unpack(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] += f[i];
        if (p.sum != nullptr) Piece<T, VEC>::store(p.sum + r * p.hidden, c, v[j]);
        if constexpr (sizeof(T) == 2)
          if (p.rest != nullptr) store_rest<VEC>(p.rest + r * p.hidden, c, v[j]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) squares = fmaf(v[j][i], v[j][i], squares);
    }
    squares = over_row<LPR>(squares, s_part, turn, Add());
    const float rstd = rsqrtf(squares * inv_hidden + p.eps);
    if (live && at.first == 0 && p.rstd != nullptr) p.rstd[r] = rstd;
    float largest = 0.f;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
      if (!live || c >= pieces) continue;
      Piece<T, VEC> w;
      w.load(p.weight, c);
      float f[VEC];
      w.unpack(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = v[j][i] * rstd * f[i];
        if (E4M3) largest = LargestBits()(largest, fabsf(v[j][i]));
      }
      if (!E4M3) Piece<T, VEC>::store(p.y + r * p.hidden, c, v[j]);
    }
    if constexpr (E4M3) {
      largest = over_row<LPR>(largest, s_part, turn, LargestBits());
      float scale = largest / 448.f;
      scale = scale < 0x1p-126f ? 0x1p-126f : scale;          // NaN stays
      const float by = 1.f / scale;
      if (live && at.first == 0) p.scales[r] = scale;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int c = at.first + j * at.step;
        if (!live || c >= pieces) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] *= by;
        store_e4m3<VEC>(p.values + r * p.hidden, c, v[j]);
      }
    }
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------
template <typename T>
struct RmsBwd {
  const T* dy;
  const T* dsum;       // may be null
  const T* v;          // x, or the sum as it was stored
  const int8_t* rest;  // of the sum; may be null (bf16)
  const T* weight;
  const float* rstd;
  T* dx;
  float* partial;      // [gridDim.x][hidden]
  int64_t rows;
  int hidden;
};

template <typename T, int VEC, int LPR, int PIECES>
__global__ void __launch_bounds__(most_threads(LPR, VEC)) rms_norm_bwd_kernel(const RmsBwd<T> p) {
  __shared__ float s_part[kPartWords];
  int turn = 0;
  extern __shared__ float s_dw[];               // [warps][hidden], where rows belong to groups of lanes
  const Place<LPR> at;
  const int pieces = p.hidden / VEC;
  const float inv_hidden = 1.f / float(p.hidden);
  float dw[PIECES][VEC];
  Piece<T, VEC> w[PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const int c = at.first + j * at.step;
    if (c < pieces) w[j].load(p.weight, c);
    else w[j].clear();
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
  }
  constexpr bool kRest = sizeof(T) == 2;
  Piece<T, VEC> next[PIECES], next_dy[PIECES], next_ds[PIECES];   // the next row, on its way
  Rest<VEC> next_rest[kRest ? PIECES : 1];
  float next_rstd;
  auto load = [&](int64_t r) {
    next_rstd = r < p.rows ? __ldg(p.rstd + r) : 0.f;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
      if (r < p.rows && c < pieces) {
        next[j].load(p.v + r * p.hidden, c);
        if constexpr (kRest) {
          if (p.rest != nullptr) next_rest[j].load(p.rest + r * p.hidden, c);
          else next_rest[j].clear();
        }
        next_dy[j].load(p.dy + r * p.hidden, c);
        if (p.dsum != nullptr) next_ds[j].load(p.dsum + r * p.hidden, c);
      } else {
        next[j].clear();
        if constexpr (kRest) next_rest[j].clear();
        next_dy[j].clear();
      }
    }
  };
  constexpr bool kAhead = LPR == 0 && row_ahead(PIECES, VEC, sizeof(T), 8);
  if (kAhead) load(at.first_row + at.row_of_cta);
  for (int64_t r0 = at.first_row; r0 < p.rows; r0 += at.rows_at_once) {
    const int64_t r = r0 + at.row_of_cta;
    const bool live = r < p.rows;
    Piece<T, VEC> v[PIECES], dy[PIECES], ds[PIECES];
    Rest<VEC> rest[kRest ? PIECES : 1];
    if (!kAhead) load(r);
    const float rstd = next_rstd;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      v[j] = next[j];
      if constexpr (kRest) rest[j] = next_rest[j];
      dy[j] = next_dy[j];
      ds[j] = next_ds[j];
    }
    if (kAhead) load(r + at.rows_at_once);
    auto values = [&](int j, float (&f)[VEC]) {
      v[j].unpack(f);
      if constexpr (kRest) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = with_rest(f[i], rest[j].at(i));
      }
    };
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      float f[VEC], d[VEC], g[VEC];
      values(j, f);
      dy[j].unpack(d);
      w[j].unpack(g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float u = f[i] * rstd;
        dw[j][i] = fmaf(d[i], u, dw[j][i]);
        dot = fmaf(d[i] * g[i], u, dot);
      }
    }
    dot = over_row<LPR>(dot, s_part, turn, Add()) * inv_hidden;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
      if (!live || c >= pieces) continue;
      float f[VEC], d[VEC], g[VEC];
      values(j, f);
      dy[j].unpack(d);
      w[j].unpack(g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[i] = rstd * (d[i] * g[i] - f[i] * rstd * dot);
      if (p.dsum != nullptr) {
        ds[j].unpack(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] += f[i];
      }
      Piece<T, VEC>::store(p.dx + r * p.hidden, c, d);
    }
  }
  release_dependents();
  float* out = p.partial + int64_t(blockIdx.x) * p.hidden;
  if constexpr (LPR == 0) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c < pieces) out[c * VEC + i] = dw[j][i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int c = at.first + j * at.step;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) dw[j][i] += __shfl_xor_sync(0xffffffffu, dw[j][i], o);
        if (threadIdx.x % 32 < LPR && c < pieces) s_dw[threadIdx.x / 32 * p.hidden + c * VEC + i] = dw[j][i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.hidden; c += kGroupThreads) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kGroupThreads / 32; ++k) s += s_dw[k * p.hidden + c];
      out[c] = s;
    }
  }
}

template <typename T>
struct WeightSum {
  const float* partial;        // [parts][hidden]
  T* dweight;
  int parts, hidden;
};
// A block adds 32 values of the CTAs' sums: 32 warps, eight in flight each.
constexpr int kSumThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kSumThreads) rms_norm_weight_grad_kernel(const WeightSum<T> p) {
  __shared__ float s_sum[32][33];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = blockIdx.x * 32 + lane;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = 0.f;
  dependent_wait();
  if (i < p.hidden)
    for (int c = warp; c < p.parts; c += 32 * 8)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + 32 * j < p.parts) s[j] += __ldcg(p.partial + int64_t(c + 32 * j) * p.hidden + i);
  s_sum[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  float v = s_sum[lane][warp];                   // of value `warp` of the block, the sums of warp `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0 && blockIdx.x * 32 + warp < p.hidden) p.dweight[blockIdx.x * 32 + warp] = T(v);
}

// ---- which kernel ----------------------------------------------------------------------------------------------------
struct Shape {
  int lpr, pieces, threads;   // lpr 0: a CTA of `threads` to a row
};
// Lanes and CTAs with two 16-byte pieces a thread where that is enough threads for the chip and rows are short enough, up to
// four (eight fp32 ones) where a row would be more threads than a CTA runs well with; single values sixteen.
Shape shape_of(int hidden, int vec) {
  const int n = hidden / vec;
  if (n <= 128) {
    int lpr = 8;
    while (lpr < 32 && 2 * lpr < n) lpr *= 2;
    const int pieces = (n + lpr - 1) / lpr;
    return {lpr, pieces <= 1 ? 1 : pieces <= 2 ? 2 : 4, kGroupThreads};
  }
  const int most = most_threads(0, vec);
  int threads = (n + 1) / 2;
  threads = threads < 128 ? 128 : threads > most ? most : (threads + 31) / 32 * 32;
  const int pieces = (n + threads - 1) / threads;
  return {0, pieces <= 2 ? 2 : pieces <= 4 ? 4 : pieces <= 8 ? 8 : 16, threads};
}

template <class F>
bool with_shape(const Shape& s, F&& f) {
  auto pieces = [&](auto lpr) {
    switch (s.pieces) {
      case 1: if constexpr (decltype(lpr)::value != 0) { f(lpr, std::integral_constant<int, 1>()); return true; } return false;
      case 2: f(lpr, std::integral_constant<int, 2>()); return true;
      case 4: f(lpr, std::integral_constant<int, 4>()); return true;
      case 8: if constexpr (decltype(lpr)::value == 0) { f(lpr, std::integral_constant<int, 8>()); return true; } return false;
      case 16: if constexpr (decltype(lpr)::value == 0) { f(lpr, std::integral_constant<int, 16>()); return true; } return false;
    }
    return false;
  };
  switch (s.lpr) {
    case 0: return pieces(std::integral_constant<int, 0>());
    case 8: return pieces(std::integral_constant<int, 8>());
    case 16: return pieces(std::integral_constant<int, 16>());
    case 32: return pieces(std::integral_constant<int, 32>());
  }
  return false;
}

// CTAs to walk the rows, no more than have any: of the backward no more than are resident together, so that all end at one
// time, nor than leave few rows of partial sums.
int grid_of(const Shape& s, int64_t rows, int ctas_per_sm) {
  const int64_t at_once = s.lpr == 0 ? 1 : kGroupThreads / s.lpr;
  const int64_t want = (rows + at_once - 1) / at_once, most = int64_t(sm_count()) * ctas_per_sm;
  return int(want < most ? want : most);
}
int forward_grid(const Shape& s, int64_t rows) { return grid_of(s, rows, 2048 / s.threads); }
int most_backward_grid(const Shape& s, int64_t rows) { return grid_of(s, rows, 1024 / s.threads); }
// resident CTAs of a kernel on an SM, asked once for each device and block size
template <auto Kernel>
int resident(int threads, int smem) {
  static std::atomic<int> cache[kMaxDevices][1024 / 32 + 1] = {};
  const int dev = current_device();
  if (dev < 0) return 1;
  std::atomic<int>& known = cache[dev][threads / 32];
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, smem) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}

int check_rows(int64_t rows, int hidden, int dtype) {
  TGT_CHECK_ARG(dtype == TGT_F32 || dtype == TGT_BF16, "dtype must be TGT_F32 or TGT_BF16");
  TGT_CHECK_ARG(rows >= 0, "rows must be >= 0");
  TGT_CHECK_ARG(hidden >= 1, "hidden must be >= 1");
  if (hidden > kMostHidden) return set_error(TGT_ERR_UNSUPPORTED, "hidden=%d: a row has at most %d values", hidden, kMostHidden);
  return TGT_OK;
}

template <typename T>
constexpr int kVec = 16 / int(sizeof(T));
template <typename T>
bool whole_pieces(int hidden, std::initializer_list<const void*> pointers) {
  if (hidden % kVec<T> != 0) return false;
  for (const void* q : pointers)
    if (!aligned16(q)) return false;
  return true;
}

template <typename T, int VEC, bool E4M3>
int launch_forward(const RmsFwd<T>& p, cudaStream_t stream) {
  const Shape s = shape_of(p.hidden, VEC);
  const bool built = with_shape(s, [&](auto lpr, auto pieces) {
    constexpr int kLpr = decltype(lpr)::value, kPieces = decltype(pieces)::value;
    if constexpr (VEC == 1 || kPieces * kVec<T> <= 32)
      rms_norm_fwd_kernel<T, VEC, kLpr, kPieces, E4M3><<<forward_grid(s, p.rows), s.threads, 0, stream>>>(p);
  });
  if (!built) return set_error(TGT_ERR_UNSUPPORTED, "no kernel for hidden=%d", p.hidden);
  TGT_CHECK_CUDA(cudaGetLastError());
  return TGT_OK;
}

template <typename T, int VEC>
int launch_backward(RmsBwd<T> p, void* dweight, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  const Shape s = shape_of(p.hidden, VEC);
  int grid = most_backward_grid(s, p.rows);
  if (scratch == nullptr || scratch_bytes < size_t(grid) * p.hidden * sizeof(float))
    return set_error(TGT_ERR_WORKSPACE, "scratch holds %zu bytes, %zu needed", scratch_bytes, size_t(grid) * p.hidden * sizeof(float));
  p.partial = static_cast<float*>(scratch);
  const size_t smem = s.lpr == 0 ? 0 : size_t(kGroupThreads / 32) * p.hidden * sizeof(float);
  const bool built = with_shape(s, [&](auto lpr, auto pieces) {
    constexpr int kLpr = decltype(lpr)::value, kPieces = decltype(pieces)::value;
    if constexpr (VEC == 1 || kPieces * kVec<T> <= 32) {
      if (s.lpr == 0) {
        const int all = sm_count() * resident<rms_norm_bwd_kernel<T, VEC, kLpr, kPieces>>(s.threads, 0);
        if (grid > all) grid = all;
      }
      rms_norm_bwd_kernel<T, VEC, kLpr, kPieces><<<grid, s.threads, smem, stream>>>(p);
    }
  });
  if (!built) return set_error(TGT_ERR_UNSUPPORTED, "no kernel for hidden=%d", p.hidden);
  TGT_CHECK_CUDA(cudaGetLastError());
  const WeightSum<T> sum{p.partial, static_cast<T*>(dweight), grid, p.hidden};
  TGT_CHECK_CUDA(launch_chained(rms_norm_weight_grad_kernel<T>, dim3((p.hidden + 31) / 32), kSumThreads, stream, kLinkStitch, sum));
  return TGT_OK;
}

template <typename T, bool E4M3>
int forward(const void* x, const void* residual, const void* weight, float eps, int64_t rows, int hidden, void* sum, int8_t* rest,
            void* y, void* values, float* scales, float* rstd, cudaStream_t stream) {
  RmsFwd<T> p{static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), static_cast<T*>(sum), rest,
              static_cast<T*>(y), static_cast<uint8_t*>(values), scales, rstd, rows, hidden, eps};
  return whole_pieces<T>(hidden, {x, residual, weight, sum, rest, y, values}) ? launch_forward<T, kVec<T>, E4M3>(p, stream)
                                                                        : launch_forward<T, 1, E4M3>(p, stream);
}

template <typename T>
int backward(const void* dy, const void* dsum, const void* v, const int8_t* rest, const void* weight, const float* rstd,
             int64_t rows, int hidden, void* dx, void* dweight, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  RmsBwd<T> p{static_cast<const T*>(dy), static_cast<const T*>(dsum), static_cast<const T*>(v), rest,
              static_cast<const T*>(weight), rstd, static_cast<T*>(dx), nullptr, rows, hidden};
  return whole_pieces<T>(hidden, {dy, dsum, v, rest, weight, dx})
             ? launch_backward<T, kVec<T>>(p, dweight, scratch, scratch_bytes, stream)
             : launch_backward<T, 1>(p, dweight, scratch, scratch_bytes, stream);
}

}  // namespace
}  // namespace tgt

extern "C" int tgt_rms_norm_fwd(const void* x, const void* residual, const void* weight, float eps, int64_t rows, int hidden,
                                int dtype, void* sum, void* rest, void* y, float* rstd, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_rows(rows, hidden, dtype);
  if (rc != TGT_OK) return rc;
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(x && weight && y, "x, weight and y must not be null");
  TGT_CHECK_ARG(sum == nullptr || residual != nullptr, "sum without a residual");
  TGT_CHECK_ARG(rest == nullptr || (sum != nullptr && dtype == TGT_BF16), "rest is of a bf16 sum");
  return dtype == TGT_F32 ? forward<float, false>(x, residual, weight, eps, rows, hidden, sum, nullptr, y, nullptr, nullptr, rstd, stream)
                          : forward<__nv_bfloat16, false>(x, residual, weight, eps, rows, hidden, sum, static_cast<int8_t*>(rest), y,
                                                          nullptr, nullptr, rstd, stream);
}

extern "C" int tgt_rms_norm_e4m3(const void* x, const void* residual, const void* weight, float eps, int64_t rows, int hidden,
                                 int dtype, void* sum, void* values, float* scales, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_rows(rows, hidden, dtype);
  if (rc != TGT_OK) return rc;
  if (rows == 0) return TGT_OK;
  TGT_CHECK_ARG(x && weight && values && scales, "x, weight, values and scales must not be null");
  TGT_CHECK_ARG(sum == nullptr || residual != nullptr, "sum without a residual");
  return dtype == TGT_F32
             ? forward<float, true>(x, residual, weight, eps, rows, hidden, sum, nullptr, nullptr, values, scales, nullptr, stream)
             : forward<__nv_bfloat16, true>(x, residual, weight, eps, rows, hidden, sum, nullptr, nullptr, values, scales, nullptr,
                                           stream);
}

extern "C" int tgt_rms_norm_bwd_scratch_bytes(int64_t rows, int hidden, int dtype, size_t* bytes) {
  using namespace tgt;
  TGT_CHECK_ARG(bytes != nullptr, "bytes is null");
  const int rc = check_rows(rows, hidden, dtype);
  if (rc != TGT_OK) return rc;
  const size_t size = dtype == TGT_F32 ? 4 : 2;
  const int vec = int(16 / size);
  // whether the pointers allow whole pieces is not known yet
  int grid = most_backward_grid(shape_of(hidden, 1), rows);
  if (hidden % vec == 0) {
    const int other = most_backward_grid(shape_of(hidden, vec), rows);
    grid = other > grid ? other : grid;
  }
  *bytes = size_t(grid) * hidden * sizeof(float);
  return TGT_OK;
}

extern "C" int tgt_rms_norm_bwd(const void* dy, const void* dsum, const void* v, const void* rest, const void* weight,
                                const float* rstd, int64_t rows, int hidden, int dtype, void* dx, void* dweight, void* scratch,
                                size_t scratch_bytes, void* stream_) {
  using namespace tgt;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_rows(rows, hidden, dtype);
  if (rc != TGT_OK) return rc;
  TGT_CHECK_ARG(dweight != nullptr, "dweight must not be null");
  if (rows == 0) {
    TGT_CHECK_CUDA(cudaMemsetAsync(dweight, 0, size_t(hidden) * (dtype == TGT_F32 ? 4 : 2), stream));
    return TGT_OK;
  }
  TGT_CHECK_ARG(dy && v && weight && rstd && dx, "dy, v, weight, rstd and dx must not be null");
  TGT_CHECK_ARG(rest == nullptr || dtype == TGT_BF16, "rest is of a bf16 sum");
  return dtype == TGT_F32
             ? backward<float>(dy, dsum, v, nullptr, weight, rstd, rows, hidden, dx, dweight, scratch, scratch_bytes, stream)
             : backward<__nv_bfloat16>(dy, dsum, v, static_cast<const int8_t*>(rest), weight, rstd, rows, hidden, dx, dweight, scratch,
                                       scratch_bytes, stream);
}
