// Root-mean-square norm of rows, with dropout and the residual's addition in front of it, an output
// in 8 bits behind it, and its gradient.
//
//   h = residual + dropout(x)      rstd = 1 / sqrt(mean(h^2) + eps)      y = h * rstd * weight
//   8 bits: for every row, or group of `group` columns, scale = max|y| / 448 and q = e4m3(y / scale)
//
//   with n = h * rstd and a = grad_y * weight:
//   grad_residual = rstd * (a - n * mean(a * n)) + grad_h      grad_x = dropout(grad_residual)
//   grad_weight   = sum over rows of grad_y * n
//
// All arithmetic is in float32; the norm is taken of the float32 h, which is rounded only where it is
// stored.  Bound by memory: a row is read once and stays in registers between the sum over it and the
// values made from it.  Up to 64 pieces of eight columns, 8 to 64 lanes of a wave hold one piece each; a longer
// row has a block to itself, as many waves as its pieces fill, one piece a lane (two above 1 024 pieces).
// Few values a lane keep the registers low and many waves in flight.  Rows of more than 2 048 pieces are
// read again for each step.
//
// Measured on 2^26 bfloat16 values with a residual, rows of 512 to 16 384: norm 90 - 105 us (5.1 - 6.0 TB/s,
// a large copy reaches 4.9), into 8 bits with groups of 128 80 - 100 us; gradient with dropout 128 - 150 us (4.5
// - 5.2 TB/s).  A wave has little work beside its loads, so instructions count: sums and maxima over lanes by
// data-parallel moves, a reciprocal square root and no division (8 bits, 16 384 x 8 192: 225 instead of 320
// vector instructions a wave, 178 -> 165 us).  With four pieces a lane (134 registers forward, 277 in the
// gradient) that call took 283 us, and rows of 4 096 206 us in the gradient.
#include "rowvec.h"

namespace hades {
namespace {

constexpr int kThreads = 256;
constexpr float kPerE4m3Max = 1.0f / 448.0f;   // of e4m3's largest value
constexpr int64_t kMaxPieces = 2048;   // of a row that stays in registers
constexpr int64_t kMostThreads = int64_t(1) << 32;   // of a launch
constexpr int64_t kCus = 256;
// Pieces of a row up to which a lane of the gradient kernel holds one, else two: from 13 waves on only one
// block of the one-piece form fits a compute unit, and nothing hides its waits for the row's sum (2^26
// bfloat16 values with dropout in rows of 7 168 / 8 192: one piece 156 / 148 us, two 134 / 132).
constexpr int64_t kGradOne = 768;
// Steps of rows that one block takes alone, without the second launch that adds the blocks' partial rows
constexpr int64_t kGradAlone = 4;

constexpr int kMaxWaves = 16;   // of a block

// A weight's piece, whose type is the rows' T or float32, as it lies in memory: nothing waits for it until it
// is used.
struct WeightPiece {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 u32x4u __attribute__((aligned(2)));
  u32x4 lo, hi;

  template <typename T>
  __device__ __forceinline__ void load(const void* p, int64_t piece, bool f32, int valid) {
    if (f32 || sizeof(T) == 4) {
      const float* const q = static_cast<const float*>(p) + piece * kPiece;
      if (valid >= kPiece) {
        lo = *reinterpret_cast<const u32x4u*>(q);
        hi = *reinterpret_cast<const u32x4u*>(q + 4);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = j < valid ? __float_as_uint(q[j]) : 0u;
          hi[j] = j + 4 < valid ? __float_as_uint(q[j + 4]) : 0u;
        }
      }
    } else {
      const uint16_t* const q = static_cast<const uint16_t*>(p) + piece * kPiece;
      if (valid >= kPiece) {
        lo = *reinterpret_cast<const u32x4u*>(q);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          lo[j] = (2 * j < valid ? uint32_t(q[2 * j]) : 0u) | (2 * j + 1 < valid ? uint32_t(q[2 * j + 1]) << 16 : 0u);
      }
    }
  }

  template <typename T>
  __device__ __forceinline__ f32x8 value(bool f32) const {
    f32x8 r;
    if (f32 || sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = __uint_as_float(lo[j]);
        r[j + 4] = __uint_as_float(hi[j]);
      }
      return r;
    }
    typename Vec8<T>::V v;
    __builtin_memcpy(&v, &lo, 16);   // (unused where T is float32)
    return __builtin_convertvector(v, f32x8);
  }
};

template <typename T>
__device__ __forceinline__ f32x8 load_weight(const void* p, int64_t piece, bool f32, int valid) {
  WeightPiece w;
  w.template load<T>(p, piece, f32, valid);
  return w.template value<T>(f32);
}

// a * b summed
__device__ __forceinline__ float dot8(f32x8 a, f32x8 b) {
  float lo = a[0] * b[0], hi = a[1] * b[1];
#pragma unroll
  for (int j = 2; j < kPiece; j += 2) {
    lo = fmaf(a[j], b[j], lo);
    hi = fmaf(a[j + 1], b[j + 1], hi);
  }
  return lo + hi;
}

// Sum over the lanes of a row: T lanes of a wave, or (T = 0) the whole block, all of whose threads
// call; `shared` has kMaxWaves values then.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* shared) {
  v = lanes_sum<T ? T : kWave>(v);
  if (T == 0) {
    const int waves = blockDim.x / kWave;
    __syncthreads();   // `shared` may still be read for the value before
    if ((threadIdx.x & (kWave - 1)) == 0) shared[threadIdx.x / kWave] = v;
    __syncthreads();
    v = shared[0];
    for (int w = 1; w < waves; ++w) v += shared[w];
  }
  return v;
}

// The largest magnitude as bits: magnitudes compare like whole numbers, and a NaN counts as larger than an
// infinity.
__device__ __forceinline__ uint32_t max8(f32x8 v) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < kPiece; ++j) m = __builtin_elementwise_maximum(m, fabsf(v[j]));
  return __float_as_uint(m) & 0x7fffffffu;
}

// The largest magnitude over 448, to half a step of float32.
__device__ __forceinline__ float e4m3_scale(uint32_t m) {
  const float top = __uint_as_float(m);
  const float s = top * kPerE4m3Max;
  return top < INFINITY ? fmaf(fmaf(-448.0f, s, top), kPerE4m3Max, s) : s;
}

// Eight values in units of `scale`, rounded to e4m3 (nearest even).  scale is the largest magnitude of
// the group over 448, to half a step: where it is a normal number a value in its units is at most 448 (1 + 2^-22),
// which rounds to 448, the type's largest.  A subnormal scale of few steps may be too small by a third, and values
// in its units would reach 672, past the type's range (a NaN); those quotients end at 448.
// Quotients by a refined reciprocal and one correction each: of 4 096 x 8 192 bfloat16 values, groups of 128, 2 827
// fall to the other side of a tie than in 64 bits; 2 838 with divisions, 3 074 with the reciprocal alone, which takes
// 1.5 % less time.  Where the reciprocal would overflow or vanish, or scale is subnormal and coarse, every value is
// divided; a group of zeros (scale 0), or of magnitudes of up to 224 * 2^-149, whose scale rounds to 0, gives zeros.
__device__ __forceinline__ void store_e4m3(uint8_t* __restrict__ p, f32x8 v, float scale, int valid) {
  f32x8 u;
  if (scale >= 0x1p-60f && scale < 0x1p100f) {
    float r = __builtin_amdgcn_rcpf(scale);
    r = fmaf(fmaf(-scale, r, 1.0f), r, r);
#pragma unroll
    for (int j = 0; j < kPiece; ++j) {
      const float q = v[j] * r;
      u[j] = fmaf(fmaf(-scale, q, v[j]), r, q);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPiece; ++j) {
      const float q = scale > 0.0f ? v[j] / scale : 0.0f;
      u[j] = q > 448.0f ? 448.0f : (q < -448.0f ? -448.0f : q);   // (a NaN stays one)
    }
  }
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[4], u[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[6], u[7], hi, true);
  if (valid >= kPiece) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef u32x2 u32x2u __attribute__((aligned(1)));
    const u32x2 w = {static_cast<uint32_t>(lo), static_cast<uint32_t>(hi)};
    *reinterpret_cast<u32x2u*>(p) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < kPiece - 1; ++j)
    if (j < valid) p[j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
}

// ---- forward ------------------------------------------------------------------------------------
struct NormArgs {
  const void* x;
  const void* residual;   // may be null
  const void* weight;     // may be null
  void* y;                // rows' type, or e4m3 with `scales`
  void* h;                // may be null
  float* rstd;            // may be null
  float* scales;
  int64_t x_stride, res_stride, rows, cols;
  int weight_f32;
  int group_lanes;        // lanes that share a scale; 0: the row
  int64_t groups;         // scales of a row
  float eps, inv_cols;
  DropArgs drop;
};

__device__ __forceinline__ int valid_of(int64_t cols, int64_t piece) {
  const int64_t left = cols - piece * kPiece;
  return left <= 0 ? 0 : (left < kPiece ? static_cast<int>(left) : kPiece);
}

template <typename X, typename S>
__device__ __forceinline__ f32x8 load_h(const NormArgs& a, const DropKeys& keys, int64_t row, int64_t piece, int valid) {
  // (raw, so that nothing waits for x before the residual's load is under way)
  const typename Vec8<X>::V raw = load8_raw(static_cast<const X*>(a.x) + row * a.x_stride + piece * kPiece, valid);
  typename Vec8<S>::V res;
  if (a.residual != nullptr)
    res = load8_raw(static_cast<const S*>(a.residual) + row * a.res_stride + piece * kPiece, valid);
  f32x8 v = __builtin_convertvector(raw, f32x8);
  if (keys.on()) v = keys.apply(v, static_cast<uint32_t>(row), static_cast<uint32_t>(piece));
  if (a.residual != nullptr) v += __builtin_convertvector(res, f32x8);
  return v;
}

// T lanes of a wave and K pieces of a row each, or T = 0: the lanes of a block
template <typename X, typename S, int T, int K, bool kEight>
__global__ __launch_bounds__(T ? kThreads : kMaxWaves* kWave) void rms_norm_kernel(NormArgs a) {
  __shared__ float shared[kMaxWaves];
  const DropKeys keys(a.drop);
  const int lanes = T ? T : blockDim.x;
  const int lane = T ? threadIdx.x % (T ? T : 1) : threadIdx.x;
  const int64_t row = T ? static_cast<int64_t>(blockIdx.x) * (kThreads / (T ? T : 1)) + threadIdx.x / (T ? T : 1)
                        : static_cast<int64_t>(blockIdx.x);
  const bool in = row < a.rows;
  f32x8 h[K];
  WeightPiece w[K];
  int valid[K];
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t piece = k * lanes + lane;
    valid[k] = in ? valid_of(a.cols, piece) : 0;
    if (a.weight != nullptr) w[k].template load<X>(a.weight, piece, a.weight_f32, valid[k]);
    h[k] = load_h<X, S>(a, keys, row, piece, valid[k]);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (a.h != nullptr) store8(static_cast<S*>(a.h) + row * a.cols + (k * lanes + lane) * kPiece, h[k], valid[k]);
    ss += dot8(h[k], h[k]);
  }
  ss = row_sum<T>(ss, shared);
  const float rstd = rsqrtf(fmaf(ss, a.inv_cols, a.eps));
  if (a.rstd != nullptr && lane == 0 && in) a.rstd[row] = rstd;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    h[k] *= rstd;
    if (a.weight != nullptr) h[k] *= w[k].template value<X>(a.weight_f32);
    if (!kEight) {
      store8(static_cast<X*>(a.y) + row * a.cols + (k * lanes + lane) * kPiece, h[k], valid[k]);
    } else if (a.group_lanes == 0) {
      const uint32_t m = max8(h[k]);
      top = m > top ? m : top;
    }
  }
  if (!kEight) return;
  if (a.group_lanes == 0) {
    __shared__ uint32_t tops[kMaxWaves];
    top = lanes_max(top, T ? T : kWave);
    if (T == 0) {
      if ((threadIdx.x & (kWave - 1)) == 0) tops[threadIdx.x / kWave] = top;
      __syncthreads();
      top = tops[0];
      for (int i = 1; i < lanes / kWave; ++i) top = tops[i] > top ? tops[i] : top;
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int piece = k * lanes + lane;
    uint32_t m = top;
    if (a.group_lanes != 0) m = lanes_max(max8(h[k]), T && a.group_lanes > T ? T : a.group_lanes);
    const float scale = e4m3_scale(m);
    const bool first = a.group_lanes == 0 ? piece == 0 : (piece & (a.group_lanes - 1)) == 0;
    if (first && valid[k] > 0) a.scales[row * a.groups + (a.group_lanes == 0 ? 0 : piece / a.group_lanes)] = scale;
    store_e4m3(static_cast<uint8_t*>(a.y) + row * a.cols + static_cast<int64_t>(piece) * kPiece, h[k], scale, valid[k]);
  }
}

// rows of more than kMaxPieces pieces: h is made again for each step
template <typename X, typename S, bool kEight>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(NormArgs a) {
  constexpr int T = 1024;
  __shared__ float shared[kMaxWaves];
  __shared__ uint32_t tops[kMaxWaves];
  const DropKeys keys(a.drop);
  const int64_t row = blockIdx.x;
  const int64_t pieces = (a.cols + kPiece - 1) / kPiece;
  const int64_t rounds = (pieces + T - 1) / T;
  float ss = 0.0f;
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t piece = k * T + threadIdx.x;
    const f32x8 h = load_h<X, S>(a, keys, row, piece, valid_of(a.cols, piece));
    ss += dot8(h, h);
  }
  ss = row_sum<0>(ss, shared);
  const float rstd = rsqrtf(fmaf(ss, a.inv_cols, a.eps));
  if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
  uint32_t top = 0;
  if (kEight && a.group_lanes == 0) {
    for (int64_t k = 0; k < rounds; ++k) {
      const int64_t piece = k * T + threadIdx.x;
      const int valid = valid_of(a.cols, piece);
      f32x8 y = load_h<X, S>(a, keys, row, piece, valid) * rstd;
      if (a.weight != nullptr) y *= load_weight<X>(a.weight, piece, a.weight_f32, valid);
      const uint32_t m = max8(y);
      top = m > top ? m : top;
    }
    top = lanes_max(top, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) tops[threadIdx.x / kWave] = top;
    __syncthreads();
    for (int i = 0; i < kMaxWaves; ++i) top = tops[i] > top ? tops[i] : top;
  }
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t piece = k * T + threadIdx.x;
    const int valid = valid_of(a.cols, piece);
    const int64_t at = row * a.cols + piece * kPiece;
    f32x8 y = load_h<X, S>(a, keys, row, piece, valid);
    if (a.h != nullptr) store8(static_cast<S*>(a.h) + at, y, valid);
    y *= rstd;
    if (a.weight != nullptr) y *= load_weight<X>(a.weight, piece, a.weight_f32, valid);
    if (!kEight) {
      store8(static_cast<X*>(a.y) + at, y, valid);
      continue;
    }
    const uint32_t m = a.group_lanes != 0 ? lanes_max(max8(y), a.group_lanes) : top;
    const float scale = e4m3_scale(m);
    const bool first = a.group_lanes == 0 ? piece == 0 : (piece & (a.group_lanes - 1)) == 0;
    if (first && valid > 0) a.scales[row * a.groups + (a.group_lanes == 0 ? 0 : piece / a.group_lanes)] = scale;
    store_e4m3(static_cast<uint8_t*>(a.y) + at, y, scale, valid);
  }
}

// ---- gradient -----------------------------------------------------------------------------------
struct NormGradArgs {
  const void* grad;      // of y, rows' type
  const void* h;         // the stream's type
  const void* weight;    // may be null
  const float* rstd;
  const void* grad_h;    // may be null; the stream's type
  void* grad_x;          // rows' type
  void* grad_res;        // may be null; the stream's type
  float* partial;        // [blocks][cols] rows of grad_weight's sum; null without grad_weight or with ...
  void* grad_weight;     // ... the result itself, of a call with one block
  int64_t grad_stride, h_stride, grad_h_stride, rows, cols;
  int weight_f32;
  DropArgs drop;
};

// A block takes every gridDim.x-th group of rows, so that a lane meets the same columns again and
// keeps its part of grad_weight in registers until the end.  Lanes as in rms_norm_kernel.
template <typename X, typename S, int T, int K>
__global__ __launch_bounds__(T ? kThreads : kMaxWaves* kWave, T == 0 && K == 1 ? 6 : 1) void rms_norm_grad_kernel(NormGradArgs a) {
  constexpr int kRows = T ? kThreads / (T ? T : 1) : 1;
  __shared__ float shared[kMaxWaves];
  __shared__ f32x8 parts[kRows > 1 ? kThreads * K : 1];
  const DropKeys keys(a.drop);
  const int lanes = T ? T : blockDim.x;
  const int lane = T ? threadIdx.x % (T ? T : 1) : threadIdx.x;
  const int sub = T ? threadIdx.x / (T ? T : 1) : 0;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f32x8 w[K], dw[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t piece = k * lanes + lane;
    dw[k] = zero;
    w[k] = a.weight != nullptr ? load_weight<X>(a.weight, piece, a.weight_f32, valid_of(a.cols, piece)) : zero + 1.0f;
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t row = base + sub;
    const bool in = row < a.rows;
    const float rstd = in ? a.rstd[row] : 0.0f;
    f32x8 g[K], n[K], gh[K];
    int valid[K];
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t piece = k * lanes + lane;
      valid[k] = in ? valid_of(a.cols, piece) : 0;
      g[k] = load8(static_cast<const X*>(a.grad) + row * a.grad_stride + piece * kPiece, valid[k]);
      n[k] = load8(static_cast<const S*>(a.h) + row * a.h_stride + piece * kPiece, valid[k]);
      if (a.grad_h != nullptr)
        gh[k] = load8(static_cast<const S*>(a.grad_h) + row * a.grad_h_stride + piece * kPiece, valid[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      n[k] *= rstd;
      dw[k] = __builtin_elementwise_fma(g[k], n[k], dw[k]);
      g[k] *= w[k];
      dot += dot8(g[k], n[k]);
    }
    const float along = row_sum<T>(dot, shared) * inv_cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t piece = k * lanes + lane;
      f32x8 d = (g[k] - n[k] * along) * rstd;
      if (a.grad_h != nullptr) d += gh[k];
      if (a.grad_res != nullptr) store8(static_cast<S*>(a.grad_res) + row * a.cols + piece * kPiece, d, valid[k]);
      if (keys.on()) d = keys.apply(d, static_cast<uint32_t>(row), static_cast<uint32_t>(piece));
      store8(static_cast<X*>(a.grad_x) + row * a.cols + piece * kPiece, d, valid[k]);
    }
  }
  if (a.partial == nullptr && a.grad_weight == nullptr) return;
  if (kRows > 1) {   // the rows of a block, in order
#pragma unroll
    for (int k = 0; k < K; ++k) parts[k * kThreads + threadIdx.x] = dw[k];
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
      for (int s = 1; s < kRows; ++s) dw[k] += parts[k * kThreads + s * T + lane];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t piece = k * lanes + lane;
    const int valid = valid_of(a.cols, piece);
    if (a.partial != nullptr) store8(a.partial + blockIdx.x * a.cols + piece * kPiece, dw[k], valid);
    else if (a.weight_f32) store8(static_cast<float*>(a.grad_weight) + piece * kPiece, dw[k], valid);
    else store8(static_cast<X*>(a.grad_weight) + piece * kPiece, dw[k], valid);
  }
}

// rows of more than kMaxPieces pieces: the row is read again behind the sum
template <typename X, typename S>
__global__ __launch_bounds__(1024) void rms_norm_grad_long_kernel(NormGradArgs a) {
  constexpr int T = 1024;
  __shared__ float shared[kMaxWaves];
  const DropKeys keys(a.drop);
  const int64_t row = blockIdx.x;
  const int64_t pieces = (a.cols + kPiece - 1) / kPiece;
  const float rstd = a.rstd[row];
  float dot = 0.0f;
  for (int64_t piece = threadIdx.x; piece < pieces; piece += T) {
    const int valid = valid_of(a.cols, piece);
    f32x8 g = load8(static_cast<const X*>(a.grad) + row * a.grad_stride + piece * kPiece, valid);
    if (a.weight != nullptr) g *= load_weight<X>(a.weight, piece, a.weight_f32, valid);
    dot += dot8(g, load8(static_cast<const S*>(a.h) + row * a.h_stride + piece * kPiece, valid) * rstd);
  }
  const float along = row_sum<0>(dot, shared) / static_cast<float>(a.cols);
  for (int64_t piece = threadIdx.x; piece < pieces; piece += T) {
    const int valid = valid_of(a.cols, piece);
    f32x8 g = load8(static_cast<const X*>(a.grad) + row * a.grad_stride + piece * kPiece, valid);
    if (a.weight != nullptr) g *= load_weight<X>(a.weight, piece, a.weight_f32, valid);
    const f32x8 n = load8(static_cast<const S*>(a.h) + row * a.h_stride + piece * kPiece, valid) * rstd;
    f32x8 d = (g - n * along) * rstd;
    if (a.grad_h != nullptr) d += load8(static_cast<const S*>(a.grad_h) + row * a.grad_h_stride + piece * kPiece, valid);
    if (a.grad_res != nullptr) store8(static_cast<S*>(a.grad_res) + row * a.cols + piece * kPiece, d, valid);
    if (keys.on()) d = keys.apply(d, static_cast<uint32_t>(row), static_cast<uint32_t>(piece));
    store8(static_cast<X*>(a.grad_x) + row * a.cols + piece * kPiece, d, valid);
  }
}

// ... and grad_weight's partial rows: block (x, y) takes kThreads pieces and every gridDim.y-th row
template <typename X, typename S>
__global__ __launch_bounds__(kThreads) void rms_norm_grad_weight_kernel(NormGradArgs a) {
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int valid = valid_of(a.cols, piece);
  if (valid == 0) return;
  f32x8 dw = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const f32x8 g = load8(static_cast<const X*>(a.grad) + row * a.grad_stride + piece * kPiece, valid);
    dw += g * (load8(static_cast<const S*>(a.h) + row * a.h_stride + piece * kPiece, valid) * a.rstd[row]);
  }
  store8(a.partial + blockIdx.y * a.cols + piece * kPiece, dw, valid);
}

// out[c] = sum of partial[0 .. blocks)[c]: 64 columns a block, 16 waves that take the rows in turn
constexpr int kFoldWaves = 16;
template <typename W>
__global__ __launch_bounds__(kFoldWaves* kWave) void fold_rows_kernel(const float* __restrict__ partial, int64_t blocks,
                                                                      int64_t cols, W* __restrict__ out) {
  constexpr int U = 8;
  __shared__ float part[kFoldWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kWave + lane;
  float acc = 0.0f;
  if (col < cols) {
    for (int64_t b = wave; b < blocks; b += kFoldWaves * U) {
      float v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t i = b + k * kFoldWaves;
        v[k] = i < blocks ? partial[i * cols + col] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) acc += v[k];
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || col >= cols) return;
  for (int w = 1; w < kFoldWaves; ++w) acc += part[w][lane];
  out[col] = static_cast<W>(acc);
}

template <typename X, typename S, bool kEight>
int launch_norm(const NormArgs& a, hipStream_t st) {
  const int64_t pieces = ceil_div(a.cols, kPiece);
#define HADES_NORM(T_, K_)                                                                            \
  do {                                                                                                \
    const int64_t block = T_ ? kThreads : ceil_div(ceil_div(pieces, K_), kWave) * kWave;              \
    const int64_t blocks = T_ ? ceil_div(a.rows, kThreads / (T_ ? T_ : 1)) : a.rows;                  \
    HADES_REQUIRE(blocks < kMostThreads / block, "rms_norm: too many rows for one call");             \
    HADES_LAUNCH((rms_norm_kernel<X, S, T_, K_, kEight>), dim3(static_cast<unsigned>(blocks)),        \
                 dim3(static_cast<unsigned>(block)), 0, st, a);                                       \
    return HADES_OK;                                                                                  \
  } while (0)
  if (pieces <= 8) HADES_NORM(8, 1);
  if (pieces <= 16) HADES_NORM(16, 1);
  if (pieces <= 32) HADES_NORM(32, 1);
  if (pieces <= 64) HADES_NORM(64, 1);
  if (pieces <= kMaxPieces / 2) HADES_NORM(0, 1);
  if (pieces <= kMaxPieces) HADES_NORM(0, 2);
#undef HADES_NORM
  HADES_REQUIRE(a.rows < kMostThreads / 1024, "rms_norm: too many rows for one call");
  HADES_LAUNCH((rms_norm_long_kernel<X, S, kEight>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, st, a);
  return HADES_OK;
}

// threads of a block of the gradient kernel
int64_t grad_threads(int64_t pieces) {
  if (pieces <= kWave) return kThreads;
  return ceil_div(ceil_div(pieces, pieces <= kGradOne ? 1 : 2), kWave) * kWave;
}

// Blocks of the gradient kernel = rows of grad_weight's partial sum.  More waves on a compute unit than it
// takes to keep memory busy cost time: 12 for 16-bit rows, 8 for float32 rows, which have twice the bytes in
// flight, but two blocks where they fit (one of them waits for its row's sum meanwhile).  16-bit rows that leave
// lanes idle want as many as are resident.  us for 2^26 bfloat16 values with dropout, 12 / 24 waves: rows of 1 024
// 131 / 146, 2 048 132 / 141, 768 203 / 147, 1 000 173 / 150; 2^25 float32 values, 8 / 16 waves: 2 048 127 / 135.
int64_t grad_blocks(int64_t rows, int64_t cols, bool f32) {
  const int64_t pieces = ceil_div(cols, kPiece);
  if (pieces > kMaxPieces) return rows < 64 ? rows : 64;
  int64_t lanes = 8;
  while (lanes < kWave && lanes < pieces) lanes *= 2;
  const int64_t blocks = pieces <= kWave ? ceil_div(rows, kThreads / lanes) : rows;
  const int64_t block = grad_threads(pieces) / kWave;
  if (blocks <= kGradAlone) return 1;
  const bool full = pieces <= kWave ? pieces == lanes : pieces % kWave == 0;
  int64_t per_cu = (f32 ? 8 : (full ? 12 : (pieces <= kWave ? 20 : 24))) / block;
  if (per_cu < 2) per_cu = pieces <= kGradOne || block <= 8 ? 2 : 1;
  return blocks < per_cu * kCus ? blocks : per_cu * kCus;
}

// bytes of the partial rows; a call with one block, or none, has none
size_t grad_bytes(int64_t rows, int64_t cols, bool f32) {
  if (grad_blocks(rows, cols, f32) <= 1 && ceil_div(cols, kPiece) <= kMaxPieces) return 0;
  const size_t b = static_cast<size_t>(grad_blocks(rows > 0 ? rows : 1, cols, f32)) * cols * sizeof(float);
  return (b + 255) & ~size_t(255);
}

template <typename X, typename S>
int launch_norm_grad(const NormGradArgs& a, hipStream_t st) {
  const int64_t pieces = ceil_div(a.cols, kPiece);
  const unsigned blocks = static_cast<unsigned>(grad_blocks(a.rows, a.cols, sizeof(X) == 4));
#define HADES_NORM_GRAD(T_, K_)                                                                        \
  do {                                                                                                 \
    HADES_LAUNCH((rms_norm_grad_kernel<X, S, T_, K_>), dim3(blocks),                                   \
                 dim3(static_cast<unsigned>(grad_threads(pieces))), 0, st, a);                         \
    return HADES_OK;                                                                                   \
  } while (0)
  if (pieces <= 8) HADES_NORM_GRAD(8, 1);
  if (pieces <= 16) HADES_NORM_GRAD(16, 1);
  if (pieces <= 32) HADES_NORM_GRAD(32, 1);
  if (pieces <= 64) HADES_NORM_GRAD(64, 1);
  if (pieces <= kGradOne) HADES_NORM_GRAD(0, 1);
  if (pieces <= kMaxPieces) HADES_NORM_GRAD(0, 2);
#undef HADES_NORM_GRAD
  HADES_REQUIRE(a.rows < kMostThreads / 1024, "rms_norm_grad: too many rows for one call");
  HADES_LAUNCH((rms_norm_grad_long_kernel<X, S>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, st, a);
  if (a.partial != nullptr)
    HADES_LAUNCH((rms_norm_grad_weight_kernel<X, S>),
                 dim3(static_cast<unsigned>(ceil_div(pieces, kThreads)), blocks), dim3(kThreads), 0, st, a);
  return HADES_OK;
}

bool row_type(int dtype) { return dtype == HADES_F32 || dtype == HADES_F16 || dtype == HADES_BF16; }

}  // namespace
}  // namespace hades

using namespace hades;

extern "C" {

int hades_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t res_stride, const void* weight,
                   void* y, float* scales, void* h, float* rstd, int64_t rows, int64_t cols, int dtype,
                   int stream_dtype, int weight_dtype, int64_t group, float eps, double p, uint64_t seed,
                   int64_t offset, const int64_t* offset_ptr, void* stream) {
  HADES_REQUIRE(rows >= 0 && cols >= 1, "rows must be >= 0 and cols >= 1");
  HADES_REQUIRE(rows < (int64_t(1) << 32) && cols < (int64_t(1) << 31), "rms_norm: rows or cols too large");
  HADES_REQUIRE(row_type(dtype), "Type can only be float, half or bfloat16");
  HADES_REQUIRE(stream_dtype == dtype || stream_dtype == HADES_F32, "the residual's type is the rows' or float");
  HADES_REQUIRE(weight_dtype == dtype || weight_dtype == HADES_F32, "the weight's type is the rows' or float");
  HADES_REQUIRE(eps >= 0.0f, "eps must be >= 0");
  HADES_REQUIRE(group == 0 || (is_pow2(group) && group >= kPiece && group <= kPiece * kWave),
                "group must be 0 or a power of two in [8, 512]");
  DropArgs drop;
  HADES_REQUIRE(make_drop(p, seed, offset, offset_ptr, 1.0, &drop), "p must lie in [0, 1]");
  if (rows == 0) return HADES_OK;
  HADES_REQUIRE(x && y, "null pointer argument");
  HADES_REQUIRE(x_stride >= cols || rows == 1, "row stride below cols");
  HADES_REQUIRE(!residual || res_stride >= cols || rows == 1, "row stride below cols");
  NormArgs a;
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.y = y;
  a.h = h;
  a.rstd = rstd;
  a.scales = scales;
  a.x_stride = x_stride;
  a.res_stride = res_stride;
  a.rows = rows;
  a.cols = cols;
  a.weight_f32 = weight_dtype == HADES_F32;
  a.group_lanes = static_cast<int>(group / kPiece);
  a.groups = group == 0 ? 1 : ceil_div(cols, group);
  a.eps = eps;
  a.inv_cols = static_cast<float>(1.0 / static_cast<double>(cols));
  a.drop = drop;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define HADES_NORM_TYPE(X_, S_) \
  return scales != nullptr ? launch_norm<X_, S_, true>(a, st) : launch_norm<X_, S_, false>(a, st)
  if (dtype == HADES_F32) HADES_NORM_TYPE(float, float);
  if (dtype == HADES_F16) {
    if (stream_dtype == HADES_F16) HADES_NORM_TYPE(f16, f16);
    HADES_NORM_TYPE(f16, float);
  }
  if (stream_dtype == HADES_BF16) HADES_NORM_TYPE(bf16, bf16);
  HADES_NORM_TYPE(bf16, float);
#undef HADES_NORM_TYPE
}

size_t hades_rms_norm_grad_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return 0;
  const size_t narrow = grad_bytes(rows, cols, false), wide = grad_bytes(rows, cols, true);
  return narrow > wide ? narrow : wide;   // of either type of rows
}

int hades_rms_norm_grad(const void* grad, int64_t grad_stride, const void* h, int64_t h_stride, const void* weight,
                        const float* rstd, const void* grad_h, int64_t grad_h_stride, void* grad_x, void* grad_res,
                        void* grad_weight, int64_t rows, int64_t cols, int dtype, int stream_dtype,
                        int weight_dtype, double p, uint64_t seed, int64_t offset, const int64_t* offset_ptr,
                        void* workspace, size_t workspace_bytes, void* stream) {
  HADES_REQUIRE(rows >= 0 && cols >= 1, "rows must be >= 0 and cols >= 1");
  HADES_REQUIRE(rows < (int64_t(1) << 32) && cols < (int64_t(1) << 31), "rms_norm_grad: rows or cols too large");
  HADES_REQUIRE(row_type(dtype), "Type can only be float, half or bfloat16");
  HADES_REQUIRE(stream_dtype == dtype || stream_dtype == HADES_F32, "the residual's type is the rows' or float");
  HADES_REQUIRE(weight_dtype == dtype || weight_dtype == HADES_F32, "the weight's type is the rows' or float");
  HADES_REQUIRE(!grad_weight || weight, "grad_weight without a weight");
  // the partial rows' sum has sixteen threads a column
  HADES_REQUIRE(!grad_weight || cols <= kMostThreads / kFoldWaves - kWave,
                "rms_norm_grad: too many columns for one call");
  DropArgs drop;
  HADES_REQUIRE(make_drop(p, seed, offset, offset_ptr, 1.0, &drop), "p must lie in [0, 1]");
  if (rows == 0 && !grad_weight) return HADES_OK;
  HADES_REQUIRE(rows == 0 || (grad && h && rstd && grad_x), "null pointer argument");
  HADES_REQUIRE(grad_stride >= cols || rows <= 1, "row stride below cols");
  HADES_REQUIRE(h_stride >= cols || rows <= 1, "row stride below cols");
  HADES_REQUIRE(!grad_h || grad_h_stride >= cols || rows <= 1, "row stride below cols");
  const size_t need = grad_weight ? grad_bytes(rows, cols, dtype == HADES_F32) : 0;
  if (need != 0 && (workspace == nullptr || workspace_bytes < need))
    return set_error(HADES_ERR_WORKSPACE, "rms_norm_grad workspace too small: need %zu bytes, got %zu", need,
                     workspace_bytes);
  HADES_REQUIRE((align_of_ptr(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  NormGradArgs a;
  a.grad = grad;
  a.h = h;
  a.weight = weight;
  a.rstd = rstd;
  a.grad_h = grad_h;
  a.grad_x = grad_x;
  a.grad_res = grad_res;
  a.partial = need != 0 ? static_cast<float*>(workspace) : nullptr;
  a.grad_weight = grad_weight;
  a.grad_stride = grad_stride;
  a.h_stride = h_stride;
  a.grad_h_stride = grad_h_stride;
  a.rows = rows;
  a.cols = cols;
  a.weight_f32 = weight_dtype == HADES_F32;
  a.drop = drop;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = HADES_OK;
  if (rows > 0) {
    if (dtype == HADES_F32) rc = launch_norm_grad<float, float>(a, st);
    else if (dtype == HADES_F16)
      rc = stream_dtype == HADES_F16 ? launch_norm_grad<f16, f16>(a, st) : launch_norm_grad<f16, float>(a, st);
    else rc = stream_dtype == HADES_BF16 ? launch_norm_grad<bf16, bf16>(a, st) : launch_norm_grad<bf16, float>(a, st);
  }
  if (rc != HADES_OK || !grad_weight || (rows > 0 && need == 0)) return rc;
  const int64_t blocks = rows > 0 ? grad_blocks(rows, cols, dtype == HADES_F32) : 0;
  const dim3 grid(static_cast<unsigned>(ceil_div(cols, kWave))), block(kFoldWaves * kWave);
#define HADES_FOLD(W_) \
  HADES_LAUNCH((fold_rows_kernel<W_>), grid, block, 0, st, a.partial, blocks, cols, static_cast<W_*>(grad_weight))
  if (weight_dtype == HADES_F32) HADES_FOLD(float);
  else if (weight_dtype == HADES_F16) HADES_FOLD(f16);
  else HADES_FOLD(bf16);
#undef HADES_FOLD
  return HADES_OK;
}

}  // extern "C"
