// Rows of float32 / float16 / bfloat16 in pieces of eight values, and the counter-based generator
// behind dropout.  Shared by embed.hip, dropout.hip and rms_norm.hip (not part of the C ABI).
#pragma once

#include "common.h"

namespace hades {

typedef _Float16 f16;
typedef __bf16 bf16;

// eight values of a row: one 16-byte access for the 16-bit types, two for float32
constexpr int kPiece = 8;

// ---- dropout's arguments ------------------------------------------------------------------------
// p as a whole number of 65536ths (0: nothing dropped), the factor of the kept values, and the
// generator's key and counter.  offset_ptr (device, may be null) is added to offset when the kernel
// runs, so that a replayed graph can draw other numbers each time.
struct DropArgs {
  uint32_t threshold;
  float factor;
  uint32_t key0, key1;
  uint64_t offset;
  const int64_t* offset_ptr;
};

// p in [0, 1] to DropArgs; `scale` is a further factor of the kept values.
inline bool make_drop(double p, uint64_t seed, int64_t offset, const int64_t* offset_ptr, double scale,
                      DropArgs* d) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  d->threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  d->factor = d->threshold >= 65536u
                  ? 0.0f : static_cast<float>(scale * (65536.0 / (65536.0 - d->threshold)));
  d->key0 = static_cast<uint32_t>(seed);
  d->key1 = static_cast<uint32_t>(seed >> 32);
  d->offset = static_cast<uint64_t>(offset);
  d->offset_ptr = offset_ptr;
  return true;
}

// Whether rows of this many bytes are read with non-temporal loads: what does not fit the last-level cache (256
// MB) cannot be there from the kernel before, and would only push other data out of it.
inline bool streamed(int64_t bytes) { return bytes >= (int64_t(1) << 28); }

// n / d for n < 2^31 as a multiplication (Granlund and Montgomery's round-up form)
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t div = 1) : d(div) {
    shift = static_cast<uint32_t>(ilog2_ceil(div));
    mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - div)) / div + 1);
  }
#if defined(__HIPCC__)
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};

#if defined(__HIPCC__)

template <typename T>
struct Vec8 {
  typedef T V __attribute__((ext_vector_type(8)));
  // a row may start at any element: the access is only as aligned as one value (gfx950 serves
  // unaligned wide accesses, a row of odd width takes the same instructions as any other)
  typedef V VU __attribute__((aligned(sizeof(T))));
};
typedef float f32x8 __attribute__((ext_vector_type(8)));

// p[0 .. 8), or its first `valid` values and zeros behind them.  kOnce / kPast: non-temporal, for rows
// that are read once and values that are not read again soon.
template <typename T, bool kOnce = false>
__device__ __forceinline__ typename Vec8<T>::V load8_raw(const T* __restrict__ p, int valid) {
  typedef typename Vec8<T>::VU VU;
  if (valid >= kPiece)
    return kOnce ? __builtin_nontemporal_load(reinterpret_cast<const VU*>(p)) : *reinterpret_cast<const VU*>(p);
  typename Vec8<T>::V r;
#pragma unroll
  for (int j = 0; j < kPiece; ++j) r[j] = j < valid ? p[j] : static_cast<T>(0.0f);
  return r;
}

// ... as float32
template <typename T, bool kOnce = false>
__device__ __forceinline__ f32x8 load8(const T* __restrict__ p, int valid) {
  return __builtin_convertvector((load8_raw<T, kOnce>(p, valid)), f32x8);
}

// rounds to nearest even, once
template <typename T, bool kPast = false>
__device__ __forceinline__ void store8(T* __restrict__ p, f32x8 v, int valid) {
  if (valid >= kPiece) {
    typedef typename Vec8<T>::V V;
    typedef typename Vec8<T>::VU VU;
    const VU r = __builtin_convertvector(v, V);
    if (kPast) __builtin_nontemporal_store(r, reinterpret_cast<VU*>(p));
    else *reinterpret_cast<VU*>(p) = r;
    return;
  }
#pragma unroll
  for (int j = 0; j < kPiece - 1; ++j)
    if (j < valid) p[j] = static_cast<T>(v[j]);
}

// The value of lanes that mirror one another, from pairs up to the halves of the wave: after the steps below `n`
// every group of n lanes has combined all its values, whatever the order of the lanes is in a step.
template <int kStep>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
  if (kStep == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);    // lanes 1 0 3 2
  if (kStep == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);    // lanes 2 3 0 1
  if (kStep == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);   // eight lanes reversed
  return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);                   // sixteen lanes reversed
}

// Sum over each group of N lanes of a full wave (N a power of two); every lane gets its group's.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  if (N > 1) v += __uint_as_float(partner<1>(__float_as_uint(v)));
  if (N > 2) v += __uint_as_float(partner<2>(__float_as_uint(v)));
  if (N > 4) v += __uint_as_float(partner<4>(__float_as_uint(v)));
  if (N > 8) v += __uint_as_float(partner<8>(__float_as_uint(v)));
  if (N > 16) {   // rows of 16 lanes: the two results hold the even rows' and the odd rows' values
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (N > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// The largest of each group of n lanes (n a power of two, the same for the whole wave)
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int n) {
  const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  if (n > 1) v = larger(v, partner<1>(v));
  if (n > 2) v = larger(v, partner<2>(v));
  if (n > 4) v = larger(v, partner<4>(v));
  if (n > 8) v = larger(v, partner<8>(v));
  if (n > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  if (n > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  return v;
}

// Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// seven rounds, the fewest that pass the paper's statistical tests: 128 bits for eight values of a row.
// Per piece 14 products of 32 x 32 bits; a dropout of bfloat16 rows stays bound by memory.
struct DropKeys {
  uint32_t threshold, key0, key1, off0, off1;
  float factor;
  __device__ __forceinline__ explicit DropKeys(const DropArgs& d)
      : threshold(d.threshold), key0(d.key0), key1(d.key1), factor(d.factor) {
    uint64_t o = d.offset;
    if (d.offset_ptr != nullptr) o += static_cast<uint64_t>(*d.offset_ptr);
    off0 = static_cast<uint32_t>(o);
    off1 = static_cast<uint32_t>(o >> 32);
  }
  __device__ __forceinline__ bool on() const { return threshold != 0u; }

  // keeps or zeroes the eight values of piece `piece` of row `row`; kept ones are multiplied by
  // factor.  A value that is dropped is 0 whatever it was, infinities and NaN too.
  __device__ __forceinline__ f32x8 apply(f32x8 v, uint32_t row, uint32_t piece) const {
    uint32_t c0 = piece, c1 = row, c2 = off0, c3 = off1, k0 = key0, k1 = key1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
      const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
      c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
      c1 = static_cast<uint32_t>(b);
      c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
      c3 = static_cast<uint32_t>(a);
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
    // both halves of a word without taking it apart: the upper one reaches the threshold if the word is
    // above threshold * 65536 - 1 (2^32 - 1 for p = 1, where nothing is kept)
    const uint32_t w[4] = {c0, c1, c2, c3};
    const uint16_t low = static_cast<uint16_t>(threshold - 1u);
    const uint32_t high = (threshold << 16) - 1u;
#pragma unroll
    for (int j = 0; j < kPiece; j += 2) {
      v[j] = static_cast<uint16_t>(w[j >> 1]) > low ? v[j] * factor : 0.0f;
      v[j + 1] = w[j >> 1] > high ? v[j + 1] * factor : 0.0f;
    }
    return v;
  }
};

#endif  // __HIPCC__

}  // namespace hades
