// Device helpers of the label-vocabulary operators (distill.hip, logits.hip, embed.hip): element
// types, and rows that start anywhere read and written in aligned 16-byte granules.
#pragma once

#include <type_traits>

#include "sbod_common.h"

namespace sbod {
namespace label {

// One element type of the ABI (SBOD_DT_*): P elements fill a 16-byte granule.  All arithmetic is
// in 32 bits; a store rounds once to nearest even (gfx950's own conversions).
template <int DT>
struct Elt;
template <>
struct Elt<SBOD_DT_F32> {
  using T = float;
  static constexpr int P = 4;
};
template <>
struct Elt<SBOD_DT_BF16> {
  using T = __bf16;
  static constexpr int P = 8;
};
template <>
struct Elt<SBOD_DT_F16> {
  using T = _Float16;
  static constexpr int P = 8;
};

inline size_t elt_bytes(int dt) { return dt == SBOD_DT_F32 ? 4 : 2; }
inline bool known_dt(int dt) { return dt == SBOD_DT_F32 || dt == SBOD_DT_BF16 || dt == SBOD_DT_F16; }

template <typename T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

__device__ __forceinline__ float ld_any(const void *p, int64_t i, int dt) {
  if (dt == SBOD_DT_F32) return static_cast<const float *>(p)[i];
  if (dt == SBOD_DT_BF16) return static_cast<float>(static_cast<const __bf16 *>(p)[i]);
  return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
}

// A label id as the caller holds it (int32 or int64); -1 for anything outside [0, v).
__device__ __forceinline__ int ld_id(const void *ids, int64_t i, bool wide, int64_t v) {
  if (wide) {
    const uint64_t id = static_cast<const uint64_t *>(ids)[i];   // (a negative id is above every label)
    return id < static_cast<uint64_t>(v) ? static_cast<int>(id) : -1;
  }
  const uint32_t id = static_cast<const uint32_t *>(ids)[i];
  return id < static_cast<uint64_t>(v) ? static_cast<int>(id) : -1;
}

// The same two in halves: loads without a branch between them or a use behind them, so that they stay in
// flight until the value is asked for.
struct RawId {
  uint32_t lo, hi;
};
__device__ __forceinline__ RawId ld_raw_id(const void *ids, int64_t i, bool wide) {
  const uint32_t *p = static_cast<const uint32_t *>(ids) + (wide ? 2 * i : i);
  return RawId{p[0], p[wide ? 1 : 0]};
}
__device__ __forceinline__ int id_of(RawId r, bool wide, int64_t v) {
  const uint64_t id = (wide ? static_cast<uint64_t>(r.hi) << 32 : 0) | r.lo;
  return id < static_cast<uint64_t>(v) ? static_cast<int>(id) : -1;
}
struct RawAny {
  uint16_t lo, hi;
};
__device__ __forceinline__ RawAny ld_raw_any(const void *q, int64_t i, int dt) {
  const uint16_t *p = static_cast<const uint16_t *>(q) + (dt == SBOD_DT_F32 ? 2 * i : i);
  return RawAny{p[0], p[dt == SBOD_DT_F32 ? 1 : 0]};
}
__device__ __forceinline__ float any_of(RawAny r, int dt) {
  if (dt == SBOD_DT_F32) return __uint_as_float(static_cast<uint32_t>(r.hi) << 16 | r.lo);
  if (dt == SBOD_DT_BF16) return __uint_as_float(static_cast<uint32_t>(r.lo) << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, r.lo));
}
// An element's bits, and its value.
template <int DT>
using bits_t = std::conditional_t<DT == SBOD_DT_F32, uint32_t, uint16_t>;
template <int DT>
__device__ __forceinline__ float bits_value(uint32_t b) {
  if (DT == SBOD_DT_F32) return __uint_as_float(b);
  if (DT == SBOD_DT_BF16) return __uint_as_float(b << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b)));
}

// Elements between the 16-byte boundary at or below p and p itself: granule g of a row at p holds
// the elements [g P - phase, (g + 1) P - phase) of it.
template <typename T>
__device__ __forceinline__ int row_phase(const T *p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// A granule's 16 bytes, and their P values.
typedef uint32_t raw16_t __attribute__((ext_vector_type(4)));
template <int DT>
__device__ __forceinline__ void raw_values(raw16_t r, float (&f)[Elt<DT>::P]) {
#pragma unroll
  for (int j = 0; j < Elt<DT>::P; ++j) {
    if (DT == SBOD_DT_F32) f[j] = __uint_as_float(r[j]);
    else f[j] = bits_value<DT>(r[j >> 1] >> (16 * (j & 1)) & 0xffff);
  }
}

// The elements [e, e + P) of a row of v at p; those outside the row read as `fill`.  p + e is
// 16-byte aligned (row_phase), so a granule inside the row is one load, and nothing outside the row
// is touched.
template <int DT>
__device__ __forceinline__ void ld_granule(const typename Elt<DT>::T *p, int64_t e, int64_t v, float fill,
                                           float (&f)[Elt<DT>::P]) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P;
  if (e >= 0 && e + P <= v) {
    const vec_t<T, P> r = *reinterpret_cast<const vec_t<T, P> *>(p + e);
#pragma unroll
    for (int j = 0; j < P; ++j) f[j] = static_cast<float>(r[j]);
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) f[j] = e + j >= 0 && e + j < v ? static_cast<float>(p[e + j]) : fill;
  }
}

// The same elements written.  `aligned`: p + e is 16-byte aligned; else element by element.  kStream: past
// the caches.
template <int DT, bool kStream = false>
__device__ __forceinline__ void st_granule(typename Elt<DT>::T *p, int64_t e, int64_t v, bool aligned,
                                           const float (&f)[Elt<DT>::P]) {
  using T = typename Elt<DT>::T;
  constexpr int P = Elt<DT>::P;
  if (aligned && e >= 0 && e + P <= v) {
    vec_t<T, P> r;
#pragma unroll
    for (int j = 0; j < P; ++j) r[j] = static_cast<T>(f[j]);
    if (kStream) __builtin_nontemporal_store(r, reinterpret_cast<vec_t<T, P> *>(p + e));
    else *reinterpret_cast<vec_t<T, P> *>(p + e) = r;
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (e + j >= 0 && e + j < v) p[e + j] = static_cast<T>(f[j]);
  }
}

// LDS written by lanes of a wave before this is seen by its other lanes after it.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Reductions over aligned groups of G lanes (a power of two), valid in each lane, without LDS: quad swaps
// and mirrors inside a row of 16 (DPP), then gfx950's row and half swaps: permlane16_swap of v with itself
// gives {row 0, row 0, row 2, row 2} and {row 1, row 1, row 3, row 3}, permlane32_swap the halves likewise.
// All lanes of a group take part; other groups of the wave need not.
template <int kCtrl>
__device__ __forceinline__ float dpp_row(float v) {
  const int x = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, kCtrl, 0xf, 0xf, false));
}
template <int G, typename Op>
__device__ __forceinline__ float group_reduce(float v, Op op) {
  if (G >= 2) v = op(v, dpp_row<0xB1>(v));     // quad_perm [1,0,3,2]
  if (G >= 4) v = op(v, dpp_row<0x4E>(v));     // quad_perm [2,3,0,1]
  if (G >= 8) v = op(v, dpp_row<0x141>(v));    // row_half_mirror
  if (G >= 16) v = op(v, dpp_row<0x140>(v));   // row_mirror
  if (G >= 32) {
    const unsigned x = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const unsigned a = r[0], b = r[1];   // (a bit cast of a vector's element takes its first one)
    v = op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
  }
  if (G >= 64) {
    const unsigned x = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const unsigned a = r[0], b = r[1];   // (a bit cast of a vector's element takes its first one)
    v = op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
  }
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
  return group_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return group_reduce<G>(v, [](float a, float b) { return a + b; });
}
template <int G>
__device__ __forceinline__ double group_sum(double v) {
#pragma unroll
  for (int m = G / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}
// Bit i: lane i of the group.
template <int G>
__device__ __forceinline__ unsigned long long group_ballot(bool b) {
  const unsigned long long m = __ballot(b);
  return G < kWave ? m >> ((threadIdx.x & 63) / G * G) & ((1ull << (G & 63)) - 1) : m;
}
template <int G>
__device__ __forceinline__ bool group_any(bool b) {
  return group_ballot<G>(b) != 0;
}
__device__ __forceinline__ float wave_max_f32(float v) { return group_max<kWave>(v); }

// 2^x by the hardware instruction (1 ulp; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// e^x and log x from it and from the hardware's log2 (1 ulp): e^x is off by |x| half steps more.
__device__ __forceinline__ float exp_hw(float x) { return exp2_hw(x * 1.44269504088896340736f); }
__device__ __forceinline__ float log_hw(float x) { return __builtin_amdgcn_logf(x) * 0.693147180559945309417f; }

}  // namespace label
}  // namespace sbod
