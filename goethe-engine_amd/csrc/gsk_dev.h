// Device helpers of the paged cache's operators: eight elements of a row between memory and fp32.
#pragma once
#include "../../include/gsk.h"
#include "gse_dev.h"

namespace gse {

template <uint32_t T>
constexpr int type_size = T == GSK_F32 ? 4 : T == GSK_BF16 || T == GSK_F16 ? 2 : 1;
template <uint32_t T>
constexpr bool type_is_8bit = T == GSK_E4M3 || T == GSK_I8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight elements as they lie in memory (8, 16 or 32 bytes).
template <uint32_t T>
struct Raw8 {
  static constexpr int N = type_size<T> * 2;
  uint32_t w[N];
};

template <uint32_t T>
__device__ __forceinline__ Raw8<T> load_raw8(const void *p) {
  Raw8<T> r;
  if constexpr (Raw8<T>::N == 2) {
    *(uint2 *)r.w = *(const uint2 *)p;
  } else {
#pragma unroll
    for (int i = 0; i < Raw8<T>::N; i += 4) *(uint4 *)(r.w + i) = ((const uint4 *)p)[i / 4];
  }
  return r;
}

template <uint32_t T>
__device__ __forceinline__ void to_f32(const Raw8<T> &r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (T == GSK_F32) x[i] = __uint_as_float(r.w[i]);
    if constexpr (T == GSK_BF16) x[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xFFFF0000u : r.w[i / 2] << 16);
    if constexpr (T == GSK_F16) x[i] = (float)__builtin_bit_cast(f16x2, r.w[i / 2])[i & 1];
    if constexpr (T == GSK_I8) x[i] = (float)((int32_t)(r.w[i / 4] << (24 - 8 * (i & 3))) >> 24);
  }
  if constexpr (T == GSK_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[i], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[i], true);
      x[4 * i] = lo[0];
      x[4 * i + 1] = lo[1];
      x[4 * i + 2] = hi[0];
      x[4 * i + 3] = hi[1];
    }
  }
}

// Rounds to nearest, ties to even; what T cannot hold becomes an infinity (8 bits: the caller keeps it in range).
template <uint32_t T>
__device__ __forceinline__ Raw8<T> from_f32(const float (&x)[8]) {
  Raw8<T> r;
  if constexpr (T == GSK_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(x[i]);
  }
  if constexpr (T == GSK_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
  }
  if constexpr (T == GSK_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
  }
  if constexpr (T == GSK_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      r.w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
    }
  }
  if constexpr (T == GSK_I8) {  // (added to 1.5 * 2^23, a number's lowest byte is its nearest whole number)
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(x[i] + 12582912.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0C0C0400u), 0x05040100u);
  }
  return r;
}

template <uint32_t T>
__device__ __forceinline__ void store_raw8(void *p, const Raw8<T> &r) {
  if constexpr (Raw8<T>::N == 2) {
    *(uint2 *)p = *(const uint2 *)r.w;
  } else {
#pragma unroll
    for (int i = 0; i < Raw8<T>::N; i += 4) ((uint4 *)p)[i / 4] = *(const uint4 *)(r.w + i);
  }
}

// Division by a number of the host's choice: the quotient by its inverse is the one wanted or one less.
struct Div {
  uint32_t d, inverse;
};
inline Div div_by(uint32_t d) { return {d, d > 1 ? (uint32_t)((1ull << 32) / d) : ~0u}; }
__device__ __forceinline__ uint32_t quotient(uint32_t x, Div v, uint32_t &rest) {
  uint32_t q = __umulhi(x, v.inverse);
  rest = x - q * v.d;
  if (rest >= v.d) rest -= v.d, ++q;
  return q;
}

// The largest of a group of 8, 16 or 32 lanes, in each of them.
template <int GL>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = max(m, dpp32<0xB1, 0xF>(0u, m));   // lane ^ 1
  m = max(m, dpp32<0x4E, 0xF>(0u, m));   // lane ^ 2
  m = max(m, dpp32<0x141, 0xF>(0u, m));  // mirrored in eight
  if constexpr (GL > 8) m = max(m, dpp32<0x140, 0xF>(0u, m));  // mirrored in sixteen
  if constexpr (GL > 16) m = max(m, shfl_xor_u32(m, 16));
  return m;
}

// The last r in [0, n) with first[r] <= x (first ascends), 0 where there is none: found by the whole wave, 64 entries a step.
__device__ __forceinline__ uint32_t wave_find(const int32_t *first, uint32_t n, int64_t x) {
  const uint32_t lane = (uint32_t)lane_id();
  uint32_t lo = 0;
  for (;;) {
    const uint32_t step = (n + WAVE - 1) / WAVE;
    const bool below = lane * step < n && first[lo + lane * step] <= x;
    const uint32_t k = (uint32_t)__popcll(ballot64(below));
    if (k == 0) return lo;
    lo += (k - 1) * step;
    if (step == 1) return lo;
    n = min(step, n - (k - 1) * step);
  }
}

}  // namespace gse
