// paged_tile.h - what the attention kernels over a paged cache share: types of
// the matrix operands, sums over a head's lanes, operands made of fp32 values.
#pragma once
#include <type_traits>

#include "moe_device.h"
#include "paged_attn.h"

namespace moe {
namespace {

enum { F32 = MOE_PAGE_F32, F16 = MOE_PAGE_F16, BF16 = MOE_PAGE_BF16, E4M3 = MOE_PAGE_E4M3 };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // queries may start at any float
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Memory that no one writes while the kernel runs, read at an address all lanes share: through the scalar cache, apart
// from the vector loads in flight.
template <class T>
__device__ __forceinline__ T scalar_load(const T* p, long long i) {
  return ((const __attribute__((address_space(4))) T*)(uintptr_t)p)[i];
}

// max over the four lanes of a head (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float head_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float head_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// sum over the wave's lanes, in all of them
__device__ __forceinline__ float wave_total(float x) {
  auto step = [&](auto ctrl, auto mask) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, decltype(mask)::value, 0xf, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Two fp32 values into the same place of three operands whose sum they are: bf16 parts by truncation (8 + 8 + 8 bits),
// f16 parts by the hardware's conversion toward zero (11 bits each).
template <bool HALF>
__device__ __forceinline__ void split2(float x, float y, uint32_t* a, uint32_t* b, uint32_t* c) {
  if constexpr (HALF) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const float x1 = x - (float)h[0], y1 = y - (float)h[1];
    const auto m = __builtin_amdgcn_cvt_pkrtz(x1, y1);
    const auto l = __builtin_amdgcn_cvt_pkrtz(x1 - (float)m[0], y1 - (float)m[1]);
    *a = __builtin_bit_cast(uint32_t, h);
    *b = __builtin_bit_cast(uint32_t, m);
    *c = __builtin_bit_cast(uint32_t, l);
  } else {
    const uint32_t xh = __float_as_uint(x), yh = __float_as_uint(y);
    const float x1 = x - __uint_as_float(xh & 0xffff0000u), y1 = y - __uint_as_float(yh & 0xffff0000u);
    const uint32_t xm = __float_as_uint(x1), ym = __float_as_uint(y1);
    const float x2 = x1 - __uint_as_float(xm & 0xffff0000u), y2 = y1 - __uint_as_float(ym & 0xffff0000u);
    *a = __builtin_amdgcn_perm(yh, xh, 0x07060302u);
    *b = __builtin_amdgcn_perm(ym, xm, 0x07060302u);
    *c = __builtin_amdgcn_perm(__float_as_uint(y2), __float_as_uint(x2), 0x07060302u);
  }
}

template <bool HALF>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (HALF)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// four 8-bit values -> two dwords of bf16 pairs (exact)
__device__ __forceinline__ u32x2 widen(uint32_t x) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true))};
}

// BYTES at p; STREAM: past the caches.
template <int BYTES, bool STREAM>
__device__ __forceinline__ void load_piece(const char* p, uint32_t* r) {
  typedef uint32_t V __attribute__((ext_vector_type(BYTES / 4)));
  V x;
  if constexpr (STREAM) x = __builtin_nontemporal_load((const V*)p);
  else x = *(const V*)p;
  if constexpr (BYTES == 4) r[0] = x.x;
  else
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) r[i] = x[i];
}

}  // namespace
}  // namespace moe
