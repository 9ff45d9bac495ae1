// Storage types of the row operators (bf16, fp16, fp32) and their loads and stores.
#pragma once

#include <type_traits>

#include "mt_common.h"

namespace mt {
namespace ops {

constexpr int kDtBF16 = 0;
constexpr int kDtFP16 = 1;
constexpr int kDtFP32 = 2;

// ---------------------------------------------------------------------------
// storage <-> fp32, 8 consecutive values at a time (16 bytes for 16-bit types,
// 32 bytes for fp32); element offsets must be multiples of 8
// ---------------------------------------------------------------------------
template <int DT>
struct IO {
  // 8 values as loaded (unpacked only where they are used: half the registers
  // of a 16-bit row while it is in flight)
  struct Raw {
    u32x4 w[DT == kDtFP32 ? 2 : 1];
  };
  static __device__ __forceinline__ Raw load_raw(const void* base, int64_t i) {
    Raw r;
    const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(base) + i * (DT == kDtFP32 ? 4 : 2));
    r.w[0] = p[0];
    if constexpr (DT == kDtFP32) r.w[1] = p[1];
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float* v) {
    if constexpr (DT == kDtFP32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(r.w[k >> 2][k & 3]);
    } else {
      using E = typename std::conditional<DT == kDtBF16, BF16, FP16>::type;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = lo_f<E>(r.w[0][k]);
        v[2 * k + 1] = hi_f<E>(r.w[0][k]);
      }
    }
  }
  static __device__ __forceinline__ void load8(const void* base, int64_t i, float* v) {
    if constexpr (DT == kDtFP32) {
      const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i);
      const f32x4 a = p[0], b = p[1];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = a[k];
        v[4 + k] = b[k];
      }
    } else {
      using E = typename std::conditional<DT == kDtBF16, BF16, FP16>::type;
      const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = lo_f<E>(w[k]);
        v[2 * k + 1] = hi_f<E>(w[k]);
      }
    }
  }
  static __device__ __forceinline__ void store8(void* base, int64_t i, const float* v) {
    if constexpr (DT == kDtFP32) {
      f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + i);
      p[0] = f32x4{v[0], v[1], v[2], v[3]};
      p[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      using E = typename std::conditional<DT == kDtBF16, BF16, FP16>::type;
      u32x4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = pack2<E>(v[2 * k], v[2 * k + 1]);
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + i) = w;
    }
  }
  static __device__ __forceinline__ float load1(const void* base, int64_t i) {
    if constexpr (DT == kDtFP32) return static_cast<const float*>(base)[i];
    else if constexpr (DT == kDtBF16) return BF16::to_f(static_cast<const uint16_t*>(base)[i]);
    else return FP16::to_f(static_cast<const uint16_t*>(base)[i]);
  }
  static __device__ __forceinline__ void store1(void* base, int64_t i, float x) {
    if constexpr (DT == kDtFP32) static_cast<float*>(base)[i] = x;
    else if constexpr (DT == kDtBF16) static_cast<uint16_t*>(base)[i] = uint16_t(pack2<BF16>(x, 0.f) & 0xffffu);
    else static_cast<uint16_t*>(base)[i] = uint16_t(pack2<FP16>(x, 0.f) & 0xffffu);
  }
  // the value x takes after a store to and a load from this storage type
  static __device__ __forceinline__ float round(float x) {
    if constexpr (DT == kDtFP32) return x;
    else if constexpr (DT == kDtBF16) return lo_f<BF16>(pack2<BF16>(x, 0.f));
    else return lo_f<FP16>(pack2<FP16>(x, 0.f));
  }
};

typedef u32x4 u32x4_any __attribute__((aligned(2)));

// 8 consecutive values at any element offset: a global access of 16 bytes takes any address
template <int DT>
__device__ __forceinline__ typename IO<DT>::Raw load8_any(const void* base, int64_t i) {
  const u32x4_any* p = reinterpret_cast<const u32x4_any*>(static_cast<const char*>(base) + i * (DT == kDtFP32 ? 4 : 2));
  typename IO<DT>::Raw r;
  r.w[0] = p[0];
  if constexpr (DT == kDtFP32) r.w[1] = p[1];
  return r;
}
// PAST: past the caches, for what is too large to stay in them
template <bool PAST>
__device__ __forceinline__ void put16(u32x4_any* p, u32x4 v) {
  if constexpr (PAST) __builtin_nontemporal_store((u32x4_any)v, p);
  else *p = v;
}
template <int DT, bool PAST = false>
__device__ __forceinline__ void store8_any(void* base, int64_t i, const float* v) {
  u32x4_any* p = reinterpret_cast<u32x4_any*>(static_cast<char*>(base) + i * (DT == kDtFP32 ? 4 : 2));
  if constexpr (DT == kDtFP32) {
    put16<PAST>(p, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    put16<PAST>(p + 1, u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
  } else {
    using E = typename std::conditional<DT == kDtBF16, BF16, FP16>::type;
    put16<PAST>(p, u32x4{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7])});
  }
}

}  // namespace ops
}  // namespace mt
