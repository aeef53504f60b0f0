// Rows over a vocabulary: what embedding.hip and vocab_logits.hip share.
//
// Dense rows are fp32, bf16 or fp16, any row stride, any base alignment that
// the element type has: 16-byte loads and stores are typed with the element's
// own alignment (gfx950 takes unaligned global accesses), so a vocabulary of
// odd size costs one more cache line a wave and no peeled head.
#pragma once
#include "common.hpp"

#include <type_traits>

namespace spmm {

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2), may_alias));   // 16 bytes at a 2- or 4-byte aligned address
typedef u32x4 u32x4_at4 __attribute__((aligned(4), may_alias));

constexpr float kInf = __builtin_inff();

template <typename T>
struct Elem;   // kN elements in a 16-byte vector; kNegInf: two (16-bit) or one negative infinity

template <>
struct Elem<float> {
  static constexpr int kN = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float cast(float x) { return x; }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
};

template <>
struct Elem<__bf16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    const uint32_t w = v[i >> 1];
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float load(const __bf16* p) { return (float)*p; }
  static __device__ __forceinline__ __bf16 cast(float x) { return (__bf16)x; }   // round to nearest even
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i]);
      const uint32_t hi = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]);
      r[i] = lo | (hi << 16);
    }
    return r;
  }
};

template <>
struct Elem<_Float16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    const uint32_t w = v[i >> 1];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)((i & 1) ? (w >> 16) : w));
  }
  static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ _Float16 cast(float x) { return (_Float16)x; }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]);
      const uint32_t hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]);
      r[i] = lo | (hi << 16);
    }
    return r;
  }
};

// 16 bytes at an address aligned to T only
template <typename T>
__device__ __forceinline__ u32x4 load_vec(const T* p) {
  using At = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
  return *reinterpret_cast<const At*>(p);
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const u32x4& v) {
  using At = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
  *reinterpret_cast<At*>(p) = v;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

__device__ __forceinline__ int wave_sum_i(int x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// Token i of an int32 or int64 array.
__device__ __forceinline__ int64_t token_at(const void* tok, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(tok)[i] : (int64_t) static_cast<const int32_t*>(tok)[i];
}

// Types of a dense operand, as the Python side numbers them.
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

#define SPMM_VOCAB_TYPE(code, NAME, ...)                 \
  switch (code) {                                        \
    case spmm::kF32: { using NAME = float; __VA_ARGS__; break; }    \
    case spmm::kBF16: { using NAME = __bf16; __VA_ARGS__; break; }  \
    case spmm::kF16: { using NAME = _Float16; __VA_ARGS__; break; } \
    default: return (int)hipErrorInvalidValue;           \
  }

// Workgroups of a launch: tasks beyond this run in the same workgroups' loops
// (a grid holds at most 2^32 threads).
constexpr int64_t kMaxGroups = 1 << 21;
inline unsigned groups_of(int64_t tasks) { return (unsigned)(tasks < kMaxGroups ? tasks : kMaxGroups); }

}  // namespace spmm
