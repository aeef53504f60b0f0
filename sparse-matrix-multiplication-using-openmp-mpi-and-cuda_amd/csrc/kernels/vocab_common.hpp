// Rows over a vocabulary: what embedding.hip and vocab_logits.hip share.
//
// Dense rows are fp32, bf16 or fp16, any row stride, any base alignment that
// the element type has: 16-byte loads and stores are typed with the element's
// own alignment, which gfx950 takes.  They cost a quarter of the bandwidth where
// they are not aligned: long rows start at the next 16-byte boundary instead
// (vocab_logits.hip Row).
#pragma once
#include "common.hpp"

#include <type_traits>

namespace spmm {

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2), may_alias));   // 16 bytes at a 2- or 4-byte aligned address
typedef u32x4 u32x4_at4 __attribute__((aligned(4), may_alias));

constexpr float kInf = __builtin_inff();

// kN elements in a 16-byte vector; kNegInf: two (16-bit) or one negative
// infinity.  Max gathers the maximum of whole vectors and single elements; a
// row with a NaN may give any of its elements.
template <typename T>
struct Elem;

__device__ __forceinline__ float max3(float a, float b, float c);

template <>
struct Elem<float> {
  static constexpr int kN = 4;
  static constexpr int kLowBits = 0;   // of an element as fp32 that are always zero
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float cast(float x) { return x; }
  struct Max {
    float m = -kInf;
    __device__ __forceinline__ void vec(const u32x4& v) {
      m = max3(m, __uint_as_float(v[0]), __uint_as_float(v[1]));
      m = max3(m, __uint_as_float(v[2]), __uint_as_float(v[3]));
    }
    __device__ __forceinline__ void one(float x) { m = fmaxf(m, x); }
    __device__ __forceinline__ float get() const { return m; }
  };
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
};

template <>
struct Elem<__bf16> {
  static constexpr int kN = 8;
  static constexpr int kLowBits = 16;   // of an element as fp32 that are always zero
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    const uint32_t w = v[i >> 1];
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float load(const __bf16* p) { return (float)*p; }
  static __device__ __forceinline__ __bf16 cast(float x) { return (__bf16)x; }   // round to nearest even
  struct Max {
    float m = -kInf;
    __device__ __forceinline__ void vec(const u32x4& v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max3(m, __uint_as_float(v[i] & 0xffff0000u), __uint_as_float(v[i] << 16));
    }
    __device__ __forceinline__ void one(float x) { m = fmaxf(m, x); }
    __device__ __forceinline__ float get() const { return m; }
  };
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
  static constexpr int kLowBits = 13;   // of an element as fp32 that are always zero
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ float get(const u32x4& v, int i) {
    const uint32_t w = v[i >> 1];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)((i & 1) ? (w >> 16) : w));
  }
  static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ _Float16 cast(float x) { return (_Float16)x; }
  struct Max {
    uint32_t m = kNegInf;   // two at a time
    float t = -kInf;
    __device__ __forceinline__ void vec(const u32x4& v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(m), "v"(v[i]));
    }
    __device__ __forceinline__ void one(float x) { t = fmaxf(t, x); }
    __device__ __forceinline__ float get() const {
      const float lo = (float)__builtin_bit_cast(_Float16, (uint16_t)m);
      return fmaxf(fmaxf(lo, (float)__builtin_bit_cast(_Float16, (uint16_t)(m >> 16))), t);
    }
  };
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

// The same past the caches' replacement order: for what is larger than the L2
// caches and not read again soon.
template <typename T>
__device__ __forceinline__ void stream_vec(T* p, const u32x4& v) {
  using At = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
  __builtin_nontemporal_store(v, reinterpret_cast<At*>(p));
}
template <typename T>
__device__ __forceinline__ u32x4 fetch_vec(const T* p) {
  using At = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
  return __builtin_nontemporal_load(reinterpret_cast<const At*>(p));
}
constexpr int64_t kStreamBytes = 16 << 20;   // outputs that are written so

// Reductions over a wave.  Lanes are paired inside rows of 16 by data-parallel
// primitives (no LDS), the four rows by lane reads: the result is uniform.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;   // quad_perm, row_half_mirror, row_mirror

// over groups of 2, 4, 8 or 16 neighbouring lanes (1: none)
template <typename F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x, int lanes, F&& f) {
  if (lanes > 1) x = f(x, dpp<kSwap1>(x));
  if (lanes > 2) x = f(x, dpp<kSwap2>(x));
  if (lanes > 4) x = f(x, dpp<kHalfMirror>(x));
  if (lanes > 8) x = f(x, dpp<kMirror>(x));
  return x;
}
template <typename F>
__device__ __forceinline__ uint32_t over_wave(uint32_t x, F&& f) {
  x = over_lanes(x, 16, f);
  const uint32_t r0 = __builtin_amdgcn_readlane(x, 0), r1 = __builtin_amdgcn_readlane(x, 16),
                 r2 = __builtin_amdgcn_readlane(x, 32), r3 = __builtin_amdgcn_readlane(x, 48);
  return f(f(r0, r1), f(r2, r3));
}
__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }

__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(over_wave(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float wave_sum(float x) {
  return __uint_as_float(over_wave(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// max(a, b, c) as one instruction, without the quieting of signalling NaNs that
// fmaxf asks for: such a NaN makes the result a NaN, which the next maximum
// passes over together with what came before it
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
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
