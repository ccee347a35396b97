// Element types of the calls that take fp32, bf16 and fp16 tensors: 16-byte accesses and conversions to and from fp32.
#pragma once
#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// a row or a tensor may begin at any element (an odd vocabulary, a view into a flat buffer): wide accesses at the
// alignment of the smallest type
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

// EV: elements of 16 bytes; at: element e of 16 bytes; one: element i of a tensor; cast: rounds to nearest even
template <int T> struct Elem;
template <> struct Elem<DVAE_F32> {
  typedef float type;
  static constexpr int EV = 4;
  static __device__ __forceinline__ float at(u32x4 r, int e) { return __uint_as_float(r[e]); }
  static __device__ __forceinline__ float one(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ float cast(float v) { return v; }
};
template <> struct Elem<DVAE_BF16> {
  typedef __bf16 type;
  static constexpr int EV = 8;
  static __device__ __forceinline__ float at(u32x4 r, int e) {
    const uint32_t w = r[e >> 1];
    return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float one(const void* p, long long i) {
    return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
  }
  static __device__ __forceinline__ __bf16 cast(float v) { return (__bf16)v; }
};
template <> struct Elem<DVAE_F16> {
  typedef _Float16 type;
  static constexpr int EV = 8;
  static __device__ __forceinline__ float at(u32x4 r, int e) {
    const uint16_t h = (uint16_t)((e & 1) ? (r[e >> 1] >> 16) : (r[e >> 1] & 0xffffu));
    return (float)__builtin_bit_cast(_Float16, h);
  }
  static __device__ __forceinline__ float one(const void* p, long long i) {
    return (float)static_cast<const _Float16*>(p)[i];
  }
  static __device__ __forceinline__ _Float16 cast(float v) { return (_Float16)v; }
};

static inline int elem_bytes(int dtype) { return dtype == DVAE_F32 ? 4 : 2; }
