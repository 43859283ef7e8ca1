// Element types of the sequence operators (ttsx_seq.h): 32-bit floats and the two 16-bit kinds, read and written 16
// bytes per lane.  Everything between a load and a store is fp32.
#pragma once
#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // rows of odd strides: global memory takes any element address
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct IoF32 {
  typedef float elem;
  static constexpr int VEC = 4;
  static constexpr uint32_t INF2 = 0x7f800000u;  // one register of +infinity
  __device__ static inline void unpack(u32x4 r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
  __device__ static inline u32x4 pack(const float* v) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    return r;
  }
};

struct IoBf16 {
  typedef __bf16 elem;
  static constexpr int VEC = 8;
  static constexpr uint32_t INF2 = 0x7f807f80u;
  __device__ static inline void unpack(u32x4 r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
  __device__ static inline u32x4 pack(const float* v) {  // to nearest, ties to even
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){v[2 * i], v[2 * i + 1]}, bf16x2));
    return r;
  }
};

struct IoF16 {
  typedef _Float16 elem;
  static constexpr int VEC = 8;
  static constexpr uint32_t INF2 = 0x7c007c00u;
  __device__ static inline void unpack(u32x4 r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[i];  // a value of its own: the cast of a vector's element takes the wrong one
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      v[2 * i] = (float)h[0];
      v[2 * i + 1] = (float)h[1];
    }
  }
  __device__ static inline u32x4 pack(const float* v) {  // to nearest, ties to even
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = v[2 * i], b = v[2 * i + 1];
      asm("" : "+v"(a), "+v"(b));  // the fp32 value is rounded, as everywhere: no fma straight into 16 bits
      const f16x2 h = {(_Float16)a, (_Float16)b};
      r[i] = __builtin_bit_cast(uint32_t, h);
    }
    return r;
  }
};

template <class IO>
__device__ static inline u32x4 load16(const typename IO::elem* p) {
  return *reinterpret_cast<const u32x4_any*>(p);
}
template <class IO>
__device__ static inline void store16(typename IO::elem* p, u32x4 r) {
  *reinterpret_cast<u32x4_any*>(p) = r;
}

// The first n (0..VEC) elements at p, the rest zero; a full vector is one load.
template <class IO>
__device__ static inline u32x4 load_some(const typename IO::elem* p, int n) {
  if (n >= IO::VEC) return load16<IO>(p);
  float v[IO::VEC];
#pragma unroll
  for (int i = 0; i < IO::VEC; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
  return IO::pack(v);
}
template <class IO>
__device__ static inline void store_some(typename IO::elem* p, u32x4 r, int n) {
  if (n >= IO::VEC) {
    store16<IO>(p, r);
    return;
  }
  float v[IO::VEC];
  IO::unpack(r, v);
#pragma unroll
  for (int i = 0; i < IO::VEC; ++i)
    if (i < n) p[i] = (typename IO::elem)v[i];
}

// VEC consecutive fp32 values (states) of which n exist.
template <int VEC>
__device__ static inline void load_f32(const float* p, int n, float* v) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = i < n ? p[i] : 0.0f;
}
template <int VEC>
__device__ static inline void store_f32(float* p, int n, const float* v) {
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < n) p[i] = v[i];
}

// A row of a ragged batch is valid below this.
__device__ static inline int valid_rows(const int32_t* lengths, int b, int T) {
  return lengths ? min(max(lengths[b], 0), T) : T;
}
