// Element types of the sequence operators (ttsx_seq.h): 32-bit floats and the two 16-bit kinds, read and written 16
// bytes per lane.  Everything between a load and a store is fp32.
#pragma once
#include <type_traits>

#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// PER: elements of a 32-bit word; INF: a word of +infinity; VEC: elements of 16 bytes.
struct IoF32 {
  typedef float elem;
  static constexpr int PER = 1, VEC = 4;
  static constexpr uint32_t INF = 0x7f800000u;
  __device__ static inline void unpack(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
  __device__ static inline uint32_t pack(const float* v) { return __float_as_uint(v[0]); }
};

struct IoBf16 {
  typedef __bf16 elem;
  static constexpr int PER = 2, VEC = 8;
  static constexpr uint32_t INF = 0x7f807f80u;
  __device__ static inline void unpack(uint32_t w, float* v) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  }
  __device__ static inline uint32_t pack(const float* v) {  // to nearest, ties to even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){v[0], v[1]}, bf16x2));
  }
};

struct IoF16 {
  typedef _Float16 elem;
  static constexpr int PER = 2, VEC = 8;
  static constexpr uint32_t INF = 0x7c007c00u;
  __device__ static inline void unpack(uint32_t w, float* v) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    v[0] = (float)h[0];
    v[1] = (float)h[1];
  }
  __device__ static inline uint32_t pack(const float* v) {  // to nearest, ties to even
    float a = v[0], b = v[1];
    asm("" : "+v"(a), "+v"(b));  // the fp32 value is rounded, as everywhere: no fma straight into 16 bits
    const f16x2 h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
  }
};

// N elements as a lane holds them (8 or 16 bytes).  Rows of odd strides: global memory takes any element address.
template <class IO, int N>
struct Lane {
  static constexpr int W = N / IO::PER;
  typedef uint32_t raw __attribute__((ext_vector_type(W)));
  typedef raw raw_any __attribute__((aligned(2)));
  typedef typename IO::elem E;
  __device__ static inline raw fill(uint32_t w) {
    raw r;
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = w;
    return r;
  }
  __device__ static inline void unpack(raw r, float* v) {
#pragma unroll
    for (int i = 0; i < W; ++i) IO::unpack(r[i], v + i * IO::PER);
  }
  __device__ static inline raw pack(const float* v) {
    raw r;
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = IO::pack(v + i * IO::PER);
    return r;
  }
  __device__ static inline raw load(const E* p) { return *reinterpret_cast<const raw_any*>(p); }
  __device__ static inline void store(E* p, raw r) { *reinterpret_cast<raw_any*>(p) = r; }
  // the first n (0..N) elements at p, the rest zero; a full vector is one load
  __device__ static inline raw load_some(const E* p, int n) {
    if (n >= N) return load(p);
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    return pack(v);
  }
  // Elements c..c+N-1 of a row of `width`, zero behind its end.  Nothing behind the row is read: the lane takes the last
  // N elements of the row (or fewer, one by one, of a row that has no N) and moves them down.
  __device__ static inline raw load_end(const E* row, int c, int width) {
    static_assert(W == 4, "16 bytes");
    const int n = min(max(width - c, 0), N);
    if (width < N) return load_some(row + min(c, width - 1), n);
    const int from = min(c, width - N), by = (c - from) * (4 / IO::PER);  // bytes
    raw r = load(row + from);
    if (by & 8) r = (raw){r[2], r[3], 0, 0};
    if (by & 4) r = (raw){r[1], r[2], r[3], 0};
    if (by & 2) r = (raw){r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    return n > 0 ? r : fill(0);
  }
  __device__ static inline void store_some(E* p, raw r, int n) {
    if (n >= N) {
      store(p, r);
      return;
    }
    float v[N];
    unpack(r, v);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (E)v[i];
  }
};

// One element per lane.
template <class IO>
struct Lane<IO, 1> {
  static constexpr int W = 1;
  typedef uint32_t raw;
  typedef typename IO::elem E;
  __device__ static inline raw fill(uint32_t w) { return w; }
  __device__ static inline void unpack(raw r, float* v) {
    float t[IO::PER];
    IO::unpack(r, t);
    v[0] = t[0];
  }
  __device__ static inline raw pack(const float* v) {
    float t[IO::PER] = {};
    t[0] = v[0];
    return IO::pack(t);
  }
  __device__ static inline raw load(const E* p) {
    if constexpr (IO::PER == 1)
      return *reinterpret_cast<const uint32_t*>(p);
    else
      return *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ static inline void store(E* p, raw r) {
    if constexpr (IO::PER == 1)
      *reinterpret_cast<uint32_t*>(p) = r;
    else
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)r;
  }
};

// N consecutive fp32 values (states).
template <int N>
__device__ static inline void load_f32(const float* p, float* v) {
  typedef float vec __attribute__((ext_vector_type(N == 1 ? 2 : N), aligned(4)));
  if constexpr (N == 1) {
    v[0] = *p;
  } else {
    const vec r = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = r[i];
  }
}
template <int N>
__device__ static inline void store_f32(float* p, const float* v) {
  typedef float vec __attribute__((ext_vector_type(N == 1 ? 2 : N), aligned(4)));
  if constexpr (N == 1) {
    *p = v[0];
  } else {
    vec r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = v[i];
    *reinterpret_cast<vec*>(p) = r;
  }
}
template <int N>
__device__ static inline void store_f32_some(float* p, int n, const float* v) {
  if (n >= N) {
    store_f32<N>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = v[i];
}

// The stride that a call goes by: a single row has no next one.
inline int64_t stride_of(int T, int64_t stride) { return T > 1 ? stride : 0; }

// The widest grid of workgroups of that many threads: a launch counts its threads in 32 bits.
constexpr int64_t most_workgroups(int threads) { return 0xffffffffLL / threads; }

// A launch and its own status: an error that an earlier call left behind is not this one's.  (hipGetLastError would report it
// although the kernel is queued, and a caller that took that for a refusal would update its state a second time.)
template <class... P>
inline int launch_kernel(const char* name, void (*kernel)(P...), int64_t grid, int threads, hipStream_t s,
                         typename std::common_type<P>::type... args) {
  void* p[] = {&args...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3(threads), p, 0, s);
  if (e == hipSuccess) return TTSX_OK;
  (void)hipGetLastError();  // reported here, and by nobody else
  ttsx_set_error("%s: launch -> %s", name, hipGetErrorString(e));
  return TTSX_ERR_HIP;
}

// A row of a ragged batch is valid below this.
__device__ static inline int valid_rows(const int32_t* lengths, int b, int T) {
  return lengths ? min(max(lengths[b], 0), T) : T;
}
