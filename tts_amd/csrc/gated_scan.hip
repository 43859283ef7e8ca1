// Gated linear recurrence (ttsx_gated_scan, ttsx_gated_scan_backward, ttsx_gated_step).
//
//   f_t = sigmoid(g_t), w_t = sigmoid(-g_t) = 1 - f_t
//   h_t = f_t h_{t-1} + w_t x_t
//
// A step is the map h -> f h + w x, and maps compose: (A2, B2) after (A1, B1) is (A2 A1, A2 B1 + B2), so the time axis
// is a prefix scan over pairs.  With G_t = dL/dh_t the gradients are
//   G_t = dh_t + f_{t+1} G_{t+1}   (the gradient of the last state enters behind the last step)
//   dx_t = w_t G_t,  dg_t = f_t w_t (h_{t-1} - x_t) G_t,  dh_0 = f_1 G_1
// and R -> f (dh + R), with R the product f G that a step hands to the one before it, composes in the same way.
//
// One pass over memory: a lane holds L consecutive steps of N channels in registers, a group of lanes covers 128 bytes
// of channels, the groups of a wave and the four waves of a workgroup are consecutive in time.  A lane folds its steps
// into one pair, the pairs are scanned by shuffles inside the wave and through LDS across the waves, and the lane then
// runs its steps from the state it starts with.  A workgroup walks the tiles of its time chunk with the state in
// registers.  Where the batch has too few channels to fill the chip the time axis is cut into chunks: a first launch
// folds every chunk into a pair, and the second combines the pairs in front of its chunk.
#include "../../include/ttsx_seq.h"
#include "seq_io.h"

namespace {

constexpr int WAVES = 4;
constexpr int BLOCK = TTSX_STATE_BLOCK;

struct ScanArgs {
  const void *x, *g, *dh;
  int64_t x_bs, g_bs, dh_bs;   // strides of the batch, in elements
  uint32_t x_ts, g_ts, dh_ts;  // strides of the rows, in bytes
  const float *h0, *dh_last, *states_in;
  const int32_t* lengths;
  int T, D, reverse, cols, chunks, per;  // per: tiles of a chunk
  void *h, *dx, *dg;                     // contiguous
  float *h_last, *states, *dh0;
  float* pairs;  // [B][chunks][2][D]
};

// How a workgroup covers a tile: N channels and L steps per lane, GROUP lanes across the channels.
template <class IO, int N_, int GROUP_, int L_>
struct Shape {
  typedef IO Type;
  typedef Lane<IO, N_> Io;
  typedef typename IO::elem E;
  static constexpr int N = N_, GROUP = GROUP_, L = L_, TGROUPS = WAVES * 64 / GROUP, TILE = TGROUPS * L;
  static_assert(TILE % BLOCK == 0 && BLOCK % L == 0, "a tile and some lane of it start at a kept state");
};

// log2(e) cut to 16 and 13 bits, and ln(2) times what was cut off.
constexpr float L2E_16 = 1.44268799f, L2E_16_REST = 4.88849537e-6f;
constexpr float L2E_13 = 1.44262695f, L2E_13_REST = 4.71948406e-5f;

// w = sigmoid(-g) = 1 / (1 + e^g) and f = sigmoid(g), each to a few units in its own last place wherever it is a normal number.
// Long memories live in w (an error d of f is one of d / w in the state), and what is left of a state behind a closed gate
// in f: below a half f is e^g w, since 1 - w has lost the digits that count (a third of f at g = -16, all of it from -17.4
// on); above it 1 - w adds half a unit.  e^g is exp2 of the rounded product with log2(e), with what was rounded away put
// back: for 16-bit logits the product with a log2(e) cut to 16 (bf16) or 13 bits (fp16) is exact and the rest of the
// constant is the correction, fp32 logits take it from a fused product.  -inf gives w = 1, +inf gives 0, a NaN stays one.
template <class IO>
__device__ static inline float gate(float g, float& f) {
  float w, e;
  if constexpr (IO::PER == 1) {
    const float c = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -126.0f), 88.0f);
    const float t = 1.44269502f * c;
    const float rest = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, c));  // c - t ln 2, ln 2 = 0.693147182 - 1.9e-9
    const float p = __builtin_amdgcn_exp2f(t);
    e = fmaf(p, rest, p);
    w = __builtin_amdgcn_rcpf(1.0f + e);
    w = g > 88.0f ? 0.0f : w;
  } else {
    constexpr bool B = IO::INF == IoBf16::INF;
    constexpr float C1 = B ? L2E_16 : L2E_13, C2 = B ? L2E_16_REST : L2E_13_REST;
    const float c = __builtin_elementwise_maximum(g, -126.0f);
    const float p = __builtin_amdgcn_exp2f(C1 * c);
    const float d = C2 * c;
    e = fmaf(p, B ? d : fmaf(0.5f * d, d, d), p);  // fp16: d is up to 4e-3 where w is no zero, its square counts
    w = __builtin_amdgcn_rcpf(1.0f + e);
  }
  f = e < 1.0f ? e * w : 1.0f - w;
  return w;
}

struct Place {
  int b, chunk, c, across, tg, wave, lane;  // c: first channel of the lane; wave: a scalar
  bool on;                                  // the lane has channels
};
template <class S>
__device__ static inline Place place(const ScanArgs& a) {
  Place q;
  const int id = blockIdx.x;
  q.chunk = id / a.cols % a.chunks;
  q.b = id / a.cols / a.chunks;
  q.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  q.lane = threadIdx.x & 63;
  q.across = q.lane & (S::GROUP - 1);
  q.tg = threadIdx.x / S::GROUP;
  q.c = (id % a.cols * S::GROUP + q.across) * S::N;
  q.on = q.c < a.D;
  return q;
}

// The rows of a tile that starts at step p0: step p is row p, or row len-1-p from right to left.  `base` is the lowest
// row, a scalar; a lane adds a 32-bit offset.  Lanes behind the end read the last row again; what they read becomes
// +infinity for g (the gate that keeps the state) and zero for the others.
template <class S>
struct Tile {
  int p0, count, reverse;
  int64_t base;
  __device__ inline Tile(int p0_, int len, int reverse_) : p0(p0_), reverse(reverse_) {
    count = min(len - p0, S::TILE);
    base = reverse ? len - p0 - count : p0;
  }
  __device__ inline uint32_t row(int tg, int i) const {
    const int k = min(tg * S::L + i, count - 1);
    return reverse ? count - 1 - k : k;
  }
  __device__ inline bool live(int tg, int i) const { return tg * S::L + i < count; }
};
template <class T>
__device__ static inline T* shifted(T* base, int64_t bytes, uint32_t lane) {
  typedef typename std::conditional<std::is_const<T>::value, const char, char>::type C;
  return reinterpret_cast<T*>(reinterpret_cast<C*>(base) + bytes + lane);
}
// A lane number the compiler takes for a new one: the rows that follow from it are computed again instead of being held
// from the loads to the stores, which the backward pass has no registers for.
__device__ static inline int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// Strides below 2^22 bytes and rows below 2^9: the product of two 24-bit numbers.
__device__ static inline uint32_t offset(uint32_t row, uint32_t stride, uint32_t c) { return __umul24(row, stride) + c; }

template <class S>
__device__ static inline void load_rows(typename S::Io::raw* r, const typename S::E* base, uint32_t stride, const Tile<S>& t,
                                        const Place& q) {
  const uint32_t c = (q.on ? q.c : 0) * sizeof(typename S::E);
  const int tg = anew(q.tg);
#pragma unroll
  for (int i = 0; i < S::L; ++i)
    r[i] = S::Io::load(shifted(base, t.base * stride, offset(t.row(tg, i), stride, c)));
}
template <class S>
__device__ static inline void blank_rows(typename S::Io::raw* r, uint32_t with, const Tile<S>& t, const Place& q) {
#pragma unroll
  for (int i = 0; i < S::L; ++i)
    if (!t.live(q.tg, i)) r[i] = S::Io::fill(with);
}
// To [T,D] contiguous; `out` begins at the tile's lowest row.
template <class S>
__device__ static inline void store_row(typename S::E* out, uint32_t pitch, const Tile<S>& t, const Place& q, int i,
                                        typename S::Io::raw r) {
  const int tg = anew(q.tg);
  if (t.live(tg, i) && q.on) S::Io::store(shifted(out, t.base * pitch, offset(t.row(tg, i), pitch, q.c * sizeof(typename S::E))), r);
}
// Zero in rows from..to-1 of the tile's span.
template <class S>
__device__ static inline void zero_rows(typename S::E* base, uint32_t pitch, int p0, int from, int to, const Place& q) {
  for (int p = max(p0, from) + q.tg; p < min(p0 + S::TILE, to); p += S::TGROUPS)
    if (q.on) S::Io::store(shifted(base, (int64_t)p * pitch, q.c * sizeof(typename S::E)), S::Io::fill(0));
}

// Inclusive scan of the pairs over the lane groups of a wave, forward in time.
template <class S>
__device__ static inline void wave_scan(float* A, float* B, int lane) {
#pragma unroll
  for (int off = S::GROUP; off < 64; off *= 2) {
    const bool on = lane >= off;
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      const float pa = __shfl_up(A[i], off, 64), pb = __shfl_up(B[i], off, 64);
      B[i] = on ? fmaf(A[i], pb, B[i]) : B[i];
      A[i] = on ? A[i] * pa : A[i];
    }
  }
}
// The same from the last group back: B folds towards the wave's first step.
template <class S>
__device__ static inline void wave_scan_back(float* A, float* B, int lane) {
#pragma unroll
  for (int off = S::GROUP; off < 64; off *= 2) {
    const bool on = lane + off < 64;
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      const float pa = __shfl_down(A[i], off, 64), pb = __shfl_down(B[i], off, 64);
      B[i] = on ? fmaf(A[i], pb, B[i]) : B[i];
      A[i] = on ? A[i] * pa : A[i];
    }
  }
}

// What a value was computed from is forgotten: later uses start from the value alone instead of keeping the parts, which
// the backward pass has no registers for.
__device__ static inline void forget(float& v) { asm("" : "+v"(v)); }
template <class S>
__device__ static inline void forget(typename S::Io::raw& r) {
  if constexpr (S::Io::W == 1) {
    asm("" : "+v"(r));
  } else {
#pragma unroll
    for (int i = 0; i < S::Io::W; ++i) {
      uint32_t w = r[i];
      asm("" : "+v"(w));
      r[i] = w;
    }
  }
}

// The totals of the waves: product, forward fold, backward fold.
template <class S>
struct Totals {
  float v[WAVES][3][S::GROUP][S::N];
};

// The pairs of `count` chunks, in order from chunk `first` on (step 1 or -1), applied to h: the lane groups take equal
// runs of them, so one round trip to memory serves them all.
template <class S>
__device__ static inline void apply_chunks(const float* pairs, int D, int first, int step, int count, const Place& q,
                                           Totals<S>& tot, float* h) {
  constexpr int N = S::N;
  const int each = ceil_div(count, S::TGROUPS), from = q.tg * each, to = min(from + each, count);
  float A[N], B[N];
#pragma unroll
  for (int j = 0; j < N; ++j) A[j] = 1.0f, B[j] = 0.0f;
  if (q.on)
    for (int k = from; k < to; ++k) {
      const float* pr = pairs + (int64_t)(first + step * k) * 2 * D + q.c;
      float ka[N], kb[N];
      load_f32<N>(pr, ka);
      load_f32<N>(pr + D, kb);
#pragma unroll
      for (int j = 0; j < N; ++j) B[j] = fmaf(ka[j], B[j], kb[j]), A[j] *= ka[j];
    }
  wave_scan<S>(A, B, q.lane);
  if (q.lane >= 64 - S::GROUP) {
#pragma unroll
    for (int j = 0; j < N; ++j) tot.v[q.wave][0][q.across][j] = A[j], tot.v[q.wave][1][q.across][j] = B[j];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WAVES; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = fmaf(tot.v[k][0][q.across][j], h[j], tot.v[k][1][q.across][j]);
}

// The pair of every chunk of a cut time axis: forwards the map of the state, BACK the map of R from the chunk's last step to
// its first.  A lane group takes one run of steps and folds them 8 at a time; nothing is exchanged until all are folded.  Bound by
// memory: the 131 MB of 1 x 32000 x 1024 bf16 in 33 us, 4.0 TB/s.
template <class S, bool BACK>
__global__ __launch_bounds__(WAVES * 64) void fold_kernel(ScanArgs a) {
  constexpr int N = S::N, U = 8;
  typedef typename S::E E;
  typedef typename S::Io Io;
  __shared__ Totals<S> tot;
  const Place q = place<S>(a);
  if (q.chunk == (BACK ? 0 : a.chunks - 1)) return;  // nothing starts behind it
  const int len = valid_rows(a.lengths, q.b, a.T);
  const int run = a.per * S::L, first = q.chunk * a.per * S::TILE + q.tg * run, last = min(first + run, len);
  const E* other = static_cast<const E*>(BACK ? a.dh : a.x) + q.b * (BACK ? a.dh_bs : a.x_bs) + (q.on ? q.c : 0);
  const E* gb = static_cast<const E*>(a.g) + q.b * a.g_bs + (q.on ? q.c : 0);
  const int64_t os = BACK ? a.dh_ts : a.x_ts, gs = a.g_ts;
  float A[N], B[N];
#pragma unroll
  for (int j = 0; j < N; ++j) A[j] = 1.0f, B[j] = 0.0f;
  const int steps = max(last - first, 0);
  for (int k0 = 0; k0 < steps; k0 += U) {
    typename Io::raw gr[U], vr[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = min(k0 + i, steps - 1), p = BACK ? last - 1 - k : first + k;
      const int64_t row = a.reverse ? len - 1 - p : p;
      gr[i] = Io::load(shifted(gb, row * gs, 0));
      vr[i] = Io::load(shifted(other, row * os, 0));
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float gv[N], v[N];
      Io::unpack(k0 + i < steps ? gr[i] : Io::fill(S::Type::INF), gv);
      Io::unpack(k0 + i < steps ? vr[i] : Io::fill(0), v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float f;
        const float w = gate<typename S::Type>(gv[j], f);
        A[j] *= f;
        B[j] = BACK ? f * (B[j] + v[j]) : fmaf(f, B[j], w * v[j]);
      }
    }
  }
  if constexpr (BACK)
    wave_scan_back<S>(A, B, q.lane);
  else
    wave_scan<S>(A, B, q.lane);
  if (BACK ? q.lane < S::GROUP : q.lane >= 64 - S::GROUP) {
#pragma unroll
    for (int j = 0; j < N; ++j) tot.v[q.wave][0][q.across][j] = A[j], tot.v[q.wave][1][q.across][j] = B[j];
  }
  __syncthreads();
  if (q.tg != 0 || !q.on) return;
#pragma unroll
  for (int j = 0; j < N; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
  for (int k = 0; k < WAVES; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float ta = tot.v[BACK ? WAVES - 1 - k : k][0][q.across][j];
      B[j] = fmaf(ta, B[j], tot.v[BACK ? WAVES - 1 - k : k][1][q.across][j]);
      A[j] *= ta;
    }
  float* pr = a.pairs + ((int64_t)q.b * a.chunks + q.chunk) * 2 * a.D + q.c;
  store_f32<N>(pr, A);
  store_f32<N>(pr + a.D, B);
}

// Forward pass.  Bound by memory: 64 x 800 x 512 fp32 with ragged ends (250 MB) in 57 us, 4.4 TB/s, where a copy of that size
// reaches 5.3; a short text is one chain of load, scan and store, 4.1 us.
template <class S, bool SAVE>
__global__ __launch_bounds__(WAVES * 64, 4) void scan_kernel(ScanArgs a) {
  constexpr int N = S::N, L = S::L;
  typedef typename S::E E;
  typedef typename S::Io Io;
  __shared__ Totals<S> tot[2];
  const Place q = place<S>(a);
  const int len = valid_rows(a.lengths, q.b, a.T), blocks = ceil_div(a.T, BLOCK);
  const E* xb = static_cast<const E*>(a.x) + q.b * a.x_bs;
  const E* gb = static_cast<const E*>(a.g) + q.b * a.g_bs;
  E* hb = static_cast<E*>(a.h) + (int64_t)q.b * a.T * a.D;
  const uint32_t pitch = a.D * sizeof(E);

  float carry[N];  // state in front of the tile
#pragma unroll
  for (int j = 0; j < N; ++j) carry[j] = 0.0f;
  if (a.h0 && q.on) load_f32<N>(a.h0 + (int64_t)q.b * a.D + q.c, carry);
  if (q.chunk > 0) apply_chunks<S>(a.pairs + (int64_t)q.b * a.chunks * 2 * a.D, a.D, 0, 1, q.chunk, q, tot[1], carry);

  const int first = q.chunk * a.per * S::TILE, last = min(first + a.per * S::TILE, a.T);
  int half = 1;  // of `tot`; the first tile that has rows takes the one that apply_chunks left alone
  for (int p0 = first; p0 < last; p0 += S::TILE) {
    const int p = p0 + q.tg * L;
    const bool keeps = SAVE && p % BLOCK == 0 && p < a.T && q.on;
    float* kept = SAVE ? a.states + ((int64_t)q.b * blocks + p / BLOCK) * a.D + q.c : nullptr;
    if (p0 >= len) {  // behind the end: zero rows, the state stays
      zero_rows<S>(hb, pitch, p0, len, a.T, q);
      if (keeps) store_f32<N>(kept, carry);
      continue;
    }
    half ^= 1;
    const Tile<S> t(p0, len, a.reverse);
    typename Io::raw xr[L], gr[L];
    load_rows<S>(gr, gb, a.g_ts, t, q);
    load_rows<S>(xr, xb, a.x_ts, t, q);
    if (t.count < S::TILE) {  // the same for the workgroup
      blank_rows<S>(gr, S::Type::INF, t, q);
      blank_rows<S>(xr, 0, t, q);
      zero_rows<S>(hb, pitch, p0, len, a.T, q);
    }
    float f[L][N], v[L][N], A[N], B[N];
#pragma unroll
    for (int j = 0; j < N; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float gv[N], xv[N];
      Io::unpack(gr[i], gv);
      Io::unpack(xr[i], xv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float w = gate<typename S::Type>(gv[j], f[i][j]);
        v[i][j] = w * xv[j];
        A[j] *= f[i][j];
        B[j] = fmaf(f[i][j], B[j], v[i][j]);
      }
    }
    wave_scan<S>(A, B, q.lane);
    if (q.lane >= 64 - S::GROUP) {
#pragma unroll
      for (int j = 0; j < N; ++j) tot[half].v[q.wave][0][q.across][j] = A[j], tot[half].v[q.wave][1][q.across][j] = B[j];
    }
    __syncthreads();  // the other half of `tot` is written next: one barrier per tile
    float h[N];       // state in front of the wave, then of the lane
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      if (k == q.wave) {
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = carry[j];
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float ta = tot[half].v[k][0][q.across][j];
        carry[j] = fmaf(ta, carry[j], tot[half].v[k][1][q.across][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float pa = __shfl_up(A[j], S::GROUP, 64), pb = __shfl_up(B[j], S::GROUP, 64);
      h[j] = q.lane >= S::GROUP ? fmaf(pa, h[j], pb) : h[j];
    }
    if (keeps) store_f32<N>(kept, h);
#pragma unroll
    for (int i = 0; i < L; ++i) {
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = fmaf(f[i][j], h[j], v[i][j]);
      store_row<S>(hb, pitch, t, q, i, Io::pack(h));
    }
  }
  if (q.tg == 0 && q.on && q.chunk == a.chunks - 1) store_f32<N>(a.h_last + (int64_t)q.b * a.D + q.c, carry);
}

// Backward pass.  Bound by memory, three streams read and two written: 64 x 800 x 1024 bf16 with ragged ends (430 MB) in 106 to
// 109 us, 4.0 TB/s; 64 x 800 x 512 fp32 (429 MB) 104.
template <class S>
__global__ __launch_bounds__(WAVES * 64, 2) void scan_backward_kernel(ScanArgs a) {
  constexpr int N = S::N, L = S::L;
  typedef typename S::E E;
  typedef typename S::Io Io;
  __shared__ Totals<S> tot[2];
  const Place q = place<S>(a);
  const int len = valid_rows(a.lengths, q.b, a.T), blocks = ceil_div(a.T, BLOCK);
  const E* xb = static_cast<const E*>(a.x) + q.b * a.x_bs;
  const E* gb = static_cast<const E*>(a.g) + q.b * a.g_bs;
  const E* db = static_cast<const E*>(a.dh) + q.b * a.dh_bs;
  E* dxb = static_cast<E*>(a.dx) + (int64_t)q.b * a.T * a.D;
  E* dgb = static_cast<E*>(a.dg) + (int64_t)q.b * a.T * a.D;
  const uint32_t pitch = a.D * sizeof(E);

  float carry[N];  // R behind the tile
#pragma unroll
  for (int j = 0; j < N; ++j) carry[j] = 0.0f;
  if (a.dh_last && q.on) load_f32<N>(a.dh_last + (int64_t)q.b * a.D + q.c, carry);
  if (q.chunk < a.chunks - 1)
    apply_chunks<S>(a.pairs + (int64_t)q.b * a.chunks * 2 * a.D, a.D, a.chunks - 1, -1, a.chunks - 1 - q.chunk, q, tot[1],
                    carry);

  const int first = q.chunk * a.per * S::TILE, last = min(first + a.per * S::TILE, a.T);
  int half = 1;  // as in scan_kernel; tiles behind the end come first here and have no barrier, so they leave it as it is
  for (int p0 = first + (ceil_div(last - first, S::TILE) - 1) * S::TILE; p0 >= first; p0 -= S::TILE) {
    if (p0 >= len) {
      zero_rows<S>(dxb, pitch, p0, len, a.T, q);
      zero_rows<S>(dgb, pitch, p0, len, a.T, q);
      continue;
    }
    half ^= 1;
    const Tile<S> t(p0, len, a.reverse);
    typename Io::raw xr[L], gr[L], dr[L];
    float h[N];  // state in front of the tile
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = 0.0f;
    load_rows<S>(gr, gb, a.g_ts, t, q);
    load_rows<S>(dr, db, a.dh_ts, t, q);
    load_rows<S>(xr, xb, a.x_ts, t, q);
    if (q.on) load_f32<N>(a.states_in + ((int64_t)q.b * blocks + p0 / BLOCK) * a.D + q.c, h);
    if (t.count < S::TILE) {  // the same for the workgroup
      blank_rows<S>(gr, S::Type::INF, t, q);
      blank_rows<S>(dr, 0, t, q);
      blank_rows<S>(xr, 0, t, q);
      zero_rows<S>(dxb, pitch, p0, len, a.T, q);
      zero_rows<S>(dgb, pitch, p0, len, a.T, q);
    }
    // A: product of f; B: the forward fold; C: the backward fold of f dh
    float f[L][N], w[L][N], A[N], A2[N], B[N], C[N];
#pragma unroll
    for (int j = 0; j < N; ++j) A[j] = 1.0f, B[j] = C[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float gv[N], xv[N];
      Io::unpack(gr[i], gv);
      Io::unpack(xr[i], xv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        w[i][j] = gate<typename S::Type>(gv[j], f[i][j]);
        forget(w[i][j]);
        forget(f[i][j]);
        A[j] *= f[i][j];
        B[j] = fmaf(f[i][j], B[j], w[i][j] * xv[j]);
      }
      forget<S>(xr[i]);
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      float dv[N];
      Io::unpack(dr[i], dv);
#pragma unroll
      for (int j = 0; j < N; ++j) C[j] = f[i][j] * (C[j] + dv[j]);
      forget<S>(dr[i]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) A2[j] = A[j];
    wave_scan_back<S>(A2, C, q.lane);
    wave_scan<S>(A, B, q.lane);
    if (q.lane < S::GROUP) {
#pragma unroll
      for (int j = 0; j < N; ++j) tot[half].v[q.wave][0][q.across][j] = A2[j], tot[half].v[q.wave][2][q.across][j] = C[j];
    }
    if (q.lane >= 64 - S::GROUP) {
#pragma unroll
      for (int j = 0; j < N; ++j) tot[half].v[q.wave][1][q.across][j] = B[j];
    }
    __syncthreads();
    float R[N];  // gradient behind the wave, then behind the lane
#pragma unroll 1
    for (int k = WAVES - 1; k >= 0; --k)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float ta = tot[half].v[k][0][q.across][j];
        if (k == q.wave) R[j] = carry[j];
        carry[j] = fmaf(ta, carry[j], tot[half].v[k][2][q.across][j]);
      }
#pragma unroll 1
    for (int k = 0; k < q.wave; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = fmaf(tot[half].v[k][0][q.across][j], h[j], tot[half].v[k][1][q.across][j]);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float pa = __shfl_up(A[j], S::GROUP, 64), pb = __shfl_up(B[j], S::GROUP, 64);
      h[j] = q.lane >= S::GROUP ? fmaf(pa, h[j], pb) : h[j];
      pa = __shfl_down(A2[j], S::GROUP, 64), pb = __shfl_down(C[j], S::GROUP, 64);
      R[j] = q.lane < 64 - S::GROUP ? fmaf(pa, R[j], pb) : R[j];
    }
    // the states of the lane's steps again; s: dg / G
    float s[L][N];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float xv[N];
      Io::unpack(xr[i], xv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        s[i][j] = f[i][j] * w[i][j] * (h[j] - xv[j]);
        h[j] = fmaf(f[i][j], h[j], w[i][j] * xv[j]);
      }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      float dv[N], gx[N], gg[N];
      Io::unpack(dr[i], dv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float G = dv[j] + R[j];
        gx[j] = w[i][j] * G;
        gg[j] = s[i][j] * G;
        R[j] = f[i][j] * G;
      }
      store_row<S>(dxb, pitch, t, q, i, Io::pack(gx));
      store_row<S>(dgb, pitch, t, q, i, Io::pack(gg));
    }
  }
  if (q.tg == 0 && q.on && q.chunk == 0) store_f32<N>(a.dh0 + (int64_t)q.b * a.D + q.c, carry);
}

// One step of every request: elementwise, shorter than its launch (256 x 2048 bf16 in 3.0 us).
template <class IO, int N>
__global__ __launch_bounds__(256) void step_kernel(const typename IO::elem* x, int64_t x_bs, const typename IO::elem* g,
                                                   int64_t g_bs, const float* h, int B, int D, typename IO::elem* y,
                                                   float* h_out) {
  typedef Lane<IO, N> Io;
  const int cols = D / N;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t b = id / cols;
  const int c = (int)(id % cols) * N;
  if (b >= B) return;
  float xv[N], gv[N], hv[N];
  Io::unpack(Io::load(x + b * x_bs + c), xv);
  Io::unpack(Io::load(g + b * g_bs + c), gv);
  load_f32<N>(h + b * D + c, hv);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float f;
    const float w = gate<IO>(gv[j], f);
    hv[j] = fmaf(f, hv[j], w * xv[j]);
  }
  Io::store(y + b * D + c, Io::pack(hv));
  store_f32<N>(h_out + b * D + c, hv);
}

// Lanes take 8 bytes of a row where D is a whole number of them, else one channel.  A tile costs its scans once, and few
// channels over many steps make that small: forwards 8 steps a lane (fp32: 16 are no faster, 60 against 58 us at 64 x 800 x 512;
// bf16: 4 take 142 us at 16 x 4000 x 1024 where 8 take 114, 35.8 and 33.3 at 48 x 800 x 512; 16-byte lanes neither), backwards
// 32 channel-steps (108 us at 64 x 800 x 1024 bf16; 16: 120, 16-byte lanes: 158).
template <class IO>
using WideFwd = Shape<IO, 2 * IO::PER, 16, 8>;
template <class IO>
using WideBwd = Shape<IO, 2 * IO::PER, 16, 16 / IO::PER>;
template <class IO>
using Narrow = Shape<IO, 1, 64, 16>;
template <class IO>
bool wide(int D) {
  return D % WideFwd<IO>::N == 0;
}

struct Plan {
  int cols, chunks, per;
};
// How the time axis is cut: enough workgroups to fill 256 CUs four times over, one tile at least to each.  It is not cut
// where that loses: from one workgroup per CU on, since the fold reads everything once more (requests of 800 x 512 fp32,
// us uncut / cut: 16 of them 21 / 25, 24 26 / 34, 32 33 / 46; below, 8 requests 17 / 16, 4 17 / 12; the backward pass 34 / 35,
// 41 / 47, 50 / 59; 27 / 20, 26 / 16), and up to three tiles forwards and two backwards, where the second launch costs more
// than the tiles in a row (300 x 512 fp32 7.1 / 8.4 us, 180 x 33 7.8 / 8.9; backwards 200 x 512 bf16 10.6 / 11.1, but its
// three tiles of 300 x 512 15.0 / 11.3).
constexpr int ENOUGH = 256, FULL = 1024;
template <class S>
Plan plan(int B, int T, int D, bool backward) {
  Plan p;
  const int tiles = ceil_div(T, S::TILE);
  p.cols = ceil_div(D, S::GROUP * S::N);
  const int64_t rows = (int64_t)B * p.cols;
  const int want = (int)(rows >= ENOUGH || tiles <= (backward ? 2 : 3) ? 1 : FULL / rows);
  p.per = ceil_div(tiles, want < tiles ? want : tiles);
  p.chunks = ceil_div(tiles, p.per);
  return p;
}
template <class S>
size_t pairs_bytes(int B, int T, int D, bool backward) {
  const Plan p = plan<S>(B, T, D, backward);
  return p.chunks == 1 ? 0 : sizeof(float) * 2 * (size_t)B * p.chunks * D;
}

template <class S, bool BACK>
int launch(ScanArgs a, int B, size_t ws_bytes, hipStream_t s) {
  const char* name = BACK ? "ttsx_gated_scan_backward" : "ttsx_gated_scan";
  const Plan p = plan<S>(B, a.T, a.D, BACK);
  a.cols = p.cols, a.chunks = p.chunks, a.per = p.per;
  TTSX_ARG(p.chunks == 1 || (a.pairs && ws_bytes >= pairs_bytes<S>(B, a.T, a.D, BACK)), "%s: workspace too small", name);
  const int64_t grid = (int64_t)B * p.cols * p.chunks;
  TTSX_ARG(grid <= most_workgroups(WAVES * 64), "%s: too many requests of so many channels", name);
  if (p.chunks > 1) {
    const int rc = launch_kernel(name, fold_kernel<S, BACK>, grid, WAVES * 64, s, a);
    if (rc != TTSX_OK) return rc;
  }
  if constexpr (BACK)
    return launch_kernel(name, scan_backward_kernel<S>, grid, WAVES * 64, s, a);
  else
    return launch_kernel(name, a.states ? scan_kernel<S, true> : scan_kernel<S, false>, grid, WAVES * 64, s, a);
}

// The offsets inside a tile fit 32 bits, and a stride in bytes the 24 of a short product.
bool stride_ok(int64_t s) { return s >= 0 && s <= TTSX_SEQ_MAX_WIDTH; }

template <class IO, bool BACK>
int run_scan(ScanArgs a, int64_t x_ts, int64_t g_ts, int64_t dh_ts, int B, size_t ws_bytes, hipStream_t s) {
  a.x_ts = (uint32_t)(x_ts * sizeof(typename IO::elem));
  a.g_ts = (uint32_t)(g_ts * sizeof(typename IO::elem));
  a.dh_ts = (uint32_t)(dh_ts * sizeof(typename IO::elem));
  if (!wide<IO>(a.D)) return launch<Narrow<IO>, BACK>(a, B, ws_bytes, s);
  return launch<typename std::conditional<BACK, WideBwd<IO>, WideFwd<IO>>::type, BACK>(a, B, ws_bytes, s);
}

template <class IO>
size_t workspace(int B, int T, int D, bool backward) {
  if (!wide<IO>(D)) return pairs_bytes<Narrow<IO>>(B, T, D, backward);
  return backward ? pairs_bytes<WideBwd<IO>>(B, T, D, true) : pairs_bytes<WideFwd<IO>>(B, T, D, false);
}

template <class IO, int N>
int launch_step(const void* x, int64_t x_bs, const void* g, int64_t g_bs, const float* h, int B, int D, void* y,
                float* h_out, hipStream_t s) {
  typedef typename IO::elem E;
  const int64_t grid = ((int64_t)B * (D / N) + 255) / 256;
  TTSX_ARG(grid <= most_workgroups(256), "ttsx_gated_step: too many requests of so many channels");
  return launch_kernel("ttsx_gated_step", step_kernel<IO, N>, grid, 256, s, static_cast<const E*>(x), x_bs,
                       static_cast<const E*>(g), g_bs, h, B, D, static_cast<E*>(y), h_out);
}
template <class IO>
int run_step(const void* x, int64_t x_bs, const void* g, int64_t g_bs, const float* h, int B, int D, void* y,
             float* h_out, hipStream_t s) {
  return D % 4 == 0 ? launch_step<IO, 4>(x, x_bs, g, g_bs, h, B, D, y, h_out, s)
                    : launch_step<IO, 1>(x, x_bs, g, g_bs, h, B, D, y, h_out, s);
}

bool shape_ok(int B, int T, int D) { return B >= 1 && T >= 1 && D >= 1 && T <= TTSX_SEQ_MAX_ROWS && D <= TTSX_SEQ_MAX_WIDTH; }
bool dtype_ok(int d) { return d == TTSX_F32 || d == TTSX_BF16 || d == TTSX_F16; }

}  // namespace

extern "C" long ttsx_gated_scan_workspace(int B, int T, int D, int dtype, int backward) {
  TTSX_ARG(shape_ok(B, T, D) && dtype_ok(dtype), "ttsx_gated_scan_workspace: bad shape or type");
  return (long)(dtype == TTSX_F32    ? workspace<IoF32>(B, T, D, backward != 0)
                : dtype == TTSX_BF16 ? workspace<IoBf16>(B, T, D, backward != 0)
                                     : workspace<IoF16>(B, T, D, backward != 0));
}

extern "C" int ttsx_gated_scan(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const void* g,
                               int64_t g_batch_stride, int64_t g_row_stride, const float* h0, const int32_t* lengths,
                               int B, int T, int D, int dtype, int reverse, void* h, float* h_last, float* states,
                               void* workspace, size_t workspace_bytes, void* stream) {
  TTSX_ARG(x && g && h && h_last, "ttsx_gated_scan: null argument");
  TTSX_ARG(shape_ok(B, T, D), "ttsx_gated_scan: bad shape B=%d T=%d D=%d", B, T, D);
  TTSX_ARG(dtype_ok(dtype), "ttsx_gated_scan: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  x_row_stride = stride_of(T, x_row_stride), g_row_stride = stride_of(T, g_row_stride);
  TTSX_ARG(stride_ok(x_row_stride) && stride_ok(g_row_stride), "ttsx_gated_scan: a row stride outside 0..%ld",
           (long)TTSX_SEQ_MAX_WIDTH);
  ScanArgs a{};
  a.x = x, a.x_bs = x_batch_stride;
  a.g = g, a.g_bs = g_batch_stride;
  a.h0 = h0, a.lengths = lengths, a.T = T, a.D = D, a.reverse = reverse != 0;
  a.h = h, a.h_last = h_last, a.states = states, a.pairs = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32    ? run_scan<IoF32, false>(a, x_row_stride, g_row_stride, 0, B, workspace_bytes, s)
         : dtype == TTSX_BF16 ? run_scan<IoBf16, false>(a, x_row_stride, g_row_stride, 0, B, workspace_bytes, s)
                              : run_scan<IoF16, false>(a, x_row_stride, g_row_stride, 0, B, workspace_bytes, s);
}

extern "C" int ttsx_gated_scan_backward(const void* dh, int64_t dh_batch_stride, int64_t dh_row_stride, const void* x,
                                        int64_t x_batch_stride, int64_t x_row_stride, const void* g,
                                        int64_t g_batch_stride, int64_t g_row_stride, const float* states,
                                        const float* dh_last, const int32_t* lengths, int B, int T, int D, int dtype,
                                        int reverse, void* dx, void* dg, float* dh0, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  TTSX_ARG(dh && x && g && states && dx && dg && dh0, "ttsx_gated_scan_backward: null argument");
  TTSX_ARG(shape_ok(B, T, D), "ttsx_gated_scan_backward: bad shape B=%d T=%d D=%d", B, T, D);
  TTSX_ARG(dtype_ok(dtype), "ttsx_gated_scan_backward: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  dh_row_stride = stride_of(T, dh_row_stride);
  x_row_stride = stride_of(T, x_row_stride), g_row_stride = stride_of(T, g_row_stride);
  TTSX_ARG(stride_ok(dh_row_stride) && stride_ok(x_row_stride) && stride_ok(g_row_stride),
           "ttsx_gated_scan_backward: a row stride outside 0..%ld", (long)TTSX_SEQ_MAX_WIDTH);
  ScanArgs a{};
  a.dh = dh, a.dh_bs = dh_batch_stride;
  a.x = x, a.x_bs = x_batch_stride;
  a.g = g, a.g_bs = g_batch_stride;
  a.states_in = states, a.dh_last = dh_last, a.lengths = lengths, a.T = T, a.D = D, a.reverse = reverse != 0;
  a.dx = dx, a.dg = dg, a.dh0 = dh0, a.pairs = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32    ? run_scan<IoF32, true>(a, x_row_stride, g_row_stride, dh_row_stride, B, workspace_bytes, s)
         : dtype == TTSX_BF16 ? run_scan<IoBf16, true>(a, x_row_stride, g_row_stride, dh_row_stride, B, workspace_bytes, s)
                              : run_scan<IoF16, true>(a, x_row_stride, g_row_stride, dh_row_stride, B, workspace_bytes, s);
}

extern "C" int ttsx_gated_step(const void* x, int64_t x_batch_stride, const void* g, int64_t g_batch_stride,
                               const float* h, int B, int D, int dtype, void* y, float* h_out, void* stream) {
  TTSX_ARG(x && g && h && y && h_out, "ttsx_gated_step: null argument");
  TTSX_ARG(shape_ok(B, 1, D), "ttsx_gated_step: bad shape B=%d D=%d", B, D);
  TTSX_ARG(dtype_ok(dtype), "ttsx_gated_step: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32    ? run_step<IoF32>(x, x_batch_stride, g, g_batch_stride, h, B, D, y, h_out, s)
         : dtype == TTSX_BF16 ? run_step<IoBf16>(x, x_batch_stride, g, g_batch_stride, h, B, D, y, h_out, s)
                              : run_step<IoF16>(x, x_batch_stride, g, g_batch_stride, h, B, D, y, h_out, s);
}
