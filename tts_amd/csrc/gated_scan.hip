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
// One pass over memory: a lane holds L consecutive steps of VEC channels (16 bytes a step) in registers, 8 lanes cover
// 128 bytes of channels, the wave's 8 lane groups and the workgroup's 4 waves are consecutive in time.  A lane folds
// its steps into one pair, the pairs are scanned by shuffles inside the wave and through LDS across the waves, and
// the lane then runs its steps from the state it starts with.  A workgroup walks the tiles of its time chunk with the
// state in registers.  Where the batch has too few channels to fill the chip the time axis is cut into chunks: a first
// launch folds every chunk into a pair, and the second combines the pairs in front of its chunk.
#include "../../include/ttsx_seq.h"
#include "seq_io.h"

namespace {

constexpr int GROUP = 8;           // lanes across the channels: 128 bytes
constexpr int WAVES = 4;
constexpr int TGROUPS = WAVES * 64 / GROUP;
constexpr int BLOCK = TTSX_STATE_BLOCK;

struct ScanArgs {
  const void *x, *g, *dh;
  int64_t x_bs, x_ts, g_bs, g_ts, dh_bs, dh_ts;  // strides of batch and time in elements
  const float *h0, *dh_last, *states_in;
  const int32_t* lengths;
  int T, D, reverse, cols, chunks, per;  // per: tiles of a chunk
  void *h, *dx, *dg;                     // contiguous
  float *h_last, *states, *dh0;
  float* pairs;  // [B][chunks][2][D]
};

// f = sigmoid(g), w = 1 - f, each to a few units in its own last place: w = e f with e = exp(-g) keeps its digits
// where f rounds to one.  Below -87 the exponential overflows: f = 0, w = 1 (f is below 2e-38 there).  Comparisons that
// a NaN fails leave it as it is.  fp32 logits carry g log2(e) in two parts; the 16-bit types' own steps are far larger.
template <class IO>
__device__ static inline void gate(float g, float& f, float& w) {
  constexpr float L2E = 1.44269502f, L2E_LO = 1.92596303e-8f;
  const bool low = g < -87.0f;
  if constexpr (IO::VEC == 4) {
    g = low ? -87.0f : g;
    g = g > 126.0f ? 126.0f : g;
    const float t = -L2E * g;
    const float lo = fmaf(-L2E, g, -t) - L2E_LO * g;
    const float p = __builtin_amdgcn_exp2f(t);
    const float e = fmaf(p, 0.693147182f * lo, p);
    f = __builtin_amdgcn_rcpf(1.0f + e);
    w = low ? 1.0f : e * f;
    f = low ? 0.0f : f;
  } else {
    const float e = __builtin_amdgcn_exp2f(-L2E * g);
    f = __builtin_amdgcn_rcpf(1.0f + e);
    w = low ? 1.0f : e * f;
  }
}

// Element row of processing step p.
__device__ static inline int row_of(int p, int len, int reverse) { return reverse ? len - 1 - p : p; }

struct Place {
  int b, chunk, col, lane8, tg, wave, lane;
};
__device__ static inline Place place(const ScanArgs& a) {
  Place q;
  const int id = blockIdx.x;
  q.col = id % a.cols;
  q.chunk = id / a.cols % a.chunks;
  q.b = id / a.cols / a.chunks;
  q.wave = threadIdx.x >> 6;
  q.lane = threadIdx.x & 63;
  q.lane8 = q.lane & (GROUP - 1);
  q.tg = threadIdx.x / GROUP;
  return q;
}

// Inclusive scan of the pairs over the 8 groups of a wave, forward in time; then the pair before each group.
template <int VEC>
__device__ static inline void wave_scan(float* A, float* B, int lane) {
#pragma unroll
  for (int off = GROUP; off < 64; off *= 2) {
    const bool on = lane >= off;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = __shfl_up(A[i], off, 64), pb = __shfl_up(B[i], off, 64);
      B[i] = on ? fmaf(A[i], pb, B[i]) : B[i];
      A[i] = on ? A[i] * pa : A[i];
    }
  }
}
// The same from the last group back: B folds towards the wave's first step.
template <int VEC>
__device__ static inline void wave_scan_back(float* A, float* B, int lane) {
#pragma unroll
  for (int off = GROUP; off < 64; off *= 2) {
    const bool on = lane + off < 64;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = __shfl_down(A[i], off, 64), pb = __shfl_down(B[i], off, 64);
      B[i] = on ? fmaf(A[i], pb, B[i]) : B[i];
      A[i] = on ? A[i] * pa : A[i];
    }
  }
}

// Forward pass.  FOLD: only the pair of a chunk (first launch of a cut time axis).
template <class IO, int L, bool FOLD, bool SAVE>
__global__ __launch_bounds__(WAVES * 64) void scan_kernel(ScanArgs a) {
  constexpr int VEC = IO::VEC, TILE = TGROUPS * L;
  typedef typename IO::elem E;
  __shared__ float tot[2][WAVES][2][GROUP][VEC];
  const Place q = place(a);
  if (FOLD && q.chunk == a.chunks - 1) return;  // nothing starts behind the last chunk
  const int c0 = (q.col * GROUP + q.lane8) * VEC;
  const int n = min(max(a.D - c0, 0), VEC);
  const int len = valid_rows(a.lengths, q.b, a.T);
  const E* xb = static_cast<const E*>(a.x) + q.b * a.x_bs + c0;
  const E* gb = static_cast<const E*>(a.g) + q.b * a.g_bs + c0;
  E* hb = static_cast<E*>(a.h) + (int64_t)q.b * a.T * a.D + c0;
  const int blocks = ceil_div(a.T, BLOCK);

  float carry[VEC], prod[VEC];  // state in front of the tile; FOLD: the pair so far
#pragma unroll
  for (int i = 0; i < VEC; ++i) carry[i] = 0.0f, prod[i] = 1.0f;
  if constexpr (!FOLD) {
    if (a.h0) load_f32<VEC>(a.h0 + (int64_t)q.b * a.D + c0, n, carry);
    const float* pr = a.pairs + (int64_t)q.b * a.chunks * 2 * a.D + c0;
    for (int k = 0; k < q.chunk; ++k, pr += 2 * (int64_t)a.D) {
      float A[VEC], B[VEC];
      load_f32<VEC>(pr, n, A);
      load_f32<VEC>(pr + a.D, n, B);
#pragma unroll
      for (int i = 0; i < VEC; ++i) carry[i] = fmaf(A[i], carry[i], B[i]);
    }
  }

  const int first = q.chunk * a.per * TILE, last = min(first + a.per * TILE, a.T);
  int flip = 0;
  for (int p0 = first; p0 < last; p0 += TILE, flip ^= 1) {
    const int p = p0 + q.tg * L;
    if (p0 >= len) {  // behind the end: zero rows, the state stays
      if constexpr (FOLD) break;
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (p + i < a.T && n > 0) store_some<IO>(hb + (int64_t)(p + i) * a.D, (u32x4){0, 0, 0, 0}, n);
      if (SAVE && p % BLOCK == 0 && p < a.T)
        store_f32<VEC>(a.states + ((int64_t)q.b * blocks + p / BLOCK) * a.D + c0, n, carry);
      continue;
    }
    u32x4 xr[L], gr[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      // a row behind the end keeps the state: f = 1, w x = 0
      gr[i] = (u32x4){IO::INF2, IO::INF2, IO::INF2, IO::INF2};
      xr[i] = (u32x4){0, 0, 0, 0};
      if (p + i < len && n > 0) {
        const int64_t t = row_of(p + i, len, a.reverse);
        gr[i] = load_some<IO>(gb + t * a.g_ts, n);
        xr[i] = load_some<IO>(xb + t * a.x_ts, n);
      }
    }
    float f[L][VEC], v[L][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.0f, B[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float gv[VEC], xv[VEC];
      IO::unpack(gr[i], gv);
      IO::unpack(xr[i], xv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float w;
        gate<IO>(gv[j], f[i][j], w);
        v[i][j] = w * xv[j];
        A[j] *= f[i][j];
        B[j] = fmaf(f[i][j], B[j], v[i][j]);
      }
    }
    wave_scan<VEC>(A, B, q.lane);
    if (q.lane >= 64 - GROUP) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) tot[flip][q.wave][0][q.lane8][j] = A[j], tot[flip][q.wave][1][q.lane8][j] = B[j];
    }
    __syncthreads();  // the other half of `tot` is written next: one barrier per tile
    if constexpr (FOLD) {
#pragma unroll
      for (int k = 0; k < WAVES; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float ta = tot[flip][k][0][q.lane8][j];
          carry[j] = fmaf(ta, carry[j], tot[flip][k][1][q.lane8][j]);
          prod[j] *= ta;
        }
    } else {
      float h[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s = carry[j], mine = s;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
          if (k == q.wave) mine = s;
          s = fmaf(tot[flip][k][0][q.lane8][j], s, tot[flip][k][1][q.lane8][j]);
        }
        carry[j] = s;
        const float pa = __shfl_up(A[j], GROUP, 64), pb = __shfl_up(B[j], GROUP, 64);
        h[j] = q.lane >= GROUP ? fmaf(pa, mine, pb) : mine;
      }
      if (SAVE && p % BLOCK == 0 && p < a.T)
        store_f32<VEC>(a.states + ((int64_t)q.b * blocks + p / BLOCK) * a.D + c0, n, h);
#pragma unroll
      for (int i = 0; i < L; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] = fmaf(f[i][j], h[j], v[i][j]);
        if (p + i < a.T && n > 0) {
          const bool live = p + i < len;
          const int64_t t = live ? row_of(p + i, len, a.reverse) : p + i;
          store_some<IO>(hb + t * a.D, live ? IO::pack(h) : (u32x4){0, 0, 0, 0}, n);
        }
      }
    }
  }
  if constexpr (FOLD) {
    float* pr = a.pairs + ((int64_t)q.b * a.chunks + q.chunk) * 2 * a.D + c0;
    if (q.tg == 0) {
      store_f32<VEC>(pr, n, prod);
      store_f32<VEC>(pr + a.D, n, carry);
    }
  } else if (q.chunk == a.chunks - 1 && q.tg == 0) {
    store_f32<VEC>(a.h_last + (int64_t)q.b * a.D + c0, n, carry);
  }
}

// Backward pass.  FOLD: only the pair (product of f, folded f dh) of a chunk, from its last step to its first.
template <class IO, int L, bool FOLD>
__global__ __launch_bounds__(WAVES * 64) void scan_backward_kernel(ScanArgs a) {
  constexpr int VEC = IO::VEC, TILE = TGROUPS * L;
  static_assert(TILE % BLOCK == 0, "a tile starts at a kept state");
  typedef typename IO::elem E;
  __shared__ float tot[2][WAVES][3][GROUP][VEC];
  const Place q = place(a);
  if (FOLD && q.chunk == 0) return;  // nothing lies in front of the first chunk
  const int c0 = (q.col * GROUP + q.lane8) * VEC;
  const int n = min(max(a.D - c0, 0), VEC);
  const int len = valid_rows(a.lengths, q.b, a.T);
  const E* xb = static_cast<const E*>(a.x) + q.b * a.x_bs + c0;
  const E* gb = static_cast<const E*>(a.g) + q.b * a.g_bs + c0;
  const E* db = static_cast<const E*>(a.dh) + q.b * a.dh_bs + c0;
  E* dxb = static_cast<E*>(a.dx) + (int64_t)q.b * a.T * a.D + c0;
  E* dgb = static_cast<E*>(a.dg) + (int64_t)q.b * a.T * a.D + c0;
  const int blocks = ceil_div(a.T, BLOCK);

  float carry[VEC], prod[VEC];  // R behind the tile; FOLD: the pair so far
#pragma unroll
  for (int i = 0; i < VEC; ++i) carry[i] = 0.0f, prod[i] = 1.0f;
  if constexpr (!FOLD) {
    if (a.dh_last) load_f32<VEC>(a.dh_last + (int64_t)q.b * a.D + c0, n, carry);
    for (int k = a.chunks - 1; k > q.chunk; --k) {
      const float* pr = a.pairs + ((int64_t)q.b * a.chunks + k) * 2 * a.D + c0;
      float A[VEC], B[VEC];
      load_f32<VEC>(pr, n, A);
      load_f32<VEC>(pr + a.D, n, B);
#pragma unroll
      for (int i = 0; i < VEC; ++i) carry[i] = fmaf(A[i], carry[i], B[i]);
    }
  }

  const int first = q.chunk * a.per * TILE, last = min(first + a.per * TILE, a.T);
  int flip = 0;
  for (int p0 = first + (ceil_div(last - first, TILE) - 1) * TILE; p0 >= first; p0 -= TILE, flip ^= 1) {
    const int p = p0 + q.tg * L;
    if (p0 >= len) {
      if constexpr (!FOLD) {
#pragma unroll
        for (int i = 0; i < L; ++i)
          if (p + i < a.T && n > 0) {
            store_some<IO>(dxb + (int64_t)(p + i) * a.D, (u32x4){0, 0, 0, 0}, n);
            store_some<IO>(dgb + (int64_t)(p + i) * a.D, (u32x4){0, 0, 0, 0}, n);
          }
      }
      continue;
    }
    u32x4 xr[L], gr[L], dr[L];
    float start[VEC];
    if constexpr (!FOLD) load_f32<VEC>(a.states_in + ((int64_t)q.b * blocks + p0 / BLOCK) * a.D + c0, n, start);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      gr[i] = (u32x4){IO::INF2, IO::INF2, IO::INF2, IO::INF2};
      xr[i] = dr[i] = (u32x4){0, 0, 0, 0};
      if (p + i < len && n > 0) {
        const int64_t t = row_of(p + i, len, a.reverse);
        gr[i] = load_some<IO>(gb + t * a.g_ts, n);
        dr[i] = load_some<IO>(db + t * a.dh_ts, n);
        if constexpr (!FOLD) xr[i] = load_some<IO>(xb + t * a.x_ts, n);
      }
    }
    // A: product of f; B: the forward fold; C: the backward fold of f dh
    float f[L][VEC], w[L][VEC], A[VEC], A2[VEC], B[VEC], C[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[j] = C[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float gv[VEC], xv[VEC];
      IO::unpack(gr[i], gv);
      IO::unpack(xr[i], xv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        gate<IO>(gv[j], f[i][j], w[i][j]);
        A[j] *= f[i][j];
        if constexpr (!FOLD) B[j] = fmaf(f[i][j], B[j], w[i][j] * xv[j]);
      }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      float dv[VEC];
      IO::unpack(dr[i], dv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) C[j] = f[i][j] * (C[j] + dv[j]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) A2[j] = A[j];
    wave_scan_back<VEC>(A2, C, q.lane);
    if constexpr (!FOLD) wave_scan<VEC>(A, B, q.lane);
    if (q.lane < GROUP) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) tot[flip][q.wave][0][q.lane8][j] = A2[j], tot[flip][q.wave][2][q.lane8][j] = C[j];
    }
    if (!FOLD && q.lane >= 64 - GROUP) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) tot[flip][q.wave][1][q.lane8][j] = B[j];
    }
    __syncthreads();
    if constexpr (FOLD) {
#pragma unroll
      for (int k = WAVES - 1; k >= 0; --k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float ta = tot[flip][k][0][q.lane8][j];
          carry[j] = fmaf(ta, carry[j], tot[flip][k][2][q.lane8][j]);
          prod[j] *= ta;
        }
    } else {
      float h[VEC], R[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s = start[j], mine = s;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
          if (k == q.wave) mine = s;
          s = fmaf(tot[flip][k][0][q.lane8][j], s, tot[flip][k][1][q.lane8][j]);
        }
        float pa = __shfl_up(A[j], GROUP, 64), pb = __shfl_up(B[j], GROUP, 64);
        h[j] = q.lane >= GROUP ? fmaf(pa, mine, pb) : mine;
        s = carry[j];
#pragma unroll
        for (int k = WAVES - 1; k >= 0; --k) {
          if (k == q.wave) mine = s;
          s = fmaf(tot[flip][k][0][q.lane8][j], s, tot[flip][k][2][q.lane8][j]);
        }
        carry[j] = s;
        pa = __shfl_down(A2[j], GROUP, 64), pb = __shfl_down(C[j], GROUP, 64);
        R[j] = q.lane < 64 - GROUP ? fmaf(pa, mine, pb) : mine;
      }
      // the states of the lane's steps again; dg_t / G_t stays in s
      float s[L][VEC];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        float xv[VEC];
        IO::unpack(xr[i], xv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s[i][j] = f[i][j] * w[i][j] * (h[j] - xv[j]);
          h[j] = fmaf(f[i][j], h[j], w[i][j] * xv[j]);
        }
      }
#pragma unroll
      for (int i = L - 1; i >= 0; --i) {
        float dv[VEC], gx[VEC], gg[VEC];
        IO::unpack(dr[i], dv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float G = dv[j] + R[j];
          gx[j] = w[i][j] * G;
          gg[j] = s[i][j] * G;
          R[j] = f[i][j] * G;
        }
        if (p + i < a.T && n > 0) {
          const bool live = p + i < len;
          const int64_t t = live ? row_of(p + i, len, a.reverse) : p + i;
          store_some<IO>(dxb + t * a.D, live ? IO::pack(gx) : (u32x4){0, 0, 0, 0}, n);
          store_some<IO>(dgb + t * a.D, live ? IO::pack(gg) : (u32x4){0, 0, 0, 0}, n);
        }
      }
    }
  }
  if constexpr (FOLD) {
    float* pr = a.pairs + ((int64_t)q.b * a.chunks + q.chunk) * 2 * a.D + c0;
    if (q.tg == 0) {
      store_f32<VEC>(pr, n, prod);
      store_f32<VEC>(pr + a.D, n, carry);
    }
  } else if (q.chunk == 0 && q.tg == 0) {
    store_f32<VEC>(a.dh0 + (int64_t)q.b * a.D + c0, n, carry);
  }
}

// One step of every request: elementwise, a lane takes 16 bytes of x.
template <class IO>
__global__ __launch_bounds__(256) void step_kernel(const typename IO::elem* x, int64_t x_bs, const typename IO::elem* g,
                                                   int64_t g_bs, const float* h, int B, int D, typename IO::elem* y,
                                                   float* h_out) {
  constexpr int VEC = IO::VEC;
  const int cols = ceil_div(D, VEC);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)(id / cols), c = (int)(id % cols) * VEC;
  if (b >= B) return;
  const int n = min(D - c, VEC);
  float xv[VEC], gv[VEC], hv[VEC];
  IO::unpack(load_some<IO>(x + b * x_bs + c, n), xv);
  IO::unpack(load_some<IO>(g + b * g_bs + c, n), gv);
  load_f32<VEC>(h + (int64_t)b * D + c, n, hv);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float f, w;
    gate<IO>(gv[j], f, w);
    hv[j] = fmaf(f, hv[j], w * xv[j]);
  }
  store_some<IO>(y + (int64_t)b * D + c, IO::pack(hv), n);
  store_f32<VEC>(h_out + (int64_t)b * D + c, n, hv);
}

// Steps a lane holds: the forward pass keeps f and w x of each, the backward pass f, w, dg / G and the inputs.
template <class IO>
constexpr int FWD_L = 8;
template <class IO>
constexpr int BWD_L = IO::VEC == 4 ? 8 : 4;

struct Plan {
  int cols, chunks, per;
};
// How the time axis is cut: enough workgroups to fill 256 CUs three times over, one tile at least to each.
Plan plan(int B, int T, int D, int vec, int L) {
  Plan p;
  const int tiles = ceil_div(T, TGROUPS * L);
  p.cols = ceil_div(D, GROUP * vec);
  const int64_t rows = (int64_t)B * p.cols;
  const int want = (int)(rows >= 768 ? 1 : 768 / rows);
  p.per = ceil_div(tiles, want < tiles ? want : tiles);
  p.chunks = ceil_div(tiles, p.per);
  return p;
}

template <class IO>
int run_scan(ScanArgs a, int B, size_t ws_bytes, hipStream_t s) {
  const Plan p = plan(B, a.T, a.D, IO::VEC, FWD_L<IO>);
  a.cols = p.cols, a.chunks = p.chunks, a.per = p.per;
  TTSX_ARG(p.chunks == 1 || (a.pairs && ws_bytes >= sizeof(float) * 2 * B * p.chunks * a.D),
           "ttsx_gated_scan: workspace too small");
  const int64_t grid = (int64_t)B * p.cols * p.chunks;
  TTSX_ARG(grid <= 0x7fffffff, "ttsx_gated_scan: too many channels");
  if (p.chunks > 1) {
    scan_kernel<IO, FWD_L<IO>, true, false><<<(unsigned)grid, WAVES * 64, 0, s>>>(a);
    TTSX_LAUNCH_CHECK();
  }
  if (a.states)
    scan_kernel<IO, FWD_L<IO>, false, true><<<(unsigned)grid, WAVES * 64, 0, s>>>(a);
  else
    scan_kernel<IO, FWD_L<IO>, false, false><<<(unsigned)grid, WAVES * 64, 0, s>>>(a);
  TTSX_LAUNCH_CHECK();
  return TTSX_OK;
}

template <class IO>
int run_backward(ScanArgs a, int B, size_t ws_bytes, hipStream_t s) {
  const Plan p = plan(B, a.T, a.D, IO::VEC, BWD_L<IO>);
  a.cols = p.cols, a.chunks = p.chunks, a.per = p.per;
  TTSX_ARG(p.chunks == 1 || (a.pairs && ws_bytes >= sizeof(float) * 2 * B * p.chunks * a.D),
           "ttsx_gated_scan_backward: workspace too small");
  const int64_t grid = (int64_t)B * p.cols * p.chunks;
  TTSX_ARG(grid <= 0x7fffffff, "ttsx_gated_scan_backward: too many channels");
  if (p.chunks > 1) {
    scan_backward_kernel<IO, BWD_L<IO>, true><<<(unsigned)grid, WAVES * 64, 0, s>>>(a);
    TTSX_LAUNCH_CHECK();
  }
  scan_backward_kernel<IO, BWD_L<IO>, false><<<(unsigned)grid, WAVES * 64, 0, s>>>(a);
  TTSX_LAUNCH_CHECK();
  return TTSX_OK;
}

template <class IO>
int run_step(const void* x, int64_t x_bs, const void* g, int64_t g_bs, const float* h, int B, int D, void* y,
             float* h_out, hipStream_t s) {
  typedef typename IO::elem E;
  const int64_t grid = ((int64_t)B * ceil_div(D, IO::VEC) + 255) / 256;
  TTSX_ARG(grid <= 0x7fffffff, "ttsx_gated_step: too many channels");
  step_kernel<IO><<<(unsigned)grid, 256, 0, s>>>(static_cast<const E*>(x), x_bs, static_cast<const E*>(g), g_bs, h, B, D,
                                                 static_cast<E*>(y), h_out);
  TTSX_LAUNCH_CHECK();
  return TTSX_OK;
}

bool shape_ok(int B, int T, int D) { return B >= 1 && T >= 1 && D >= 1 && T <= (1 << 30) && D <= (1 << 24); }
bool dtype_ok(int d) { return d == TTSX_F32 || d == TTSX_BF16 || d == TTSX_F16; }

size_t pairs_bytes(int B, int T, int D, int dtype, int lf, int lh) {
  const bool wide = dtype == TTSX_F32;
  const Plan p = plan(B, T, D, wide ? 4 : 8, wide ? lf : lh);
  return p.chunks == 1 ? 0 : sizeof(float) * 2 * (size_t)B * p.chunks * D;
}

}  // namespace

extern "C" long ttsx_gated_scan_workspace(int B, int T, int D, int dtype, int backward) {
  TTSX_ARG(shape_ok(B, T, D) && dtype_ok(dtype), "ttsx_gated_scan_workspace: bad shape or type");
  return (long)(backward ? pairs_bytes(B, T, D, dtype, BWD_L<IoF32>, BWD_L<IoBf16>)
                         : pairs_bytes(B, T, D, dtype, FWD_L<IoF32>, FWD_L<IoBf16>));
}

extern "C" int ttsx_gated_scan(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const void* g,
                               int64_t g_batch_stride, int64_t g_row_stride, const float* h0, const int32_t* lengths,
                               int B, int T, int D, int dtype, int reverse, void* h, float* h_last, float* states,
                               void* workspace, size_t workspace_bytes, void* stream) {
  TTSX_ARG(x && g && h && h_last, "ttsx_gated_scan: null argument");
  TTSX_ARG(shape_ok(B, T, D), "ttsx_gated_scan: bad shape B=%d T=%d D=%d", B, T, D);
  TTSX_ARG(dtype_ok(dtype), "ttsx_gated_scan: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  ScanArgs a{};
  a.x = x, a.x_bs = x_batch_stride, a.x_ts = x_row_stride;
  a.g = g, a.g_bs = g_batch_stride, a.g_ts = g_row_stride;
  a.h0 = h0, a.lengths = lengths, a.T = T, a.D = D, a.reverse = reverse != 0;
  a.h = h, a.h_last = h_last, a.states = states, a.pairs = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32    ? run_scan<IoF32>(a, B, workspace_bytes, s)
         : dtype == TTSX_BF16 ? run_scan<IoBf16>(a, B, workspace_bytes, s)
                              : run_scan<IoF16>(a, B, workspace_bytes, s);
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
  ScanArgs a{};
  a.dh = dh, a.dh_bs = dh_batch_stride, a.dh_ts = dh_row_stride;
  a.x = x, a.x_bs = x_batch_stride, a.x_ts = x_row_stride;
  a.g = g, a.g_bs = g_batch_stride, a.g_ts = g_row_stride;
  a.states_in = states, a.dh_last = dh_last, a.lengths = lengths, a.T = T, a.D = D, a.reverse = reverse != 0;
  a.dx = dx, a.dg = dg, a.dh0 = dh0, a.pairs = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32    ? run_backward<IoF32>(a, B, workspace_bytes, s)
         : dtype == TTSX_BF16 ? run_backward<IoBf16>(a, B, workspace_bytes, s)
                              : run_backward<IoF16>(a, B, workspace_bytes, s);
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
