// Low-rank adapters of many voices beside a shared projection (ttsx_adapter_add, ttsx_adapter_backward).
//
//   out[b,t,:] = y[b,t,:] + s_v (x[b,t,:] A_v^T) B_v,   v = voices[b],   A_v = down[v] [R,K], B_v = up[v] [R,N]
//
//   du = s_v dy B_v^T;  dx = du A_v;  dA_v = sum of du^T x,  dB_v = sum of s_v (x A_v^T)^T dy over the rows of a voice
//
// A and B both have their long axis contiguous, so "contract the long axis" and "expand from R" are one kernel each way:
// dx is the same call as the forward pass with dy in the place of x and the two matrices swapped.
//
// One launch does both products of a tile of 32 (or 16) rows of one request: the four waves share the long axis of the first
// (each streams x and A from memory straight into matrix operands), the partial sums meet in LDS, and then the waves
// take blocks of 16 VEC output columns each, read B once per block, and add to y as they write.  u = x A^T never
// leaves the chip, and y is read and written once: the launch is bound by x, y and out.
//
// 16-bit types: the first product is exact up to its fp32 sums.  u is fp32 and is handed on as a sum of 16-bit numbers that
// holds all of it: three of bf16's 8 bits, or two of fp16's 11 (24 bits leave a remainder below 2^12 units behind the first,
// which the second holds to one unit: a rounding of u to 2^-23).  fp16 has no range for that, so its rows of u are scaled by a
// power of two first.
// Where a column block's lanes read 16 bytes of B from 8 ranks, the 8 x 8 block is transposed in registers; lane
// l & 15 then owns VEC neighbouring columns, so y and out move 16 bytes per lane.
#include "../../include/ttsx_seq.h"
#include "seq_io.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class IO>
using Full = Lane<IO, IO::VEC>;  // 16 bytes of a lane

constexpr int ROWS = 32;  // rows of a tile of kept hidden values; the first kernel takes them in one piece or in halves

// A first product: x [.,K] of a request's rows with the voice's matrix m [R,K].
struct Product {
  const void *x, *m;
  int64_t bs;  // stride of the batch in elements
  uint32_t ts;  // of the rows, in bytes
  int K;
  float* keep;  // [B][tiles][RP][ROWS]: s u for the weights' gradients (keep_hidden)
};
struct AddArgs {
  Product first, second;  // the second one is only kept
  const void *y, *up;
  void* out;
  int64_t y_bs, o_bs;
  uint32_t y_ts, o_ts;
  const int32_t *voices, *lengths;
  const float* scale;
  int T, N, R, V, tiles, splits, in_place;
};

template <class IO>
__device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (IO::VEC == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  } else if constexpr (IO::INF == IoBf16::INF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// 8 x 8 of 16-bit elements: r[i] holds row i, t[j] is column j.
__device__ static inline void transpose8(const u32x4* r, u32x4* t) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const uint32_t a = r[2 * m][c], b = r[2 * m + 1][c];
      t[2 * c][m] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      t[2 * c + 1][m] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
}

// Two fp32 values as sums of numbers of the 16-bit type, a word of pairs each, the largest first.
template <class IO>
constexpr int PARTS = IO::INF == IoBf16::INF ? 3 : 2;
template <class IO>
__device__ static inline void parts_of(float v0, float v1, uint32_t* p) {
  float v[2] = {v0, v1}, h[2];
#pragma unroll
  for (int k = 0; k < PARTS<IO>; ++k) {
    p[k] = IO::pack(v);
    IO::unpack(p[k], h);
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] -= h[i];
  }
}
// A sum over parts is no number where a factor is infinite: the other parts of u may be zero or of the other sign, those of an
// infinite u are none.  The first parts alone give the infinity (or NaN) of the sum (a multiple of it does too); where they
// give a number the sum stands.  `unsure`: whether the wave has such a sum.
template <int N>
__device__ static inline bool unsure(const f32x4* z) {
  float t = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) t = fmaf(z[j][i], 0.0f, t);
  return __any(t != 0.0f);
}
__device__ static inline void settle(f32x4& z, f32x4 first) {
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = fabsf(z[i]) < INFINITY || fabsf(first[i]) < INFINITY ? z[i] : first[i];
}

__device__ static inline int voice_of(const int32_t* voices, int b, int V) {
  const int v = voices[b];
  return v >= 0 && v < V ? v : -1;
}

// Zero in the place of infinities and NaN.
__device__ static inline u32x4 finite_bf16(u32x4 r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = r[i];
    w = (w & 0x7f80u) == 0x7f80u ? w & 0xffff0000u : w;
    r[i] = (w & 0x7f800000u) == 0x7f800000u ? w & 0xffffu : w;
  }
  return r;
}

// u of a tile, as the matrix operand of the second product: [H][RP] fp32, or its parts in 16-bit planes and a factor per row.
template <class IO, int RP, int H>
struct alignas(16) Hidden {
  typename IO::elem part[PARTS<IO>][H][RP + 8];
  float factor[H];
};
template <int RP, int H>
struct Hidden<IoF32, RP, H> {
  float u[H][RP + 4];
};

// Rank of a lane's i-th row of B: 16-bit types take 8 ranks at a time (up to rank 16 the upper half of the lanes has
// them again, for the second part of u), fp32 a quarter of them.
template <class IO, int RP>
__device__ static inline int rank_of(int q, int i) {
  if (IO::VEC == 4) return q * (RP / 4) + i;
  return RP == 16 ? 8 * (q & 1) + i : i / 8 * 32 + 8 * q + i % 8;
}

// u for the weights' gradients, where it is contracted over rows: per tile of 32 rows and 16 ranks two times 1 KB of fp32 in the
// order of the matrix operand, lane 16 q + rank with rows 8 q .. 8 q + 7, the first four in the first KB.
template <int RP>
__device__ static inline void keep_hidden(float* keep, int64_t tile, int row, int c0, const float* u) {
#pragma unroll
  for (int c = 0; c < RP / 8; ++c) {
    const int rank = c0 + c, lane = 16 * (row >> 3) + (rank & 15);
    float* at = keep + (tile * (RP / 16) + (rank >> 4)) * 512;
    at[(row >> 2 & 1) * 256 + lane * 4 + (row & 3)] = u[c];
  }
}
// Rows 16 .. 31 of a tile whose request ends in front of them: zero.
template <int RP>
__device__ static inline void keep_no_upper(float* keep, int64_t tile, int thread, int threads) {
  for (int i = thread; i < RP * 16; i += threads) keep[tile * RP * 32 + i / 128 * 256 + 128 + i % 128] = 0.0f;
}
template <int RP>
__device__ static inline void hidden_rows(const float* keep, int64_t tile, int j, int lane, u32x4* r) {
  const u32x4* at = reinterpret_cast<const u32x4*>(keep + (tile * (RP / 16) + j) * 512) + lane;
  r[0] = at[0];
  r[1] = at[64];
}

// A scalar base and a lane's offset in bytes.
template <class T>
__device__ static inline T* shifted(T* base, uint32_t bytes) {
  typedef typename std::conditional<std::is_const<T>::value, const char, char>::type C;
  return reinterpret_cast<T*>(reinterpret_cast<C*>(base) + bytes);
}

// A lane number the compiler takes for a new one: what follows from it is computed again instead of being held in
// registers around a loop, which the operands need.
__device__ static inline int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

template <class T>
__device__ static inline T* row_at(T* base, int64_t row, uint32_t stride) {
  typedef typename std::conditional<std::is_const<T>::value, const char, char>::type C;
  return reinterpret_cast<T*>(reinterpret_cast<C*>(base) + row * stride);
}

// Four registers of four neighbouring lanes, transposed: register j of lane i becomes register i of lane j.
__device__ static inline void quad_transpose(u32x4* r, int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t v[4] = {r[0][w], r[1][w], r[2][w], r[3][w]};
#pragma unroll
    for (int j = 0; j < 4; j += 2) {  // lanes 1 apart: quad_perm 1,0,3,2
      const uint32_t a = __builtin_amdgcn_mov_dpp(v[j], 0xb1, 0xf, 0xf, true);
      const uint32_t b = __builtin_amdgcn_mov_dpp(v[j + 1], 0xb1, 0xf, 0xf, true);
      v[j] = odd ? b : v[j];
      v[j + 1] = odd ? v[j + 1] : a;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // lanes 2 apart: quad_perm 2,3,0,1
      const uint32_t a = __builtin_amdgcn_mov_dpp(v[j], 0x4e, 0xf, 0xf, true);
      const uint32_t b = __builtin_amdgcn_mov_dpp(v[j + 2], 0x4e, 0xf, 0xf, true);
      v[j] = high ? b : v[j];
      v[j + 2] = high ? v[j + 2] : a;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j][w] = v[j];
  }
}

// The waves' shares of u = x A^T, 256 bytes of every row at a time.  A matrix operand wants 16 rows in 16 neighbouring
// lanes, which as a load is 64 separate accesses (the first form of this kernel was bound by them: 50 cache accesses to
// an instruction).  So four loads bring four rows each, 16 neighbouring lanes to a row, and the lanes' quads are
// transposed: lane 16 q + r then holds chunks 4 q .. 4 q + 3 of 16 bytes of row r, one per register, the same of x and of
// A.  Rows and ranks that do not exist repeat the last one and are dropped in the sum.
template <class IO, int RP, int WV, int MF>
__device__ static inline void first_product(const Product& p, const typename IO::elem* xb, int v, int R, int live, int wave,
                                            int lane, float (*part)[16 * MF][RP + 1]) {
  constexpr int VEC = IO::VEC, NJ = RP / 16, STEP = VEC * 16;
  typedef typename IO::elem E;
  typedef Full<IO> Io;
  const E* A = static_cast<const E*>(p.m) + (int64_t)v * R * p.K;
  f32x4 acc[MF][NJ];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[m][j] = (f32x4){0, 0, 0, 0};
  for (int k0 = wave * STEP; k0 < p.K; k0 += WV * STEP) {
    u32x4 xr[MF][4], ar[NJ][4];
    const uint32_t pitch = p.K * sizeof(E);
    const int l = anew(lane), row = l >> 2 & 3, k = ((l >> 4) * 4 + (l & 3)) * VEC;  // of load j: row 4 row + j
    if (k0 + STEP <= p.K) {  // the same for the wave
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xr[m][j] = Io::load(shifted(xb + k0, min(16 * m + 4 * row + j, live - 1) * p.ts + (uint32_t)(k * sizeof(E))));
#pragma unroll
      for (int n = 0; n < NJ; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ar[n][j] = Io::load(shifted(A + k0, min(16 * n + 4 * row + j, R - 1) * pitch + (uint32_t)(k * sizeof(E))));
    } else {
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xr[m][j] = Io::load_end(shifted(xb, min(16 * m + 4 * row + j, live - 1) * p.ts), k0 + k, p.K);
#pragma unroll
      for (int n = 0; n < NJ; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ar[n][j] = Io::load_end(shifted(A, min(16 * n + 4 * row + j, R - 1) * pitch), k0 + k, p.K);
    }
#pragma unroll
    for (int m = 0; m < MF; ++m) quad_transpose(xr[m], lane);
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      quad_transpose(ar[n], lane);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < MF; ++m) acc[m][n] = mma<IO>(xr[m][j], ar[n][j], acc[m][n]);
    }
  }
  const int q = lane >> 4, l16 = lane & 15;
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][16 * m + 4 * q + i][16 * j + l16] = acc[m][j][i];
}

// Ranks c0.. of row r of s u, from the waves' shares; zero where the row or the rank does not exist.
template <int RP, int WV, int H>
__device__ static inline void sum_shares(float (*part)[H][RP + 1], int r, int c0, int live, int R, float s, float* u) {
#pragma unroll
  for (int c = 0; c < RP / 8; ++c) {
    u[c] = 0.0f;
#pragma unroll
    for (int w = 0; w < WV; ++w) u[c] += part[w][r][c0 + c];
    u[c] = r < live && c0 + c < R ? u[c] * s : 0.0f;
  }
}

// ADD: out = y + z.  Else out = z, and the hidden rows of both products are kept.  Bound by memory where tiles are many: 64 x 800 x
// 256 -> 1025 rank 16 fp32 with ragged ends (452 MB) in 111 us, 4.1 TB/s (1024 columns, whose rows share no cache lines, 4.4;
// bf16 5.3);
// kept, 64 x 800 x (2048 -> 512) rank 32 bf16 in 57 us, 3.7 TB/s.  By its chain of dependent parts where they are few: 64 rows of
// 1024 -> 4096 in 6.8 us, 64 x 128 x 512 -> 2048 rank 32 bf16 (73 MB, a tile to a CU) in 16.7 us, 4.4 TB/s.
template <class IO, int RP, int WV, int MF, bool ADD>
__global__ __launch_bounds__(WV * 64, WV > 4 || RP == 64 ? 2 : 3) void adapter_kernel(AddArgs a) {
  constexpr int VEC = IO::VEC, CB = 16 * VEC, H = 16 * MF;  // H: rows of a tile
  constexpr bool WIDE = VEC == 4;
  typedef typename IO::elem E;
  typedef Full<IO> Io;
  __shared__ float part[ADD ? 1 : 2][WV][H][RP + 1];
  __shared__ Hidden<IO, RP, H> hid;
  const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits % a.tiles, b = blockIdx.x / a.splits / a.tiles;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, l16 = lane & 15;
  const int row0 = tile * H, rows = min(H, a.T - row0);
  const int len = valid_rows(a.lengths, b, a.T), v = voice_of(a.voices, b, a.V);
  const int live = min(rows, len - row0);  // rows of the tile that count (may be negative)
  const int64_t kept = (int64_t)b * ceil_div(a.T, ROWS) + row0 / ROWS;
  const E* yb = row_at(static_cast<const E*>(a.y) + b * a.y_bs, row0, a.y_ts);
  E* ob = row_at(static_cast<E*>(a.out) + b * a.o_bs, row0, a.o_ts);
  // A few columns behind the last whole block are no block of their own: the threads that add up u have their products as
  // well, and the waves are left with equal shares (64 x 800 x 256 -> 1025 bf16 64.9 -> 59.9 us, 1028 58.1 -> 51.1; fp32 with
  // ragged ends 117 -> 114).  More of them would take more registers than they save time.
  constexpr int REST = 64 / RP;
  const int rest = a.N > CB && a.N % CB <= REST ? a.N % CB : 0, blocks = ceil_div(a.N - rest, CB);

  if (v < 0 || live <= 0) {
    if (ADD && a.in_place) return;
    if (!ADD && v >= 0 && split == 0 && row0 % ROWS > 0 && len > row0 - H) {
      keep_no_upper<RP>(a.first.keep, kept, threadIdx.x, WV * 64);
      keep_no_upper<RP>(a.second.keep, kept, threadIdx.x, WV * 64);
    }
    // a row per wave, 64 lanes across
    for (int r = split * WV + wave; r < rows; r += a.splits * WV) {
      const E* from = shifted(yb, r * a.y_ts);
      E* to = shifted(ob, r * a.o_ts);
      constexpr int SPAN = 64 * VEC;
      int c = lane * VEC;
      for (; c + 3 * SPAN + VEC <= a.N; c += 4 * SPAN) {
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = ADD ? Io::load(from + c + i * SPAN) : Io::fill(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) Io::store(to + c + i * SPAN, w[i]);
      }
      for (; c + VEC <= a.N; c += SPAN) Io::store(to + c, ADD ? Io::load(from + c) : Io::fill(0));
      for (; c < a.N; ++c) to[c] = ADD ? from[c] : (E)0.0f;  // the one lane whose columns the row ends in
    }
    return;
  }

  // A piece is 16 rows of a column block.  The waves take neighbouring blocks at a time, since rows that are no multiple
  // of 128 bytes share a line at every border and the line should be whole when it leaves the L2; the blocks that are
  // left over are dealt out piece by piece.  A wave reads its next piece's y (and B, where registers allow) while it
  // multiplies, and its first piece's y before anything else.
  constexpr int KB = WIDE ? 1 : (RP + 31) / 32;  // blocks of 32 ranks
  constexpr int NB = WIDE ? RP / 4 : KB * 8;     // ranks of a lane
  constexpr bool AHEAD = WV == 4;
  const int pieces = ceil_div(rows, 16), lanes = a.splits * WV, me = split * WV + wave;
  const int rounds = blocks / lanes, left = blocks - rounds * lanes;
  const bool dealt = left * pieces <= lanes;
  const int all = rounds * pieces + (dealt ? (me < left * pieces ? 1 : 0) : me < left ? pieces : 0);
  const auto block_of = [&](int k) {
    return k < rounds * pieces ? k / pieces * lanes + me : rounds * lanes + (dealt ? me / pieces : me);
  };
  const auto piece_of = [&](int k) { return k >= rounds * pieces && dealt ? me % pieces : k % pieces; };
  const E* Bm = static_cast<const E*>(a.up) + (int64_t)v * a.R * a.N;
  const uint32_t b_pitch = a.N * sizeof(E);
  const auto fetch_b = [&](int cb, u32x4* br) {
    const int q = anew(lane >> 4), l16 = anew(lane & 15);
    if (cb * CB + CB <= a.N) {  // the same for the wave
#pragma unroll
      for (int i = 0; i < NB; ++i)
        br[i] = Io::load(shifted(Bm + cb * CB, min(rank_of<IO, RP>(q, i), a.R - 1) * b_pitch + (uint32_t)(l16 * 16)));
    } else {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        br[i] = Io::load_end(shifted(Bm, min(rank_of<IO, RP>(q, i), a.R - 1) * b_pitch), cb * CB + l16 * VEC, a.N);
    }
  };
  const auto fetch_y = [&](int cb, int m, u32x4* yr) {
    const int q = anew(lane >> 4), l16 = anew(lane & 15);
    if (cb * CB + CB <= a.N) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        yr[i] = Io::load(shifted(yb + cb * CB, min(16 * m + 4 * q + i, rows - 1) * a.y_ts + (uint32_t)(l16 * 16)));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        yr[i] = Io::load_end(shifted(yb, min(16 * m + 4 * q + i, rows - 1) * a.y_ts), cb * CB + l16 * VEC, a.N);
    }
  };
  u32x4 br[NB], bn[AHEAD ? NB : 1], yr[4], yn[4];
  if (ADD && all > 0) fetch_y(block_of(0), piece_of(0), yn);

  const float s = a.scale ? a.scale[v] : 1.0f;
  const int r = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * (RP / 8);  // of the sums: 8 threads to a row
  first_product<IO, RP, WV, MF>(a.first, row_at(static_cast<const E*>(a.first.x) + b * a.first.bs, row0, a.first.ts), v, a.R,
                            live, wave, lane, part[0]);
  if constexpr (!ADD) {
    // its 256 bytes go to the waves the first product leaves off at
    if (split == 0)
      first_product<IO, RP, WV, MF>(a.second, row_at(static_cast<const E*>(a.second.x) + b * a.second.bs, row0, a.second.ts),
                                v, a.R, live, (wave + WV - ceil_div(a.first.K, 16 * VEC) % WV) % WV, lane, part[1]);
  }
  if (all > 0) fetch_b(block_of(0), AHEAD ? bn : br);
  typedef Lane<IO, 1> One;
  const bool owns_rest = rest > 0 && split == 0 && r < H;
  typename One::raw rest_b[RP / 8][REST], rest_y = One::fill(0);
  if (owns_rest) {
#pragma unroll
    for (int c = 0; c < RP / 8; ++c)
#pragma unroll
      for (int j = 0; j < REST; ++j) rest_b[c][j] = One::load(Bm + min(c0 + c, a.R - 1) * a.N + a.N - max(rest - j, 1));
    if (ADD) rest_y = One::load(shifted(yb, min(r, rows - 1) * a.y_ts) + a.N - max(rest - (int)(threadIdx.x & 7), 1));
  }
  __syncthreads();
  if (r < H) {
    float u[RP / 8];
    if (!ADD && split == 0) {
      sum_shares<RP, WV, H>(part[ADD ? 0 : 1], r, c0, live, a.R, s, u);
      keep_hidden<RP>(a.second.keep, kept, row0 % ROWS + r, c0, u);
    }
    sum_shares<RP, WV, H>(part[0], r, c0, live, a.R, s, u);
    if (!ADD && split == 0) keep_hidden<RP>(a.first.keep, kept, row0 % ROWS + r, c0, u);
    if (owns_rest) {
      float sum = 0.0f, y;
#pragma unroll
      for (int j = 0; j < REST; ++j) {
        float z = 0.0f;
#pragma unroll
        for (int c = 0; c < RP / 8; ++c) {
          float m;
          One::unpack(rest_b[c][j], &m);
          z = c0 + c < a.R ? fmaf(u[c], m, z) : z;
        }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) z += __shfl_xor(z, o, 64);
        if ((int)(threadIdx.x & 7) == j) sum = z;
      }
      One::unpack(rest_y, &y);
      y += sum;
      if ((int)(threadIdx.x & 7) < rest && r < rows && !(ADD && a.in_place && r >= live))
        One::store(shifted(ob, r * a.o_ts) + a.N - rest + (threadIdx.x & 7), r < live ? One::pack(&y) : rest_y);
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int c = 0; c < RP / 8; ++c) hid.u[r][c0 + c] = u[c];
    } else {
      float up = 1.0f;
      if constexpr (IO::INF == IoF16::INF) {
        // the row's largest magnitude to [2^13, 2^14): both parts and their products stay inside fp16 and fp32
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < RP / 8; ++c) top = fmaxf(top, fabsf(u[c]));
        top = fmaxf(top, __shfl_xor(top, 1, 64));
        top = fmaxf(top, __shfl_xor(top, 2, 64));
        top = fmaxf(top, __shfl_xor(top, 4, 64));
        if (top > 1e-30f && top < INFINITY) {
          int e;
          frexpf(top, &e);
          up = ldexpf(1.0f, 14 - e);
        }
        if ((threadIdx.x & 7) == 0) hid.factor[r] = 1.0f / up;
      }
#pragma unroll
      for (int c = 0; c < RP / 8; c += 2) {
        uint32_t p[PARTS<IO>];
        parts_of<IO>(u[c] * up, u[c + 1] * up, p);
#pragma unroll
        for (int k = 0; k < PARTS<IO>; ++k) *reinterpret_cast<uint32_t*>(&hid.part[k][r][c0 + c]) = p[k];
      }
    }
  }
  __syncthreads();

  int held = -1;
  for (int k = 0; k < all; ++k) {
    const int cb = block_of(k), m = piece_of(k);
#pragma unroll
    for (int i = 0; i < 4; ++i) yr[i] = ADD ? yn[i] : Io::fill(0);
    if (cb != held) {
      held = cb;
      if (!AHEAD && k > 0) fetch_b(cb, br);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if constexpr (AHEAD) br[i] = bn[i];
        if (rank_of<IO, RP>(q, i) >= a.R) br[i] = Io::fill(0);
      }
      if constexpr (!WIDE) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          u32x4 t[8];
          transpose8(br + 8 * kb, t);
#pragma unroll
          for (int i = 0; i < 8; ++i) br[8 * kb + i] = t[i];
        }
      }
    }
    if (k + 1 < all) {
      if constexpr (ADD) fetch_y(block_of(k + 1), piece_of(k + 1), yn);
      if (AHEAD && block_of(k + 1) != cb) fetch_b(block_of(k + 1), bn);
    }
    f32x4 z[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[j] = (f32x4){0, 0, 0, 0};
    const int ur = 16 * m + l16;
    if constexpr (WIDE) {
#pragma unroll
      for (int t = 0; t < RP / 4; ++t) {
        const float u = hid.u[ur][q * (RP / 4) + t];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          z[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(u, __uint_as_float(br[t][j]), z[j], 0, 0, 0);
      }
    } else if constexpr (RP == 16) {
      // both halves of the lanes have these ranks of B: two parts of u to an instruction
#pragma unroll
      for (int k = (PARTS<IO> - 1) / 2 * 2; k >= 0; k -= 2) {
        u32x4 u = Io::fill(0);
        if (k + 1 < PARTS<IO> || q < 2) u = *reinterpret_cast<const u32x4*>(&hid.part[k + q / 2][ur][8 * (q & 1)]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[j] = mma<IO>(u, br[j], z[j]);
      }
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int k = PARTS<IO> - 1; k >= 0; --k) {
          const u32x4 u = *reinterpret_cast<const u32x4*>(&hid.part[k][ur][32 * kb + 8 * q]);
#pragma unroll
          for (int j = 0; j < VEC; ++j) z[j] = mma<IO>(u, br[8 * kb + j], z[j]);
        }
      }
    }
    if constexpr (!WIDE) {
      if (unsure<VEC>(z)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f32x4 first = (f32x4){0, 0, 0, 0};
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {  // up to rank 16 in both halves of the lanes: twice the sum
            const u32x4 u = *reinterpret_cast<const u32x4*>(&hid.part[0][ur][32 * kb + 8 * (RP > 16 ? q : q & 1)]);
            first = mma<IO>(u, br[8 * kb + j], first);
          }
          settle(z[j], first);
        }
      }
    }
    const int sl = anew(l16), n = min(max(a.N - cb * CB - sl * VEC, 0), VEC);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * m + 4 * (lane >> 4) + i;
      float o[VEC];
      u32x4 w = yr[i];
      Io::unpack(w, o);
      float f = 1.0f;
      if constexpr (!WIDE && IO::INF == IoF16::INF) f = hid.factor[row];
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = fmaf(f, z[j][i], o[j]);
      if (row < live) w = Io::pack(o);
      if (row < rows && !(ADD && a.in_place && row >= live))
        Io::store_some(shifted(ob + cb * CB, row * a.o_ts + (uint32_t)(sl * 16)), w, n);
    }
  }
}

// Weights' gradients, one request (and slice of its rows) at a time: part[b][chunk][rank][column] = sum of u x over
// the slice's rows, the columns of x (from du) first, those of dy (from u) behind them.  A workgroup owns 16 VEC columns,
// its waves take every fourth 32 rows, 8 of them and VEC columns to a lane; their sums meet in LDS, the upper two waves'
// first.  Three workgroups to a CU hide the loads (fetching the next rows ahead leaves room for two and is no faster).
// 64 x 800 x (512 + 2048) rank 32 bf16 with ragged ends: 163 MB in 37 us, 4.4 TB/s.
struct OuterArgs {
  const void *x, *dy;
  int64_t x_bs, dy_bs;
  uint32_t x_ts, dy_ts;
  const float *du, *u;  // as keep_hidden left them
  const int32_t *voices, *lengths;
  float* part;
  int T, K, N, V, chunks, span, tiles;
};

constexpr int WAVES = 4;
// Above rank 32 the 16-bit types' sums (VEC to a lane and rank) leave room for one workgroup a CU: two take half of the ranks
// each (32 x 128 x (512 + 2048) rank 64 bf16: the whole backward pass 45.7 -> 36.1 us a call; fp32, half as many, loses 0 to 2 %).
template <class IO, int RP>
constexpr int RANK_PARTS = RP > 32 && IO::VEC == 8 ? RP / 32 : 1;
template <class IO, int RP>
__global__ __launch_bounds__(WAVES * 64, 3) void outer_kernel(OuterArgs a) {
  constexpr int VEC = IO::VEC, SHARES = RANK_PARTS<IO, RP>, NJ = RP / 16 / SHARES, CB = 16 * VEC;
  typedef typename IO::elem E;
  typedef Full<IO> Io;
  const int j0 = blockIdx.x % SHARES * NJ;  // first sixteen of ranks
  const int kblocks = ceil_div(a.K, CB), groups = kblocks + ceil_div(a.N, CB);
  const int id = blockIdx.x / SHARES;
  int cb = id % groups;
  const int chunk = id / groups % a.chunks, b = id / groups / a.chunks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, l16 = lane & 15;
  __shared__ f32x4 sums[2][NJ * VEC][64];
  const int len = valid_rows(a.lengths, b, a.T);
  const int first = chunk * a.span, last = min(first + a.span, len);
  if (voice_of(a.voices, b, a.V) < 0 || first >= last) return;
  const bool of_x = cb < kblocks;
  if (!of_x) cb -= kblocks;
  const int width = of_x ? a.K : a.N;
  const int c = cb * CB + l16 * VEC, n = min(max(width - c, 0), VEC);
  const bool whole = cb * CB + CB <= width;
  const uint32_t ts = of_x ? a.x_ts : a.dy_ts;
  const E* src = of_x ? static_cast<const E*>(a.x) + b * a.x_bs : static_cast<const E*>(a.dy) + b * a.dy_bs;
  const float* ub = of_x ? a.du : a.u;
  f32x4 acc[NJ][VEC];
  // rows first + r0 .. + 31, this lane the 8 from 8 q on; rows behind the last are zero (and so is their u)
  const auto fetch = [&](int r0, u32x4* xr, u32x4 (*ur)[2]) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        xr[i] = Io::load(shifted(row_at(src + cb * CB, r0, ts), min(8 * q + i, last - 1 - r0) * ts + (uint32_t)(l16 * 16)));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        xr[i] = Io::load_end(shifted(row_at(src, r0, ts), min(8 * q + i, last - 1 - r0) * ts), c, width);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) hidden_rows<RP>(ub, (int64_t)b * a.tiles + r0 / ROWS, j0 + j, lane, ur[j]);
  };
  // A sum over parts is no number where a factor is infinite (see `unsure`).  The wave then takes its rows once more with zero
  // in the place of what is not finite wherever other parts than the first are multiplied.
  constexpr bool SPLIT = IO::INF == IoBf16::INF;
  bool again = false;
  do {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[j][i] = (f32x4){0, 0, 0, 0};
    for (int r0 = first + wave * ROWS; r0 < last; r0 += WAVES * ROWS) {
      u32x4 xr[8], ur[NJ][2];
      fetch(r0, xr, ur);
      if (r0 + ROWS > last) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r0 + 8 * q + i >= last) xr[i] = Io::fill(0);
      }
      if constexpr (SPLIT) {
        u32x4 bt[8], part[NJ][PARTS<IO>];
        transpose8(xr, bt);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            uint32_t p[PARTS<IO>];
            const u32x4 r = ur[j][m / 2];
            parts_of<IO>(__uint_as_float(r[m % 2 * 2]), __uint_as_float(r[m % 2 * 2 + 1]), p);
#pragma unroll
            for (int k = 0; k < PARTS<IO>; ++k) part[j][k][m] = p[k];
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[j][i] = mma<IO>(part[j][0], bt[i], acc[j][i]);
        }
        if (again) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) bt[i] = finite_bf16(bt[i]);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int k = 1; k < PARTS<IO>; ++k) part[j][k] = finite_bf16(part[j][k]);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int k = 1; k < PARTS<IO>; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[j][i] = mma<IO>(part[j][k], bt[i], acc[j][i]);
      } else {  // fp16 has no range for parts here: a factor per row would not come out of the sum
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          float xv[VEC];
          Io::unpack(xr[s], xv);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ur[j][s / 4][s % 4]), xv[i], acc[j][i], 0, 0, 0);
        }
      }
    }
    if (again) break;
#pragma unroll
    for (int j = 0; j < NJ; ++j) again |= SPLIT && unsure<VEC>(acc[j]);
  } while (again);
#pragma unroll
  for (int half = 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sums[wave - half][j * VEC + i][lane] = acc[j][i];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[j][i] += sums[wave][j * VEC + i][lane];
    }
    __syncthreads();
  }
  if (wave > 0) return;
  const int total = a.K + a.N;
  float* out = a.part + (int64_t)(b * a.chunks + chunk) * RP * total + (of_x ? 0 : a.K) + c;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) o[k] = acc[j][k][i];
      store_f32_some<VEC>(out + (int64_t)(16 * (j0 + j) + 4 * q + i) * total, n, o);
    }
}

// Sum over the requests of a voice, in their order.  A thread takes four columns; the requests of the voice are listed
// first, so that the loads of several are in flight: 5 to 6 us, most of them the chain of list, load and store.
struct GatherArgs {
  const float* part;
  const int32_t *voices, *lengths;
  void *ddown, *dup;
  int B, T, K, N, R, RP, chunks, span;
};
constexpr int LISTED = 256;  // threads of the gather: one looks at one slice
template <class IO>
__global__ __launch_bounds__(LISTED) void gather_kernel(GatherArgs a) {
  typedef typename IO::elem E;
  __shared__ int slices[LISTED], count[LISTED / 64];
  const int total = a.K + a.N, cols = ceil_div(total, LISTED * 4);
  const int col = (blockIdx.x % cols * LISTED + threadIdx.x) * 4, r = blockIdx.x / cols % a.R, v = blockIdx.x / cols / a.R;
  const int64_t pitch = (int64_t)a.RP * total;
  // the last thread of a row that ends inside its four columns takes the row's last four (a row has two at least)
  const int at0 = min(col, max(total - 4, 0));
  const float* p = a.part + (int64_t)r * total + at0;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int from = 0; from < a.B * a.chunks; from += LISTED) {
    // in order: a thread's slice goes where the slices in front of it leave off
    const int k = from + threadIdx.x, b = k / a.chunks;
    const bool mine = k < a.B * a.chunks && a.voices[b] == v && k % a.chunks * a.span < valid_rows(a.lengths, b, a.T);
    const uint64_t wave = __ballot(mine);
    if ((threadIdx.x & 63) == 0) count[threadIdx.x >> 6] = __popcll(wave);
    __syncthreads();
    int at = __popcll(wave & ((1ull << (threadIdx.x & 63)) - 1)), all = 0;
    for (int w = 0; w < LISTED / 64; ++w) {
      if (w < (int)(threadIdx.x >> 6)) at += count[w];
      all += count[w];
    }
    if (mine) slices[at] = k;
    __syncthreads();
    const auto take = [&](int k, float* t) {
      if (total >= 4)
        load_f32<4>(p + slices[k] * pitch, t);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = j < total ? p[slices[k] * pitch + j] : 0.0f;
    };
    int i = 0;
    for (; i + 4 <= all; i += 4) {
      float t[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) take(i + k, t[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += t[k][j];
    }
    for (; i < all; ++i) {
      float t[4];
      take(i, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += t[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = at0 + j;
    if (c < col || c >= total) continue;
    if (c < a.K)
      static_cast<E*>(a.ddown)[((int64_t)v * a.R + r) * a.K + c] = (E)s[j];
    else
      static_cast<E*>(a.dup)[((int64_t)v * a.R + r) * a.N + c - a.K] = (E)s[j];
  }
}

int padded_rank(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : 64; }

template <class IO, int RP, int WV, int MF, bool ADD>
int launch_waves(AddArgs a, int64_t tiles, int splits, hipStream_t s) {
  a.splits = splits;
  const char* name = ADD ? "ttsx_adapter_add" : "ttsx_adapter_backward";
  TTSX_ARG(tiles * splits <= most_workgroups(WV * 64), "%s: too many rows", name);
  return launch_kernel(name, adapter_kernel<IO, RP, WV, MF, ADD>, tiles * splits, WV * 64, s, a);
}
// Four waves to a tile where the tiles fill 256 CUs twice.  Fewer tiles get a workgroup of 16 waves each (8 at rank 64,
// whose operands need the registers) and share their columns among up to 256 workgroups; each of those repeats the
// first product, so no more of them than N is longer than K.  Up to 128 tiles are cut into halves of 16 rows, a CU to each:
// the chain of one tile is what is waited for then (32 x 128 x 512 -> 2048 rank 16 bf16 13.7 -> 10.9 us, its backward pass
// in fp32 36 -> 31; at 256 tiles, 64 x 128 rank 32, A read twice as often costs more: bf16 21.0 -> 25.7, fp32 35.4 -> 39.3).
constexpr int64_t HALVES = 128;
template <class IO, int RP, bool ADD>
int launch_tiles(AddArgs a, int B, hipStream_t s) {
  constexpr int MANY = RP == 64 ? 8 : 16;
  a.tiles = ceil_div(a.T, ROWS);
  int64_t tiles = (int64_t)B * a.tiles;
  if (tiles >= 512) return launch_waves<IO, RP, 4, 2, ADD>(a, tiles, 1, s);
  const int blocks = ceil_div(a.N, 16 * IO::VEC);
  const bool halves = tiles <= HALVES;
  if (halves) {
    a.tiles = ADD ? ceil_div(a.T, ROWS / 2) : 2 * a.tiles;  // both halves of a tile of kept values are written
    tiles = (int64_t)B * a.tiles;
  }
  const int pieces = ceil_div(min(a.T, halves ? ROWS / 2 : ROWS), 16);
  const int splits = min(min(ceil_div(blocks * pieces, MANY), max(1, (int)(256 / tiles))), max(1, a.N / a.first.K));
  return halves ? launch_waves<IO, RP, MANY, 1, ADD>(a, tiles, splits, s) : launch_waves<IO, RP, MANY, 2, ADD>(a, tiles, splits, s);
}

template <class IO>
int run_add(const AddArgs& a, int B, hipStream_t s) {
  switch (padded_rank(a.R)) {
    case 16: return launch_tiles<IO, 16, true>(a, B, s);
    case 32: return launch_tiles<IO, 32, true>(a, B, s);
    default: return launch_tiles<IO, 64, true>(a, B, s);
  }
}

struct BackPlan {
  int RP, chunks, span;
  size_t hidden, part;  // floats
};
// Slices of a request's rows: enough workgroups (one per 16 VEC columns and slice) to fill 256 CUs twice, 128 rows at
// least; every slice more is written and read again.
BackPlan back_plan(int B, int T, int K, int N, int R, int vec) {
  BackPlan p;
  p.RP = padded_rank(R);
  const int64_t groups = (int64_t)B * (ceil_div(K, 16 * vec) + ceil_div(N, 16 * vec));
  const int want = groups >= 512 ? 1 : (int)((512 + groups - 1) / groups), most = ceil_div(T, WAVES * ROWS);
  p.span = round_up(ceil_div(T, want < most ? want : most), ROWS);
  p.chunks = ceil_div(T, p.span);
  p.hidden = (size_t)B * p.RP * round_up(T, ROWS);
  p.part = (size_t)B * p.chunks * p.RP * ((size_t)K + N);
  return p;
}

template <class IO, int RP>
int run_backward(AddArgs a, const BackPlan& p, int B, float* ws, void* ddown, void* dup, hipStream_t s) {
  float *du = ws, *u = du + p.hidden, *part = u + p.hidden;
  a.first.keep = du, a.second.keep = u;
  OuterArgs o{};
  o.x = a.second.x, o.x_bs = a.second.bs, o.x_ts = a.second.ts;
  o.dy = a.first.x, o.dy_bs = a.first.bs, o.dy_ts = a.first.ts;
  o.du = du, o.u = u, o.voices = a.voices, o.lengths = a.lengths, o.part = part;
  o.T = a.T, o.K = a.second.K, o.N = a.first.K, o.V = a.V, o.chunks = p.chunks, o.span = p.span, o.tiles = ceil_div(a.T, ROWS);
  const int64_t grid = (int64_t)B * p.chunks * (ceil_div(o.K, 16 * IO::VEC) + ceil_div(o.N, 16 * IO::VEC)) * RANK_PARTS<IO, RP>;
  GatherArgs g{};
  g.part = part, g.voices = a.voices, g.lengths = a.lengths, g.ddown = ddown, g.dup = dup;
  g.B = B, g.T = a.T, g.K = o.K, g.N = o.N, g.R = a.R, g.RP = RP, g.chunks = p.chunks, g.span = p.span;
  const int64_t outs = (int64_t)a.V * a.R * ceil_div(o.K + o.N, LISTED * 4);
  // nothing is queued before all is known to fit
  const char* name = "ttsx_adapter_backward";
  TTSX_ARG(grid <= most_workgroups(WAVES * 64), "%s: too many rows", name);
  TTSX_ARG(outs <= most_workgroups(LISTED), "%s: too many voices", name);
  int rc = launch_tiles<IO, RP, false>(a, B, s);
  if (rc == TTSX_OK) rc = launch_kernel(name, outer_kernel<IO, RP>, grid, WAVES * 64, s, o);
  if (rc == TTSX_OK) rc = launch_kernel(name, gather_kernel<IO>, outs, LISTED, s, g);
  return rc;
}

template <class IO>
int run_backward_any(const AddArgs& a, const BackPlan& p, int B, float* ws, void* ddown, void* dup, hipStream_t s) {
  switch (p.RP) {
    case 16: return run_backward<IO, 16>(a, p, B, ws, ddown, dup, s);
    case 32: return run_backward<IO, 32>(a, p, B, ws, ddown, dup, s);
    default: return run_backward<IO, 64>(a, p, B, ws, ddown, dup, s);
  }
}

// The offsets inside a tile, and inside an adapter, fit 32 bits.
bool stride_ok(int64_t s) { return s >= 0 && s <= TTSX_SEQ_MAX_WIDTH; }
bool shape_ok(int B, int T, int K, int N, int R, int V) {
  return B >= 1 && T >= 1 && K >= 1 && N >= 1 && R >= 1 && R <= TTSX_ADAPTER_MAX_RANK && V >= 1 && T <= TTSX_SEQ_MAX_ROWS &&
         K <= TTSX_SEQ_MAX_WIDTH && N <= TTSX_SEQ_MAX_WIDTH && V <= TTSX_SEQ_MAX_VOICES;
}
bool dtype_ok(int d) { return d == TTSX_F32 || d == TTSX_BF16 || d == TTSX_F16; }

}  // namespace

extern "C" int ttsx_adapter_add(const void* y, int64_t y_batch_stride, int64_t y_row_stride, const void* x,
                                int64_t x_batch_stride, int64_t x_row_stride, const void* down, const void* up,
                                const int32_t* voices, const float* scale, const int32_t* lengths, int B, int T, int K,
                                int N, int R, int V, int dtype, void* out, int64_t out_batch_stride,
                                int64_t out_row_stride, void* stream) {
  TTSX_ARG(y && x && down && up && voices && out, "ttsx_adapter_add: null argument");
  TTSX_ARG(shape_ok(B, T, K, N, R, V), "ttsx_adapter_add: bad shape B=%d T=%d K=%d N=%d R=%d V=%d (1 <= R <= %d)", B, T,
           K, N, R, V, TTSX_ADAPTER_MAX_RANK);
  TTSX_ARG(dtype_ok(dtype), "ttsx_adapter_add: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  y_row_stride = stride_of(T, y_row_stride), x_row_stride = stride_of(T, x_row_stride);
  out_row_stride = stride_of(T, out_row_stride);
  TTSX_ARG(stride_ok(y_row_stride) && stride_ok(x_row_stride) && stride_ok(out_row_stride),
           "ttsx_adapter_add: a row stride outside 0..%ld", (long)TTSX_SEQ_MAX_WIDTH);
  TTSX_ARG(out != y || (out_batch_stride == y_batch_stride && out_row_stride == y_row_stride),
           "ttsx_adapter_add: out is y with other strides");
  AddArgs a{};
  const int64_t size = dtype == TTSX_F32 ? 4 : 2;
  a.first = {x, down, x_batch_stride, (uint32_t)(x_row_stride * size), K, nullptr};
  a.y = y, a.y_bs = y_batch_stride, a.y_ts = (uint32_t)(y_row_stride * size), a.up = up;
  a.out = out, a.o_bs = out_batch_stride, a.o_ts = (uint32_t)(out_row_stride * size);
  a.voices = voices, a.scale = scale, a.lengths = lengths, a.T = T, a.N = N, a.R = R, a.V = V;
  a.in_place = out == y;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TTSX_F32 ? run_add<IoF32>(a, B, s) : dtype == TTSX_BF16 ? run_add<IoBf16>(a, B, s) : run_add<IoF16>(a, B, s);
}

extern "C" long ttsx_adapter_backward_workspace(int B, int T, int K, int N, int R, int dtype) {
  TTSX_ARG(shape_ok(B, T, K, N, R, 1) && dtype_ok(dtype), "ttsx_adapter_backward_workspace: bad shape or type");
  const BackPlan p = back_plan(B, T, K, N, R, dtype == TTSX_F32 ? 4 : 8);
  return (long)(sizeof(float) * (2 * p.hidden + p.part));
}

extern "C" int ttsx_adapter_backward(const void* dy, int64_t dy_batch_stride, int64_t dy_row_stride, const void* x,
                                     int64_t x_batch_stride, int64_t x_row_stride, const void* down, const void* up,
                                     const int32_t* voices, const float* scale, const int32_t* lengths, int B, int T,
                                     int K, int N, int R, int V, int dtype, void* dx, void* ddown, void* dup,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  TTSX_ARG(dy && x && down && up && voices && dx && ddown && dup && workspace, "ttsx_adapter_backward: null argument");
  TTSX_ARG(shape_ok(B, T, K, N, R, V), "ttsx_adapter_backward: bad shape B=%d T=%d K=%d N=%d R=%d V=%d (1 <= R <= %d)",
           B, T, K, N, R, V, TTSX_ADAPTER_MAX_RANK);
  TTSX_ARG(dtype_ok(dtype), "ttsx_adapter_backward: dtype=%d is none of TTSX_F32, TTSX_BF16, TTSX_F16", dtype);
  dy_row_stride = stride_of(T, dy_row_stride), x_row_stride = stride_of(T, x_row_stride);
  TTSX_ARG(stride_ok(dy_row_stride) && stride_ok(x_row_stride), "ttsx_adapter_backward: a row stride outside 0..%ld",
           (long)TTSX_SEQ_MAX_WIDTH);
  const BackPlan p = back_plan(B, T, K, N, R, dtype == TTSX_F32 ? 4 : 8);
  TTSX_ARG(workspace_bytes >= sizeof(float) * (2 * p.hidden + p.part) && (uintptr_t)workspace % 16 == 0,
           "ttsx_adapter_backward: workspace too small or not aligned to 16 bytes");
  // the forward kernel with dy for x and the matrices swapped; x A^T is only kept
  AddArgs a{};
  const int64_t size = dtype == TTSX_F32 ? 4 : 2;
  a.first = {dy, up, dy_batch_stride, (uint32_t)(dy_row_stride * size), N, nullptr};
  a.second = {x, down, x_batch_stride, (uint32_t)(x_row_stride * size), K, nullptr};
  a.out = dx, a.o_bs = (int64_t)T * K, a.o_ts = (uint32_t)(K * size), a.up = down;
  a.voices = voices, a.scale = scale, a.lengths = lengths, a.T = T, a.N = K, a.R = R, a.V = V;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  return dtype == TTSX_F32    ? run_backward_any<IoF32>(a, p, B, ws, ddown, dup, s)
         : dtype == TTSX_BF16 ? run_backward_any<IoBf16>(a, p, B, ws, ddown, dup, s)
                              : run_backward_any<IoF16>(a, p, B, ws, ddown, dup, s);
}
