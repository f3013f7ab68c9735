// The gated projection of a feed-forward block and its gradients: the tiled matrix product that all of its
// parts run on. Instantiated for float32, bfloat16 and float16 in a translation unit each.
//
//     g = x Wg^T + bg,   u = x Wu^T + bu,   y = act(g) * u                              (forward, one kernel)
//     dg = dy u act'(g), du = dy act(g)       with g and u formed again                 (backward 1, one kernel)
//     dx = [dg du] [Wg; Wu]                                                             (backward 2)
//     [dWg; dWu] = [dg du]^T x,   [dbg; dbu] = column sums of [dg du]                   (backward 3)
//
// dg and du are rounded to the tensors' type once, as the operands that the matrix instructions take: 0.0023 of a bf16
// gradient against 0.0017 by its own rounding alone. In two terms they would double both products behind them (8192 x
// 1024 to 2730: 210 us more of 480) and the bytes of dh. In fp16 they have that type's range, which callers are told.
//
// One product form: out[q][p] = sum_k P[p][k] Q[q][k], 16 x 16 tiles with p along the four registers of a
// lane, so that a lane stores four neighbours of a row. Either operand may lie in memory with k contiguous
// (rows) or with its own index contiguous (columns: dx reads the weights as they are, backward 3 both dh and x).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <cstdint>

#include "cet_internal.h"

namespace cet {
namespace gated {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

// An operand in memory. Rows (k contiguous): element (i, k) at p[i * ld + k]. Columns: at p[k * ld + i].
// Where `split` is below the length of the divided index (the rows; with columns, k), what lies from there on
// comes from p1, and of each part only `part` entries exist.
struct Operand {
  const void *p, *p1;
  long ld, ld1;
  int split, part;
};

struct Args {
  Operand P, Q;
  int np, nq, nk;     // lengths of p, q and k
  int tiles_p, tiles_q, splits, k_per_split;
  int F, Fp;          // features of the hidden layer, and the same rounded up to whole 16-byte pieces
  int activation;
  const void *bias_g, *bias_u;
  const void* dy;
  long ld_dy;
  int dy_step;        // elements that a row of dy can be read at once: 8, 4, 2 or 1
  void *out, *out1;   // out[q][p], rows from `out_split` on to out1
  long ld_out;
  int out_split, out_step;
  float* part;        // column sums per block of rows, or the splits' partial products
};

enum { FORWARD, BACKWARD, PLAIN, PARTIAL };

template <typename T>
struct Type;
template <>
struct Type<float> {
  static constexpr int E = 4;
};
template <>
struct Type<__bf16> {
  static constexpr int E = 2;
};
template <>
struct Type<_Float16> {
  static constexpr int E = 2;
};

// 16 bytes of an operand: 8 or 4 values of k
typedef uint32_t Frag __attribute__((ext_vector_type(4)));

template <typename T>
__device__ inline f4 mma(const Frag& a, const Frag& b, f4 c) {
  if constexpr (__is_same(T, float)) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], y[r], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}

__device__ inline unsigned lds_address(const void* p) {
  return (unsigned)(unsigned long)(const __attribute__((address_space(3))) char*)p;
}
// 16 bytes per lane straight into LDS at lds + 16 * lane. In assembly so that the compiler does not hold back
// every later LDS read until it has landed; the wait before the barrier orders it.
__device__ inline void dma16(const void* src, unsigned lds_wave) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(src), "s"(lds_wave)
      : "memory");
}

static __device__ const uint4 zeros = {0, 0, 0, 0};

// A tile of ROWS indices by 128 bytes of k in LDS, in 16-byte pieces whose places are permuted so that the
// reads of a wave touch every bank equally often (LDS takes the pieces in the order of the lanes, so the
// permutation is made on the memory side).
//   rows:    piece kc of row r (8 to a row of 128 bytes) at kc ^ (r >> 1 & 7): 16 rows of one kc are 256
//            different bytes of the banks' 256.
//   columns: a row of the tile is one k; piece mc at mc ^ turn(k). 16-bit values are read transposed, 8 bytes
//            of rows 8g..8g+3 (then +4) by each group of 16 lanes; fp32 ones singly, rows 4g + r.
template <typename T, int ROWS, int NT, bool COLS>
struct Tile {
  static constexpr int E = Type<T>::E, VEC = 16 / E, BK = 128 / E;
  static constexpr int PER_ROW = COLS ? ROWS / VEC : 8, TOTAL = ROWS * 8, N = TOTAL / NT, BYTES = ROWS * 128;
  static_assert(TOTAL % NT == 0, "whole pieces per thread");

  __device__ static int turn(int k) { return (E == 2 ? 2 * ((k & 3) | (k >> 3 & 1) << 2) : 4 * (k >> 2 & 3)) & (PER_ROW - 1); }

  // Rows: the addresses of this thread's pieces are carried along, 128 bytes a tile; all of them are the same piece
  // kc of their rows (NT / 8 rows apart, a multiple of the permutation's period).
  const char* row_at[COLS ? 1 : N];

  __device__ static int piece() { return (threadIdx.x & 7) ^ (threadIdx.x >> 4 & 7); }
  // The first tile to fetch starts at index i0 and k0.
  __device__ void init(const Operand& o, int i0, int len, int k0) {
    if constexpr (!COLS) {
      static_assert(NT % 128 == 0, "rows of a thread's pieces a multiple of 16 apart");
#pragma unroll
      for (int u = 0; u < N; ++u) {
        // FORWARD and BACKWARD take rows of both weights in one tile: the second half from p1
        const int r = (u * NT + (int)threadIdx.x) / 8;
        const bool second = o.split < ROWS && r >= o.split;
        const int i = min(i0 + (second ? r - o.split : r), len - 1);
        row_at[u] = reinterpret_cast<const char*>(static_cast<const T*>(second ? o.p1 : o.p) + (long)i * (second ? o.ld1 : o.ld) + k0 + piece() * VEC);
      }
    }
  }
  // piece of memory that goes to place `at`: index i0.. of the operand, k0.. of the summed axis
  __device__ static const char* source(const Operand& o, int at, int i0, int len, int k0, int k_end) {
    const int kr = at / PER_ROW, mc = at % PER_ROW ^ turn(kr);
    int k = k0 + kr;
    const bool second = k >= o.split;
    bool live = k < k_end;
    if (second) k -= o.split;
    live = live && k < o.part;
    const int i = min(i0 + mc * VEC, (len - 1) / VEC * VEC);
    const T* p = static_cast<const T*>(second ? o.p1 : o.p) + (long)k * (second ? o.ld1 : o.ld) + i;
    return live ? reinterpret_cast<const char*>(p) : reinterpret_cast<const char*>(&zeros);
  }
  // The tiles follow each other: k0 is BK behind that of the call before.
  __device__ void fetch(const Operand& o, unsigned lds, int i0, int len, int k0, int k_end) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned to = lds + wave * 1024;
    if constexpr (COLS) {
#pragma unroll
      for (int u = 0; u < N; ++u) dma16(source(o, u * NT + (int)threadIdx.x, i0, len, k0, k_end), to + u * NT * 16);
    } else {
      const bool live = k0 + piece() * VEC < k_end;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        dma16(live ? row_at[u] : reinterpret_cast<const char*>(&zeros), to + u * NT * 16);
        row_at[u] += 128;
      }
    }
  }
  // indices r0..r0+15 of step kk (64 bytes of k) as an operand of the matrix instructions
  __device__ static Frag read(const char* t, int r0, int kk, int i, int g) {
    if constexpr (!COLS) {
      const int r = r0 + i, kc = kk * 4 + g;
      return *reinterpret_cast<const Frag*>(t + r * 128 + ((kc ^ (r >> 1 & 7)) << 4));
    } else if constexpr (E == 2) {
      // k = 32 kk + 8 g + 4 half + i / 4, whose turn is that of the lane alone; pieces of 16 indices: 2 X, 2 X + 1
      typedef __attribute__((address_space(3))) s4* lds_s4;
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      const int th = ((i >> 2) | (g & 1) << 2) & (PER_ROW / 2 - 1);
      const char* p = t + (8 * g + (i >> 2)) * (ROWS * E) + (i & 1) * 8 + ((r0 / 16 ^ th) << 5) + ((i >> 1 & 1) << 4) + kk * 32 * ROWS * E;
      const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p));
      const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * ROWS * E)));
      return Frag{a[0], a[1], b[0], b[1]};
    } else {
      Frag f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int k = kk * 16 + 4 * g + r, m = r0 + i;
        f[r] = *reinterpret_cast<const uint32_t*>(t + k * (ROWS * E) + ((m / 4 ^ turn(k)) << 4) + (m & 3) * 4);
      }
      return f;
    }
  }
};

enum { SILU, GELU, RELU };

__device__ inline float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// The activation and its slope. silu: s = 1 / (1 + e^-g). gelu: the normal distribution's density e = e^(-g^2/2) and
// its tail P(-|g|) = e R(|g|), R a polynomial of t = 1 / (1 + 0.3 |g|) fitted by least maximum of its relative error (1.5e-7 for |g| up to
// 14), so that the tail keeps its bits as far as e does; without a branch between two ranges (erff took half the
// time of a narrow layer's pass). Exponential and reciprocal are the hardware's, 1 ulp each.
template <int KIND>
__device__ inline void act1(float g, float& a, float& slope) {
  if constexpr (KIND == SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + fast_exp(-g));
    a = g * s;
    slope = s * fmaf(g, 1.f - s, 1.f);
  } else if constexpr (KIND == GELU) {
    const float e = fast_exp(-0.5f * g * g);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(g), 1.f));
    float r = fmaf(t, 0.035674780f, -0.15720310f);
    r = fmaf(t, fmaf(t, r, 0.20635351f), -0.053683635f);
    r = fmaf(t, fmaf(t, r, 0.12856161f), 0.099913498f);
    r = fmaf(t, fmaf(t, r, 0.12075395f), 0.11962930f);
    const float tail = e * (t * r);
    const float p = g < 0.f ? tail : 1.f - tail;
    a = g * p;
    slope = fmaf(g * 0.39894228040143267794f, e, p);
  } else {
    a = g <= 0.f ? 0.f : g;  // (a NaN stays one)
    slope = g <= 0.f ? 0.f : 1.f;
  }
}
__device__ inline void act4(int kind, const f4& g, f4& a, f4& slope) {
  if (kind == SILU) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x, y;
      act1<SILU>(g[r], x, y);
      a[r] = x, slope[r] = y;
    }
  } else if (kind == GELU) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x, y;
      act1<GELU>(g[r], x, y);
      a[r] = x, slope[r] = y;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x, y;
      act1<RELU>(g[r], x, y);
      a[r] = x, slope[r] = y;
    }
  }
}

template <typename T>
__device__ inline void store4(T* p, const f4& v, int n, int step) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  if (n >= 4 && step >= 4) {
    *reinterpret_cast<t4*>(p) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else if (n >= 4 && step == 2) {
    *reinterpret_cast<t2*>(p) = t2{(T)v[0], (T)v[1]};
    *reinterpret_cast<t2*>(p + 2) = t2{(T)v[2], (T)v[3]};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) p[r] = (T)v[r];
  }
}
template <typename T>
__device__ inline f4 load4(const T* p, int n, int step) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4 && step >= 4) {
    const t4 x = *reinterpret_cast<const t4*>(p);
    v = f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
  } else if (n >= 4 && step == 2) {
    const t2 x = *reinterpret_cast<const t2*>(p), y = *reinterpret_cast<const t2*>(p + 2);
    v = f4{(float)x[0], (float)x[1], (float)y[0], (float)y[1]};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) v[r] = (float)p[r];
  }
  return v;
}

// n values of a 16-byte piece at a time: whole where rows start on 16 bytes (step 16 / sizeof(T)), in 4 bytes or singly
template <typename T>
__device__ inline uint4 load_piece(const T* p, int n, int step) {
  constexpr int VEC = 16 / sizeof(T), W = 4 / sizeof(T);
  if (n >= VEC && step >= VEC) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
  if (n >= VEC && step >= W) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const uint32_t*>(p)[j];
  } else {
    T e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = j < n ? p[j] : (T)0.f;
    __builtin_memcpy(w, e, 16);
  }
  return uint4{w[0], w[1], w[2], w[3]};
}
template <typename T>
__device__ inline void store_piece(T* p, const uint4& raw, int n, int step) {
  constexpr int VEC = 16 / sizeof(T), W = 4 / sizeof(T);
  if (n >= VEC && step >= VEC) {
    *reinterpret_cast<uint4*>(p) = raw;
  } else if (n >= VEC && step >= W) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(p)[j] = w[j];
  } else {
    T e[VEC];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (j < n) p[j] = e[j];
  }
}

template <int N>
struct Half {
  static constexpr int value = N;
};

template <typename T, int BP, int BQ, int WP, int WQ, bool PC, bool QC, int KIND>
__global__ __launch_bounds__(64 * WP * WQ, 2) void product(const Args a) {
  constexpr int NT = 64 * WP * WQ, NPT = BP / WP / 16, NQT = BQ / WQ / 16;
  constexpr bool GATED = KIND == FORWARD || KIND == BACKWARD;
  typedef Tile<T, BP, NT, PC> TP;
  typedef Tile<T, BQ, NT, QC> TQ;
  constexpr int BK = TP::BK;
  extern __shared__ __align__(1024) char lds[];  // two of [P tile | Q tile]
  constexpr int BUF = TP::BYTES + TQ::BYTES;

  // Workgroups go to the 8 XCDs in turn: each XCD is given one run of tiles, in blocks of eight rows of
  // tiles, so that the tiles that its L2 holds are shared by the workgroups that run on it together.
  const int total = a.tiles_p * a.tiles_q * a.splits;
  int id = blockIdx.x;
  {
    const int per = total / 8, rest = total % 8, xcd = id % 8, at = id / 8;
    id = xcd * per + min(xcd, rest) + at;
  }
  const int split = id / (a.tiles_p * a.tiles_q);
  id -= split * a.tiles_p * a.tiles_q;
  const int block = id / (8 * a.tiles_p), in = id - block * 8 * a.tiles_p;
  const int high = min(8, a.tiles_q - 8 * block);
  const int tq = 8 * block + in % high, tp = in / high;
  const int q0 = tq * BQ, p0 = tp * (GATED ? BP / 2 : BP);

  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = wave % WP, wq = wave / WP;
  const int k_first = split * a.k_per_split, k_end = min(a.nk, k_first + a.k_per_split);
  const unsigned base = lds_address(lds);

  f4 acc[NPT][NQT];
#pragma unroll
  for (int x = 0; x < NPT; ++x)
#pragma unroll
    for (int y = 0; y < NQT; ++y) acc[x][y] = f4{0.f, 0.f, 0.f, 0.f};

  TP from_p;
  TQ from_q;
  from_p.init(a.P, p0, a.np, k_first);
  from_q.init(a.Q, q0, a.nq, k_first);
  auto fetch_p = [&](int k0, int buf) { from_p.fetch(a.P, base + buf * BUF, p0, a.np, k0, k_end); };
  auto fetch_q = [&](int k0, int buf) { from_q.fetch(a.Q, base + buf * BUF + TP::BYTES, q0, a.nq, k0, k_end); };
  // first row of the wave's tile x of P: gate rows, then the up rows of the same features
  auto p_row = [&](int x) {
    return GATED ? (x < NPT / 2 ? wp * (BP / 2 / WP) + 16 * x : BP / 2 + wp * (BP / 2 / WP) + 16 * (x - NPT / 2)) : wp * (BP / WP) + 16 * x;
  };

  // A tile is worked on in four steps: half of its 128 bytes of k and half of the wave's tiles of P each. The
  // operands of a step travel from LDS into one set of registers while the matrix instructions work on the other,
  // across the barrier too: before the last step of a tile the next tile has landed, this one is all in registers,
  // and its buffer takes the rows of the tile after, P's at once and Q's behind the next step (3 % over both at
  // once). (Whole steps of k need 32 registers more and spilled where operands are read by columns.)
  constexpr int HP = NPT / 2;
  Frag p0_[HP], p1_[HP], q0_[NQT], q1_[NQT];
  auto load_p = [&](Frag (&fp)[HP], int buf, int kk, int half) {
    const char* pt = lds + buf * BUF;
#pragma unroll
    for (int x = 0; x < HP; ++x) fp[x] = TP::read(pt, p_row(half * HP + x), kk, i, g);
  };
  auto load_q = [&](Frag (&fq)[NQT], int buf, int kk) {
    const char* qt = lds + buf * BUF + TP::BYTES;
#pragma unroll
    for (int y = 0; y < NQT; ++y) fq[y] = TQ::read(qt, wq * (BQ / WQ) + 16 * y, kk, i, g);
  };
  auto multiply = [&](const Frag (&fp)[HP], const Frag (&fq)[NQT], auto half) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < HP; ++x)
#pragma unroll
      for (int y = 0; y < NQT; ++y) acc[decltype(half)::value * HP + x][y] = mma<T>(fp[x], fq[y], acc[decltype(half)::value * HP + x][y]);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (k_first < k_end) {
    fetch_p(k_first, 0);
    fetch_q(k_first, 0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (k_first + BK < k_end) fetch_p(k_first + BK, 1);
  if (k_first < k_end) {
    load_q(q0_, 0, 0);
    load_p(p0_, 0, 0, 0);
  }
  int buf = 0;
  for (int k0 = k_first; k0 < k_end; k0 += BK, buf ^= 1) {
    load_p(p1_, buf, 0, 1);
    if (k0 + BK < k_end) fetch_q(k0 + BK, buf ^ 1);
    multiply(p0_, q0_, Half<0>());
    load_q(q1_, buf, 1);
    load_p(p0_, buf, 1, 0);
    multiply(p1_, q0_, Half<1>());
    load_p(p1_, buf, 1, 1);
    multiply(p0_, q1_, Half<0>());
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + 2 * BK < k_end) fetch_p(k0 + 2 * BK, buf);
    if (k0 + BK < k_end) {
      load_q(q0_, buf ^ 1, 0);
      load_p(p0_, buf ^ 1, 0, 0);
    }
    multiply(p1_, q1_, Half<1>());
  }

  if constexpr (GATED) {
    // Results (and dy on its way in) go through LDS, so that memory sees whole pieces of 16 bytes along the rows: a
    // lane holds 4 features of a row, 16 rows apart from its neighbours'. (dy and dh read and written from the
    // accumulators' places: 66 us over the forward product's time at 8192 x 1024 x 2730, this way 30.) Rows of 256
    // bytes at most, so fp32 takes two rounds in the large tile.
    constexpr int E = Type<T>::E, VEC = 16 / E, XT = NPT / 2 * E > 8 ? 2 : NPT / 2, ROUNDS = NPT / 2 / XT;
    constexpr int PIECES = WP * 16 * XT / VEC, SHARE = 16 / PIECES;
    static_assert(2 * BQ * PIECES * 16 <= 2 * BUF, "two tiles of results in the operands' buffers");
    char* const first = lds;
    char* const second = lds + BQ * PIECES * 16;
    auto turn = [](int row) { return row / SHARE & (PIECES - 1); };
    // feature behind p0 of piece p in a round
    auto feature = [](int p, int round) { return p * VEC / (16 * XT) * (BP / 2 / WP) + round * 16 * XT + p * VEC % (16 * XT); };
    for (int round = 0; round < ROUNDS; ++round) {
      if (round) __syncthreads();
      if constexpr (KIND == BACKWARD) {
        for (int at = threadIdx.x; at < BQ * PIECES; at += NT) {
          const int row = at / PIECES, p = at % PIECES, q = q0 + row, f = p0 + feature(p, round), n = a.F - f;
          uint4 raw = {0, 0, 0, 0};
          if (q < a.nq && n > 0) raw = load_piece(static_cast<const T*>(a.dy) + (long)q * a.ld_dy + f, n, a.dy_step);
          *reinterpret_cast<uint4*>(first + (row * PIECES + (p ^ turn(row))) * 16) = raw;
        }
        __syncthreads();
      }
#pragma unroll
      for (int xr = 0; xr < NPT / 2; ++xr) {
        if (xr / XT != round) continue;
        const int f = p0 + wp * (BP / 2 / WP) + 16 * xr + 4 * g, n = a.F - f;
        const int byte = (wp * 16 * XT + 16 * (xr % XT) + 4 * g) * E;
        f4 bg = {0.f, 0.f, 0.f, 0.f}, bu = bg, sg = bg, su = bg;
        if (a.bias_g) bg = load4(static_cast<const T*>(a.bias_g) + f, n, 1);
        if (a.bias_u) bu = load4(static_cast<const T*>(a.bias_u) + f, n, 1);
#pragma unroll
        for (int y = 0; y < NQT; ++y) {
          const int row = wq * (BQ / WQ) + 16 * y + i;
          T* const place = reinterpret_cast<T*>(first + (row * PIECES + (byte / 16 ^ turn(row))) * 16 + byte % 16);
          f4 gv = acc[xr][y] + bg, uv = acc[xr + NPT / 2][y] + bu, v, slope;
          act4(a.activation, gv, v, slope);
          if constexpr (KIND == FORWARD) {
            store4(place, v * uv, 4, 4);
          } else {
            const f4 d = load4(place, 4, 4);
            f4 dg = {0.f, 0.f, 0.f, 0.f}, du = dg;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (r < n && q0 + row < a.nq) {  // columns behind F are summed over in the products behind this one: zero
                dg[r] = d[r] * uv[r] * slope[r];
                du[r] = d[r] * v[r];
              }
            }
            sg += dg;
            su += du;
            store4(place, dg, 4, 4);
            store4(reinterpret_cast<T*>(reinterpret_cast<char*>(place) + (second - first)), du, 4, 4);
          }
        }
        if constexpr (KIND == BACKWARD) {
          if (a.part) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int off = 1; off < 16; off *= 2) {
                sg[r] += __shfl_xor(sg[r], off);
                su[r] += __shfl_xor(su[r], off);
              }
            if (i == 0 && f < a.Fp) {
              float* to = a.part + (long)(tq * WQ + wq) * 2 * a.Fp + f;
              *reinterpret_cast<f4*>(to) = sg;
              *reinterpret_cast<f4*>(to + a.Fp) = su;
            }
          }
        }
      }
      __syncthreads();
      if (KIND == FORWARD && E == 2 && a.out_step == 1) {
        // Rows of an odd number of 2-byte values: every other one starts between two words, and its pieces are
        // stored as words from the value before them on (102,400 x 441 in fp16: 91 us, by single values 127).
        static_assert(E == 4 || 16 * XT == BP / 2 / WP, "a tile's pieces follow each other along the row");
        for (int at = threadIdx.x; at < BQ * PIECES; at += NT) {
          const int row = at / PIECES, p = at % PIECES, q = q0 + row, f = p0 + feature(p, round);
          if (q >= a.nq || f >= a.F) continue;
          const uint4 raw = *reinterpret_cast<const uint4*>(first + (row * PIECES + (p ^ turn(row))) * 16);
          T* const to = static_cast<T*>(a.out) + (long)q * a.ld_out + f;
          if (a.F - f < VEC || (reinterpret_cast<uintptr_t>(to) & 2) == 0) {
            store_piece(to, raw, a.F - f, 2);
            continue;
          }
          uint32_t* const w = reinterpret_cast<uint32_t*>(reinterpret_cast<uintptr_t>(to) - 2);
          unsigned short* const e = reinterpret_cast<unsigned short*>(to);
          if (p)
            w[0] = *reinterpret_cast<const unsigned short*>(first + (row * PIECES + ((p - 1) ^ turn(row))) * 16 + 14) | raw.x << 16;
          else
            e[0] = (unsigned short)raw.x;  // the word's other half is the tile's before this one
          w[1] = raw.x >> 16 | raw.y << 16;
          w[2] = raw.y >> 16 | raw.z << 16;
          w[3] = raw.z >> 16 | raw.w << 16;
          if (p == PIECES - 1 || a.F - f < 2 * VEC) e[7] = (unsigned short)(raw.w >> 16);  // no whole piece behind
        }
        continue;
      }
      for (int at = threadIdx.x; at < BQ * PIECES; at += NT) {
        const int row = at / PIECES, p = at % PIECES, q = q0 + row, f = p0 + feature(p, round);
        const int from = (row * PIECES + (p ^ turn(row))) * 16;
        if (q >= a.nq) continue;
        if constexpr (KIND == FORWARD) {
          if (f < a.F) store_piece(static_cast<T*>(a.out) + (long)q * a.ld_out + f, *reinterpret_cast<const uint4*>(first + from), a.F - f, a.out_step);
        } else if (f < a.Fp) {
          T* to = static_cast<T*>(a.out) + (long)q * a.ld_out + f;
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(first + from);
          *reinterpret_cast<uint4*>(to + a.Fp) = *reinterpret_cast<const uint4*>(second + from);
        }
      }
    }
  } else {
#pragma unroll
    for (int x = 0; x < NPT; ++x) {
      const int p = p0 + p_row(x) + 4 * g, n = a.np - p;
#pragma unroll
      for (int y = 0; y < NQT; ++y) {
        const int q = q0 + wq * (BQ / WQ) + 16 * y + i;
        if (q >= a.nq || n <= 0) continue;
        if constexpr (KIND == PARTIAL) {
          store4(a.part + ((long)split * a.nq + q) * a.ld_out + p, acc[x][y], n, a.ld_out % 4 == 0 ? 4 : 1);
        } else {
          const bool second = q >= a.out_split;
          const int row = second ? q - a.out_split : q;
          if (a.F && row >= a.F) continue;  // weights' gradients: rows behind F do not exist
          store4(static_cast<T*>(second ? a.out1 : a.out) + (long)row * a.ld_out + p, acc[x][y], n, a.out_step);
        }
      }
    }
  }
}

int run_f32(const Args& a, int kind, int tile, hipStream_t s);
int run_bf16(const Args& a, int kind, int tile, hipStream_t s);
int run_f16(const Args& a, int kind, int tile, hipStream_t s);

// Which product: KIND and the operands' layouts go together.
enum { STEP_FORWARD, STEP_DH, STEP_DX, STEP_DW, STEP_DW_PARTIAL, STEP_DX_PARTIAL };

template <typename T, int BP, int BQ, int WP, int WQ, bool PC, bool QC, int KIND>
inline int run1(const Args& a, hipStream_t s) {
  constexpr int LDS = 2 * (BP + BQ) * 128;
  auto* f = &product<T, BP, BQ, WP, WQ, PC, QC, KIND>;
  if (LDS > 65536) CET_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  f<<<(unsigned)(a.tiles_p * a.tiles_q * a.splits), 64 * WP * WQ, LDS, s>>>(a);
  CET_HIP(hipGetLastError());
  return CET_OK;
}
template <typename T, int BP, int BQ, int WP, int WQ>
inline int run2(const Args& a, int step, hipStream_t s) {
  switch (step) {
    case STEP_FORWARD: return run1<T, BP, BQ, WP, WQ, false, false, FORWARD>(a, s);
    case STEP_DH: return run1<T, BP, BQ, WP, WQ, false, false, BACKWARD>(a, s);
    case STEP_DX: return run1<T, BP, BQ, WP, WQ, true, false, PLAIN>(a, s);
    case STEP_DX_PARTIAL: return run1<T, BP, BQ, WP, WQ, true, false, PARTIAL>(a, s);
    case STEP_DW: return run1<T, BP, BQ, WP, WQ, true, true, PLAIN>(a, s);
    default: return run1<T, BP, BQ, WP, WQ, true, true, PARTIAL>(a, s);
  }
}
template <typename T>
inline int run(const Args& a, int step, int tile, hipStream_t s) {
  return tile == 256 ? run2<T, 256, 256, 2, 4>(a, step, s) : tile == 128 ? run2<T, 128, 128, 2, 2>(a, step, s) : run2<T, 64, 64, 2, 2>(a, step, s);
}

}  // namespace gated
}  // namespace cet
