// Linear attention with a decay per head, chunked form: the kernel template shared by the translation
// units that instantiate it for float32, bfloat16 and float16 tensors.
//
// Per sequence and head, with d = exp(log_decay[h]) and a state S of K x V held in fp32:
//     S_t = d S_{t-1} + k_t^T v_t,      o_t = scale * q_t S_t.
// A chunk of C slots is taken at once (i, j: places in the chunk, n of them in use, S before the chunk):
//     o_i = d^(i+1) scale q_i S + sum_{j<=i} d^(i-j) scale (q_i k_j) v_j
//     S'  = d^n S + sum_j d^(n-1-j) k_j^T v_j.
// The gradients are the same recurrence with other operands: dq is (do, v, k) for (q, k, v) forward in
// time; dk is (v, do, q) and dv is (k, q, do) backward in time from the gradient of the last state, and
// the state that this leaves is the gradient of the first. Backward in time the state enters with the
// exponents moved by one (`e` below): what the kernel carries is d R_{t+1}, so that the gradient of the
// last state enters the last slot undecayed and the carry at the end is that of the first state.
//
// One wave owns 16 NV columns of V and all of K: S stays in its accumulators from the first chunk to
// the last, and the waves of a workgroup share nothing but the staged rows of q, k and v and the scores, so a chunk
// costs one or two barriers. All products are laid out so that an accumulator is the next product's operand
// without a move: a 16 x 16 tile holds, in lane (i = l % 16, g = l / 16), rows 4g..4g+3 of column i,
// and an operand of the matrix instructions holds k = 4g..4g+3 of row i, the same values:
//     P^T = K Q^T (columns: slots of q)     -> O^T += V^T P^T takes P^T as it is,
//     S  += K^T V (rows K, columns V)       -> O^T += S^T Q^T takes S as it is.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <cstdint>

#include "cet_internal.h"

namespace cet {
namespace la {

struct Strides {
  long b, t, h;  // elements; the feature axis is contiguous
};

struct Args {
  const void *q, *k, *v;
  void* o;
  const float* init;       // state before the first slot (nullptr: zero), element (k, v) at k * init_k + v * init_v
  float* fin;              // state after the last slot [B * H][K][V] (nullptr: not wanted)
  const float* log_decay;  // [H]
  const void* lengths;     // [B] int32 or int64 (nullptr: all T)
  float* ws;               // states between segments: [B * H][nseg - 1] states, element (k, v) at k * ws_k + v * ws_v
  Strides sq, sk, sv, so;
  int B, T, H, K, V;
  int init_k, init_v, ws_k, ws_v;
  int lengths64, reverse;
  int seg_len, nseg, nslice;
  int vec_o;  // rows of o start on the boundaries that stores of four need (those of q, k and v always do)
  float s_inter, s_intra, s_kv;
};

// Passes of one shape in one launch (the gradients).
struct Passes {
  Args a[3];
  int n;
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <bool B, typename X, typename Y>
struct Pick {
  typedef X T;
};
template <typename X, typename Y>
struct Pick<false, X, Y> {
  typedef Y T;
};

// d^n with d^0 = 1 also for d = 0 (a log decay of minus infinity)
__device__ inline float pw(float g2, int n) { return n == 0 ? 1.f : exp2f((float)n * g2); }
// the same without denormal results (below 2^-126 they are zero), in one instruction
__device__ inline float pw_fast(float g2, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f((float)n * g2); }

// slots of sequence b that are in use
__device__ inline int row_count(const void* lengths, int lengths64, int T, int b) {
  if (!lengths) return T;
  const long n = lengths64 ? static_cast<const long*>(lengths)[b] : (long)static_cast<const int*>(lengths)[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}
__device__ inline int row_count(const Args& a, int b) { return row_count(a.lengths, a.lengths64, a.T, b); }

// The arithmetic of a tensor type. float32 and float16 tensors are multiplied in fp32 (a float16
// state or score would leave that type's range on long histories), bfloat16 ones in bf16.

// Slots of a chunk: 32 with outputs, 64 where only states are formed (fewer barriers; no scores to hold). In fp32 half
// as many or fewer as soon as the rows are long: two workgroups (K up to 128) or three buffers then fit a CU's LDS, and
// one wave holds all of K (2 x 6 heads of 128 x 128, 4096 slots: 59 us; 32 slots, K in halves by two waves and one
// workgroup of 64 columns per CU 75; 186 heads of 256 x 256, 702 slots: 560 us, by slices of 32 columns 870).
// Four blocks of K by eight waves too: with 32 slots nine of their 128 registers spilled, at the same times.
constexpr int OUT_SLOTS = 32, STATE_SLOTS = 64;
constexpr int chunk_slots(bool bf, size_t bytes, bool out, int nk, int wc) {
  if (out) return bf || nk < 4 || (nk == 4 && !(bytes == 4 && wc == 8)) ? 32 : 16;
  return bf ? 64 : nk > 8 ? 16 : nk > 4 || wc == 8 ? 32 : 64;
}

template <typename IO>
struct Type {
  typedef IO V4 __attribute__((ext_vector_type(4)));
  static constexpr bool BF = __is_same(IO, __bf16);
  typedef typename Pick<BF, bf4, f4>::T Quad;  // four values of an operand: k = 4g..4g+3
  typedef typename Pick<BF, bf8, f4>::T Score; // four fp32 values as an operand: in bf16 two terms of each, x and what is left
  __device__ static Quad quad(const V4& v) {
    if constexpr (BF || __is_same(IO, float))
      return v;
    else
      return f4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  // said to be global memory: stores through a generic pointer are waited for with the LDS reads
  __device__ static void store(IO* p, float v) { *(__attribute__((address_space(1))) IO*)p = (IO)v; }
  __device__ static void store4(IO* p, const f4& v) {
    *(__attribute__((address_space(1))) V4*)p = V4{(IO)v[0], (IO)v[1], (IO)v[2], (IO)v[3]};
  }
};

// acc += A B over 16 values of k in one tile (fp32: four instructions of k = 4)
__device__ inline f4 mma16(const f4& a, const f4& b, f4 c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
  return c;
}
// over 32 values of k: two quads of each operand
__device__ inline f4 mma32(const bf4& a0, const bf4& a1, const bf4& b0, const bf4& b1, f4 c) {
  const bf8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
  const bf8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline bf4 to_bf(const f4& v) { return __builtin_convertvector(v, bf4); }
// (whole vectors one way and bits the other: of single conversions the compiler made the packed values and each by itself)
__device__ inline f4 to_f(const bf4& v) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 w = __builtin_bit_cast(u2, v);
  return f4{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16),
            __builtin_bit_cast(float, w[1] & 0xffff0000u)};
}
// An fp32 operand of bf16 products in two terms, 2^-16 of it at most left out: scores and states are sums in fp32, and
// rounded to one term they made the outputs' error 1.4 times that of their own rounding. (8 x 16 heads x 2048 slots of
// 128 x 128: 126 us forward and 293 for the gradients, with one term 119 and 271; 96 heads of 256 x 256: 255, 229.)
__device__ inline bf8 two_terms(const f4& v) {
  const bf4 hi = to_bf(v);
  return __builtin_shufflevector(hi, to_bf(v - to_f(hi)), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ inline bf4 first_term(const bf8& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3); }
__device__ inline bf4 second_term(const bf8& v) { return __builtin_shufflevector(v, v, 4, 5, 6, 7); }

__device__ inline unsigned lds_address(const void* p) {
  return (unsigned)(unsigned long)(const __attribute__((address_space(3))) char*)p;
}
// 16 bytes per lane straight into LDS at lds + 16 * lane, in assembly: loads into registers are waited for by the
// compiler wherever it merges or copies them, which left a chunk's rows no time to travel. The waits below order them.
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

// The SLOTS rows of a chunk in LDS, COLS columns in 16-byte pieces. Piece p of row r lies at p ^ turn(r), so that the
// reads of a wave touch all banks equally often; LDS takes the pieces in the order of the lanes, so the
// permutation is made on the memory side. Rows as an operand: 16 rows of one piece (fp32) or of one half piece.
// Columns as an operand: fp32 rows 4g + r of four pieces each, 2-byte types rows of two pieces each through the
// transposing read, which hands lane i of each 16 the column i of the four rows that they read 8 bytes of each.
template <typename IO, int COLS, int SLOTS>
struct Tile {
  static constexpr int E = sizeof(IO), VEC = 16 / E, P = COLS / VEC, PB = P < 16 ? P : 16, SHARE256 = 16 / PB;
  static constexpr int BYTES = SLOTS * COLS * E, PARTS = BYTES / 1024;  // a part: what one instruction of a wave brings
  typedef typename Type<IO>::V4 V4;
  typedef typename Type<IO>::Quad Quad;

  __device__ static int turn(int r) {
    const int u = r / SHARE256;  // rows of this many share the banks' 256 bytes
    return E == 2 ? ((u & (PB / 2 - 1)) << 1 | (r >> 3 & 1)) & (PB - 1) : u & (PB - 1);
  }
  // A lane's address for the 16 x 16 tile (sb, x): rows 16 sb.., columns 16 x... The pieces of column tile x differ from
  // those of tile 0 in bits that the permutation only flips, so one address per operand and an exclusive or serve
  // all of them (addresses kept for each tile took a hundred registers).
  static constexpr int ROW = COLS * E, SHIFT = E == 2 ? 5 : 6;
  template <typename X>
  __device__ static X at(unsigned p) {
    return *reinterpret_cast<const __attribute__((address_space(3))) X*>(p);
  }
  __device__ static unsigned rows_base(int i, int g) {
    return E == 2 ? i * ROW + (((g >> 1) ^ turn(i)) << 4) + (g & 1) * 8 : i * ROW + ((g ^ turn(i)) << 4);
  }
  __device__ static unsigned cols_base(int i, int g, int j) {  // fp32: one for each of the four rows
    const int r = 4 * g + (E == 2 ? i >> 2 : j);
    return E == 2 ? r * ROW + (((i >> 1 & 1) ^ turn(r)) << 4) + (i & 1) * 8 : r * ROW + (((i >> 2) ^ turn(r)) << 4) + (i & 3) * 4;
  }
  __device__ static Quad rows(unsigned base, int sb, int x) { return Type<IO>::quad(at<V4>((base ^ x << SHIFT) + sb * 16 * ROW)); }
  __device__ static Quad cols(const unsigned (&base)[E == 2 ? 1 : 4], int sb, int x) {
    if constexpr (E == 2) {
      typedef __attribute__((address_space(3))) s4* lds_s4;
      const s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(unsigned long)((base[0] ^ x << SHIFT) + sb * 16 * ROW));
      return Type<IO>::quad(__builtin_bit_cast(V4, r));
    } else {
      f4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = at<float>((base[j] ^ x << SHIFT) + sb * 16 * ROW);
      return v;
    }
  }
};

// One operand in memory: place i of the sequence is slot i, or rows - 1 - i backward in time. Places from `end`
// on and columns from `cols` on do not exist and are zero.
struct Source {
  const char* base;  // first place, first column
  long st;           // bytes from place to place
  int end, cols;

  template <typename Ti>
  __device__ void fetch(int part, int i0, unsigned lds, int lane) const {
    const int at = part * 64 + lane, r = at / Ti::P, c = (at % Ti::P ^ Ti::turn(r)) * Ti::VEC;
    const char* p = base + (i0 + r) * st + c * Ti::E;
    dma16(i0 + r < end && c < cols ? p : reinterpret_cast<const char*>(&zeros), lds + part * 1024);
  }
};
template <typename IO>
__device__ inline Source source(const IO* p, long st, int rows, int end, int reverse, int c0, int cols) {
  return Source{reinterpret_cast<const char*>(p + c0 + (reverse ? (rows - 1) * st : 0)), (reverse ? -st : st) * (long)sizeof(IO), end, cols - c0};
}

// Columns of the staged rows of q and k: a power of two, for the permutation, and 64 bytes at least.
constexpr int row_width(int nk, size_t bytes) {
  int w = bytes == 2 ? 32 : 16;
  while (w < 16 * nk) w *= 2;
  return w;
}

template <int NK, int NV>
__device__ inline void multiply_out(f4 (&S)[NK][NV], float f) {
#pragma unroll
  for (int x = 0; x < NK; ++x)
#pragma unroll
    for (int y = 0; y < NV; ++y) S[x][y] *= f;
}

// A workgroup is WC x KH waves: WC side by side along V, 16 NV columns each, and KH (1 or 2) that share the K of
// those columns. OUT: with outputs; without, only the state that a segment of slots adds is formed (into ws).
//
// Per chunk and wave: its blocks of the scores into LDS; its part of q S; what the chunk adds to its part of S; the
// one barrier; the rows of a later chunk asked for; scores times v, and the outputs. With two waves to the K of a
// column each finishes the outputs of one block of 16 slots, with the other's half of q S for it, which comes
// through LDS behind the same barrier.
template <typename IO, int NK, int NV, int WC, int KH, bool OUT>
__global__ __launch_bounds__(64 * WC * KH, WC == 8 && NK <= 8 ? 4 : WC * KH == 1 ? 1 : 2) void chunks(const Passes passes) {
  typedef Type<IO> Ty;
  typedef typename Ty::Quad Quad;
  typedef typename Ty::Score Score;
  constexpr int C = chunk_slots(Ty::BF, sizeof(IO), OUT, NK, WC), NB = C / 16;
  constexpr int NW = WC * KH, DK = row_width(NK, sizeof(IO)), NKW = NK / KH, SL = 16 * NV * WC;
  constexpr bool SHARE = NW > 1;  // one wave keeps its scores
  constexpr int BLOCKS = NB * (NB + 1) / 2, MINE = KH == 2 ? 1 : NB;
  // The scores of a chunk of 16 slots are one block: the waves take its K in parts, and each adds the parts up.
  constexpr bool SPLIT = OUT && NB == 1;
  constexpr int SCORES = SPLIT ? (NK < NW ? NK : NW) : BLOCKS;
  static_assert(KH <= 2 && NK % KH == 0 && (!OUT || NB == 2 || (NB == 1 && KH == 1 && SHARE)), "one or two blocks of slots in a chunk with outputs");
  typedef Tile<IO, DK, C> TK;
  typedef Tile<IO, SL, C> TV;
  // Buffers in a ring: rows of chunk c + BUFS are asked for when everybody has left chunk c.
  constexpr int BUF = (OUT ? 2 : 1) * TK::BYTES + TV::BYTES;
  // Three where that leaves room for two workgroups on a CU, or where two would not either.
  constexpr int REST = (OUT && SHARE ? 2 * SCORES * 64 * (int)sizeof(Score) : 0) + (OUT && KH == 2 ? 2 * NW * NV * 1024 : 0);
  constexpr int BUFS = SHARE && (3 * BUF + REST <= 81920 || (2 * BUF + REST > 81920 && 3 * BUF + REST <= 163840)) ? 3 : 2;
  constexpr int PARTS = BUF / 1024, PER = PARTS / NW, EXTRA = PARTS % NW;  // of a chunk; of each wave; of the first waves
  __shared__ __align__(1024) char tiles[BUFS][BUF];
  __shared__ Score ps[2][OUT && SHARE ? SCORES : 1][64];
  __shared__ f4 xs[2][OUT && KH == 2 ? NW : 1][NV][64];

  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wc = wave % WC, kh = wave / WC;
  // Workgroups go to the 8 XCDs in turn: the slices and passes of a segment, which read the same rows, are given to
  // one, and share its L2 (the three gradients of 8 x 16 heads of 128 x 128, 2048 slots, bf16: 543 MB fetched, 700 in the
  // order of the ids, in the same time; the whole backward call 255 us, with a launch for each gradient 281); the segments of
  // a sequence are spread over all, so that long ones keep no XCD busy alone (32 sequences, the first four full and the
  // others of 64 slots, 16 heads, bf16: 220 us forward and 256 for the gradients, by runs of workgroups 286 and 763).
  const int inner = passes.n * passes.a[0].nslice;
  unsigned id = blockIdx.x;
  int slice;
  if (const unsigned eight = 8 * inner, whole = gridDim.x / eight * eight; id < whole) {
    slice = id / 8 % inner;
    id = id / eight * 8 + id % 8;
  } else {
    slice = id % inner;
    id /= inner;
  }
  const Args a = passes.a[slice / passes.a[0].nslice];
  slice %= passes.a[0].nslice;
  const int nseg_here = OUT ? a.nseg : a.nseg - 1;  // without outputs the last segment has nothing to add
  const int seg = id % nseg_here;
  const long bh = id / nseg_here;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H);
  const int rows = row_count(a, b);
  const int first = seg * a.seg_len;
  const int end = min(rows, first + a.seg_len);
  const int c0 = slice * SL, col = c0 + wc * 16 * NV;  // first column of V: of the workgroup, of the wave
  const int k0 = kh * NKW * 16;                        // first row of the wave's part of S
  const bool busy = col < a.V;  // the last slice may leave waves with nothing but their share of rows and scores

  const IO* q = static_cast<const IO*>(a.q) + b * a.sq.b + h * a.sq.h;
  const IO* k = static_cast<const IO*>(a.k) + b * a.sk.b + h * a.sk.h;
  const IO* v = static_cast<const IO*>(a.v) + b * a.sv.b + h * a.sv.h;
  IO* o = OUT ? static_cast<IO*>(a.o) + b * a.so.b + h * a.so.h : nullptr;

  const Source from_q = source(q, a.sq.t, rows, end, a.reverse, 0, a.K), from_k = source(k, a.sk.t, rows, end, a.reverse, 0, a.K);
  const Source from_v = source(v, a.sv.t, rows, end, a.reverse, c0, a.V);
  const unsigned lds = lds_address(tiles);
  auto fetch = [&](int at, int buf) {  // this wave's parts of a chunk's rows: k, v, q one behind the other
    const unsigned to = lds + buf * BUF;
#pragma unroll
    for (int u = 0; u < PER + (EXTRA ? 1 : 0); ++u) {
      const int part = u * NW + wave;
      if (part < TK::PARTS)
        from_k.fetch<TK>(part, at, to, lane);
      else if (part < TK::PARTS + TV::PARTS)
        from_v.fetch<TV>(part - TK::PARTS, at, to + TK::BYTES, lane);
      else if (OUT && part < PARTS)
        from_q.fetch<TK>(part - TK::PARTS - TV::PARTS, at, to + TK::BYTES + TV::BYTES, lane);
    }
  };
#pragma unroll
  for (int u = 0; u < BUFS; ++u)
    if (first + u * C < end) fetch(first + u * C, u);

  f4 S[NKW][NV];
#pragma unroll
  for (int x = 0; x < NKW; ++x)
#pragma unroll
    for (int y = 0; y < NV; ++y) S[x][y] = f4{0.f, 0.f, 0.f, 0.f};

  const long states = (long)a.K * a.V;
  bool have = false;  // S is not all zero
  if (OUT) {
    const float* from = seg ? a.ws + (bh * (a.nseg - 1) + seg - 1) * states : a.init ? a.init + bh * states : nullptr;
    const int fk = seg ? a.ws_k : a.init_k, fv = seg ? a.ws_v : a.init_v;
    have = from != nullptr && (first < end || seg == 0);
    if (have && fk == 1 && a.K % 4 == 0) {  // a transposed state: four neighbours at once (states start on 16 bytes)
#pragma unroll
      for (int x = 0; x < NKW; ++x)
#pragma unroll
        for (int y = 0; y < NV; ++y) {
          const int kk = k0 + 16 * x + 4 * g, vv = col + 16 * y + i;
          if (kk < a.K && vv < a.V) S[x][y] = *reinterpret_cast<const f4*>(from + kk + (long)vv * fv);
        }
    } else if (have) {
#pragma unroll
      for (int x = 0; x < NKW; ++x)
#pragma unroll
        for (int y = 0; y < NV; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kk = k0 + 16 * x + 4 * g + r, vv = col + 16 * y + i;
            if (kk < a.K && vv < a.V) S[x][y][r] = from[(long)kk * fk + (long)vv * fv];
          }
    }
  }

  const float g2 = a.log_decay[h] * 1.44269504088896340736f;
  const int e = a.reverse ? 0 : 1;
  float wd[4], wo[4];  // scores of a block with itself (masked) and with the one before
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int s = 4 * g + r;
    wd[r] = i >= s ? pw(g2, i - s) * a.s_intra : 0.f;
    wo[r] = pw(g2, 16 + i - s) * a.s_intra;
  }
  const float rf[2] = {pw(g2, i + e) * a.s_inter, pw(g2, 16 + i + e) * a.s_inter};
  // A state that fades slowly is kept as S / d^m, m slots since it was last multiplied out: a chunk then adds
  // its keys and values by the weights d^-(m + 1 + j) and touches no element of S otherwise, and the weight of
  // a slot far back is not rounded once per chunk. It is multiplied out when d^m would leave 2^+-20. Where 2^-16
  // is passed within one chunk S is multiplied by d^n for each, and the weights are d^(n-1-j).
  const bool slow = fabsf(g2) * C < 16.f;
  int m = 0;
  float wk[NB][4];
#pragma unroll
  for (int sb = 0; sb < NB; ++sb)
#pragma unroll
    for (int r = 0; r < 4; ++r) wk[sb][r] = slow ? pw(g2, -(16 * sb + 4 * g + r + e)) * a.s_kv : 0.f;

  // block (tb, sb) of the scores, decayed, as an operand
  auto scores = [&](unsigned qr, unsigned kr, int tb, int sb) {
    f4 p = f4{0.f, 0.f, 0.f, 0.f};
    if constexpr (Ty::BF) {
#pragma unroll
      for (int x = 0; x < NK; x += 2) p = mma32(TK::rows(kr, sb, x), TK::rows(kr, sb, x + 1), TK::rows(qr, tb, x), TK::rows(qr, tb, x + 1), p);
    } else {
#pragma unroll
      for (int x = 0; x < NK; ++x) p = mma16(TK::rows(kr, sb, x), TK::rows(qr, tb, x), p);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = sb == tb ? (i >= 4 * g + r ? p[r] * wd[r] : 0.f) : p[r] * wo[r];
    if constexpr (Ty::BF)
      return two_terms(p);
    else
      return p;
  };

  IO* po[MINE];  // where this lane's slots of the chunk go
  const long po_step = (a.reverse ? -C : C) * a.so.t;
#pragma unroll
  for (int t = 0; t < MINE; ++t) {
    const long place = first + 16 * (KH == 2 ? kh : t) + i;
    po[t] = o + (a.reverse ? rows - 1 - place : place) * a.so.t + col + 4 * g;
  }

  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  constexpr int CB = sizeof(IO) == 2 ? 1 : 4;
  const unsigned row_lane = TK::rows_base(i, g);
  unsigned k_lane[CB], v_lane[CB];
#pragma unroll
  for (int j = 0; j < CB; ++j) k_lane[j] = TK::cols_base(i, g, j), v_lane[j] = TV::cols_base(i, g, j);
  int buf = 0;
  for (int at = first; at < end; at += C) {
    const int n = min(C, end - at);
    const unsigned kt = lds + buf * BUF, vt = kt + TK::BYTES, kr = kt + row_lane, qr = vt + TV::BYTES + row_lane;
    unsigned kc[CB], vc[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) kc[j] = kt + k_lane[j], vc[j] = vt + v_lane[j];

    Quad vf[NB][NV];
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int y = 0; y < NV; ++y) vf[sb][y] = TV::cols(vc, sb, wc * NV + y);

    f4 acc[OUT ? NB : 1][NV];
    Score pf[OUT ? BLOCKS : 1];
    const int flip = (at / C) & 1;
    if (OUT) {
      constexpr int TB[3] = {0, 1, 1}, SB[3] = {0, 0, 1};  // the blocks on and below the diagonal
      if constexpr (SPLIT) {
        f4 p = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NK; u += NW)
          if (u + wave < NK) p = mma16(TK::rows(kr, 0, u + wave), TK::rows(qr, 0, u + wave), p);
        if (wave < SCORES) ps[flip][wave][lane] = p;
      }
#pragma unroll
      for (int x = 0; x < (SPLIT ? 0 : BLOCKS); ++x) {
        if constexpr (SHARE) {
          if (x % NW == wave) ps[flip][x][lane] = scores(qr, kr, TB[x], SB[x]);
        } else {
          pf[x] = scores(qr, kr, TB[x], SB[x]);
        }
      }
#pragma unroll
      for (int tb = 0; tb < NB; ++tb)
#pragma unroll
        for (int y = 0; y < NV; ++y) acc[tb][y] = f4{0.f, 0.f, 0.f, 0.f};
      if (have && busy) {
        const float dm = pw_fast(g2, m);
#pragma unroll
        for (int x = 0; x < NKW; x += Ty::BF ? 2 : 1) {
          if constexpr (Ty::BF) {
#pragma unroll
            for (int y = 0; y < NV; ++y) {
              const bf8 s0 = two_terms(S[x][y]), s1 = two_terms(S[x + 1][y]);
#pragma unroll
              for (int tb = 0; tb < NB; ++tb) {
                const Quad q0 = TK::rows(qr, tb, k0 / 16 + x), q1 = TK::rows(qr, tb, k0 / 16 + x + 1);
                acc[tb][y] = mma32(second_term(s0), second_term(s1), q0, q1, acc[tb][y]);
                acc[tb][y] = mma32(first_term(s0), first_term(s1), q0, q1, acc[tb][y]);
              }
            }
          } else {
#pragma unroll
            for (int tb = 0; tb < NB; ++tb) {
              const Quad q0 = TK::rows(qr, tb, k0 / 16 + x);
#pragma unroll
              for (int y = 0; y < NV; ++y) acc[tb][y] = mma16(S[x][y], q0, acc[tb][y]);
            }
          }
        }
#pragma unroll
        for (int tb = 0; tb < NB; ++tb)
#pragma unroll
          for (int y = 0; y < NV; ++y) acc[tb][y] *= rf[tb] * dm;
      }
      if constexpr (KH == 2) {
#pragma unroll
        for (int y = 0; y < NV; ++y) xs[flip][wave][y][lane] = kh ? acc[0][y] : acc[NB - 1][y];
      }
    }

    if (busy && (!OUT || at + C < end || a.fin)) {  // nobody reads the state behind the last slot otherwise
      float w[NB][4];
      if (slow) {
        if (fabsf(g2) * (float)(m + C) > 20.f) {
          multiply_out(S, pw(g2, m));
          m = 0;
        }
        const float f = pw_fast(g2, -m);
#pragma unroll
        for (int sb = 0; sb < NB; ++sb)
#pragma unroll
          for (int r = 0; r < 4; ++r) w[sb][r] = wk[sb][r] * f;
        m += n;
      } else {
        multiply_out(S, pw(g2, n));
#pragma unroll
        for (int sb = 0; sb < NB; ++sb)
#pragma unroll
          for (int r = 0; r < 4; ++r) w[sb][r] = pw_fast(g2, max(0, n - e - (16 * sb + 4 * g + r))) * a.s_kv;
      }
      if constexpr (Ty::BF) {
#pragma unroll
       for (int sb = 0; sb < NB; sb += 2) {
        if (16 * sb >= n) break;
        // the decayed v in three bf16 terms (24 bits): the state is as exact as products of the tensors in fp32
        bf4 t0[2][NV], t1[2][NV], t2[2][NV];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int y = 0; y < NV; ++y) {
            f4 x = to_f(vf[sb + u][y]);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] *= w[sb + u][r];
            t0[u][y] = to_bf(x);
            const f4 x1 = x - to_f(t0[u][y]);
            t1[u][y] = to_bf(x1);
            t2[u][y] = to_bf(x1 - to_f(t1[u][y]));
          }
#pragma unroll
        for (int x = 0; x < NKW; ++x) {
          const bf4 kq0 = TK::cols(kc, sb, k0 / 16 + x), kq1 = TK::cols(kc, sb + 1, k0 / 16 + x);
#pragma unroll
          for (int y = 0; y < NV; ++y) {
            S[x][y] = mma32(kq0, kq1, t2[0][y], t2[1][y], S[x][y]);
            S[x][y] = mma32(kq0, kq1, t1[0][y], t1[1][y], S[x][y]);
            S[x][y] = mma32(kq0, kq1, t0[0][y], t0[1][y], S[x][y]);
          }
        }
       }
      } else {
#pragma unroll
        for (int sb = 0; sb < NB; ++sb) {
          if (16 * sb >= n) break;
          f4 vw[NV];
#pragma unroll
          for (int y = 0; y < NV; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) vw[y][r] = vf[sb][y][r] * w[sb][r];
#pragma unroll
          for (int x = 0; x < NKW; ++x) {
            const f4 kq = TK::cols(kc, sb, k0 / 16 + x);
#pragma unroll
            for (int y = 0; y < NV; ++y) S[x][y] = mma16(kq, vw[y], S[x][y]);
          }
        }
      }
      have = true;
    }

    // The next chunk's rows have landed. In a ring of three the rows of the chunk behind it may still travel: as
    // many instructions of this wave as it has parts (stores between them only make the wait longer).
    if (BUFS == 3 && at + 2 * C < end) {
      if (wave < EXTRA)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER + 1) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
    if (at + BUFS * C < end) fetch(at + BUFS * C, buf);
    buf = buf == BUFS - 1 ? 0 : buf + 1;

    if (OUT && busy) {
      if constexpr (SPLIT) {
        f4 p = ps[flip][0][lane];
#pragma unroll
        for (int x = 1; x < SCORES; ++x) p += ps[flip][x][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = i >= 4 * g + r ? p[r] * wd[r] : 0.f;
        pf[0] = p;
      } else if constexpr (SHARE) {
#pragma unroll
        for (int x = 0; x < BLOCKS; ++x) pf[x] = ps[flip][x][lane];
      }
#pragma unroll
      for (int t = 0; t < MINE; ++t) {
        const int tb = KH == 2 ? kh : t;
        if (16 * tb >= n) break;
        f4 out[NV];
#pragma unroll
        for (int y = 0; y < NV; ++y) {
          out[y] = KH == 2 ? (kh ? acc[NB - 1][y] : acc[0][y]) : acc[t][y];
          if constexpr (KH == 2) out[y] += xs[flip][kh ? wave - WC : wave + WC][y][lane];
          if constexpr (Ty::BF) {
            const bf4 none = bf4{(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f}, v1 = tb ? vf[1][y] : none;
            const Score p0 = tb ? pf[1] : pf[0];
            out[y] = mma32(vf[0][y], v1, second_term(p0), tb ? second_term(pf[2]) : none, out[y]);
            out[y] = mma32(vf[0][y], v1, first_term(p0), tb ? first_term(pf[2]) : none, out[y]);
          } else {
            if constexpr (NB == 1) {
              out[y] = mma16(vf[0][y], pf[0], out[y]);
            } else {
              out[y] = mma16(vf[0][y], tb ? pf[1] : pf[0], out[y]);
              if (tb) out[y] = mma16(vf[1][y], pf[2], out[y]);
            }
          }
        }
        if (16 * tb + i < n) {
#pragma unroll
          for (int y = 0; y < NV; ++y) {
            const int vv = col + 16 * y + 4 * g;
            if (a.vec_o && vv + 4 <= a.V) {
              Ty::store4(po[t] + 16 * y, out[y]);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (vv + r < a.V) Ty::store(po[t] + 16 * y + r, out[y][r]);
            }
          }
        }
        po[t] += po_step;
      }
    }
  }

  if (OUT) {
    // slots behind the sequence's end: four columns a thread
    constexpr int LPR = SL / 4;
    const int to = min(a.T, first + a.seg_len), vv = c0 + 4 * (int)(threadIdx.x % LPR);
    for (int at = max(rows, first) + (int)(threadIdx.x / LPR); at < to; at += 64 * NW / LPR) {
      IO* p = o + at * a.so.t + vv;
      if (a.vec_o && vv + 4 <= a.V) {
        Ty::store4(p, f4{0.f, 0.f, 0.f, 0.f});
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (vv + r < a.V) Ty::store(p + r, 0.f);
      }
    }
  }
  if (m) multiply_out(S, pw(g2, m));
  float* to = nullptr;
  int tk = a.ws_k, tv = a.ws_v;
  if (OUT) {
    const int owner = rows > 0 ? (rows - 1) / a.seg_len : 0;
    if (a.fin && seg == owner) to = a.fin + bh * states, tk = a.V, tv = 1;
  } else {
    to = a.ws + (bh * (a.nseg - 1) + seg) * states;
  }
  if (to) {
#pragma unroll
    for (int x = 0; x < NKW; ++x)
#pragma unroll
      for (int y = 0; y < NV; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kk = k0 + 16 * x + 4 * g + r, vv = col + 16 * y + i;
          if (kk < a.K && vv < a.V) to[(long)kk * tk + (long)vv * tv] = S[x][y][r];
        }
  }
}

// Columns of V that a workgroup takes: 16 (one wave, as long as that wave can bring in the rows of K in few
// instructions), else 64 or, from 65 on, 128: in bf16 up to K = 128 by four waves that hold their state in 64 registers
// each, otherwise by eight. (Forward and gradients in us, bf16, 128 x 128, 16 heads x 2048 slots, 32 sequences: 300 and 820,
// by 64 columns with eight waves, two to the K of a column, 370 and 1015; 8 sequences 128 and 255, 124 and 288; 12 sequences, where
// the coarser slices leave a round half empty, 197 and 389, 164 and 403. 256 x 256, 16 x 6 heads: 255 and 727, 328 and 803.
// fp32, 40 x 72, 16 x 6 heads of up to 777 slots, a pass: 35, 50.)
inline int slice_columns(int K, int V) {
  if (V <= 16 && K <= 64) return 16;
  return V > 64 ? 128 : 64;
}

// How many of them a CU holds at once and keeps busy: single waves as many as LDS takes; one where rows of 256 fill
// it, two otherwise.
inline int workgroups_per_cu(int dtype, int K, int V) {
  if (slice_columns(K, V) == 16) return K > 32 ? 4 : 8;
  return K > 128 && (dtype == CET_BF16 || V > 64) ? 1 : 2;
}

template <typename IO, int NK, bool OUT>
inline void launch_k(const Passes& p, unsigned blocks, hipStream_t s) {
  constexpr bool BF = Type<IO>::BF;
  const int cols = slice_columns(p.a[0].K, p.a[0].V);
  if constexpr (NK <= 4)
    if (cols == 16) return chunks<IO, NK, 1, 1, 1, OUT><<<blocks, 64, 0, s>>>(p);
  if constexpr (!BF || NK > 8)
    if (cols == 128) return chunks<IO, NK, 1, 8, 1, OUT><<<blocks, 512, 0, s>>>(p);
  if constexpr (NK <= 8 && BF)
    if (cols == 128) return chunks<IO, NK, 2, 4, 1, OUT><<<blocks, 256, 0, s>>>(p);
  if constexpr (NK <= 4 || (!BF && (OUT || NK <= 8)))
    chunks<IO, NK, 1, 4, 1, OUT><<<blocks, 256, 0, s>>>(p);
  else
    chunks<IO, NK, 1, 4, 2, OUT><<<blocks, 512, 0, s>>>(p);
}

// K in blocks of 16. In fp32 the matrix instructions are what counts, and there are more sizes than powers of two:
// none is issued for blocks that do not exist (16 x 6 heads of up to 777 slots, K = 40: 35 us a pass, as K = 64 38).
inline int k_blocks(int dtype, int K) {
  const int n = (K + 15) / 16;
  if (dtype == CET_BF16) return n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : n <= 12 ? 12 : 16;
  return n <= 4 ? n : n <= 6 ? 6 : n <= 8 ? 8 : n <= 12 ? 12 : 16;
}
// Passes of one launch have the same kernel and slices.
inline bool alike(int dtype, const Args& a, const Args& b) {
  const int cols = slice_columns(a.K, a.V);
  return k_blocks(dtype, a.K) == k_blocks(dtype, b.K) && cols == slice_columns(b.K, b.V) &&
         (a.V + cols - 1) / cols == (b.V + cols - 1) / cols;
}

template <typename IO, bool OUT>
inline void launch(const Passes& p, unsigned blocks, hipStream_t s) {
  constexpr bool BF = Type<IO>::BF;
  switch (k_blocks(BF ? CET_BF16 : CET_F32, p.a[0].K)) {
    case 1:
      if constexpr (!BF) launch_k<IO, 1, OUT>(p, blocks, s);
      break;
    case 2: launch_k<IO, 2, OUT>(p, blocks, s); break;
    case 3:
      if constexpr (!BF) launch_k<IO, 3, OUT>(p, blocks, s);
      break;
    case 4: launch_k<IO, 4, OUT>(p, blocks, s); break;
    case 6:
      if constexpr (!BF) launch_k<IO, 6, OUT>(p, blocks, s);
      break;
    case 8: launch_k<IO, 8, OUT>(p, blocks, s); break;
    case 12: launch_k<IO, 12, OUT>(p, blocks, s); break;
    default: launch_k<IO, 16, OUT>(p, blocks, s);
  }
}

// one translation unit each
void launch_f32(const Passes& p, bool out, unsigned blocks, hipStream_t s);
void launch_f16(const Passes& p, bool out, unsigned blocks, hipStream_t s);
void launch_bf16(const Passes& p, bool out, unsigned blocks, hipStream_t s);

}  // namespace la
}  // namespace cet
