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
// the last, and the waves of a workgroup share nothing but the staged rows of q, k and v, so a chunk
// costs two barriers. All products are laid out so that an accumulator is the next product's operand
// without a move: a 16 x 16 tile holds, in lane (i = l % 16, g = l / 16), rows 4g..4g+3 of column i,
// and an operand of the matrix instructions holds k = 4g..4g+3 of row i, the same values:
//     P^T = K Q^T (columns: slots of q)     -> O^T += V^T P^T takes P^T as it is,
//     S  += K^T V (rows K, columns V)       -> O^T += S^T Q^T takes S as it is.
// The columns of V that each wave recomputes P for cost 16 x 16 x K operations per block; handing P
// over through LDS instead would cost a third barrier per chunk.
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
  float* fin;              // state after the last slot (nullptr: not wanted), same addressing
  const float* log_decay;  // [H]
  const void* lengths;     // [B] int32 or int64 (nullptr: all T)
  float* ws;               // [B * H][nseg - 1][K * V]
  Strides sq, sk, sv, so;
  int B, T, H, K, V;
  int init_k, init_v, fin_k, fin_v;
  int lengths64, reverse;
  int seg_len, nseg, nslice;
  int vec_o;  // rows of o start on the boundaries that stores of four need (those of q, k and v always do)
  float s_inter, s_intra, s_kv;
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// d^n with d^0 = 1 also for d = 0 (a log decay of minus infinity)
__device__ inline float pw(float g2, int n) { return n == 0 ? 1.f : exp2f((float)n * g2); }

__device__ inline int row_count(const Args& a, int b) {
  if (!a.lengths) return a.T;
  const long n = a.lengths64 ? static_cast<const long*>(a.lengths)[b] : (long)static_cast<const int*>(a.lengths)[b];
  return n < 0 ? 0 : n > a.T ? a.T : (int)n;
}

// The arithmetic of a tensor type. float32 and float16 tensors are multiplied in fp32 (a float16
// state or score would leave that type's range on long histories), bfloat16 ones in bf16.
template <typename IO>
struct Type;

template <>
struct Type<float> {
  typedef float Lds;
  typedef f4 Quad;  // four values of an operand: k = 4g..4g+3
  static constexpr bool BF = false;
  static constexpr int VEC = 4, C = 32, LDPAD = 4;
  __device__ static void to_lds(float* p, const uint4& raw) { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ static float load(const float* p) { return *p; }
  __device__ static void store(float* p, float v) { *p = v; }
  __device__ static void store4(float* p, const f4& v) { *reinterpret_cast<f4*>(p) = v; }
};

template <>
struct Type<_Float16> {
  typedef float Lds;
  typedef f4 Quad;
  static constexpr bool BF = false;
  static constexpr int VEC = 8, C = 32, LDPAD = 4;
  __device__ static void to_lds(float* p, const uint4& raw) {
    const h8 v = *reinterpret_cast<const h8*>(&raw);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<f4*>(p + 4 * i) = f4{(float)v[4 * i], (float)v[4 * i + 1], (float)v[4 * i + 2], (float)v[4 * i + 3]};
  }
  __device__ static float load(const _Float16* p) { return (float)*p; }
  __device__ static void store(_Float16* p, float v) { *p = (_Float16)v; }
  __device__ static void store4(_Float16* p, const f4& v) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4*>(p) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
};

template <>
struct Type<__bf16> {
  typedef __bf16 Lds;
  typedef bf4 Quad;
  static constexpr bool BF = true;
  static constexpr int VEC = 8, C = 32, LDPAD = 8;
  __device__ static void to_lds(__bf16* p, const uint4& raw) { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ static float load(const __bf16* p) { return (float)*p; }
  __device__ static void store(__bf16* p, float v) { *p = (__bf16)v; }
  __device__ static void store4(__bf16* p, const f4& v) {
    *reinterpret_cast<bf4*>(p) = bf4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
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
__device__ inline bf4 to_bf(const f4& v) { return bf4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]}; }
__device__ inline f4 to_f(const bf4& v) { return f4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }

// rows r0..r0+15, k columns c0..c0+15 of a row-major tile as an operand (k = columns)
__device__ inline f4 quad_rows(const float* t, int ld, int r0, int c0, int i, int g) {
  return *reinterpret_cast<const f4*>(t + (r0 + i) * ld + c0 + 4 * g);
}
__device__ inline bf4 quad_rows(const __bf16* t, int ld, int r0, int c0, int i, int g) {
  return *reinterpret_cast<const bf4*>(t + (r0 + i) * ld + c0 + 4 * g);
}
// the same tile as an operand with k = rows: bf16 through the transposing LDS read, which hands lane
// i of each 16 the column i of the four rows that the 16 lanes read 8 bytes of each
__device__ inline f4 quad_cols(const float* t, int ld, int r0, int c0, int i, int g) {
  const float* p = t + (r0 + 4 * g) * ld + c0 + i;
  return f4{p[0], p[ld], p[2 * ld], p[3 * ld]};
}
__device__ inline bf4 quad_cols(const __bf16* t, int ld, int r0, int c0, int i, int g) {
  typedef __attribute__((address_space(3))) s4* lds_s4;
  const __bf16* p = t + (r0 + 4 * g + (i >> 2)) * ld + c0 + 4 * (i & 3);
  const s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
  return __builtin_bit_cast(bf4, r);
}

// Rows of consecutive chunks on their way from memory to LDS: C rows of COLS columns over NT threads. A
// thread keeps the address of each of its pieces and moves it on by a chunk with every fetch.
template <typename IO, int C, int COLS, int NT>
struct Rows {
  typedef Type<IO> Ty;
  static constexpr int VEC = Ty::VEC, PER_ROW = COLS / VEC, TOTAL = C * PER_ROW, N = (TOTAL + NT - 1) / NT;
  uint4 raw[N];
  const char* at[N];
  long step;  // bytes from chunk to chunk

  __device__ static int row_of(int u) { return (u * NT + (int)threadIdx.x) / PER_ROW; }
  __device__ static int col_of(int u) { return (u * NT + (int)threadIdx.x) % PER_ROW * VEC; }

  // place i of the sequence is slot i, or rows - 1 - i backward in time; the first fetch takes places i0..
  __device__ void init(const IO* p, long st, int i0, int rows, int reverse, int c0) {
    step = (reverse ? -C : C) * st * (long)sizeof(IO);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const long place = i0 + row_of(u);
      at[u] = reinterpret_cast<const char*>(p + (reverse ? rows - 1 - place : place) * st + c0 + col_of(u));
    }
  }
  // rows from n on and columns from `cols` (counted from c0) on are zero
  __device__ void fetch(int n, int cols) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      raw[u] = uint4{0, 0, 0, 0};
      if (row_of(u) < n && col_of(u) < cols) raw[u] = *reinterpret_cast<const uint4*>(at[u]);
      at[u] += step;
    }
  }
  __device__ void put(typename Ty::Lds* lds, int ld) const {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (TOTAL % NT == 0 || row_of(u) < C) Ty::to_lds(lds + row_of(u) * ld + col_of(u), raw[u]);
  }
};

template <int NK, int NV>
__device__ inline void multiply_out(f4 (&S)[NK][NV], float f) {
#pragma unroll
  for (int x = 0; x < NK; ++x)
#pragma unroll
    for (int y = 0; y < NV; ++y) S[x][y] *= f;
}

// OUT: with outputs; without, only the state that a segment of slots adds is formed (into ws).
template <typename IO, int NK, int NV, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW, NK >= 16 || NW == 1 ? 1 : 2) void chunks(const Args a) {
  typedef Type<IO> Ty;
  typedef typename Ty::Lds Lds;
  typedef typename Ty::Quad Quad;
  constexpr int C = Ty::C, NB = C / 16, NT = 64 * NW, DK = 16 * NK, SL = 16 * NV * NW;
  constexpr int LK = DK + Ty::LDPAD, LV = SL + Ty::LDPAD;
  __shared__ __align__(16) Lds qs[OUT ? C * LK : 1];
  __shared__ __align__(16) Lds ks[C * LK];
  __shared__ __align__(16) Lds vs[C * LV];

  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned id = blockIdx.x;
  const int slice = id % a.nslice;
  id /= a.nslice;
  const int nseg_here = OUT ? a.nseg : a.nseg - 1;  // without outputs the last segment has nothing to add
  const int seg = id % nseg_here;
  const long bh = id / nseg_here;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H);
  const int rows = row_count(a, b);
  const int first = seg * a.seg_len;
  const int end = min(rows, first + a.seg_len);
  const int c0 = slice * SL, col = c0 + wave * 16 * NV;  // first column of V: of the workgroup, of the wave

  const IO* q = static_cast<const IO*>(a.q) + b * a.sq.b + h * a.sq.h;
  const IO* k = static_cast<const IO*>(a.k) + b * a.sk.b + h * a.sk.h;
  const IO* v = static_cast<const IO*>(a.v) + b * a.sv.b + h * a.sv.h;
  IO* o = OUT ? static_cast<IO*>(a.o) + b * a.so.b + h * a.so.h : nullptr;

  f4 S[NK][NV];
#pragma unroll
  for (int x = 0; x < NK; ++x)
#pragma unroll
    for (int y = 0; y < NV; ++y) S[x][y] = f4{0.f, 0.f, 0.f, 0.f};

  const long states = (long)a.K * a.V;
  bool have = false;  // S is not all zero
  if (OUT) {
    const float* from = seg ? a.ws + (bh * (a.nseg - 1) + seg - 1) * states : a.init ? a.init + bh * states : nullptr;
    const int fk = seg ? a.V : a.init_k, fv = seg ? 1 : a.init_v;
    have = from != nullptr && (first < end || seg == 0);
    if (have) {
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int y = 0; y < NV; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kk = 16 * x + 4 * g + r, vv = col + 16 * y + i;
            if (kk < a.K && vv < a.V) S[x][y][r] = from[(long)kk * fk + (long)vv * fv];
          }
    }
  }

  const float g2 = a.log_decay[h] * 1.44269504088896340736f;
  const int e = a.reverse ? 0 : 1;
  // scores: same block (masked), next block; further blocks by d^16 each
  float wd[4], wo[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int s = 4 * g + r;
    wd[r] = i >= s ? pw(g2, i - s) * a.s_intra : 0.f;
    wo[r] = pw(g2, 16 + i - s) * a.s_intra;
  }
  float d16[NB];
#pragma unroll
  for (int x = 0; x < NB; ++x) d16[x] = pw(g2, 16 * x);
  const float rf = pw(g2, i + e) * a.s_inter;
  // A state that fades slowly is kept as S / d^m, m slots since it was last multiplied out: a chunk then adds
  // its keys and values by the weights d^-(m + 1 + j) and touches no element of S otherwise (multiplying S by
  // d^C per chunk took 512 of some 3,300 cycles of a chunk's issue, and rounded the weight of a far slot once
  // per chunk). It is multiplied out when d^m would leave 2^+-20. Where 2^-16 is passed within one chunk S is
  // multiplied by d^n for each, and the weights are d^(n-1-j).
  const bool slow = fabsf(g2) * C < 16.f;
  int m = 0;
  float wk[NB][4];
#pragma unroll
  for (int sb = 0; sb < NB; ++sb)
#pragma unroll
    for (int r = 0; r < 4; ++r) wk[sb][r] = slow ? pw(g2, -(16 * sb + 4 * g + r + e)) * a.s_kv : 0.f;

  Rows<IO, C, DK, NT> rq, rk;
  Rows<IO, C, SL, NT> rv;
  if (OUT) rq.init(q, a.sq.t, first, rows, a.reverse, 0);
  rk.init(k, a.sk.t, first, rows, a.reverse, 0);
  rv.init(v, a.sv.t, first, rows, a.reverse, c0);
  auto fetch = [&](int at) {
    const int n = min(C, end - at);
    if (OUT) rq.fetch(n, a.K);
    rk.fetch(n, a.K);
    rv.fetch(n, a.V - c0);
  };
  if (first < end) fetch(first);
  for (int at = first; at < end; at += C) {
    const int n = min(C, end - at);
    if (at != first) __syncthreads();  // the products of the chunk before have read their rows
    if (OUT) rq.put(qs, LK);
    rk.put(ks, LK);
    rv.put(vs, LV);
    __syncthreads();
    if (at + C < end) fetch(at + C);  // on their way while this chunk is computed

    Quad vf[NB][NV];
#pragma unroll
    for (int sb = 0; sb < NB; ++sb)
#pragma unroll
      for (int y = 0; y < NV; ++y) vf[sb][y] = quad_cols(vs, LV, 16 * sb, wave * 16 * NV + 16 * y, i, g);

    if (OUT) {
      const float dm = pw(g2, m);
      Quad sf[Ty::BF ? NK : 1][Ty::BF ? NV : 1];
      if constexpr (Ty::BF) {
        // the state enters this product rounded to bf16, the only place where it is: an error of at most
        // half a step of the output's own type on its share of the sum
#pragma unroll
        for (int x = 0; x < NK; ++x)
#pragma unroll
          for (int y = 0; y < NV; ++y) sf[x][y] = to_bf(S[x][y]);
      }
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) {
        if (16 * tb >= n) break;
        Quad qf[NK];
#pragma unroll
        for (int x = 0; x < NK; ++x) qf[x] = quad_rows(qs, LK, 16 * tb, 16 * x, i, g);
        f4 acc[NV];
#pragma unroll
        for (int y = 0; y < NV; ++y) acc[y] = f4{0.f, 0.f, 0.f, 0.f};
        if (have) {
          if constexpr (Ty::BF) {
#pragma unroll
            for (int x = 0; x < NK; x += 2)
#pragma unroll
              for (int y = 0; y < NV; ++y) acc[y] = mma32(sf[x][y], sf[x + 1][y], qf[x], qf[x + 1], acc[y]);
          } else {
#pragma unroll
            for (int x = 0; x < NK; ++x)
#pragma unroll
              for (int y = 0; y < NV; ++y) acc[y] = mma16(S[x][y], qf[x], acc[y]);
          }
          const float f = rf * d16[tb] * dm;
#pragma unroll
          for (int y = 0; y < NV; ++y) acc[y] *= f;
        }
        Quad pf[NB];
#pragma unroll
        for (int sb = 0; sb < NB; ++sb) {
          if (sb > tb) continue;
          f4 p = f4{0.f, 0.f, 0.f, 0.f};
          if constexpr (Ty::BF) {
#pragma unroll
            for (int x = 0; x < NK; x += 2)
              p = mma32(quad_rows(ks, LK, 16 * sb, 16 * x, i, g), quad_rows(ks, LK, 16 * sb, 16 * x + 16, i, g), qf[x], qf[x + 1], p);
          } else {
#pragma unroll
            for (int x = 0; x < NK; ++x) p = mma16(quad_rows(ks, LK, 16 * sb, 16 * x, i, g), qf[x], p);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = sb == tb ? (i >= 4 * g + r ? p[r] * wd[r] : 0.f) : p[r] * (wo[r] * d16[tb - sb - 1]);
          if constexpr (Ty::BF) {
            pf[sb] = to_bf(p);  // scores rounded to the tensors' type for the second product, as their sum will be
          } else {
            pf[sb] = p;
          }
        }
        if constexpr (Ty::BF) {
          const bf4 none = bf4{(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};
#pragma unroll
          for (int sb = 0; sb < NB; sb += 2) {
            if (sb > tb) continue;
#pragma unroll
            for (int y = 0; y < NV; ++y)
              acc[y] = mma32(vf[sb][y], sb + 1 <= tb ? vf[sb + 1][y] : none, pf[sb], sb + 1 <= tb ? pf[sb + 1] : none, acc[y]);
          }
        } else {
#pragma unroll
          for (int sb = 0; sb < NB; ++sb) {
            if (sb > tb) continue;
#pragma unroll
            for (int y = 0; y < NV; ++y) acc[y] = mma16(vf[sb][y], pf[sb], acc[y]);
          }
        }
        const int place = 16 * tb + i;
        if (place < n) {
          IO* po = o + (long)(a.reverse ? rows - 1 - (at + place) : at + place) * a.so.t;
#pragma unroll
          for (int y = 0; y < NV; ++y) {
            const int vv = col + 16 * y + 4 * g;
            if (a.vec_o && vv + 4 <= a.V) {
              Ty::store4(po + vv, acc[y]);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (vv + r < a.V) Ty::store(po + vv + r, acc[y][r]);
            }
          }
        }
      }
    }

    if (OUT && at + C >= end && !a.fin) break;  // nobody reads the state behind the last slot
    float w[NB][4];
    if (slow) {
      if (fabsf(g2) * (float)(m + C) > 20.f) {
        multiply_out(S, pw(g2, m));
        m = 0;
      }
      const float f = pw(g2, -m);
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
        for (int r = 0; r < 4; ++r) w[sb][r] = pw(g2, max(0, n - e - (16 * sb + 4 * g + r))) * a.s_kv;
    }
    have = true;
    if constexpr (Ty::BF) {
      // the decayed v in three bf16 terms (24 bits): the state is as exact as products of the tensors in fp32
#pragma unroll
      for (int sb = 0; sb < NB; sb += 2) {
        if (16 * sb >= n) break;
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
        for (int x = 0; x < NK; ++x) {
          const bf4 k0 = quad_cols(ks, LK, 16 * sb, 16 * x, i, g), k1 = quad_cols(ks, LK, 16 * sb + 16, 16 * x, i, g);
#pragma unroll
          for (int y = 0; y < NV; ++y) {
            S[x][y] = mma32(k0, k1, t2[0][y], t2[1][y], S[x][y]);
            S[x][y] = mma32(k0, k1, t1[0][y], t1[1][y], S[x][y]);
            S[x][y] = mma32(k0, k1, t0[0][y], t0[1][y], S[x][y]);
          }
        }
      }
    } else {
#pragma unroll
      for (int sb = 0; sb < NB; ++sb) {
        if (16 * sb >= n) break;
#pragma unroll
        for (int y = 0; y < NV; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) vf[sb][y][r] *= w[sb][r];
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          const f4 kq = quad_cols(ks, LK, 16 * sb, 16 * x, i, g);
#pragma unroll
          for (int y = 0; y < NV; ++y) S[x][y] = mma16(kq, vf[sb][y], S[x][y]);
        }
      }
    }
  }

  if (OUT) {
    // slots behind the sequence's end
    const int from = max(rows, first), to = min(a.T, first + a.seg_len);
    const int wide = min(a.V, c0 + SL) - c0;
    for (long at = (long)from * wide + threadIdx.x; at < (long)to * wide; at += NT)
      Ty::store(o + at / wide * a.so.t + c0 + at % wide, 0.f);
  }
  if (m) multiply_out(S, pw(g2, m));
  float* to = nullptr;
  int tk = a.V, tv = 1;
  if (OUT) {
    const int owner = rows > 0 ? (rows - 1) / a.seg_len : 0;
    if (a.fin && seg == owner) to = a.fin + bh * states, tk = a.fin_k, tv = a.fin_v;
  } else {
    to = a.ws + (bh * (a.nseg - 1) + seg) * states;
  }
  if (to) {
#pragma unroll
    for (int x = 0; x < NK; ++x)
#pragma unroll
      for (int y = 0; y < NV; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kk = 16 * x + 4 * g + r, vv = col + 16 * y + i;
          if (kk < a.K && vv < a.V) to[(long)kk * tk + (long)vv * tv] = S[x][y][r];
        }
  }
}

// Columns of V that a workgroup takes: 16 (one wave, as long as that wave can stage the rows of K in
// few loads), 64, or 128 as long as its share of the state leaves a wave registers to work with.
inline int slice_columns(int K, int V) { return V <= 16 && K <= 64 ? 16 : V <= 64 || K > 128 ? 64 : 128; }
inline int chunk_slots(int dtype) { return dtype == CET_BF16 ? Type<__bf16>::C : Type<float>::C; }

template <typename IO, int NK, bool OUT>
inline void launch_k(const Args& a, unsigned blocks, hipStream_t s) {
  const int cols = slice_columns(a.K, a.V);
  if (cols == 16) {
    if constexpr (NK <= 4) chunks<IO, NK, 1, 1, OUT><<<blocks, 64, 0, s>>>(a);
  } else if (cols == 64) {
    chunks<IO, NK, 1, 4, OUT><<<blocks, 256, 0, s>>>(a);
  } else {
    if constexpr (NK <= 8) chunks<IO, NK, 2, 4, OUT><<<blocks, 256, 0, s>>>(a);
  }
}

template <typename IO, bool OUT>
inline void launch(const Args& a, unsigned blocks, hipStream_t s) {
  if (!Type<IO>::BF && a.K <= 16)
    launch_k<IO, Type<IO>::BF ? 2 : 1, OUT>(a, blocks, s);
  else if (a.K <= 32)
    launch_k<IO, 2, OUT>(a, blocks, s);
  else if (a.K <= 64)
    launch_k<IO, 4, OUT>(a, blocks, s);
  else if (a.K <= 128)
    launch_k<IO, 8, OUT>(a, blocks, s);
  else
    launch_k<IO, 16, OUT>(a, blocks, s);
}

// one translation unit each
void launch_f32(const Args& a, bool out, unsigned blocks, hipStream_t s);
void launch_f16(const Args& a, bool out, unsigned blocks, hipStream_t s);
void launch_bf16(const Args& a, bool out, unsigned blocks, hipStream_t s);

}  // namespace la
}  // namespace cet
