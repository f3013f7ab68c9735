// Rotary positions: every pair (a, b) of the first R features of a head is turned by position * f[pair]
// and scaled by a gain,
//     (a, b) -> gain (a cos - b sin, a sin + b cos),
// pairs (j, j + R / 2) ("half") or (2j, 2j + 1) ("interleaved"); the other features pass through. The
// gradient is the turn by the opposite angle.
//
// HBM-bound: every element is read and written once, queries and keys in one launch. The angles are formed
// in fp64 (a position of a million at one radian per slot leaves fp32 no fraction of a turn worth having),
// reduced to an eighth of a turn, and only then rounded to fp32. One workgroup forms the cosines and sines
// of its slots once, in LDS, for all of its heads.
#include <algorithm>
#include <cmath>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "cet_internal.h"

namespace cet {
namespace {

// n / d for n < 2^31 by one multiplication
struct Div {
  unsigned d, mul, shift;
  explicit Div(unsigned d_) : d(d_), mul(0), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct RotArgs {
  const void *q, *k;
  void *qo, *ko;
  long qs[3], ks[3];  // sequence, slot, head
  const void* pos;
  const double* freq;
  long pos_b, pos_t;
  int pos64, B, T, Hq, Hk, D, pairs, tile, heads_per_wg, head_groups, turn_units;
  float gain, sign;
  Div per_seq, units, heads;  // slots of a sequence, units of a row, heads of a workgroup
};

typedef float v4 __attribute__((ext_vector_type(4)));

template <typename E, int VEC>
struct Vec {
  typedef E type __attribute__((ext_vector_type(VEC)));
  type v;
  __device__ void load(const E* p) { v = *reinterpret_cast<const type*>(p); }
  __device__ void store(E* p) const { *reinterpret_cast<type*>(p) = v; }
};
template <typename E>
struct Vec<E, 1> {
  E v[1];
  __device__ void load(const E* p) { v[0] = *p; }
  __device__ void store(E* p) const { *p = v[0]; }
};

// A unit of work is VEC pairs (half: two pieces of VEC features) or VEC / 2 pairs (interleaved: one
// piece; one pair where VEC is 1), or one piece of VEC features that only pass through.
template <typename E, int VEC, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a) {
  extern __shared__ float2 cs[];  // [tile][pairs]
  const unsigned group = blockIdx.x % a.head_groups;
  const long first = (long)(blockIdx.x / a.head_groups) * a.tile;
  const int slots = (int)min((long)a.tile, (long)a.B * a.T - first);
  for (int at = threadIdx.x; at < slots * a.pairs; at += 256) {
    const int s = at / a.pairs, j = at - s * a.pairs;
    const unsigned n = (unsigned)(first + s), b = a.per_seq.div(n), t = n - b * a.T;
    const long p = b * a.pos_b + t * a.pos_t;
    const double pos = a.pos64 ? (double)static_cast<const long*>(a.pos)[p] : (double)static_cast<const int*>(a.pos)[p];
    const double quarters = pos * a.freq[j] * 0.63661977236758134308;  // of a turn
    const double whole = rint(quarters);
    float sn, cn;
    sincospif((float)(quarters - whole) * 0.5f, &sn, &cn);
    const int quadrant = (int)(whole - 4.0 * floor(0.25 * whole));
    const float c = quadrant == 0 ? cn : quadrant == 1 ? -sn : quadrant == 2 ? -cn : sn;
    const float d = quadrant == 0 ? sn : quadrant == 1 ? cn : quadrant == 2 ? -sn : -cn;
    cs[at] = make_float2(c * a.gain, d * a.gain * a.sign);
  }
  __syncthreads();
  const int h0 = group * a.heads_per_wg, nh = min(a.heads_per_wg, a.Hq + a.Hk - h0);
  const unsigned total = (unsigned)slots * nh * a.units.d;
  for (unsigned at = threadIdx.x; at < total; at += 256) {
    const unsigned row = a.units.div(at), u = at - row * a.units.d;
    const unsigned s = nh == (int)a.heads.d ? a.heads.div(row) : row / nh;
    const int h = h0 + (int)(row - s * nh);
    const unsigned n = (unsigned)(first + s), b = a.per_seq.div(n), t = n - b * a.T;
    const bool is_q = h < a.Hq;
    const int hh = is_q ? h : h - a.Hq;
    const E* in = static_cast<const E*>(is_q ? a.q : a.k) + (is_q ? b * a.qs[0] + t * a.qs[1] + hh * a.qs[2] : b * a.ks[0] + t * a.ks[1] + hh * a.ks[2]);
    E* out = static_cast<E*>(is_q ? a.qo : a.ko) + ((long)n * (is_q ? a.Hq : a.Hk) + hh) * a.D;
    if ((int)u >= a.turn_units) {
      const int c = 2 * a.pairs + (int)(u - a.turn_units) * VEC;
      Vec<E, VEC> x;
      x.load(in + c);
      x.store(out + c);
    } else if (HALF || VEC == 1) {
      const int j = (int)u * VEC, pa = HALF ? j : 2 * j, pb = HALF ? j + a.pairs : 2 * j + 1;
      Vec<E, VEC> x, y, xo, yo;
      x.load(in + pa);
      y.load(in + pb);
      const float2* w = cs + s * a.pairs + j;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 r = w[e];
        const float p = (float)x.v[e], q = (float)y.v[e];
        xo.v[e] = (E)fmaf(p, r.x, -q * r.y);
        yo.v[e] = (E)fmaf(p, r.y, q * r.x);
      }
      xo.store(out + pa);
      yo.store(out + pb);
    } else {
      const int c = (int)u * VEC;
      Vec<E, VEC> x, xo;
      x.load(in + c);
      const float2* w = cs + s * a.pairs + c / 2;
#pragma unroll
      for (int e = 0; e + 1 < VEC; e += 2) {
        const float2 r = w[e / 2];
        const float p = (float)x.v[e], q = (float)x.v[e + 1];
        xo.v[e] = (E)fmaf(p, r.x, -q * r.y);
        xo.v[e + 1] = (E)fmaf(p, r.y, q * r.x);
      }
      xo.store(out + c);
    }
  }
}

template <typename E, int vec>
int launch(RotArgs a, int interleaved, hipStream_t s) {
  const int rest = a.D - 2 * a.pairs;
  a.turn_units = vec == 1 || !interleaved ? a.pairs / vec : 2 * a.pairs / vec;
  const int units = a.turn_units + rest / vec, heads = a.Hq + a.Hk;
  const long n = (long)a.B * a.T;
  // Slots per workgroup: four rounds of its threads, as long as that leaves two workgroups per CU; then
  // (few slots) heads are split too.
  long tile = std::max<long>(1, 1024 / ((long)units * heads));
  tile = std::min<long>(std::min<long>(tile, 8192 / (a.pairs * 8)), 16);
  while (tile > 1 && (n + tile - 1) / tile < 512) tile /= 2;
  a.tile = (int)tile;
  a.head_groups = 1;
  if ((n + tile - 1) / tile < 512) a.head_groups = (int)std::min<long>(heads, std::max<long>(1, std::min<long>(512 / n, (long)units * heads / 256)));
  a.heads_per_wg = (heads + a.head_groups - 1) / a.head_groups;
  a.head_groups = (heads + a.heads_per_wg - 1) / a.heads_per_wg;
  a.units = Div((unsigned)units);
  a.heads = Div((unsigned)a.heads_per_wg);
  const long blocks = (n + tile - 1) / tile * a.head_groups;
  if (blocks >= 1 << 24) return CET_ERR_UNSUPPORTED;  // a launch holds fewer than 2^32 threads
  const size_t lds = (size_t)tile * a.pairs * sizeof(float2);
  if (interleaved)
    rotary_kernel<E, vec, false><<<(unsigned)blocks, 256, lds, s>>>(a);
  else
    rotary_kernel<E, vec, true><<<(unsigned)blocks, 256, lds, s>>>(a);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

template <typename E>
int launch(const RotArgs& a, int interleaved, int vec, hipStream_t s) {
  if constexpr (sizeof(E) == 2)
    if (vec == 8) return launch<E, 8>(a, interleaved, s);
  return vec == 4 ? launch<E, 4>(a, interleaved, s) : vec == 2 ? launch<E, 2>(a, interleaved, s) : launch<E, 1>(a, interleaved, s);
}

}  // namespace
}  // namespace cet

using namespace cet;

extern "C" int cet_rotary(const cet_rotary_desc* d, const void* q, const void* k, const void* positions,
                          const double* inv_freq, int inverse, void* q_out, void* k_out, void* stream) {
  if (!d || d->dtype < CET_F32 || d->dtype > CET_F16 || d->B < 0 || d->T < 0 || d->Hq < 0 || d->Hk < 0 || d->D < 1 ||
      d->pairs < 1 || 2L * d->pairs > d->D || !std::isfinite(d->gain) || d->interleaved < 0 || d->interleaved > 1)
    return CET_ERR_INVALID_ARG;
  if (d->D > 1024 || d->Hq > 65536 || d->Hk > 65536 || (double)d->B * d->T > 2e9) return CET_ERR_UNSUPPORTED;
  if ((long)d->B * d->T == 0 || d->Hq + d->Hk == 0) return CET_OK;
  if (!positions || !inv_freq || (d->Hq && (!q || !q_out)) || (d->Hk && (!k || !k_out))) return CET_ERR_INVALID_ARG;
  RotArgs a{q, k, q_out, k_out, {d->q[0], d->q[1], d->q[2]}, {d->k[0], d->k[1], d->k[2]}, positions, inv_freq, d->pos[0], d->pos[1],
            d->positions64, d->B, d->T, d->Hq, d->Hk, d->D, d->pairs, 1, 1, 1, 1, d->gain, inverse ? -1.f : 1.f, Div((unsigned)d->T), Div(1), Div(1)};
  const int size = d->dtype == CET_F32 ? 4 : 2;
  uintptr_t at = 0;
  long strides = 0;
  if (d->Hq) at |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out), strides |= d->q[0] | d->q[1] | d->q[2];
  if (d->Hk) at |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out), strides |= d->k[0] | d->k[1] | d->k[2];
  // The widest pieces of up to 16 bytes that every row and both halves of the turned part are whole numbers of and
  // start on (22 x 3036 slots, 6 heads of 48, 6 pairs in fp16: 31 us by 4 bytes, 51 by single values; 20 x 1772 slots,
  // 7 heads of 80, 20 pairs in bf16: 19 us by 8 bytes, 47).
  int vec = 16 / size;
  while (vec > 1 && (at % (vec * size) || strides % vec || d->D % vec || (d->interleaved ? 2 * d->pairs : d->pairs) % vec)) vec /= 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == CET_F32) return launch<float>(a, d->interleaved, vec, s);
  if (d->dtype == CET_F16) return launch<_Float16>(a, d->interleaved, vec, s);
  return launch<__bf16>(a, d->interleaved, vec, s);
}
