// Linear attention with a decay per head: entry points, the join of the segments' states, the copy of
// operands that wide loads cannot take, and the form for single slots. The chunk kernels are in linattn.h.
#include <algorithm>
#include <cmath>

#include "linattn.h"

namespace cet {
namespace la {
namespace {

constexpr size_t align_up(size_t n) { return (n + 255) & ~(size_t)255; }
constexpr int elem_bytes(int dtype) { return dtype == CET_F32 ? 4 : 2; }

// ws[bh][s] holds what segment s adds to the state; afterwards the state behind segment s (the one that
// segment s + 1 starts from). A thread takes W state elements, segments in order; blockIdx.y is the head.
template <int W>
__global__ __launch_bounds__(256) void join_segments(const Args a) {
  typedef float vec __attribute__((ext_vector_type(W)));
  const int states = a.K * a.V, e = (blockIdx.x * 256 + threadIdx.x) * W;
  if (e >= states) return;
  const long bh = blockIdx.y;
  const float d = pw(a.log_decay[bh % a.H] * 1.44269504088896340736f, a.seg_len);
  vec cur = {};
  if (a.init) cur = *reinterpret_cast<const vec*>(a.init + bh * states + e);
  float* p = a.ws + bh * (a.nseg - 1) * states + e;
  for (int s0 = 0; s0 < a.nseg - 1; s0 += 8) {
    vec add[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) add[j] = *reinterpret_cast<const vec*>(p + (long)min(s0 + j, a.nseg - 2) * states);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cur = cur * d + add[j];
      if (s0 + j < a.nseg - 1) *reinterpret_cast<vec*>(p + (long)(s0 + j) * states) = cur;
    }
  }
}

// [B,T,H,D] with any strides -> contiguous with D rounded up to a multiple of 16 bytes, zeros behind D. Slots at and behind a
// sequence's length are not read, here or by the kernels that take the copy, and nothing is written for them.
template <typename E>
__global__ __launch_bounds__(256) void pack_rows(const E* __restrict__ src, Strides s, E* __restrict__ dst, const void* lengths,
                                                 int lengths64, int T, int H, int D, int per_row, long total) {
  constexpr int VEC = 16 / sizeof(E);
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long)gridDim.x * 256) {
    const int c = (int)(at % per_row) * VEC;
    const long row = at / per_row, h = row % H, t = row / H % T, b = row / H / T;
    if (t >= row_count(lengths, lengths64, T, (int)b)) continue;
    const E* p = src + b * s.b + t * s.t + h * s.h;
    E e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = c + j < D ? p[c + j] : E(0);
    uint4 raw;
    __builtin_memcpy(&raw, e, 16);
    reinterpret_cast<uint4*>(dst)[at] = raw;
  }
}

// d = exp(log_decay) in two parts: a state that is multiplied slot by slot would hold a rounding of d raised to the
// number of slots, 1e-4 of a weight 4,000 slots back.
__device__ inline void decay_of(float log_decay, float& hi, float& lo) {
  const double d = exp((double)log_decay);
  hi = (float)d;
  lo = (float)(d - (double)hi);
}

// Small heads (K and V up to 16) on many sequences, the predictors' own batches: a lane takes one column of V
// of one head of one sequence, holds that column's state in K registers and walks the slots one by one; lanes of
// a head read the same q and k. 100 instructions a head and 25 slots, where a wave with matrix instructions on a
// head of its own took 1,180 and was bound by issuing them (4096 x 8 heads of 8, 25 slots, fp32: 67 us).
template <typename IO, int KP>
__global__ __launch_bounds__(256, 4) void columns(const Args a, int step_q, int step_k) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  const bool live = c < (long)a.B * a.H * a.V;
  const unsigned bh = live ? (unsigned)(c / a.V) : 0;
  const int vv = live ? (int)(c - (long)bh * a.V) : 0, b = bh / a.H, h = bh - b * a.H;
  const int n = live ? row_count(a, b) : 0;
  const long states = (long)a.K * a.V;
  float S[KP];
#pragma unroll
  for (int k = 0; k < KP; ++k) S[k] = live && a.init && k < a.K ? a.init[bh * states + (long)k * a.init_k + (long)vv * a.init_v] : 0.f;
  float d, d_lo;
  decay_of(a.log_decay[h], d, d_lo);
  const long from = a.reverse ? n - 1 : 0, dir = a.reverse ? -1 : 1;
  const IO* q = static_cast<const IO*>(a.q) + b * a.sq.b + h * a.sq.h + from * a.sq.t;
  const IO* k = static_cast<const IO*>(a.k) + b * a.sk.b + h * a.sk.h + from * a.sk.t;
  const IO* v = static_cast<const IO*>(a.v) + b * a.sv.b + h * a.sv.h + from * a.sv.t + vv;
  IO* const o0 = static_cast<IO*>(a.o) + b * a.so.b + h * a.so.h + vv;
  IO* o = o0 + from * a.so.t;
  auto row = [&](float (&x)[KP], const IO* p, int step) {
    typedef typename Type<IO>::V4 V4;
#pragma unroll
    for (int j = 0; j < KP; j += 4) {
      if (step == 4) {
        V4 y = {};
        if (j < a.K) y = *reinterpret_cast<const V4*>(p + j);  // K is a multiple of four
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j + r] = (float)y[r];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j + r] = j + r < a.K ? (float)p[j + r] : 0.f;
      }
    }
  };
  float qn[KP], kn[KP], vn = 0.f;  // the next slot's, on their way
  if (n > 0) {
    row(qn, q, step_q);
    row(kn, k, step_k);
    vn = (float)*v;
  }
  for (int t = 0; t < n; ++t) {
    float qr[KP], kr[KP];
    const float vr = vn * a.s_kv;
#pragma unroll
    for (int j = 0; j < KP; ++j) qr[j] = qn[j], kr[j] = kn[j];
    if (t + 1 < n) {
      q += dir * a.sq.t, k += dir * a.sk.t, v += dir * a.sv.t;
      row(qn, q, step_q);
      row(kn, k, step_k);
      vn = (float)*v;
    }
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      S[j] = a.reverse ? fmaf(kr[j], vr, S[j]) : fmaf(S[j], d, fmaf(S[j], d_lo, kr[j] * vr));
      sum[j & 3] = fmaf(qr[j], S[j], sum[j & 3]);
    }
    if (a.reverse) {
#pragma unroll
      for (int j = 0; j < KP; ++j) S[j] = fmaf(S[j], d, S[j] * d_lo);
    }
    *o = (IO)(((sum[0] + sum[1]) + (sum[2] + sum[3])) * a.s_inter);
    o += dir * a.so.t;
  }
  if (!live) return;
  for (long t = n; t < a.T; ++t) o0[t * a.so.t] = (IO)0.f;
  if (a.fin)
#pragma unroll
    for (int j = 0; j < KP; ++j)
      if (j < a.K) a.fin[bh * states + (long)j * a.V + vv] = S[j];
}

// One slot. A workgroup takes 4 TX (or TX, where rows of V are no multiple of four) columns of one head's
// state of one stream; the rows of K are spread over TY = 256 / TX threads per column group, whose partial
// sums of q S are added over the lanes of a wave and then over the four waves in LDS.
template <typename IO>
struct Step {
  const IO *q, *k, *v;
  long qb, qh, kb, kh, vb, vh;
  const float* log_decay;
  const float* in;
  float* out;
  const void* slots;
  const int* owner;  // first stream of the call in each row of the pool, where a table was made (else nullptr)
  IO* o;
  int B, H, K, V, rows, slots64, nslice;
  float scale;
};

__device__ inline long slot_of(const void* slots, int wide, int b) {
  return wide ? static_cast<const long*>(slots)[b] : (long)static_cast<const int*>(slots)[b];
}

// owner[row] = the first stream of the call whose slot is that row, for the rows that are some stream's. The first
// launch clears these, the second takes the least; the rest of the table is neither written nor read.
template <bool CLAIM>
__global__ __launch_bounds__(256) void claim_rows(const void* __restrict__ slots, int wide, int B, int rows, int* owner) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const long row = slot_of(slots, wide, b);
  if (row < 0 || row >= rows) return;
  if (CLAIM)
    atomicMin(owner + row, b);
  else
    owner[row] = 0x7fffffff;
}

template <typename IO, int TX, int W>
__global__ __launch_bounds__(256) void step(const Step<IO> a) {
  constexpr int TY = 256 / TX, COLS = TX * W;
  __shared__ float ks[256], qs[256], part[4][COLS];
  const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
  unsigned id = blockIdx.x;
  const int c = (int)(id % a.nslice) * COLS + tx * W;
  id /= a.nslice;
  const int h = (int)(id % a.H), b = (int)(id / a.H);
  long row = b;
  float idle = 0.f;
  bool live = true;
  if (a.slots) {
    row = slot_of(a.slots, a.slots64, b);
    // a slot that an earlier stream of this call has: two workgroups would update one state
    bool twice = false;
    if (a.owner) {
      twice = row >= 0 && row < a.rows && a.owner[row] != b;
    } else {
      if (row >= 0 && row < a.rows)
        for (int e = tid; e < b; e += 256) twice |= slot_of(a.slots, a.slots64, e) == row;
      twice = __syncthreads_or(twice);
    }
    live = row >= 0 && row < a.rows && !twice;
    if (row >= 0 && !live) idle = __builtin_nanf("");
  }
  if (live) {
    if (tid < a.K) {
      ks[tid] = (float)a.k[b * a.kb + h * a.kh + tid];
      qs[tid] = (float)a.q[b * a.qb + h * a.qh + tid] * a.scale;
    }
    float d, d_lo;
    decay_of(a.log_decay[h], d, d_lo);
    float v[W], acc[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      v[w] = c + w < a.V ? (float)a.v[b * a.vb + h * a.vh + c + w] : 0.f;
      acc[w] = 0.f;
    }
    __syncthreads();
    const long base = (row * a.H + h) * a.K * a.V + c;
    if (c < a.V) {  // V is a multiple of W
#pragma unroll 4
      for (int x = ty; x < a.K; x += TY) {
        const float* p = a.in + base + (long)x * a.V;
        float* to = a.out + base + (long)x * a.V;
        float s[W];
        if constexpr (W == 4) {
          *reinterpret_cast<f4*>(s) = *reinterpret_cast<const f4*>(p);
        } else {
          s[0] = *p;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          s[w] = fmaf(s[w], d, fmaf(s[w], d_lo, ks[x] * v[w]));
          acc[w] = fmaf(qs[x], s[w], acc[w]);
        }
        if constexpr (W == 4) {
          *reinterpret_cast<f4*>(to) = *reinterpret_cast<f4*>(s);
        } else {
          *to = s[0];
        }
      }
    }
#pragma unroll
    for (int off = TX; off < 64; off *= 2)
#pragma unroll
      for (int w = 0; w < W; ++w) acc[w] += __shfl_xor(acc[w], off);
    if ((tid & 63) < TX)
#pragma unroll
      for (int w = 0; w < W; ++w) part[tid >> 6][tx * W + w] = acc[w];
  }
  __syncthreads();
  const int first = (int)(blockIdx.x % a.nslice) * COLS;
  for (int x = tid; x < COLS; x += 256)
    if (first + x < a.V) {
      const float r = live ? part[0][x] + part[1][x] + part[2][x] + part[3][x] : idle;
      a.o[((long)b * a.H + h) * a.V + first + x] = (IO)r;
    }
}

int cu_count() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
    return 256;
  return n;
}

bool by_columns(const cet_linattn_desc& d);

struct Operand {
  const void* p;
  Strides s;
  int D;
  size_t copy = 0;  // bytes of its packed copy, 0 where it is read in place

  Operand(const void* ptr, const int64_t* st, int D, const cet_linattn_desc& d) : p(ptr), s{st[0], st[1], st[2]}, D(D) {
    const int vec = 16 / elem_bytes(d.dtype);
    const bool wide = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && D % vec == 0 && (s.b % vec == 0 || d.B == 1) &&
                      (s.t % vec == 0 || d.T == 1) && (s.h % vec == 0 || d.H == 1);
    if (!wide && !by_columns(d)) copy = align_up((size_t)d.B * d.T * d.H * ((D + vec - 1) / vec) * 16);
  }
  int pack(const cet_linattn_desc& d, const void* lengths, char*& ws, hipStream_t stream) {
    if (!copy) return CET_OK;
    const int vec = 16 / elem_bytes(d.dtype), per_row = (D + vec - 1) / vec;
    const long total = (long)d.B * d.T * d.H * per_row;
    const unsigned blocks = (unsigned)std::min<long>((total + 255) / 256, 1 << 20);
    if (d.dtype == CET_F32)
      pack_rows<uint32_t><<<blocks, 256, 0, stream>>>(static_cast<const uint32_t*>(p), s, reinterpret_cast<uint32_t*>(ws), lengths, d.lengths64, d.T, d.H, D, per_row, total);
    else
      pack_rows<uint16_t><<<blocks, 256, 0, stream>>>(static_cast<const uint16_t*>(p), s, reinterpret_cast<uint16_t*>(ws), lengths, d.lengths64, d.T, d.H, D, per_row, total);
    CET_HIP(hipGetLastError());
    const long row = (long)per_row * vec;
    p = ws;
    s = Strides{(long)d.T * d.H * row, d.H * row, row};
    ws += copy;
    return CET_OK;
  }
};

// How the time axis is cut: into segments where heads, sequences and slices alone are fewer than two workgroups
// per CU, none shorter than 128 slots, as many as make the workgroups' rounds over the chip times the length of a
// segment least (forward and gradients in us, bf16, 128 x 128, 16 heads x 2048 slots, 12 sequences: two segments in one round 197 and
// 389, three in two rounds 210 and 372; 8 sequences: 128 and 255, three 137 and 267, as for four workgroups per CU 158 and
// 290). Forward and backward cut it alike, and share the segments' states.
struct Cut {
  int nseg, seg_len;
  size_t states;  // bytes of the states between segments, K x V per head
};

// A lane per column: small heads, as long as there are waves for two to every SIMD or too few slots to cut.
bool by_columns(const cet_linattn_desc& d) {
  return d.K <= 16 && d.V <= 16 && (d.T <= OUT_SLOTS || (long)d.B * d.H * std::min(d.K, d.V) >= 64L * 8 * cu_count());
}

Cut cut(const cet_linattn_desc& d) {
  if (by_columns(d)) return Cut{1, std::max(d.T, 1), 0};
  const int cols = slice_columns(d.K, d.V);
  const long tasks = (long)d.B * d.H * ((d.V + cols - 1) / cols), chunks = (d.T + STATE_SLOTS - 1) / STATE_SLOTS;
  const long room = (long)cu_count() * workgroups_per_cu(d.dtype, d.K, d.V);
  long per = std::max<long>(chunks, 1), best = (tasks + room - 1) / room * per;
  for (const long most : {tasks ? room / tasks : 1, tasks ? (room + tasks - 1) / tasks : 1}) {  // within a round, and one more
    const long n = std::min(most, chunks / 2);
    if (n < 2) continue;
    const long p = (chunks + n - 1) / n, cost = (tasks * ((chunks + p - 1) / p) + room - 1) / room * p;
    if (cost < best) per = p, best = cost;
  }
  Cut c;
  c.seg_len = (int)(per * STATE_SLOTS);
  c.nseg = (int)std::max<long>((chunks + per - 1) / per, 1);
  c.states = c.nseg > 1 ? align_up((size_t)d.B * d.H * (c.nseg - 1) * d.K * d.V * sizeof(float)) : 0;
  return c;
}

// A launch of passes of one shape; `nseg`: segments that have work.
int launch(Passes& p, bool out, int nseg, int dtype, hipStream_t s) {
  const Args& a = p.a[0];
  const int cols = slice_columns(a.K, a.V);
  for (int i = 0; i < p.n; ++i) p.a[i].nslice = (a.V + cols - 1) / cols;
  const unsigned blocks = (unsigned)((long)a.B * a.H * nseg * a.nslice * p.n);
  if (dtype == CET_F32)
    launch_f32(p, out, blocks, s);
  else if (dtype == CET_F16)
    launch_f16(p, out, blocks, s);
  else
    launch_bf16(p, out, blocks, s);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

// The states between segments from (k, v) into ws, as K x V.
int segment_states(Args a, const Cut& c, int dtype, hipStream_t s) {
  if (c.nseg == 1) return CET_OK;
  a.nseg = c.nseg, a.seg_len = c.seg_len;
  a.ws_k = a.V, a.ws_v = 1;
  Passes p{{a}, 1};
  if (const int rc = launch(p, false, c.nseg - 1, dtype, s)) return rc;
  const unsigned heads = (unsigned)((long)a.B * a.H), states = (unsigned)(a.K * a.V);
  if (states % 4 == 0 && (reinterpret_cast<uintptr_t>(a.init) & 15) == 0)
    join_segments<4><<<dim3((states / 4 + 255) / 256, heads), 256, 0, s>>>(a);
  else
    join_segments<1><<<dim3((states + 255) / 256, heads), 256, 0, s>>>(a);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

template <typename IO>
void launch_columns(const Args& a, hipStream_t s) {
  const auto step = [&](const void* p, const Strides& t) {
    return a.K % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(IO)) == 0 && (t.b | t.t | t.h) % 4 == 0 ? 4 : 1;
  };
  const unsigned blocks = (unsigned)(((long)a.B * a.H * a.V + 255) / 256);
  if (a.K <= 8)
    columns<IO, 8><<<blocks, 256, 0, s>>>(a, step(a.q, a.sq), step(a.k, a.sk));
  else
    columns<IO, 16><<<blocks, 256, 0, s>>>(a, step(a.q, a.sq), step(a.k, a.sk));
}

// Passes of the recurrence, segments from their states in ws (`transposed`: of the operands' roles exchanged). Those of
// one shape share a launch.
double threads(const Args& a, int nseg) { return (double)a.B * a.H * nseg * ((a.V + 63) / 64) * 512; }  // at most
struct Run {
  Args a;
  bool transposed;
};
int run(Run* r, int n, const Cut& c, bool columns, int dtype, hipStream_t s) {
  Passes p{};
  for (int i = 0; i < n; ++i) {
    Args& a = r[i].a;
    a.nseg = c.nseg, a.seg_len = c.seg_len;
    a.ws_k = a.init_k = r[i].transposed ? 1 : a.V;
    a.ws_v = a.init_v = r[i].transposed ? a.K : 1;
    a.vec_o = a.V % 4 == 0 && (reinterpret_cast<uintptr_t>(a.o) & 15) == 0;
    if (columns) {
      if (dtype == CET_F32)
        launch_columns<float>(a, s);
      else if (dtype == CET_F16)
        launch_columns<_Float16>(a, s);
      else
        launch_columns<__bf16>(a, s);
      CET_HIP(hipGetLastError());
      continue;
    }
    p.a[p.n++] = a;
    if (i + 1 < n && alike(dtype, a, r[i + 1].a) && threads(a, c.nseg) * (p.n + 1) < 4294967296.) continue;
    if (const int rc = launch(p, true, c.nseg, dtype, s)) return rc;
    p.n = 0;
  }
  return CET_OK;
}

bool bad_desc(const cet_linattn_desc* d) {
  return !d || d->dtype < CET_F32 || d->dtype > CET_F16 || d->B < 0 || d->T < 0 || d->H < 0 || d->K < 1 || d->V < 1 ||
         d->T > (1 << 30) || !std::isfinite(d->scale);
}
// (a launch holds fewer than 2^32 threads: at most 512 for each head of each sequence and 64 columns)
bool too_large(const cet_linattn_desc& d) {
  return d.K > 256 || d.V > 256 || (double)d.B * d.H * ((std::max(d.K, d.V) + 63) / 64) > (1 << 22);
}
Strides contiguous(const cet_linattn_desc& d, int D) { return Strides{(long)d.T * d.H * D, (long)d.H * D, D}; }

template <typename IO, int W>
void launch_step(const Step<IO>& a0, int cus, hipStream_t s) {
  Step<IO> a = a0;
  const long heads = (long)a.B * a.H;
  // columns in as few workgroups as keep every CU at two or more
  int tx = 64;
  while (tx > 4 && (tx * W / 2 >= a.V || heads * ((a.V + tx * W - 1) / (tx * W)) < 2L * cus)) tx /= 2;
  a.nslice = (a.V + tx * W - 1) / (tx * W);
  const unsigned blocks = (unsigned)(heads * a.nslice);
  switch (tx) {
    case 64: step<IO, 64, W><<<blocks, 256, 0, s>>>(a); break;
    case 32: step<IO, 32, W><<<blocks, 256, 0, s>>>(a); break;
    case 16: step<IO, 16, W><<<blocks, 256, 0, s>>>(a); break;
    case 8: step<IO, 8, W><<<blocks, 256, 0, s>>>(a); break;
    default: step<IO, 4, W><<<blocks, 256, 0, s>>>(a);
  }
}

template <typename IO>
void run_step(int B, int H, int K, int V, const int64_t* qs, const int64_t* ks, const int64_t* vs, const void* q,
              const void* k, const void* v, const float* log_decay, float scale, const float* in, float* out, int rows,
              const void* slots, int slots64, const int* owner, void* o, hipStream_t s) {
  const Step<IO> a{static_cast<const IO*>(q), static_cast<const IO*>(k), static_cast<const IO*>(v), qs[0], qs[1], ks[0], ks[1],
                   vs[0], vs[1], log_decay, in, out, slots, owner, static_cast<IO*>(o), B, H, K, V, rows, slots64, 1, scale};
  const bool wide = V % 4 == 0 && ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (wide)
    launch_step<IO, 4>(a, cu_count(), s);
  else
    launch_step<IO, 1>(a, cu_count(), s);
}

// Streams up to which every workgroup looks for its slot among those before it; for more a table of the rows' owners is
// made first, by two launches. (Without slots, looking, with the table: 1024 streams of 2 heads of 16 x 16 4.9, 6.3, 8.8 us; 1024 of 8
// heads of 128 x 128 209, 225, 229; 2048 of 8 of 64 x 64 87, 116, 104; 4096 197, 256, 226; 262,144 of one of 8 x 8 a call 282, 14,490, 366.)
constexpr int FEW_STREAMS = 1024;

int step_call(int dtype, int B, int H, int K, int V, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
              const void* q, const void* k, const void* v, const float* log_decay, float scale, const float* state_in,
              float* state_out, int rows, const void* slots, int slots64, int* owner, void* o, hipStream_t s) {
  if (dtype < CET_F32 || dtype > CET_F16 || B < 0 || H < 0 || K < 1 || V < 1 || rows < 0 || !std::isfinite(scale))
    return CET_ERR_INVALID_ARG;
  if (K > 256 || V > 256 || (double)B * H > (1 << 21)) return CET_ERR_UNSUPPORTED;
  if ((long)B * H == 0) return CET_OK;
  if (!q_strides || !k_strides || !v_strides || !q || !k || !v || !log_decay || !o) return CET_ERR_INVALID_ARG;
  if (rows > 0 && (!state_in || !state_out)) return CET_ERR_INVALID_ARG;
  if (slots ? state_in != state_out : rows < B) return CET_ERR_INVALID_ARG;
  const uintptr_t a = reinterpret_cast<uintptr_t>(state_in), z = reinterpret_cast<uintptr_t>(state_out);
  const uintptr_t bytes = (uintptr_t)B * H * K * V * sizeof(float);
  if (a != z && (a < z ? z - a : a - z) < bytes) return CET_ERR_INVALID_ARG;  // half overlapping
  if (owner) {
    const unsigned blocks = (unsigned)((B + 255) / 256);
    claim_rows<false><<<blocks, 256, 0, s>>>(slots, slots64, B, rows, owner);
    CET_HIP(hipGetLastError());
    claim_rows<true><<<blocks, 256, 0, s>>>(slots, slots64, B, rows, owner);
    CET_HIP(hipGetLastError());
  }
  if (dtype == CET_F32)
    run_step<float>(B, H, K, V, q_strides, k_strides, v_strides, q, k, v, log_decay, scale, state_in, state_out, rows, slots, slots64, owner, o, s);
  else if (dtype == CET_F16)
    run_step<_Float16>(B, H, K, V, q_strides, k_strides, v_strides, q, k, v, log_decay, scale, state_in, state_out, rows, slots, slots64, owner, o, s);
  else
    run_step<__bf16>(B, H, K, V, q_strides, k_strides, v_strides, q, k, v, log_decay, scale, state_in, state_out, rows, slots, slots64, owner, o, s);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

}  // namespace
}  // namespace la
}  // namespace cet

using namespace cet;
using namespace cet::la;

extern "C" {

size_t cet_linear_attention_states(const cet_linattn_desc* d) {
  return bad_desc(d) || too_large(*d) ? 0 : cut(*d).states;
}

size_t cet_linear_attention_workspace(const cet_linattn_desc* d, const void* q, const void* k, const void* v,
                                      const void* d_o, int backward) {
  if (bad_desc(d) || too_large(*d)) return 0;
  size_t n = Operand(q, d->q, d->K, *d).copy + Operand(k, d->k, d->K, *d).copy + Operand(v, d->v, d->V, *d).copy;
  if (backward) n += Operand(d_o, d->d_o, d->V, *d).copy;
  return n + cut(*d).states * (backward ? 2 : 1);
}

int cet_linear_attention(const cet_linattn_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                         const float* initial, const void* lengths, void* o, float* final_state, float* states,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_desc(d)) return CET_ERR_INVALID_ARG;
  if (too_large(*d)) return CET_ERR_UNSUPPORTED;
  if ((long)d->B * d->H == 0) return CET_OK;
  if (!log_decay || (d->T > 0 && (!q || !k || !v || !o))) return CET_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(states) | reinterpret_cast<uintptr_t>(initial)) & 15)
    return CET_ERR_INVALID_ARG;
  const size_t need = cet_linear_attention_workspace(d, q, k, v, nullptr, 0) - (states ? cut(*d).states : 0);
  if (need > workspace_bytes || (need && !workspace)) return CET_ERR_INVALID_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  Operand oq(q, d->q, d->K, *d), ok(k, d->k, d->K, *d), ov(v, d->v, d->V, *d);
  for (Operand* x : {&oq, &ok, &ov})
    if (const int rc = x->pack(*d, lengths, ws, s)) return rc;
  const Cut c = cut(*d);
  const bool columns = by_columns(*d);
  Args a{};
  a.q = oq.p, a.k = ok.p, a.v = ov.p, a.o = o;
  a.sq = oq.s, a.sk = ok.s, a.sv = ov.s, a.so = contiguous(*d, d->V);
  a.init = initial, a.fin = final_state;
  a.log_decay = log_decay, a.lengths = lengths, a.lengths64 = d->lengths64;
  a.ws = states ? states : reinterpret_cast<float*>(ws);
  a.B = d->B, a.T = d->T, a.H = d->H, a.K = d->K, a.V = d->V;
  a.s_inter = a.s_intra = d->scale, a.s_kv = 1.f;
  if (const int rc = segment_states(a, c, d->dtype, s)) return rc;
  Run r{a, false};
  return run(&r, 1, c, columns, d->dtype, s);
}

int cet_linear_attention_backward(const cet_linattn_desc* d, const void* q, const void* k, const void* v,
                                  const float* log_decay, const float* initial, const void* lengths, const float* states,
                                  const void* d_o, const float* d_final, void* dq, void* dk, void* dv,
                                  float* d_initial, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_desc(d)) return CET_ERR_INVALID_ARG;
  if (too_large(*d)) return CET_ERR_UNSUPPORTED;
  if ((long)d->B * d->H == 0) return CET_OK;
  if (!log_decay || (d->T > 0 && (!q || !k || !v || !d_o || !dq || !dk || !dv))) return CET_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(states) | reinterpret_cast<uintptr_t>(initial) |
       reinterpret_cast<uintptr_t>(d_final)) & 15)
    return CET_ERR_INVALID_ARG;
  const size_t need = cet_linear_attention_workspace(d, q, k, v, d_o, 1) - (states ? cut(*d).states : 0);
  if (need > workspace_bytes || (need && !workspace)) return CET_ERR_INVALID_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  Operand oq(q, d->q, d->K, *d), ok(k, d->k, d->K, *d), ov(v, d->v, d->V, *d), og(d_o, d->d_o, d->V, *d);
  for (Operand* x : {&oq, &ok, &ov, &og})
    if (const int rc = x->pack(*d, lengths, ws, s)) return rc;
  const Cut c = cut(*d);
  const bool columns = by_columns(*d);
  float* const forward = states ? const_cast<float*>(states) : reinterpret_cast<float*>(ws);  // only read where given
  float* const back = reinterpret_cast<float*>(ws + (states ? 0 : c.states));
  Args a{};
  a.log_decay = log_decay, a.lengths = lengths, a.lengths64 = d->lengths64;
  a.B = d->B, a.T = d->T, a.H = d->H;
  a.so = contiguous(*d, d->K);
  a.ws = forward;
  a.init = initial;
  if (!states) {
    a.k = ok.p, a.sk = ok.s, a.v = ov.p, a.sv = ov.s;
    a.K = d->K, a.V = d->V, a.s_kv = 1.f;
    if (const int rc = segment_states(a, c, d->dtype, s)) return rc;
  }
  Run r[3];
  // dq: (do, v, k) forward in time, states transposed
  a.q = og.p, a.sq = og.s, a.k = ov.p, a.sk = ov.s, a.v = ok.p, a.sv = ok.s;
  a.o = dq;
  a.K = d->V, a.V = d->K;
  a.s_inter = a.s_intra = d->scale, a.s_kv = 1.f;
  r[0] = Run{a, true};
  // the gradients of the states, backward in time, which the two other passes share
  a.ws = back;
  a.init = d_final;
  a.reverse = 1, a.s_inter = 1.f, a.s_intra = a.s_kv = d->scale;
  a.k = oq.p, a.sk = oq.s, a.v = og.p, a.sv = og.s;
  a.K = d->K, a.V = d->V;
  if (const int rc = segment_states(a, c, d->dtype, s)) return rc;
  // dk: (v, do, q) backward in time, states transposed
  a.q = ov.p, a.sq = ov.s, a.k = og.p, a.sk = og.s, a.v = oq.p, a.sv = oq.s;
  a.o = dk;
  a.K = d->V, a.V = d->K;
  r[1] = Run{a, true};
  // dv: (k, q, do) backward in time; the carry at the end is the gradient of the first state
  a.q = ok.p, a.sq = ok.s, a.k = oq.p, a.sk = oq.s, a.v = og.p, a.sv = og.s;
  a.o = dv, a.so = contiguous(*d, d->V);
  a.K = d->K, a.V = d->V;
  a.fin = d_initial;
  r[2] = Run{a, false};
  return run(r, 3, c, columns, d->dtype, s);
}

int cet_linear_attention_step(int dtype, int B, int H, int K, int V, const int64_t* q_strides, const int64_t* k_strides,
                              const int64_t* v_strides, const void* q, const void* k, const void* v,
                              const float* log_decay, float scale, const float* state_in, float* state_out, int rows,
                              const void* slots, int slots64, void* o, void* stream) {
  return step_call(dtype, B, H, K, V, q_strides, k_strides, v_strides, q, k, v, log_decay, scale, state_in, state_out, rows, slots,
                   slots64, nullptr, o, static_cast<hipStream_t>(stream));
}

size_t cet_linear_attention_step_pool_workspace(int B, int rows) { return B > FEW_STREAMS && rows > 0 ? align_up((size_t)rows * sizeof(int)) : 0; }

int cet_linear_attention_step_pool(int dtype, int B, int H, int K, int V, const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* v_strides, const void* q, const void* k, const void* v,
                                   const float* log_decay, float scale, float* states, int rows, const void* slots,
                                   int slots64, void* o, void* workspace, size_t workspace_bytes, void* stream) {
  const size_t need = cet_linear_attention_step_pool_workspace(B, rows);
  if (!slots || need > workspace_bytes || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return CET_ERR_INVALID_ARG;
  return step_call(dtype, B, H, K, V, q_strides, k_strides, v_strides, q, k, v, log_decay, scale, states, states, rows, slots,
                   slots64, need ? static_cast<int*>(workspace) : nullptr, o, static_cast<hipStream_t>(stream));
}

}  // extern "C"
