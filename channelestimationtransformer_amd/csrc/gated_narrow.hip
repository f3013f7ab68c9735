// The gated projection of narrow layers, D and F up to 64 (the Transformer predictor's own sizes): both weights
// fit one CU, so that a pass over the rows does everything. Waves are persistent; each takes 16 rows at a time
// straight into registers. Multiplied in fp32 whatever the tensors' type: what bounds these sizes is memory
// (102,400 rows of 64 to 64 in fp32: 52 MB, 11 us at the rate of a large copy) and the fp32 matrix rate (11 us)
// alike. Forward takes 34 us and backward 79; the tiled products took 40 and 375, most of it in passes over dh and
// in launches.
//
//   forward:  the weights stay in a wave's registers; D tiles hold 4 neighbouring features of a row per lane.
//   backward: the projections are formed again, their gradients stay in registers as the operand of dx and go
//             through the wave's own LDS once, turned, as the operand of dW; dW and db are summed in registers
//             over all rows of a wave, over the waves of a workgroup in LDS, and over workgroups in a second launch.
#include "gated.h"

namespace cet {
namespace gated {
namespace {

struct Narrow {
  const void *x, *wg, *wu, *bg, *bu, *dy;
  void *out, *dx;
  float* part;  // [workgroups][2 * 64 * 64 + 2 * 64]
  long ld_x, ld_g, ld_u, ld_dy;
  int N, D, F, activation;
  int x_step, g_step, u_step, dy_step, out_step, dx_step;
};

constexpr int PART = 2 * 64 * 64 + 2 * 64;

__device__ inline f4 mma4(const f4& a, const f4& b, f4 c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
  return c;
}

// What lanes of a wave read of each other in LDS stays behind what they wrote (LDS takes a wave's accesses in order: only the
// compiler has to be told).
__device__ inline void between_lanes() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 16 rows from `row` on as operands (k along the features): lane (i, g) holds features 16 kk + 4 g.. of row i
template <typename T, int NK>
__device__ inline void load_rows(f4 (&q)[NK], const void* p, long ld, long row, long rows, int cols, int step, int i, int g) {
  const bool live = row + i < rows;
  const T* at = static_cast<const T*>(p) + (live ? row + i : 0) * ld;
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) q[kk] = load4(at + 16 * kk + 4 * g, live ? cols - 16 * kk - 4 * g : 0, step);
}

// Both weights as operands (k along the inputs) into LDS, once per workgroup: [gate tiles, up tiles][ND][lane]
template <typename T, int ND, int NF, int NT>
__device__ inline void stage_weights(const Narrow& a, f4 (*w)[ND][64]) {
  for (int at = threadIdx.x; at < 2 * NF * ND * 64; at += NT) {
    const int l = at & 63, li = l & 15, lg = l >> 4, kk = at / 64 % ND, f = at / 64 / ND;
    const bool up = f >= NF;
    const int row = 16 * (up ? f - NF : f) + li, c = 16 * kk + 4 * lg;
    const T* p = static_cast<const T*>(up ? a.wu : a.wg) + (long)(row < a.F ? row : 0) * (up ? a.ld_u : a.ld_g) + c;
    w[f][kk][l] = load4(p, row < a.F ? a.D - c : 0, up ? a.u_step : a.g_step);
  }
}

template <typename T, int ND, int NF>
__global__ __launch_bounds__(512, 2) void narrow_forward(const Narrow a) {
  __shared__ f4 w[2 * NF][ND][64];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const long wave = (long)blockIdx.x * 8 + (threadIdx.x >> 6), waves = (long)gridDim.x * 8, tiles = ((long)a.N + 15) / 16;
  f4 x[ND], next[ND];
  if (wave < tiles) load_rows<T, ND>(x, a.x, a.ld_x, wave * 16, a.N, a.D, a.x_step, i, g);
  stage_weights<T, ND, NF, 512>(a, w);
  f4 wg[NF][ND], wu[NF][ND], bg[NF], bu[NF];
  __syncthreads();
#pragma unroll
  for (int f = 0; f < NF; ++f) {
#pragma unroll
    for (int kk = 0; kk < ND; ++kk) wg[f][kk] = w[f][kk][lane], wu[f][kk] = w[NF + f][kk][lane];
    const int at = 16 * f + 4 * g, n = a.F - at;
    bg[f] = bu[f] = f4{0.f, 0.f, 0.f, 0.f};
    if (a.bg) bg[f] = load4(static_cast<const T*>(a.bg) + at, n, 1);
    if (a.bu) bu[f] = load4(static_cast<const T*>(a.bu) + at, n, 1);
  }
  for (long t = wave; t < tiles; t += waves) {
    if (t + waves < tiles) load_rows<T, ND>(next, a.x, a.ld_x, (t + waves) * 16, a.N, a.D, a.x_step, i, g);
    const long row = t * 16 + i;
    f4 gv[NF], uv[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) gv[f] = bg[f], uv[f] = bu[f];
#pragma unroll
    for (int kk = 0; kk < ND; ++kk)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        gv[f] = mma4(wg[f][kk], x[kk], gv[f]);
        uv[f] = mma4(wu[f][kk], x[kk], uv[f]);
      }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      f4 v, slope;
      act4(a.activation, gv[f], v, slope);
      const int at = 16 * f + 4 * g;
      if (row < a.N && at < a.F) store4(static_cast<T*>(a.out) + row * a.F + at, v * uv[f], a.F - at, a.out_step);
    }
#pragma unroll
    for (int kk = 0; kk < ND; ++kk) x[kk] = next[kk];
  }
}

template <typename T, int ND, int NF>
__global__ __launch_bounds__(256, 1) void narrow_backward(const Narrow a) {
  constexpr int XLD = 16 * ND + 4, HLD = 32 * NF + 4;  // rows of the turned tiles, off the banks' period
  __shared__ f4 w[2 * NF][ND][64];   // weights as operands, k along the inputs
  __shared__ f4 wt[ND][2 * NF][64];  // and along the features
  __shared__ __align__(16) float xs[4][16 * XLD], hs[4][16 * HLD];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wv = threadIdx.x >> 6;
  const long wave = (long)blockIdx.x * 4 + wv, waves = (long)gridDim.x * 4, tiles = ((long)a.N + 15) / 16;
  stage_weights<T, ND, NF, 256>(a, w);
  __syncthreads();
  for (int at = threadIdx.x; at < 2 * NF * ND * 64; at += 256) {
    // element (feature 16 f + 4 lg + r, input 16 d + li) of the weights as laid down above
    const int l = at & 63, li = l & 15, lg = l >> 4, f = at / 64 % (2 * NF), d = at / 64 / (2 * NF);
    f4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = w[f][d][(4 * lg + r) + 16 * (li >> 2)][li & 3];
    wt[d][f][l] = v;
  }
  f4 bg[NF], bu[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int at = 16 * f + 4 * g, n = a.F - at;
    bg[f] = bu[f] = f4{0.f, 0.f, 0.f, 0.f};
    if (a.bg) bg[f] = load4(static_cast<const T*>(a.bg) + at, n, 1);
    if (a.bu) bu[f] = load4(static_cast<const T*>(a.bu) + at, n, 1);
  }
  f4 dw[2 * NF][ND], db[2 * NF];
#pragma unroll
  for (int f = 0; f < 2 * NF; ++f) {
    db[f] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < ND; ++d) dw[f][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  f4 x[ND], dy[NF];
  if (wave < tiles) {
    load_rows<T, ND>(x, a.x, a.ld_x, wave * 16, a.N, a.D, a.x_step, i, g);
    load_rows<T, NF>(dy, a.dy, a.ld_dy, wave * 16, a.N, a.F, a.dy_step, i, g);
  }
  __syncthreads();
  f4 wr[2 * NF][ND];
#pragma unroll
  for (int f = 0; f < 2 * NF; ++f)
#pragma unroll
    for (int kk = 0; kk < ND; ++kk) wr[f][kk] = w[f][kk][lane];
  float* const xt = xs[wv];
  float* const ht = hs[wv];
  for (long t = wave; t < tiles; t += waves) {
    f4 dh[2 * NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) dh[f] = bg[f], dh[NF + f] = bu[f];
#pragma unroll
    for (int kk = 0; kk < ND; ++kk)
#pragma unroll
      for (int f = 0; f < 2 * NF; ++f) dh[f] = mma4(wr[f][kk], x[kk], dh[f]);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      f4 v, slope;
      act4(a.activation, dh[f], v, slope);
      const f4 uv = dh[NF + f];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool live = 16 * f + 4 * g + r < a.F && t * 16 + i < a.N;
        dh[f][r] = live ? dy[f][r] * uv[r] * slope[r] : 0.f;
        dh[NF + f][r] = live ? dy[f][r] * v[r] : 0.f;
      }
      db[f] += dh[f];
      db[NF + f] += dh[NF + f];
    }
    // both operands of dW with the rows along k: through this wave's own LDS
#pragma unroll
    for (int kk = 0; kk < ND; ++kk) *reinterpret_cast<f4*>(xt + i * XLD + 16 * kk + 4 * g) = x[kk];
#pragma unroll
    for (int f = 0; f < 2 * NF; ++f) *reinterpret_cast<f4*>(ht + i * HLD + 16 * f + 4 * g) = dh[f];
    if (t + waves < tiles) {
      load_rows<T, ND>(x, a.x, a.ld_x, (t + waves) * 16, a.N, a.D, a.x_step, i, g);
      load_rows<T, NF>(dy, a.dy, a.ld_dy, (t + waves) * 16, a.N, a.F, a.dy_step, i, g);
    }
    if (a.dx) {
      const long row = t * 16 + i;
      f4 v[ND];
#pragma unroll
      for (int d = 0; d < ND; ++d) v[d] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < 2 * NF; ++f)
#pragma unroll
        for (int d = 0; d < ND; ++d) v[d] = mma4(wt[d][f][lane], dh[f], v[d]);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const int at = 16 * d + 4 * g;
        if (row < a.N && at < a.D) store4(static_cast<T*>(a.dx) + row * a.D + at, v[d], a.D - at, a.dx_step);
      }
    }
    between_lanes();
    f4 xq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) xq[d][r] = xt[(4 * g + r) * XLD + 16 * d + i];
#pragma unroll
    for (int f = 0; f < 2 * NF; ++f) {
      f4 hq;
#pragma unroll
      for (int r = 0; r < 4; ++r) hq[r] = ht[(4 * g + r) * HLD + 16 * f + i];
#pragma unroll
      for (int d = 0; d < ND; ++d) dw[f][d] = mma4(xq[d], hq, dw[f][d]);
    }
    between_lanes();
  }
  if (!a.part) return;
  // sums over the four waves, one after the other, in the space of the weights; lane (i, g) of tile (f, d) holds
  // inputs 16 d + 4 g.. of feature 16 f + i
  f4* const sum = &w[0][0][0];
  float* const bsum = reinterpret_cast<float*>(xs);
#pragma unroll
  for (int f = 0; f < 2 * NF; ++f)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int off = 1; off < 16; off *= 2) db[f][r] += __shfl_xor(db[f][r], off);
  for (int turn = 0; turn < 4; ++turn) {
    __syncthreads();
    if (wv != turn) continue;
#pragma unroll
    for (int f = 0; f < 2 * NF; ++f) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f4* p = sum + (f * ND + d) * 64 + lane;
        *p = turn ? *p + dw[f][d] : dw[f][d];
      }
      if (i == 0) {
        f4* p = reinterpret_cast<f4*>(bsum + 16 * f + 4 * g);
        *p = turn ? *p + db[f] : db[f];
      }
    }
  }
  __syncthreads();
  float* part = a.part + (long)blockIdx.x * PART;
  for (int at = threadIdx.x; at < 2 * NF * ND * 64; at += 256) {
    const int l = at & 63, li = l & 15, lg = l >> 4, d = at / 64 % ND, f = at / 64 / ND;
    const int feature = 16 * (f % NF) + li + (f >= NF ? 64 : 0);
    *reinterpret_cast<f4*>(part + feature * 64 + 16 * d + 4 * lg) = sum[at];
  }
  for (int at = threadIdx.x; at < 32 * NF; at += 256)
    part[2 * 64 * 64 + (at < 16 * NF ? at : 64 + at - 16 * NF)] = bsum[at];
}

// dW and db from the workgroups' sums, in their order
template <typename T>
__global__ __launch_bounds__(1024) void sum_narrow(const float* __restrict__ part, int groups, int F, int D, T* dwg, T* dwu, T* dbg, T* dbu) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6, row = blockIdx.x;  // rows 0..127: features; 128, 129: the biases
  const bool bias = row >= 128;
  const int f = row & 63;
  if (bias ? !dbg : !dwg || f >= F) return;
  float s = 0.f;
  if (c < (bias ? F : D)) {
    const float* p = part + (long)row * 64 + c;
#pragma unroll 4
    for (int r = r0; r < groups; r += 16) s += p[(long)r * PART];
  }
  red[r0][c] = s;
  __syncthreads();
  if (r0 == 0 && c < (bias ? F : D)) {
#pragma unroll
    for (int r = 1; r < 16; ++r) s += red[r][c];
    if (bias)
      (row == 128 ? dbg : dbu)[c] = (T)s;
    else
      (row < 64 ? dwg : dwu)[(long)f * D + c] = (T)s;
  }
}

template <typename T, int ND, int NF>
void launch(const Narrow& a, bool backward, unsigned groups, hipStream_t s) {
  if (backward)
    narrow_backward<T, ND, NF><<<groups, 256, 0, s>>>(a);
  else
    narrow_forward<T, ND, NF><<<groups, 512, 0, s>>>(a);
}
template <typename T>
void launch(const Narrow& a, bool backward, unsigned groups, hipStream_t s) {
  if (a.D <= 32)
    a.F <= 32 ? launch<T, 2, 2>(a, backward, groups, s) : launch<T, 2, 4>(a, backward, groups, s);
  else
    a.F <= 32 ? launch<T, 4, 2>(a, backward, groups, s) : launch<T, 4, 4>(a, backward, groups, s);
}
void launch(const Narrow& a, int dtype, bool backward, unsigned groups, hipStream_t s) {
  if (dtype == CET_F32)
    launch<float>(a, backward, groups, s);
  else if (dtype == CET_F16)
    launch<_Float16>(a, backward, groups, s);
  else
    launch<__bf16>(a, backward, groups, s);
}

int step_of(const void* p, long ld, int dtype) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) / (dtype == CET_F32 ? 4 : 2);
  return (at | ld) % 4 == 0 ? 4 : (at | ld) % 2 == 0 ? 2 : 1;
}

// Workgroups, at most one per CU, for waves with 16 rows at least.
unsigned groups_of(long N, int waves, unsigned most) {
  const long n = (N + 16 * waves - 1) / (16 * waves);
  return (unsigned)(n < 1 ? 1 : n < most ? n : most);
}

Narrow base(const cet_gated_desc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu) {
  Narrow a{};
  a.x = x, a.wg = wg, a.wu = wu, a.bg = bg, a.bu = bu;
  a.ld_x = d.ld_x, a.ld_g = d.ld_gate, a.ld_u = d.ld_up;
  a.N = d.N, a.D = d.D, a.F = d.F, a.activation = d.activation;
  a.x_step = step_of(x, d.ld_x, d.dtype), a.g_step = step_of(wg, d.ld_gate, d.dtype), a.u_step = step_of(wu, d.ld_up, d.dtype);
  return a;
}

}  // namespace

bool narrow(const cet_gated_desc& d) { return d.D <= 64 && d.F <= 64; }

size_t narrow_workspace(const cet_gated_desc& d, int cus) { return (size_t)groups_of(d.N, 4, cus) * PART * sizeof(float); }

int narrow_forward_run(const cet_gated_desc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                       void* out, int cus, hipStream_t s) {
  Narrow a = base(d, x, wg, wu, bg, bu);
  a.out = out, a.out_step = step_of(out, d.F, d.dtype);
  launch(a, d.dtype, false, groups_of(d.N, 8, cus), s);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

int narrow_backward_run(const cet_gated_desc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                        const void* dy, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, float* part, int cus, hipStream_t s) {
  Narrow a = base(d, x, wg, wu, bg, bu);
  a.dy = dy, a.ld_dy = d.ld_dy, a.dy_step = step_of(dy, d.ld_dy, d.dtype);
  a.dx = dx, a.dx_step = step_of(dx, d.D, d.dtype);
  a.part = dwg || dbg ? part : nullptr;
  const unsigned groups = groups_of(d.N, 4, cus);
  launch(a, d.dtype, true, groups, s);
  CET_HIP(hipGetLastError());
  if (a.part) {
    if (d.dtype == CET_F32)
      sum_narrow<float><<<130, 1024, 0, s>>>(part, (int)groups, d.F, d.D, (float*)dwg, (float*)dwu, (float*)dbg, (float*)dbu);
    else if (d.dtype == CET_F16)
      sum_narrow<_Float16><<<130, 1024, 0, s>>>(part, (int)groups, d.F, d.D, (_Float16*)dwg, (_Float16*)dwu, (_Float16*)dbg, (_Float16*)dbu);
    else
      sum_narrow<__bf16><<<130, 1024, 0, s>>>(part, (int)groups, d.F, d.D, (__bf16*)dwg, (__bf16*)dwu, (__bf16*)dbg, (__bf16*)dbu);
    CET_HIP(hipGetLastError());
  }
  return CET_OK;
}

}  // namespace gated
}  // namespace cet
