// The gated projection of a feed-forward block: entry points, the choice of tiles, the kernel for few rows
// (weights streamed once) and the sums over blocks and splits. The tiled products are in gated.h.
#include <algorithm>
#include <climits>
#include <cmath>

#include "gated.h"

namespace cet {
namespace gated {

// gated_narrow.hip
bool narrow(const cet_gated_desc& d);
size_t narrow_workspace(const cet_gated_desc& d, int cus);
int narrow_forward_run(const cet_gated_desc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                       void* out, int cus, hipStream_t s);
int narrow_backward_run(const cet_gated_desc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                        const void* dy, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, float* part, int cus, hipStream_t s);

namespace {

constexpr size_t align_up(size_t n) { return (n + 255) & ~(size_t)255; }
constexpr int elem_bytes(int dtype) { return dtype == CET_F32 ? 4 : 2; }

// rows of D values at any stride -> rows of whole 16-byte pieces, zeros behind D
template <typename E>
__global__ __launch_bounds__(256) void pack_rows(const E* __restrict__ src, long ld, E* __restrict__ dst, int D, int per_row, long total) {
  constexpr int VEC = 16 / sizeof(E);
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long)gridDim.x * 256) {
    const int c = (int)(at % per_row) * VEC;
    const E* p = src + at / per_row * ld;
    E e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = c + j < D ? p[c + j] : E(0);
    uint4 raw;
    __builtin_memcpy(&raw, e, 16);
    reinterpret_cast<uint4*>(dst)[at] = raw;
  }
}

// db = column sums of dh, from the sums that the blocks of rows left in fp32 (in their order)
template <typename T>
__global__ __launch_bounds__(1024) void sum_blocks(const float* __restrict__ part, int rows, int F, int Fp, T* dg, T* du) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < 2 * Fp)
    for (int r = r0; r < rows; r += 64) s += part[(long)r * 2 * Fp + col];
  red[r0][c] = s;
  __syncthreads();
  if (r0 == 0 && col < 2 * Fp) {
    for (int r = 1; r < 64; ++r) s += red[r][c];
    const int f = col < Fp ? col : col - Fp;
    if (f < F) (col < Fp ? dg : du)[f] = (T)s;
  }
}

// out = sum of the splits' products, rounded once
template <typename T>
__global__ __launch_bounds__(256) void sum_splits(const float* __restrict__ part, int splits, int nq, int np, T* out, T* out1, int out_split, int F) {
  const long total = (long)nq * np, vec = np % 4 == 0 ? 4 : 1;
  for (long at = ((long)blockIdx.x * 256 + threadIdx.x) * vec; at < total; at += (long)gridDim.x * 256 * vec) {
    const int q = (int)(at / np), p = (int)(at - (long)q * np);
    const bool second = q >= out_split;
    const int row = second ? q - out_split : q;
    if (F && row >= F) continue;
    T* to = (second ? out1 : out) + (long)row * np + p;
    if (vec == 4) {
      f4 s = *reinterpret_cast<const f4*>(part + at);
      for (int x = 1; x < splits; ++x) s += *reinterpret_cast<const f4*>(part + x * total + at);
      const bool wide = (reinterpret_cast<uintptr_t>(to) & (4 * sizeof(T) - 1)) == 0;
      store4(to, s, 4, wide ? 4 : 1);
    } else {
      float s = part[at];
      for (int x = 1; x < splits; ++x) s += part[x * total + at];
      *to = (T)s;
    }
  }
}

// At most 64 rows: bound by the weights, which are read once and straight into registers. A workgroup takes
// 16 features; its 8 waves share the summed axis and add up in LDS. x comes from the caches.
template <typename T, int NQT>
__global__ __launch_bounds__(512) void few_rows(const Args a) {
  constexpr int E = Type<T>::E, VEC = 16 / E, STEP = 4 * VEC;
  __shared__ f4 red[8][2 * NQT][64];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = blockIdx.x * 16, fr = min(f0 + i, a.F - 1);
  const T* wg = static_cast<const T*>(a.P.p) + (long)fr * a.P.ld;
  const T* wu = static_cast<const T*>(a.P.p1) + (long)fr * a.P.ld1;
  const T* x[NQT];
#pragma unroll
  for (int y = 0; y < NQT; ++y) x[y] = static_cast<const T*>(a.Q.p) + (long)min(16 * y + i, a.nq - 1) * a.Q.ld;
  f4 ag[NQT], au[NQT];
#pragma unroll
  for (int y = 0; y < NQT; ++y) ag[y] = au[y] = f4{0.f, 0.f, 0.f, 0.f};
  const Frag none = {0, 0, 0, 0};
  const int steps = (a.nk + STEP - 1) / STEP;
  for (int s = wave; s < steps; s += 8) {
    const int k = s * STEP + g * VEC;
    const bool live = k < a.nk;  // whole pieces: rows are padded to them
    const Frag pg = live ? __builtin_nontemporal_load(reinterpret_cast<const Frag*>(wg + k)) : none;
    const Frag pu = live ? __builtin_nontemporal_load(reinterpret_cast<const Frag*>(wu + k)) : none;
#pragma unroll
    for (int y = 0; y < NQT; ++y) {
      const Frag q = live ? *reinterpret_cast<const Frag*>(x[y] + k) : none;
      ag[y] = mma<T>(pg, q, ag[y]);
      au[y] = mma<T>(pu, q, au[y]);
    }
  }
#pragma unroll
  for (int y = 0; y < NQT; ++y) {
    red[wave][2 * y][lane] = ag[y];
    red[wave][2 * y + 1][lane] = au[y];
  }
  __syncthreads();
  for (int y = wave; y < NQT; y += 8) {
    f4 gv = red[0][2 * y][lane], uv = red[0][2 * y + 1][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      gv += red[w][2 * y][lane];
      uv += red[w][2 * y + 1][lane];
    }
    const int f = f0 + 4 * g, n = a.F - f, q = 16 * y + i;
    if (a.bias_g) gv += load4(static_cast<const T*>(a.bias_g) + f, n, 1);
    if (a.bias_u) uv += load4(static_cast<const T*>(a.bias_u) + f, n, 1);
    f4 v, slope;
    act4(a.activation, gv, v, slope);
    if (q < a.nq && n > 0) store4(static_cast<T*>(a.out) + (long)q * a.ld_out + f, v * uv, n, a.out_step);
  }
}

template <typename T>
void launch_few(const Args& a, hipStream_t s) {
  const unsigned blocks = (unsigned)((a.F + 15) / 16);
  if (a.nq <= 16)
    few_rows<T, 1><<<blocks, 512, 0, s>>>(a);
  else if (a.nq <= 32)
    few_rows<T, 2><<<blocks, 512, 0, s>>>(a);
  else
    few_rows<T, 4><<<blocks, 512, 0, s>>>(a);
}

int cu_count() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
    return 256;
  return n;
}

// Tiles of 256 x 256 (one workgroup per CU), 128 x 128 (two) or 64 x 64 (four), and for sums that may be split, in how
// many pieces: the least estimate, from times measured per tile and 128 bytes of k, of a workgroup alone on its CU
// (its latency) and of one among several (its share of the CU), and per tile's results; 1.3 times as much where operands
// are read by columns, half of the results' time where they are stored as they are; the splits' partial products
// written and read at 8 TB/s, as they stay in the caches between. Forward times in us by 256, 128 and 64: bf16 500 rows,
// 2048 to 759: 55, 30, 21; 1073 rows, 1024 to 2177: 35, 24, 27; 8192 rows, 1024 to 2730: 115, 133, 179; fp32 1262 rows,
// 2048 to 1925: 490, 278, 213; 20,000 rows, 500 to 1001: 414, 391, 423.
struct Cut {
  int tile;
  int splits, k_per_split;
  size_t ws;
};
struct TileTimes {
  long b;
  double alone, shared, results;  // us
};
constexpr TileTimes TIMES[2][3] = {{{256, 1.55, 1.55, 10}, {128, 0.85, 0.58, 2.6}, {64, 0.58, 0.23, 1.1}},
                                   {{256, 7.5, 7.5, 20}, {128, 2.1, 2.1, 4}, {64, 0.65, 0.65, 1}}};  // fp32

Cut cut(int dtype, long np, long nq, long nk, bool gated, bool may_split, int cus) {
  const int bk = 128 / elem_bytes(dtype);
  Cut best{128, 1, 0, 0};
  double cost = 1e30;
  for (const TileTimes& x : TIMES[dtype == CET_F32]) {
    const long bp = gated ? x.b / 2 : x.b, tiles = ((np + bp - 1) / bp) * ((nq + x.b - 1) / x.b), slots = cus * (256 / x.b);
    for (int s = 1; s <= (may_split ? 512 : 1); s += s < 32 ? 1 : s / 8) {
      const long per = std::max<long>(((nk + s - 1) / s + bk - 1) / bk * bk, bk);
      const long used = std::max<long>((nk + per - 1) / per, 1);
      if (used != s) continue;
      const double rounds = (double)((tiles * s + slots - 1) / slots), share = (double)((tiles * s + cus - 1) / cus);
      const double steps = (double)(per / bk) * (gated ? 1 : 1.3);
      double t = std::max(rounds * steps * x.alone, share * steps * x.shared) + share * x.results * (gated ? 1 : 0.5);
      if (s > 1) t += 8.0 * s * np * nq / 8e6 + 4;
      if (t < cost) {
        cost = t;
        best = Cut{(int)x.b, s, (int)per, s > 1 ? align_up((size_t)s * np * nq * sizeof(float)) : 0};
      }
    }
  }
  return best;
}

void set_tiles(Args& a, const Cut& c, bool gated) {
  const int b = c.tile, bp = gated ? b / 2 : b;
  a.tiles_p = (a.np + bp - 1) / bp;
  a.tiles_q = (a.nq + b - 1) / b;
  a.splits = c.splits;
  a.k_per_split = c.splits > 1 ? c.k_per_split : a.nk;
  if (gated) a.P.split = b / 2;
}

int run(int dtype, const Args& a, int step, int tile, hipStream_t s) {
  return dtype == CET_F32 ? run_f32(a, step, tile, s) : dtype == CET_F16 ? run_f16(a, step, tile, s) : run_bf16(a, step, tile, s);
}

// A row-major matrix that the products read: in place where its rows are whole 16-byte pieces, else copied.
struct Matrix {
  const void* p;
  long ld, rows;
  int cols;
  size_t copy = 0;

  Matrix(const void* p, long ld, long rows, int cols, int dtype) : p(p), ld(ld), rows(rows), cols(cols) {
    const int vec = 16 / elem_bytes(dtype);
    if ((reinterpret_cast<uintptr_t>(p) & 15) || cols % vec || (ld % vec && rows > 1))
      copy = align_up((size_t)rows * ((cols + vec - 1) / vec) * 16);
  }
  int pack(int dtype, char*& ws, hipStream_t s) {
    if (!copy) return CET_OK;
    const int vec = 16 / elem_bytes(dtype), per_row = (cols + vec - 1) / vec;
    const long total = rows * per_row;
    const unsigned blocks = (unsigned)std::min<long>((total + 255) / 256, 1 << 20);
    if (dtype == CET_F32)
      pack_rows<uint32_t><<<blocks, 256, 0, s>>>(static_cast<const uint32_t*>(p), ld, reinterpret_cast<uint32_t*>(ws), cols, per_row, total);
    else
      pack_rows<uint16_t><<<blocks, 256, 0, s>>>(static_cast<const uint16_t*>(p), ld, reinterpret_cast<uint16_t*>(ws), cols, per_row, total);
    CET_HIP(hipGetLastError());
    p = ws;
    ld = (long)per_row * vec;
    ws += copy;
    return CET_OK;
  }
};

int step_of(const void* p, long ld, int dtype) {  // elements that a row can be read or written at once
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) / elem_bytes(dtype);
  return (at | ld) % 8 == 0 ? 8 : (at | ld) % 4 == 0 ? 4 : (at | ld) % 2 == 0 ? 2 : 1;
}

constexpr int FEW = 64;

bool bad_desc(const cet_gated_desc* d) {
  return !d || d->dtype < CET_F32 || d->dtype > CET_F16 || d->activation < 0 || d->activation > 2 || d->N < 0 || d->D < 1 || d->F < 1;
}
// (a launch holds fewer than 2^32 threads)
bool too_large(const cet_gated_desc& d) {
  return d.N > (1 << 28) || d.D > (1 << 20) || d.F > (1 << 20) || (double)d.N * d.F > 6e10 || (double)d.N * d.D > 6e10 || (double)d.D * d.F > 6e10;
}

struct Plan {
  Matrix x, wg, wu;
  int Fp;
  Cut forward, dx, dw;
  size_t packs, dh, blocks, splits;
  long block_rows;

  Plan(const cet_gated_desc& d, const void* xp, const void* wgp, const void* wup, bool backward)
      : x(xp, d.ld_x, d.N, d.D, d.dtype), wg(wgp, d.ld_gate, d.F, d.D, d.dtype), wu(wup, d.ld_up, d.F, d.D, d.dtype) {
    const int vec = 16 / elem_bytes(d.dtype), cus = cu_count();
    Fp = (d.F + vec - 1) / vec * vec;
    packs = x.copy + wg.copy + wu.copy;
    forward = cut(d.dtype, d.F, d.N, d.D, true, false, cus);
    dh = blocks = splits = 0;
    block_rows = 0;
    if (backward) {
      dx = cut(d.dtype, d.D, d.N, 2L * Fp, false, true, cus);
      dw = cut(d.dtype, d.D, 2L * Fp, d.N, false, true, cus);
      dh = align_up((size_t)d.N * 2 * Fp * elem_bytes(d.dtype));
      // one row of column sums per tile and wave along the rows (4 waves in the largest tile, 2 in the others)
      block_rows = ((long)d.N + forward.tile - 1) / forward.tile * (forward.tile == 256 ? 4 : 2);
      blocks = align_up((size_t)block_rows * 2 * Fp * sizeof(float));
      splits = std::max(dx.ws, dw.ws);
    }
  }
  size_t bytes() const { return packs + dh + blocks + splits; }
};

template <typename T>
void launch_sum_blocks(const float* part, long rows, int F, int Fp, void* dg, void* du, hipStream_t s) {
  sum_blocks<T><<<(unsigned)((2 * Fp + 15) / 16), 1024, 0, s>>>(part, (int)rows, F, Fp, static_cast<T*>(dg), static_cast<T*>(du));
}
template <typename T>
void launch_sum_splits(const Args& a, hipStream_t s) {
  const long vec = a.np % 4 == 0 ? 4 : 1, n = ((long)a.nq * a.np / vec + 255) / 256;
  sum_splits<T><<<(unsigned)std::min<long>(n, 1 << 16), 256, 0, s>>>(a.part, a.splits, a.nq, a.np, static_cast<T*>(a.out), static_cast<T*>(a.out1), a.out_split, a.F);
}

// A product of `dh` with another operand, split over the summed axis where the plan says so.
int product_of_dh(int dtype, Args a, const Cut& c, int step, int step_partial, float* splits, hipStream_t s) {
  set_tiles(a, c, false);
  if (c.splits == 1) return run(dtype, a, step, c.tile, s);
  a.part = splits;
  Args b = a;
  b.ld_out = a.np;
  if (const int rc = run(dtype, b, step_partial, c.tile, s)) return rc;
  if (dtype == CET_F32)
    launch_sum_splits<float>(a, s);
  else if (dtype == CET_F16)
    launch_sum_splits<_Float16>(a, s);
  else
    launch_sum_splits<__bf16>(a, s);
  CET_HIP(hipGetLastError());
  return CET_OK;
}

Args base(const cet_gated_desc& d, const Plan& p, const void* bg, const void* bu) {
  Args a{};
  a.P = Operand{p.wg.p, p.wu.p, p.wg.ld, p.wu.ld, INT_MAX, INT_MAX};
  a.Q = Operand{p.x.p, nullptr, p.x.ld, 0, INT_MAX, INT_MAX};
  a.np = a.F = d.F, a.nq = d.N, a.nk = d.D;
  a.Fp = p.Fp;
  a.activation = d.activation;
  a.bias_g = bg, a.bias_u = bu;
  a.out_split = INT_MAX;
  return a;
}

}  // namespace
}  // namespace gated
}  // namespace cet

using namespace cet;
using namespace cet::gated;

extern "C" {

size_t cet_gated_linear_workspace(const cet_gated_desc* d, const void* x, const void* w_gate, const void* w_up, int backward) {
  if (bad_desc(d) || too_large(*d)) return 0;
  if (narrow(*d)) return backward ? narrow_workspace(*d, cu_count()) : 0;
  return Plan(*d, x, w_gate, w_up, backward != 0).bytes();
}

int cet_gated_linear(const cet_gated_desc* d, const void* x, const void* w_gate, const void* w_up, const void* b_gate,
                     const void* b_up, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_desc(d)) return CET_ERR_INVALID_ARG;
  if (too_large(*d)) return CET_ERR_UNSUPPORTED;
  if (d->N == 0) return CET_OK;
  if (!x || !w_gate || !w_up || !out || (reinterpret_cast<uintptr_t>(workspace) & 15)) return CET_ERR_INVALID_ARG;
  if (narrow(*d)) return narrow_forward_run(*d, x, w_gate, w_up, b_gate, b_up, out, cu_count(), static_cast<hipStream_t>(stream));
  Plan p(*d, x, w_gate, w_up, false);
  if (p.bytes() > workspace_bytes || (p.bytes() && !workspace)) return CET_ERR_INVALID_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  for (Matrix* m : {&p.x, &p.wg, &p.wu})
    if (const int rc = m->pack(d->dtype, ws, s)) return rc;
  Args a = base(*d, p, b_gate, b_up);
  a.out = out, a.ld_out = d->F, a.out_step = step_of(out, d->F, d->dtype);
  if (d->N <= FEW) {
    if (d->dtype == CET_F32)
      launch_few<float>(a, s);
    else if (d->dtype == CET_F16)
      launch_few<_Float16>(a, s);
    else
      launch_few<__bf16>(a, s);
    CET_HIP(hipGetLastError());
    return CET_OK;
  }
  set_tiles(a, p.forward, true);
  return run(d->dtype, a, STEP_FORWARD, p.forward.tile, s);
}

int cet_gated_linear_backward(const cet_gated_desc* d, const void* x, const void* w_gate, const void* w_up,
                              const void* b_gate, const void* b_up, const void* dy, void* dx, void* dw_gate, void* dw_up,
                              void* db_gate, void* db_up, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_desc(d)) return CET_ERR_INVALID_ARG;
  if (too_large(*d)) return CET_ERR_UNSUPPORTED;
  if (!w_gate || !w_up || (d->N > 0 && (!x || !dy))) return CET_ERR_INVALID_ARG;
  if ((dw_gate == nullptr) != (dw_up == nullptr) || (db_gate == nullptr) != (db_up == nullptr)) return CET_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return CET_ERR_INVALID_ARG;
  if (narrow(*d)) {
    const int cus = cu_count();
    if (narrow_workspace(*d, cus) > workspace_bytes || !workspace) return CET_ERR_INVALID_ARG;
    return narrow_backward_run(*d, x, w_gate, w_up, b_gate, b_up, dy, dx, dw_gate, dw_up, db_gate, db_up,
                               static_cast<float*>(workspace), cus, static_cast<hipStream_t>(stream));
  }
  Plan p(*d, x, w_gate, w_up, true);
  if (p.bytes() > workspace_bytes || (p.bytes() && !workspace)) return CET_ERR_INVALID_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  for (Matrix* m : {&p.x, &p.wg, &p.wu})
    if (const int rc = m->pack(d->dtype, ws, s)) return rc;
  void* dh = ws;
  float* blocks = reinterpret_cast<float*>(ws + p.dh);
  float* splits = reinterpret_cast<float*>(ws + p.dh + p.blocks);
  if (d->N > 0) {
    Args a = base(*d, p, b_gate, b_up);
    a.dy = dy, a.ld_dy = d->ld_dy, a.dy_step = step_of(dy, d->ld_dy, d->dtype);
    a.out = dh, a.ld_out = 2L * p.Fp;
    a.part = db_gate ? blocks : nullptr;
    set_tiles(a, p.forward, true);
    if (const int rc = run(d->dtype, a, STEP_DH, p.forward.tile, s)) return rc;
  }
  if (db_gate) {
    if (d->dtype == CET_F32)
      launch_sum_blocks<float>(blocks, p.block_rows, d->F, p.Fp, db_gate, db_up, s);
    else if (d->dtype == CET_F16)
      launch_sum_blocks<_Float16>(blocks, p.block_rows, d->F, p.Fp, db_gate, db_up, s);
    else
      launch_sum_blocks<__bf16>(blocks, p.block_rows, d->F, p.Fp, db_gate, db_up, s);
    CET_HIP(hipGetLastError());
  }
  if (dx && d->N > 0) {
    Args a{};
    a.P = Operand{p.wg.p, p.wu.p, p.wg.ld, p.wu.ld, p.Fp, d->F};
    a.Q = Operand{dh, nullptr, 2L * p.Fp, 0, INT_MAX, INT_MAX};
    a.np = d->D, a.nq = d->N, a.nk = 2 * p.Fp;
    a.out = dx, a.ld_out = d->D, a.out_split = INT_MAX, a.out_step = step_of(dx, d->D, d->dtype);
    if (const int rc = product_of_dh(d->dtype, a, p.dx, STEP_DX, STEP_DX_PARTIAL, splits, s)) return rc;
  }
  if (dw_gate) {
    Args a{};
    a.P = Operand{p.x.p, nullptr, p.x.ld, 0, INT_MAX, d->N};
    a.Q = Operand{dh, nullptr, 2L * p.Fp, 0, INT_MAX, d->N};
    a.np = d->D, a.nq = 2 * p.Fp, a.nk = d->N;
    a.F = d->F;
    a.out = dw_gate, a.out1 = dw_up, a.ld_out = d->D, a.out_split = p.Fp;
    a.out_step = std::min(step_of(dw_gate, d->D, d->dtype), step_of(dw_up, d->D, d->dtype));
    if (const int rc = product_of_dh(d->dtype, a, p.dw, STEP_DW, STEP_DW_PARTIAL, splits, s)) return rc;
  }
  return CET_OK;
}

}  // extern "C"
