// Activations kept in 8 bits between forward and backward (format: fm_act8.h), and the two
// element-wise layers that keep their inputs so:
//   fm_act8_compress, fm_act8_restore   rows into the format and back (the rows of an index)
//   fm_act8_swiglu, .._swiglu_backward  h = silu(g) u, g and u kept; dg, du from what was kept
//   fm_act8_rmsnorm, .._rmsnorm_backward  y = x r w, x kept; dx, dw from what was kept
// All of them move bytes: one pass each, every value read and written once.  A lane holds eight
// neighbours (16 bytes of bf16), four lanes a block, so a block's scale costs two exchanges within
// quads and no LDS.
#include <type_traits>

#include "fm_act8.h"
#include "fm_lanes.h"
#include "fm_silu.h"
#include "../../include/fm_hip.h"

namespace fm {
namespace {

// How a call passes the caches, by the bytes of its widest tensor (STREAM of the kernels; wide: of 16- or 32-bit values).
//   0  as usual
//   1  from 32 MiB on, the second-level caches together: wide outputs are stored past them.  2999 x 2831 fp32: the norm's three
//      launches 45.3 -> 38.2 us; 16384 x 4096 bf16 kept and restored in 33792 rows 107.7 -> 95.5.  (The payload, which
//      the backward wants, is stored as usual: past the caches the latter takes 107.3.)
//   2  from 128 MiB on, half of the last-level cache: the backward's gradients and the compressed activation are loaded past them
//      too, so that what was kept stays: norm of 16384 x 7168 228 -> 204 us, SwiGLU of 16384 x 14336 667 -> 654.  At 34 MB
//      that costs: 38.2 -> 42.5 us.
constexpr int64_t kStreamOut = int64_t(32) << 20, kStreamIn = int64_t(128) << 20;
inline int stream_level(int64_t bytes) { return bytes >= kStreamIn ? 2 : bytes >= kStreamOut ? 1 : 0; }

// ------------------------------------------------------------ rows of eight ----
// Eight neighbours of a row as they are stored, n of them in the row (zeros behind).  TAIL: n may lie between 0 and 8.
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];
  template <bool TAIL = true, bool NT = false>
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4_el v = NT ? __builtin_nontemporal_load(FM_GLOBAL(const u32x4_el, p) + i) : *(FM_GLOBAL(const u32x4_el, p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if constexpr (!TAIL) return;
#pragma unroll
    for (int i = 0; i < 7; ++i) {
      if constexpr (sizeof(T) == 2) w[i / 2] |= i < n ? uint32_t(p[i]) << (16 * (i & 1)) : 0u;
      else w[i] = i < n ? f2u(p[i]) : 0u;
    }
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = u2f(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      else v[i] = u2f(w[i]);
    }
  }
};

// The first n of eight values, rounded to T.
template <typename T, bool TAIL = true, bool NT = false>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  uint32_t w[Eight<T>::kWords];
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 2) w[i] = hw_bf16x2(v[2 * i], v[2 * i + 1]);
    else w[i] = f2u(v[i]);
  }
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < Eight<T>::kWords / 4; ++i) {
      const u32x4_el v = {w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      if constexpr (NT) __builtin_nontemporal_store(v, FM_GLOBAL(u32x4_el, p) + i);
      else *(FM_GLOBAL(u32x4_el, p) + i) = v;
    }
    return;
  }
  if constexpr (!TAIL) return;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    if (i >= n) break;
    if constexpr (sizeof(T) == 2) st_global(p + i, uint16_t(w[i / 2] >> (16 * (i & 1))));
    else st_global(reinterpret_cast<uint32_t*>(p) + i, w[i]);
  }
}

// Division of 0 <= n < 2^31 by a fixed d >= 1: (n + mulhi(n, m)) >> l (Granlund and Montgomery, PLDI 1994).
struct FastDiv {
  uint32_t m, l, d;
  explicit FastDiv(uint32_t div) : d(div) {
    l = 0;
    while ((uint64_t(1) << l) < div) ++l;
    m = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << l) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (n + __umulhi(n, m)) >> l; }
};

// A matrix's eights (fours, where EACH is 4), row by row, ld_q / EACH to a row: eight i is columns [8 (i % per), + 8) of row i / per.
struct Items {
  FastDiv per;
  uint32_t n;      // fewer than 2^31
  int64_t row0;    // first row
  int cols;
};
struct Item {
  int64_t row;
  int col, n;      // n of the eight lie in the row (at most 0 behind it)
  bool in;
};
// Eights u of U of a thread; one past the last stands for the last and is not stored.
template <int U, int EACH = 8>
__device__ __forceinline__ Item item_of(const Items& t, int u) {
  const uint32_t i = blockIdx.x * (256u * U) + u * 256u + threadIdx.x;
  const uint32_t j = i < t.n ? i : t.n - 1;
  const uint32_t r = t.per.quotient(j);
  const int col = int(j - r * t.per.d) * EACH;
  return Item{t.row0 + r, col, t.cols - col, i < t.n};
}

__device__ __forceinline__ void store_kept(uint8_t* q, int64_t ld_q, uint8_t* codes, int64_t ld_c, int64_t row, int col, uint2 b,
                                           uint32_t code) {
  st_global(q + row * ld_q + col, b);
  if ((threadIdx.x & 3) == 0) st_global(codes + row * ld_c + (col >> 5), uint8_t(code));
}

// --------------------------------------------------------------- compress ----
struct CompressArgs {
  const void* x;
  int64_t ld_x;
  uint8_t* q;
  int64_t ld_q;
  uint8_t* codes;
  int64_t ld_c;
  const int32_t* tile_valid;   // rows of 128-row tiles with a negative entry are left alone; null: none
};

template <typename T, int U, int STREAM>
__global__ __launch_bounds__(256) void compress_kernel(Items t, CompressArgs a) {
  Item it[U];
  Eight<T> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    it[u] = item_of<U>(t, u);
    if (a.tile_valid && a.tile_valid[it[u].row >> 7] < 0) it[u].in = false;
    x[u].template load<true, (STREAM > 1)>(static_cast<const T*>(a.x) + it[u].row * a.ld_x + it[u].col, it[u].in ? it[u].n : 0);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8];
    x[u].widen(v);
    uint32_t code;
    const uint2 b = act_encode8(v, code);
    if (it[u].in) store_kept(a.q, a.ld_q, a.codes, a.ld_c, it[u].row, it[u].col, b, code);
  }
}

// ---------------------------------------------------------------- restore ----
struct RestoreArgs {
  Act8 x;
  const int32_t* index;   // output row r is row index[r] of x, zeros where it is outside [0, src_rows); null: row r
  int64_t src_rows;
  void* out;
  int64_t ld_out;
};

// A lane stores 16 bytes: eight bf16 values or four fp32 ones.  (Eight fp32 values as two stores, each to every other 16 bytes, went past
// the caches at half the rate: 65536 x 1024 108 us, of fours 49.)
template <typename T, int U, bool GATHER, int STREAM>
__global__ __launch_bounds__(256) void restore_kernel(Items t, RestoreArgs a) {
  constexpr int kEach = 16 / sizeof(T);
  Item it[U];
  uint32_t b[U][kEach / 4], code[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    it[u] = item_of<U, kEach>(t, u);
    int64_t r = it[u].row;
    bool zero = false;
    if constexpr (GATHER) {
      r = a.index[r];
      zero = r < 0 || r >= a.src_rows;
    }
    code[u] = zero ? 0u : a.x.code(r, it[u].col);
    if constexpr (kEach == 8) {
      const uint2 w = zero ? make_uint2(0, 0) : a.x.bytes(r, it[u].col);
      b[u][0] = w.x;
      b[u][1] = w.y;
    } else {
      b[u][0] = zero ? 0u : *reinterpret_cast<const uint32_t*>(a.x.q + r * a.x.ld_q + it[u].col);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8];
    const float s = act_scale(code[u]);
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) act_decode4(b[u][i], s, v + 4 * i);
    if (!it[u].in) continue;
    T* p = static_cast<T*>(a.out) + it[u].row * a.ld_out + it[u].col;
    if constexpr (kEach == 8) {
      store8<T, true, (STREAM > 0)>(p, v, it[u].n);
    } else if (it[u].n >= 4) {
      const u32x4_el w = {f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
      if constexpr (STREAM > 0) __builtin_nontemporal_store(w, FM_GLOBAL(u32x4_el, p));
      else *FM_GLOBAL(u32x4_el, p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < it[u].n) st_global(p + i, v[i]);
    }
  }
}

// ----------------------------------------------------------------- SwiGLU ----
struct SwigluArgs {
  const void *g, *u;
  int64_t ld_g, ld_u;
  void* h;
  int64_t ld_h;
  uint8_t *qg, *qu, *cg, *cu;
  int64_t ld_q, ld_c;
};

template <typename T, int U, int STREAM>
__global__ __launch_bounds__(256) void swiglu_kernel(Items t, SwigluArgs a) {
  Item it[U];
  Eight<T> g[U], up[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    it[u] = item_of<U>(t, u);
    g[u].template load<true>(static_cast<const T*>(a.g) + it[u].row * a.ld_g + it[u].col, it[u].n);
    up[u].template load<true>(static_cast<const T*>(a.u) + it[u].row * a.ld_u + it[u].col, it[u].n);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float gv[8], uv[8], h[8];
    g[u].widen(gv);
    up[u].widen(uv);
    swiglu8(gv, uv, h);
    if (it[u].in) store8<T, true, (STREAM > 0)>(static_cast<T*>(a.h) + it[u].row * a.ld_h + it[u].col, h, it[u].n);
    if (a.qg == nullptr) continue;   // no backward: h alone
    uint32_t gc, uc;
    const uint2 gb = act_encode8(gv, gc), ub = act_encode8(uv, uc);
    if (!it[u].in) continue;
    store_kept(a.qg, a.ld_q, a.cg, a.ld_c, it[u].row, it[u].col, gb, gc);
    store_kept(a.qu, a.ld_q, a.cu, a.ld_c, it[u].row, it[u].col, ub, uc);
  }
}

struct SwigluBwdArgs {
  const void* dh;
  int64_t ld_dh;
  Act8 g, u;
  void *dg, *du;
  int64_t ld_dg, ld_du;
};

template <typename T, int U, int STREAM>
__global__ __launch_bounds__(256) void swiglu_backward_kernel(Items t, SwigluBwdArgs a) {
  Item it[U];
  Eight<T> dh[U];
  uint2 g[U], up[U];
  uint32_t gc[U], uc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    it[u] = item_of<U>(t, u);
    g[u] = a.g.bytes(it[u].row, it[u].col);
    up[u] = a.u.bytes(it[u].row, it[u].col);
    gc[u] = a.g.code(it[u].row, it[u].col);
    uc[u] = a.u.code(it[u].row, it[u].col);
    dh[u].template load<true, (STREAM > 1)>(static_cast<const T*>(a.dh) + it[u].row * a.ld_dh + it[u].col, it[u].n);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float gv[8], uv[8], dv[8], dg[8], du[8];
    act_decode8(g[u], act_scale(gc[u]), gv);
    act_decode8(up[u], act_scale(uc[u]), uv);
    dh[u].widen(dv);
    swiglu8_backward(gv, uv, dv, dg, du);
    if (!it[u].in) continue;
    store8<T, true, (STREAM > 0)>(static_cast<T*>(a.dg) + it[u].row * a.ld_dg + it[u].col, dg, it[u].n);
    store8<T, true, (STREAM > 0)>(static_cast<T*>(a.du) + it[u].row * a.ld_du + it[u].col, du, it[u].n);
  }
}

// ---------------------------------------------------------------- RMSNorm ----
// A row sits in the registers of W waves: lane l of them holds columns 8 l .. + 8 and, of rows wider than 512, 8 l + 512 W .. + 8
// too.  Up to 512 columns a row takes L = 8, 16, 32 or 64 lanes of a wave, 64 / L rows side by side (1.6 M rows of 40: a whole wave to a
// row took 385 us forward and 415 backward, eight lanes 62 and 75); wider rows take a workgroup of W = ceil(D / 1024)
// waves each, so the lanes of any width are busy.  (One eight a lane and twice the waves was slower, 16384 rows of 7168:
// forward 132 us against 100, backward 162 against 129: fewer rows on a CU, and each waits for its slowest wave.)
struct NormArgs {
  const void* x;
  int64_t ld_x, T;
  int D;
  const void* w;
  float eps;
  void* y;
  int64_t ld_y;
  uint8_t* q;
  int64_t ld_q;
  uint8_t* codes;
  int64_t ld_c;
  float* rstd;
};

// Sum over a row's L lanes, or (L 0) its waves [first, + waves) of the workgroup's, in wave order; `parity` alternates between rows, so one barrier is enough.
template <int L>
__device__ __forceinline__ float row_sum(float v, float (*sums)[16], int parity, int first, int waves) {
  v = group_sum<L == 0 ? 64 : L>(v);
  if constexpr (L == 0) {
    if ((threadIdx.x & 63) == 0) sums[parity][threadIdx.x >> 6] = v;
    __syncthreads();
    v = sums[parity][first];
    for (int i = 1; i < waves; ++i) v += sums[parity][first + i];
  }
  return v;
}

template <typename T, typename WT, int NC, int L, bool TAIL, int STREAM>
__global__ __launch_bounds__(L > 0 ? 256 : 1024) void norm_kernel(NormArgs a) {
  __shared__ float sums[1][16];
  const int lane = L > 0 ? threadIdx.x & (L - 1) : threadIdx.x;
  const int step = int(blockDim.x) * 8;   // (of a second eight, of wide rows alone)
  const int64_t mine = L > 0 ? int64_t(blockIdx.x) * (256 / (L > 0 ? L : 1)) + threadIdx.x / (L > 0 ? L : 1) : int64_t(blockIdx.x);
  const bool in = mine < a.T;
  const int64_t row = in ? mine : a.T - 1;   // past the end: the last row again, not stored
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  Eight<T> xr[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) xr[c].template load<TAIL>(x + step * c + 8 * lane, a.D - (step * c + 8 * lane));
  Eight<WT> wr[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    wr[c].template load<TAIL>(static_cast<const WT*>(a.w) + step * c + 8 * lane, a.D - (step * c + 8 * lane));
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float v[8];
    xr[c].widen(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
  }
  ss = row_sum<L>(ss, sums, 0, 0, int(blockDim.x >> 6));
  const float r = 1.0f / sqrtf(ss / float(a.D) + a.eps);
  if (!in) return;
  if (lane == 0 && a.q) st_global(a.rstd + row, r);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = step * c + 8 * lane;
    if (col >= a.ld_q) break;
    float v[8], wv[8], yv[8];
    xr[c].widen(v);
    wr[c].widen(wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) yv[j] = (v[j] * r) * wv[j];
    store8<T, TAIL, (STREAM > 0)>(static_cast<T*>(a.y) + row * a.ld_y + col, yv, a.D - col);
    if (a.q == nullptr) continue;   // no backward: y alone
    uint32_t code;
    const uint2 b = act_encode8(v, code);
    store_kept(a.q, a.ld_q, a.codes, a.ld_c, row, col, b, code);
  }
}

// A workgroup of G teams of W waves takes the rows [slice * rps, + rps), a team every G-th of them, and writes the slice's share of
// dw: the teams' shares, added in order.  Eight waves or so to a workgroup, two of them to a CU: 16384 rows of 2048 take 65 us with one
// team to a workgroup (four waves to a CU), 35 with four.
struct NormBwdArgs {
  const void* dy;
  int64_t ld_dy;
  Act8 x;
  int64_t T;
  int D;
  const void* w;
  const float* rstd;
  void* dx;
  int64_t ld_dx;
  float* part;      // [slices, ld_p], or null: no dw
  int64_t ld_p, rps;
  int waves, teams;  // W and G
};

template <typename T, int NC, bool TAIL, int STREAM>
struct NormRow {
  uint2 q[NC];
  uint32_t code[NC];
  Eight<T> dy[NC];
  float r;
  // in: else a dy of zeros
  __device__ __forceinline__ void load(const NormBwdArgs& a, int64_t row, bool in, int lane, int step) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = step * c + 8 * lane;
      const int at = col < a.x.ld_q ? col : 0;   // behind the row: its first bytes, with a dy of zeros
      q[c] = a.x.bytes(row, at);
      code[c] = a.x.code(row, at);
      dy[c].template load<TAIL, (STREAM > 1)>(static_cast<const T*>(a.dy) + row * a.ld_dy + col, in ? a.D - col : 0);
    }
    r = a.rstd[row];
  }
};

template <typename T, typename WT, int NC, int L, bool TAIL, int STREAM>
__global__ __launch_bounds__(L > 0 ? 512 : 1024) void norm_backward_kernel(NormBwdArgs a) {
  extern __shared__ float4 shares4[];   // a team's dw [ld_p], if there are several
  __shared__ float sums[2][16];
  const int width = L > 0 ? L : 64 * a.waves;   // threads of a team
  const int team = int(threadIdx.x) / width, lane = int(threadIdx.x) - team * width;
  const int step = 8 * width;
  const int64_t r0 = int64_t(blockIdx.x) * a.rps, r1 = r0 + a.rps < a.T ? r0 + a.rps : a.T;
  const float inv_d = 1.0f / float(a.D);
  float wv[NC][8], pdw[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = step * c + 8 * lane;
    Eight<WT> wr;
    wr.template load<TAIL>(static_cast<const WT*>(a.w) + col, a.D - col);
    wr.widen(wv[c]);
#pragma unroll
    for (int j = 0; j < 8; ++j) pdw[c][j] = 0.f;
  }
  int parity = 0;
  // the next row's loads are in flight while this one is summed, where 128 registers hold both
  constexpr bool kNext = L > 0 || (sizeof(T) == 2 && !TAIL);
  NormRow<T, NC, TAIL, STREAM> n, next;
  // a team without a row of its own reads the slice's last one again, with a dy of zeros
  auto load = [&](NormRow<T, NC, TAIL, STREAM>& to, int64_t i) {
    const bool in = i + team < r1;
    to.load(a, in ? i + team : r1 - 1, in, lane, step);
  };
  if constexpr (kNext) load(next, r0);
  for (int64_t i = r0; i < r1; i += a.teams, parity ^= 1) {
    const int64_t row = i + team;
    if constexpr (kNext) {
      n = next;
      if (i + a.teams < r1) load(next, i + a.teams);
    } else {
      load(n, i);
    }
    // x r from the bytes in one product (s r is exact), and dx = r (a - (sum a x r / D) x r)
    float xr[NC][8], g[NC][8], dot = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      act_decode8(n.q[c], act_scale(n.code[c]) * n.r, xr[c]);
      n.dy[c].widen(g[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pdw[c][j] = fmaf(g[c][j], xr[c][j], pdw[c][j]);
        g[c][j] *= wv[c][j];
        dot = fmaf(g[c][j], xr[c][j], dot);
      }
    }
    const float m = row_sum<L>(dot, sums, parity, team * a.waves, a.waves) * inv_d;
    if (row >= r1) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = step * c + 8 * lane;
      if (col >= a.D) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) g[c][j] = n.r * fmaf(-m, xr[c][j], g[c][j]);
      store8<T, TAIL, (STREAM > 0)>(static_cast<T*>(a.dx) + row * a.ld_dx + col, g[c], a.D - col);
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + blockIdx.x * a.ld_p;   // ld_p is D rounded up to 8
  // the rows side by side in a wave, then waves (L > 0) or teams one after the other
  if constexpr (L > 0) {
#pragma unroll
    for (int off = L; off < 64; off <<= 1)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) pdw[c][j] += __shfl_xor(pdw[c][j], off);
  }
  const int turns = L > 0 ? int(blockDim.x >> 6) : a.teams, turn = L > 0 ? int(threadIdx.x >> 6) : team;
  const bool one = L == 0 || (threadIdx.x & 63) < (L > 0 ? L : 64);
  if (turns == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = step * c + 8 * lane;
      if (one && col < a.D) store8<float, false>(part + col, pdw[c], 8);
    }
    return;
  }
  for (int t = 0; t < turns; ++t) {
    if (t > 0) __syncthreads();
    if (turn != t || !one) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = step * c + 8 * lane;
      if (col >= a.D) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 v = make_float4(pdw[c][4 * h], pdw[c][4 * h + 1], pdw[c][4 * h + 2], pdw[c][4 * h + 3]);
        if (t > 0) {
          const float4 before = shares4[col / 4 + h];
          v = make_float4(before.x + v.x, before.y + v.y, before.z + v.z, before.w + v.w);
        }
        shares4[col / 4 + h] = v;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < int(a.ld_p) / 4; i += blockDim.x) st_global(part + 4 * i, shares4[i]);
}

// dw from the slices' shares: a workgroup takes 16 columns, 64 rows of threads every 64th slice each, then the sums of
// sixteen rows of a wave and of the four waves, in a fixed order.
template <typename WT>
__global__ __launch_bounds__(256) void norm_dw_kernel(const float* part, int64_t ld_p, int slices, int D, WT* dw) {
  __shared__ float4 acc[4][4];
  const int q = threadIdx.x & 3, g = threadIdx.x >> 2;
  const int col = blockIdx.x * 16 + q * 4;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < ld_p) {
#pragma unroll 4
    for (int s = g; s < slices; s += 64) {
      const float4 v = *reinterpret_cast<const float4*>(part + s * ld_p + col);
      t.x += v.x;
      t.y += v.y;
      t.z += v.z;
      t.w += v.w;
    }
  }
#pragma unroll
  for (int off = 4; off < 64; off <<= 1) {
    t.x += __shfl_xor(t.x, off);
    t.y += __shfl_xor(t.y, off);
    t.z += __shfl_xor(t.z, off);
    t.w += __shfl_xor(t.w, off);
  }
  if ((threadIdx.x & 63) < 4) acc[threadIdx.x >> 6][q] = t;
  __syncthreads();
  const int c = blockIdx.x * 16 + threadIdx.x;
  if (threadIdx.x >= 16 || c >= D) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += reinterpret_cast<const float*>(&acc[i][0])[threadIdx.x];
  if constexpr (sizeof(WT) == 2) st_global(dw + c, f32_to_bf16(s));
  else st_global(dw + c, s);
}

// ----------------------------------------------------------------- launches ----
constexpr int64_t kMaxItems = int64_t(1) << 30;   // of one launch; longer matrices go in runs of rows
constexpr int64_t kMaxCols = (int64_t(1) << 24) - 1;   // 128 rows stay below twice that
constexpr int kNormMaxD = 16384;

// Calls go(items, unroll tag, workgroups) over the eights of a [rows, cols] matrix.  Four eights a thread keep 64
// bytes a lane in flight; a matrix that then leaves CUs without two workgroups takes one a thread.
template <int UMAX, int EACH = 8, typename F>
int for_items(int64_t rows, int64_t cols, F go) {
  const int64_t per = (cols + kActBlock - 1) / kActBlock * (kActBlock / EACH);
  int64_t run = kMaxItems / per;
  run = run < 128 ? run : run / 128 * 128;   // whole 128-row tiles
  for (int64_t r = 0; r < rows; r += run) {
    const int64_t n = (rows - r < run ? rows - r : run) * per;
    const Items t{FastDiv(uint32_t(per)), uint32_t(n), r, int(cols)};
    if (n >= int64_t(512) * UMAX * device_cus()) go(t, std::integral_constant<int, UMAX>{}, unsigned((n + 256 * UMAX - 1) / (256 * UMAX)));
    else go(t, std::integral_constant<int, 1>{}, unsigned((n + 255) / 256));
  }
  return 0;
}

// go(tag of the level, one of LEVELS)
template <int... LEVELS, typename F>
void for_stream(int64_t bytes, F go) {
  const int level = stream_level(bytes);
  int best = 0;
  ((best = LEVELS <= level ? LEVELS : best), ...);
  ((best == LEVELS ? go(std::integral_constant<int, LEVELS>{}) : void()), ...);
}

template <typename F>
void for_dtype(int dtype, F go) {
  if (dtype == FM_DTYPE_BF16) go(uint16_t{});
  else go(float{});
}

bool dtype_ok(int d) { return d == FM_DTYPE_BF16 || d == FM_DTYPE_F32; }

// ---- the norm's shapes
int norm_waves(int64_t D) { return int((D + 1023) / 1024); }
// Lanes of a narrow row, 0 for a wide one's waves.
int norm_lanes(int64_t D) { return D > 512 ? 0 : D > 256 ? 64 : D > 128 ? 32 : D > 64 ? 16 : 8; }
// Waves of a workgroup of the backward, and its teams (rows side by side): the fewest while 512 workgroups take all rows at once; else
// eight waves or so, one round of the workgroups that fit (sixteen waves to a CU), but no more than 512 of them: each writes D sums
// that the second launch reads.
int norm_group_waves(int64_t T, int64_t D) {
  const int w = D <= 512 ? 1 : norm_waves(D);
  return T <= 512 || w > 4 ? w : 8 / w * w;
}
int norm_teams(int64_t T, int64_t D) {
  const int waves = norm_group_waves(T, D);
  return D <= 512 ? waves * 64 / norm_lanes(D) : waves / norm_waves(D);
}
int64_t norm_rows_per_slice(int64_t T, int64_t D) {
  const int teams = norm_teams(T, D);
  int64_t most = int64_t(device_cus()) * (16 / norm_group_waves(T, D));
  most = most < 512 ? most : 512;
  const int64_t r = (T + most - 1) / most;
  return (r + teams - 1) / teams * teams;
}

// go(eights a lane, lanes of a row (0: waves), a width that is no multiple of 8)
template <typename F>
void for_norm(int64_t D, F go) {
  auto with_tail = [&](auto nc, auto lanes) {
    if (D % 8) go(nc, lanes, std::true_type{});
    else go(nc, lanes, std::false_type{});
  };
  using one = std::integral_constant<int, 1>;
  switch (norm_lanes(D)) {
    case 8: with_tail(one{}, std::integral_constant<int, 8>{}); break;
    case 16: with_tail(one{}, std::integral_constant<int, 16>{}); break;
    case 32: with_tail(one{}, std::integral_constant<int, 32>{}); break;
    case 64: with_tail(one{}, std::integral_constant<int, 64>{}); break;
    default: with_tail(std::integral_constant<int, 2>{}, std::integral_constant<int, 0>{}); break;
  }
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" {

int fm_act8_compress(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld_x, void* q, int64_t ld_q, void* codes,
                     int64_t ld_c, const int32_t* tile_valid, void* stream) {
  FM_REQUIRE(rows >= 0 && cols >= 1 && cols <= kMaxCols, "fm_act8_compress: bad sizes");
  FM_REQUIRE(dtype_ok(x_dtype), "fm_act8_compress: x must be bf16 or fp32");
  if (rows == 0) return 0;
  FM_REQUIRE(x && ld_x >= 0, "fm_act8_compress: null x or negative pitch");
  FM_REQUIRE(kept_ok(q, ld_q, codes, ld_c, cols) && ld_q == (cols + 31) / 32 * 32, "fm_act8_compress: the payload's pitch is cols rounded up to 32, "
             "on 8 bytes, a code to 32 columns");
  const CompressArgs a{x, ld_x, static_cast<uint8_t*>(q), ld_q, static_cast<uint8_t*>(codes), ld_c, tile_valid};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for_dtype(x_dtype, [&](auto t) {
    for_stream<0, 2>(rows * cols * int64_t(sizeof(t)), [&](auto stream_) {
      for_items<4>(rows, cols, [&](const Items& items, auto u, unsigned wgs) {
        hipLaunchKernelGGL((compress_kernel<decltype(t), decltype(u)::value, decltype(stream_)::value>), dim3(wgs), dim3(256), 0, s, items, a);
      });
    });
  });
  return check_launch("fm_act8_compress");
}

int fm_act8_restore(const void* q, int64_t ld_q, const void* codes, int64_t ld_c, int64_t src_rows, int64_t cols, const int32_t* index,
                    int64_t rows, void* out, int out_dtype, int64_t ld_out, void* stream) {
  FM_REQUIRE(rows >= 0 && src_rows >= 0 && cols >= 1 && cols <= kMaxCols, "fm_act8_restore: bad sizes");
  FM_REQUIRE(dtype_ok(out_dtype), "fm_act8_restore: the output must be bf16 or fp32");
  FM_REQUIRE(index || rows <= src_rows, "fm_act8_restore: more rows than there are");
  if (rows == 0) return 0;
  FM_REQUIRE(out && ld_out >= cols, "fm_act8_restore: null output or a pitch below cols");
  FM_REQUIRE(src_rows == 0 || kept_ok(q, ld_q, codes, ld_c, cols), "fm_act8_restore: bad payload, codes or pitches");
  const RestoreArgs a{Act8{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(codes), ld_q, ld_c}, index, src_rows, out, ld_out};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for_dtype(out_dtype, [&](auto t) {
    for_stream<0, 1>(rows * cols * int64_t(sizeof(t)), [&](auto stream_) {
      constexpr int kStream = decltype(stream_)::value;
      for_items<4, 16 / sizeof(t)>(rows, cols, [&](const Items& items, auto u, unsigned wgs) {
        constexpr int U = decltype(u)::value;
        if (index) hipLaunchKernelGGL((restore_kernel<decltype(t), U, true, kStream>), dim3(wgs), dim3(256), 0, s, items, a);
        else hipLaunchKernelGGL((restore_kernel<decltype(t), U, false, kStream>), dim3(wgs), dim3(256), 0, s, items, a);
      });
    });
  });
  return check_launch("fm_act8_restore");
}

int fm_act8_swiglu(const void* g, int64_t ld_g, const void* u, int64_t ld_u, int dtype, int64_t rows, int64_t H, void* h, int64_t ld_h,
                   void* qg, void* cg, void* qu, void* cu, int64_t ld_q, int64_t ld_c, void* stream) {
  FM_REQUIRE(rows >= 0 && H >= 1 && H <= kMaxCols, "fm_act8_swiglu: bad sizes");
  FM_REQUIRE(dtype_ok(dtype), "fm_act8_swiglu: gate and up must be bf16 or fp32");
  if (rows == 0) return 0;
  FM_REQUIRE(g && u && h && ld_g >= 0 && ld_u >= 0 && ld_h >= H, "fm_act8_swiglu: null pointer or bad pitch");
  const bool keep = qg || cg || qu || cu;
  FM_REQUIRE(!keep || (kept_ok(qg, ld_q, cg, ld_c, H) && kept_ok(qu, ld_q, cu, ld_c, H)), "fm_act8_swiglu: bad payload, codes or pitches");
  const SwigluArgs a{g, u, ld_g, ld_u, h, ld_h, static_cast<uint8_t*>(qg), static_cast<uint8_t*>(qu), static_cast<uint8_t*>(cg),
                     static_cast<uint8_t*>(cu), ld_q, ld_c};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for_dtype(dtype, [&](auto t) {
    for_stream<0, 1>(rows * H * int64_t(sizeof(t)), [&](auto stream_) {
      for_items<2>(rows, H, [&](const Items& items, auto n, unsigned wgs) {
        hipLaunchKernelGGL((swiglu_kernel<decltype(t), decltype(n)::value, decltype(stream_)::value>), dim3(wgs), dim3(256), 0, s, items, a);
      });
    });
  });
  return check_launch("fm_act8_swiglu");
}

int fm_act8_swiglu_backward(const void* dh, int64_t ld_dh, int dtype, int64_t rows, int64_t H, const void* qg, const void* cg, const void* qu,
                            const void* cu, int64_t ld_q, int64_t ld_c, void* dg, int64_t ld_dg, void* du, int64_t ld_du, void* stream) {
  FM_REQUIRE(rows >= 0 && H >= 1 && H <= kMaxCols, "fm_act8_swiglu_backward: bad sizes");
  FM_REQUIRE(dtype_ok(dtype), "fm_act8_swiglu_backward: dh must be bf16 or fp32");
  if (rows == 0) return 0;
  FM_REQUIRE(dh && dg && du && ld_dh >= 0 && ld_dg >= H && ld_du >= H, "fm_act8_swiglu_backward: null pointer or bad pitch");
  FM_REQUIRE(kept_ok(qg, ld_q, cg, ld_c, H) && kept_ok(qu, ld_q, cu, ld_c, H), "fm_act8_swiglu_backward: bad payload, codes or pitches");
  const SwigluBwdArgs a{dh, ld_dh, Act8{static_cast<const uint8_t*>(qg), static_cast<const uint8_t*>(cg), ld_q, ld_c},
                        Act8{static_cast<const uint8_t*>(qu), static_cast<const uint8_t*>(cu), ld_q, ld_c}, dg, du, ld_dg, ld_du};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for_dtype(dtype, [&](auto t) {
    for_stream<0, 1, 2>(rows * H * int64_t(sizeof(t)), [&](auto stream_) {
      for_items<2>(rows, H, [&](const Items& items, auto n, unsigned wgs) {
        hipLaunchKernelGGL((swiglu_backward_kernel<decltype(t), decltype(n)::value, decltype(stream_)::value>), dim3(wgs), dim3(256), 0, s,
                           items, a);
      });
    });
  });
  return check_launch("fm_act8_swiglu_backward");
}

int fm_act8_rmsnorm(const void* x, int dtype, int64_t ld_x, int64_t T, int64_t D, const void* w, int w_dtype, float eps, void* y, int64_t ld_y,
                    void* q, int64_t ld_q, void* codes, int64_t ld_c, float* rstd, void* stream) {
  FM_REQUIRE(T >= 0 && T < (int64_t(1) << 31) && D >= 1 && D <= kNormMaxD, "fm_act8_rmsnorm: D must be 1 to %d, T below 2^31", kNormMaxD);
  FM_REQUIRE(dtype_ok(dtype) && dtype_ok(w_dtype), "fm_act8_rmsnorm: x and the weight must be bf16 or fp32");
  if (T == 0) return 0;
  const bool keep = q || codes || rstd;
  FM_REQUIRE(x && w && y && (rstd || !keep) && ld_x >= 0 && ld_y >= D, "fm_act8_rmsnorm: null pointer or bad pitch");
  FM_REQUIRE(ld_q == (D + 31) / 32 * 32 && (!keep || kept_ok(q, ld_q, codes, ld_c, D)), "fm_act8_rmsnorm: bad payload, codes or pitches");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int lanes = norm_lanes(D), threads = lanes ? 256 : 64 * norm_waves(D), rows = lanes ? 256 / lanes : 1;   // of a workgroup
  const int64_t run = (int64_t(1) << 31) / threads * rows;   // a launch has fewer than 2^32 threads
  for (int64_t r = 0; r < T; r += run) {
    const int64_t n = T - r < run ? T - r : run;
    for_dtype(dtype, [&](auto t) {
      const NormArgs a{static_cast<const decltype(t)*>(x) + r * ld_x, ld_x, n, int(D), w, eps, static_cast<decltype(t)*>(y) + r * ld_y, ld_y,
                       keep ? static_cast<uint8_t*>(q) + r * ld_q : nullptr, ld_q, keep ? static_cast<uint8_t*>(codes) + r * ld_c : nullptr, ld_c,
                       keep ? rstd + r : nullptr};
      for_dtype(w_dtype, [&](auto wt) {
        for_norm(D, [&](auto nc, auto l, auto tail) {
          for_stream<0, 1>(T * D * int64_t(sizeof(t)), [&](auto stream_) {
            hipLaunchKernelGGL((norm_kernel<decltype(t), decltype(wt), decltype(nc)::value, decltype(l)::value, decltype(tail)::value,
                                            decltype(stream_)::value>),
                               dim3(unsigned((n + rows - 1) / rows)), dim3(threads), 0, s, a);
          });
        });
      });
    });
  }
  return check_launch("fm_act8_rmsnorm");
}

int64_t fm_act8_rmsnorm_backward_workspace_bytes(int64_t T, int64_t D) {
  if (T <= 0 || D <= 0) return 0;
  const int64_t rps = norm_rows_per_slice(T, D);
  return (T + rps - 1) / rps * ((D + 7) / 8 * 8) * int64_t(sizeof(float));
}

int fm_act8_rmsnorm_backward(const void* dy, int64_t ld_dy, int dtype, int64_t T, int64_t D, const void* q, int64_t ld_q, const void* codes,
                             int64_t ld_c, const void* w, int w_dtype, const float* rstd, void* dx, int64_t ld_dx, void* dw,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  FM_REQUIRE(T >= 1 && T < (int64_t(1) << 31) && D >= 1 && D <= kNormMaxD, "fm_act8_rmsnorm_backward: D must be 1 to %d, T 1 to 2^31 - 1", kNormMaxD);
  FM_REQUIRE(dtype_ok(dtype) && dtype_ok(w_dtype), "fm_act8_rmsnorm_backward: dy and the weight must be bf16 or fp32");
  FM_REQUIRE(dy && w && rstd && dx && ld_dy >= 0 && ld_dx >= D, "fm_act8_rmsnorm_backward: null pointer or bad pitch");
  FM_REQUIRE(kept_ok(q, ld_q, codes, ld_c, D), "fm_act8_rmsnorm_backward: bad payload, codes or pitches");
  FM_REQUIRE(dw == nullptr || (workspace && aligned16(workspace) && workspace_bytes >= fm_act8_rmsnorm_backward_workspace_bytes(T, D)),
             "fm_act8_rmsnorm_backward: dw needs a workspace of fm_act8_rmsnorm_backward_workspace_bytes(T, D) bytes on 16");
  const int64_t rps = norm_rows_per_slice(T, D), slices = (T + rps - 1) / rps, ld_p = (D + 7) / 8 * 8;
  const int waves = norm_group_waves(T, D), turns = D <= 512 ? waves : norm_teams(T, D);   // shares of dw that meet in LDS
  float* part = static_cast<float*>(workspace);
  const NormBwdArgs a{dy, ld_dy, Act8{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(codes), ld_q, ld_c}, T, int(D), w, rstd,
                      dx, ld_dx, dw ? part : nullptr, ld_p, rps, D <= 512 ? 1 : norm_waves(D), norm_teams(T, D)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for_dtype(dtype, [&](auto t) {
    for_dtype(w_dtype, [&](auto wt) {
      for_norm(D, [&](auto nc, auto l, auto tail) {
        for_stream<0, 1, 2>(T * D * int64_t(sizeof(t)), [&](auto stream_) {
          hipLaunchKernelGGL((norm_backward_kernel<decltype(t), decltype(wt), decltype(nc)::value, decltype(l)::value, decltype(tail)::value,
                                                   decltype(stream_)::value>),
                             dim3(unsigned(slices)), dim3(64 * waves), dw && turns > 1 ? unsigned(ld_p * 4) : 0u, s, a);
        });
      });
    });
  });
  if (int rc = check_launch("fm_act8_rmsnorm_backward")) return rc;
  if (dw == nullptr) return 0;
  for_dtype(w_dtype, [&](auto wt) {
    using WT = decltype(wt);
    hipLaunchKernelGGL(norm_dw_kernel<WT>, dim3(unsigned((D + 15) / 16)), dim3(256), 0, s, part, ld_p, int(slices), int(D), static_cast<WT*>(dw));
  });
  return check_launch("fm_act8_rmsnorm_backward");
}

}  // extern "C"
