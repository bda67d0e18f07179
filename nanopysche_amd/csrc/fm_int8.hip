// Products in 8-bit integers with a scale for each token and each channel:
//
//   s_r = max(max_k |x_rk|, 1e-12) / 127,  q_rk = rint(x_rk / s_r)        (rows of an operand)
//   out[t, n] = (sum_k qx[t, k] qw[n, k]) sx[t] sw[n] (+ bias[n])
//
// and their forms over a routing plan's groups, with SwiGLU behind the gate|up product.
// The sums are int32, exact for K < 2^17, so a product does not depend on how it is cut.
// s and x / s are rounded fp32 quotients: an x of exactly half its row's maximum (one bf16 element
// in 800) lies at 63.5 steps and becomes 63 or 64 as the last bit of s falls (64 in 95% of them).
// A row that holds a NaN or an infinity gets that scale and zero payload: its outputs are NaN.
//
// Layout.  An operand [R, K] lies in tiles of 16 rows x 64 columns, 1 KiB each, in the
// order of the matrix cores' fragments: element (r, k) of tile (r / 16, k / 64) at byte
// (k % 64 / 16 * 16 + r % 16) * 16 + k % 16, tiles of a row of tiles one after the other,
// R padded to 16 and K to 128 with zeros.  Every load of a wave, from memory to LDS and
// from LDS or memory to registers, then takes 1 KiB in order: whole lines, no bank
// conflicts, no swizzle, and odd sizes need no bounds in the loops.
#include <type_traits>

#include "fm_common.h"
#include "fm_dma.h"
#include "../../include/fm_hip.h"

namespace fm {

namespace {

constexpr int kMaxK = 131072;   // K below this: 127 * 127 K (and 128 * 128 K - 1 step) fits int32

// 16 bytes at any address of the element's alignment
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// ---------------------------------------------------------------- quantise ----
struct QuantArgs {
  const void* x;
  int64_t ld, R, C;
  const int32_t* assign;   // row r of the output is row assign[r] / top_k of x (negative: zeros); null: row r
  int top_k;
  const int32_t* limit;    // rows from *limit on are left alone; null: none
  const uint32_t* top;     // the rows' largest magnitudes as bits where they are known, or null
  uint32_t* clear;         // [rows, padded to 16] set to 0, or null
  uint8_t* q;
  float* s;
  int kt;
};

// 16 elements of a row from column c on, as bits, zeros from column C on.
template <bool F32>
struct Raw {
  fm_u32x4 v[F32 ? 4 : 2];
  __device__ __forceinline__ void load(const void* row, int64_t c, int64_t C) {
    constexpr int kEach = F32 ? 4 : 8;
    if (c + 16 <= C) {
#pragma unroll
      for (int i = 0; i < 16 / kEach; ++i)
        v[i] = *FM_GLOBAL(const u32x4_any, static_cast<const uint8_t*>(row) + (c + i * kEach) * (F32 ? 4 : 2));
      return;
    }
#pragma unroll
    for (int i = 0; i < 16 / kEach; ++i) v[i] = fm_u32x4{0, 0, 0, 0};
    if (c >= C) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (c + i >= C) break;
      if constexpr (F32) v[i / 4][i % 4] = f2u(*FM_GLOBAL(const float, static_cast<const float*>(row) + c + i));
      else v[i / 8][i / 2 % 4] |= uint32_t(*FM_GLOBAL(const uint16_t, static_cast<const uint16_t*>(row) + c + i)) << (i % 2 * 16);
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (F32) return u2f(v[i / 4][i % 4]);
    else return u2f(i % 2 ? v[i / 8][i / 2 % 4] & 0xffff0000u : v[i / 8][i / 2 % 4] << 16);
  }
  // the largest magnitude as bits: a NaN is above infinity, infinity above every number
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t b = v[i / 4][i % 4] & 0x7fffffffu;
        m = b > m ? b : m;
      }
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 t = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, v[i / 4][i % 4] & 0x7fff7fffu));
      const uint32_t b = uint32_t(t[0] > t[1] ? t[0] : t[1]) << 16;
      m = b > m ? b : m;
    }
    return m;
  }
};

__device__ __forceinline__ float int8_scale(uint32_t top) {
  return top <= 0x7f7fffffu ? fmaxf(u2f(top), kAmaxFloor) / 127.0f : u2f(top);
}
// 16 quotients rounded to whole numbers as bytes; `finite`: else zeros
template <bool F32>
__device__ __forceinline__ fm_u32x4 int8_round(const Raw<F32>& v, Recip d, bool finite) {
  fm_u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t b[4];
    // adding 1.5 * 2^23 rounds to the nearest whole number (ties to even) in the low byte
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = f2u(div_rn(v.at(4 * i + j), d) + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    o[i] = finite ? lo | hi : 0u;
  }
  return o;
}

// A workgroup takes RW rows, a lane 16 columns of one row, a wave 64 / RW such chunks side by
// side: of 16 rows a tile's payload leaves in one 1 KiB store, of 4 in pieces of 64 bytes.  The NT
// chunks of a lane stay in registers between the maximum and the rounding (NT = 0: read
// twice).  GIVEN: the maxima are known, and gridDim.y workgroups share the columns.  Bound:
// reading x and writing q once (8192 x 4096 bf16 in 20.4 us, 4.9 TB/s), by few rows what a CU
// can have in flight.  So a workgroup takes 2 or 4 rows while no more workgroups than CUs come
// of it, else 8.  us with 16 / 8 / 4 / 2 rows: 16 x 4096 bf16 7.4 / 4.9 / 3.6 / 3.0; 64 x 14336
// 28.7 / 11.9 / 7.1 / 4.3; 512 x 14336 29.7 / 13.4 / 8.6 / 7.6; 1024 x 8192 14.8 / 9.3 / 7.5 / 7.9;
// 1409 x 2817 fp32 9.6 / 6.7 / 6.8 / 7.1; 2048 x 14336 36.9 / 19.8 / 21.9 / 25.0; 8192 x 4096 20.4 /
// 20.4 / 21.9 / 27.8; 16384 x 2048 20.9 / 18.8 / 20.9 / 28.6.
constexpr int kQuantWaves = 8;
template <bool F32, int NT, bool GIVEN, int RW>
__global__ __launch_bounds__(64 * kQuantWaves) void int8_quant_kernel(QuantArgs a) {
  constexpr int kSide = 64 / RW;
  __shared__ uint32_t tops[kQuantWaves][RW];
  const int lane = threadIdx.x & 63, r = lane % RW, wave = threadIdx.x >> 6;
  const int64_t r0 = int64_t(blockIdx.x) * RW;
  if (a.limit && r0 >= *a.limit) return;
  if (a.clear && threadIdx.x < RW) st_global(a.clear + r0 + threadIdx.x, 0u);
  int64_t src = r0 + r;
  bool valid = src < a.R;
  if (a.assign) {
    const int as = valid ? a.assign[src] : -1;
    valid = as >= 0;
    src = valid ? as / a.top_k : 0;
  }
  if (!valid) src = 0;
  const void* row = static_cast<const uint8_t*>(a.x) + src * a.ld * (F32 ? 4 : 2);
  const int64_t C = valid ? a.C : 0;
  const int n = a.kt * 4, c0 = wave * kSide + lane / RW, step = kQuantWaves * kSide;   // chunks of a row; the lane's are c0 + step i
  uint8_t* const q = a.q + (r0 / 16 * a.kt * 64 + r0 % 16 + r) * 16;
  auto put = [&](const Raw<F32>& v, Recip d, bool finite, int c) {
    const fm_u32x4 o = int8_round(v, d, finite);
    st_global(q + int64_t(c) * 256, make_uint4(o[0], o[1], o[2], o[3]));
  };
  if constexpr (GIVEN) {
    const uint32_t top = valid ? a.top[r0 + r] : 0u;
    const float s = int8_scale(top);
    if (blockIdx.y == 0 && threadIdx.x < RW && r0 + r < a.R) st_global(a.s + r0 + r, s);
    const Recip d = recip_of(s);
    const int64_t read = top ? C : 0;   // a row of zeros (a plan's padding) need not be there
#pragma unroll 4
    for (int c = c0 + step * blockIdx.y; c < n; c += step * gridDim.y) {
      Raw<F32> v;
      v.load(row, int64_t(c) * 16, read);
      put(v, d, top <= 0x7f7fffffu, c);
    }
  } else {
    Raw<F32> held[NT ? NT : 1];
    uint32_t top = 0;
    if constexpr (NT > 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i) held[i].load(row, int64_t(c0 + step * i) * 16, C);
#pragma unroll
      for (int i = 0; i < NT; ++i) top = held[i].top(top);
    } else {
#pragma unroll 4
      for (int c = c0; c < n; c += step) {
        Raw<F32> v;
        v.load(row, int64_t(c) * 16, C);
        top = v.top(top);
      }
    }
#pragma unroll
    for (int off = RW; off < 64; off <<= 1) {
      const uint32_t o = __shfl_xor(top, off);
      top = o > top ? o : top;
    }
    if (lane < RW) tops[wave][r] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantWaves; ++w) top = tops[w][r] > top ? tops[w][r] : top;
    const float s = int8_scale(top);
    const bool finite = top <= 0x7f7fffffu;
    if (threadIdx.x < RW && r0 + r < a.R) st_global(a.s + r0 + r, valid ? s : 0.f);   // 0 marks a plan's padding
    const Recip d = recip_of(s);
    if constexpr (NT > 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (c0 + step * i < n) put(held[i], d, finite, c0 + step * i);
    } else {
#pragma unroll 2
      for (int c = c0; c < n; c += step) {
        Raw<F32> v;
        v.load(row, int64_t(c) * 16, C);
        put(v, d, finite, c);
      }
    }
  }
}

// Int8 values (any strides, in bytes) into tiles, groups one after the other, a tile a wave.
// Rows of contiguous columns: a lane's 16 bytes in one load.  Columns of contiguous rows (w2 as
// the expert block stores it): a lane loads the tile's 16 rows of one column, and the wave
// turns them in LDS.  A byte at a time otherwise and at the edges.  us for 8 x 14336 x 4096
// (470 MB): rows 160, columns 246; by bytes 840 and 560, and 670 to 880 with a gap between.
__global__ __launch_bounds__(256) void int8_pack_kernel(const uint8_t* x, int64_t gs, int64_t rs, int64_t cs, int64_t R, int64_t C,
                                                        int kt, int64_t tiles, uint8_t* q) {
  __shared__ __attribute__((aligned(16))) uint8_t turn[4][64 * 20];   // 20 bytes a column: 64 columns' dwords on distinct banks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int64_t t = int64_t(blockIdx.x) * 4 + wave;
  if (t >= tiles) return;
  const int64_t rt = (R + 15) / 16, g = t / (rt * kt), r0 = t / kt % rt * 16, c0 = t % kt * 64;
  const int64_t r = r0 + (lane & 15), c = c0 + (lane >> 4) * 16;
  uint32_t o[4] = {0, 0, 0, 0};
  if (cs != 1 && rs == 1 && r0 + 16 <= R && c0 + 64 <= C) {
    const fm_u32x4 v = *FM_GLOBAL(const u32x4_any, x + g * gs + r0 + (c0 + lane) * cs);
    uint8_t* mine = turn[wave];
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(mine + lane * 20 + 4 * i) = v[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // LDS keeps a wave's order
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i / 4] |= uint32_t(mine[((lane >> 4) * 16 + i) * 20 + (lane & 15)]) << (i % 4 * 8);
  } else if (r < R) {
    const uint8_t* p = x + g * gs + r * rs;
    if (cs == 1 && c + 16 <= C) {
      const fm_u32x4 v = *FM_GLOBAL(const u32x4_any, p + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < C) o[i / 4] |= uint32_t(*FM_GLOBAL(const uint8_t, p + (c + i) * cs)) << (i % 4 * 8);
    }
  }
  st_global(q + (t * 64 + lane) * 16, make_uint4(o[0], o[1], o[2], o[3]));
}

// Tiles back to rows: q s as bf16 or fp32, or q itself.
enum Unpacked : int { UP_BF16 = FM_INT8_TO_BF16, UP_F32 = FM_INT8_TO_F32, UP_I8 = FM_INT8_TO_I8 };
template <int OUT>
__global__ __launch_bounds__(256) void int8_unpack_kernel(const uint8_t* q, const float* s, int64_t R, int64_t C, int kt,
                                                          int64_t tiles, uint8_t* out, int64_t ld) {
  constexpr int kSize = OUT == UP_BF16 ? 2 : OUT == UP_F32 ? 4 : 1;
  const int lane = threadIdx.x & 63;
  const int64_t t = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= tiles) return;
  const int64_t r = t / kt * 16 + (lane & 15), c = t % kt * 64 + (lane >> 4) * 16;
  const fm_u32x4 v = *FM_GLOBAL(const fm_u32x4, q + (t * 64 + lane) * 16);
  if (r >= R || c >= C) return;
  fm_u32x4 o[kSize];
  if constexpr (OUT == UP_I8) {
    o[0] = v;
  } else {
    const float sc = s[r];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = float(int8_t(v[i] >> (8 * j))) * sc;
      if constexpr (OUT == UP_F32) {
        o[i] = fm_u32x4{f2u(f[0]), f2u(f[1]), f2u(f[2]), f2u(f[3])};
      } else {
        o[i / 2][i % 2 * 2] = hw_bf16x2(f[0], f[1]);
        o[i / 2][i % 2 * 2 + 1] = hw_bf16x2(f[2], f[3]);
      }
    }
  }
  uint8_t* p = out + (r * ld + c) * kSize;
  if (c + 16 <= C) {
#pragma unroll
    for (int i = 0; i < kSize; ++i) *FM_GLOBAL(u32x4_any, p + 16 * i) = o[i];
    return;
  }
  const int left = int(C - c);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (i >= left) continue;
    const int at = i * kSize;
    const uint32_t w = o[at / 16][at / 4 % 4];
    if constexpr (OUT == UP_F32) *FM_GLOBAL(uint32_t, p + at) = w;
    else if constexpr (OUT == UP_BF16) *FM_GLOBAL(uint16_t, p + at) = uint16_t(w >> (at % 4 * 8));
    else *FM_GLOBAL(uint8_t, p + at) = uint8_t(w >> (at % 4 * 8));
  }
}

// 4 scales or biases of channels from n on (n a multiple of 4), zeros from N on.
__device__ __forceinline__ v4f four_of(const float* p, int64_t n, int64_t N) {
  typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
  if (n + 4 <= N) return *FM_GLOBAL(const v4f_any, p + n);
  v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (n + i < N) v[i] = *FM_GLOBAL(const float, p + n + i);
  return v;
}

// ------------------------------------------------------------ few tokens ----
// out[t, n], bound by reading the weights once for up to 32 tokens and by the latency of a
// chain over K for more.  A workgroup owns 16 channels and TF tiles of 16 tokens; its 4 waves
// take a quarter of K each, tiles straight from memory into 16x16x64 MFMA fragments, U of them
// in flight beside the ones in use, and the four int32 sums meet in LDS.  More tokens are
// further passes over the weights.
struct ProductArgs {
  const uint8_t *a, *w, *w2;   // tiles of tokens and channels; w2: SwiGLU's up rows (else null)
  const float *sa, *sw, *sw2;
  int64_t w_gs, sw_gs;         // of an expert: bytes, scales
  int kt;
  int64_t M, N;                // rows of tokens (padded groups: of the buffer), channels (SwiGLU: hidden units)
  const int32_t* offsets;      // [E + 1] group starts, or null: one group of M rows
  int E;
  const float* bias;
  void* out;
  int64_t ld_out;
  int out_f32;
  uint32_t* top;               // SwiGLU: the rows' largest |h| as bits, raised by every wave
};

// QUANT 1 (bf16) or 2 (fp32): the tokens (at most kFusedRows) come as floats and every
// workgroup quantises them into LDS while its first weights are on their way: a launch and
// a round trip through memory fewer, for 2 or 4 M K bytes more from the caches a workgroup.
constexpr int kFusedRows = 4, kFusedBytes = 32 * 1024;
struct FusedRows {
  const void* x;
  int64_t ld, K;
};

template <bool F32>
__device__ __forceinline__ void quantise_rows(const FusedRows& x, int M, int kt, uint8_t* q, float* scale, uint32_t (*tops)[kFusedRows]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunks = kt * 4;
  for (int r = 0; r < M; ++r) {
    const void* row = static_cast<const uint8_t*>(x.x) + r * x.ld * (F32 ? 4 : 2);
    uint32_t top = 0;
    for (int c = tid; c < chunks; c += 256) {
      Raw<F32> v;
      v.load(row, int64_t(c) * 16, x.K);
      top = v.top(top);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = __shfl_xor(top, off);
      top = o > top ? o : top;
    }
    if (lane == 0) tops[wave][r] = top;
  }
  __syncthreads();
  for (int r = 0; r < M; ++r) {
    const void* row = static_cast<const uint8_t*>(x.x) + r * x.ld * (F32 ? 4 : 2);
    uint32_t top = tops[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = tops[w][r] > top ? tops[w][r] : top;
    const float s = int8_scale(top);
    if (tid == 0) scale[r] = s;
    const Recip d = recip_of(s);
    for (int c = tid; c < chunks; c += 256) {
      Raw<F32> v;
      v.load(row, int64_t(c) * 16, x.K);
      *reinterpret_cast<fm_u32x4*>(q + (r * chunks + c) * 16) = int8_round(v, d, top <= 0x7f7fffffu);
    }
  }
  __syncthreads();
}

template <int TF, int QUANT>
__global__ __launch_bounds__(256) void int8_few_kernel(ProductArgs p, FusedRows x, int passes) {
  __shared__ v4i red[3][TF][64];
  __shared__ __attribute__((aligned(16))) uint8_t held[QUANT ? kFusedBytes : 16];
  __shared__ float held_scale[kFusedRows];
  __shared__ uint32_t tops[4][kFusedRows];
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  // an XCD takes a run of channel tiles with all of their passes, so its L2 holds the weights for
  // them; weights that are read once go in order (1 x 4096 -> 14336: 11.6 us, in runs 12.4)
  const int64_t id = passes == 1 ? blockIdx.x : int64_t(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8, nt = id / passes;
  if (nt * 16 >= p.N) return;
  const int t0 = int(id % passes) * TF, last = int((p.M - 1) / 16);   // token tiles
  const int k0 = p.kt * wave / 4, k1 = p.kt * (wave + 1) / 4;
  constexpr int U = TF == 1 ? 8 : 4;
  const uint8_t* w = p.w + (nt * p.kt * 64 + lane) * 16;
  const uint8_t* a[TF];
#pragma unroll
  for (int f = 0; f < TF; ++f) a[f] = p.a + (int64_t(t0 + f < last ? t0 + f : last) * p.kt * 64 + lane) * 16;
  const uint8_t* mine = held + ((m < p.M ? m : 0) * p.kt * 4 + q) * 16;
  v4i acc[TF];
#pragma unroll
  for (int f = 0; f < TF; ++f) acc[f] = v4i{0, 0, 0, 0};
  v4i wv[2][U], av[2][U][TF];
  auto load = [&](int b, int k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = k + u < k1 ? k + u : k1 - 1;   // past the end: read again, not used
      wv[b][u] = *FM_GLOBAL(const v4i, w + t * 1024);
      if constexpr (QUANT == 0)
#pragma unroll
        for (int f = 0; f < TF; ++f) av[b][u][f] = *FM_GLOBAL(const v4i, a[f] + t * 1024);
    }
  };
  auto use = [&](int b, int k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u >= k1) break;
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        v4i tok;
        if constexpr (QUANT) tok = *reinterpret_cast<const v4i*>(mine + (k + u) * 64);
        else tok = av[b][u][f];
        acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[b][u], tok, acc[f], 0, 0, 0);
      }
    }
  };
  if (k0 < k1) load(0, k0), load(1, k0 + U);
  if constexpr (QUANT) quantise_rows<QUANT == 2>(x, int(p.M), p.kt, held, held_scale, tops);
  for (int k = k0; k < k1; k += 2 * U) {
    use(0, k);
    if (k + 2 * U < k1) load(0, k + 2 * U);
    use(1, k + U);
    if (k + 3 * U < k1) load(1, k + 3 * U);
  }
  if (wave)
#pragma unroll
    for (int f = 0; f < TF; ++f) red[wave - 1][f][lane] = acc[f];
  __syncthreads();
  if (wave) return;
  const int64_t n = nt * 16 + 4 * q;
  if (n >= p.N) return;
  const v4f sw = four_of(p.sw, n, p.N), bias = p.bias ? four_of(p.bias, n, p.N) : v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int f = 0; f < TF; ++f) {
    const int64_t t = 16 * (t0 + f) + m;
    if (t >= p.M) break;
    const v4i s = acc[f] + red[0][f][lane] + red[1][f][lane] + red[2][f][lane];
    const float sa = QUANT ? held_scale[m] : p.sa[t];
    v4f v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = float(s[i]) * sa * sw[i] + bias[i];
    if (n + 4 <= p.N) {
      if (p.out_f32) *FM_GLOBAL(u32x4_any, static_cast<float*>(p.out) + t * p.ld_out + n) = __builtin_bit_cast(fm_u32x4, v);
      else *FM_GLOBAL(u32x2_any, static_cast<uint16_t*>(p.out) + t * p.ld_out + n) = fm_u32x2{hw_bf16x2(v[0], v[1]), hw_bf16x2(v[2], v[3])};
      continue;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (n + i >= p.N) break;
      if (p.out_f32) st_global(static_cast<float*>(p.out) + t * p.ld_out + n + i, v[i]);
      else st_global(static_cast<uint16_t*>(p.out) + t * p.ld_out + n + i, uint16_t(hw_bf16x2(v[i], v[i])));
    }
  }
}

// ------------------------------------------------------------- many tokens ----
// out tile of TI channels x TJ tokens, WI x WJ waves of FA x FB 16x16x64 MFMA blocks; K runs in
// steps of 64 KS through a ring of NS LDS slots: while one step is multiplied from
// registers the next is read from LDS and the NS - 2 after it are on their way from memory.
// Persistent: the ring runs on into the workgroup's next output tile, so its stores and
// the next tile's first loads overlap.  SWIGLU: half of a wave's rows are gate rows, the
// others the same hidden units' up rows, and h = silu(g) u leaves in fp32.
template <int WI_, int WJ_, int FA_, int FB_, int KS_, int NS_>
struct Shape {
  static constexpr int WI = WI_, WJ = WJ_, FA = FA_, FB = FB_, W = WI * WJ;
  static constexpr int KS = KS_, NS = NS_;   // 64s of K in a step; slots of the ring
  static constexpr int TI = 16 * FA * WI, TJ = 16 * FB * WJ;
  static constexpr int PI = TI / 16 / W, PJ = TJ / 16 / W;   // row tiles that a wave moves
  static constexpr int kSlot = (TI + TJ) * 64 * KS;
  static constexpr int kStage = W * 2048;
  static constexpr bool kHalves = W == 8 && WJ % 2 == 0;   // waves 0..3 hold the first half of the tokens, 4..7 the second
  static_assert(TI % (16 * W) == 0 && TJ % (16 * W) == 0 && (KS == 1 || KS == 2), "whole pieces; K is a multiple of 128");
};
constexpr int kProductExperts = 1024;

struct OutTile {
  int e, i, j0, j1;   // expert, channel tile, rows [j0, j1)
};

// A wave's blocks of an output tile: block (x, y) holds token lane % 16 of y, channels
// 4 (lane / 16) + 0..3 of x.  bf16 rows go through the wave's 2 KiB of LDS, so that a
// store covers 64 bytes of 16 rows.  The lane is asked for again, so that nothing derived
// from it stays in registers through the loop over K, which leaves none to spare.
template <typename S, bool SWIGLU>
__device__ __forceinline__ void store_tile(const ProductArgs& p, const OutTile& cur, const v4i (&acc)[S::FA][S::FB], uint8_t* stage,
                                           int wi, int wj) {
  constexpr int FA = S::FA, FB = S::FB;
  const int lane = fresh_lane(), m = lane & 15, q = lane >> 4;
  const float *sw = p.sw + cur.e * p.sw_gs, *sw2 = p.sw2 + cur.e * p.sw_gs;
  const int64_t iw = int64_t(cur.i) * (SWIGLU ? S::TI / 2 : S::TI) + wi * (SWIGLU ? 8 * FA : 16 * FA);
  const int64_t tw = cur.j0 + wj * FB * 16;
  float sa[FB];
#pragma unroll
  for (int y = 0; y < FB; ++y) sa[y] = tw + 16 * y + m < cur.j1 ? *FM_GLOBAL(const float, p.sa + tw + 16 * y + m) : 0.f;
  if constexpr (SWIGLU) {
    // rows of scale 0 are none or a plan's padding, whose h nothing reads
    uint32_t top[FB];
#pragma unroll
    for (int y = 0; y < FB; ++y) top[y] = 0;
#pragma unroll
    for (int x = 0; x < FA / 2; ++x) {
      const int64_t n = iw + x * 16 + 4 * q;   // H is a multiple of 128: inside
      const v4f s1 = *FM_GLOBAL(const v4f, sw + n), s3 = *FM_GLOBAL(const v4f, sw2 + n);
#pragma unroll
      for (int y = 0; y < FB; ++y) {
        const int64_t t = tw + 16 * y + m;
        float h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gate = float(acc[x][y][i]) * sa[y] * s1[i], up = float(acc[x + FA / 2][y][i]) * sa[y] * s3[i];
          h[i] = gate / (1.f + expf(-gate)) * up;
          const uint32_t b = f2u(h[i]) & 0x7fffffffu;   // a NaN is above infinity, infinity above every number
          top[y] = b > top[y] ? b : top[y];
        }
        if (sa[y] != 0.f) st_global(static_cast<float*>(p.out) + t * p.ld_out + n, make_float4(h[0], h[1], h[2], h[3]));
      }
    }
    // a maximum does not depend on the order in which the waves raise it
#pragma unroll
    for (int y = 0; y < FB; ++y) {
#pragma unroll
      for (int off = 16; off < 64; off <<= 1) {
        const uint32_t o = __shfl_xor(top[y], off);
        top[y] = o > top[y] ? o : top[y];
      }
      if (q == 0 && sa[y] != 0.f) atomicMax(p.top + tw + 16 * y + m, top[y]);
    }
  } else {
    static_assert(FA % 2 == 0 && FB % 2 == 0, "blocks in squares of four");
#pragma unroll
    for (int x = 0; x < FA; x += 2) {
      const int64_t n0 = iw + x * 16;
      if (n0 >= p.N) break;
      v4f s[2], bias[2];
#pragma unroll
      for (int xx = 0; xx < 2; ++xx) {
        s[xx] = four_of(sw, n0 + 16 * xx + 4 * q, p.N);
        bias[xx] = p.bias ? four_of(p.bias, n0 + 16 * xx + 4 * q, p.N) : v4f{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int y = 0; y < FB; y += 2) {
#pragma unroll
        for (int yy = 0; yy < 2; ++yy)
#pragma unroll
          for (int xx = 0; xx < 2; ++xx) {
            v4f v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = float(acc[x + xx][y + yy][i]) * sa[y + yy] * s[xx][i] + bias[xx][i];
            if (p.out_f32) {
              const int64_t t = tw + 16 * (y + yy) + m, n = n0 + 16 * xx + 4 * q;
              float* o = static_cast<float*>(p.out) + t * p.ld_out + n;
              if (t < cur.j1) {
                if (n + 4 <= p.N) {
                  *FM_GLOBAL(u32x4_any, o) = __builtin_bit_cast(fm_u32x4, v);
                } else {
#pragma unroll
                  for (int i = 0; i < 3; ++i)
                    if (n + i < p.N) st_global(o + i, v[i]);
                }
              }
            } else {
              // 32 tokens x 64 bytes, 16-byte unit u of row t at u ^ (t / 2 % 4)
              const int tr = 16 * yy + m, u = 2 * xx + (q >> 1);
              *reinterpret_cast<fm_u32x2*>(stage + tr * 64 + ((u ^ (tr >> 1)) & 3) * 16 + (q & 1) * 8) =
                  fm_u32x2{hw_bf16x2(v[0], v[1]), hw_bf16x2(v[2], v[3])};
            }
          }
        if (!p.out_f32) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int tr = b * 16 + (lane >> 2), u = lane & 3;
            const fm_u32x4 o = *reinterpret_cast<const fm_u32x4*>(stage + tr * 64 + ((u ^ (tr >> 1)) & 3) * 16);
            const int64_t t = tw + 16 * y + tr, n = n0 + 8 * u;
            uint16_t* d = static_cast<uint16_t*>(p.out) + t * p.ld_out + n;
            if (t >= cur.j1) continue;
            if (n + 8 <= p.N) {
              *FM_GLOBAL(u32x4_any, d) = o;
            } else {
#pragma unroll
              for (int i = 0; i < 7; ++i)
                if (n + i < p.N) st_global(d + i, uint16_t(o[i / 2] >> (i % 2 * 16)));
            }
          }
        }
      }
    }
  }
}

template <typename S, bool SWIGLU>
__global__ __launch_bounds__(64 * S::W) void int8_product_kernel(ProductArgs p) {
  constexpr int FA = S::FA, FB = S::FB;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S::NS * S::kSlot + S::kStage];
  __shared__ int first[kProductExperts + 1];   // token tiles before each expert
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave % S::WI, wj = wave / S::WI;   // a SIMD's two waves hold different tokens

  // token tiles of every expert, added up
  const int rows_i = SWIGLU ? S::TI / 2 : S::TI;
  const int NI = int((p.N + rows_i - 1) / rows_i);
  if (p.offsets) {
    for (int e = tid; e < p.E; e += 64 * S::W) first[e + 1] = (p.offsets[e + 1] - p.offsets[e] + S::TJ - 1) / S::TJ;
    __syncthreads();
    if (wave == 0) {
      int sum = 0;
      for (int e0 = 0; e0 < p.E; e0 += 64) {
        int v = e0 + lane < p.E ? first[e0 + lane + 1] : 0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int o = __shfl_up(v, off);
          if (lane >= off) v += o;
        }
        if (e0 + lane < p.E) first[e0 + lane + 1] = sum + v;
        sum += __shfl(v, 63);
      }
      if (lane == 0) first[0] = 0;
    }
  } else if (tid == 0) {
    first[0] = 0;
    first[1] = int((p.M + S::TJ - 1) / S::TJ);
  }
  __syncthreads();
  const int n_tiles = __builtin_amdgcn_readfirstlane(first[p.E]) * NI;   // below 2^31 (launcher)
  // an XCD takes a run of tiles, its workgroups in turn, so those running together share operands in its L2
  const int xcd = blockIdx.x & 7, nbx = gridDim.x / 8;
  const int each = n_tiles / 8, more_x = n_tiles % 8;
  const int lo = each * xcd + (xcd < more_x ? xcd : more_x), hi = lo + each + (xcd < more_x);
  // where the last round leaves half or more of an XCD's workgroups idle, two share a tile's
  // tokens: half of them take half of the time where each SIMD holds a wave of either half
  const int mine = blockIdx.x / 8, whole = (hi - lo) / nbx, rem = (hi - lo) % nbx;
  const bool halves = S::kHalves && 2 * rem <= nbx;
  auto tile_at = [&](int c, OutTile& t) -> bool {
    int at = lo + c * nbx + mine;
    const bool halve = halves && c == whole && mine >= rem;   // the second half of the tile of `mine - rem`
    if (halve) at -= rem;
    if (c > whole || at >= hi) return false;
    int e = 0, n = p.E;   // the last expert whose tiles start at or before
    while (n > 1) {
      const int h = n / 2;
      if (__builtin_amdgcn_readfirstlane(first[e + h]) * NI <= at) e += h, n -= h;
      else n = h;
    }
    const int f0 = __builtin_amdgcn_readfirstlane(first[e]), nj = __builtin_amdgcn_readfirstlane(first[e + 1]) - f0;
    const int l = at - f0 * NI, g = l / (8 * NI), gj = nj - 8 * g < 8 ? nj - 8 * g : 8, r = l - g * 8 * NI;
    t.e = e;
    t.i = r / gj;
    const int j = 8 * g + r % gj;
    const int b = p.offsets ? __builtin_amdgcn_readfirstlane(p.offsets[e]) : 0;
    const int end = p.offsets ? __builtin_amdgcn_readfirstlane(p.offsets[e + 1]) : int(p.M);
    t.j0 = b + j * S::TJ;
    t.j1 = t.j0 + S::TJ < end ? t.j0 + S::TJ : end;
    if (halves && c == whole) {
      const int mid = t.j0 + S::TJ / 2;
      if (halve) t.j0 = mid;
      else if (mid < t.j1) t.j1 = mid;
    }
    return t.j0 < t.j1;
  };

  // what the wave moves: its tiles of the operands, row tiles past the end read from the last one
  v4i src[S::PI + S::PJ];
  const int64_t row_bytes = int64_t(p.kt) * 1024;
  auto aim = [&](const OutTile& t) {
#pragma unroll
    for (int u = 0; u < S::PI; ++u) {
      int rt = wave * S::PI + u;
      const uint8_t* base = p.w;
      if constexpr (SWIGLU) {
        // of a wave's FA row tiles the first half are gate rows, the others the same units' up rows
        if (rt / (FA / 2) % 2) base = p.w2;
        rt = t.i * (S::TI / 32) + rt / FA * (FA / 2) + rt % (FA / 2);
      } else {
        rt += t.i * (S::TI / 16);
      }
      const int last = int((p.N + 15) / 16) - 1;
      src[u] = make_rsrc(base + t.e * p.w_gs + (rt < last ? rt : last) * row_bytes);
    }
#pragma unroll
    for (int u = 0; u < S::PJ; ++u) {
      const int rt = t.j0 / 16 + wave * S::PJ + u, last = (t.j1 - 1) / 16;
      src[S::PI + u] = make_rsrc(p.a + (rt < last ? rt : last) * row_bytes);
    }
  };
  const uint32_t ring = lds_addr(smem);
  auto issue = [&](int slot, int k) {   // step k: tiles KS k .. of each row tile
#pragma unroll
    for (int u = 0; u < S::PI + S::PJ; ++u) {
      const int row = u < S::PI ? wave * S::PI + u : S::TI / 16 + wave * S::PJ + u - S::PI;
#pragma unroll
      for (int i = 0; i < S::KS; ++i)
        bdma16(src[u], lane * 16, uint32_t(k * S::KS + i) * 1024, ring + slot * S::kSlot + (row * S::KS + i) * 1024);
    }
  };

  struct Frags {
    v4i a[S::KS][FA], b[S::KS][FB];
  };
  auto read = [&](int slot, Frags& f) {
    const uint8_t* st = smem + slot * S::kSlot + lane * 16;   // a tile lies as its fragment is read
#pragma unroll
    for (int k = 0; k < S::KS; ++k) {
#pragma unroll
      for (int y = 0; y < FB; ++y) f.b[k][y] = *reinterpret_cast<const v4i*>(st + (S::TI / 16 + wj * FB + y) * S::KS * 1024 + k * 1024);
#pragma unroll
      for (int x = 0; x < FA; ++x) f.a[k][x] = *reinterpret_cast<const v4i*>(st + (wi * FA + x) * S::KS * 1024 + k * 1024);
    }
  };
  v4i acc[FA][FB];
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int k = 0; k < S::KS; ++k)
#pragma unroll
      for (int x = 0; x < FA; ++x)
#pragma unroll
        for (int y = 0; y < FB; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[k][x], f.b[k][y], acc[x][y], 0, 0, 0);
  };

  // the tile that is issued runs up to NS steps ahead of the one that is multiplied
  OutTile cur;
  if (!tile_at(0, cur)) return;
  int ca = 0;
  int ka = 0;
  const int steps = p.kt / S::KS;
  aim(cur);
  // a wave whose tokens lie behind the group's end only moves data: such a tile takes about half as long
  bool active = cur.j0 + wj * FB * 16 < cur.j1;
  bool more = true;
  auto advance = [&]() {
    if (ka == steps) {   // on to the next tile; behind the last one its last step again, which nothing reads
      OutTile t;
      more = more && tile_at(ca + 1, t);
      if (more) {
        ++ca;
        ka = 0;
        aim(t);
      } else {
        ka = steps - 1;
      }
    }
  };
  constexpr int kPer = (S::PI + S::PJ) * S::KS;
  // one step: the next one has landed (the others in flight; stores of the tile before,
  // if any, only make this wait longer) and every wave has read the one in `now`, whose slot
  // takes the step after those.  The reads of the next step go out under the first MFMAs: left
  // to itself the compiler reads after them, and every step waits for LDS.
  auto one_step = [&](int slot, const Frags& now, Frags& next) {
    advance();
    FM_WAIT_VMCNT((S::NS - 2) * kPer);
    block_barrier();
    issue(slot, ka++);
    if (!active) return;
    read(slot + 1 == S::NS ? 0 : slot + 1, next);
    multiply(now);
#pragma unroll
    for (int i = 0; i < (FA + FB) * S::KS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // one read of LDS
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
    }
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int s = 0; s < S::NS; ++s) {
    advance();
    issue(s, ka);
    ++ka;
  }
  FM_WAIT_VMCNT((S::NS - 1) * kPer);
  block_barrier();
  Frags f0, f1;
  read(0, f0);
  int g = 0;   // slot of the step in f0
  uint8_t* stage = smem + S::NS * S::kSlot + wave * 2048;
  for (int c = 0;; ++c) {
#pragma unroll
    for (int x = 0; x < FA; ++x)
#pragma unroll
      for (int y = 0; y < FB; ++y) acc[x][y] = v4i{0, 0, 0, 0};
    auto after = [](int slot) { return slot + 1 == S::NS ? 0 : slot + 1; };
#pragma unroll 1
    for (int k = 0;;) {
      one_step(g, f0, f1);
      g = after(g);
      if (++k == steps) break;
      one_step(g, f1, f0);
      g = after(g);
      if (++k == steps) break;
    }
    if (active) store_tile<S, SWIGLU>(p, cur, acc, stage, wi, wj);
    if (!tile_at(c + 1, cur)) break;
    active = cur.j0 + wj * FB * 16 < cur.j1;
    // the next tile's first step, read now rather than kept in registers while the tile was
    // stored; its slot is refilled after the next barrier
    read(g, f0);
  }
  FM_WAIT_VMCNT(0);
}

// out[t] = sum_k w[t, k] y[row of (t, k)], y fp32
__global__ __launch_bounds__(256) void int8_combine_kernel(const float* y, int64_t D, const int32_t* row_of, const float* w, int K,
                                                           void* out, int out_f32) {
  const int64_t t = blockIdx.y, c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (c >= D) return;
  fm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const int r = row_of[t * K + k];
    if (r >= 0) sum += *FM_GLOBAL(const fm_f32x4, y + r * D + c) * w[t * K + k];
  }
  if (out_f32) st_global(static_cast<float*>(out) + t * D + c, make_float4(sum[0], sum[1], sum[2], sum[3]));
  else st_global(static_cast<uint16_t*>(out) + t * D + c, make_uint2(hw_bf16x2(sum[0], sum[1]), hw_bf16x2(sum[2], sum[3])));
}

template <bool F32, int RW>
void launch_rows(const QuantArgs& a, int64_t row_tiles, hipStream_t s) {
  const dim3 grid{unsigned(row_tiles * (16 / RW))}, block(64 * kQuantWaves);
  constexpr int kStep = kQuantWaves * 64 / RW;
  const int each = (a.kt * 4 + kStep - 1) / kStep;   // chunks of a lane
  if (each <= 2) hipLaunchKernelGGL((int8_quant_kernel<F32, 2, false, RW>), grid, block, 0, s, a);
  else if (each <= 4) hipLaunchKernelGGL((int8_quant_kernel<F32, 4, false, RW>), grid, block, 0, s, a);
  else if (each <= 8) hipLaunchKernelGGL((int8_quant_kernel<F32, 8, false, RW>), grid, block, 0, s, a);
  else if (!F32 && each <= 16) hipLaunchKernelGGL((int8_quant_kernel<F32, F32 ? 8 : 16, false, RW>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((int8_quant_kernel<F32, 0, false, RW>), grid, block, 0, s, a);
}

template <bool F32>
void launch_quant(const QuantArgs& a, int64_t row_tiles, hipStream_t s) {
  if (a.top) {
    constexpr int RW = 8;
    // columns shared until the workgroups fill the chip twice, eight chunks a lane at least
    const int64_t rows = row_tiles * (16 / RW), y = (4 * device_cus() + rows - 1) / rows;
    const int64_t each = 8 * kQuantWaves * (64 / RW), most = (a.kt * 4 + each - 1) / each;
    hipLaunchKernelGGL((int8_quant_kernel<F32, 0, true, RW>), dim3(unsigned(rows), unsigned(y < most ? y : most)), dim3(64 * kQuantWaves), 0, s, a);
  } else if (row_tiles * 8 <= device_cus()) {
    launch_rows<F32, 2>(a, row_tiles, s);
  } else if (row_tiles * 4 <= device_cus()) {
    launch_rows<F32, 4>(a, row_tiles, s);
  } else {
    launch_rows<F32, 8>(a, row_tiles, s);
  }
}

using Large = Shape<2, 4, 8, 4, 1, 4>;
using Medium = Shape<2, 4, 8, 2, 1, 4>;
using Small = Shape<2, 2, 4, 2, 1, 5>;   // two workgroups to a CU

template <typename S, bool SWIGLU>
void launch_product(const ProductArgs& p, int64_t token_tiles, hipStream_t s) {
  const int rows_i = SWIGLU ? S::TI / 2 : S::TI;
  const int64_t tiles = token_tiles * ((p.N + rows_i - 1) / rows_i);
  static const int64_t fit = resident_workgroups(int8_product_kernel<S, SWIGLU>, 64 * S::W);
  int64_t grid = tiles * (S::kHalves ? 2 : 1) < fit ? tiles * (S::kHalves ? 2 : 1) : fit;
  grid = (grid + 7) / 8 * 8;   // a multiple of the XCDs
  hipLaunchKernelGGL((int8_product_kernel<S, SWIGLU>), dim3{unsigned(grid)}, dim3(64 * S::W), 0, s, p);
}

// The shape that is fastest by what 64 of K cost on it and the rounds of output tiles that a
// launch needs: 0.95 us for the 256 x 256 tile, 0.59 for 256 x 128, one workgroup a CU, 0.68
// and 0.43 for a round of halved tiles; 0.32 for 128 x 64 while it has a CU to itself, 0.42 when
// two share one.  Measured (us, small, medium, large, dense M x N x K): 77 x 2831 x 1409 9.6 /
// 15.5 / 18.1; 512 x 5632 x 2048 15.5 / 16.2 / 28.8; 512 x 4096 x 14336 53 / 85 / 102;
// 1024 x 4096 x 4096 25.9 / 25.1 / 33.8; 1500 x 3500 x 3000 27.7 / 25.9 / 39.2; 2048 x 4096 x
// 4096 46 / 36 / 39; 4096 x 2816 x 2048 37.3 / 35.7 / 34.1; 4096 x 4096 x 14336 308 / 224 / 194;
// 8192 x 14336 x 4096 652 / 538 / 424.  Halved last rounds: the large shape 47 -> 33.8 at
// 1024 x 4096 x 4096 and 348 -> 304 for 4096 slots on 8 experts x 4096 x 14336.
// Over a plan whose groups hold a token tile of the 256 x 128 shape or less, weights that are read
// once bound every shape, and that one reads them fastest: us of gate|up and down, small / medium /
// large, 65 tokens x 2 on 8 experts of 4096 x 14336 248 / 193 / 218 and 126 / 129 / 139; 128 x 8 on 32
// of 7168 x 2048 248 / 207 / 213 and 133 / 119 / 128; 1024 x 6 on 64 of 2048 x 1408 102 / 98 / 104
// and 70 / 62 / 63; 512 x 2 on 8 of 4096 x 14336 331 / 260 / 239 and 158 / 135 / 138.
// tokens over `groups` groups (dense: one); rows: of the padded buffer, or 0.
template <bool SWIGLU>
void launch_shape(const ProductArgs& p, int64_t tokens, int64_t groups, int64_t rows, hipStream_t s) {
  const int64_t cus = device_cus(), up = SWIGLU ? 2 : 1;
  // output tiles, about: the tokens' and, over a plan, a partly filled one for every other group
  auto tiles = [&](int64_t ti, int64_t tj) {
    const int64_t j = rows ? tokens / tj + (groups + 1) / 2 : (tokens + tj - 1) / tj;
    return j * ((p.N * up + ti - 1) / ti);
  };
  auto rounds = [](int64_t n, int64_t at_once) { return (n + at_once - 1) / at_once; };
  // a last round of half the workgroups or fewer is one of halved tiles
  auto cost = [&](int64_t n, int64_t one, int64_t half) { return one * (n / cus) + (n % cus == 0 ? 0 : n % cus * 2 <= cus ? half : one); };
  const int64_t small = tiles(Small::TI, Small::TJ);
  const int64_t large_us = cost(tiles(Large::TI, Large::TJ), 95, 68), medium_us = cost(tiles(Medium::TI, Medium::TJ), 59, 43);
  const int64_t small_us = small <= cus ? 32 : 42 * rounds(small, 2 * cus);
  // a bound of the token tiles: every group is a multiple of 128 rows
  auto most = [&](int64_t tj) { return rows ? rows / 128 * (tj < 128 ? 128 / tj : 1) : (tokens + tj - 1) / tj; };
  const bool stream = rows && tokens <= groups * Medium::TJ && groups * ((p.N * up + Medium::TI - 1) / Medium::TI) * 2 >= cus;
  if (stream) launch_product<Medium, SWIGLU>(p, most(Medium::TJ), s);
  else if (small_us <= medium_us && small_us <= large_us) launch_product<Small, SWIGLU>(p, most(Small::TJ), s);
  else if (large_us <= medium_us * 108 / 100) launch_product<Large, SWIGLU>(p, most(Large::TJ), s);
  else launch_product<Medium, SWIGLU>(p, most(Medium::TJ), s);
}

// Whether int8_few_kernel takes a product of 16-row tiles of tokens and of channels: up to 6
// workgroups a CU, or one pass over the weights.  us, it / the 128 x 64 tile (N x K at M): 512 x 4096
// at 16 3.2 / 14.8, at 512 6.8 / 15.8; 2831 x 1409 at 96 5.8 / 9.1, at 256 8.9 / 9.5, at 384 11.5 / 9.7;
// 4096 x 4096 at 128 10.4 / 15.9, at 192 14.0 / 16.2, at 256 17.3 / 16.2; 4096 x 14336 at 96 32.3 / 45.8,
// at 192 52.5 / 50.0; 14336 x 4096 at 32 19.5 / 22.2, at 64 25.2 / 24.1; 28672 x 4096 at 16 24.0 /
// 26.3, at 32 31.9 / 27.1.
bool few_rounds(int64_t tiles, int64_t channels) { return tiles == 1 || (tiles + 1) / 2 * channels <= 6 * int64_t(device_cus()); }

// Whether fm_int8_linear quantises in its product's kernel: rows that fit its LDS.
bool fused_rows(int64_t M, int64_t K) { return M <= kFusedRows && M * ((K + 127) / 128 * 128) <= kFusedBytes; }

bool product_sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && M < (int64_t(1) << 31) - 256 && N >= 1 && N < (int64_t(1) << 31) - 256 && K >= 1 && K < kMaxK;
}

}  // namespace

}  // namespace fm

using namespace fm;

extern "C" {

int fm_int8_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld_x, const int32_t* assign_of_row,
                     int top_k, const int32_t* limit, const uint32_t* top, uint32_t* clear, void* q, float* s, void* stream) {
  FM_REQUIRE(x && q && s, "fm_int8_quantize: null pointer");
  FM_REQUIRE(x_dtype == FM_DTYPE_BF16 || x_dtype == FM_DTYPE_F32, "fm_int8_quantize: x must be bf16 or fp32");
  FM_REQUIRE(product_sizes_ok(rows, 1, cols) && ld_x >= cols, "fm_int8_quantize: needs 1 <= columns < 131072 and a pitch that covers them");
  FM_REQUIRE(!assign_of_row || top_k >= 1, "fm_int8_quantize: top_k must be positive");
  FM_REQUIRE(aligned16(q) && reinterpret_cast<uintptr_t>(x) % (x_dtype == FM_DTYPE_F32 ? 4 : 2) == 0, "fm_int8_quantize: misaligned buffer");
  if (rows == 0) return 0;
  const QuantArgs a{x, ld_x, rows, cols, assign_of_row, top_k, limit, top, clear, static_cast<uint8_t*>(q), s, int((cols + 127) / 128 * 2)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == FM_DTYPE_F32) launch_quant<true>(a, (rows + 15) / 16, st);
  else launch_quant<false>(a, (rows + 15) / 16, st);
  return check_launch("fm_int8_quantize");
}

int fm_int8_pack(const void* x, int64_t groups, int64_t rows, int64_t cols, int64_t group_stride, int64_t row_stride,
                 int64_t col_stride, void* q, void* stream) {
  FM_REQUIRE(x && q && aligned16(q), "fm_int8_pack: null or misaligned pointer");
  FM_REQUIRE(groups >= 1 && rows >= 1 && product_sizes_ok(rows, 1, cols) && (groups == 1 || rows % 16 == 0),
             "fm_int8_pack: needs 1 <= columns < 131072, and groups of a multiple of 16 rows");
  const int64_t kt = (cols + 127) / 128 * 2, tiles = groups * ((rows + 15) / 16) * kt;
  FM_REQUIRE(tiles < (int64_t(1) << 32), "fm_int8_pack: too large");
  hipLaunchKernelGGL(int8_pack_kernel, dim3{unsigned((tiles + 3) / 4)}, dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(x), group_stride, row_stride, col_stride, rows, cols, int(kt), tiles,
                     static_cast<uint8_t*>(q));
  return check_launch("fm_int8_pack");
}

int fm_int8_unpack(const void* q, const float* s, int64_t rows, int64_t cols, void* out, int out_kind, int64_t ld_out, void* stream) {
  FM_REQUIRE(q && out && aligned16(q) && (s || out_kind == UP_I8), "fm_int8_unpack: null or misaligned pointer");
  FM_REQUIRE(product_sizes_ok(rows, 1, cols) && ld_out >= cols && out_kind >= UP_BF16 && out_kind <= UP_I8, "fm_int8_unpack: bad sizes or kind");
  if (rows == 0) return 0;
  const int kt = int((cols + 127) / 128 * 2);
  const int64_t tiles = (rows + 15) / 16 * kt;
  FM_REQUIRE(tiles < (int64_t(1) << 32), "fm_int8_unpack: too large");
  const dim3 grid{unsigned((tiles + 3) / 4)}, block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint8_t* p = static_cast<const uint8_t*>(q);
  uint8_t* o = static_cast<uint8_t*>(out);
  if (out_kind == UP_BF16) hipLaunchKernelGGL(int8_unpack_kernel<UP_BF16>, grid, block, 0, st, p, s, rows, cols, kt, tiles, o, ld_out);
  else if (out_kind == UP_F32) hipLaunchKernelGGL(int8_unpack_kernel<UP_F32>, grid, block, 0, st, p, s, rows, cols, kt, tiles, o, ld_out);
  else hipLaunchKernelGGL(int8_unpack_kernel<UP_I8>, grid, block, 0, st, p, s, rows, cols, kt, tiles, o, ld_out);
  return check_launch("fm_int8_unpack");
}

int fm_int8_matmul(const void* a, const float* sa, int64_t M, const void* w, const float* sw, int64_t N, int64_t K, const float* bias,
                   void* out, int out_dtype, int64_t ld_out, void* stream) {
  FM_REQUIRE(a && sa && w && sw && out && aligned16(a) && aligned16(w), "fm_int8_matmul: null or misaligned pointer");
  FM_REQUIRE(product_sizes_ok(M, N, K), "fm_int8_matmul: needs sizes of at least 1 and K < 131072");
  FM_REQUIRE((out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32) && ld_out >= N, "fm_int8_matmul: bad output type or pitch");
  if (M == 0) return 0;
  const ProductArgs p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(w), nullptr, sa, sw, nullptr, 0, 0,
                      int((K + 127) / 128 * 2), M, N, nullptr, 1, bias, out, ld_out, int(out_dtype == FM_DTYPE_F32), nullptr};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t tiles = (M + 15) / 16, channels = (N + 15) / 16;
  if (few_rounds(tiles, channels)) {
    const FusedRows none{nullptr, 0, 0};
    const bool one = tiles * channels <= device_cus() || tiles == 1;
    const int64_t passes = one ? tiles : (tiles + 1) / 2;
    const dim3 grid{unsigned((channels * passes + 7) / 8 * 8)}, block(256);
    if (one) hipLaunchKernelGGL((int8_few_kernel<1, 0>), grid, block, 0, st, p, none, int(passes));
    else hipLaunchKernelGGL((int8_few_kernel<2, 0>), grid, block, 0, st, p, none, int(passes));
  } else {
    launch_shape<false>(p, M, 1, 0, st);
  }
  return check_launch("fm_int8_matmul");
}

int64_t fm_int8_linear_workspace_bytes(int64_t M, int64_t K) {
  if (!product_sizes_ok(M, 1, K)) return -1;
  const int64_t tiles = (M + 15) / 16;
  return fused_rows(M, K) ? 0 : tiles * ((K + 127) / 128) * 2048 + tiles * 64;
}

int fm_int8_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, const void* w, const float* sw, int64_t N,
                   const float* bias, void* out, int out_dtype, int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  FM_REQUIRE(x && w && sw && out && aligned16(w), "fm_int8_linear: null or misaligned pointer");
  FM_REQUIRE(product_sizes_ok(M, N, K) && ld_x >= K, "fm_int8_linear: needs sizes of at least 1, K < 131072 and a pitch that covers a row");
  FM_REQUIRE((x_dtype == FM_DTYPE_BF16 || x_dtype == FM_DTYPE_F32) && reinterpret_cast<uintptr_t>(x) % (x_dtype == FM_DTYPE_F32 ? 4 : 2) == 0,
             "fm_int8_linear: x must be bf16 or fp32, aligned to its elements");
  FM_REQUIRE((out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32) && ld_out >= N, "fm_int8_linear: bad output type or pitch");
  if (M == 0) return 0;
  if (fused_rows(M, K)) {
    const ProductArgs p{nullptr, static_cast<const uint8_t*>(w), nullptr, nullptr, sw, nullptr, 0, 0, int((K + 127) / 128 * 2), M, N, nullptr, 1,
                        bias, out, ld_out, int(out_dtype == FM_DTYPE_F32), nullptr};
    const FusedRows r{x, ld_x, K};
    const dim3 grid{unsigned(((N + 15) / 16 + 7) / 8 * 8)}, block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == FM_DTYPE_F32) hipLaunchKernelGGL((int8_few_kernel<1, 2>), grid, block, 0, st, p, r, 1);
    else hipLaunchKernelGGL((int8_few_kernel<1, 1>), grid, block, 0, st, p, r, 1);
    return check_launch("fm_int8_linear");
  }
  FM_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= fm_int8_linear_workspace_bytes(M, K),
             "fm_int8_linear: the workspace must be fm_int8_linear_workspace_bytes bytes, 16-byte aligned");
  float* s = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (M + 15) / 16 * ((K + 127) / 128) * 2048);
  if (int rc = fm_int8_quantize(x, x_dtype, M, K, ld_x, nullptr, 1, nullptr, nullptr, nullptr, workspace, s, stream)) return rc;
  return fm_int8_matmul(workspace, s, M, w, sw, N, K, bias, out, out_dtype, ld_out, stream);
}

int fm_int8_grouped_gemm(const void* a, const float* sa, int64_t rows, const int32_t* offsets, int E, const void* w, const float* sw,
                         const void* w_up, const float* sw_up, uint32_t* top, int64_t N, int64_t K, int64_t tokens, void* out, int out_dtype,
                         int64_t ld_out, void* stream) {
  FM_REQUIRE(a && sa && offsets && w && sw && out && aligned16(a) && aligned16(w) && aligned16(w_up), "fm_int8_grouped_gemm: null or misaligned pointer");
  FM_REQUIRE(E >= 1 && E <= kProductExperts && rows >= 0 && rows % 128 == 0 && product_sizes_ok(rows, N, K) && K % 128 == 0 && N % 16 == 0,
             "fm_int8_grouped_gemm: needs rows and K multiples of 128, N of 16, and at most 1024 experts");
  FM_REQUIRE((w_up == nullptr) == (sw_up == nullptr) && (w_up == nullptr) == (top == nullptr) && (!w_up || (N % 128 == 0 && out_dtype == FM_DTYPE_F32 && ld_out % 4 == 0 && aligned16(out) && aligned16(sw) && aligned16(sw_up))),
             "fm_int8_grouped_gemm: SwiGLU needs the row maxima, N a multiple of 128 and an aligned fp32 output");
  FM_REQUIRE((out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32) && ld_out >= N, "fm_int8_grouped_gemm: bad output type or pitch");
  if (rows == 0) return 0;
  const ProductArgs p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(w_up), sa, sw, sw_up, N * K, N,
                      int(K / 64), rows, N, offsets, E, nullptr, out, ld_out, int(out_dtype == FM_DTYPE_F32), top};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (w_up) launch_shape<true>(p, tokens, tokens < E ? tokens : E, rows, st);
  else launch_shape<false>(p, tokens, tokens < E ? tokens : E, rows, st);
  return check_launch("fm_int8_grouped_gemm");
}

int fm_int8_combine(const float* y, int64_t D, const int32_t* row_of, const float* weights, int64_t T, int K, void* out, int out_dtype,
                    void* stream) {
  FM_REQUIRE(y && row_of && weights && out && aligned16(y) && aligned16(out), "fm_int8_combine: null or misaligned pointer");
  FM_REQUIRE(T >= 0 && T < 65536LL * 1024 && K >= 1 && D >= 4 && D % 4 == 0 && (out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32),
             "fm_int8_combine: bad sizes");
  if (T == 0) return 0;
  for (int64_t t0 = 0; t0 < T; t0 += 65535) {
    const int64_t n = T - t0 < 65535 ? T - t0 : 65535;
    hipLaunchKernelGGL(int8_combine_kernel, dim3(unsigned((D / 4 + 255) / 256), unsigned(n)), dim3(256), 0, static_cast<hipStream_t>(stream), y, D,
                       row_of + t0 * K, weights + t0 * K, K, static_cast<uint8_t*>(out) + t0 * D * (out_dtype == FM_DTYPE_F32 ? 4 : 2),
                       int(out_dtype == FM_DTYPE_F32));
  }
  return check_launch("fm_int8_combine");
}

}  // extern "C"
