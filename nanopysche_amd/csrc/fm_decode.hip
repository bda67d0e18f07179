// A MoE layer for a few tokens (a decoding step): router, the experts that the
// tokens reach, an optional shared expert, and the sum over a token's experts.
//
//   xn     = x                          or  x rsqrt(mean(x^2) + eps) g   (pre-norm)
//   logits = xn G^T + b + s, the K largest; their weights (softmax over the K, or
//            sigmoid / (sum + 1e-8); optionally divided by their l2 norm + 1e-8)
//   out[t] = sum_k w[t, k] y_e(t, k) (xn[t])  (+ the shared expert's y)
//   y_e(x) = (silu(x W1_e^T) * (x W3_e^T)) W2_e,   W1, W3, W2 stored [H, D]
//
// What bounds it is reading the reached experts' weights once: 3 H D elements of
// 2 bytes (bf16, as the layer stores them) or 1 (int8 with a scale per channel).
// Four launches: the router (a workgroup a token; a large gate over many workgroups and a
// launch of its own for the picks), gate|up (a workgroup takes 16 to 64 hidden units of
// one expert over all of its tokens and leaves h), down (512 output columns of one expert
// over a share of the hidden units), and the sum of the shares per token, in a fixed order.  Weights go from
// memory straight into MFMA fragments: with at most 16 tokens each feeds one MFMA, and
// LDS would only add latency.  The tokens' operand goes through LDS, a chunk at a time.
//
// Streaming rates measured on the same access patterns alone (2 GiB, MI355X): 1 KiB in
// order 6.2 to 6.9 TB/s; 16 rows x 64 bytes, the order of a row-major fragment, 5.5 to 6.0
// when a wave fetches 1 KiB of each row at a time and 3.7 to 4.6 when it fetches 512 bytes
// of two matrices in turn.  So a gate|up unit is 1 KiB of 16 rows of one matrix.
//
// W2's rows run along the output columns, but the MFMA wants the contracted index
// (a row) contiguous in a lane.  A lane loads 8 rows x 8 columns and transposes
// them in registers with 32 v_perm_b32; the 8 results are the fragments of 8
// interleaved sets of 16 columns.  Int8 weights are laid out once in 16 x 64 tiles
// in fragment order, W2 transposed.
//
// Sums, gate, up and SwiGLU are fp32.  h (and xn under a norm) enters the matrix
// cores as two bf16 pieces, hi + lo (remainder 2^-17 of the value), since a second
// MFMA costs nothing beside the weights' bytes; x itself and int8 weights are
// exact in bf16.
#include <type_traits>

#include "fm_common.h"
#include "../../include/fm_hip.h"

namespace fm {

namespace {

constexpr int kDecodeTokens = 64;    // most tokens of a call
constexpr int kDecodeTopK = 16;      // most experts of a token
constexpr int kDecodeExperts = 1024; // most experts
constexpr int kDecodeDim = 14336;    // widest token

// ------------------------------------------------------------------ router ----
constexpr int64_t kRouterOne = 64 * 1024;   // elements of a gate that one workgroup reads for a token

struct RouterArgs {
  const uint16_t* x;
  int64_t ld_x;
  int T, D;
  const void* gate;
  int gate_f32;
  int64_t ld_g;
  const void* bias;         // [E] or null
  int bias_f32;
  const float* score_bias;  // [E] or null
  const void* norm;         // [D] or null
  int norm_f32;
  float eps;
  int E, K, sigmoid, l2;
  float* logits;            // [T, E]
  uint16_t *xhi, *xlo;      // [T, D] with a norm
  float* w;                 // [T, K]
  int64_t* idx;             // [T, K]
};

__device__ __forceinline__ float load_f(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// 8 elements from column c of a row (16-byte boundary for bf16, 16 for fp32).
__device__ __forceinline__ void load8(const void* p, int f32, int64_t at, float (&v)[8]) {
  if (f32) {
    const fm_f32x4* s = reinterpret_cast<const fm_f32x4*>(static_cast<const float*>(p) + at);
    const fm_f32x4 a = s[0], b = s[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    const fm_u32x4 a = *reinterpret_cast<const fm_u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = u2f(a[i] << 16), v[2 * i + 1] = u2f(a[i] & 0xffff0000u);
  }
}

// Eight elements held as they were loaded.
template <bool F32>
struct Eight;
template <>
struct Eight<false> {
  fm_u32x4 w;
  __device__ __forceinline__ void load(const void* p, int64_t at) { w = *FM_GLOBAL(const fm_u32x4, static_cast<const uint16_t*>(p) + at); }
  __device__ __forceinline__ float at(int j) const { return u2f(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16); }
};
template <>
struct Eight<true> {
  float f[8];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const float* s = static_cast<const float*>(p) + at;
    const fm_f32x4 a = *FM_GLOBAL(const fm_f32x4, s), b = *FM_GLOBAL(const fm_f32x4, s + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  }
  __device__ __forceinline__ float at(int j) const { return f[j]; }
};

// The sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  // row_shr 1, 2, 4, 8: lane 15 of a row of 16 has its sum
  v += u2f(uint32_t(__builtin_amdgcn_update_dpp(0, int(f2u(v)), 0x111, 0xf, 0xf, true)));
  v += u2f(uint32_t(__builtin_amdgcn_update_dpp(0, int(f2u(v)), 0x112, 0xf, 0xf, true)));
  v += u2f(uint32_t(__builtin_amdgcn_update_dpp(0, int(f2u(v)), 0x114, 0xf, 0xf, true)));
  v += u2f(uint32_t(__builtin_amdgcn_update_dpp(0, int(f2u(v)), 0x118, 0xf, 0xf, true)));
  const float a = u2f(__builtin_amdgcn_readlane(f2u(v), 15)), b = u2f(__builtin_amdgcn_readlane(f2u(v), 31));
  const float c = u2f(__builtin_amdgcn_readlane(f2u(v), 47)), d = u2f(__builtin_amdgcn_readlane(f2u(v), 63));
  return (a + b) + (c + d);
}

// Selection order as a whole number: NaN above every number, then by value (-0 as 0).
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = f2u(v + 0.f);
  return v != v ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
}

// The workgroup picks token t's experts from its logits l[0, E) in LDS: an expert's place is
// the number of experts before it (a larger score, or an equal one and a lower index), counted
// by 512 / E' threads an expert (E' = E rounded up to a power of two).
constexpr int kRouterThreads = 512;
struct Gate {
  float l[kDecodeExperts];
  uint32_t key[kDecodeExperts];
  int place[kDecodeExperts], pick[kDecodeTopK];
};
__device__ __forceinline__ float sigmoid_of(float v) { return 1.f / (1.f + expf(-v)); }
__device__ __forceinline__ void gate_token(const RouterArgs& a, Gate& s, int t) {
  const int tid = threadIdx.x;
  for (int e = tid; e < a.E; e += kRouterThreads) {
    s.key[e] = order_of(a.sigmoid ? sigmoid_of(s.l[e]) : s.l[e]);
    s.place[e] = 0;
  }
  __syncthreads();
  int shift = 0;
  while ((1 << shift) < a.E) ++shift;
  const int parts = shift < 9 ? kRouterThreads >> shift : 1, each = (a.E + parts - 1) / parts;
  for (int i = tid; i < (parts << shift); i += kRouterThreads) {
    const int e = i & ((1 << shift) - 1), j0 = (i >> shift) * each, j1 = j0 + each < a.E ? j0 + each : a.E;
    if (e >= a.E) continue;
    const uint32_t mine = s.key[e];
    int n = 0;
    for (int j = j0; j < j1; ++j) n += s.key[j] > mine || (s.key[j] == mine && j < e);
    if (parts > 1) atomicAdd(&s.place[e], n);
    else s.place[e] = n;
  }
  __syncthreads();
  for (int e = tid; e < a.E; e += kRouterThreads)
    if (s.place[e] < a.K) s.pick[s.place[e]] = e;
  __syncthreads();
  if (tid >= 64) return;
  const int e = s.pick[tid < a.K ? tid : 0];
  const float l = s.l[e];
  const float v = tid >= a.K ? 0.f : a.sigmoid ? sigmoid_of(l) : expf(l - s.l[s.pick[0]]);
  const float sum = wave_sum(v);
  float w = a.sigmoid ? v / (sum + 1e-8f) : v / sum;
  if (a.l2) w = w / (sqrtf(wave_sum(tid < a.K ? w * w : 0.f)) + 1e-8f);
  if (tid < a.K) {
    st_global(a.w + int64_t(t) * a.K + tid, w);
    *FM_GLOBAL(int64_t, a.idx + int64_t(t) * a.K + tid) = e;
  }
}

// Workgroup: one token, experts [e0, e0 + per).  Every wave runs over the whole token for EP
// experts at a time and, under a norm, its sum of squares, so no wave waits for another
// before the picks; the logits take the norm's rsqrt at the end.  The waves of the first
// workgroup write the normed row's two pieces.
template <int EP, bool NORM, bool GF32>
__global__ __launch_bounds__(kRouterThreads) void decode_router_kernel(RouterArgs a, int per, int gate) {
  // U: steps of 512 columns whose loads leave together
  constexpr int NW = kRouterThreads / 64, U = (EP == 8 || (EP == 4 && NORM) ? 4 : 8) / (GF32 ? 2 : 1);
  __shared__ Gate s;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int t = blockIdx.y, e0 = blockIdx.x * per, e1 = e0 + per < a.E ? e0 + per : a.E;
  const uint16_t* x = a.x + int64_t(t) * a.ld_x;
  float rstd = 1.f;
  for (int e = e0 + wave * EP; e < e1 || (NORM && e < e0 + NW * EP); e += NW * EP) {   // with a norm every wave needs the sum
    float acc[EP], ss = 0.f;
    int64_t row[EP];
#pragma unroll
    for (int i = 0; i < EP; ++i) acc[i] = 0.f, row[i] = int64_t(e + i < e1 ? e + i : e1 - 1) * a.ld_g;
    for (int c0 = lane * 8; c0 < a.D; c0 += 512 * U) {
      Eight<false> v[U];
      Eight<GF32> g[U][EP];
      Eight<true> n[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + 512 * u < a.D ? c0 + 512 * u : lane * 8 % a.D;   // past the end: read again, not used
        v[u].load(x, c);
#pragma unroll
        for (int i = 0; i < EP; ++i) g[u][i].load(a.gate, row[i] + c);
        if constexpr (NORM) load8(a.norm, a.norm_f32, c, n[u].f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + 512 * u >= a.D) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float y = v[u].at(j);
          if constexpr (NORM) ss = fmaf(y, y, ss), y *= n[u].f[j];
#pragma unroll
          for (int i = 0; i < EP; ++i) acc[i] = fmaf(y, g[u][i].at(j), acc[i]);
        }
      }
    }
    if constexpr (NORM) rstd = 1.f / sqrtf(wave_sum(ss) / float(a.D) + a.eps);
#pragma unroll
    for (int i = 0; i < EP; ++i) {
      float l = wave_sum(acc[i]) * rstd;
      if (e + i < e1) {
        if (a.bias) l += load_f(a.bias, a.bias_f32, e + i);
        if (a.score_bias) l += a.score_bias[e + i];
        if (lane == 0) {
          if (gate) s.l[e + i] = l;
          else st_global(a.logits + int64_t(t) * a.E + e + i, l);
        }
      }
    }
  }
  if constexpr (NORM) {
    if (blockIdx.x == 0) {
      for (int c = threadIdx.x * 8; c < a.D; c += kRouterThreads * 8) {
        float v[8], n[8];
        load8(x, 0, c, v);
        load8(a.norm, a.norm_f32, c, n);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y0 = v[2 * j] * n[2 * j] * rstd, y1 = v[2 * j + 1] * n[2 * j + 1] * rstd;
          hi[j] = hw_bf16x2(y0, y1);
          lo[j] = hw_bf16x2(y0 - u2f(hi[j] << 16), y1 - u2f(hi[j] & 0xffff0000u));
        }
        st_global(a.xhi + int64_t(t) * a.D + c, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        st_global(a.xlo + int64_t(t) * a.D + c, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      }
    }
  }
  if (!gate) return;
  __syncthreads();
  gate_token(a, s, t);
}

// The picks from the logits of a launch whose workgroups each held some of the experts.
__global__ __launch_bounds__(kRouterThreads) void decode_gate_kernel(RouterArgs a) {
  __shared__ Gate s;
  const int t = blockIdx.x;
  for (int e = threadIdx.x; e < a.E; e += kRouterThreads) s.l[e] = a.logits[int64_t(t) * a.E + e];
  __syncthreads();
  gate_token(a, s, t);
}

template <int EP>
void launch_router(const RouterArgs& a, int per, bool gate, hipStream_t s) {
  const dim3 grid(unsigned((a.E + per - 1) / per), unsigned(a.T)), block(kRouterThreads);
  const int g = gate;
  if (a.norm && a.gate_f32) hipLaunchKernelGGL((decode_router_kernel<EP, true, true>), grid, block, 0, s, a, per, g);
  else if (a.norm) hipLaunchKernelGGL((decode_router_kernel<EP, true, false>), grid, block, 0, s, a, per, g);
  else if (a.gate_f32) hipLaunchKernelGGL((decode_router_kernel<EP, false, true>), grid, block, 0, s, a, per, g);
  else hipLaunchKernelGGL((decode_router_kernel<EP, false, false>), grid, block, 0, s, a, per, g);
}

// ----------------------------------------------------------------- experts ----
struct Expert {
  const uint8_t *w1, *w3, *w2;       // bf16 [E * H, D]; int8: tiles (W1 and W3 [H][D], W2 transposed [D][H])
  const float *s1, *s3, *s2;         // int8: [E * H], [E * H], [E, D]
  int H, S;                          // hidden units; workgroups of an expert in gate|up
  int R, P;                          // hidden units of a share of the down product, shares
  uint16_t *hhi, *hlo;               // [assignments][H]
  float* part;                       // [assignments][P][D]
};

struct ExpertArgs {
  const uint16_t *xhi, *xlo;         // [T, ld_x]; xlo null: x is its own first piece
  int64_t ld_x;
  int T, D, K, E;
  const void* idx;                   // [T, K]
  int idx_i64;
  int64_t offset;                    // index of the first expert held here
  Expert r, s;                       // routed, shared (S = P = 0: none)
};

__device__ __forceinline__ int expert_of(const ExpertArgs& a, int i) {
  const int64_t e = (a.idx_i64 ? static_cast<const int64_t*>(a.idx)[i] : int64_t(static_cast<const int32_t*>(a.idx)[i])) - a.offset;
  return e >= 0 && e < a.E ? int(e) : -1;
}

// eight int8 (two dwords) as bf16, exactly
__device__ __forceinline__ v8bf i8_to_bf16(uint32_t lo, uint32_t hi) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = i ? hi : lo;
    o[2 * i] = hw_bf16x2(float(int8_t(w)), float(int8_t(w >> 8)));
    o[2 * i + 1] = hw_bf16x2(float(int8_t(w >> 16)), float(int8_t(w >> 24)));
  }
  return __builtin_bit_cast(v8bf, fm_u32x4{o[0], o[1], o[2], o[3]});
}

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Loads of a buffer through a descriptor: a 32-bit lane offset that stays the same and a
// uniform one, so a load in flight holds no address registers; past the end they give 0.
// kOnce: weights that are read once leave the caches first (whole lines only: half lines
// would be fetched twice).
__device__ __forceinline__ auto buffer_of(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(uint32_t(bytes)), 0x00020000);
}
constexpr int kOnce = 2;
template <typename V, int POLICY = 0, typename B>
__device__ __forceinline__ V load_buffer(B rsrc, int voff, int soff) {
  if constexpr (sizeof(V) == 16) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff, soff, POLICY));
  else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(rsrc, voff, soff, POLICY));
}

// A barrier that does not wait for loads from memory in flight.
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The tokens' operand of a workgroup: rows of XL pieces, a chunk of 64 C columns at a time
// through two LDS buffers; rows of 64 C + 8 elements, so that 16 rows' reads fall on
// distinct banks.
template <int XL, int TF>
struct Tokens {
  static constexpr int C = XL * TF <= 2 ? 8 : 16 / (XL * TF);     // steps of 64 in a chunk
  static constexpr int P = 64 * C + 8, N = 16 * TF * C * 8 / 256; // 16-byte loads of a thread and piece
  static constexpr int kBytes = 2 * XL * 16 * TF * P * 2;
  static_assert(16 * TF * C * 8 % 256 == 0, "whole loads");
  int from[N], to[N];
  fm_u32x4 v[XL][N];
  // row(i): the element offset of token i < n's row
  template <typename F>
  __device__ __forceinline__ void aim(int n, F&& row) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int at = int(threadIdx.x) + 256 * j, r = at / (8 * C), c = at % (8 * C);
      from[j] = int((row(r < n ? r : n - 1) + 8 * c) * 2);
      to[j] = r * P + 8 * c;
    }
  }
  template <typename B>
  __device__ __forceinline__ void load(B hi, B lo, int step) {   // past a row's end: not used
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int p = 0; p < XL; ++p) v[p][j] = load_buffer<fm_u32x4>(p ? lo : hi, from[j], step * 128);
  }
  __device__ __forceinline__ void put(uint16_t* lds, int buf) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int p = 0; p < XL; ++p) *reinterpret_cast<fm_u32x4*>(lds + (buf * XL + p) * 16 * TF * P + to[j]) = v[p][j];
  }
  // the fragment of token tile f, piece p: 8 columns from `col` of the chunk
  static __device__ __forceinline__ v8bf get(const uint16_t* lds, int buf, int p, int f, int col) {
    return *reinterpret_cast<const v8bf*>(lds + ((buf * XL + p) * 16 * TF + 16 * f + int(threadIdx.x & 15)) * P + col);
  }
};

// h = silu(g) u of 16 hidden units (rows 4 q + v) and the lane's token, as two pieces
__device__ __forceinline__ void store_h(const Expert& x, bool i8, int e, int hid, int assign, const v4f& g, const v4f& u) {
  const int q = (threadIdx.x & 63) >> 4;
  v4f g1 = {1.f, 1.f, 1.f, 1.f}, g3 = g1;
  if (i8) {
    const int64_t at = int64_t(e) * x.H + hid + 4 * q;
    g1 = *FM_GLOBAL(const v4f, x.s1 + at);
    g3 = *FM_GLOBAL(const v4f, x.s3 + at);
  }
  float h[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float gate = g[v] * g1[v];
    h[v] = gate / (1.f + expf(-gate)) * (u[v] * g3[v]);
  }
  const uint32_t h0 = hw_bf16x2(h[0], h[1]), h1 = hw_bf16x2(h[2], h[3]);
  const uint32_t l0 = hw_bf16x2(h[0] - u2f(h0 << 16), h[1] - u2f(h0 & 0xffff0000u));
  const uint32_t l1 = hw_bf16x2(h[2] - u2f(h1 << 16), h[3] - u2f(h1 & 0xffff0000u));
  const int64_t at = int64_t(assign) * x.H + hid + 4 * q;
  st_global(x.hhi + at, make_uint2(h0, h1));
  st_global(x.hlo + at, make_uint2(l0, l1));
}

// Gate and up of one expert's tokens: RG row groups of 16 hidden units and KG parts of D over
// the 4 waves.  A unit is 16 rows x a chunk of one matrix; one of w1 and one of w3 are in
// flight or in use.
template <bool I8, bool LO, int RG, int TF>
__device__ __forceinline__ void up_pass(const ExpertArgs& a, const Expert& x, int e, int slice, const int* list, int n, int per,
                                        uint8_t* lds) {
  constexpr int KG = 4 / RG, XL = LO ? 2 : 1;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int rg = wave % RG, kg = wave / RG, D = a.D;
  // a step is 64 of D, two MFMAs deep.  bf16: lane q holds columns 8 q and 32 + 8 q; int8:
  // columns 16 q .. + 16 in one load
  typedef Tokens<XL, TF> Tok;
  constexpr int C = KG == 1 ? Tok::C : XL * TF == 1 ? 8 : XL * TF == 2 ? 4 : XL * TF == 4 ? 2 : 1, WL = I8 ? 1 : 2;
  const int steps = D / 64, s0 = steps * kg / KG, s1 = steps * (kg + 1) / KG;
  const int hid = slice * 16 * RG + rg * 16;
  const int row_bytes = I8 ? D : 2 * D;
  const int64_t first = (int64_t(e) * x.H + hid) * row_bytes;
  const auto r1 = buffer_of(x.w1 + first, 16 * row_bytes), r3 = buffer_of(x.w3 + first, 16 * row_bytes);
  const int w_off = I8 ? lane * 16 : m * row_bytes + 16 * q;   // int8: a row tile is 16 D bytes
  auto load_w = [&](fm_u32x4 (&w)[C][WL], const auto& r, int s) {
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int k = s + u < s1 ? s + u : s1 - 1;   // past the end: read again, not used
#pragma unroll
      for (int l = 0; l < WL; ++l) w[u][l] = load_buffer<fm_u32x4, I8 ? kOnce : 0>(r, w_off, k * (I8 ? 1024 : 128) + l * 64);
    }
  };
  v4f acc[2][TF];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int f = 0; f < TF; ++f) acc[b][f] = v4f{0.f, 0.f, 0.f, 0.f};
  auto use_w = [&](const fm_u32x4 (&w)[C][WL], v4f (&c)[TF], int s, auto&& token) {   // token(u, l, p, f)
#pragma unroll
    for (int u = 0; u < C; ++u) {
      if (s + u >= s1) break;
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        v8bf wf;
        if constexpr (I8) wf = i8_to_bf16(w[u][0][2 * l], w[u][0][2 * l + 1]);
        else wf = __builtin_bit_cast(v8bf, w[u][l]);
#pragma unroll
        for (int f = 0; f < TF; ++f)
#pragma unroll
          for (int p = 0; p < XL; ++p) c[f] = mfma(wf, token(u, l, p, f), c[f]);
      }
    }
  };
  const int64_t x_bytes = ((a.T - 1) * a.ld_x + D) * 2;
  const auto rx = buffer_of(a.xhi, x_bytes), rl = buffer_of(LO ? a.xlo : a.xhi, x_bytes);
  fm_u32x4 wa[C][WL], wb[C][WL];
  if constexpr (KG == 1) {
    uint16_t* xs = reinterpret_cast<uint16_t*>(lds);
    Tok t;
    t.aim(n, [&](int i) { return int64_t(list[i] / per) * a.ld_x; });
    // workgroups start at different chunks, so that rows a power of two apart do not meet in one memory channel
    const int chunks = (steps + C - 1) / C, c0 = int(blockIdx.x * 5u % unsigned(chunks));
    auto at = [&](int c) { return (c + c0 < chunks ? c + c0 : c + c0 - chunks) * C; };
    t.load(rx, rl, at(0));
    load_w(wa, r1, at(0));
    load_w(wb, r3, at(0));
    t.put(xs, 0);
    auto chunk = [&](int c, auto more) {   // more: another chunk follows
      const int s = at(c), next = more ? at(c + 1) : 0, buf = c & 1;
      auto token = [&](int u, int l, int p, int f) { return Tok::get(xs, buf, p, f, 64 * u + (I8 ? 16 * q + 8 * l : 8 * q + 32 * l)); };
      if constexpr (more) t.load(rx, rl, next);
      wg_barrier();
      use_w(wa, acc[0], s, token);
      if constexpr (more) load_w(wa, r1, next);
      use_w(wb, acc[1], s, token);
      if constexpr (more) {
        load_w(wb, r3, next);
        t.put(xs, buf ^ 1);
      }
    };
    for (int c = 0; c + 1 < chunks; ++c) chunk(c, std::true_type{});
    chunk(chunks - 1, std::false_type{});
  } else {
    int xo[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f)
      xo[f] = int((list[16 * f + m < n ? 16 * f + m : n - 1] / per * a.ld_x + (I8 ? 16 : 8) * q) * 2);
    fm_u32x4 xv[C][2][XL][TF];
    auto load_x = [&](int s) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int k = s + u < s1 ? s + u : s1 - 1;
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
          for (int p = 0; p < XL; ++p)
#pragma unroll
            for (int f = 0; f < TF; ++f)
              xv[u][l][p][f] = load_buffer<fm_u32x4>(p ? rl : rx, xo[f], k * 128 + l * (I8 ? 16 : 64));
      }
    };
    auto token = [&](int u, int l, int p, int f) { return __builtin_bit_cast(v8bf, xv[u][l][p][f]); };
    if (s0 < s1) {
      load_x(s0);
      load_w(wa, r1, s0);
      load_w(wb, r3, s0);
      for (int s = s0;;) {
        use_w(wa, acc[0], s, token);
        if (s + C < s1) load_w(wa, r1, s + C);
        use_w(wb, acc[1], s, token);
        s += C;
        if (s >= s1) break;
        load_x(s);
        load_w(wb, r3, s);
      }
    }
    // the parts of D meet in LDS in their order
    fm_f32x4* red = reinterpret_cast<fm_f32x4*>(lds);
    auto slot = [&](int k, int b, int f) { return red + (((k * RG + rg) * 2 + b) * TF + f) * 64 + lane; };
    if (kg > 0) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int f = 0; f < TF; ++f) *slot(kg - 1, b, f) = __builtin_bit_cast(fm_f32x4, acc[b][f]);
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int k = 0; k < KG - 1; ++k)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int f = 0; f < TF; ++f) acc[b][f] += __builtin_bit_cast(v4f, *slot(k, b, f));
    }
  }
  if (kg == 0) {
#pragma unroll
    for (int f = 0; f < TF; ++f)
      if (16 * f + m < n) store_h(x, I8, e, hid, list[16 * f + m], acc[0][f], acc[1][f]);
  }
  __syncthreads();   // LDS is read before the next pass's writes
}

// The down product of hidden units [k0, k1) into columns [col, col + 128) of the wave.
template <bool I8, int TF>
__device__ __forceinline__ void down_pass(const ExpertArgs& a, const Expert& x, int e, int col, int k0, int k1, int share,
                                          const int* list, int n, int rows, uint8_t* lds) {
  typedef Tokens<2, TF> Tok;
  constexpr int C = Tok::C;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4, D = a.D;
  const bool mine = col < D;   // D is a multiple of 128
  float* part[TF];
#pragma unroll
  for (int f = 0; f < TF; ++f) {
    const int i = 16 * f + m;
    part[f] = mine && i < n ? x.part + (int64_t(list[i]) * x.P + share) * D : nullptr;
  }
  const int64_t h_bytes = int64_t(rows) * x.H * 2;
  const auto rh = buffer_of(x.hhi, h_bytes), rl = buffer_of(x.hlo, h_bytes);
  uint16_t* hs = reinterpret_cast<uint16_t*>(lds);
  Tok t;
  t.aim(n, [&](int i) { return int64_t(list[i]) * x.H; });
  const int chunks = (k1 - k0 + 64 * C - 1) / (64 * C);
  if constexpr (I8) {
    // a unit is UT tiles of 16 columns x a chunk.  64 tokens: the wave's columns in two turns of 64
    constexpr int CT = TF == 4 ? 4 : 8, UT = 8 / C, UN = CT / UT;
    static_assert(UN == 1 || UN % 2 == 0, "units in pairs");
    const int tile_row = x.H / 64 * 1024;   // bytes of 16 output columns
    const auto r2 = buffer_of(x.w2 + int64_t(e) * x.H * D + int64_t(mine ? col / 16 : 0) * tile_row, 8 * int64_t(tile_row));
    const int last = k1 / 64 - 1;
    for (int sub = 0; sub < 8 / CT; ++sub) {
      fm_u32x4 wa[UT][C], wb[UT][C];
      auto load_w = [&](fm_u32x4 (&w)[UT][C], int c, int unit) {
#pragma unroll
        for (int i = 0; i < UT; ++i)
#pragma unroll
          for (int u = 0; u < C; ++u) {
            const int k = k0 / 64 + c * C + u;
            w[i][u] = load_buffer<fm_u32x4, kOnce>(r2, lane * 16, (sub * CT + unit * UT + i) * tile_row + (k < last ? k : last) * 1024);
          }
      };
      v4f o[CT][TF];
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int f = 0; f < TF; ++f) o[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
      auto use = [&](const fm_u32x4 (&w)[UT][C], int unit, int buf, int left) {
#pragma unroll
        for (int u = 0; u < C; ++u) {
          if (u >= left) break;
#pragma unroll
          for (int l = 0; l < 2; ++l)
#pragma unroll
            for (int f = 0; f < TF; ++f) {
              const v8bf hv = Tok::get(hs, buf, 0, f, 64 * u + 16 * q + 8 * l), lv = Tok::get(hs, buf, 1, f, 64 * u + 16 * q + 8 * l);
#pragma unroll
              for (int i = 0; i < UT; ++i) {
                const v8bf wf = i8_to_bf16(w[i][u][2 * l], w[i][u][2 * l + 1]);
                o[unit * UT + i][f] = mfma(wf, lv, mfma(wf, hv, o[unit * UT + i][f]));
              }
            }
        }
      };
      t.load(rh, rl, k0 / 64);
      load_w(wa, 0, 0);
      t.put(hs, 0);
      auto chunk = [&](int c, auto more) {   // more: another chunk follows
        const int buf = c & 1, left = (k1 - k0) / 64 - c * C;
        if constexpr (more) t.load(rh, rl, k0 / 64 + (c + 1) * C);
        wg_barrier();
        if constexpr (UN == 1) {
          if constexpr (more) load_w(wb, c + 1, 0);
          use(wa, 0, buf, left);
#pragma unroll
          for (int i = 0; i < UT; ++i)
#pragma unroll
            for (int u = 0; u < C; ++u) wa[i][u] = wb[i][u];
        } else {
#pragma unroll
          for (int unit = 0; unit < UN; unit += 2) {
            load_w(wb, c, unit + 1);
            use(wa, unit, buf, left);
            if (unit + 2 < UN) load_w(wa, c, unit + 2);
            else if constexpr (more) load_w(wa, c + 1, 0);
            use(wb, unit + 1, buf, left);
          }
        }
        if constexpr (more) t.put(hs, buf ^ 1);
      };
      for (int c = 0; c + 1 < chunks; ++c) chunk(c, std::true_type{});
      chunk(chunks - 1, std::false_type{});
      // the channels' scales come in with the sum over shares
#pragma unroll
      for (int f = 0; f < TF; ++f)
        if (part[f])
#pragma unroll
          for (int c = 0; c < CT; ++c)
            st_global(part[f] + col + 16 * (sub * CT + c) + 4 * q, make_float4(o[c][f][0], o[c][f][1], o[c][f][2], o[c][f][3]));
      if (sub + 1 < 8 / CT) wg_barrier();   // the chunks are read before the next turn's
    }
  } else {
    // a unit is 32 KU hidden units x 16 CW columns: lane (m, q) loads rows 8 q + i of each 32,
    // columns CW m .. + CW.  64 tokens: the wave's columns in two turns of 64
    constexpr int CW = TF == 4 ? 4 : 8, KU = TF == 2 ? 1 : 2, UC = 2 * C / KU;   // UC: units of a chunk
    typedef std::conditional_t<CW == 8, fm_u32x4, fm_u32x2> Row;
    const auto r2 = buffer_of(x.w2 + (int64_t(e) * x.H + k0) * D * 2, int64_t(k1 - k0) * D * 2);
    const int units = (k1 - k0) / (32 * KU);
    for (int sub = 0; sub < 8 / CW; ++sub) {
      const int c_at = (mine ? col : 0) + sub * 64, v_off = (8 * q * D + c_at + CW * m) * 2;
      Row wa[KU][8], wb[KU][8];
      auto load_w = [&](Row (&w)[KU][8], int unit) {
        const int k = unit * 32 * KU;
#pragma unroll
        for (int kk = 0; kk < KU; ++kk)
#pragma unroll
          for (int i = 0; i < 8; ++i) w[kk][i] = load_buffer<Row, kOnce>(r2, v_off, (k + 32 * kk + i) * D * 2);
      };
      v4f o[CW][TF];
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int f = 0; f < TF; ++f) o[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
      t.load(rh, rl, k0 / 64);
      load_w(wa, 0);
      t.put(hs, 0);
      int unit = 0;
      for (int c = 0; c < chunks; ++c) {
        const int buf = c & 1;
        if (c + 1 < chunks) t.load(rh, rl, k0 / 64 + (c + 1) * C);
        wg_barrier();
        auto use = [&](const Row (&w)[KU][8], int u) {
#pragma unroll
          for (int kk = 0; kk < KU; ++kk) {
            v8bf hv[TF], lv[TF];
#pragma unroll
            for (int f = 0; f < TF; ++f) {
              hv[f] = Tok::get(hs, buf, 0, f, 32 * (KU * u + kk) + 8 * q);
              lv[f] = Tok::get(hs, buf, 1, f, 32 * (KU * u + kk) + 8 * q);
            }
            // fragment 2 j + p: column CW r + 2 j + p of row r, from the halves p of dword j of the lane's rows
#pragma unroll
            for (int j = 0; j < CW / 2; ++j)
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                fm_u32x4 d;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  d[i] = __builtin_amdgcn_perm(w[kk][2 * i + 1][j], w[kk][2 * i][j], p ? 0x07060302u : 0x05040100u);
                const v8bf wf = __builtin_bit_cast(v8bf, d);
#pragma unroll
                for (int f = 0; f < TF; ++f) o[2 * j + p][f] = mfma(wf, lv[f], mfma(wf, hv[f], o[2 * j + p][f]));
              }
          }
        };
#pragma unroll 1
        for (int u = 0; u < UC && unit < units; u += 2, unit += 2) {
          if (unit + 1 < units) load_w(wb, unit + 1);
          use(wa, u);
          if (unit + 2 < units) load_w(wa, unit + 2);
          if (unit + 1 < units) use(wb, u + 1);
        }
        if (c + 1 < chunks) t.put(hs, buf ^ 1);
      }
      // fragment c's row 4 q + i is column CW (4 q + i) + c
#pragma unroll
      for (int f = 0; f < TF; ++f)
        if (part[f])
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < CW; c += 4)
              st_global(part[f] + c_at + CW * (4 * q + i) + c, make_float4(o[c][f][i], o[c + 1][f][i], o[c + 2][f][i], o[c + 3][f][i]));
      if (sub + 1 < 8 / CW) wg_barrier();   // the chunks are read before the next turn's
    }
  }
  __syncthreads();   // LDS is read before the next pass's writes
}

// The pick-th reached expert and its assignments in order, by every thread of the
// workgroup; -1 if fewer are reached.
struct Picked {
  int list[kDecodeTokens * kDecodeTopK];
  uint32_t bits[kDecodeExperts / 32];
  int e, n;
};
__device__ __forceinline__ void pick_expert(const ExpertArgs& a, int pick, Picked& s) {
  const int tid = threadIdx.x, lane = tid & 63, A = a.T * a.K;
  if (A <= 64) {
    // every wave by itself, in the order of the experts' first assignments; all write the same
    const int mine = lane < A ? expert_of(a, lane) : -1;
    bool again = mine < 0;
    for (int i = 0; i < A; ++i) again |= i < lane && __builtin_amdgcn_readlane(mine, i) == mine;
    uint64_t firsts = __ballot(!again);
    for (int i = 0; i < pick; ++i) firsts &= firsts - 1;
    int e = -1, n = 0;
    if (firsts) {
      e = __builtin_amdgcn_readlane(mine, __ffsll(static_cast<unsigned long long>(firsts)) - 1);
      const uint64_t hits = __ballot(mine == e);
      if (mine == e) s.list[__popcll(hits & ((uint64_t(1) << lane) - 1))] = lane;
      n = __popcll(hits);
    }
    s.e = e;
    s.n = n;
    __syncthreads();
    return;
  }
  for (int i = tid; i < kDecodeExperts / 32; i += 256) s.bits[i] = 0;
  if (tid == 0) s.e = -1;
  __syncthreads();
  for (int i = tid; i < A; i += 256) {
    const int v = expert_of(a, i);
    if (v >= 0) atomicOr(&s.bits[v >> 5], 1u << (v & 31));
  }
  __syncthreads();
  if (tid < 64) {
    const uint32_t w = lane < kDecodeExperts / 32 ? s.bits[lane] : 0;
    int before = __popc(w);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(before, off);
      if (lane >= off) before += o;
    }
    before -= __popc(w);
    const int in = pick - before;
    const uint64_t has = __ballot(in >= 0 && in < __popc(w));
    if (has) {
      uint32_t v = w;
      for (int i = 0; i < in && v; ++i) v &= v - 1;
      const int e = __shfl(lane * 32 + __ffs(v) - 1, __ffsll(static_cast<unsigned long long>(has)) - 1);
      int at = 0;
      for (int i0 = 0; i0 < A; i0 += 64) {
        const bool hit = i0 + lane < A && expert_of(a, i0 + lane) == e;
        const uint64_t bal = __ballot(hit);
        if (hit) s.list[at + __popcll(bal & ((uint64_t(1) << lane) - 1))] = i0 + lane;
        at += __popcll(bal);
      }
      if (lane == 0) s.e = e, s.n = at;
    }
  }
  __syncthreads();
}

template <bool I8, bool LO, int RG>
__global__ __launch_bounds__(256, 2) void decode_up_kernel(ExpertArgs a) {
  constexpr int XL = LO ? 2 : 1, KG = 4 / RG;
  constexpr int kX = Tokens<XL, 4>::kBytes > Tokens<XL, 1>::kBytes ? Tokens<XL, 4>::kBytes : Tokens<XL, 1>::kBytes;
  constexpr int kX2 = Tokens<XL, 2>::kBytes > kX ? Tokens<XL, 2>::kBytes : kX;
  constexpr int kRed = (KG - 1) * RG * 2 * 4 * 64 * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[KG == 1 ? kX2 : kRed];
  __shared__ Picked s;
  const bool shared = int(blockIdx.x) < a.s.S;
  int slice = blockIdx.x;
  if (shared) {
    for (int i = threadIdx.x; i < a.T; i += 256) s.list[i] = i;
    if (threadIdx.x == 0) s.e = 0, s.n = a.T;
    __syncthreads();
  } else {
    const int b = int(blockIdx.x) - a.s.S;
    pick_expert(a, b / a.r.S, s);
    slice = b % a.r.S;
  }
  const int e = __builtin_amdgcn_readfirstlane(s.e), n = e < 0 ? 0 : __builtin_amdgcn_readfirstlane(s.n);
  const Expert x = shared ? a.s : a.r;
  const int per = shared ? 1 : a.K;
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int left = n - t0;
    if (left > 32) up_pass<I8, LO, RG, 4>(a, x, e, slice, s.list + t0, left, per, lds);
    else if (left > 16) up_pass<I8, LO, RG, 2>(a, x, e, slice, s.list + t0, left, per, lds);
    else up_pass<I8, LO, RG, 1>(a, x, e, slice, s.list + t0, left, per, lds);
  }
}

template <bool I8>
__global__ __launch_bounds__(256, 2) void decode_down_kernel(ExpertArgs a) {
  constexpr int kX = Tokens<2, 4>::kBytes > Tokens<2, 1>::kBytes ? Tokens<2, 4>::kBytes : Tokens<2, 1>::kBytes;
  __shared__ __attribute__((aligned(16))) uint8_t lds[Tokens<2, 2>::kBytes > kX ? Tokens<2, 2>::kBytes : kX];
  __shared__ Picked s;
  const int cols = (a.D + 511) / 512, ns = a.s.P * cols;
  const bool shared = int(blockIdx.x) < ns;
  const Expert x = shared ? a.s : a.r;
  int b = blockIdx.x;
  if (shared) {
    for (int i = threadIdx.x; i < a.T; i += 256) s.list[i] = i;
    if (threadIdx.x == 0) s.e = 0, s.n = a.T;
    __syncthreads();
  } else {
    b -= ns;
    pick_expert(a, b / (x.P * cols), s);
    b %= x.P * cols;
  }
  const int e = __builtin_amdgcn_readfirstlane(s.e), n = e < 0 ? 0 : __builtin_amdgcn_readfirstlane(s.n);
  const int share = b / cols, k0 = share * x.R, k1 = k0 + x.R < x.H ? k0 + x.R : x.H;
  const int rows = shared ? a.T : a.T * a.K;
  const int col = b % cols * 512 + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) * 128;
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int left = n - t0;
    if (left > 32) down_pass<I8, 4>(a, x, e, col, k0, k1, share, s.list + t0, left, rows, lds);
    else if (left > 16) down_pass<I8, 2>(a, x, e, col, k0, k1, share, s.list + t0, left, rows, lds);
    else down_pass<I8, 1>(a, x, e, col, k0, k1, share, s.list + t0, left, rows, lds);
  }
}

// out[t] = sum_k w[t, k] (sum over the down product's shares) + the shared expert's shares.  A
// workgroup takes 64 columns of one token: 16 lanes of 4 columns, 16 groups over
// the shares in strides, the groups' sums added in order.
__global__ __launch_bounds__(256) void decode_combine_kernel(ExpertArgs a, const float* w, void* out, int out_f32, int64_t ld_o) {
  __shared__ fm_f32x4 red[16][16];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, t = blockIdx.y;
  const int64_t col = int64_t(blockIdx.x) * 64 + c * 4;
  fm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int shares = a.K * a.r.P;
#pragma unroll 2
  for (int i = g; i < shares; i += 16) {
    const int slot = t * a.K + i / a.r.P, e = expert_of(a, slot);
    if (e < 0) continue;
    fm_f32x4 y = *FM_GLOBAL(const fm_f32x4, a.r.part + (int64_t(slot) * a.r.P + i % a.r.P) * a.D + col);
    if (a.r.s2) y *= *FM_GLOBAL(const fm_f32x4, a.r.s2 + int64_t(e) * a.D + col);
    sum += y * w[slot];
  }
  if (a.s.P) {
    fm_f32x4 one = {1.f, 1.f, 1.f, 1.f};
    if (a.s.s2) one = *FM_GLOBAL(const fm_f32x4, a.s.s2 + col);
#pragma unroll 2
    for (int i = g; i < a.s.P; i += 16) sum += *FM_GLOBAL(const fm_f32x4, a.s.part + (int64_t(t) * a.s.P + i) * a.D + col) * one;
  }
  red[g][c] = sum;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += red[i][c];
  if (out_f32) st_global(static_cast<float*>(out) + t * ld_o + col, make_float4(sum[0], sum[1], sum[2], sum[3]));
  else st_global(static_cast<uint16_t*>(out) + t * ld_o + col, make_uint2(hw_bf16x2(sum[0], sum[1]), hw_bf16x2(sum[2], sum[3])));
}

// The launch: hidden units of a gate|up workgroup and of a share of the down product.
// Gate|up: 64 share the tokens' chunks among four waves and win from about three tokens an
// expert on; with fewer, 32 (or 16, below 128 workgroups) give more workgroups with less to
// wait for.  us a layer at 64 / 32 / 16 hidden units (MI355X): 64 tokens, 4 experts of 4096 x
// 4096 105 / 128 / 126; 64 tokens, 32 int8 experts of 7168 x 2048 291 / 340 / 352; 5 tokens,
// 64 experts of 2048 x 1408 105 / 98 / 98; 1 token, 8 of 128 experts of 2048 x 768 41 / 34 / 37;
// 1 token, 2 of 8 experts of 2048 x 1408 32.3 / 28.3 / 27.9.
// Down: as few shares as give every CU a workgroup, since each writes and the last kernel
// reads 4 D bytes a token (512 instead of 256 workgroups: 1 to 3% slower at 5 and 17 tokens).
struct DecodePlan {
  int hs, R, Rs;               // hidden units: of a gate|up workgroup; of a share, the shared expert's
  int P, Ps;                   // shares
  int64_t reach;               // most experts reached
  int64_t h, hs_at, part, part_s, bytes;   // offsets of h (two pieces), the shared expert's h, the shares, its shares
};
inline DecodePlan decode_plan(int64_t T, int64_t D, int64_t K, int64_t E, int64_t H, int64_t Hs) {
  constexpr int64_t kFill = 256;   // workgroups
  DecodePlan p;
  p.reach = E < T * K ? E : T * K;
  const int64_t units = p.reach * H + Hs;
  p.hs = T * K >= 3 * p.reach ? 64 : units / 32 >= kFill / 2 ? 32 : 16;
  const int64_t cols = (D + 511) / 512;
  // shares of at least 64 hidden units
  auto shares = [&](int64_t h, int& R, int& P) {
    int64_t want = (kFill * h + units * cols - 1) / (units * cols);
    const int64_t most = h / 64;
    want = want < 1 ? 1 : want > most ? most : want;
    R = int((h / 64 + want - 1) / want * 64);
    P = int((h + R - 1) / R);
  };
  shares(H, p.R, p.P);
  p.Rs = p.Ps = 0;
  if (Hs) shares(Hs, p.Rs, p.Ps);
  p.h = 0;
  p.hs_at = p.h + T * K * H * 4;
  p.part = p.hs_at + T * Hs * 4;
  p.part_s = p.part + T * K * p.P * D * 4;
  p.bytes = p.part_s + T * p.Ps * D * 4;
  return p;
}

template <bool I8, bool LO>
void launch_up(const ExpertArgs& a, int hs, int64_t blocks, hipStream_t s) {
  const dim3 grid{unsigned(blocks)}, block(256);
  if (hs == 64) hipLaunchKernelGGL((decode_up_kernel<I8, LO, 4>), grid, block, 0, s, a);
  else if (hs == 32) hipLaunchKernelGGL((decode_up_kernel<I8, LO, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((decode_up_kernel<I8, LO, 1>), grid, block, 0, s, a);
}

int expert_of_weights(const FmDecodeWeights* w, bool i8, Expert& x) {
  FM_REQUIRE(w->w1 && w->w2 && w->w3 && aligned16(w->w1) && aligned16(w->w2) && aligned16(w->w3),
             "fm_decode_experts: expert weights must be given and 16-byte aligned");
  FM_REQUIRE(!i8 || (w->s1 && w->s2 && w->s3 && aligned16(w->s1) && aligned16(w->s2) && aligned16(w->s3)),
             "fm_decode_experts: int8 weights need their scales, 16-byte aligned");
  FM_REQUIRE((w->kind == FM_DECODE_INT8) == i8, "fm_decode_experts: routed and shared experts must be of one kind");
  x = Expert{static_cast<const uint8_t*>(w->w1), static_cast<const uint8_t*>(w->w3), static_cast<const uint8_t*>(w->w2),
             i8 ? w->s1 : nullptr, i8 ? w->s3 : nullptr, i8 ? w->s2 : nullptr, int(w->H), 0, 0, 0, nullptr, nullptr, nullptr};
  return 0;
}

// Weights, output and pitch of x, before anything is launched.
int decode_operands_ok(int64_t ld_x, int64_t D, const FmDecodeWeights* experts, const FmDecodeWeights* shared, const void* out,
                       int out_dtype, int64_t ld_out, Expert& r, Expert& s) {
  FM_REQUIRE(experts->kind == FM_DECODE_BF16 || experts->kind == FM_DECODE_INT8, "fm_decode_experts: bad weight kind");
  FM_REQUIRE(ld_x >= D && ld_x % 8 == 0 && ld_x <= (1 << 23), "fm_decode_experts: rows must start on 16-byte boundaries, at a pitch of at most 2^23");
  FM_REQUIRE((out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32) && aligned16(out) && ld_out >= D && ld_out % 4 == 0,
             "fm_decode_experts: output must be bf16 or fp32, 16-byte aligned, its pitch at least D and a multiple of 4");
  const bool i8 = experts->kind == FM_DECODE_INT8;
  if (int rc = expert_of_weights(experts, i8, r)) return rc;
  return shared ? expert_of_weights(shared, i8, s) : 0;
}

int64_t decode_router_bytes(int64_t T, int64_t D, int64_t E) { return T * D * 4 + T * E * 4; }

bool decode_sizes_ok(int64_t T, int64_t D, int64_t K, int64_t E, int64_t H, int64_t Hs) {
  return T >= 1 && T <= kDecodeTokens && D >= 128 && D <= kDecodeDim && D % 128 == 0 && K >= 1 && K <= kDecodeTopK &&
         E >= 1 && E <= kDecodeExperts && H >= 128 && H % 128 == 0 && H <= (1 << 20) && Hs >= 0 && Hs % 128 == 0 &&
         Hs <= (1 << 20) && (H > Hs ? H : Hs) * D < (int64_t(1) << 30);   // a matrix's bytes are below 2^31
}

}  // namespace

}  // namespace fm

using namespace fm;

extern "C" {

int fm_moe_decode(const void* x, int64_t ld_x, int64_t T, int64_t D, const void* gate, int gate_dtype, int64_t ld_g,
                  const void* bias, int bias_dtype, const float* score_bias, const void* norm, int norm_dtype, float eps,
                  int E, int K, int gating, int flags, const FmDecodeWeights* experts, const FmDecodeWeights* shared,
                  float* weights, int64_t* indices, void* out, int out_dtype, int64_t ld_out, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  FM_REQUIRE(x && gate && weights && indices && experts && out && workspace, "fm_moe_decode: null pointer");
  FM_REQUIRE(decode_sizes_ok(T, D, K, E, 128, 0) && K <= E,
             "fm_moe_decode: needs 1..64 tokens, D a multiple of 128 up to 14336, at most 1024 experts and K <= min(E, 16)");
  FM_REQUIRE((gate_dtype == FM_DTYPE_BF16 || gate_dtype == FM_DTYPE_F32) && (bias_dtype == FM_DTYPE_BF16 || bias_dtype == FM_DTYPE_F32) &&
                 (norm_dtype == FM_DTYPE_BF16 || norm_dtype == FM_DTYPE_F32), "fm_moe_decode: bad dtype");
  FM_REQUIRE(gating == FM_GATING_SOFTMAX || gating == FM_GATING_SIGMOID, "fm_moe_decode: bad gating");
  FM_REQUIRE(aligned16(x) && ld_x >= D && ld_x % 8 == 0 && aligned16(gate) && ld_g >= D && ld_g % (gate_dtype == FM_DTYPE_F32 ? 4 : 8) == 0 &&
                 aligned16(norm), "fm_moe_decode: rows must start on 16-byte boundaries");
  const int64_t need = fm_decode_workspace_bytes(T, D, K, E, experts->H, shared ? shared->H : 0);
  FM_REQUIRE(need >= 0 && (!shared || shared->H > 0) && aligned16(workspace) && workspace_bytes >= need + decode_router_bytes(T, D, E),
             "fm_moe_decode: hidden sizes must be multiples of 128 and the workspace fm_moe_decode_workspace_bytes bytes");
  Expert routed{}, shared_expert{};
  if (int rc = decode_operands_ok(norm ? D : ld_x, D, experts, shared, out, out_dtype, ld_out, routed, shared_expert)) return rc;
  // behind the experts' workspace: the normed rows' two pieces, the logits
  uint8_t* own = static_cast<uint8_t*>(workspace) + need;
  uint16_t *x_hi = reinterpret_cast<uint16_t*>(own), *x_lo = x_hi + T * D;
  float* logits = reinterpret_cast<float*>(x_lo + T * D);
  const RouterArgs a{static_cast<const uint16_t*>(x), ld_x, int(T), int(D), gate, gate_dtype == FM_DTYPE_F32, ld_g, bias,
                     bias_dtype == FM_DTYPE_F32, score_bias, norm, norm_dtype == FM_DTYPE_F32, eps, E, K,
                     gating == FM_GATING_SIGMOID, (flags & FM_GATING_L2_NORMALIZE) != 0, logits,
                     x_hi, x_lo, weights, indices};
  hipStream_t s = static_cast<hipStream_t>(stream);
  // one workgroup a token where a gate is small enough for one CU to read; else eight experts a workgroup and a second launch
  const bool one = int64_t(E) * D <= kRouterOne;
  if (!one) {
    launch_router<1>(a, kRouterThreads / 64, false, s);
    hipLaunchKernelGGL(decode_gate_kernel, dim3{unsigned(T)}, dim3(kRouterThreads), 0, s, a);
  } else if (E <= 8) {
    launch_router<1>(a, E, true, s);
  } else if (E <= 16) {
    launch_router<2>(a, E, true, s);
  } else if (E <= 32) {
    launch_router<4>(a, E, true, s);
  } else {
    launch_router<8>(a, E, true, s);
  }
  if (int rc = check_launch("fm_moe_decode")) return rc;
  return fm_decode_experts(norm ? x_hi : x, norm ? x_lo : nullptr, norm ? D : ld_x, T, D, weights, indices, 1, K, 0, E, experts, shared,
                           out, out_dtype, ld_out, workspace, need, stream);
}

int64_t fm_moe_decode_workspace_bytes(int64_t T, int64_t D, int K, int E, int64_t H, int64_t H_shared) {
  const int64_t n = fm_decode_workspace_bytes(T, D, K, E, H, H_shared);
  return n < 0 ? n : n + decode_router_bytes(T, D, E);
}

int64_t fm_decode_workspace_bytes(int64_t T, int64_t D, int K, int E, int64_t H, int64_t H_shared) {
  if (!decode_sizes_ok(T, D, K, E, H, H_shared)) return -1;
  return decode_plan(T, D, K, E, H, H_shared).bytes;
}

int fm_decode_experts(const void* x, const void* x_lo, int64_t ld_x, int64_t T, int64_t D, const float* weights,
                      const void* indices, int indices_i64, int K, int64_t expert_offset, int E,
                      const FmDecodeWeights* experts, const FmDecodeWeights* shared, void* out, int out_dtype,
                      int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  FM_REQUIRE(x && weights && indices && experts && out && workspace, "fm_decode_experts: null pointer");
  const int64_t Hs = shared ? shared->H : 0;
  FM_REQUIRE(decode_sizes_ok(T, D, K, E, experts->H, Hs) && (!shared || Hs > 0),
             "fm_decode_experts: needs 1..64 tokens, D and hidden sizes multiples of 128 (D up to 14336), K <= 16 and at most 1024 experts");
  FM_REQUIRE(aligned16(x) && aligned16(x_lo) && aligned16(workspace), "fm_decode_experts: rows and workspace must start on 16-byte boundaries");
  Expert routed{}, shared_expert{};
  if (int rc = decode_operands_ok(ld_x, D, experts, shared, out, out_dtype, ld_out, routed, shared_expert)) return rc;
  const bool i8 = experts->kind == FM_DECODE_INT8;
  const DecodePlan p = decode_plan(T, D, K, E, experts->H, Hs);
  FM_REQUIRE(workspace_bytes >= p.bytes, "fm_decode_experts: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)p.bytes);
  ExpertArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(x_lo), ld_x, int(T), int(D), K, E, indices,
               indices_i64, expert_offset, routed, shared_expert};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto place = [&](Expert& e, int64_t rows, int R, int P, int64_t h, int64_t part) {
    e.S = e.H / p.hs;
    e.R = R;
    e.P = P;
    e.hhi = reinterpret_cast<uint16_t*>(ws + h);
    e.hlo = e.hhi + rows * e.H;
    e.part = reinterpret_cast<float*>(ws + part);
  };
  place(a.r, T * K, p.R, p.P, p.h, p.part);
  if (shared) place(a.s, T, p.Rs, p.Ps, p.hs_at, p.part_s);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t up = p.reach * a.r.S + a.s.S, down = (p.reach * a.r.P + a.s.P) * ((D + 511) / 512);
  if (i8) {
    if (x_lo) launch_up<true, true>(a, p.hs, up, s);
    else launch_up<true, false>(a, p.hs, up, s);
    hipLaunchKernelGGL(decode_down_kernel<true>, dim3{unsigned(down)}, dim3(256), 0, s, a);
  } else {
    if (x_lo) launch_up<false, true>(a, p.hs, up, s);
    else launch_up<false, false>(a, p.hs, up, s);
    hipLaunchKernelGGL(decode_down_kernel<false>, dim3{unsigned(down)}, dim3(256), 0, s, a);
  }
  hipLaunchKernelGGL(decode_combine_kernel, dim3(unsigned(D / 64), unsigned(T)), dim3(256), 0, s, a, weights, out,
                     int(out_dtype == FM_DTYPE_F32), ld_out);
  return check_launch("fm_decode_experts");
}

}  // extern "C"
