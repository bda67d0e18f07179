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
// A workgroup therefore takes one slice of HS hidden units of one expert through
// both products: the slice's rows of W1 and W3 give its HS columns of h for the
// expert's tokens, which stay in LDS, and its rows of W2 give the slice's share of
// y, which goes to the workspace in fp32 (8 D bytes out and back a token, against
// 6 HS D or 3 HS D of weights); the last kernel adds the shares in a fixed order.
// No phase waits for another workgroup.  Weights go from memory straight into MFMA
// fragments (no LDS): with at most 16 tokens a fragment's 16 x 32 weights feed one
// MFMA, so LDS staging would only add latency.
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
constexpr int kDecodeDim = 14336;    // widest token (the router holds it in LDS in fp32)

// ------------------------------------------------------------------ router ----
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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// NaN above every number, then the larger value, then the lower index.
__device__ __forceinline__ bool gate_beats(float av, int ai, float bv, int bi) {
  const bool an = av != av, bn = bv != bv;
  if (an || bn) return an && (!bn || ai < bi);
  return av > bv || (av == bv && ai < bi);
}

// One wave picks token t's experts from its logits l[0, E) in LDS, which it may
// overwrite.  Every round is an arg-max over the experts not yet taken.
__device__ __forceinline__ void gate_token(const RouterArgs& a, const float* l, int t, int lane) {
  uint32_t taken = 0;   // bit i: expert 64 i + lane
  float top = 0.f, sum = 0.f, mine = 0.f;
  int my_e = 0;
  for (int k = 0; k < a.K; ++k) {
    float bv = -INFINITY, bl = 0.f;
    int be = 0x7fffffff;
    for (int e = lane, i = 0; e < a.E; e += 64, ++i) {
      if ((taken >> i) & 1) continue;
      const float lg = l[e];
      const float sc = a.sigmoid ? 1.f / (1.f + expf(-lg)) : lg;
      if (be == 0x7fffffff || gate_beats(sc, e, bv, be)) bv = sc, bl = lg, be = e;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float ov = __shfl_xor(bv, off), ol = __shfl_xor(bl, off);
      const int oe = __shfl_xor(be, off);
      if (oe != 0x7fffffff && (be == 0x7fffffff || gate_beats(ov, oe, bv, be))) bv = ov, bl = ol, be = oe;
    }
    if ((be & 63) == lane) taken |= 1u << (be >> 6);
    if (k == 0) top = bl;
    const float wk = a.sigmoid ? bv : expf(bl - top);
    sum += wk;
    if (lane == k) mine = wk, my_e = be;
  }
  float w = a.sigmoid ? mine / (sum + 1e-8f) : mine / sum;
  if (a.l2) w = w / (sqrtf(wave_sum(lane < a.K ? w * w : 0.f)) + 1e-8f);
  if (lane < a.K) {
    st_global(a.w + int64_t(t) * a.K + lane, w);
    *FM_GLOBAL(int64_t, a.idx + int64_t(t) * a.K + lane) = my_e;
  }
}

// Workgroup: NW waves, one token, experts [e0, e1).  The token's row (times the
// norm weight) goes to LDS in fp32, every wave forms the logits of four experts at
// a time, and with `gate` wave 0 picks the experts.  The workgroup of the first
// experts writes the normed row's two pieces.
template <int NW>
__global__ __launch_bounds__(64 * NW) void decode_router_kernel(RouterArgs a, int per, int gate) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  float* xs = sm;              // [D]
  float* lg = sm + a.D;        // [per]
  float* red = lg + per;       // [NW]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int t = blockIdx.y, e0 = blockIdx.x * per, e1 = e0 + per < a.E ? e0 + per : a.E;
  const uint16_t* x = a.x + int64_t(t) * a.ld_x;
  float ss = 0.f;
  for (int c = threadIdx.x * 8; c < a.D; c += NW * 64 * 8) {
    float v[8];
    load8(x, 0, c, v);
    if (a.norm) {
      float g[8];
      load8(a.norm, a.norm_f32, c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss), v[i] *= g[i];
    }
    *reinterpret_cast<fm_f32x4*>(xs + c) = fm_f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<fm_f32x4*>(xs + c + 4) = fm_f32x4{v[4], v[5], v[6], v[7]};
  }
  float rstd = 1.f;
  if (a.norm) {
    ss = wave_sum(ss);
    if (lane == 0) red[wave] = ss;
  }
  __syncthreads();
  if (a.norm) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) s += red[i];
    rstd = 1.f / sqrtf(s / float(a.D) + a.eps);
    if (blockIdx.x == 0) {
      for (int c = threadIdx.x * 2; c < a.D; c += NW * 128) {
        const float v0 = xs[c] * rstd, v1 = xs[c + 1] * rstd;
        const uint32_t hi = hw_bf16x2(v0, v1);
        const uint32_t lo = hw_bf16x2(v0 - u2f(hi << 16), v1 - u2f(hi & 0xffff0000u));
        st_global(reinterpret_cast<uint32_t*>(a.xhi + int64_t(t) * a.D + c), hi);
        st_global(reinterpret_cast<uint32_t*>(a.xlo + int64_t(t) * a.D + c), lo);
      }
    }
  }
  for (int e = e0 + wave * 4; e < e1; e += NW * 4) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = int64_t(e + i < e1 ? e + i : e1 - 1) * a.ld_g;
    for (int c = lane * 8; c < a.D; c += 512) {
      const fm_f32x4 xa = *reinterpret_cast<const fm_f32x4*>(xs + c), xb = *reinterpret_cast<const fm_f32x4*>(xs + c + 4);
      float g[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) load8(a.gate, a.gate_f32, row[i] + c, g[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i] = fmaf(xb[j], g[i][4 + j], fmaf(xa[j], g[i][j], acc[i]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = wave_sum(acc[i]) * rstd;
      if (e + i < e1) {
        if (a.bias) v += load_f(a.bias, a.bias_f32, e + i);
        if (a.score_bias) v += a.score_bias[e + i];
        if (lane == 0) {
          if (gate) lg[e + i - e0] = v;
          else st_global(a.logits + int64_t(t) * a.E + e + i, v);
        }
      }
    }
  }
  if (!gate) return;
  __syncthreads();
  if (wave == 0) gate_token(a, lg, t, lane);
}

// The gating of logits from a launch whose workgroups each hold some of the experts: a wave a token.
__global__ __launch_bounds__(64) void decode_gate_kernel(RouterArgs a) {
  __shared__ float lg[kDecodeExperts];
  const int t = blockIdx.x, lane = threadIdx.x;
  for (int e = lane; e < a.E; e += 64) lg[e] = a.logits[int64_t(t) * a.E + e];
  __syncthreads();
  gate_token(a, lg, t, lane);
}

// ----------------------------------------------------------------- experts ----
struct Expert {
  const uint8_t *w1, *w3, *w2;       // bf16 [E * H, D]; int8: tiles (W1 and W3 [H][D], W2 transposed [D][H])
  const float *s1, *s3, *s2;         // int8: [E * H], [E * H], [E, D]
  int H, S;                          // hidden units; slices of an expert
  float* part;                       // [assignments][S][D]
};

struct ExpertArgs {
  const uint16_t *xhi, *xlo;         // [T, ld_x]; xlo null: x is its own first piece
  int64_t ld_x;
  int T, D, K, E;
  const void* idx;                   // [T, K]
  int idx_i64;
  int64_t offset;                    // index of the first expert held here
  Expert r, s;                       // routed, shared (S = 0: none)
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
__device__ __forceinline__ auto buffer_of(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(uint32_t(bytes)), 0x00020000);
}
#define FM_BUFFER_LOAD16(rsrc, voff, soff) \
  __builtin_bit_cast(fm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, int(voff), int(soff), 0))

template <typename V, typename B>
__device__ __forceinline__ V load_row(B rsrc, int voff, int soff) {
  if constexpr (sizeof(V) == 16) return FM_BUFFER_LOAD16(rsrc, voff, soff);
  else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(rsrc, voff, soff, 0));
}

// A barrier that does not wait for loads from memory in flight.
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A workgroup's slice: RG row groups of NR x 16 hidden units and KG parts of D
// over the 4 waves (RG * KG = 4), HS = 16 NR RG.
template <bool I8, bool LO, int NR, int RG>
struct Slice {
  static constexpr int KG = 4 / RG, HS = 16 * NR * RG;
  static constexpr int kPitch = HS + 8;                 // of h in LDS, elements
};

template <bool I8, bool LO, int NR, int RG, int TF>
__device__ __forceinline__ void slice_pass(const ExpertArgs& a, const Expert& x, int e, int slice, const int* list, int n,
                                           int per, uint8_t* lds) {
  using S = Slice<I8, LO, NR, RG>;
  constexpr int HS = S::HS, KG = S::KG, P = S::kPitch;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int rg = wave % RG, kg = wave / RG;
  const int64_t D = a.D;

  // ---- gate and up: rows hidden units, columns tokens
  v4f acc[2][NR][TF];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int f = 0; f < TF; ++f) acc[b][r][f] = v4f{0.f, 0.f, 0.f, 0.f};
  // a step is 64 of D: two MFMAs deep.  bf16: lane q holds columns 8 q and 32 + 8 q;
  // int8: columns 16 q .. + 16 in one load.  A chunk is C steps; the weights of the next
  // chunk are in flight while one is multiplied
  constexpr int XL = LO ? 2 : 1, C = KG == 1 ? (I8 && TF == 1 ? 4 : 4 / (NR * (TF == 4 ? 2 : 1))) : (TF * XL == 1 ? 4 : TF * XL == 2 ? 2 : 1);
  const int steps = a.D / 64, s0 = steps * kg / KG, s1 = steps * (kg + 1) / KG;
  constexpr int WL = I8 ? 1 : 2;                        // loads of a row's step
  const int hid = slice * HS + rg * 16 * NR;            // the wave's first hidden unit
  const int64_t row_bytes = I8 ? D : 2 * D, first = (int64_t(e) * x.H + hid) * row_bytes, mine = 16 * NR * row_bytes;
  const auto r1 = buffer_of(x.w1 + first, mine), r3 = buffer_of(x.w3 + first, mine);
  const int w_off = I8 ? lane * 16 : m * int(row_bytes) + 16 * q;    // int8: a row tile is 16 D bytes
  auto load_w = [&](fm_u32x4 (&w)[C][2][NR][WL], int s) {
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int k = s + u < s1 ? s + u : s1 - 1;    // past the end: read again, not used
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int l = 0; l < WL; ++l) {
          const int at = 16 * r * int(row_bytes) + k * (I8 ? 1024 : 128) + l * 64;
          w[u][0][r][l] = FM_BUFFER_LOAD16(r1, w_off, at);
          w[u][1][r][l] = FM_BUFFER_LOAD16(r3, w_off, at);
        }
    }
  };
  const int64_t x_bytes = ((a.T - 1) * a.ld_x + D) * 2;
  const auto rx = buffer_of(a.xhi, x_bytes), rl = buffer_of(LO ? a.xlo : a.xhi, x_bytes);
  auto step = [&](const fm_u32x4 (&w)[2][NR][WL], auto&& xf) {   // xf(piece, l, f): the fragment of tokens
#pragma unroll
    for (int l = 0; l < 2; ++l) {
      v8bf xv[XL][TF];
#pragma unroll
      for (int p = 0; p < XL; ++p)
#pragma unroll
        for (int f = 0; f < TF; ++f) xv[p][f] = xf(p, l, f);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          v8bf wf;
          if constexpr (I8) wf = i8_to_bf16(w[b][r][0][2 * l], w[b][r][0][2 * l + 1]);
          else wf = __builtin_bit_cast(v8bf, w[b][r][l]);
#pragma unroll
          for (int f = 0; f < TF; ++f)
#pragma unroll
            for (int p = 0; p < XL; ++p) acc[b][r][f] = mfma(wf, xv[p][f], acc[b][r][f]);
        }
    }
  };
  if constexpr (KG == 1) {
    // every wave runs over all of D: the chunk's tokens go through LDS once, in two
    // buffers, rows of 64 C elements + 8 (16 rows' reads fall on distinct banks)
    constexpr int XP = 64 * C + 8, NX = 16 * TF * C * 8 / 256;   // 16-byte loads of a thread and piece
    static_assert(16 * TF * C * 8 % 256 == 0, "whole loads");
    uint16_t* xs = reinterpret_cast<uint16_t*>(lds);             // [buffer][piece][16 TF][XP]
    const int tid = threadIdx.x;
    int from[NX], to[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const int at = tid + 256 * j, row = at / (8 * C), c = at % (8 * C);
      from[j] = (list[row < n ? row : n - 1] / per * int(a.ld_x) + 8 * c) * 2;
      to[j] = row * XP + 8 * c;
    }
    fm_u32x4 xr[XL][NX], wa[C][2][NR][WL], wb[C][2][NR][WL];
    auto load_x = [&](int s) {
#pragma unroll
      for (int j = 0; j < NX; ++j) {
#pragma unroll
        for (int p = 0; p < XL; ++p) xr[p][j] = FM_BUFFER_LOAD16(p ? rl : rx, from[j], s * 128);   // past D: not used
      }
    };
    auto put_x = [&](int buf) {
#pragma unroll
      for (int j = 0; j < NX; ++j)
#pragma unroll
        for (int p = 0; p < XL; ++p)
          *reinterpret_cast<fm_u32x4*>(xs + (buf * XL + p) * 16 * TF * XP + to[j]) = xr[p][j];
    };
    auto use = [&](const fm_u32x4 (&w)[C][2][NR][WL], int buf, int s) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        if (s + u >= s1) break;
        step(w[u], [&](int p, int l, int f) {
          return *reinterpret_cast<const v8bf*>(xs + ((buf * XL + p) * 16 * TF + 16 * f + m) * XP + 64 * u +
                                                (I8 ? 16 * q + 8 * l : 8 * q + 32 * l));
        });
      }
    };
    // a buffer is filled while the other is read: one barrier a chunk
    load_x(0);
    load_w(wa, 0);
    put_x(0);
    for (int s = 0;; s += 2 * C) {
      load_x(s + C);
      load_w(wb, s + C);
      wg_barrier();
      use(wa, 0, s);
      if (s + C >= s1) break;
      put_x(1);
      load_x(s + 2 * C);
      load_w(wa, s + 2 * C);
      wg_barrier();
      use(wb, 1, s + C);
      if (s + 2 * C >= s1) break;
      put_x(0);
    }
    wg_barrier();   // the buffers are read
  } else if (s0 < s1) {
    int xo[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f)
      xo[f] = (list[16 * f + m < n ? 16 * f + m : n - 1] / per * int(a.ld_x) + (I8 ? 16 : 8) * q) * 2;
    fm_u32x4 wa[C][2][NR][WL], wb[C][2][NR][WL];
    auto use = [&](const fm_u32x4 (&w)[C][2][NR][WL], const fm_u32x4 (&x)[C][XL][TF][2], int s) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        if (s + u >= s1) break;
        step(w[u], [&](int p, int l, int f) { return __builtin_bit_cast(v8bf, x[u][p][f][l]); });
      }
    };
    fm_u32x4 xa[C][XL][TF][2], xb[C][XL][TF][2];
    auto load_x = [&](fm_u32x4 (&x)[C][XL][TF][2], int s) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        const int k = s + u < s1 ? s + u : s1 - 1;
#pragma unroll
        for (int p = 0; p < XL; ++p)
#pragma unroll
          for (int f = 0; f < TF; ++f)
#pragma unroll
            for (int l = 0; l < 2; ++l)
              x[u][p][f][l] = FM_BUFFER_LOAD16(p ? rl : rx, xo[f], k * 128 + l * (I8 ? 16 : 64));
      }
    };
    load_x(xa, s0);
    load_w(wa, s0);
    for (int s = s0; s < s1; s += 2 * C) {
      load_x(xb, s + C);
      load_w(wb, s + C);
      use(wa, xa, s);
      load_x(xa, s + 2 * C);
      load_w(wa, s + 2 * C);
      use(wb, xb, s + C);
    }
  }

  uint16_t* hh = reinterpret_cast<uint16_t*>(lds);      // [16 TF][P] high pieces, then low
  uint16_t* hl = hh + 16 * TF * P;
  if constexpr (KG > 1) {
    // the parts of D meet in LDS in their order; [part][gate|up][NR][TF][lane] of 16 bytes
    fm_f32x4* red = reinterpret_cast<fm_f32x4*>(lds);
    constexpr int N = 2 * NR * TF;
    if (kg > 0) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int f = 0; f < TF; ++f)
            red[(((kg - 1) * RG + rg) * N + (b * NR + r) * TF + f) * 64 + lane] = __builtin_bit_cast(fm_f32x4, acc[b][r][f]);
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int p = 0; p < KG - 1; ++p)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int f = 0; f < TF; ++f)
              acc[b][r][f] += __builtin_bit_cast(v4f, red[((p * RG + rg) * N + (b * NR + r) * TF + f) * 64 + lane]);
    }
    __syncthreads();
  }
  if (kg == 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      v4f g1 = {1.f, 1.f, 1.f, 1.f}, g3 = g1;
      if constexpr (I8) {
        const int64_t at = int64_t(e) * x.H + hid + 16 * r + 4 * q;
        g1 = *reinterpret_cast<const v4f*>(x.s1 + at);
        g3 = *reinterpret_cast<const v4f*>(x.s3 + at);
      }
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        float h[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float g = I8 ? acc[0][r][f][v] * g1[v] : acc[0][r][f][v];
          const float u = I8 ? acc[1][r][f][v] * g3[v] : acc[1][r][f][v];
          h[v] = g / (1.f + expf(-g)) * u;
        }
        const uint32_t h0 = hw_bf16x2(h[0], h[1]), h1 = hw_bf16x2(h[2], h[3]);
        const uint32_t l0 = hw_bf16x2(h[0] - u2f(h0 << 16), h[1] - u2f(h0 & 0xffff0000u));
        const uint32_t l1 = hw_bf16x2(h[2] - u2f(h1 << 16), h[3] - u2f(h1 & 0xffff0000u));
        const int at = (16 * f + m) * P + rg * 16 * NR + 16 * r + 4 * q;
        *reinterpret_cast<fm_u32x2*>(hh + at) = fm_u32x2{h0, h1};
        *reinterpret_cast<fm_u32x2*>(hl + at) = fm_u32x2{l0, l1};
      }
    }
  }
  __syncthreads();

  // ---- down: rows output columns, columns tokens
  float* part[TF];
#pragma unroll
  for (int f = 0; f < TF; ++f) {
    const int i = 16 * f + m;
    part[f] = i < n ? x.part + (int64_t(list[i]) * x.S + slice) * D : nullptr;
  }
  if constexpr (I8) {
    static_assert(HS % 64 == 0, "whole tiles of W2");
    constexpr int KT = HS / 64, C2 = TF * KT > 4 ? 2 : TF * KT > 2 ? 4 : 8;    // output tiles of a step
    const int tile_row = x.H / 64 * 1024;                // bytes of 16 output columns
    const int64_t down = int64_t(x.H) * D;               // bytes of an expert's W2; the slice's tiles start at slice * KT
    const auto r2 = buffer_of(x.w2 + e * down, down);
    const int v_off = lane * 16 + slice * KT * 1024;
    const int tiles = a.D / 16;
    auto load2 = [&](fm_u32x4 (&v)[C2][KT], int d) {
#pragma unroll
      for (int c = 0; c < C2; ++c) {
        const int dt = d + c < tiles ? d + c : tiles - 1;
#pragma unroll
        for (int k = 0; k < KT; ++k) v[c][k] = FM_BUFFER_LOAD16(r2, v_off, dt * tile_row + k * 1024);
      }
    };
    auto use2 = [&](const fm_u32x4 (&v)[C2][KT], int d) {
      v4f o[C2][TF];
#pragma unroll
      for (int c = 0; c < C2; ++c)
#pragma unroll
        for (int f = 0; f < TF; ++f) o[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          v8bf hv[TF], lv[TF];
#pragma unroll
          for (int f = 0; f < TF; ++f) {
            const int at = (16 * f + m) * P + 64 * k + 16 * q + 8 * l;
            hv[f] = *reinterpret_cast<const v8bf*>(hh + at);
            lv[f] = *reinterpret_cast<const v8bf*>(hl + at);
          }
#pragma unroll
          for (int c = 0; c < C2; ++c) {
            const v8bf w = i8_to_bf16(v[c][k][2 * l], v[c][k][2 * l + 1]);
#pragma unroll
            for (int f = 0; f < TF; ++f) o[c][f] = mfma(w, lv[f], mfma(w, hv[f], o[c][f]));
          }
        }
#pragma unroll
      for (int c = 0; c < C2; ++c) {   // the channels' scales come in with the sum over slices
        if (d + c >= tiles) break;
#pragma unroll
        for (int f = 0; f < TF; ++f)
          if (part[f]) st_global(part[f] + (d + c) * 16 + 4 * q, make_float4(o[c][f][0], o[c][f][1], o[c][f][2], o[c][f][3]));
      }
    };
    fm_u32x4 va[C2][KT], vb[C2][KT];
    constexpr int kAll = 4 * C2;   // tiles of a step of the four waves
    if (wave * C2 < tiles) {
      load2(va, wave * C2);
      for (int d = wave * C2;; d += 2 * kAll) {
        load2(vb, d + kAll);
        use2(va, d);
        if (d + kAll >= tiles) break;
        load2(va, d + 2 * kAll);
        use2(vb, d + kAll);
        if (d + 2 * kAll >= tiles) break;
      }
    }
  } else {
    // 16 CW output columns a block: lane (m, q) loads rows 8 q + i of each 32, columns CW m .. + CW;
    // a unit is UK such 32s (HS = 16: 4 rows a lane, in fragments 16 deep)
    constexpr int CW = TF == 4 ? 4 : 8, KB = (HS + 31) / 32, UK = KB == 1 ? 1 : 2, NU = KB / UK;
    typedef std::conditional_t<CW == 8, fm_u32x4, fm_u32x2> Row;
    constexpr int R = HS < 32 ? HS / 4 : 8;
    const auto r2 = buffer_of(x.w2 + (int64_t(e) * x.H + slice * HS) * D * 2, HS * D * 2);
    const int v_off = (R * q * a.D + CW * m) * 2;
    const int blocks = a.D / (16 * CW);
    v4f o[CW][TF];
    auto load2 = [&](Row (&v)[UK][R], int unit) {   // the wave's unit: block 4 (unit / NU) + wave
      const int d = unit / NU * 4 + wave;
      const int dd = d < blocks ? d : blocks - 1;
#pragma unroll
      for (int k = 0; k < UK; ++k)
#pragma unroll
        for (int i = 0; i < R; ++i)
          v[k][i] = load_row<Row>(r2, v_off, ((32 * (unit % NU * UK + k) + i) * a.D + dd * 16 * CW) * 2);
    };
    auto use2 = [&](const Row (&v)[UK][R], int unit) {
      if (unit % NU == 0) {
#pragma unroll
        for (int c = 0; c < CW; ++c)
#pragma unroll
          for (int f = 0; f < TF; ++f) o[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int k = 0; k < UK; ++k) {
        const int kb = unit % NU * UK + k;
        // fragment 2 j + p: column CW r + 2 j + p of row r, from the halves p of dword j of the lane's rows
        if constexpr (R == 8) {
          v8bf hv[TF], lv[TF];
#pragma unroll
          for (int f = 0; f < TF; ++f) {
            const int at = (16 * f + m) * P + 32 * kb + 8 * q;
            hv[f] = *reinterpret_cast<const v8bf*>(hh + at);
            lv[f] = *reinterpret_cast<const v8bf*>(hl + at);
          }
#pragma unroll
          for (int j = 0; j < CW / 2; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              fm_u32x4 w;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = __builtin_amdgcn_perm(v[k][2 * i + 1][j], v[k][2 * i][j], p ? 0x07060302u : 0x05040100u);
              const v8bf wf = __builtin_bit_cast(v8bf, w);
#pragma unroll
              for (int f = 0; f < TF; ++f) o[2 * j + p][f] = mfma(wf, lv[f], mfma(wf, hv[f], o[2 * j + p][f]));
            }
        } else {
          v4s16 hv[TF], lv[TF];
#pragma unroll
          for (int f = 0; f < TF; ++f) {
            const int at = (16 * f + m) * P + 4 * q;
            hv[f] = *reinterpret_cast<const v4s16*>(hh + at);
            lv[f] = *reinterpret_cast<const v4s16*>(hl + at);
          }
#pragma unroll
          for (int j = 0; j < CW / 2; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              fm_u32x2 w;
#pragma unroll
              for (int i = 0; i < 2; ++i)
                w[i] = __builtin_amdgcn_perm(v[k][2 * i + 1][j], v[k][2 * i][j], p ? 0x07060302u : 0x05040100u);
              const v4s16 wf = __builtin_bit_cast(v4s16, w);
#pragma unroll
              for (int f = 0; f < TF; ++f) {
                v4f& t = o[2 * j + p][f];
                t = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(wf, hv[f], t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(wf, lv[f], t, 0, 0, 0);
              }
            }
        }
      }
      if (unit % NU != NU - 1) return;
      // fragment c's row 4 q + i is column CW (4 q + i) + c
      const int d = unit / NU * 4 + wave;
#pragma unroll
      for (int f = 0; f < TF; ++f)
        if (part[f]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* p = part[f] + d * 16 * CW + CW * (4 * q + i);
#pragma unroll
            for (int c = 0; c < CW; c += 4)
              st_global(p + c, make_float4(o[c][f][i], o[c + 1][f][i], o[c + 2][f][i], o[c + 3][f][i]));
          }
        }
    };
    const int units = wave < blocks ? (blocks - wave + 3) / 4 * NU : 0;
    Row va[UK][R], vb[UK][R];
    if (units > 0) {
      load2(va, 0);
      for (int u = 0;; u += 2) {
        load2(vb, u + 1);
        use2(va, u);
        if (u + 1 >= units) break;
        load2(va, u + 2);
        use2(vb, u + 1);
        if (u + 2 >= units) break;
      }
    }
  }
  __syncthreads();   // h is read before the next pass's
}

template <bool I8, bool LO, int NR, int RG>
__global__ __launch_bounds__(256, 2) void decode_experts_kernel(ExpertArgs a) {
  using S = Slice<I8, LO, NR, RG>;
  constexpr int kH = 16 * 4 * S::kPitch * 2 * 2;                                        // h of 64 tokens, two pieces
  constexpr int kRed = S::KG > 1 ? (S::KG - 1) * RG * 2 * NR * 4 * 64 * 16 : 0;        // the parts of D
  constexpr int kX = S::KG == 1 ? 2 * (LO ? 2 : 1) * 64 * (64 * 2 + 8) * 2 : 0;          // the tokens' chunks (TF 2 and 4 need this, TF 1 half)
  constexpr int kXR = kH > kRed ? kH : kRed;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kX > kXR ? kX : kXR];
  __shared__ int list[kDecodeTokens * kDecodeTopK];
  __shared__ uint32_t bits[kDecodeExperts / 32];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool shared = int(blockIdx.x) < a.s.S;
  int n, e, slice;
  if (shared) {
    slice = blockIdx.x;
    e = 0;
    n = a.T;
    for (int i = tid; i < n; i += 256) list[i] = i;
  } else {
    const int b = int(blockIdx.x) - a.s.S, pick = b / a.r.S, A = a.T * a.K;
    slice = b - pick * a.r.S;
    for (int i = tid; i < kDecodeExperts / 32; i += 256) bits[i] = 0;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int i = tid; i < A; i += 256) {
      const int v = expert_of(a, i);
      if (v >= 0) atomicOr(&bits[v >> 5], 1u << (v & 31));
    }
    __syncthreads();
    if (tid < 64) {   // the pick-th reached expert, then its assignments in order
      const uint32_t w = lane < kDecodeExperts / 32 ? bits[lane] : 0;
      int before = __popc(w);
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(before, off);
        if (lane >= off) before += o;
      }
      before -= __popc(w);
      const int in = pick - before;
      if (in >= 0 && in < __popc(w)) {
        uint32_t v = w;
        for (int i = 0; i < in; ++i) v &= v - 1;
        found[0] = lane * 32 + __ffs(v) - 1;
      }
    }
    __syncthreads();
    e = found[0];
    if (e < 0) return;   // the same for the whole workgroup
    if (tid < 64) {
      int at = 0;
      for (int i0 = 0; i0 < A; i0 += 64) {
        const bool hit = i0 + lane < A && expert_of(a, i0 + lane) == e;
        const uint64_t bal = __ballot(hit);
        if (hit) list[at + __popcll(bal & ((uint64_t(1) << lane) - 1))] = i0 + lane;
        at += __popcll(bal);
      }
      if (lane == 0) found[1] = at;
    }
  }
  __syncthreads();
  if (!shared) n = found[1];
  e = __builtin_amdgcn_readfirstlane(e);
  n = __builtin_amdgcn_readfirstlane(n);
  slice = __builtin_amdgcn_readfirstlane(slice);
  const Expert x = shared ? a.s : a.r;
  const int per = shared ? 1 : a.K;
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int left = n - t0;
    if (left > 32) slice_pass<I8, LO, NR, RG, 4>(a, x, e, slice, list + t0, left, per, lds);
    else if (left > 16) slice_pass<I8, LO, NR, RG, 2>(a, x, e, slice, list + t0, left, per, lds);
    else slice_pass<I8, LO, NR, RG, 1>(a, x, e, slice, list + t0, left, per, lds);
  }
}

// out[t] = sum_k w[t, k] (sum over slices) + the shared expert's slices.  A
// workgroup takes 64 columns of one token: 16 lanes of 4 columns, 16 groups over
// the shares in strides, the groups' sums added in order.
__global__ __launch_bounds__(256) void decode_combine_kernel(ExpertArgs a, const float* w, void* out, int out_f32, int64_t ld_o) {
  __shared__ fm_f32x4 red[16][16];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, t = blockIdx.y;
  const int64_t col = int64_t(blockIdx.x) * 64 + c * 4;
  fm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.K; ++k) {
    const int i = t * a.K + k;
    const int e = expert_of(a, i);
    if (e < 0) continue;
    const float* p = a.r.part + int64_t(i) * a.r.S * a.D + col;
    fm_f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = g; s < a.r.S; s += 16) y += *reinterpret_cast<const fm_f32x4*>(p + int64_t(s) * a.D);
    if (a.r.s2) y *= *reinterpret_cast<const fm_f32x4*>(a.r.s2 + int64_t(e) * a.D + col);
    sum += y * w[i];
  }
  fm_f32x4 ys = {0.f, 0.f, 0.f, 0.f};
  const float* p = a.s.part + int64_t(t) * a.s.S * a.D + col;
#pragma unroll 4
  for (int s = g; s < a.s.S; s += 16) ys += *reinterpret_cast<const fm_f32x4*>(p + int64_t(s) * a.D);
  if (a.s.S && a.s.s2) ys *= *reinterpret_cast<const fm_f32x4*>(a.s.s2 + col);
  sum += ys;
  red[g][c] = sum;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += red[i][c];
  if (out_f32) st_global(static_cast<float*>(out) + t * ld_o + col, make_float4(sum[0], sum[1], sum[2], sum[3]));
  else st_global(static_cast<uint16_t*>(out) + t * ld_o + col, make_uint2(hw_bf16x2(sum[0], sum[1]), hw_bf16x2(sum[2], sum[3])));
}

// Hidden units of a workgroup: 128 where the reached experts still give about two
// workgroups a CU, fewer where they do not.  Int8 tiles of W2 are 64 deep.
inline int slice_of(int64_t H, int64_t experts, bool i8) {
  const int64_t want = 2 * 256;
  for (int hs : {128, 64, 32}) {
    if (hs < 64 && i8) break;
    if (H % hs == 0 && experts * (H / hs) >= want) return hs;
  }
  return i8 ? 64 : 16;
}

struct DecodePlan {
  int hs;
  int64_t reach, part, bytes;   // part: the routed experts' shares
};
inline DecodePlan decode_plan(int64_t T, int64_t D, int64_t K, int64_t E, int64_t H, int64_t Hs, bool i8) {
  DecodePlan p;
  p.reach = E < T * K ? E : T * K;
  p.hs = slice_of(H, p.reach, i8);
  p.part = T * K * (H / p.hs) * D * 4;
  p.bytes = p.part + T * (Hs / p.hs) * D * 4;
  return p;
}

template <bool I8, bool LO>
void launch_experts(const ExpertArgs& a, int hs, int64_t blocks, hipStream_t s) {
  const dim3 grid{unsigned(blocks)}, block(256);
  if (hs == 128) hipLaunchKernelGGL((decode_experts_kernel<I8, LO, 2, 4>), grid, block, 0, s, a);
  else if (hs == 64) hipLaunchKernelGGL((decode_experts_kernel<I8, LO, 1, 4>), grid, block, 0, s, a);
  else if constexpr (!I8) {
    if (hs == 32) hipLaunchKernelGGL((decode_experts_kernel<I8, LO, 1, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((decode_experts_kernel<I8, LO, 1, 1>), grid, block, 0, s, a);
  }
}

int expert_of_weights(const FmDecodeWeights* w, bool i8, int S, float* part, Expert& x) {
  FM_REQUIRE(w->w1 && w->w2 && w->w3 && aligned16(w->w1) && aligned16(w->w2) && aligned16(w->w3),
             "fm_decode_experts: expert weights must be given and 16-byte aligned");
  FM_REQUIRE(!i8 || (w->s1 && w->s2 && w->s3 && aligned16(w->s1) && aligned16(w->s2) && aligned16(w->s3)),
             "fm_decode_experts: int8 weights need their scales, 16-byte aligned");
  FM_REQUIRE((w->kind == FM_DECODE_INT8) == i8, "fm_decode_experts: routed and shared experts must be of one kind");
  x = Expert{static_cast<const uint8_t*>(w->w1), static_cast<const uint8_t*>(w->w3), static_cast<const uint8_t*>(w->w2),
             i8 ? w->s1 : nullptr, i8 ? w->s3 : nullptr, i8 ? w->s2 : nullptr, int(w->H), S, part};
  return 0;
}

bool decode_sizes_ok(int64_t T, int64_t D, int64_t K, int64_t E, int64_t H, int64_t Hs) {
  return T >= 1 && T <= kDecodeTokens && D >= 128 && D <= kDecodeDim && D % 128 == 0 && K >= 1 && K <= kDecodeTopK &&
         E >= 1 && E <= kDecodeExperts && H >= 128 && H % 128 == 0 && H <= (1 << 20) && Hs >= 0 && Hs % 128 == 0 &&
         Hs <= (1 << 20) && (H > Hs ? H : Hs) * D < (int64_t(1) << 31);
}

}  // namespace

}  // namespace fm

using namespace fm;

extern "C" {

int fm_decode_router(const void* x, int64_t ld_x, int64_t T, int64_t D, const void* gate, int gate_dtype, int64_t ld_g,
                     const void* bias, int bias_dtype, const float* score_bias, const void* norm, int norm_dtype,
                     float eps, int E, int K, int gating, int flags, float* logits, void* x_hi, void* x_lo,
                     float* weights, int64_t* indices, void* stream) {
  FM_REQUIRE(x && gate && weights && indices, "fm_decode_router: null pointer");
  FM_REQUIRE(decode_sizes_ok(T, D, K, E, 128, 0) && K <= E,
             "fm_decode_router: needs 1..64 tokens, D a multiple of 128 up to 14336, at most 1024 experts and K <= min(E, 16)");
  FM_REQUIRE((gate_dtype == FM_DTYPE_BF16 || gate_dtype == FM_DTYPE_F32) && (bias_dtype == FM_DTYPE_BF16 || bias_dtype == FM_DTYPE_F32) &&
                 (norm_dtype == FM_DTYPE_BF16 || norm_dtype == FM_DTYPE_F32), "fm_decode_router: bad dtype");
  FM_REQUIRE(gating == FM_GATING_SOFTMAX || gating == FM_GATING_SIGMOID, "fm_decode_router: bad gating");
  FM_REQUIRE(aligned16(x) && ld_x >= D && ld_x % 8 == 0 && aligned16(gate) && ld_g >= D && ld_g % (gate_dtype == FM_DTYPE_F32 ? 4 : 8) == 0 &&
                 aligned16(norm), "fm_decode_router: rows must start on 16-byte boundaries");
  FM_REQUIRE(!norm || (x_hi && x_lo && aligned16(x_hi) && aligned16(x_lo)), "fm_decode_router: a norm needs x_hi and x_lo");
  const RouterArgs a{static_cast<const uint16_t*>(x), ld_x, int(T), int(D), gate, gate_dtype == FM_DTYPE_F32, ld_g, bias,
                     bias_dtype == FM_DTYPE_F32, score_bias, norm, norm_dtype == FM_DTYPE_F32, eps, E, K,
                     gating == FM_GATING_SIGMOID, (flags & FM_GATING_L2_NORMALIZE) != 0, logits,
                     static_cast<uint16_t*>(x_hi), static_cast<uint16_t*>(x_lo), weights, indices};
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int NW = 8;
  // one workgroup a token where a gate is small enough for one CU to read; else 32 experts a workgroup and a second launch
  const bool one = int64_t(E) * D <= 64 * 1024;
  const int per = one ? E : 32;
  FM_REQUIRE(one || logits, "fm_decode_router: this gate needs logits [T, E]");
  const size_t lds = size_t(D + per + NW) * 4;
  hipLaunchKernelGGL(decode_router_kernel<NW>, dim3(unsigned((E + per - 1) / per), unsigned(T)), dim3(64 * NW), lds, s, a, per,
                     int(one));
  if (!one) hipLaunchKernelGGL(decode_gate_kernel, dim3{unsigned(T)}, dim3(64), 0, s, a);
  return check_launch("fm_decode_router");
}

int64_t fm_decode_workspace_bytes(int64_t T, int64_t D, int K, int E, int64_t H, int64_t H_shared, int kind) {
  if (!decode_sizes_ok(T, D, K, E, H, H_shared)) return -1;
  return decode_plan(T, D, K, E, H, H_shared, kind == FM_DECODE_INT8).bytes;
}

int fm_decode_experts(const void* x, const void* x_lo, int64_t ld_x, int64_t T, int64_t D, const float* weights,
                      const void* indices, int indices_i64, int K, int64_t expert_offset, int E,
                      const FmDecodeWeights* experts, const FmDecodeWeights* shared, void* out, int out_dtype,
                      int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  FM_REQUIRE(x && weights && indices && experts && out && workspace, "fm_decode_experts: null pointer");
  const int64_t Hs = shared ? shared->H : 0;
  FM_REQUIRE(decode_sizes_ok(T, D, K, E, experts->H, Hs) && (!shared || Hs > 0),
             "fm_decode_experts: needs 1..64 tokens, D and hidden sizes multiples of 128 (D up to 14336), K <= 16 and at most 1024 experts");
  FM_REQUIRE(experts->kind == FM_DECODE_BF16 || experts->kind == FM_DECODE_INT8, "fm_decode_experts: bad weight kind");
  FM_REQUIRE(aligned16(x) && aligned16(x_lo) && ld_x >= D && ld_x % 8 == 0 && ld_x <= (1 << 23) && aligned16(workspace),
             "fm_decode_experts: rows must start on 16-byte boundaries, at a pitch of at most 2^23");
  FM_REQUIRE((out_dtype == FM_DTYPE_BF16 || out_dtype == FM_DTYPE_F32) && aligned16(out) && ld_out >= D && ld_out % 4 == 0,
             "fm_decode_experts: output must be bf16 or fp32, 16-byte aligned, its pitch at least D and a multiple of 4");
  const bool i8 = experts->kind == FM_DECODE_INT8;
  const DecodePlan p = decode_plan(T, D, K, E, experts->H, Hs, i8);
  FM_REQUIRE(workspace_bytes >= p.bytes, "fm_decode_experts: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)p.bytes);
  float* part = static_cast<float*>(workspace);
  ExpertArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(x_lo), ld_x, int(T), int(D), K, E, indices,
               indices_i64, expert_offset, {}, {}};
  if (int rc = expert_of_weights(experts, i8, int(experts->H / p.hs), part, a.r)) return rc;
  if (shared) {
    if (int rc = expert_of_weights(shared, i8, int(Hs / p.hs), part + p.part / 4, a.s)) return rc;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t blocks = p.reach * a.r.S + a.s.S;
  if (i8) {
    if (x_lo) launch_experts<true, true>(a, p.hs, blocks, s);
    else launch_experts<true, false>(a, p.hs, blocks, s);
  } else {
    if (x_lo) launch_experts<false, true>(a, p.hs, blocks, s);
    else launch_experts<false, false>(a, p.hs, blocks, s);
  }
  hipLaunchKernelGGL(decode_combine_kernel, dim3(unsigned(D / 64), unsigned(T)), dim3(256), 0, s, a, weights, out,
                     int(out_dtype == FM_DTYPE_F32), ld_out);
  return check_launch("fm_decode_experts");
}

}  // extern "C"
