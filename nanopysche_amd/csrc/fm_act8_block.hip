// The expert block's backward from activations in 8 bits (fm_act8.h): the operands of its grouped products, made from the
// kept gate|up, tokens and expert outputs by the tile producers of the 16-bit ones.  The first and the fourth take the place of
// passes there; the others are passes more, whose results the 16-bit block has from its forward, or (the last) forms with the gating's gradient.
//   fm_act8_swiglu_keep_quantize      the forward's h, as fm_swiglu_quantize, keeping gate|up on the way
//   fm_act8_permute                   the tokens in expert order, as fm_permute
//   fm_act8_swiglu_quantize           h = silu(g) u of the kept g and u, as fm_swiglu_quantize
//   fm_act8_swiglu_backward_quantize  [dg | du], as fm_swiglu_backward
//   fm_act8_router_weight_grad        dw[t, k] = <dout[t], y[row(t, k)]>, as fm_router_weight_grad
// 33664 rows, H 1408, D 2048, bf16 operands: 80, 80, 76, 172 and 25 us, of 62, 28, 31, 92 and 22 for the bytes: the transposed outputs.
// The tile producer's 128 columns are four of the format's blocks, so a lane's eight values have one code.
#include "fm_act8.h"
#include "fm_lanes.h"
#include "fm_silu.h"
#include "../../include/fm_hip.h"

namespace fm {
namespace {

struct KeptGatherSrc {
  static constexpr int kOut = 1;
  Act8 x;
  const int32_t* assign_of_row;
  int K;
  struct Raw {
    uint2 b;
    uint32_t code;
    bool ok;
  };
  __device__ __forceinline__ Raw fetch(int64_t row, int64_t col) const {
    const int32_t a = assign_of_row[row];
    const int64_t t = (a >= 0 ? a : 0) / K;   // a pad row reads token 0 and is zeroed below
    return Raw{x.bytes(t, col), x.code(t, col), a >= 0};
  }
  __device__ __forceinline__ void compute(const Raw& r, float v[][8]) const {
    float f[8];
    act_decode8(r.b, act_scale(r.code), f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0][i] = r.ok ? f[i] : 0.f;
  }
};

// No tokens: pad rows alone.
struct NoTokensSrc {
  static constexpr int kOut = 1;
  struct Raw {};
  __device__ __forceinline__ Raw fetch(int64_t, int64_t) const { return Raw{}; }
  __device__ __forceinline__ void compute(const Raw&, float v[][8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0][i] = 0.f;
  }
};

struct KeptSwigluSrc {
  static constexpr int kOut = 1;
  Act8 gu;      // gate's columns, then up's
  int64_t H;
  struct Raw {
    uint2 g, u;
    uint32_t gc, uc;
  };
  __device__ __forceinline__ Raw fetch(int64_t row, int64_t col) const {
    return Raw{gu.bytes(row, col), gu.bytes(row, col + H), gu.code(row, col), gu.code(row, col + H)};
  }
  __device__ __forceinline__ void compute(const Raw& r, float v[][8]) const {
    float g[8], u[8];
    act_decode8(r.g, act_scale(r.gc), g);
    act_decode8(r.u, act_scale(r.uc), u);
    swiglu8(g, u, v[0]);
  }
};

// The forward: h of bf16 gate|up, which compute stores in 8 bits as well.  Row outputs only: the producer then computes every row
// in range once, its quads of lanes together.
struct KeepSwigluSrc {
  static constexpr int kOut = 1;
  const uint16_t* gu;   // bf16 [rows, ld]
  int64_t ld, H;
  uint8_t* q;
  int64_t ld_q;
  uint8_t* codes;
  int64_t ld_c;
  struct Raw {
    uint4 g, u;
    int64_t row, col;
  };
  __device__ __forceinline__ Raw fetch(int64_t row, int64_t col) const {
    const uint16_t* p = gu + row * ld + col;
    return Raw{*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + H), row, col};
  }
  __device__ __forceinline__ void keep(const float (&v)[8], int64_t row, int64_t col) const {
    uint32_t code;
    const uint2 b = act_encode8(v, code);
    st_global(q + row * ld_q + col, b);
    if ((threadIdx.x & 3) == 0) st_global(codes + row * ld_c + (col >> 5), uint8_t(code));
  }
  __device__ __forceinline__ void compute(const Raw& r, float v[][8]) const {
    float g[8], u[8];
    unpack8_bf16(r.g, g);
    unpack8_bf16(r.u, u);
    keep(g, r.row, r.col);
    keep(u, r.row, r.col + H);
    swiglu8(g, u, v[0]);
  }
};

struct KeptSwigluBwdSrc {
  static constexpr int kOut = 2;
  KeptSwigluSrc kept;
  const uint16_t* dh;
  int64_t ld_dh;
  struct Raw {
    KeptSwigluSrc::Raw kept;
    uint4 dh;
  };
  __device__ __forceinline__ Raw fetch(int64_t row, int64_t col) const {
    return Raw{kept.fetch(row, col), *reinterpret_cast<const uint4*>(dh + row * ld_dh + col)};
  }
  __device__ __forceinline__ void compute(const Raw& r, float v[][8]) const {
    float g[8], u[8], d[8];
    act_decode8(r.kept.g, act_scale(r.kept.gc), g);
    act_decode8(r.kept.u, act_scale(r.kept.uc), u);
    unpack8_bf16(r.dh, d);
    swiglu8_backward(g, u, d, v[0], v[1]);
  }
};

// One wave an assignment: four 512-column chunks' loads before their products, then a sum over the lanes.
__global__ __launch_bounds__(256) void kept_router_grad_kernel(const uint16_t* __restrict__ dout, int64_t ld_do, Act8 y,
                                                               const int32_t* __restrict__ row_of, int64_t A, int K, int64_t D,
                                                               float* __restrict__ dw) {
  const int lane = threadIdx.x & 63;
  for (int64_t a = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); a < A; a += int64_t(gridDim.x) * 4) {
    const int32_t r = row_of[a];
    float acc = 0.f;
    if (r >= 0) {
      const uint16_t* g = dout + (a / K) * ld_do;
      for (int64_t c0 = 0; c0 < D; c0 += 4 * 512) {
        uint4 p[4];
        uint2 q[4];
        uint32_t code[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t c = c0 + 512 * u + 8 * lane, at = c < D ? c : 0;
          p[u] = c < D ? *reinterpret_cast<const uint4*>(g + c) : make_uint4(0, 0, 0, 0);
          q[u] = y.bytes(r, at);
          code[u] = c < D ? y.code(r, at) : 0u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float d[8], v[8];
          unpack8_bf16(p[u], d);
          act_decode8(q[u], act_scale(code[u]), v);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc = fmaf(d[i], v[i], acc);
        }
      }
    }
    acc = group_sum<64>(acc);
    if (lane == 0) st_global(dw + a, acc);
  }
}

Act8 kept_of(const void* q, int64_t ld_q, const void* codes, int64_t ld_c) {
  return Act8{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(codes), ld_q, ld_c};
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" {

int fm_act8_permute(const void* xq, int64_t ld_xq, const void* codes, int64_t ld_c, int64_t T, int64_t D, const int32_t* assign_of_row,
                    int64_t rows, int K, int kind, void* q, int64_t ld_q, void* s, int64_t ld_s, void* qt, int64_t ld_qt, void* st,
                    int64_t ld_st, const int32_t* tile_valid, void* stream) {
  FM_REQUIRE(T >= 0 && K >= 1 && assign_of_row, "fm_act8_permute: bad sizes or null assign_of_row");
  FM_REQUIRE(T == 0 || kept_ok(xq, ld_xq, codes, ld_c, D), "fm_act8_permute: bad payload, codes or pitches");
  const TileOut o = make_tile_out(kind, q, ld_q, s, ld_s, qt, ld_qt, st, ld_st, 0, 0, tile_valid);
  if (T == 0) return launch_tile_producer(NoTokensSrc{}, o, rows, D, static_cast<hipStream_t>(stream), "fm_act8_permute");
  return launch_tile_producer(KeptGatherSrc{kept_of(xq, ld_xq, codes, ld_c), assign_of_row, K}, o, rows, D,
                              static_cast<hipStream_t>(stream), "fm_act8_permute");
}

int fm_act8_swiglu_keep_quantize(const void* gu, int64_t ld_gu, int64_t rows, int64_t H, void* q8, int64_t ld_q8, void* codes, int64_t ld_c,
                                 int kind, void* q, int64_t ld_q, void* s, int64_t ld_s, const int32_t* tile_valid, void* stream) {
  FM_REQUIRE(H >= 128 && H % 128 == 0 && rows % 128 == 0, "fm_act8_swiglu_keep_quantize: H and rows must be multiples of 128");
  FM_REQUIRE(rows == 0 || (gu && aligned16(gu) && ld_gu >= 2 * H && ld_gu % 8 == 0),
             "fm_act8_swiglu_keep_quantize: gate|up must lie on 16 bytes, its pitch a multiple of 8");
  FM_REQUIRE(rows == 0 || kept_ok(q8, ld_q8, codes, ld_c, 2 * H), "fm_act8_swiglu_keep_quantize: bad payload, codes or pitches");
  const TileOut o = make_tile_out(kind, q, ld_q, s, ld_s, nullptr, 0, nullptr, 0, 0, 0, tile_valid);
  return launch_tile_producer(KeepSwigluSrc{static_cast<const uint16_t*>(gu), ld_gu, H, static_cast<uint8_t*>(q8), ld_q8,
                                            static_cast<uint8_t*>(codes), ld_c},
                              o, rows, H, static_cast<hipStream_t>(stream), "fm_act8_swiglu_keep_quantize");
}

int fm_act8_swiglu_quantize(const void* gu, int64_t ld_gu, const void* codes, int64_t ld_c, int64_t rows, int64_t H, int kind, void* q,
                            int64_t ld_q, void* s, int64_t ld_s, void* qt, int64_t ld_qt, void* st, int64_t ld_st,
                            const int32_t* tile_valid, void* stream) {
  FM_REQUIRE(H >= 128 && H % 128 == 0, "fm_act8_swiglu_quantize: H must be a positive multiple of 128");
  FM_REQUIRE(rows == 0 || kept_ok(gu, ld_gu, codes, ld_c, 2 * H), "fm_act8_swiglu_quantize: bad payload, codes or pitches");
  const TileOut o = make_tile_out(kind, q, ld_q, s, ld_s, qt, ld_qt, st, ld_st, 0, 0, tile_valid);
  return launch_tile_producer(KeptSwigluSrc{kept_of(gu, ld_gu, codes, ld_c), H}, o, rows, H, static_cast<hipStream_t>(stream),
                              "fm_act8_swiglu_quantize");
}

int fm_act8_swiglu_backward_quantize(const void* gu, int64_t ld_gu, const void* codes, int64_t ld_c, const void* dh, int64_t ld_dh,
                                     int64_t rows, int64_t H, int kind, void* q, int64_t ld_q, void* s, int64_t ld_s, void* qt,
                                     int64_t ld_qt, void* st, int64_t ld_st, const int32_t* tile_valid, void* stream) {
  FM_REQUIRE(H >= 128 && H % 128 == 0, "fm_act8_swiglu_backward_quantize: H must be a positive multiple of 128");
  FM_REQUIRE(rows == 0 || kept_ok(gu, ld_gu, codes, ld_c, 2 * H), "fm_act8_swiglu_backward_quantize: bad payload, codes or pitches");
  FM_REQUIRE(rows == 0 || (dh && aligned16(dh) && ld_dh >= H && ld_dh % 8 == 0),
             "fm_act8_swiglu_backward_quantize: dh must lie on 16 bytes, its pitch a multiple of 8");
  const TileOut o = make_tile_out(kind, q, ld_q, s, ld_s, qt, ld_qt, st, ld_st, 0, H, tile_valid);
  return launch_tile_producer(KeptSwigluBwdSrc{{kept_of(gu, ld_gu, codes, ld_c), H}, static_cast<const uint16_t*>(dh), ld_dh}, o, rows, H,
                              static_cast<hipStream_t>(stream), "fm_act8_swiglu_backward_quantize");
}

int fm_act8_router_weight_grad(const void* dout, int64_t ld_do, const void* y, int64_t ld_y, const void* codes, int64_t ld_c,
                               const int32_t* row_of, int64_t T, int K, int64_t D, float* dw, void* stream) {
  FM_REQUIRE(T >= 0 && K >= 1 && D >= 8 && D % 8 == 0, "fm_act8_router_weight_grad: bad sizes");
  if (T == 0) return 0;
  FM_REQUIRE(dout && row_of && dw && aligned16(dout) && ld_do >= D && ld_do % 8 == 0, "fm_act8_router_weight_grad: null pointer, or dout off "
             "16 bytes");
  FM_REQUIRE(kept_ok(y, ld_y, codes, ld_c, D), "fm_act8_router_weight_grad: bad payload, codes or pitches");
  const int64_t A = T * K;
  const unsigned blocks = unsigned(A / 4 + 1 < 16384 ? A / 4 + 1 : 16384);
  hipLaunchKernelGGL(kept_router_grad_kernel, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(dout),
                     ld_do, kept_of(y, ld_y, codes, ld_c), row_of, A, K, D, dw);
  return check_launch("fm_act8_router_weight_grad");
}

}  // extern "C"
