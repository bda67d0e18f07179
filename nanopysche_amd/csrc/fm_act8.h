// Activations in 8 bits: the format, and its conversions in registers.
//
// A row's blocks of 32 values share a power of two s = 2^k (an e8m0 code):
//   k = max(floor(log2 max|x|) - 6, -127), q = min(max(rint(x / s), -127), 127), code = k + 127.
// The values are those of OCP MX int8, the bytes are not: its element is q 2^-6, so its code of the same block is 6
// above this one, and its smallest scale 2^-133.
// x / s is exact, so q is the correctly rounded quotient (ties to even) in every order of work, and q s,
// a 7-bit whole number times a power of two, is exact in bf16 as in fp32: what a kernel
// rounds is the value once, in the forward.  |x - q s| <= s / 2 (s where |x| is above 127.5 s, which no
// bf16 is), s at most max|x| / 64.  A block that holds a NaN or an infinity gets code 255 and
// stands for NaNs.
//
// Payload: int8 [rows, ld_q], ld_q = cols rounded up to 32, zeros behind cols; codes [rows, ld_q / 32].
// 33 bytes hold 32 values.  A power of two of 32 neighbours rather than a factor of 128: the
// same bytes with an fp32 factor, and an outlier costs its 31 neighbours precision, not 127.
#pragma once

#include "fm_tile.h"

namespace fm {

constexpr int kActBlock = 32;
constexpr uint32_t kActNan = 255;

// vectors at any address of the element's alignment: rows of odd lengths start anywhere
typedef uint32_t u32x4_el __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16_el __attribute__((aligned(2)));

// Code of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t act_code(uint32_t top) {
  const int e = int(top >> 23);   // 255: NaN or infinity
  return e == 255 ? kActNan : uint32_t(max(e - 6, 0));
}
// 2^(127 - code): 1 / s (codes end at 248), 0 for a block of NaNs.
__device__ __forceinline__ float act_inverse(uint32_t code) { return u2f(code == kActNan ? 0u : (254u - code) << 23); }
// s = 2^(code - 127); 2^-127 is a subnormal.
__device__ __forceinline__ float act_scale(uint32_t code) {
  return u2f(code == kActNan ? 0x7fc00000u : max(code << 23, 0x00400000u));
}

// Four values as bytes.  x / s added to 3 * 2^22 leaves the rounded quotient in the sum's low bits (its ulp is 1 there, the
// product exact inside the FMA); the bounds are those of the sum.  A NaN gives any byte.
__device__ __forceinline__ uint32_t act_bytes4(const float* v, float inv) {
  constexpr float kBias = 12582912.f;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = f2u(__builtin_amdgcn_fmed3f(fmaf(v[i], inv, kBias), kBias - 127.f, kBias + 127.f));
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
  return lo | (hi << 16);
}
// Eight neighbours' bytes, and the code they share with the three lanes beside (lanes in fours hold a block).
__device__ __forceinline__ uint2 act_encode8(const float (&v)[8], uint32_t& code) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, f2u(v[i]) & 0x7fffffffu);
  top = max(top, uint32_t(dpp_move<kDppQuadSwap1>(int(top))));
  top = max(top, uint32_t(dpp_move<kDppQuadSwap2>(int(top))));
  code = act_code(top);
  const float inv = act_inverse(code);
  return make_uint2(act_bytes4(v, inv), act_bytes4(v + 4, inv));
}
// q s of four bytes (the conversion takes a sign-extended byte of the word).
__device__ __forceinline__ void act_decode4(uint32_t w, float s, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = float(int8_t(w >> (8 * i))) * s;
}
__device__ __forceinline__ void act_decode8(uint2 w, float s, float (&v)[8]) {
  act_decode4(w.x, s, v);
  act_decode4(w.y, s, v + 4);
}

// A stored matrix as the kernels read it.
struct Act8 {
  const uint8_t* q;      // [rows, ld_q] int8
  const uint8_t* codes;  // [rows, ld_c]
  int64_t ld_q, ld_c;
  __device__ __forceinline__ uint2 bytes(int64_t row, int64_t col) const {
    return *reinterpret_cast<const uint2*>(q + row * ld_q + col);
  }
  __device__ __forceinline__ uint32_t code(int64_t row, int64_t col) const { return codes[row * ld_c + (col >> 5)]; }
};

// Whether a caller's payload and codes are such a matrix of cols columns.
inline bool kept_ok(const void* q, int64_t ld_q, const void* codes, int64_t ld_c, int64_t cols) {
  return q && codes && ld_q >= cols && ld_q % kActBlock == 0 && ld_c * kActBlock >= ld_q && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
}

}  // namespace fm
