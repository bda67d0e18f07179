// The balance loss of packed and padded sequences, its per-expert counts, and its gradient:
//
//   n_s: counting tokens of sequence s;  f_se = (their slots at expert e) / n_s;  P_se = mean of their p_te
//   loss = (E / S') sum_s sum_e f_se P_se + z mean_t lse_t^2,   S': sequences with n_s > 0
//   d loss / d l_te = E / (S' n_s) p_te (f_se - sum_j f_sj p_tj) + (2 z / N) lse_t softmax(l_t)_e   (softmax scores)
//
// p is softmax(l), or sigma / (sum sigma + 1e-8) of sigma = sigmoid(l), then with
// (f_se - sum_j f_sj p_tj) / (sum sigma + 1e-8) sigma (1 - sigma) in place of p (f - sum f p).
// A token counts if it lies in a sequence and its mask says so; the others' logits may hold anything.
//
// Forward: one pass over the logits and indices.  A wave takes a run of C tokens; a token's logits sit in L
// lanes (64 / L tokens side by side), whose column sums stay in registers; the slots are counted in LDS.
// At the end of each sequence in its run the wave writes sums and counts to its own place in the workspace:
// run c and sequence s meet at most once, and runs and sequences both ascend, so place c + s is theirs
// alone.  A second launch adds each sequence's places in order (no float atomics: the same bits each time)
// and leaves E cnt / n^2 for the backward, a third adds the sequences.  Backward: one pass, logits in, gradient out.
#include <type_traits>

#include "fm_lanes.h"
#include "fm_silu.h"
#include "../../include/fm_hip.h"

namespace fm {
namespace {

constexpr int kMaxExperts = 1024;
constexpr float kSumFloor = 1e-8f;

typedef float f32x4_el __attribute__((ext_vector_type(4), aligned(4)));

// e^d for d <= 0 (or NaN) to about an ulp: 2^(d log2 e) by the hardware, the product's rounding error as a factor.
__device__ __forceinline__ float exp_below(float d) {
#pragma clang fp contract(off)
  constexpr float kL = 1.44269502162933349609375f, kLlo = 1.925963033500011e-08f, kLn2 = 0.693147180559945f;
  d = d < -110.f ? -110.f : d;   // 0 there; an infinity has no product error to speak of
  const float h = d * kL;
  const float e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, fmaf(d, kLlo, fmaf(d, kL, -h)) * kLn2, e);
}

struct BalanceArgs {
  const float* logits;
  int64_t ld;
  int64_t T;
  int E, K;
  const void* idx;
  int idx_i64;
  const int32_t* cu;       // [S + 1], or null: one sequence of all tokens
  int64_t S;
  const uint8_t* mask;     // [T], or null
  int sigmoid;
  int want_z;
  int run;                 // tokens of a wave
  float* sums;             // [places, E]
  int32_t* slots;          // [places, E]
  int32_t* tokens;         // [places]
  float* z;                // [places]
};

__device__ __forceinline__ int64_t border(const BalanceArgs& a, int64_t s) {
  if (a.cu == nullptr) return s == 0 ? 0 : a.T;
  const int64_t b = a.cu[s];
  return b < 0 ? 0 : (b > a.T ? a.T : b);
}

// The first sequence that may hold token t: the largest s with border s at or before t (0 if none).  64 candidates a round.
__device__ __forceinline__ int64_t sequence_of(const BalanceArgs& a, int64_t t, int lane) {
  if (a.cu == nullptr) return 0;
  int64_t lo = 0, n = a.S + 1;   // the answer is in [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const int64_t at = lo + lane * step;
    const uint64_t m = __ballot(lane * step < n && a.cu[at < a.S ? at : a.S] <= t);
    const int k = m == 0 ? 0 : 63 - __builtin_clzll(m);
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
    if (m == 0) return 0;
  }
  return lo;
}

// A token's logits over L lanes, NV to a lane (quads: NV / 4 times four neighbours).
template <int L, int NV, bool QUADS>
struct Row {
  float v[NV];
  static __device__ __forceinline__ int column(int l, int i) { return QUADS ? 4 * (l + L * (i / 4)) + i % 4 : l + L * i; }
  __device__ __forceinline__ void load(const float* p, int E, int l) {
    if constexpr (QUADS) {
#pragma unroll
      for (int i = 0; i < NV; i += 4) {
        const int c = column(l, i);
        f32x4_el q = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (c < E) q = *reinterpret_cast<const f32x4_el*>(p + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = q[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = column(l, i);
        v[i] = c < E ? p[c] : -INFINITY;
      }
    }
  }
  // softmax in place; the log of the sum of exponentials
  __device__ __forceinline__ float softmax() {
    float m = v[0], s = 0.f;
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, v[i]);
    m = group_max<L>(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = exp_below(v[i] - m);
      s += v[i];
    }
    s = group_sum<L>(s);
    const float r = 1.f / s;
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] *= r;
    return m + logf(s);
  }
  // sigmoids in place (0 behind the last expert); 1 / (their sum + floor)
  __device__ __forceinline__ float sigmoids(int E, int l) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = column(l, i) < E ? sigmoid_only(v[i]) : 0.f;
      s += v[i];
    }
    return 1.f / (group_sum<L>(s) + kSumFloor);
  }
};

// Steps whose loads are in flight at once: four, as long as they stay within the shortest run.
template <int L>
constexpr int ahead() {
  return 32 * L / 64 >= 4 ? 4 : (32 * L / 64 >= 2 ? 2 : 1);
}

template <int L, int NV, bool QUADS>
__global__ __launch_bounds__(256) void balance_sums_kernel(BalanceArgs a) {
  extern __shared__ int32_t hist_all[];
  const int lane = threadIdx.x & 63, l = lane & (L - 1), sub = lane / L;
  constexpr int kSide = 64 / L, kAhead = ahead<L>();   // tokens side by side
  int32_t* hist = hist_all + (threadIdx.x >> 6) * a.E;
  const int64_t c = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t t0 = c * a.run, t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  if (t0 >= t1) return;
  for (int64_t s = sequence_of(a, t0, lane); s < a.S; ++s) {
    int64_t lo = border(a, s), hi = border(a, s + 1);
    if (lo >= t1) break;
    lo = lo > t0 ? lo : t0;
    hi = hi < t1 ? hi : t1;
    if (lo >= hi) continue;
    for (int e = lane; e < a.E; e += 64) hist[e] = 0;
    float acc[NV], z = 0.f;
    int count = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.f;
    for (int64_t t = lo; t < hi; t += kSide * kAhead) {
      Row<L, NV, QUADS> row[kAhead];
      bool in[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t mine = t + k * kSide + sub, at = mine < hi ? mine : hi - 1;
        in[k] = mine < hi && (a.mask == nullptr || a.mask[at] != 0);
        row[k].load(a.logits + at * a.ld, a.E, l);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float lse = 0.f, r = 1.f;
        Row<L, NV, QUADS> p = row[k];
        if (a.sigmoid) {
          r = p.sigmoids(a.E, l);
          if (a.want_z) lse = row[k].softmax();
        } else {
          lse = p.softmax();
        }
        count += in[k];
        if (a.want_z) z += in[k] ? lse * lse : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] += in[k] ? p.v[i] * r : 0.f;
      }
    }
    const uint32_t n = uint32_t(hi - lo) * uint32_t(a.K);   // of one run: T / 4096 tokens of K <= 1024
    for (uint32_t i = lane; i < n; i += 64) {
      const int64_t at = lo * a.K + i;
      const int64_t e = a.idx_i64 ? static_cast<const int64_t*>(a.idx)[at] : int64_t(static_cast<const int32_t*>(a.idx)[at]);
      if (e >= 0 && e < a.E && (a.mask == nullptr || a.mask[lo + i / uint32_t(a.K)] != 0)) atomicAdd(&hist[e], 1);
    }
    __builtin_amdgcn_wave_barrier();
    // the tokens side by side, in a fixed order
#pragma unroll
    for (int off = L; off < 64; off <<= 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] += __shfl_xor(acc[i], off);
      z += __shfl_xor(z, off);
      count += __shfl_xor(count, off);
    }
    const int64_t place = c + s;
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = Row<L, NV, QUADS>::column(l, i);
        if (e < a.E) st_global(a.sums + place * a.E + e, acc[i]);
      }
    }
    if (lane == 0) {
      st_global(reinterpret_cast<uint32_t*>(a.tokens) + place, uint32_t(count));
      st_global(a.z + place, z);
    }
    for (int e = lane; e < a.E; e += 64) st_global(reinterpret_cast<uint32_t*>(a.slots) + place * a.E + e, uint32_t(hist[e]));
    __builtin_amdgcn_wave_barrier();
  }
}

struct FoldArgs {
  BalanceArgs b;
  float* f;             // [S, E]: E cnt / n^2
  int32_t* counts;      // [S, E]
  int32_t* seq_tokens;  // [S]
  float* seq_z;         // [S]
  float* loss_part;     // [workgroups of the fold]
};

// Sum of v over a workgroup of up to 1024 threads, in a fixed order; valid in thread 0.
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < int(blockDim.x >> 6); ++i) s += lds[i];
  __syncthreads();
  return s;
}

// A sequence's places, one after the other: first and how many (0 for an empty sequence).
__device__ __forceinline__ void places_of(const BalanceArgs& b, int64_t s, int64_t& first, int64_t& n) {
  const int64_t lo = border(b, s), hi = border(b, s + 1);
  first = lo / b.run + s;
  n = hi > lo ? (hi - 1) / b.run - lo / b.run + 1 : 0;
}

// Workgroup (column group, sequence): 16 columns, blockDim / 16 rows of threads that each add every so many places, then each other.
__global__ __launch_bounds__(1024) void balance_fold_kernel(FoldArgs a) {
  __shared__ float sum[64][16];
  __shared__ int32_t cnt[64][16];
  __shared__ int32_t tok[64];
  __shared__ float lds[16];
  const int64_t s = blockIdx.y;
  const int q = threadIdx.x & 15, g = threadIdx.x >> 4, groups = int(blockDim.x >> 4);
  const int e = int(blockIdx.x) * 16 + q;
  int64_t first, n;
  places_of(a.b, s, first, n);
  float p = 0.f;
  int32_t m = 0, t = 0;
  float z = 0.f;
  for (int64_t i = g; i < n; i += groups) {
    const int64_t at = first + i;
    if (e < a.b.E) {
      p += a.b.sums[at * a.b.E + e];
      m += a.b.slots[at * a.b.E + e];
    }
    if (q == 0) {
      t += a.b.tokens[at];
      z += a.b.z[at];
    }
  }
  sum[g][q] = p;
  cnt[g][q] = m;
  if (q == 0) tok[g] = t;
  const float zsum = block_sum(z, lds);   // (a barrier for the others too)
  float part = 0.f;
  if (threadIdx.x < 16) {
    p = 0.f;
    m = t = 0;
    for (int i = 0; i < groups; ++i) {
      p += sum[i][q];
      m += cnt[i][q];
      t += tok[i];
    }
    if (e < a.b.E) {
      const float inv = t > 0 ? 1.f / float(t) : 0.f;
      const float f = float(a.b.E) * float(m) * inv;
      st_global(a.f + s * a.b.E + e, f * inv);
      st_global(reinterpret_cast<uint32_t*>(a.counts) + s * a.b.E + e, uint32_t(m));
      part = f * (p * inv);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      st_global(reinterpret_cast<uint32_t*>(a.seq_tokens) + s, uint32_t(t));
      st_global(a.seq_z + s, zsum);
    }
  }
  const float total = block_sum(part, lds);
  if (threadIdx.x == 0) st_global(a.loss_part + s * gridDim.x + blockIdx.x, total);
}

// Sequences of a few places: one thread to a sequence's column.
__global__ __launch_bounds__(256) void balance_fold_short_kernel(FoldArgs a) {
  __shared__ float lds[4];
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  float part = 0.f;
  if (i < a.b.S * a.b.E) {
    const int64_t s = i / a.b.E, e = i - s * a.b.E;
    int64_t first, n;
    places_of(a.b, s, first, n);
    float p = 0.f, z = 0.f;
    int32_t m = 0, t = 0;
    for (int64_t k = first; k < first + n; ++k) {
      p += a.b.sums[k * a.b.E + e];
      m += a.b.slots[k * a.b.E + e];
      t += a.b.tokens[k];
      if (e == 0) z += a.b.z[k];
    }
    const float inv = t > 0 ? 1.f / float(t) : 0.f;
    const float f = float(a.b.E) * float(m) * inv;
    st_global(a.f + i, f * inv);
    st_global(reinterpret_cast<uint32_t*>(a.counts) + i, uint32_t(m));
    part = f * (p * inv);
    if (e == 0) {
      st_global(reinterpret_cast<uint32_t*>(a.seq_tokens) + s, uint32_t(t));
      st_global(a.seq_z + s, z);
    }
  }
  const float total = block_sum(part, lds);
  if (threadIdx.x == 0) st_global(a.loss_part + blockIdx.x, total);
}

// loss, and {1 / S', 1 / N} for the backward; the running totals of a load tracker.
struct FinishArgs {
  const float* loss_part;
  int64_t parts, S;
  const int32_t* seq_tokens;
  const float* seq_z;
  float z_mult;
  float* loss;
  float* inverse;        // [2]
  int64_t* acc_total;    // [1] or null
};

__global__ __launch_bounds__(1024) void balance_finish_kernel(FinishArgs a) {
  __shared__ float lds[16];
  __shared__ int64_t ilds[16];
  float loss = 0.f, z = 0.f, filled = 0.f;
  int64_t n = 0;
  for (int64_t i = threadIdx.x; i < a.parts; i += 1024) loss += a.loss_part[i];
  for (int64_t i = threadIdx.x; i < a.S; i += 1024) {
    const int32_t t = a.seq_tokens[i];
    n += t;
    filled += t > 0 ? 1.f : 0.f;
    z += a.seq_z[i];
  }
  loss = block_sum(loss, lds);
  z = block_sum(z, lds);
  filled = block_sum(filled, lds);   // whole numbers below 2^24
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off);
  if ((threadIdx.x & 63) == 0) ilds[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x != 0) return;
  n = 0;
  for (int i = 0; i < 16; ++i) n += ilds[i];
  const float inv_s = filled > 0.f ? 1.f / filled : 0.f, inv_n = n > 0 ? 1.f / float(n) : 0.f;
  st_global(a.loss, loss * inv_s + a.z_mult * (z * inv_n));
  st_global(a.inverse, inv_s);
  st_global(a.inverse + 1, inv_n);
  if (a.acc_total) *FM_GLOBAL(int64_t, a.acc_total) = a.acc_total[0] + n;
}

// acc[e] += sum of the sequences' counts: one workgroup to an expert
__global__ __launch_bounds__(256) void balance_track_kernel(const int32_t* counts, int64_t S, int E, int64_t* acc) {
  __shared__ int64_t lds[4];
  int64_t n = 0;
  for (int64_t s = threadIdx.x; s < S; s += 256) n += counts[s * E + blockIdx.x];
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) *FM_GLOBAL(int64_t, acc + blockIdx.x) = acc[blockIdx.x] + ((lds[0] + lds[1]) + (lds[2] + lds[3]));
}

struct BalanceBwdArgs {
  BalanceArgs b;
  const float* f;        // [S, E]
  const float* inverse;  // [2]
  const float* dloss;    // scalar
  float z_mult;
  float* dlogits;
  int64_t ld_d;
  int add;               // dlogits += rather than =
};

template <int L, int NV, bool QUADS>
__device__ __forceinline__ void put(const BalanceBwdArgs& a, int64_t t, int l, float (&g)[NV]) {
  float* p = a.dlogits + t * a.ld_d;
  using R = Row<L, NV, QUADS>;
  if constexpr (QUADS) {
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      const int c = R::column(l, i);
      if (c >= a.b.E) continue;
      f32x4_el q = {g[i], g[i + 1], g[i + 2], g[i + 3]};
      if (a.add) q += *reinterpret_cast<const f32x4_el*>(p + c);
      *FM_GLOBAL(f32x4_el, reinterpret_cast<f32x4_el*>(p + c)) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = R::column(l, i);
      if (c < a.b.E) st_global(p + c, a.add ? p[c] + g[i] : g[i]);
    }
  }
}

template <int L, int NV, bool QUADS>
__global__ __launch_bounds__(256) void balance_backward_kernel(BalanceBwdArgs a) {
  const BalanceArgs& b = a.b;
  const int lane = threadIdx.x & 63, l = lane & (L - 1), sub = lane / L;
  constexpr int kSide = 64 / L, kAhead = ahead<L>();
  const int64_t c = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t t0 = c * b.run, t1 = t0 + b.run < b.T ? t0 + b.run : b.T;
  if (t0 >= t1) return;
  const float g = a.dloss[0] * a.inverse[0];
  const float gz = 2.f * a.z_mult * (a.dloss[0] * a.inverse[1]);
  float zero[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) zero[i] = 0.f;
  int64_t done = t0;   // tokens before it are written
  auto skip_to = [&](int64_t end) {   // tokens of no sequence
    if (!a.add)
      for (int64_t t = done + sub; t < end; t += kSide) put<L, NV, QUADS>(a, t, l, zero);
    done = end;
  };
  for (int64_t s = sequence_of(b, t0, lane); s < b.S; ++s) {
    int64_t lo = border(b, s), hi = border(b, s + 1);
    if (lo >= t1) break;
    lo = lo > done ? lo : done;
    hi = hi < t1 ? hi : t1;
    if (lo >= hi) continue;
    skip_to(lo);
    float f[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = Row<L, NV, QUADS>::column(l, i);
      f[i] = e < b.E ? g * a.f[s * b.E + e] : 0.f;
    }
    for (int64_t t = lo; t < hi; t += kSide * kAhead) {
      Row<L, NV, QUADS> row[kAhead];
      bool in[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t mine = t + k * kSide + sub, at = mine < hi ? mine : hi - 1;
        in[k] = b.mask == nullptr || b.mask[at] != 0;
        row[k].load(b.logits + at * b.ld, b.E, l);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t mine = t + k * kSide + sub;
        Row<L, NV, QUADS> p = row[k];
        float out[NV], inner = 0.f;
        if (b.sigmoid) {
          const float r = p.sigmoids(b.E, l);
#pragma unroll
          for (int i = 0; i < NV; ++i) inner = fmaf(f[i], p.v[i], inner);
          inner = group_sum<L>(inner) * r;
#pragma unroll
          for (int i = 0; i < NV; ++i) out[i] = (f[i] - inner) * r * (p.v[i] * (1.f - p.v[i]));
          if (gz != 0.f) {
            const float lse = row[k].softmax();
#pragma unroll
            for (int i = 0; i < NV; ++i) out[i] = fmaf(gz * lse, row[k].v[i], out[i]);
          }
        } else {
          const float lse = p.softmax();
#pragma unroll
          for (int i = 0; i < NV; ++i) inner = fmaf(f[i], p.v[i], inner);
          inner = group_sum<L>(inner) - gz * lse;
#pragma unroll
          for (int i = 0; i < NV; ++i) out[i] = p.v[i] * (f[i] - inner);
        }
        if (mine < hi) put<L, NV, QUADS>(a, mine, l, in[k] ? out : zero);
      }
    }
    done = hi;
  }
  skip_to(t1);
}

// -------------------------------------------------------------------- launches ----
// go(lanes to a token, values to a lane, quads)
template <typename F>
void for_experts(int E, F go) {
#define FM_ROW(l, n, q) go(std::integral_constant<int, l>{}, std::integral_constant<int, n>{}, std::integral_constant<bool, q>{})
  if (E % 4 == 0) {
    if (E <= 4) FM_ROW(1, 4, true);
    else if (E <= 8) FM_ROW(2, 4, true);
    else if (E <= 16) FM_ROW(4, 4, true);
    else if (E <= 32) FM_ROW(8, 4, true);
    else if (E <= 64) FM_ROW(16, 4, true);
    else if (E <= 128) FM_ROW(32, 4, true);
    else if (E <= 256) FM_ROW(64, 4, true);
    else if (E <= 512) FM_ROW(64, 8, true);
    else FM_ROW(64, 16, true);
  } else {
    if (E <= 4) FM_ROW(4, 1, false);
    else if (E <= 16) FM_ROW(16, 1, false);
    else if (E <= 64) FM_ROW(64, 1, false);
    else if (E <= 256) FM_ROW(64, 4, false);
    else FM_ROW(64, 16, false);
  }
#undef FM_ROW
}

// Tokens of a wave: 32 at least (a place of the workspace is 8 E bytes beside the 4 E of a token's logits), and no more waves than
// sixteen to a CU of 256.
int run_of(int64_t T) {
  const int64_t r = (T + 4095) / 4096;
  return int(r < 32 ? 32 : r);
}

struct Space {
  int64_t places, sums, slots, tokens, z, seq_tokens, seq_z, loss_part, bytes;   // offsets in bytes
};
Space space_of(int64_t T, int E, int64_t S) {
  Space w{};
  w.bytes = 256;   // never none: no tokens and no sequences are a call too
  w.places = (T + run_of(T) - 1) / run_of(T) + S;
  auto take = [&](int64_t n) {
    const int64_t at = w.bytes;
    w.bytes += (n * 4 + 255) / 256 * 256;
    return at;
  };
  w.sums = take(w.places * E);
  w.slots = take(w.places * E);
  w.tokens = take(w.places);
  w.z = take(w.places);
  w.seq_tokens = take(S);
  w.seq_z = take(S);
  w.loss_part = take((S * E + 255) / 256 + S * ((E + 15) / 16));
  return w;
}

int check_balance(const BalanceArgs& a, const char* what) {
  FM_REQUIRE(a.T >= 0 && a.T < (int64_t(1) << 31), "%s: T must be below 2^31", what);
  FM_REQUIRE(a.E >= 1 && a.E <= kMaxExperts, "%s: E must be 1 to %d (got %d)", what, kMaxExperts, a.E);
  FM_REQUIRE(a.S >= 0 && a.S < (int64_t(1) << 24), "%s: fewer than 2^24 sequences", what);
  FM_REQUIRE(a.cu || a.S == 1, "%s: without borders there is one sequence", what);
  FM_REQUIRE(a.T == 0 || (a.logits && a.ld >= a.E), "%s: null logits or a pitch below E", what);
  return 0;
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" {

int64_t fm_balance_workspace_bytes(int64_t T, int E, int64_t S) {
  return T < 0 || E < 1 || E > kMaxExperts || S < 0 ? 0 : space_of(T, E, S).bytes;
}

int fm_balance_forward(const float* logits, int64_t ld, int64_t T, int E, const void* indices, int indices_i64, int K, const int32_t* cu,
                       int64_t S, const uint8_t* mask, int sigmoid, float z_mult, float* f, int32_t* counts, float* inverse, float* loss,
                       int64_t* acc, int64_t* acc_total, void* workspace, int64_t workspace_bytes, void* stream) {
  char* ws = static_cast<char*>(workspace);
  BalanceArgs b{logits, ld, T, E, K, indices, indices_i64, cu, S, mask, sigmoid, z_mult != 0.f, run_of(T), nullptr, nullptr, nullptr, nullptr};
  if (int rc = check_balance(b, "fm_balance_forward")) return rc;
  FM_REQUIRE(K >= 1 && K <= 1024 && (T == 0 || indices), "fm_balance_forward: null indices or bad K");
  FM_REQUIRE(inverse && loss && (S == 0 || (f && counts)), "fm_balance_forward: null output");
  const Space w = space_of(T, E, S);
  FM_REQUIRE(ws && aligned16(ws) && workspace_bytes >= w.bytes, "fm_balance_forward: the workspace must hold fm_balance_workspace_bytes(T, E, S) "
             "bytes on 16");
  b.sums = reinterpret_cast<float*>(ws + w.sums);
  b.slots = reinterpret_cast<int32_t*>(ws + w.slots);
  b.tokens = reinterpret_cast<int32_t*>(ws + w.tokens);
  b.z = reinterpret_cast<float*>(ws + w.z);
  const FoldArgs fold{b, f, counts, reinterpret_cast<int32_t*>(ws + w.seq_tokens), reinterpret_cast<float*>(ws + w.seq_z),
                      reinterpret_cast<float*>(ws + w.loss_part)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t runs = (T + b.run - 1) / b.run;
  if (runs > 0 && S > 0)
    for_experts(E, [&](auto l, auto n, auto q) {
      hipLaunchKernelGGL((balance_sums_kernel<decltype(l)::value, decltype(n)::value, decltype(q)::value>), dim3(unsigned((runs + 3) / 4)),
                         dim3(256), unsigned(4 * E * sizeof(int32_t)), s, b);
    });
  int64_t parts = 0;
  if (S > 0) {
    // sequences of eight places or fewer on average: a thread to a column; of many, a workgroup of 1024
    if (w.places <= 8 * S || S > 65535) {
      parts = (S * E + 255) / 256;
      hipLaunchKernelGGL(balance_fold_short_kernel, dim3(unsigned(parts)), dim3(256), 0, s, fold);
    } else {
      const unsigned groups = unsigned((E + 15) / 16);
      parts = S * groups;
      hipLaunchKernelGGL(balance_fold_kernel, dim3(groups, unsigned(S)), dim3(w.places > 64 * S ? 1024 : 256), 0, s, fold);
    }
  }
  const FinishArgs fin{fold.loss_part, parts, S, fold.seq_tokens, fold.seq_z, z_mult, loss, inverse, acc_total};
  hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, s, fin);
  if (acc && S > 0) hipLaunchKernelGGL(balance_track_kernel, dim3(unsigned(E)), dim3(256), 0, s, counts, S, E, acc);
  return check_launch("fm_balance_forward");
}

int fm_balance_backward(const float* logits, int64_t ld, int64_t T, int E, const int32_t* cu, int64_t S, const uint8_t* mask, int sigmoid,
                        float z_mult, const float* f, const float* inverse, const float* dloss, float* dlogits, int64_t ld_d, int add,
                        void* stream) {
  const BalanceArgs b{logits, ld, T, E, 1, nullptr, 0, cu, S, mask, sigmoid, z_mult != 0.f, run_of(T), nullptr, nullptr, nullptr, nullptr};
  if (int rc = check_balance(b, "fm_balance_backward")) return rc;
  if (T == 0) return 0;
  FM_REQUIRE(inverse && dloss && dlogits && ld_d >= E && (S == 0 || f), "fm_balance_backward: null pointer or a pitch below E");
  const BalanceBwdArgs a{b, f, inverse, dloss, z_mult, dlogits, ld_d, add};
  const int64_t runs = (T + b.run - 1) / b.run;
  for_experts(E, [&](auto l, auto n, auto q) {
    hipLaunchKernelGGL((balance_backward_kernel<decltype(l)::value, decltype(n)::value, decltype(q)::value>), dim3(unsigned((runs + 3) / 4)),
                       dim3(256), 0, static_cast<hipStream_t>(stream), a);
  });
  return check_launch("fm_balance_backward");
}

}  // extern "C"
