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
// Forward: one pass over the logits and indices.  The batch is cut at sequence borders and into runs of tokens; run c and
// sequence s meet at most once, and runs and sequences both ascend, so the number c + s names each piece, and a piece finds its
// run and sequence from its number by a search of the borders.  A piece is the work of a wave, or of four or sixteen where sequences are
// long: a token's logits sit in L lanes (64 / L tokens side by side) whose column sums stay in registers, the slots are counted in
// LDS, and both go to the piece's place in the workspace.  A second launch adds each sequence's places in order (no float
// atomics: the same bits each time) and leaves E cnt / n^2 for the backward, a third adds the sequences; few tokens take one launch
// for all of it.  Backward: the same pieces, logits in, gradient out; the tokens before the first border and behind the last
// are two sequences more, of zeros.
#include <type_traits>

#include "fm_lanes.h"
#include "../../include/fm_hip.h"

namespace fm {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int64_t kMaxSequences = int64_t(1) << 20;   // 64 column groups of a wave each stay below 2^32 threads
constexpr float kSumFloor = 1e-8f;

typedef float f32x4_el __attribute__((ext_vector_type(4), aligned(4)));

// e^d for -110 <= d <= 0: 2^(d log2 e) by the hardware, with the product's rounding error as a factor (without it an ulp more for each
// 2^k <= |d|).
__device__ __forceinline__ float exp_below(float d) {
#pragma clang fp contract(off)
  constexpr float kL = 1.44269502162933349609375f, kLn2 = 0.693147180559945f;
  const float h = d * kL;
  const float e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, fmaf(d, kL, -h) * kLn2, e);
}

// 1 / d of a normal d to about an ulp.
__device__ __forceinline__ float reciprocal(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  return fmaf(fmaf(-d, r, 1.f), r, r);
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
  int run;                 // tokens of a piece at most
  int64_t places;          // pieces
  float* sums;             // [places, E]
  int32_t* slots;          // [places, E]
  int32_t* tokens;         // [places]
  float* z;                // [places]
};

// Start of sequence a - 1: a = 0 is the rest before the first border, a = S + 1 the rest behind the last.
__device__ __forceinline__ int64_t border(const BalanceArgs& b, int64_t a) {
  if (a <= 0) return 0;
  if (a > b.S + 1) return b.T;
  if (b.cu == nullptr) return a == 1 ? 0 : b.T;
  const int64_t t = b.cu[a - 1];
  return t < 0 ? 0 : (t > b.T ? b.T : t);
}

// Piece p: sequence a - 1 and its tokens [lo, hi) of run p - a.  a is the largest with border(a) + a run < (p + 1) run: a sequence that meets
// run p - a starts before the run's end, and the next one does not.  64 candidates a round; in the last they are
// neighbours, which hold lo and hi.
struct Piece {
  int64_t a, lo, hi;
};
__device__ __forceinline__ Piece piece_of(const BalanceArgs& b, int64_t p, int lane) {
  int64_t a = 0, lo, hi;
  if (b.cu == nullptr) {
    a = 1;
    lo = 0;
    hi = b.T;
  } else {
    const int64_t end = (p + 1) * b.run;
    int64_t n = b.S + 2;   // a is in [a, a + n)
    while (n > 63) {
      const int64_t step = (n + 63) / 64, at = a + lane * step;
      const uint64_t m = __ballot(lane * step < n && border(b, at) + at * b.run < end);
      const int64_t k = m == 0 ? 0 : 63 - __builtin_clzll(m);
      a += k * step;
      n = n - k * step < step ? n - k * step : step;
    }
    const int64_t t = border(b, a + lane);
    const uint64_t m = __ballot(lane < n && t + (a + lane) * b.run < end);
    const int k = m == 0 ? 0 : 63 - __builtin_clzll(m);
    a += k;
    lo = __builtin_amdgcn_readlane(int(t), k);
    hi = __builtin_amdgcn_readlane(int(t), k + 1);
  }
  const int64_t c0 = (p - a) * b.run, c1 = c0 + b.run;
  lo = lo > c0 ? lo : c0;
  hi = hi < c1 ? hi : c1;
  return Piece{a, lo, c0 < 0 ? lo : hi};
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
  // Columns behind the last expert hold -infinity: exponentials and sigmoids of 0.
  // softmax in place; the log of the sum of exponentials, where wanted
  // A NaN, or a largest logit of +-infinity, makes the factor NaN: the bound below would hide the NaN's own exponential.
  __device__ __forceinline__ float softmax(bool want_log) {
    float m = v[0], s = 0.f;
#pragma unroll
    for (int i = 1; i < NV; ++i) m = __builtin_elementwise_maximum(m, v[i]);
    m = group_fold<L>(m, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = exp_below(fmaxf(v[i] - m, -110.f));
      s += v[i];
    }
    s = group_sum<L>(s);
    const float r = fmaf(m, 0.f, reciprocal(s));
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] *= r;
    return want_log ? m + logf(s) : 0.f;
  }
  // sigmoids in place: 1 or e^-|l| over 1 + e^-|l| (half an ulp of l's exponent and two more of the sigmoid); 1 / (their sum + floor)
  __device__ __forceinline__ float sigmoids() {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float e = __builtin_amdgcn_exp2f(-fabsf(v[i]) * 1.44269502162933349609375f);
      v[i] = (v[i] < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
      s += v[i];
    }
    return reciprocal(group_sum<L>(s) + kSumFloor);
  }
};

// Steps whose loads are in flight at once: four, as long as they stay within the shortest run; two of eight values side by side.
template <int L, int NV>
constexpr int ahead() {
  return 16 * L / 64 >= 4 ? (NV > 4 && L < 64 ? 2 : 4) : (16 * L / 64 >= 2 ? 2 : 1);
}

// Piece p's sums and counts, by one wave (its own hist) or a workgroup of TEAM (one hist; sums and small hold a row for each wave).
template <int L, int NV, bool QUADS, int TEAM>
__device__ __forceinline__ void sum_piece(const BalanceArgs& a, int64_t p, int32_t* hist, float* sums, float (*small)[2]) {
  using R = Row<L, NV, QUADS>;
  constexpr int kSide = 64 / L, kAhead = ahead<L, NV>();   // tokens side by side
  const int lane = threadIdx.x & 63, l = lane & (L - 1), sub = lane / L;
  const int wave = TEAM == 1 ? 0 : threadIdx.x >> 6, me = TEAM == 1 ? lane : threadIdx.x;
  const Piece piece = piece_of(a, p, lane);
  const int64_t lo = piece.lo, hi = piece.hi;
  if (piece.a < 1 || piece.a > a.S || lo >= hi) return;
  auto team_sync = [] {
    if constexpr (TEAM > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
  };
  // the first indices come in beside the logits
  const uint32_t n = uint32_t(hi - lo) * uint32_t(a.K);   // of one run: some hundred tokens of K <= 1024
  auto slot = [&](uint32_t i) {
    const int64_t at = lo * a.K + i;
    const int64_t e = a.idx_i64 ? static_cast<const int64_t*>(a.idx)[at] : int64_t(static_cast<const int32_t*>(a.idx)[at]);
    const bool counts = a.mask == nullptr || a.mask[lo + i / uint32_t(a.K)] != 0;
    return counts && e >= 0 && e < a.E ? int(e) : -1;
  };
  const uint32_t i0 = me, i1 = me + 64 * TEAM;
  const int e0 = i0 < n ? slot(i0) : -1, e1 = i1 < n ? slot(i1) : -1;
  for (int e = me; e < a.E; e += 64 * TEAM) hist[e] = 0;
  team_sync();
  float acc[NV], z = 0.f;
  int count = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  // the next steps' logits come in while these are summed
  R next[kAhead];
  bool use[kAhead];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t mine = t + k * TEAM * kSide + sub, at = mine < hi ? mine : hi - 1;
      use[k] = mine < hi && (a.mask == nullptr || a.mask[at] != 0);
      next[k].load(a.logits + at * a.ld, a.E, l);
    }
  };
  int64_t t = lo + wave * kSide;
  if (t < hi) fetch(t);
  while (t < hi) {
    R row[kAhead];
    bool in[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      row[k] = next[k];
      in[k] = use[k];
    }
    t += TEAM * kSide * kAhead;
    if (t < hi) fetch(t);
    if (a.mask) {   // what a mask leaves out may be a NaN; a row past the end is the last one again
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int i = 0; i < NV; ++i) row[k].v[i] = in[k] ? row[k].v[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float one = in[k] ? 1.f : 0.f;
      R p = row[k];
      count += in[k];
      if (a.sigmoid) {
        const float r = p.sigmoids() * one;
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = fmaf(p.v[i], r, acc[i]);
        if (a.want_z) {
          const float lse = row[k].softmax(true);
          z = fmaf(lse * one, lse, z);
        }
      } else {
        const float lse = p.softmax(a.want_z);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = fmaf(p.v[i], one, acc[i]);
        z = fmaf(lse * one, lse, z);
      }
    }
  }
  if (e0 >= 0) atomicAdd(&hist[e0], 1);
  if (e1 >= 0) atomicAdd(&hist[e1], 1);
  for (uint32_t i = me + 128 * TEAM; i < n; i += 64 * TEAM) {
    const int e = slot(i);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  // the tokens side by side, in a fixed order
#pragma unroll
  for (int off = L; off < 64; off <<= 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] += __shfl_xor(acc[i], off);
    z += __shfl_xor(z, off);
    count += __shfl_xor(count, off);
  }
  if constexpr (TEAM == 1) {
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = R::column(l, i);
        if (e < a.E) st_global(a.sums + p * a.E + e, acc[i]);
      }
    }
    if (lane == 0) {
      st_global(reinterpret_cast<uint32_t*>(a.tokens) + p, uint32_t(count));
      st_global(a.z + p, z);
    }
    team_sync();
  } else {
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = R::column(l, i);
        if (e < a.E) sums[wave * a.E + e] = acc[i];
      }
    }
    if (lane == 0) {
      small[wave][0] = float(count);
      small[wave][1] = z;
    }
    team_sync();
    for (int e = me; e < a.E; e += 64 * TEAM) {
      float v = sums[e];
#pragma unroll
      for (int w = 1; w < TEAM; ++w) v += sums[w * a.E + e];
      st_global(a.sums + p * a.E + e, v);
    }
    if (me == 0) {
      float c = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) {
        c += small[w][0];
        v += small[w][1];
      }
      st_global(reinterpret_cast<uint32_t*>(a.tokens) + p, uint32_t(c));   // whole numbers of a run
      st_global(a.z + p, v);
    }
  }
  for (int e = me; e < a.E; e += 64 * TEAM) st_global(reinterpret_cast<uint32_t*>(a.slots) + p * a.E + e, uint32_t(hist[e]));
}

template <int L, int NV, bool QUADS, int TEAM>
__global__ __launch_bounds__(TEAM == 16 ? 1024 : 256) void balance_sums_kernel(BalanceArgs a) {
  extern __shared__ int32_t lds[];   // TEAM 1: four hists; else one, and the waves' sums
  __shared__ float small[TEAM][2];
  const int64_t p = TEAM == 1 ? int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6) : int64_t(blockIdx.x);
  if (p >= a.places) return;
  sum_piece<L, NV, QUADS, TEAM>(a, p, TEAM == 1 ? lds + (threadIdx.x >> 6) * a.E : lds, reinterpret_cast<float*>(lds + a.E), small);
}

// A workgroup's share of the loss: sum_e f P of its columns; its sequences' tokens, how many of them have any, and their z
// (with the first columns alone).
struct alignas(16) Share {
  float loss, z;
  int32_t tokens, filled;   // below T < 2^31 in any sum
};

struct FoldArgs {
  BalanceArgs b;
  float* f;             // [S, E]: E cnt / n^2
  int32_t* counts;      // [S, E]
  Share* shares;        // [workgroups of the fold]
};

// The sum over a workgroup's threads, in a fixed order; valid in thread 0.
__device__ __forceinline__ Share block_sum(Share v) {
  __shared__ Share waves[16];
  v.loss = group_sum<64>(v.loss);
  v.z = group_sum<64>(v.z);
  for (int off = 32; off > 0; off >>= 1) {
    v.tokens += __shfl_xor(v.tokens, off);
    v.filled += __shfl_xor(v.filled, off);
  }
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < int(blockDim.x >> 6); ++i) {
      v.loss += waves[i].loss;
      v.z += waves[i].z;
      v.tokens += waves[i].tokens;
      v.filled += waves[i].filled;
    }
  }
  return v;
}

// loss, and {1 / S', 1 / N} for the backward; the running totals of a load tracker.
struct FinishArgs {
  const Share* shares;
  int64_t parts;
  float z_mult;
  float* loss;
  float* inverse;        // [2]
  int64_t* acc_total;    // [1] or null
};

// By one workgroup, from each thread's share of the sums.
__device__ __forceinline__ void finish(const FinishArgs& a, Share v) {
  v = block_sum(v);
  if (threadIdx.x != 0) return;
  const float inv_s = v.filled > 0 ? 1.f / float(v.filled) : 0.f, inv_n = v.tokens > 0 ? 1.f / float(v.tokens) : 0.f;
  st_global(a.loss, v.loss * inv_s + a.z_mult * (v.z * inv_n));
  st_global(a.inverse, inv_s);
  st_global(a.inverse + 1, inv_n);
  if (a.acc_total) *FM_GLOBAL(int64_t, a.acc_total) = a.acc_total[0] + v.tokens;
}

__global__ __launch_bounds__(1024) void balance_finish_kernel(FinishArgs a) {
  Share v{0.f, 0.f, 0, 0};
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < a.parts; i += 1024) {
    const Share s = a.shares[i];
    v.loss += s.loss;
    v.z += s.z;
    v.tokens += s.tokens;
    v.filled += s.filled;
  }
  finish(a, v);
}

// A sequence's places, one after the other: first and how many (0 for an empty sequence).
__device__ __forceinline__ void places_of(const BalanceArgs& b, int64_t s, int64_t& first, int64_t& n) {
  const int64_t lo = border(b, s + 1), hi = border(b, s + 2);
  first = lo / b.run + s + 1;
  n = hi > lo ? (hi - 1) / b.run - lo / b.run + 1 : 0;
}

// What a sequence's places add up to, of one column.
struct Column {
  float p, z;
  int32_t slots, tokens;
  // places first + g, first + g + step, ..: the loads of U places at once
  template <int U>
  __device__ __forceinline__ void add(const BalanceArgs& b, int64_t first, int64_t n, int g, int step, int col) {
    for (int64_t k = g; k < n; k += U * step) {
      float pk[U] = {}, zk[U] = {};
      int32_t mk[U] = {}, tk[U] = {};
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (k + i * step >= n) continue;
        const int64_t at = first + k + i * step;
        pk[i] = b.sums[at * b.E + col];
        mk[i] = b.slots[at * b.E + col];
        tk[i] = b.tokens[at];
        zk[i] = b.z[at];
      }
#pragma unroll
      for (int i = 0; i < U; ++i) add(Column{pk[i], zk[i], mk[i], tk[i]});
    }
  }
  __device__ __forceinline__ void add(const Column& c) {
    p += c.p;
    z += c.z;
    slots += c.slots;
    tokens += c.tokens;
  }
  // the sum over lanes `from`, 2 from, .. below `to` apart
  __device__ __forceinline__ void join(int from, int to) {
    for (int off = from; off < to; off <<= 1) add(Column{__shfl_xor(p, off), __shfl_xor(z, off), __shfl_xor(slots, off), __shfl_xor(tokens, off)});
  }
  // writes f and the count; this column's share of the loss
  __device__ __forceinline__ float write(const FoldArgs& a, int64_t at) const {
    const float inv = tokens > 0 ? 1.f / float(tokens) : 0.f;
    const float f = float(a.b.E) * float(slots) * inv;
    st_global(a.f + at, f * inv);
    st_global(reinterpret_cast<uint32_t*>(a.counts) + at, uint32_t(slots));
    return f * (p * inv);
  }
};

// C columns of each of 1024 / (C ROWS) sequences to a workgroup: a sequence's ROWS rows of threads (of one wave, or of all sixteen) add every
// so many places, then the rows' sums meet in order.  Sequences of more than LONG places, which would hold their rows up, are the whole
// workgroup's, one after the other.  The only workgroup finishes the loss too.
template <int C, int ROWS, int LONG>
__global__ __launch_bounds__(1024, ROWS == 1 ? 8 : 4) void balance_fold_kernel(FoldArgs a, int parts, FinishArgs fin) {
  constexpr int kSeqs = 1024 / (C * ROWS), kAtOnce = ROWS == 1 ? 2 : 4;
  __shared__ Column waves[16][C];
  __shared__ bool many[kSeqs];
  const int64_t block = blockIdx.x / uint32_t(parts);
  const int q = threadIdx.x & (C - 1), row = (threadIdx.x / C) & (ROWS - 1), mine = threadIdx.x / (C * ROWS);
  const int e = int(blockIdx.x - block * parts) * C + q, col = e < a.b.E ? e : a.b.E - 1;
  const int64_t s = block * kSeqs + mine;
  int64_t first = 0, n = 0;
  if (s < a.b.S) places_of(a.b, s, first, n);
  Share v{0.f, 0.f, 0, 0};
  auto done = [&](const Column& c, int64_t seq) {
    if (e < a.b.E) v.loss += c.write(a, seq * a.b.E + e);
    if (e == 0) {
      v.z += c.z;
      v.tokens += c.tokens;
      v.filled += c.tokens > 0;
    }
  };
  if (q == 0 && row == 0) many[mine] = n > LONG;
  Column c{0.f, 0.f, 0, 0};
  if (n <= LONG) c.add<kAtOnce>(a.b, first, n, row, ROWS, col);
  if constexpr (ROWS * C <= 64) c.join(C, C * ROWS);   // else there are none to add
  if (row == 0 && s < a.b.S && n <= LONG) done(c, s);
  if (__syncthreads_or(n > LONG)) {
    for (int i = 0; i < kSeqs; ++i) {
      if (!many[i]) continue;
      places_of(a.b, block * kSeqs + i, first, n);
      Column d{0.f, 0.f, 0, 0};
      d.add<kAtOnce>(a.b, first, n, threadIdx.x / C, 1024 / C, col);
      d.join(C, 64);
      if ((threadIdx.x & 63) < C) waves[threadIdx.x >> 6][q] = d;
      __syncthreads();
      if (threadIdx.x < C) {
        d = waves[0][q];
        for (int w = 1; w < 16; ++w) d.add(waves[w][q]);
        done(d, block * kSeqs + i);
      }
      __syncthreads();
    }
  }
  if (gridDim.x == 1) {
    finish(fin, v);
    return;
  }
  v = block_sum(v);
  if (threadIdx.x == 0) st_global(a.shares + blockIdx.x, make_uint4(f2u(v.loss), f2u(v.z), uint32_t(v.tokens), uint32_t(v.filled)));
}

// Few logits in few pieces: all of the forward in one workgroup, its sixteen waves taking the pieces in turn; the runs give each a piece at
// most, of one run or of four.  Against three launches, whose host's 5.8 us more hide up to that much of the device's time, us on the
// device: 512 tokens of 8 experts 6.9 and 7.1, 1024 7.0 and 8.4, 2048 9.2 and 8.5; 4096 of 4 9.2 and 8.8; 1000 of 7 13.3 and 7.6; beyond
// sixteen pieces 1700 of 7 19.5 and 8.6.  (Pieces of four runs at 512 < T: 576 of 8 in pieces of one 7.5, of four 6.6.)
constexpr int64_t kOnePieces = 32, kOneLogits = 16384, kOneColumns = 4096;
template <int L, int NV, bool QUADS>
__global__ __launch_bounds__(1024) void balance_one_kernel(FoldArgs a, FinishArgs fin) {
  extern __shared__ int32_t lds[];   // a hist for each wave
  for (int64_t p = threadIdx.x >> 6; p < a.b.places; p += blockDim.x >> 6)
    sum_piece<L, NV, QUADS, 1>(a.b, p, lds + (threadIdx.x >> 6) * a.b.E, nullptr, nullptr);
  __syncthreads();
  Share v{0.f, 0.f, 0, 0};
  for (int i = threadIdx.x; i < int(a.b.S) * a.b.E; i += blockDim.x) {
    const int s = i / a.b.E, e = i - s * a.b.E;
    Column c{0.f, 0.f, 0, 0};
    int64_t first, n;
    places_of(a.b, s, first, n);
    c.add<4>(a.b, first, n, 0, 1, e);
    v.loss += c.write(a, i);
    if (e == 0) {
      v.z += c.z;
      v.tokens += c.tokens;
      v.filled += c.tokens > 0;
    }
  }
  finish(fin, v);
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
  using R = Row<L, NV, QUADS>;
  const BalanceArgs& b = a.b;
  const int lane = threadIdx.x & 63, l = lane & (L - 1), sub = lane / L;
  constexpr int kSide = 64 / L, kAhead = ahead<L, NV>();
  const int64_t p = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (p >= b.places) return;
  const Piece piece = piece_of(b, p, lane);
  const int64_t lo = piece.lo, hi = piece.hi;
  if (lo >= hi) return;
  float zero[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) zero[i] = 0.f;
  if (piece.a < 1 || piece.a > b.S) {   // tokens of no sequence
    if (!a.add)
      for (int64_t t = lo + sub; t < hi; t += kSide) put<L, NV, QUADS>(a, t, l, zero);
    return;
  }
  const float g = a.dloss[0] * a.inverse[0];
  const float gz = 2.f * a.z_mult * (a.dloss[0] * a.inverse[1]);
  R f;
  f.load(a.f + (piece.a - 1) * b.E, b.E, l);
#pragma unroll
  for (int i = 0; i < NV; ++i) f.v[i] = R::column(l, i) < b.E ? g * f.v[i] : 0.f;
  R next[kAhead];
  bool use[kAhead];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t mine = t + k * kSide + sub, at = mine < hi ? mine : hi - 1;
      use[k] = b.mask == nullptr || b.mask[at] != 0;
      next[k].load(b.logits + at * b.ld, b.E, l);
    }
  };
  fetch(lo);
  for (int64_t t = lo; t < hi; t += kSide * kAhead) {
    R row[kAhead];
    bool in[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      row[k] = next[k];
      in[k] = use[k];
    }
    if (t + kSide * kAhead < hi) fetch(t + kSide * kAhead);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t mine = t + k * kSide + sub;
      R q = row[k];
      float out[NV], inner = 0.f;
      if (b.sigmoid) {
        const float r = q.sigmoids();
#pragma unroll
        for (int i = 0; i < NV; ++i) inner = fmaf(f.v[i], q.v[i], inner);
        inner = group_sum<L>(inner) * r;
#pragma unroll
        for (int i = 0; i < NV; ++i) out[i] = (f.v[i] - inner) * r * (q.v[i] * (1.f - q.v[i]));
        if (a.z_mult != 0.f) {
          const float lse = row[k].softmax(true);
#pragma unroll
          for (int i = 0; i < NV; ++i) out[i] = fmaf(gz * lse, row[k].v[i], out[i]);
        }
      } else {
        const float lse = q.softmax(a.z_mult != 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) inner = fmaf(f.v[i], q.v[i], inner);
        inner = group_sum<L>(inner);
        if (a.z_mult != 0.f) inner -= gz * lse;
#pragma unroll
        for (int i = 0; i < NV; ++i) out[i] = q.v[i] * (f.v[i] - inner);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) out[i] = in[k] ? out[i] : 0.f;
      if (mine < hi) put<L, NV, QUADS>(a, mine, l, out);
    }
  }
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
    else if (E <= 256) FM_ROW(32, 8, true);   // 65536 x 256: sums 19.3 us, backward 25.3; of (64, 4): 21 and 26.5
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

// Tokens side by side in a wave, as for_experts takes them.
int side_of(int E) {
  int side = 1;
  for_experts(E, [&](auto l, auto, auto) { side = 64 / decltype(l)::value; });
  return side;
}

// Tokens of a wave: 16 at least (or one step of what lies side by side), the more the longer the batch: no more than 4096 waves, sixteen
// to a CU.
int run_of(int64_t T, int E) {
  const int side = side_of(E), least = side < 16 ? 16 : side;
  const int64_t r = (T + 4095) / 4096;
  return int(r <= least ? least : (r + least - 1) / least * least);
}
// Waves to a piece: four where sequences have 64 tokens on average, sixteen from 1024 on; the fewer places to write and add.  One
// sequence of 65536 tokens, 256 experts: sums and fold 18.6 + 23.0 us of 4096 places, 17.0 + 6.7 of 256.
// (Sixteen waves' registers do not fit where a lane holds sixteen values of a row: beyond 512 experts, beyond 256 of no multiple of 4.
// 65536 x 511 of one sequence: 57 us the forward in pieces of four, 249 in pieces cut for sixteen and taken by one.)
constexpr int kTeamMaxValues = 8;   // of a lane, for sixteen waves
int team_of(int64_t T, int E, int64_t S) {
  if (T <= 16 * run_of(T, E) || T < 64 * S) return 1;
  int values = 0;
  for_experts(E, [&](auto, auto n, auto) { values = decltype(n)::value; });
  return T < 1024 * S || values > kTeamMaxValues ? 4 : 16;
}

struct Space {
  int64_t runs, places, sums, slots, tokens, z, shares, bytes;   // offsets in bytes
  int team, run;
  bool one;   // all of it in one launch, a wave to a piece
};
Space space_of(int64_t T, int E, int64_t S) {
  Space w{};
  w.bytes = 256;   // never none: no tokens and no sequences are a call too
  const int run = run_of(T, E);
  const int longer = T > 16 * run ? 4 : 1;   // runs to a piece of the one launch
  w.one = T <= 16 * longer * run && (T + longer * run - 1) / (longer * run) + S + 2 <= kOnePieces && T * E <= kOneLogits && E <= 256 &&
          S * E <= kOneColumns;
  w.team = w.one ? 1 : team_of(T, E, S);
  w.run = (w.one ? longer : w.team) * run;
  w.runs = (T + w.run - 1) / w.run;
  w.places = w.runs + S + 2;
  auto take = [&](int64_t n) {
    const int64_t at = w.bytes;
    w.bytes += (n * 4 + 255) / 256 * 256;
    return at;
  };
  w.sums = take(w.places * E);
  w.slots = take(w.places * E);
  w.tokens = take(w.places);
  w.z = take(w.places);
  w.shares = take(4 * S * ((E + 15) / 16));
  return w;
}

int check_balance(const BalanceArgs& a, const char* what) {
  FM_REQUIRE(a.T >= 0 && a.T < (int64_t(1) << 31), "%s: T must be below 2^31", what);
  FM_REQUIRE(a.E >= 1 && a.E <= kMaxExperts, "%s: E must be 1 to %d (got %d)", what, kMaxExperts, a.E);
  FM_REQUIRE(a.S >= 0 && a.S < kMaxSequences, "%s: fewer than 2^20 sequences", what);
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
  BalanceArgs b{logits, ld, T, E, K, indices, indices_i64, cu, S, mask, sigmoid, z_mult != 0.f, 0, 0, nullptr, nullptr, nullptr, nullptr};
  if (int rc = check_balance(b, "fm_balance_forward")) return rc;
  FM_REQUIRE(K >= 1 && K <= 1024 && (T == 0 || indices), "fm_balance_forward: null indices or bad K");
  FM_REQUIRE(inverse && loss && (S == 0 || (f && counts)), "fm_balance_forward: null output");
  FM_REQUIRE(T * K < (int64_t(1) << 31), "fm_balance_forward: fewer than 2^31 slots");
  const Space w = space_of(T, E, S);
  FM_REQUIRE(ws && aligned16(ws) && workspace_bytes >= w.bytes, "fm_balance_forward: the workspace must hold fm_balance_workspace_bytes(T, E, S) "
             "bytes on 16");
  b.run = w.run;
  b.places = w.places;
  b.sums = reinterpret_cast<float*>(ws + w.sums);
  b.slots = reinterpret_cast<int32_t*>(ws + w.slots);
  b.tokens = reinterpret_cast<int32_t*>(ws + w.tokens);
  b.z = reinterpret_cast<float*>(ws + w.z);
  const FoldArgs fold{b, f, counts, reinterpret_cast<Share*>(ws + w.shares)};
  FinishArgs fin{fold.shares, 0, z_mult, loss, inverse, acc_total};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (w.one) {
    const int64_t waves = w.places < 16 ? w.places : 16;
    for_experts(E, [&](auto l, auto n, auto q) {
      if constexpr (decltype(n)::value <= 8)
        hipLaunchKernelGGL((balance_one_kernel<decltype(l)::value, decltype(n)::value, decltype(q)::value>), dim3(1), dim3(unsigned(64 * waves)),
                           unsigned(waves * E * sizeof(int32_t)), s, fold, fin);
    });
  } else {
    // pieces are cut for w.team waves: another kernel's would leave waves idle
    bool fits = true;
    if (w.runs > 0 && S > 0)
      for_experts(E, [&](auto l, auto n, auto q) {
        constexpr int L = decltype(l)::value, N = decltype(n)::value;
        constexpr bool Q = decltype(q)::value;
        if constexpr (N <= kTeamMaxValues) {
          if (w.team == 16) {
            hipLaunchKernelGGL((balance_sums_kernel<L, N, Q, 16>), dim3(unsigned(w.places)), dim3(1024), unsigned(17 * E * 4), s, b);
            return;
          }
        }
        if (w.team == 4) hipLaunchKernelGGL((balance_sums_kernel<L, N, Q, 4>), dim3(unsigned(w.places)), dim3(256), unsigned(5 * E * 4), s, b);
        else if (w.team == 1) hipLaunchKernelGGL((balance_sums_kernel<L, N, Q, 1>), dim3(unsigned((w.places + 3) / 4)), dim3(256), unsigned(4 * E * 4), s, b);
        else fits = false;
      });
    FM_REQUIRE(fits, "fm_balance_forward: no kernel for pieces of %d waves", w.team);
    // Sequences of more than 64 places on average take a workgroup for 16 columns (one of 65536 tokens, 256 experts: 6.7 us, by four rows 19.6).
    // From four on, while the rows do not fill the CUs, and up to twice that from two on, four rows of a wave; below that a row.  By four
    // rows and by one, us: 131072 tokens of 64, 30000 sequences 107 and 20; 65536 of 256, 512 sequences (two places each) 9.0 and 6.7, 1300
    // sequences 23 and 15, 400 9.0 and 10.6; 65536 of 32, 2048 sequences 6.2 and 13.2, 4000 8.8 and 6.0; 65536 of 128, 700 8.7 and 6.1.
    auto fold_by = [&](auto c, auto rows, auto most) {
      constexpr int C = decltype(c)::value, R = decltype(rows)::value, M = decltype(most)::value, G = 1024 / (C * R);
      const int parts = (E + C - 1) / C;
      fin.parts = (S + G - 1) / G * parts;
      if (S > 0) hipLaunchKernelGGL((balance_fold_kernel<C, R, M>), dim3(unsigned(fin.parts)), dim3(1024), 0, s, fold, parts, fin);
    };
    if (w.runs > 64 * S) fold_by(std::integral_constant<int, 16>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 0>{});
    else if (w.runs > 4 * S || S * E <= 1 << 16 || (w.runs > 2 * S && S * E <= 1 << 17)) fold_by(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{}, std::integral_constant<int, 256>{});
    else if (E > 32) fold_by(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
    else fold_by(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
    if (fin.parts != 1) hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, s, fin);
  }
  if (acc && S > 0) hipLaunchKernelGGL(balance_track_kernel, dim3(unsigned(E)), dim3(256), 0, s, counts, S, E, acc);
  return check_launch("fm_balance_forward");
}

int fm_balance_backward(const float* logits, int64_t ld, int64_t T, int E, const int32_t* cu, int64_t S, const uint8_t* mask, int sigmoid,
                        float z_mult, const float* f, const float* inverse, const float* dloss, float* dlogits, int64_t ld_d, int add,
                        void* stream) {
  BalanceArgs b{logits, ld, T, E, 1, nullptr, 0, cu, S, mask, sigmoid, z_mult != 0.f, 0, 0, nullptr, nullptr, nullptr, nullptr};
  if (int rc = check_balance(b, "fm_balance_backward")) return rc;
  if (T == 0) return 0;
  FM_REQUIRE(inverse && dloss && dlogits && ld_d >= E && (S == 0 || f), "fm_balance_backward: null pointer or a pitch below E");
  b.run = run_of(T, E);
  b.places = (T + b.run - 1) / b.run + S + 2;
  const BalanceBwdArgs a{b, f, inverse, dloss, z_mult, dlogits, ld_d, add};
  for_experts(E, [&](auto l, auto n, auto q) {
    hipLaunchKernelGGL((balance_backward_kernel<decltype(l)::value, decltype(n)::value, decltype(q)::value>), dim3(unsigned((b.places + 3) / 4)),
                       dim3(256), 0, static_cast<hipStream_t>(stream), a);
  });
  return check_launch("fm_balance_backward");
}

}  // extern "C"
