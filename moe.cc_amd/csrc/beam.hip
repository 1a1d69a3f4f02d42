// beam.hip - the selection of a beam search (moe_beam_select_dev, include/moehip.h).
//
// Rows (beams) in groups of n_beam, each with the logits x_v of its next token
// and the log probability `score` it has so far:
//   value(row, v) = score + x_v - lse,   lse = log sum_v exp(x_v),
// and of each group's candidates the n_beam with the largest value * weight.
//
// One read of the logits bounds it.  The first kernel cuts a row into blocks;
// a wave takes 1024 logits a step, sums their exponentials and keeps the
// n_beam best as a list sorted over its lanes.  The second, a block a group,
// joins the rows' sums and lists and ranks the candidates of all rows.  One
// group of 4 beams over 151936 tokens takes 11.5 us, of which the launches and
// the chain of a block's own work are most; 24 groups of 8 (117 MB, 104 of them
// of rows that go on) 37.5 us, the first kernel's 31 of them at 3.4 TB/s, where
// vector instructions take 62 % of the cycles at 4 each (an exponential takes
// more) and waves wait 45 % of theirs.
//
// Order.  Inside a row candidates are ordered by (logit, token), which a
// 64-bit whole number holds exactly: the logit's bits as an ordered whole
// number above, the token's complement below.  Between rows by value * weight
// in 64 bits, of values that are as exact as the sums: exp(x) = 2^(x log2(e)),
// the product carried in two floats and split into a whole number and what is
// left, so that a term's error is that of the hardware's exp2 on [-1/2, 1/2]
// (2^-23 of it, either way) and 2^-25; four terms are added in fp32 (2^-23), the
// rest in 64 bits.  Errors of many terms average out; of a token that holds
// nearly all of its row's probability they do not: lse is within 2^-21 (5e-7),
// and rows whose values differ by less than twice that may change places.
#include <math.h>

#include <type_traits>

#include "moe_device.h"
#include "moe_lib.h"
#include "paged_attn.h"

namespace moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMostBeams = kWave;          // a list is a lane a beam
// From here on a wave collects its candidates, sorts 64 at a time and merges them into its list, and blocks' lists are merged by
// a kernel of their own; below, candidates are inserted one by one (one group over 151936 tokens, us with the first and the
// second: 8 beams 23.7, 14.8; 16 25.9, 23.2; 24 27.7, about 43; 32 29.3, about 57; 24 groups of 8 51.6, 38.0; 200 groups of 64
// over 1000 tokens, whole steps, 158, 707).
constexpr int kMergedBeams = 17;
// Blocks that rows are cut into, about: 16 waves a CU, and few enough lists for the second kernel (us at 512, 1024 and 2048, 8
// beams: 24 groups 44.7, 38.1, 38.6; 64 groups 70.5, 63.8, 65.5; one group alike; one of 64 37.6, 36.3, 41.7).
constexpr int kBlocks = 1024;
// Rows of up to this many tokens, one step of a wave, go in quarters to all four (us with whole steps and quarters: 200 groups of
// 64 beams over 1000 tokens 136, 86, over 300 116, 105; of 4 beams 11.6, 11.1, 11.2, 10.9; over 3000 tokens 112, 133).
constexpr int kShort = 1024;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Sum of a part of a row: sum * exp(at); nothing there: 0 at -inf.
struct Part {
  double sum, at;
};

__device__ __forceinline__ double part_at(const Part& p, double at) {
  return p.at == at || p.at == -(double)INFINITY ? p.sum : p.sum * exp(p.at - at);
}

struct SelectArgs {
  moe_beam_select a;
  int blocks;       // of a row
  int each, rest;   // steps of a block, one more for the first `rest`
  Part* parts;      // work [rows][blocks]
  int merged;       // the blocks' lists are merged by a kernel of their own
  uint64_t* keys;   // work [rows][n_beam][blocks], or merged [rows][blocks][n_beam]: each block's best, in order; 0: none
};

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // (-0 is 0)
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
}
constexpr uint32_t kOrderedNone = 0x007fffffu;   // of -inf, which is no candidate
// The float before that of an ordered number (before 0 lies -0, which is 0).
__device__ __forceinline__ float before(uint32_t u) { return unordered(u - (u == 0x80000000u ? 2 : 1)); }

__device__ __forceinline__ uint64_t read_lane(uint64_t x, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}

// The value of lane ^ C, C a power of two.
template <int C>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (C == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, false);   // quad_perm [1,0,3,2]
  if constexpr (C == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, false);   // quad_perm [2,3,0,1]
  if constexpr (C == 4) {   // row_half_mirror (^ 7), quad_perm [3,2,1,0]
    x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, false);
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x1B, 0xf, 0xf, false);
  }
  if constexpr (C == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false);  // row_ror 8
  if constexpr (C == 16) {
    auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? p[0] : p[1];
  }
  if constexpr (C == 32) {
    auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? p[0] : p[1];
  }
}
// Of lane 63 - i.
__device__ __forceinline__ uint32_t lane_mirror(uint32_t x) {
  x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, false);   // row_mirror
  return lane_xor<32>(lane_xor<16>(x));
}
template <int C>
__device__ __forceinline__ uint64_t lane_xor(uint64_t x) {
  return (uint64_t)lane_xor<C>((uint32_t)(x >> 32)) << 32 | lane_xor<C>((uint32_t)x);
}
template <int C>
__device__ __forceinline__ double lane_xor(double x) { return __longlong_as_double((long long)lane_xor<C>((uint64_t)__double_as_longlong(x))); }
__device__ __forceinline__ uint64_t lane_mirror(uint64_t x) {
  return (uint64_t)lane_mirror((uint32_t)(x >> 32)) << 32 | lane_mirror((uint32_t)x);
}

// A candidate of a group: its place in the order of all (larger first; 0: none), then row * 64 + its place in the row's list
// (the lower goes first where ranks are equal).
struct Best {
  uint64_t rank;
  uint32_t from;
};
template <int C>
__device__ __forceinline__ Best lane_xor(Best x) { return {lane_xor<C>(x.rank), lane_xor<C>(x.from)}; }
__device__ __forceinline__ Best lane_mirror(Best x) { return {lane_mirror(x.rank), lane_mirror(x.from)}; }

__device__ __forceinline__ bool precedes(uint64_t x, uint64_t y) { return x > y; }
__device__ __forceinline__ bool precedes(Best x, Best y) { return x.rank > y.rank || (x.rank == y.rank && x.from < y.from); }

// Runs of 2 C lanes that rise and fall once, sorted: the first to the lowest lane where `down`, else to the highest.
template <int C, class T>
__device__ __forceinline__ T sort_runs(T x, bool down) {
  const T y = lane_xor<C>(x);
  if (precedes(x, y) != (((threadIdx.x & C) == 0) == down)) x = y;
  if constexpr (C > 1) x = sort_runs<C / 2>(x, down);
  return x;
}

// The lanes', sorted, the first to lane 0 (bitonic); of which only the first n hold any.
template <class T>
__device__ __forceinline__ T sort_lanes(T x, int n = kWave) {
  const int lane = threadIdx.x % kWave;
  if (n > 1) x = sort_runs<1>(x, !(lane & 2));
  if (n > 2) x = sort_runs<2>(x, !(lane & 4));
  if (n > 4) x = sort_runs<4>(x, !(lane & 8));
  if (n > 8) x = sort_runs<8>(x, !(lane & 16));
  if (n > 16) x = sort_runs<16>(x, !(lane & 32));
  if (n > 32) x = sort_runs<32>(x, true);
  return x;
}

// The first 64 of two lists sorted over the lanes, sorted: of lane i's and the other's 63 - i'th the first, which fall and rise
// once.
template <class T>
__device__ __forceinline__ T merge_lists(T a, T b) {
  const T other = lane_mirror(b);
  return sort_runs<32>(precedes(other, a) ? other : a, true);
}

// A list sorted over the lanes, the largest first; 0: nothing there.
struct List {
  uint64_t key = 0;
  uint64_t last = 0;   // of lane n - 1, in all lanes

  __device__ __forceinline__ void insert(uint64_t k, int n) {
    const int lane = threadIdx.x % kWave, at = __popcll(__ballot(key > k));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)key, 0x138, 0xf, 0xf, false);   // wave_shr 1
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(key >> 32), 0x138, 0xf, 0xf, false);
    key = lane < at ? key : lane == at ? k : (uint64_t)hi << 32 | lo;
    last = read_lane(key, n - 1);
  }
};

// The n-th largest of the lanes' numbers (0 where that is 0), or a number between it and the next smaller one.
__device__ __forceinline__ uint32_t nth_largest(uint32_t x, int n) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t up = t | 1u << bit;
    const int c = __popcll(__ballot(x >= up));
    if (c >= n) t = up;
    if (c == n) break;
  }
  return t;
}

// Largest of the lanes' numbers (of floats: that are numbers), in all of them.
template <class T>
__device__ __forceinline__ T wave_max(T x) {
  auto larger = [](uint32_t y, uint32_t z) {
    if constexpr (std::is_same_v<T, float>) return fmaxf(__uint_as_float(y), __uint_as_float(z));
    else return y > z ? y : z;
  };
  auto bits = [&]() { return __builtin_bit_cast(uint32_t, x); };
  x = larger(bits(), __builtin_amdgcn_update_dpp(0, bits(), 0xB1, 0xf, 0xf, false));    // quad_perm [1,0,3,2], [2,3,0,1]
  x = larger(bits(), __builtin_amdgcn_update_dpp(0, bits(), 0x4E, 0xf, 0xf, false));
  x = larger(bits(), __builtin_amdgcn_update_dpp(0, bits(), 0x141, 0xf, 0xf, false));   // row_half_mirror, row_mirror
  x = larger(bits(), __builtin_amdgcn_update_dpp(0, bits(), 0x140, 0xf, 0xf, false));
  auto p = __builtin_amdgcn_permlane32_swap(bits(), bits(), false, false);
  x = larger(p[0], p[1]);
  auto q = __builtin_amdgcn_permlane16_swap(bits(), bits(), false, false);
  return larger(q[0], q[1]);
}

__device__ __forceinline__ double wave_max_f64(double x) {
  x = fmax(x, lane_xor<1>(x)), x = fmax(x, lane_xor<2>(x)), x = fmax(x, lane_xor<4>(x));
  x = fmax(x, lane_xor<8>(x)), x = fmax(x, lane_xor<16>(x));
  return fmax(x, lane_xor<32>(x));
}

__device__ __forceinline__ double wave_sum(double x) {
  x += lane_xor<1>(x), x += lane_xor<2>(x), x += lane_xor<4>(x), x += lane_xor<8>(x), x += lane_xor<16>(x);
  return x + lane_xor<32>(x);
}

constexpr float kLog2eHi = 1.44269504088896340736f;
constexpr float kLog2eLo = (float)(1.44269504088896340736 - (double)kLog2eHi);

// exp(x - m); 0 below exp(-200).
__device__ __forceinline__ float exp_from(float x, float m) {
  float d = x - m;
  const float b = x - d;
  float e = (x - (d + b)) + (b - m);   // x - m = d + e
  if (d < -200.0f) d = -200.0f, e = 0.0f;
  const float hi = d * kLog2eHi;
  const float lo = fmaf(e, kLog2eHi, fmaf(d, kLog2eLo, fmaf(d, kLog2eHi, -hi)));
  const float y = __builtin_amdgcn_exp2f(hi);
  return fmaf(y, lo * 0.69314718055994530942f, y);
}

// exp(x) * 2^-at, for x under `floor` that of floor; at a whole number, |at| and the product's whole part below 2^21, the
// result a normal number.  A NaN counts as floor.
__device__ __forceinline__ float exp_at(float x, float floor, float at) {
  constexpr float kWhole = 12582912.0f;   // 1.5 * 2^23: a sum with it is a whole number, whose last bits are its own
  x = fmaxf(x, floor);
  const float p = x * kLog2eHi, low = fmaf(x, kLog2eLo, fmaf(x, kLog2eHi, -p));
  const float u = p + (kWhole - at), rest = p - (u - (kWhole - at));
  return __uint_as_float(__float_as_uint(__builtin_amdgcn_exp2f(rest + low)) + (__float_as_uint(u) << 23));
}

// A row has candidates from its logits: it is neither ended nor none at all.
__device__ __forceinline__ bool usable(const moe_beam_select& a, int r) {
  const float w = a.weight ? a.weight[r] : 1.0f;
  return fabsf(a.score[r]) < INFINITY && w > 0.0f && w < INFINITY;
}

// A wave's step: 16 bytes of a lane, J times.
template <int J>
__global__ __launch_bounds__(kThreads) void select_rows_kernel(SelectArgs s) {
  constexpr int N = 4 * J, STEP = N * kWave;
  const moe_beam_select& a = s.a;
  const int row = (int)blockIdx.y, b = (int)blockIdx.x, K = a.n_beam;
  if (!usable(a, row) || (a.done && a.done[row])) return;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int first = s.each * b + min(b, s.rest), end = first + s.each + (b < s.rest);
  const float* x0 = a.logits + (size_t)row * a.ld;
  const int active = min(kWaves, end - first);
  List list;
  float from = -INFINITY, power = 0.0f, floor = 0.0f;   // the logit that sums are taken from, its power of two
  double at = -(double)INFINITY;                        // as Part's
  bool far = false;                                     // logits too far from 0 for exp_at
  float least = -INFINITY;                              // what a logit has to pass
  double sum = 0.0;
  // what the block's n_beam-th has to reach at least, as an ordered number: after the first step the least of the waves'
  // share-th (share: n_beam by the waves that have a step, rounded up), then any wave's n_beam-th
  __shared__ uint32_t share_s[kWaves], least_s;
  __shared__ uint64_t pending_s[kWaves][2 * kWave];
  f32x4 next[J];
  auto load = [&](int step) {
    const int v0 = step * STEP + 4 * lane;
    if ((step + 1) * STEP <= a.vocab) {
#pragma unroll
      for (int j = 0; j < J; ++j) next[j] = *(const f32x4u*)(x0 + v0 + j * 4 * kWave);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int v = v0 + j / 4 * 4 * kWave + j % 4;
        next[j / 4][j % 4] = v < a.vocab ? x0[v] : -INFINITY;
      }
    }
  };
  if (threadIdx.x == 0) least_s = 0;
  if (first + wave < end) {
    load(first + wave);
  } else {   // a wave without a step comes to the first one's barrier all the same
    if (lane == 0) share_s[wave] = 0xffffffffu;
    __syncthreads();
  }
  for (int step = first + wave; step < end; step += kWaves) {
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = next[j / 4][j % 4];
    if (step + kWaves < end) load(step + kWaves);
    float top = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, x[j]);
    // ---- the sum.  Its power of two moves only when a term would leave fp32; terms below 2^-100 of that count as 2^-100
    const float most = wave_max(top);
    if (!(most < INFINITY)) sum = NAN;
    if (most > from + 40.0f && most < INFINITY) {
      far = fabsf(most) > 1e6f;
      power = rintf(most * kLog2eHi);
      const double now = far ? (double)most : (double)power * 0.693147180559945309417;
      if (from > -INFINITY) sum *= exp(at - now);
      at = now, from = most, floor = (power - 100.0f) * 0.693147180559945309417f;
    }
    if (far) {
#pragma unroll
      for (int j = 0; j < N; ++j) sum += (double)exp_from(x[j], from);
    } else if (from > -INFINITY) {
      float check = 0.0f;
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        check += (x[j] + x[j + 1]) + (x[j + 2] + x[j + 3]);
        sum += (double)((exp_at(x[j], floor, power) + exp_at(x[j + 1], floor, power)) + (exp_at(x[j + 2], floor, power) + exp_at(x[j + 3], floor, power)));
      }
      if (check != check) sum = NAN;   // one of them is (no infinity but -inf is left)
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) sum += x[j] == -INFINITY ? 0.0 : (double)NAN;
    }
    // ---- the best
    if (step == first + wave) {
      const int share = active >= kWaves ? (K + kWaves - 1) / kWaves : active == 3 ? (K + 2) / 3 : active == 2 ? (K + 1) / 2 : K;
      const uint32_t mine = share > 1 ? nth_largest(top > -INFINITY ? ordered(top) : 0u, share) : most > -INFINITY ? ordered(most) : 0u;
      if (lane == 0) share_s[wave] = mine;
      __syncthreads();
      uint32_t all = share_s[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) all = min(all, share_s[w]);
      least = all > kOrderedNone ? before(all) : -INFINITY;
      if (lane == 0) atomicMax(&least_s, all);
    } else {
      const uint32_t others = least_s;
      if (others > kOrderedNone) least = fmaxf(least, before(others));   // (as good as theirs may be an earlier token)
    }
    const uint64_t better = __ballot(top > least);
    if (!better) continue;
    // of the lanes' largest the K-th bounds the K-th of all from below
    uint32_t bound = kOrderedNone + 1;
    if (__popcll(better) > K) bound = max(bound, nth_largest(top > least ? ordered(top) : 0u, K));
    float pass = fmaxf(before(bound), least);
    if (K >= kMergedBeams) {   // many: 64 at a time, sorted and merged
      auto take = [&](int n) {
        list.key = merge_lists(list.key, sort_lanes(lane < n ? pending_s[wave][lane] : 0));
        list.last = read_lane(list.key, K - 1);
        if (list.last) pass = fmaxf(pass, before((uint32_t)(list.last >> 32)));
      };
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint64_t who = __ballot(x[j] > pass);
        if (!who) continue;
        const uint32_t token = (uint32_t)(step * STEP + j / 4 * 4 * kWave + 4 * lane + j % 4);
        if (x[j] > pass)
          pending_s[wave][n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] =
              (uint64_t)ordered(x[j]) << 32 | (0xffffffffu - token);
        n += __popcll(who);
        if (n < kWave) continue;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        take(kWave);
        n -= kWave;
        const uint64_t rest = pending_s[wave][kWave + lane];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        pending_s[wave][lane] = rest;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (n) take(n);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int j = 0; j < N && K < kMergedBeams; ++j) {
      uint64_t who = __ballot(x[j] > pass);
      while (who) {
        const int l = __builtin_ctzll(who);
        who &= who - 1;
        const uint32_t token = (uint32_t)(step * STEP + j / 4 * 4 * kWave + 4 * l + j % 4);
        const uint64_t k = (uint64_t)ordered(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x[j]), l))) << 32 | (0xffffffffu - token);
        if (k > list.last) list.insert(k, K);
      }
    }
    if (list.last) {
      least = fmaxf(least, unordered((uint32_t)(list.last >> 32)));
      if (lane == 0) atomicMax(&least_s, (uint32_t)(list.last >> 32));
    }
  }
  // ---- the waves' lists and sums joined
  __shared__ uint64_t key_s[kWaves][kMostBeams], best_s[kMostBeams];
  __shared__ Part part_s[kWaves];
  const double all = wave_sum(sum);
  key_s[wave][lane] = lane < K ? list.key : 0;
  if (wave == 0) best_s[lane] = 0;
  if (lane == 0) part_s[wave] = Part{all, at};
  __syncthreads();
  const int mine = threadIdx.x % kWave;
  if (mine < K && key_s[wave][mine]) {
    const uint64_t k = key_s[wave][mine];
    int before[kWaves] = {}, rank = 0;   // of each wave's list, by bisection
    for (int half = 1 << (31 - __builtin_clz(K)); half; half /= 2)
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (before[w] + half <= K && key_s[w][before[w] + half - 1] > k) before[w] += half;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) rank += before[w];
    if (rank < K) best_s[rank] = k;
  }
  __syncthreads();
  if ((int)threadIdx.x < K)
    s.keys[(size_t)row * K * s.blocks + (s.merged ? (size_t)b * K + threadIdx.x : (size_t)threadIdx.x * s.blocks + b)] = best_s[threadIdx.x];
  if (wave == 1) {   // (the first stores the list) a lane of four a wave's
    static_assert(kWaves == 4);
    const Part p = part_s[lane % kWaves];
    double most = fmax(p.at, lane_xor<1>(p.at));
    most = fmax(most, lane_xor<2>(most));
    double total = part_at(p, most);
    total += lane_xor<1>(total);
    total += lane_xor<2>(total);
    if (lane == 0) s.parts[(size_t)row * s.blocks + b] = Part{total, most};
  }
}

// exp's sum of a row from its parts, as what a logit is added to: score - lse; NaN where there is none.
__device__ __forceinline__ double base_of(const SelectArgs& s, int row, float score) {
  const int lane = threadIdx.x % kWave;
  const Part* p = s.parts + (size_t)row * s.blocks;
  const Part first = lane < s.blocks ? p[lane] : Part{0.0, -(double)INFINITY};
  double most = first.at;
  for (int c = lane + kWave; c < s.blocks; c += kWave) most = fmax(most, p[c].at);
  most = wave_max_f64(most);
  double sum = part_at(first, most);
  for (int c = lane + kWave; c < s.blocks; c += kWave) sum += part_at(p[c], most);
  sum = wave_sum(sum);
  if (!(sum > 0.0 && sum < (double)INFINITY)) return NAN;   // (a NaN or +inf among the logits makes it NaN)
  return (double)score - (most + log(sum));
}

// A candidate's place in the order of all, larger first: value * weight as an ordered whole number, above 0.
__device__ __forceinline__ uint64_t rank_of(double value, double weight) {
  const uint64_t bits = (uint64_t)__double_as_longlong(value * weight + 0.0);
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}

__device__ __forceinline__ double value_of(double base, uint64_t key) { return base + (double)unordered((uint32_t)(key >> 32)); }

__device__ __forceinline__ void write_choice(const moe_beam_select& a, int to, int parent, bool done, double value, uint64_t key) {
  const int token = done ? a.pad : (int)(0xffffffffu - (uint32_t)key), ends = done || token == a.eos;
  a.parent[to] = parent;
  a.token[to] = token;
  a.score_out[to] = (float)value;
  a.done_out[to] = ends;
  a.fresh[to] = !ends;
}

__device__ __forceinline__ void write_none(const moe_beam_select& a, int to) {
  a.parent[to] = a.token[to] = -1, a.score_out[to] = -INFINITY, a.done_out[to] = a.fresh[to] = 0;
}

// Many beams: a block a row merges its blocks' lists, into the first one's place, and its sums.
__global__ __launch_bounds__(kThreads) void select_merge_kernel(SelectArgs s) {
  const moe_beam_select& a = s.a;
  const int row = (int)blockIdx.x, K = a.n_beam, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  if (!usable(a, row) || (a.done && a.done[row])) return;
  uint64_t* keys = s.keys + (size_t)row * K * s.blocks;
  auto load = [&](int b) { return lane < K && b < s.blocks ? keys[(size_t)b * K + lane] : 0; };
  uint64_t best = load(wave), next = load(wave + kWaves);
  for (int b = wave + kWaves; b < s.blocks; b += kWaves) {
    const uint64_t now = next;
    next = load(b + kWaves);
    if (__any(now > read_lane(best, K - 1))) best = merge_lists(best, now);
  }
  __shared__ uint64_t list_s[kWaves][kWave];
  list_s[wave][lane] = best;
  __syncthreads();
  if (wave == 1) {
    const double base = base_of(s, row, a.score[row]);
    if (lane == 0) s.parts[(size_t)row * s.blocks].sum = base;
  }
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) best = merge_lists(best, list_s[w][lane]);
  if (lane < K) keys[lane] = best;
}

// Then a block a group: a wave merges every sixteenth row's candidates, four of the waves theirs, the first these.
__global__ __launch_bounds__(1024) void select_many_kernel(SelectArgs s) {
  const moe_beam_select& a = s.a;
  constexpr int W = 1024 / kWave, R = kMostBeams / W;
  const int K = a.n_beam, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, row0 = (int)blockIdx.x * K;
  __shared__ uint64_t key_s[kMostBeams][kMostBeams], rank_s[W][kWave];
  __shared__ uint32_t from_s[W][kWave];
  __shared__ int done_s[kMostBeams];
  __shared__ double base_s[kMostBeams];
  Best best[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int mine = wave + i * W, row = row0 + min(mine, K - 1);
    const bool use = mine < K && usable(a, row), done = a.done && a.done[row];
    const float score = a.score[row];
    const double weight = a.weight ? (double)a.weight[row] : 1.0, base = done ? (double)score : use ? s.parts[(size_t)row * s.blocks].sum : NAN;
    const uint64_t key = !use || base != base ? 0 : done ? lane == 0 : lane < K ? s.keys[(size_t)row * K * s.blocks + lane] : 0;
    best[i].rank = key ? rank_of(done ? base : value_of(base, key), weight) : 0;
    best[i].from = mine * kWave + lane;
    key_s[mine][lane] = key;
    if (lane == 0) base_s[mine] = base, done_s[mine] = done;
  }
#pragma unroll
  for (int i = 1; i < R; ++i) best[0] = merge_lists(best[0], best[i]);
  for (int n = W; n > 1; n /= 4) {
    if (wave < n) rank_s[wave][lane] = best[0].rank, from_s[wave][lane] = best[0].from;
    __syncthreads();
    if (wave < n / 4)
      for (int i = 1; i < 4; ++i) best[0] = merge_lists(best[0], Best{rank_s[wave + i * (n / 4)][lane], from_s[wave + i * (n / 4)][lane]});
    __syncthreads();
  }
  if (wave || lane >= K) return;
  const int mine = best[0].from / kWave;
  if (!best[0].rank) return write_none(a, row0 + lane);
  const uint64_t key = key_s[mine][best[0].from % kWave];
  const bool done = done_s[mine];
  write_choice(a, row0 + lane, row0 + mine, done, done ? base_s[mine] : value_of(base_s[mine], key), key);
}

// A block a group: a wave a row, then all rows' candidates sorted at once (taken one by one, the best of a lane a row each time,
// 8 beams take 0.9 us more, 16 2.5).  One beam has nothing to sort: the code of it, jumped over, costs 1 us of 10 in fetches.
constexpr int kSorted = 4;   // waves that sort: 16 beams of up to 16 candidates
static_assert(kMergedBeams <= 17);
__global__ __launch_bounds__(1024) void select_groups_kernel(SelectArgs s) {
  const moe_beam_select& a = s.a;
  constexpr int W = 1024 / kWave;
  const int K = a.n_beam, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, row0 = (int)blockIdx.x * K;
  __shared__ uint64_t key_s[kMergedBeams][kMergedBeams];
  __shared__ double base_s[kMergedBeams], weight_s[kMergedBeams];
  __shared__ int count_s[kMergedBeams], done_s[kMergedBeams];
  __shared__ uint64_t rank_s[kSorted][kWave];
  __shared__ uint32_t from_s[kSorted][kWave];
  for (int i = wave; i < K; i += W) {
    const int row = row0 + i;
    const bool use = usable(a, row), done = a.done && a.done[row];
    const float score = a.score[row];
    const double weight = a.weight ? (double)a.weight[row] : 1.0;
    List list;
    double base = score;
    int count = 0;
    if (use && done) {
      count = 1;
      list.key = lane == 0 ? 1 : 0;
    } else if (use) {
      const uint64_t* keys = s.keys + (size_t)row * K * s.blocks;
      auto load = [&](int c0) { return c0 + lane < K * s.blocks ? keys[c0 + lane] : 0; };
      uint64_t next = load(0), after = load(kWave);   // (two ahead)
      base = base_of(s, row, score);
      if (base == base) {
        for (int c0 = 0; c0 < K * s.blocks; c0 += kWave) {
          const uint64_t k = next;
          next = after;
          after = load(c0 + 2 * kWave);
          if (!__any(k > list.last)) continue;
          const uint32_t bound = nth_largest(k > list.last ? (uint32_t)(k >> 32) : 0u, K);
          uint64_t who = __ballot(k > list.last && (uint32_t)(k >> 32) >= bound);
          while (who) {
            const int l = __builtin_ctzll(who);
            who &= who - 1;
            const uint64_t x = read_lane(k, l);
            if (x > list.last) list.insert(x, K);
          }
        }
        count = __popcll(__ballot(lane < K && list.key != 0));
      }
    }
    if (lane < K) key_s[i][lane] = list.key;
    if (lane == 0) count_s[i] = count, base_s[i] = base, done_s[i] = done, weight_s[i] = weight;
  }
  __syncthreads();
  // ---- all candidates a lane each, 1 << side lanes a row, sorted; past 64 of them by as many waves, whose lists the first one
  // merges
  const int side = K <= 1 ? 0 : 32 - __builtin_clz(K - 1), waves = ((K << side) + kWave - 1) / kWave;
  Best best = {0, (uint32_t)tid};
  if (wave < waves) {
    const int mine = min(tid >> side, K - 1), at = tid & ((1 << side) - 1);
    best.from = (uint32_t)(mine * kWave + at);
    if (tid >> side < K && at < count_s[mine]) best.rank = rank_of(done_s[mine] ? base_s[mine] : value_of(base_s[mine], key_s[mine][at]), weight_s[mine]);
    if (K > 1) best = sort_lanes(best, K << side);
  }
  if (waves > 1) {
    if (wave < waves) rank_s[wave][lane] = best.rank, from_s[wave][lane] = best.from;
    __syncthreads();
  }
  if (wave) return;
  for (int w = 1; w < waves; ++w) best = merge_lists(best, Best{rank_s[w][lane], from_s[w][lane]});
  if (lane >= K) return;
  if (!best.rank) return write_none(a, row0 + lane);
  const int mine = (int)best.from / kWave;
  const uint64_t key = key_s[mine][best.from % kWave];
  const bool done = done_s[mine];
  write_choice(a, row0 + lane, row0 + mine, done, done ? base_s[mine] : value_of(base_s[mine], key), key);
}

// Logits of a wave's step.
int step_for(int vocab) { return vocab <= kShort ? 4 * kWave : 16 * kWave; }

// Blocks that a row is cut into: as many steps a wave as leave about kBlocks in all.
int blocks_for(long long rows, int vocab) {
  const long long step = step_for(vocab), steps = (vocab + step - 1) / step, most = (steps + kWaves - 1) / kWaves;
  const long long want = kBlocks / rows;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

constexpr long long kMostSelected = 65535;   // rows: a launch's second dimension

}  // namespace

moe_status check_select(const moe_beam_select* a) {
  if (!a) return set_error(MOE_ERR_ARG, "beam_select: null argument");
  if (a->n_groups < 0 || a->n_beam < 1 || a->vocab < 1)
    return set_error(MOE_ERR_ARG, "beam_select: %d groups of %d beams, %d tokens", a->n_groups, a->n_beam, a->vocab);
  if (a->n_beam > kMostBeams || (long long)a->n_groups * a->n_beam > kMostSelected || a->vocab > (1 << 30))
    return set_error(MOE_ERR_UNSUPPORTED, "beam_select: %d groups of %d beams, %d tokens (at most %d beams, %lld rows, 2^30 tokens)",
                     a->n_groups, a->n_beam, a->vocab, kMostBeams, kMostSelected);
  if (a->ld < a->vocab) return set_error(MOE_ERR_ARG, "beam_select: rows of %lld floats for %d tokens", a->ld, a->vocab);
  if (a->n_groups == 0) return MOE_OK;
  if (!a->logits || !a->score || !a->parent || !a->token || !a->score_out || !a->done_out || !a->fresh || !a->work)
    return set_error(MOE_ERR_ARG, "beam_select: null pointer");
  const size_t need = ::moe_beam_select_work_bytes(a->n_groups, a->n_beam, a->vocab);
  if (a->work_bytes < need || (uintptr_t)a->work % 16)
    return set_error(MOE_ERR_ARG, "beam_select: %zu bytes of work at %p, %zu needed, 16-byte aligned", a->work_bytes, a->work, need);
  return MOE_OK;
}

}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_beam_select_work_bytes(int n_groups, int n_beam, int vocab) {
  if (n_groups < 0 || n_beam < 1 || n_beam > kMostBeams || vocab < 1 || (long long)n_groups * n_beam > kMostSelected) return 0;
  const size_t rows = (size_t)n_groups * n_beam;
  return rows ? rows * blocks_for((long long)rows, vocab) * (sizeof(Part) + 8 * (size_t)n_beam) : 16;
}

moe_status moe_beam_select_dev(const moe_beam_select* a) {
  moe_status st = check_select(a);
  if (st || a->n_groups == 0 || (st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const int rows = a->n_groups * a->n_beam;
  SelectArgs s;
  s.a = *a;
  s.blocks = blocks_for(rows, a->vocab);
  const int steps = (a->vocab + step_for(a->vocab) - 1) / step_for(a->vocab);
  s.each = steps / s.blocks, s.rest = steps % s.blocks;
  s.merged = a->n_beam >= kMergedBeams;
  s.parts = (Part*)a->work;
  s.keys = (uint64_t*)(s.parts + (size_t)rows * s.blocks);
  hipLaunchKernelGGL(a->vocab <= kShort ? select_rows_kernel<1> : select_rows_kernel<4>, dim3((unsigned)s.blocks, (unsigned)rows), dim3(kThreads), 0, stream(), s);
  if ((st = check_hip(hipGetLastError(), "beam_select launch"))) return st;
  if (s.merged) {
    hipLaunchKernelGGL(select_merge_kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream(), s);
    if ((st = check_hip(hipGetLastError(), "beam_select launch"))) return st;
  }
  hipLaunchKernelGGL(s.merged ? select_many_kernel : select_groups_kernel, dim3((unsigned)a->n_groups), dim3(1024), 0, stream(), s);
  return check_hip(hipGetLastError(), "beam_select launch");
}

}  // extern "C"
