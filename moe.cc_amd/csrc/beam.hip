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
// joins the rows' sums and lists and ranks the candidates of all rows.
//
// Order.  Inside a row candidates are ordered by (logit, token), which a
// 64-bit whole number holds exactly: the logit's bits as an ordered whole
// number above, the token's complement below.  Between rows by value * weight
// in 64 bits, so that two candidates are told apart unless they are 1e-8 close
// to each other; that is also how exact the sums are.  Sums: exp(x - m) with
// x - m and its product with log2(e) carried in two floats each, so that a
// term's only error is that of the hardware's exp2 (2^-23 of it, either way);
// four terms are added in fp32, the rest in 64 bits.
#include <math.h>

#include "moe_device.h"
#include "moe_lib.h"

namespace moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMostBeams = kWave;          // a list is a lane a beam
constexpr int kStep = 16 * kWave;          // logits of a wave's step
constexpr int kBlocks = 2048;              // blocks that rows are cut into, about

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Sum of a part of a row: sum * exp(at); nothing there: 0 at -inf.
struct Part {
  double sum;
  float at, pad;
};

__device__ __forceinline__ double part_at(const Part& p, float at) {
  return p.at == at || p.at == -INFINITY ? p.sum : p.sum * exp((double)p.at - (double)at);
}

struct SelectArgs {
  moe_beam_select a;
  int blocks;       // of a row
  Part* parts;      // work [rows][blocks]
  uint64_t* keys;   // work [rows][n_beam][blocks]: each block's best, in order; 0: none
};

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // (-0 is 0)
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
}
constexpr uint32_t kOrderedNone = 0x007fffffu;   // of -inf, which is no candidate

__device__ __forceinline__ uint64_t read_lane(uint64_t x, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, l);
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

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int c = 32; c; c /= 2) x = fmaxf(x, __shfl_xor(x, c));
  return x;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int c = 32; c; c /= 2) x += __shfl_xor(x, c);
  return x;
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

// A row has candidates from its logits: it is neither ended nor none at all.
__device__ __forceinline__ bool usable(const moe_beam_select& a, int r) {
  const float w = a.weight ? a.weight[r] : 1.0f;
  return fabsf(a.score[r]) < INFINITY && w > 0.0f && w < INFINITY;
}

__global__ __launch_bounds__(kThreads) void select_rows_kernel(SelectArgs s) {
  const moe_beam_select& a = s.a;
  const int row = (int)blockIdx.y, b = (int)blockIdx.x, K = a.n_beam;
  if (!usable(a, row) || (a.done && a.done[row])) return;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int steps = (a.vocab + kStep - 1) / kStep;
  const int first = (int)((long long)b * steps / s.blocks), end = (int)((long long)(b + 1) * steps / s.blocks);
  const float* x0 = a.logits + (size_t)row * a.ld;
  List list;
  float at = -INFINITY, least = -INFINITY;   // at: as Part's; least: what a logit has to pass
  double sum = 0.0;
  for (int step = first + wave; step < end; step += kWaves) {
    const int v0 = step * kStep + 4 * lane;
    float x[16];
    if ((step + 1) * kStep <= a.vocab) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 y = *(const f32x4u*)(x0 + v0 + j * 4 * kWave);
        x[4 * j] = y[0], x[4 * j + 1] = y[1], x[4 * j + 2] = y[2], x[4 * j + 3] = y[3];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int v = v0 + j / 4 * 4 * kWave + j % 4;
        x[j] = v < a.vocab ? x0[v] : -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]);
    // ---- the sum.  What it is taken from moves only when a term would leave fp32
    const float most = wave_max(top);
    if (most > at + 40.0f) {
      if (at > -INFINITY) sum *= exp((double)at - (double)most);
      at = most;
    }
    if (at > -INFINITY) {
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        sum += (double)((exp_from(x[j], at) + exp_from(x[j + 1], at)) + (exp_from(x[j + 2], at) + exp_from(x[j + 3], at)));
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) sum += x[j] == -INFINITY ? 0.0 : (double)NAN;
    }
    // ---- the best.  Of the lanes' largest the K-th bounds the K-th of all from below
    const uint32_t bound = max(nth_largest(top > least ? ordered(top) : 0u, K), kOrderedNone + 1);
    if (!__any(top > least)) continue;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      uint64_t who = __ballot(ordered(x[j]) >= bound && x[j] > least);
      while (who) {
        const int l = __builtin_ctzll(who);
        who &= who - 1;
        const uint32_t token = (uint32_t)(step * kStep + j / 4 * 4 * kWave + 4 * l + j % 4);
        const uint64_t k = (uint64_t)ordered(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x[j]), l))) << 32 | (0xffffffffu - token);
        if (k > list.last) list.insert(k, K);
      }
    }
    if (list.last) least = unordered((uint32_t)(list.last >> 32));
  }
  // ---- the waves' lists and sums joined
  __shared__ uint64_t key_s[kWaves][kMostBeams], best_s[kMostBeams];
  __shared__ Part part_s[kWaves];
  const double all = wave_sum(sum);
  key_s[wave][lane] = lane < K ? list.key : 0;
  if (wave == 0) best_s[lane] = 0;
  if (lane == 0) part_s[wave] = Part{all, at, 0.0f};
  __syncthreads();
  const int mine = threadIdx.x % kWave;
  if (mine < K && key_s[wave][mine]) {
    const uint64_t k = key_s[wave][mine];
    int rank = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      for (int i = 0; i < K; ++i) rank += key_s[w][i] > k;
    if (rank < K) best_s[rank] = k;
  }
  __syncthreads();
  if ((int)threadIdx.x < K) s.keys[((size_t)row * K + threadIdx.x) * s.blocks + b] = best_s[threadIdx.x];
  if (threadIdx.x == 0) {
    float most = part_s[0].at;
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, part_s[w].at);
    double total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += part_at(part_s[w], most);
    s.parts[(size_t)row * s.blocks + b] = Part{total, most, 0.0f};
  }
}

// A block a group; a wave a row, then all rows' lists against each other.
__global__ __launch_bounds__(1024) void select_groups_kernel(SelectArgs s) {
  const moe_beam_select& a = s.a;
  constexpr int W = 1024 / kWave;
  const int K = a.n_beam, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, row0 = (int)blockIdx.x * K;
  __shared__ uint64_t key_s[kMostBeams][kMostBeams];
  __shared__ double base_s[kMostBeams], weight_s[kMostBeams];
  __shared__ int count_s[kMostBeams], place_s[kMostBeams * kMostBeams], out_s[kMostBeams], done_s[kMostBeams];
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
      const Part* p = s.parts + (size_t)row * s.blocks;
      float most = -INFINITY;
      for (int c = lane; c < s.blocks; c += kWave) most = fmaxf(most, p[c].at);
      most = wave_max(most);
      double sum = 0.0;
      for (int c = lane; c < s.blocks; c += kWave) sum += part_at(p[c], most);
      sum = wave_sum(sum);
      if (sum > 0.0 && sum < (double)INFINITY) {   // (a NaN or +inf among the logits makes it NaN)
        base = (double)score - ((double)most + log(sum));
        const uint64_t* keys = s.keys + (size_t)row * K * s.blocks;
        for (int c0 = 0; c0 < K * s.blocks; c0 += kWave) {
          const uint64_t k = c0 + lane < K * s.blocks ? keys[c0 + lane] : 0;
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
  auto value_of = [&](int row, int c) {
    return done_s[row] ? base_s[row] : base_s[row] + (double)unordered((uint32_t)(key_s[row][c] >> 32));
  };
  for (int i = tid; i < K * K; i += 1024) place_s[i] = 0;
  if (tid < K) out_s[tid] = -1;
  __syncthreads();
  // the place of each candidate: how many of every row come before it
  for (int i = tid; i < K * K * K; i += 1024) {
    const int at = i / K, other = i % K, row = at / K, c = at % K;
    if (c >= count_s[row]) continue;
    int n;
    if (other == row) {
      n = c;
    } else {
      const double x = value_of(row, c) * weight_s[row];
      int lo = 0, hi = count_s[other];   // equal ranks: the lower row first
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double y = value_of(other, mid) * weight_s[other];
        if (y > x || (y == x && other < row)) lo = mid + 1;
        else hi = mid;
      }
      n = lo;
    }
    if (n) atomicAdd(&place_s[at], n);
  }
  __syncthreads();
  for (int i = tid; i < K * K; i += 1024)
    if (i % K < count_s[i / K] && place_s[i] < K) out_s[place_s[i]] = i;
  __syncthreads();
  if (tid < K) {
    const int from = out_s[tid], to = row0 + tid;
    int parent = -1, token = -1, done = 0;
    double value = -(double)INFINITY;
    if (from >= 0) {
      const int row = from / K, c = from % K;
      const uint64_t k = key_s[row][c];
      parent = row0 + row;
      done = done_s[row] != 0;
      token = done ? a.pad : (int)(0xffffffffu - (uint32_t)k);
      value = value_of(row, c);
      done = done || token == a.eos;
    }
    a.parent[to] = parent;
    a.token[to] = token;
    a.score_out[to] = (float)value;
    a.done_out[to] = done;
    a.fresh[to] = parent >= 0 && !done;
  }
}

// Blocks that a row is cut into: as many steps a wave as leave about kBlocks in all.
int blocks_for(long long rows, int vocab) {
  const long long steps = (vocab + kStep - 1) / kStep, most = (steps + kWaves - 1) / kWaves;
  const long long want = kBlocks / rows;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

constexpr long long kMostRows = 65535;   // a launch's second dimension

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_beam_select_work_bytes(int n_groups, int n_beam, int vocab) {
  if (n_groups < 0 || n_beam < 1 || n_beam > kMostBeams || vocab < 1 || (long long)n_groups * n_beam > kMostRows) return 0;
  const size_t rows = (size_t)n_groups * n_beam;
  return rows ? rows * blocks_for((long long)rows, vocab) * (sizeof(Part) + 8 * (size_t)n_beam) : 16;
}

moe_status moe_beam_select_dev(const moe_beam_select* a) {
  if (!a) return set_error(MOE_ERR_ARG, "beam_select: null argument");
  if (a->n_groups < 0 || a->n_beam < 1 || a->vocab < 1)
    return set_error(MOE_ERR_ARG, "beam_select: %d groups of %d beams, %d tokens", a->n_groups, a->n_beam, a->vocab);
  if (a->n_beam > kMostBeams || (long long)a->n_groups * a->n_beam > kMostRows || a->vocab > (1 << 30))
    return set_error(MOE_ERR_UNSUPPORTED, "beam_select: %d groups of %d beams, %d tokens (at most %d beams, %lld rows, 2^30 tokens)",
                     a->n_groups, a->n_beam, a->vocab, kMostBeams, kMostRows);
  if (a->ld < a->vocab) return set_error(MOE_ERR_ARG, "beam_select: rows of %lld floats for %d tokens", a->ld, a->vocab);
  if (a->n_groups == 0) return MOE_OK;
  if (!a->logits || !a->score || !a->parent || !a->token || !a->score_out || !a->done_out || !a->fresh || !a->work)
    return set_error(MOE_ERR_ARG, "beam_select: null pointer");
  const size_t need = moe_beam_select_work_bytes(a->n_groups, a->n_beam, a->vocab);
  if (a->work_bytes < need || (uintptr_t)a->work % 16)
    return set_error(MOE_ERR_ARG, "beam_select: %zu bytes of work at %p, %zu needed, 16-byte aligned", a->work_bytes, a->work, need);
  moe_status st = ensure_init();
  if (st) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const int rows = a->n_groups * a->n_beam;
  SelectArgs s;
  s.a = *a;
  s.blocks = blocks_for(rows, a->vocab);
  s.parts = (Part*)a->work;
  s.keys = (uint64_t*)(s.parts + (size_t)rows * s.blocks);
  hipLaunchKernelGGL(select_rows_kernel, dim3((unsigned)s.blocks, (unsigned)rows), dim3(kThreads), 0, stream(), s);
  if ((st = check_hip(hipGetLastError(), "beam_select launch"))) return st;
  hipLaunchKernelGGL(select_groups_kernel, dim3((unsigned)a->n_groups), dim3(1024), 0, stream(), s);
  return check_hip(hipGetLastError(), "beam_select launch");
}

}  // extern "C"
