// paged_attn.hip - attention of new tokens over a paged cache
// (moe_paged_attn_dev, include/moehip.h).
//
// For a row (token) and one key-value head, with its G = n_q / n_kv query
// heads q_h and the row's positions j:
//   s_hj = scale q_h . k_j,  out_h = sum_j exp(s_hj - m_h) v_j / sum_j exp(s_hj - m_h)
// in one pass over the pages with a running maximum m_h.  The bytes of K and V
// bound it (4 G operations a cached element), so a K or V byte is loaded once,
// 16 bytes a lane, straight into the registers that the matrix instructions
// read, with no LDS and no barrier in the loop:
//   scores   16 keys x 16 heads a tile: lane l holds 16-byte pieces of key l % 16, and the matching query values of
//            head l % 16; any order of the dimensions will do as long as both sides share it
//   weights  come out as keys 4 (l / 16) + i of head l % 16, and go back in as the second operand from the same lane:
//            the instruction's sum runs over the keys in that order
//   values   lane l holds the keys 4 (l / 16) + i of both tiles at its 1 / 16 of the dimensions; pairs of keys are put
//            side by side by byte permutes; the sums come out as 16 dimensions x 16 heads, so a lane rescales its own head
// Rounding: the products run on 16-bit operands with fp32 sums.  Keys and values enter as they are stored (8-bit ones are
// exact in bf16); the fp32 queries and weights are split into three 16-bit parts that hold all their bits, so that
// nothing is lost against an fp32 evaluation.  (f16 parts hold what lies above 2^-38 of a head's largest query value or
// weight; below it bits drop out of the products, of a weight those with its value, while its sum counts it.)  The matrix units this triples the work of are busy a seventh of the long batches' time.
// fp32 pages use the fp32 instruction (16 x 16 x 4) on the same layouts.
//
// Work is split over the length too.  The rows' positions, in units of kUnit, are laid end to end and cut into as many
// even pieces as the chip holds blocks at once; a block walks the rows of its piece, whose place it finds in the rows'
// lengths by itself (find_piece).  Parts of a row that pieces cut go to `work` and are joined by a second kernel.  (Joined
// in the same launch they would need a device-scope release a block, an L2 write-back here: 24 rows 18 -> 29 us, where the
// second launch costs 4.)
//
// 32 / 4 heads of 128: 256 bf16 rows of 1..8192 positions 354-386 us (5.6-6.1 TB/s), one of 131072 49 us (5.5), 64 e4m3
// rows of 512..8192 55-61 us (4.7-5.2), 24 bf16 rows of 64..2048 17 us (3.0), a row of 40 in fp32 6.7 us.  The long ones are bound by the
// bytes (the GEMVs of this library read 6.5 TB/s), the short ones by what comes one after another: launch, lengths, page
// numbers, keys, the join.  128 rows of 4096 bf16 positions in head-major pages 172 us (6.2 TB/s), slot-major, where a
// head's rows lie 256 bytes in every 1024, 180-185.  (Blocks with the heads side by side instead of one after another:
// 172 and 195.)
#include <math.h>

#include <type_traits>

#include "moe_device.h"
#include "paged_attn.h"

namespace moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
// Bytes of K's pages, attended or not (the lengths are on the device), from which loads pass the caches, since nothing of
// them is there at the next step: 64 e4m3 rows
// (142 MB) 56 us against 63 through them, 256 bf16 rows 393 against 417; below, 8 bf16 rows of 1000..7000 (33 MB) 21 us
// through the caches, 24 past them.
constexpr long long kStreamBytes = 64ll << 20;

enum { F32 = MOE_PAGE_F32, F16 = MOE_PAGE_F16, BF16 = MOE_PAGE_BF16, E4M3 = MOE_PAGE_E4M3 };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // queries may start at any float
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Memory that no one writes while the kernel runs, read at an address all lanes share: through the scalar cache, apart
// from the vector loads in flight.
template <class T>
__device__ __forceinline__ T scalar_load(const T* p, long long i) {
  return ((const __attribute__((address_space(4))) T*)(uintptr_t)p)[i];
}

// ---------------------------------------------------------------- the items

struct AttnLaunch {
  AttnPages g;
  int head_tiles;   // of 16 query heads, a key-value head
  int pieces;       // 0: rows are not cut, a block a row (SHARE: `share` rows)
  Divider each;     // by the pieces
  int share;        // SHARE: rows that the 16 columns of a tile hold; else 1
  Divider by_share, by_group;   // by share, by n_q / n_kv
  int by_row;       // joins are listed a row (T <= pieces) or a piece (`share` of each)
  int4* joins;      // work: row, parts, the piece its first lies in, its place in a run; of a piece: of the rows that end there
  float* part_ml;   // [2 pieces][share][n_q][2] work: maximum and sum of a part
  float* part_o;    // [2 pieces][share][n_q][head_dim] work: its values' sums
};

__device__ __forceinline__ int length_of(const AttnPages& g, int req, int pos) {
  return row_length(req, pos, g.a.n_req, g.a.max_pages * g.map.page_size);
}

// Sums over the lanes up to each one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ float wave_total(float x) {
  auto step = [&](auto ctrl, auto mask) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, decltype(mask)::value, 0xf, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

// Where a block's piece starts: units begin .. end - 1 of all, in row `row` of request `req`, whose first unit is `at`.
struct Piece {
  uint32_t begin, end, per;   // per: units of a piece
  int row, req, len;          // len: as length_of
  uint32_t at;
};

struct PieceShared {
  uint32_t scan[kWaves];
  Piece piece;
};

// SHARE: rows of one request that follow one another and lie among the same `share` rows (counted from 0) are a run: one
// item, whose columns are the heads of its rows, as long as the longest of them.  A prompt of 2048 bf16 positions, 8
// heads to a key-value head, 2 rows a run: 211 us, each row for itself 538; 300 rows at position 8000 194 and 447; 1000
// rows with a key-value head for each of 32 heads, 16 a run: 75 and 1052.

// The run that starts at `row`; a lane holds the length of row + lane.
struct Run {
  int n, req, longest, shortest;   // rows; longest: as length_of
  int len;
};
__device__ __forceinline__ Run run_at(const AttnLaunch& L, int row, int req, int pos) {
  const int lane = threadIdx.x % kWave;
  const int past = min(((int)divide((uint32_t)row, L.by_share) + 1) * L.share, L.g.a.T) - row;
  Run r;
  r.len = lane < past ? length_of(L.g, req, pos) : kNone;
  r.req = __builtin_amdgcn_readfirstlane(req);
  const int len0 = __builtin_amdgcn_readfirstlane(r.len);
  const uint64_t same = __ballot(r.len >= 0 && len0 >= 0 && req == r.req);
  r.n = len0 >= 0 ? __builtin_ctzll(~same) : 1;   // (lanes past the run's 16 rows at most hold kNone)
  int hi = lane < r.n ? r.len : kNone, lo = lane < r.n ? r.len : 0x7fffffff;
#pragma unroll
  for (int c = 8; c; c /= 2) hi = max(hi, __shfl_xor(hi, c)), lo = min(lo, __shfl_xor(lo, c));
  r.longest = __builtin_amdgcn_readfirstlane(hi);
  r.shortest = __builtin_amdgcn_readfirstlane(lo);
  return r;
}

// Finds piece b of the runs' units, whole groups of `share` rows a thread.
__device__ __forceinline__ void find_runs(const AttnLaunch& L, uint32_t b, bool lists, PieceShared& sh) {
  constexpr int PER = 16;   // rows a thread at most: kSplitRows are 8 each, in groups of up to 16
  const AttnPages& g = L.g;
  const int T = g.a.T, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, share = L.share;
  const int groups = (int)divide((uint32_t)(T + share - 1), L.by_share), per = (groups + kThreads - 1) / kThreads * share, t0 = tid * per;
  int len[PER], req[PER];
  uint32_t units[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = min(t0 + min(i, per - 1), T - 1);
    req[i] = g.a.req[t];
    len[i] = g.a.pos[t];
  }
  uint32_t follows = 0;   // bit i: row i belongs to the run of the row before it
  int at_share = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    len[i] = i < per && t0 + i < T ? length_of(g, req[i], len[i]) : kNone;
    if (i && at_share && len[i] >= 0 && len[i - 1] >= 0 && req[i] == req[i - 1]) follows |= 1u << i;
    at_share = at_share + 1 == share ? 0 : at_share + 1;
    if (len[i] == kPadding && L.by_row && b == 0 && lists) L.joins[t0 + i] = int4{0, 0, 0, 0};
  }
  uint32_t mine = 0;
  int longest = kNone;
#pragma unroll
  for (int i = PER - 1; i >= 0; --i) {
    longest = max(len[i], longest);
    units[i] = follows >> i & 1 ? 0 : weight_of(longest);
    if (!(follows >> i & 1)) longest = kNone;
    mine += units[i];
  }
  const uint32_t scan = wave_scan(mine);
  if (lane == kWave - 1) sh.scan[wave] = scan;
  if (tid == 0) sh.piece.row = -1;
  if (tid < share && !L.by_row && lists) L.joins[b * share + tid] = int4{0, 0, 0, 0};
  __syncthreads();
  uint32_t at = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at += sh.scan[w];
    total += sh.scan[w];
  }
  const uint32_t each = piece_units(total, L.each), begin = b * each;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (begin >= at && begin - at < units[i]) sh.piece = Piece{begin, min(begin + each, total), each, t0 + i, 0, 0, at};
    at += units[i];
  }
  __syncthreads();
}

// Finds piece b; PER rows a thread.  The host sees to it that the units' sum and the pieces fit 31 bits.
template <int PER>
__device__ __forceinline__ void find_first(const AttnLaunch& L, uint32_t b, PieceShared& sh) {
  const AttnPages& g = L.g;
  const int T = g.a.T, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int per = PER == 1 ? 1 : (T + kThreads - 1) / kThreads, t0 = tid * per;
  int len[PER], req[PER];
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = min(t0 + i, T - 1);
    req[i] = g.a.req ? g.a.req[t] : t;
    len[i] = g.a.pos[t];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    len[i] = i < per && t0 + i < T ? length_of(g, req[i], len[i]) : kNone;
    mine += units_of(len[i]);
    if (len[i] == kPadding && L.by_row && b == 0 && blockIdx.y == 0) L.joins[t0 + i] = int4{0, 0, 0, 0};
  }
  const uint32_t scan = wave_scan(mine);
  if (lane == kWave - 1) sh.scan[wave] = scan;
  if (tid == 0) {
    sh.piece.row = -1;
    if (!L.by_row && blockIdx.y == 0) L.joins[b] = int4{0, 0, 0, 0};
  }
  __syncthreads();
  uint32_t at = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at += sh.scan[w];
    total += sh.scan[w];
  }
  const uint32_t each = piece_units(total, L.each), begin = b * each;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t n = units_of(len[i]);
    if (begin >= at && begin - at < n) sh.piece = Piece{begin, min(begin + each, total), each, t0 + i, req[i], len[i], at};
    at += n;
  }
  __syncthreads();
}

template <bool SHARE>
__device__ __forceinline__ bool find_piece(const AttnLaunch& L, int b, bool lists, Piece* out) {
  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  if (SHARE && !L.pieces) {
    *out = Piece{0, 1u << 30, 1u << 30, b * L.share, 0, 0, 0};
    return true;
  }
  if (!L.pieces) {
    const int req = a.req ? scalar_load(a.req, b) : b, len = length_of(g, req, scalar_load(a.pos, b));
    const uint32_t n = units_of(len);
    *out = Piece{0, n, n, b, req, len, 0};
    return n > 0;
  }
  if (!SHARE && a.T <= kWave) {   // every wave by itself, a row a lane: no barrier (24 rows 17.9 us, 18.4 with the block's sums)
    const int lane = threadIdx.x % kWave, t = min(lane, a.T - 1);
    const int req = a.req ? a.req[t] : t, len = lane < a.T ? length_of(g, req, a.pos[t]) : kNone;
    const uint32_t n = units_of(len), scan = wave_scan(n), at = scan - n;
    const uint32_t total = __builtin_amdgcn_readlane(scan, kWave - 1);
    if (len == kPadding && L.by_row && b == 0 && blockIdx.y == 0 && threadIdx.x < kWave) L.joins[lane] = int4{0, 0, 0, 0};
    if (!L.by_row && blockIdx.y == 0 && threadIdx.x == 0) L.joins[b] = int4{0, 0, 0, 0};
    const uint32_t each = piece_units(total, L.each), begin = (uint32_t)b * each;
    const uint64_t mine = __ballot(begin >= at && begin - at < n);
    if (!mine) return false;
    const int row = __builtin_ctzll(mine);
    *out = Piece{begin, min(begin + each, total), each, row, __builtin_amdgcn_readlane(req, row),
                 __builtin_amdgcn_readlane(len, row), (uint32_t)__builtin_amdgcn_readlane(at, row)};
    return true;
  }
  __shared__ PieceShared sh;
  if constexpr (SHARE) find_runs(L, (uint32_t)b, lists, sh);
  else if (a.T <= kThreads) find_first<1>(L, (uint32_t)b, sh);
  else find_first<kSplitRows / kThreads>(L, (uint32_t)b, sh);
  auto get = [](auto x) { return (decltype(x))__builtin_amdgcn_readfirstlane((int)x); };
  *out = Piece{get(sh.piece.begin), get(sh.piece.end), get(sh.piece.per), get(sh.piece.row), get(sh.piece.req),
               get(sh.piece.len), get(sh.piece.at)};
  return out->row >= 0;
}

// ---------------------------------------------------------------- pieces

// max over the four lanes of a head (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float head_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float head_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Two fp32 values into the same place of three operands whose sum they are: bf16 parts by truncation (8 + 8 + 8 bits),
// f16 parts by the hardware's conversion toward zero (11 bits each).
template <bool HALF>
__device__ __forceinline__ void split2(float x, float y, uint32_t* a, uint32_t* b, uint32_t* c) {
  if constexpr (HALF) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const float x1 = x - (float)h[0], y1 = y - (float)h[1];
    const auto m = __builtin_amdgcn_cvt_pkrtz(x1, y1);
    const auto l = __builtin_amdgcn_cvt_pkrtz(x1 - (float)m[0], y1 - (float)m[1]);
    *a = __builtin_bit_cast(uint32_t, h);
    *b = __builtin_bit_cast(uint32_t, m);
    *c = __builtin_bit_cast(uint32_t, l);
  } else {
    const uint32_t xh = __float_as_uint(x), yh = __float_as_uint(y);
    const float x1 = x - __uint_as_float(xh & 0xffff0000u), y1 = y - __uint_as_float(yh & 0xffff0000u);
    const uint32_t xm = __float_as_uint(x1), ym = __float_as_uint(y1);
    const float x2 = x1 - __uint_as_float(xm & 0xffff0000u), y2 = y1 - __uint_as_float(ym & 0xffff0000u);
    *a = __builtin_amdgcn_perm(yh, xh, 0x07060302u);
    *b = __builtin_amdgcn_perm(ym, xm, 0x07060302u);
    *c = __builtin_amdgcn_perm(__float_as_uint(y2), __float_as_uint(x2), 0x07060302u);
  }
}

template <bool HALF>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (HALF)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// four 8-bit values -> two dwords of bf16 pairs (exact)
__device__ __forceinline__ u32x2 widen(uint32_t x) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true))};
}

// Not zero where one of the dword's values is an infinity or a NaN.
template <int CT>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  constexpr uint32_t exps = CT == F32 ? 0x7f800000u : CT == BF16 ? 0x7f807f80u : CT == F16 ? 0x7c007c00u : 0x7f7f7f7fu;
  constexpr uint32_t ones = CT == F32 ? 0x00800000u : CT == BF16 ? 0x00800080u : CT == F16 ? 0x04000400u : 0x01010101u;
  constexpr uint32_t tops = CT == F32 ? 0x80000000u : CT == E4M3 ? 0x80808080u : 0x80008000u;
  return ((x & exps) + ones) & tops;
}

// BYTES at p; STREAM: past the caches.
template <int BYTES, bool STREAM>
__device__ __forceinline__ void load_piece(const char* p, uint32_t* r) {
  typedef uint32_t V __attribute__((ext_vector_type(BYTES / 4)));
  V x;
  if constexpr (STREAM) x = __builtin_nontemporal_load((const V*)p);
  else x = *(const V*)p;
  if constexpr (BYTES == 4) r[0] = x.x;
  else
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) r[i] = x[i];
}

// ---------------------------------------------------------------- the kernel

// CT: the pages' type.  HDP: head_dim, or the next of 64, 128, 256 (the pieces past head_dim repeat its last one against
// zero queries, and their sums are not stored).  WHOLE: a tile of 16 positions lies in one page (page_size % 16 == 0), so
// its address is one scalar lookup; otherwise each lane looks up one position and the lanes exchange addresses (on pages
// of 16 and more that takes 57.9 us for the e4m3 batch where WHOLE takes 54.9, 7.3 / 6.9 for one short row, 36.2 / 34.6
// for heads of 64, 17.5 / 18.0 for 24 bf16 rows).  STREAM: loads past the caches.  SHARE: a run of rows of one request
// fills the tile's columns, so that a prompt's rows read the cache together.
template <int CT, int HDP, bool WHOLE, bool STREAM, bool SHARE>
__global__ __launch_bounds__(kThreads, HDP <= 128 ? 2 : 1) void paged_attn_kernel(AttnLaunch L) {
  constexpr bool HALF = CT == F16;
  constexpr int S = CT == F32 ? 4 : CT == E4M3 ? 1 : 2;
  constexpr int E = 16 / S;                        // elements of a 16-byte piece
  constexpr int NK = HDP / E / 4;                  // a lane's pieces of a key
  constexpr int VE = HDP / 16;                     // a lane's dimensions of a value
  constexpr int EV = VE < E ? VE : E, NV = VE / EV, VW = EV * S / 4;   // its pieces: elements, number, dwords
  constexpr int KT = CT == F32 && HDP == 256 ? 1 : 2;                  // tiles of 16 positions a step
  constexpr int NQ = CT == F32 ? 1 : HDP / 32;     // query operands of 8 values
  constexpr int STEP = 16 * KT;
  // weights are held times 2^14 where their parts are f16, far from its smallest numbers
  constexpr float kLift = HALF ? 14.0f : 0.0f;

  // SHARE: blocks of one L2 (every eighth) take neighbouring pieces of the same heads (512 rows at position 8000 312 us,
  // in the grid's order 379)
  int block = (int)blockIdx.x, heads_at = (int)blockIdx.y;
  if (const uint32_t n = gridDim.x * gridDim.y; SHARE && L.pieces && n % 8 == 0) {
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, at = id % 8 * (n / 8) + id / 8;
    heads_at = (int)(at / gridDim.x), block = (int)(at % gridDim.x);
  }
  Piece pc;
  if (!find_piece<SHARE>(L, block, heads_at == 0, &pc)) return;
  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int hd = g.map.head_dim;
  const int G = a.n_q / g.map.n_kv, kv = heads_at / L.head_tiles, tile = heads_at % L.head_tiles;
  const int head0 = kv * G + tile * 16;   // this block's query heads
  const float scale = a.scale * (g.k_scale ? scalar_load(g.k_scale, kv) : 1.0f) * 1.44269504088896340736f;
  const float vs = g.v_scale ? scalar_load(g.v_scale, kv) : 1.0f;
  const long long head_at = (long long)kv * g.map.head_stride;
  const char* kbase = (const char*)g.k + head_at * S;
  const char* vbase = (const char*)g.v + head_at * S;
  const uint32_t slot_bytes = (uint32_t)(g.map.slot_stride * S);   // WHOLE: below 2^24
  // SHARE: the rows from the next one on, a lane each, and the first that is none of the block's
  const int row_end = L.pieces ? a.T : min(pc.row + L.share, a.T);
  int next_req = 0, next_pos = 0;
  auto ask = [&](int row) {
    const int t = min(row + (int)(threadIdx.x % kWave), a.T - 1);
    next_req = a.req[t], next_pos = a.pos[t];
  };
  if constexpr (SHARE) ask(pc.row);
  for (;;) {   // the rows of the piece
  Run run = {1, 0, 0, 0, 0};
  if constexpr (SHARE) {
    run = run_at(L, pc.row, next_req, next_pos);
    pc.len = run.longest, pc.req = run.req;
    ask(pc.row + run.n);
    if (units_of(pc.len) == 0) {   // a row of no request
      if (++pc.row >= row_end) return;
      continue;
    }
  }
  const int heads = SHARE ? run.n * G : min(16, G - tile * 16);   // columns
  // (the lane's places anew for every row: addresses made from them once would fill the registers that the loop needs)
  int col = lane % 16, quad = lane / 16;
  asm volatile("" : "+v"(col), "+v"(quad));
  const uint32_t units = units_of(pc.len);
  const auto [unit0, unit1] = units_in(pc.begin, pc.end, pc.at, units);
  if (SHARE && unit0 >= units) {
    pc.at += units + kRunUnits;
    if (pc.at >= pc.end || (pc.row += run.n) >= row_end) return;
    continue;
  }
  const int first = (int)unit0 * kUnit, end = (int)min((long long)max(pc.len, 0), (long long)unit1 * kUnit);
  // the row after this one, asked for now
  const int row2 = min(pc.row + 1, a.T - 1), req2 = SHARE ? 0 : a.req ? scalar_load(a.req, row2) : row2, pos2 = SHARE ? 0 : scalar_load(a.pos, row2);
  // SHARE: the column's row of the run, its positions; all columns have those before `lo`
  const int run_row = SHARE ? min((int)divide((uint32_t)col, L.by_group), run.n - 1) : 0;
  const int my_len = SHARE ? max(__shfl(run.len, run_row), 0) : 0, my_end = min(my_len, end), lo = min(run.shortest, end);

  // WHOLE: a scalar base a tile and 32-bit lane offsets; else a 64-bit row address a lane
  uint32_t kpiece[NK], vpiece[NV];
#pragma unroll
  for (int j = 0; j < NK; ++j) kpiece[j] = (uint32_t)min((4 * j + quad) * 16, hd * S - 16);
#pragma unroll
  for (int h = 0; h < NV; ++h) vpiece[h] = (uint32_t)min((16 * h + col) * EV * S, hd * S - EV * S);

  // ---- queries: requested first, used after the first keys are requested
  const float* q = a.q + (size_t)(pc.row + run_row) * a.ldq + (size_t)(head0 + min(col, heads - 1) - run_row * G) * hd;
  f32x4 x[CT == F32 ? NK : 2 * NQ];
  auto query_dim = [&](int s) {   // of x[s]
    return CT == F32 ? (4 * s + quad) * 4 : CT == E4M3 ? (4 * (s / 4) + quad) * 16 + 4 * (s % 4) : (4 * (s / 2) + quad) * 8 + 4 * (s % 2);
  };
  constexpr int NX = CT == F32 ? NK : 2 * NQ;
#pragma unroll
  for (int s = 0; s < NX; ++s) x[s] = *(const f32x4u*)(q + min(query_dim(s), hd - 4));

  // ---- addresses
  const int* table = a.tables + (size_t)(pc.len == kOutside ? 0 : pc.req) * a.max_pages;
  // something wrong; SHARE: from this position on
  constexpr int kGood = SHARE ? 0x7fffffff : 0;
  int bad = pc.len == kOutside ? SHARE ? -1 : 1 : kGood;
  auto base_of = [&](int step) { return first + (step * kWaves + wave) * STEP; };
  // page numbers of a step: WHOLE: of its tiles; else of the lane's position
  struct Look { int p[WHOLE ? KT : 1]; };
  auto look = [&](int step) {
    Look r;
    const int base = base_of(step);
    if constexpr (WHOLE) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const int tb = min(base + 16 * t, (end - 1) & ~15);   // tiles past the end repeat the last one
        r.p[t] = scalar_load(table, divide((uint32_t)tb, g.map.per));
      }
    } else {
      r.p[0] = table[divide((uint32_t)min(base + lane, end - 1), g.map.per)];
    }
    return r;
  };
  // byte offsets: WHOLE: of a step's tiles, and the last position of each that counts; else of the lane's position.
  // Positions past the end take the last one's row, whose numbers are the request's own
  struct At { long long tile[WHOLE ? KT : 1]; int lim[WHOLE ? KT : 1]; };
  auto place = [&](int step, const Look& r) {
    At o;
    const int base = base_of(step);
    if constexpr (WHOLE) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const int tb = min(base + 16 * t, (end - 1) & ~15);
        int pg = r.p[t];
        if (!page_ok(g.map, pg)) bad = SHARE ? min(bad, tb) : 1, pg = 0;
        const int off = tb - (int)divide((uint32_t)tb, g.map.per) * g.map.page_size;
        o.tile[t] = ((long long)pg * g.map.page_stride + (long long)off * g.map.slot_stride) * S;
        o.lim[t] = min(end - 1 - tb, 15);
      }
    } else {
      const int p = min(base + lane, end - 1);
      int pg = r.p[0];
      if (!page_ok(g.map, pg)) bad = SHARE ? min(bad, p) : 1, pg = 0;
      const int off = p - (int)divide((uint32_t)p, g.map.per) * g.map.page_size;
      o.tile[0] = ((long long)pg * g.map.page_stride + (long long)off * g.map.slot_stride) * S;
      o.lim[0] = 15;
    }
    return o;
  };
  uint32_t kr[KT][NK][4], vr[4 * KT][NV][VW];
  auto load_k = [&](const At& o) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const char* base = WHOLE ? kbase + o.tile[t] : kbase + __shfl(o.tile[0], 16 * t + col);
      const uint32_t off = WHOLE ? __umul24((uint32_t)min(col, o.lim[t]), slot_bytes) : 0;
#pragma unroll
      for (int j = 0; j < NK; ++j) load_piece<16, STREAM>(base + (off + kpiece[j]), kr[t][j]);
    }
  };
  auto load_v = [&](const At& o) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* base = WHOLE ? vbase + o.tile[t] : vbase + __shfl(o.tile[0], 16 * t + 4 * quad + i);
        const uint32_t off = WHOLE ? __umul24((uint32_t)min(4 * quad + i, o.lim[t]), slot_bytes) : 0;
#pragma unroll
        for (int h = 0; h < NV; ++h) load_piece<EV * S, STREAM>(base + (off + vpiece[h]), vr[4 * t + i][h]);
      }
  };

  f32x4 o[VE];
#pragma unroll
  for (int c = 0; c < VE; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  f32x4 s[KT];
  u32x4 qa[NQ], qb[NQ], qc[NQ];
  float unlift = 1.0f;
  auto score = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < KT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        if constexpr (CT == F32) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[t][j][c]), x[j][c], s[t], 0, 0, 0);
        } else if constexpr (CT == E4M3) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u32x2 x = widen(kr[t][j][2 * u]), y = widen(kr[t][j][2 * u + 1]);
            const u32x4 k = {x[0], x[1], y[0], y[1]};
            s[t] = mfma32<HALF>(k, qa[2 * j + u], s[t]);
            s[t] = mfma32<HALF>(k, qb[2 * j + u], s[t]);
            s[t] = mfma32<HALF>(k, qc[2 * j + u], s[t]);
          }
        } else {
          const u32x4 k = {kr[t][j][0], kr[t][j][1], kr[t][j][2], kr[t][j][3]};
          s[t] = mfma32<HALF>(k, qa[j], s[t]);
          s[t] = mfma32<HALF>(k, qb[j], s[t]);
          s[t] = mfma32<HALF>(k, qc[j], s[t]);
        }
      }
  };
  // the scores' weights and their sums over the values; base: the step's first position
  auto gather = [&](int base) __attribute__((always_inline)) {
    // ---- weights
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (HALF) s[t][i] *= unlift;
        if (base + STEP > (SHARE ? lo : end) && base + 16 * t + 4 * quad + i >= (SHARE ? my_end : end)) s[t][i] = -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    top = fmaxf(m, head_max(top));
    if (__any(top > m)) {
      const float keep = top == -INFINITY ? 1.0f : exp2_hw(m - top);
      l *= keep;
#pragma unroll
      for (int c = 0; c < VE; ++c) o[c] *= keep;
      m = top;
    }
    const float from = (m == -INFINITY ? 0.0f : m) - kLift;
    float p[KT][4];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[t][i] = exp2_hw(s[t][i] - from);
        l += p[t][i];
      }
    // SHARE: a value that is no number, at a position that some columns do not have, counts as zero (their weight for it,
    // zero, would not make it one), and those that have it lose their sum
    if (SHARE && base + STEP > lo) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t odd = 0;
#pragma unroll
          for (int h = 0; h < NV; ++h)
#pragma unroll
            for (int d = 0; d < VW; ++d) odd |= not_finite<CT>(vr[4 * t + i][h][d]);
          if (__ballot(odd) >> (16 * quad) & 0xffff) {
            if (base + 16 * t + 4 * quad + i < my_end) l = p[t][i] = NAN;
#pragma unroll
            for (int h = 0; h < NV; ++h)
#pragma unroll
              for (int d = 0; d < VW; ++d) vr[4 * t + i][h][d] = 0;
          }
        }
    }
    // ---- values
    if constexpr (CT == F32) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < VE; ++c)
            o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[4 * t + i][c / EV][c % EV]), p[t][i], o[c], 0, 0, 0);
    } else {
      u32x4 pa, pb, pc;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t u, v, w;
        split2<HALF>(p[c / 2][2 * (c % 2)], p[c / 2][2 * (c % 2) + 1], &u, &v, &w);
        pa[c] = u, pb[c] = v, pc[c] = w;
      }
#pragma unroll
      for (int h = 0; h < NV; ++h) {
        constexpr int W16 = EV / 2;   // dwords of 16-bit pairs of a piece
        uint32_t w16[8][W16];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int d = 0; d < VW; ++d) {
            if constexpr (CT == E4M3) {
              const u32x2 x = widen(vr[k][h][d]);
              w16[k][2 * d] = x[0], w16[k][2 * d + 1] = x[1];
            } else {
              w16[k][d] = vr[k][h][d];
            }
          }
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          u32x4 x;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            x[c] = __builtin_amdgcn_perm(w16[2 * c + 1][e / 2], w16[2 * c][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
          o[h * EV + e] = mfma32<HALF>(x, pa, o[h * EV + e]);
          o[h * EV + e] = mfma32<HALF>(x, pb, o[h * EV + e]);
          o[h * EV + e] = mfma32<HALF>(x, pc, o[h * EV + e]);
        }
      }
    }
  };

  if (base_of(0) < end) {
    At at = place(0, look(0));
    load_k(at);
    load_v(at);
    Look next = look(1);
    // ---- queries times scale and log2(e): scores are powers of two
    float lift = 1.0f;
#pragma unroll
    for (int s = 0; s < NX; ++s) x[s] *= query_dim(s) < hd && col < heads ? scale : 0.0f;
    if constexpr (HALF) {   // the head's largest value to 2^14 .. 2^15, so that f16 parts hold the others against it
      float big = 0.0f;
#pragma unroll
      for (int s = 0; s < NX; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) big = fmaxf(big, fabsf(x[s][c]));
      big = head_max(big);
      if (big > 0.0f && big < INFINITY) {
        const int e = max((int)(__float_as_uint(big) >> 23) - 127, -100);
        lift = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        unlift = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      }
    }
    if constexpr (CT != F32)
#pragma unroll
      for (int s = 0; s < NQ; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4 y = x[2 * s + c / 2];
          uint32_t u, v, w;
          split2<HALF>(y[2 * (c % 2)] * lift, y[2 * (c % 2) + 1] * lift, &u, &v, &w);
          qa[s][c] = u, qb[s][c] = v, qc[s][c] = w;
        }

    // keys are requested a step ahead while the weights and values are worked on, values while the scores are
    int step = 0;
    for (; base_of(step + 1) < end; ++step) {
      score();
      at = place(step + 1, next);
      load_k(at);
      next = look(step + 2);
      gather(base_of(step));
      load_v(at);
    }
    score();
    gather(base_of(step));
  }
  l = head_sum(l);
  if (__any(bad != kGood)) {
    if constexpr (SHARE) {
#pragma unroll
      for (int c = 32; c; c /= 2) bad = min(bad, __shfl_xor(bad, c));
    }
    if (!SHARE || bad < my_len) l = NAN;
  }

  // ---- the waves' sums joined, 128 dimensions at a time
  asm volatile("" : "+v"(col), "+v"(quad));
  constexpr int PASS = HDP > 128 ? 2 : 1, VP = VE / PASS;
  __shared__ float o_s[kWaves][16 * VP][17], m_s[kWaves][16], l_s[kWaves][16];
  if (quad == 0) m_s[wave][col] = m, l_s[wave][col] = l;
  __syncthreads();
  float top = m_s[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_s[w][col]);
  const float from = top == -INFINITY ? 0.0f : top;
  const float mine = exp2_hw(m - from);
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += l_s[w][col] * exp2_hw(m_s[w][col] - from);
  // a row that goes on in other pieces leaves its part
  const RowParts parts = parts_of(pc.at, units, pc.per);
  const bool cut = L.pieces && parts.count > 1;
  const size_t part = (size_t)part_place(block - (unit0 != 0), unit0 != 0);
  __shared__ float div_s[16];
  if (wave == 0 && quad == 0) {
    div_s[col] = sum == 0.0f ? 0.0f : vs / sum;
    if (cut && col < heads) {
      float* ml = L.part_ml + ((SHARE ? part * L.share + run_row : part) * a.n_q + head0 + col - run_row * G) * 2;
      ml[0] = top;
      ml[1] = sum;
    }
    if (heads_at == 0 && col < run.n) {
      const int row = pc.row + col;
      const bool last = pc.end >= pc.at + units;
      if (cut) {
        if (L.by_row ? unit0 == 0 : last) L.joins[L.by_row ? row : block * L.share + col] = int4{row, parts.count, parts.first, col};
      } else if (L.by_row && unit0 == 0) {
        L.joins[row] = int4{0, 0, 0, 0};
      }
    }
  }
#pragma unroll
  for (int ps = 0; ps < PASS; ++ps) {
#pragma unroll
    for (int c = 0; c < VP; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_s[wave][(4 * quad + i) * VP + c][col] = o[ps * VP + c][i] * mine;
    __syncthreads();
    for (int x = threadIdx.x; x < heads * 16 * VP; x += kThreads) {
      const int h = x / (16 * VP), at = x % (16 * VP), c = ps * VP + at % VP;
      const int d = c / EV * 16 * EV + at / VP * EV + c % EV;
      if (d >= hd) continue;
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) y += o_s[w][at][h];
      const int of = SHARE ? (int)divide((uint32_t)h, L.by_group) : 0, head = head0 + h - of * G;
      if (cut) {
        L.part_o[((SHARE ? part * L.share + of : part) * a.n_q + head) * hd + d] = y;
      } else {
        a.out[(size_t)(pc.row + of) * a.ldo + (size_t)head * hd + d] = y * div_s[h];
      }
    }
    if (ps + 1 < PASS) __syncthreads();
  }

  pc.at += SHARE ? units + kRunUnits : units;
  if (pc.at >= pc.end) return;
  if constexpr (SHARE) {
    if ((pc.row += run.n) >= row_end) return;
    continue;
  }
  pc.row = row2, pc.req = req2, pc.len = length_of(g, req2, pos2);
  while (units_of(pc.len) == 0) {   // rows of no request between
    ++pc.row;
    pc.req = a.req ? scalar_load(a.req, pc.row) : pc.row;
    pc.len = length_of(g, pc.req, scalar_load(a.pos, pc.row));
  }
  }
}

// A block a (cut row, query head, `slice` dimensions): its parts joined, four dimensions a thread, so that WAVES 64 /
// (slice / 4) parts are read side by side.  Latency: the parts' first rows are requested with their maxima.
template <int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void paged_join_kernel(AttnLaunch L, int slice) {
  constexpr int N = WAVES * kWave, U = 4;
  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  const int head = (int)blockIdx.y, hd = g.map.head_dim;
  const int4 r = L.joins[blockIdx.x];   // row, parts, first piece, place in its run
  const int parts = r.y;
  if (!join_ok(r.x, r.y, r.z, r.w, a.T, L.pieces, L.share)) return;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int width = slice / 4, rows = N / width, row = tid / width, d = (int)blockIdx.z * slice + tid % width * 4;
  __shared__ float by_s[WAVES][kMaxParts];
  __shared__ f32x4 acc_s[N];
  const float* ml = L.part_ml + ((size_t)r.w * a.n_q + head) * 2;
  const float* o = L.part_o + ((size_t)r.w * a.n_q + head) * hd + d;
  const size_t step = (size_t)L.share * a.n_q * 2, next = (size_t)L.share * a.n_q * hd;
  f32x4 y[U];
#pragma unroll
  for (int c = 0; c < U; ++c) {
    const int i = row + c * rows;
    y[c] = *(const f32x4*)(o + part_place(r.z, i < parts ? i : 0) * next);
  }
  // what each part counts for; every wave for itself, the first 64 parts' numbers kept between the two passes
  const float* mine = ml + part_place(r.z, min(lane, parts - 1)) * step;
  const float m0 = mine[0], l0 = mine[1];
  float top = m0, sum = 0.0f;
  for (int i = lane + kWave; i < parts; i += kWave) top = fmaxf(top, ml[part_place(r.z, i) * step]);
#pragma unroll
  for (int c = 32; c; c /= 2) top = fmaxf(top, __shfl_xor(top, c));
  if (top == -INFINITY) top = 0.0f;
  if (lane < parts) {
    by_s[wave][lane] = exp2_hw(m0 - top);
    sum = l0 * exp2_hw(m0 - top);
  }
  for (int i = lane + kWave; i < parts; i += kWave) {
    const float* p = ml + part_place(r.z, i) * step;
    const float f = exp2_hw(p[0] - top);
    by_s[wave][i] = f;
    sum += p[1] * f;
  }
  sum = wave_total(sum);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < rows) {
#pragma unroll
    for (int c = 0; c < U; ++c)
      if (row + c * rows < parts) acc += y[c] * by_s[wave][row + c * rows];
    int i = row + U * rows;
    for (; i + (U - 1) * rows < parts; i += U * rows) {
#pragma unroll
      for (int c = 0; c < U; ++c) y[c] = *(const f32x4*)(o + part_place(r.z, i + c * rows) * next);
#pragma unroll
      for (int c = 0; c < U; ++c) acc += y[c] * by_s[wave][i + c * rows];
    }
    for (; i < parts; i += rows) acc += *(const f32x4*)(o + part_place(r.z, i) * next) * by_s[wave][i];
  }
  acc_s[tid] = acc;
  __syncthreads();
  if (row == 0) {
    for (int i = 1; i < rows && i < parts; ++i) acc += acc_s[i * width + tid];
    const float vs = g.v_scale ? g.v_scale[head / (a.n_q / g.map.n_kv)] : 1.0f;
    float* out = a.out + (size_t)r.x * a.ldo + (size_t)head * hd + d;
#pragma unroll
    for (int c = 0; c < 4; ++c) out[c] = sum == 0.0f ? 0.0f : acc[c] / sum * vs;
  }
}

template <int CT, int HDP>
hipError_t launch(const AttnLaunch& L, bool whole, bool stream, dim3 grid, hipStream_t s) {
  using std::false_type;
  using std::true_type;
  auto go = [&](auto w, auto n, auto r) {
    hipLaunchKernelGGL((paged_attn_kernel<CT, HDP, decltype(w)::value, decltype(n)::value, decltype(r)::value>), grid, dim3(kThreads), 0, s, L);
  };
  if (L.share > 1 && whole) go(true_type{}, false_type{}, true_type{});
  else if (L.share > 1) go(false_type{}, false_type{}, true_type{});
  else if (whole && stream) go(true_type{}, true_type{}, false_type{});
  else if (whole) go(true_type{}, false_type{}, false_type{});
  else if (stream) go(false_type{}, true_type{}, false_type{});
  else go(false_type{}, false_type{}, false_type{});
  return hipGetLastError();
}

template <int CT>
hipError_t launch(const AttnLaunch& L, bool whole, bool stream, dim3 grid, hipStream_t s) {
  const int hd = L.g.map.head_dim;
  return hd <= 64    ? launch<CT, 64>(L, whole, stream, grid, s)
         : hd <= 128 ? launch<CT, 128>(L, whole, stream, grid, s)
                     : launch<CT, 256>(L, whole, stream, grid, s);
}

}  // namespace

size_t paged_attn_work(int T, int n_q, int n_kv, int head_dim) {
  const size_t pieces = (size_t)pieces_for(n_q, n_kv, head_dim), rows = (size_t)rows_shared(n_q, n_kv);
  return ((size_t)T <= pieces ? T : pieces * rows) * sizeof(int4) + 2 * pieces * rows * n_q * (2 + (size_t)head_dim) * 4 + 16;
}

hipError_t launch_paged_attn(const AttnPages& p, int dtype, hipStream_t s) {
  const moe_paged_attn& a = p.a;
  const PageMap& map = p.map;
  AttnLaunch L;
  L.g = p;
  L.head_tiles = (a.n_q / map.n_kv + 15) / 16;
  const AttnCut cut = cut_rows(a.T, a.n_req, a.req, (long long)a.max_pages * map.page_size, a.n_q, map.n_kv, map.head_dim);
  L.share = cut.share;
  L.by_share = make_divider((uint32_t)L.share);
  L.by_group = make_divider((uint32_t)(a.n_q / map.n_kv));
  L.pieces = cut.pieces;
  L.each = make_divider((uint32_t)cut.most);
  L.by_row = cut.by_row;
  L.joins = (int4*)a.work;
  L.part_o = (float*)(L.joins + (L.by_row ? a.T : (size_t)cut.most * L.share));
  L.part_ml = L.part_o + 2 * (size_t)cut.most * L.share * a.n_q * map.head_dim;
  const dim3 grid((unsigned)cut.blocks, (unsigned)(map.n_kv * L.head_tiles));
  const bool whole = map.page_size % 16 == 0 && map.slot_stride < (1 << 22);
  const int size = dtype == F32 ? 4 : dtype == E4M3 ? 1 : 2;
  const bool stream = (long long)map.n_pages * map.page_stride * size >= kStreamBytes;
  const hipError_t e = dtype == F32    ? launch<F32>(L, whole, stream, grid, s)
                       : dtype == F16  ? launch<F16>(L, whole, stream, grid, s)
                       : dtype == BF16 ? launch<BF16>(L, whole, stream, grid, s)
                                       : launch<E4M3>(L, whole, stream, grid, s);
  if (e != hipSuccess || !L.pieces) return e;
  // few rows may have many parts each: four waves to 16 rows (one row of 16000 15.2 us, 16.7 with one wave; 64 rows 34.7
  // with four, 33.6 with one), and slices of the dimensions to 4 rows (15.7 against 17.3 whole)
  const int slice = a.T > 4 ? map.head_dim : map.head_dim % 32 ? 16 : 32;
  const dim3 joins(L.by_row ? (unsigned)a.T : grid.x * L.share, (unsigned)a.n_q, (unsigned)(map.head_dim / slice));
  if (a.T <= 16) hipLaunchKernelGGL(paged_join_kernel<4>, joins, dim3(4 * kWave), 0, s, L, slice);
  else hipLaunchKernelGGL(paged_join_kernel<1>, joins, dim3(kWave), 0, s, L, slice);
  return hipGetLastError();
}

}  // namespace moe
