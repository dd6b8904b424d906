// Attention over the paged cache (paged_cache.h): what its kernels share.
//
// A code times its scale is exact in bf16, so keys and values enter the matrix instructions without a rounding, and
// precision is in how many bf16 terms a query or a probability is split into: bf16 queries are one term,
// f16 ones two and fp32 ones three (8 + 8 + 8 bits), exactly.
//
// Rows: the `group` heads that share a key head stand together, row r of a key head being token r / group of head
// r % group, so that a tile of keys serves them all.
//
// Work split over the keys: the host does not know the lengths, so the grid holds `slots` pieces more than sequences, and
// each work-group cuts the sequences' tokens into pieces of one length, which the grid holds whatever the lengths
// are.  Tiles of rows that see one piece alone are written at once, the others' pieces leave their sums in the workspace
// for a join.
#pragma once

#include "paged_cache.h"

namespace vgo {
namespace paged {

typedef __attribute__((__vector_size__(16))) uint32_t u32x4;

struct Attend {
  Pages pages;
  const void* q;
  void* out;
  float* sums;   // [piece][key head][row tile][rows of a tile] of D sums of values, then as many (maximum, sum) pairs
  float2* ends;
  int2* firsts;  // [batch]: a sequence's first piece, tokens of a piece
  int64_t q_stride[3], out_stride[3];
  const int32_t* lengths;
  const int32_t* counts;
  int64_t batch;
  int32_t n_query, group;
  int32_t first_row, last_row;  // the rows of this launch: from .. to before
  int32_t tiles, tile_rows;   // row tiles of a key head, rows of one
  int32_t slots, least;       // pieces beside one a sequence (0: no splitting), tokens of a piece at least
  int32_t held;               // work-groups that the chip holds at once
  int32_t causal;
  float scale, per_scale;     // times log2(e); 1 / the scale itself
};

__device__ __forceinline__ int64_t capacity_of(const Attend& a) { return a.pages.width << a.pages.shift; }
__device__ __forceinline__ int length_of(const Attend& a, int64_t b) {
  return static_cast<int>(min(max(static_cast<int64_t>(a.lengths[b]), int64_t{0}), capacity_of(a)));
}
__device__ __forceinline__ int count_of(const Attend& a, int64_t b) {
  return a.counts ? min(max(a.counts[b], 0), a.n_query) : a.n_query;
}

// Where a sequence's first query stands.  (Past every table: seen from there all is earlier, and sums of places fit 32 bits.)
__device__ __forceinline__ int first_place(const Attend& a, int64_t b, int count) {
  return min(max(a.lengths[b], 0), 1 << 30) - count;
}

// Reductions over a wave stay in the vector unit (a shuffle through LDS takes a hundred cycles, and a step of a short
// sequence is little else).  Their results are said to be the wave's, so that what follows from them is scalar: a page
// looked up by vector loads waits for all that are on their way.
template <int kCtrl, int kRows = 0xF>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xF, false));
}
// Sums over the lanes up to each (row_shr 1, 2, 4, 8 within 16 lanes, then their last lanes' to the rows behind).
__device__ __forceinline__ uint32_t sums_upto(uint32_t v) {
  v += moved<0x111>(v);
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<0x142, 0xA>(v);
  v += moved<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  return __builtin_amdgcn_readlane(static_cast<int>(sums_upto(v)), 63);
}

__device__ __forceinline__ int pieces_of(int length, int tokens) { return max(1, (length - 1) / tokens + 1); }

// The sequences' pieces, as every work-group reckons them: all lanes of a wave together, the same in each.
struct Pieces {
  int mine;    // length of sequence `lane`, of the first 64
  int tokens;  // of a piece: a multiple of 64
};
// Row tiles of a sequence that have queries (one at least).
__device__ __forceinline__ int busy_tiles(const Attend& a, int64_t b) {
  const int rows = min(count_of(a, b) * a.group, a.last_row) - a.first_row;
  return max(1, (rows + a.tile_rows - 1) / a.tile_rows);
}
// The shortest pieces of which no more than `slots` beside one a sequence are needed, or nearly so, and (kMany), since
// sequences differ in queries too, whose work-groups that have queries fill the chip about once, or twice where a single
// round would leave it ragged (2 x 2,058 queries at most over 16,464 tokens of 128 channels, both ragged: one round 282 us, so 242).
template <bool kMany>
__device__ __forceinline__ Pieces pieces(const Attend& a) {
  const bool here = lane_id() < a.batch;
  Pieces p{here ? length_of(a, lane_id()) : 0, INT32_MAX};
  if (a.slots == 0) return p;
  const int weight = kMany && here ? busy_tiles(a, lane_id()) : 1;
  const auto over_all = [&](auto of) {  // at most 2^25 a lane, so that 64 of them fit
    int64_t sum = here ? of(p.mine, weight) : 0;
    for (int64_t b = lane_id() + 64; b < a.batch; b += 64) sum += of(length_of(a, b), kMany ? busy_tiles(a, b) : 1);
    return static_cast<int64_t>(wave_sum(static_cast<uint32_t>(min(sum, int64_t{1} << 25))));
  };
  const int most = a.slots + static_cast<int>(a.batch);
  const auto rounded = [&](int64_t units) {  // of 64 tokens
    return static_cast<int>(min(max(units * 64, static_cast<int64_t>(a.least)), static_cast<int64_t>(INT32_MAX)));
  };
  int64_t target = most;
  if constexpr (kMany) {
    const int64_t busy = over_all([&](int, int w) { return static_cast<int64_t>(w) * a.pages.kv_heads; });
    if (10 * busy >= 9 * static_cast<int64_t>(a.held)) return p;
    target = 100 * (a.held / busy * busy) >= 85 * static_cast<int64_t>(a.held) ? a.held : 2 * a.held;
  }
  const int each = kMany ? a.pages.kv_heads : 1;
  const int64_t sum = over_all([&](int length, int w) { return (static_cast<int64_t>(length) + 63) / 64 * w * each; });
  // (more than the sums hold: a piece a sequence)
  if (sum >= int64_t{1} << 25) return p;
  p.tokens = rounded((sum + target - 1) / target);
  for (int round = 0; round < 4; ++round) {
    const int tokens = p.tokens;
    const int64_t n = over_all([&](int length, int) { return static_cast<int64_t>(pieces_of(length, tokens)); });
    int64_t groups = n;
    if constexpr (kMany) groups = over_all([&](int length, int w) { return static_cast<int64_t>(pieces_of(length, tokens)) * w * each; });
    if (n <= most && (groups <= target || round == 3)) return p;
    const int64_t by_n = p.tokens / 64 * n / most + 1, by_groups = p.tokens / 64 * groups / target + 1;
    p.tokens = rounded(max(n > most ? by_n : 0, by_groups));
  }
  // (at most one more a sequence than all the tokens / tokens)
  const int64_t all = kMany ? over_all([](int length, int) { return (static_cast<int64_t>(length) + 63) / 64; }) : sum;
  p.tokens = rounded((all + a.slots - 1) / a.slots);
  return p;
}

struct Piece {
  int64_t b;           // -1: there is no such piece
  int begin, end;      // its tokens
  int length;          // of the sequence
  int tokens;          // of a piece
};

// Pieces of all sequences together.
__device__ __forceinline__ int pieces_in_all(const Attend& a, const Pieces& all) {
  int n = lane_id() < a.batch ? pieces_of(all.mine, all.tokens) : 0;
  for (int64_t b = lane_id() + 64; b < a.batch; b += 64) n += pieces_of(length_of(a, b), all.tokens);
  return static_cast<int>(wave_sum(static_cast<uint32_t>(n)));
}
// Piece x of all sequences' pieces in a row.
__device__ __forceinline__ Piece piece_of(const Attend& a, const Pieces& all, int x) {
  int before = 0;
  for (int64_t b0 = 0; b0 < a.batch; b0 += 64) {
    const int64_t b = b0 + lane_id();
    const int length = b0 == 0 ? all.mine : b < a.batch ? length_of(a, b) : 0;
    const int n = b < a.batch ? pieces_of(length, all.tokens) : 0;
    const int upto = static_cast<int>(sums_upto(static_cast<uint32_t>(n)));
    const uint64_t past = __ballot(x < before + upto);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      const int mine = x - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
      Piece p;
      p.b = b0 + at;
      p.length = __builtin_amdgcn_readlane(length, at);
      p.begin = mine == 0 ? 0 : mine * all.tokens;
      p.end = min(p.length, p.begin + min(all.tokens, INT32_MAX - p.begin));
      p.tokens = all.tokens;
      return p;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0, 0};
}
// What the join asks of a sequence: its first piece and their length, left by that piece.
__device__ __forceinline__ void leave(const Attend& a, const Piece& piece, int x, bool one) {
  if (a.slots > 0 && piece.begin == 0 && one) a.firsts[piece.b] = {x, piece.tokens};
}

// Tokens that any row of the tile at row `row0` sees: from 0 to before this one.
__device__ __forceinline__ int stop_of(const Attend& a, int length, int count, int place0, int row0) {
  const int last = min(min(row0 + a.tile_rows, a.last_row), count * a.group) - 1;
  return last < row0 ? 0 : a.causal ? max(0, min(length, place0 + last / a.group + 1)) : length;
}

// Exponents are z scale - reference in one instruction, whose product is not rounded while the reference's was: they are off by
// its rounding, the same for all of a row, which normalising takes out.  From references of this size on, where that could
// pass what an exponential holds (a row of a type's lowest values, say), the difference is taken before the scale.
constexpr float kFar = 0x1p20f;

// A mass as the kernels take it: a type's lowest value is a number, and with the scales that are allowed it stays one.
__device__ __forceinline__ float mass_of(float mass) {
  return mass == -INFINITY ? mass : fminf(fmaxf(mass, -1e30f), 1e30f);
}

// bf16 terms that a query, and a probability, is split into (many bf16 queries: one each, see ManyTerms).
template <typename T>
struct Terms;
template <>
struct Terms<bf16_t> {
  static constexpr int kQuery = 1, kWeight = 2;
};
template <>
struct Terms<f16_t> {
  static constexpr int kQuery = 2, kWeight = 2;
};
template <>
struct Terms<float> {
  static constexpr int kQuery = 3, kWeight = 3;
};

union Operand {
  bf16x8 v;
  u32x4 u;
  uint32_t w[4];
};

// Two numbers of byte kAt of a word, as bf16 or f16.
template <bool kHalf, int kAt>
__device__ __forceinline__ uint32_t two_of(uint32_t word, float scale) {
  if constexpr (kHalf) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, kAt));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, kAt));
}
// Eight channels of a key: a word of codes, one scale.
template <bool kHalf = false>
__device__ __forceinline__ u32x4 key_operand(uint32_t word, float scale) {
  return u32x4{two_of<kHalf, 0>(word, scale), two_of<kHalf, 1>(word, scale), two_of<kHalf, 2>(word, scale),
               two_of<kHalf, 3>(word, scale)};
}
// A channel pair of eight tokens, a scale each: the even channel's operand and the odd one's.
template <bool kHalf = false>
__device__ __forceinline__ void value_operands(uint2 codes, uint2 scales, u32x4& even, u32x4& odd) {
  const uint32_t t[8] = {two_of<kHalf, 0>(codes.x, scale_of<0>(scales.x)), two_of<kHalf, 1>(codes.x, scale_of<1>(scales.x)),
                         two_of<kHalf, 2>(codes.x, scale_of<2>(scales.x)), two_of<kHalf, 3>(codes.x, scale_of<3>(scales.x)),
                         two_of<kHalf, 0>(codes.y, scale_of<0>(scales.y)), two_of<kHalf, 1>(codes.y, scale_of<1>(scales.y)),
                         two_of<kHalf, 2>(codes.y, scale_of<2>(scales.y)), two_of<kHalf, 3>(codes.y, scale_of<3>(scales.y))};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    even[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100);
    odd[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302);
  }
}
// Scale bytes of eight tokens with those from `valid` on as zero: what lies past a length may be anything, and a scale of
// 255 would make a probability of zero NaN.
__device__ __forceinline__ uint2 kept_scales(uint2 s, int valid) {
  const uint64_t keep = valid >= 8 ? ~uint64_t{0} : valid <= 0 ? 0 : (uint64_t{1} << (8 * valid)) - 1;
  return {s.x & static_cast<uint32_t>(keep), s.y & static_cast<uint32_t>(keep >> 32)};
}
// x as kTerms terms, the first ones rounded to nearest: exact but for what the last one leaves.
template <int kTerms, typename N>
__device__ __forceinline__ void split(float x, N (&t)[kTerms]) {
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    t[i] = static_cast<N>(x);
    x -= static_cast<float>(t[i]);
  }
}

// The two kernels: few rows beside a key head (cached_attention_few.hip), many (cached_attention_many.h, a file a type).
constexpr int kFewRows = 64;
int few_tile(int64_t rows);  // rows of a tile
int launch_few(const Attend& a, int64_t pieces, int head_dim, int dtype, hipStream_t s);
struct ManyShape {
  int tile_rows, resident;  // rows of a work-group, work-groups that a CU holds
};
template <typename T>
ManyShape many_shape(int head_dim, bool causal);
template <typename T>
int launch_many(const Attend& a, int64_t pieces, int head_dim, hipStream_t s);

}  // namespace paged
}  // namespace vgo
