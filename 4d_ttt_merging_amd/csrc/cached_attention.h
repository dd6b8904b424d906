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

#include <type_traits>

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
  float lazy;                 // kLazy / scale
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

__device__ __forceinline__ int wave_max(int v) {
  // (a lane without another sees zero there, or its own)
  const auto step = [&](auto at, auto rows) {
    v = max(v, static_cast<int>(__builtin_amdgcn_update_dpp(v, v, decltype(at)::value, decltype(rows)::value, 0xF, false)));
  };
  using All = std::integral_constant<int, 0xF>;
  step(std::integral_constant<int, 0x111>(), All());
  step(std::integral_constant<int, 0x112>(), All());
  step(std::integral_constant<int, 0x114>(), All());
  step(std::integral_constant<int, 0x118>(), All());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xA>());
  step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xC>());
  return __builtin_amdgcn_readlane(v, 63);
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
  return max(1, (rows + a.tile_rows - 1) >> __builtin_ctz(a.tile_rows));
}
// Few queries: the shortest pieces of which no more than `slots` beside one a sequence are needed, or nearly so.
__device__ __forceinline__ Pieces few_pieces(const Attend& a) {
  const bool here = lane_id() < a.batch;
  Pieces p{here ? length_of(a, lane_id()) : 0, INT32_MAX};
  if (a.slots == 0) return p;
  const auto over_all = [&](auto of) {  // at most 2^25 a lane, so that 64 of them fit
    int64_t sum = here ? of(p.mine) : 0;
    for (int64_t b = lane_id() + 64; b < a.batch; b += 64) sum += of(length_of(a, b));
    return static_cast<int64_t>(wave_sum(static_cast<uint32_t>(min(sum, int64_t{1} << 25))));
  };
  const int most = a.slots + static_cast<int>(a.batch);
  const auto rounded = [&](int64_t units) {  // of 64 tokens
    return static_cast<int>(min(max(units * 64, static_cast<int64_t>(a.least)), static_cast<int64_t>(INT32_MAX)));
  };
  const int64_t sum = over_all([](int length) { return (static_cast<int64_t>(length) + 63) / 64; });
  // (more than the sums hold: a piece a sequence)
  if (sum >= int64_t{1} << 25) return p;
  p.tokens = rounded((sum + most - 1) / most);
  for (int round = 0; round < 4; ++round) {
    const int tokens = p.tokens;
    const int64_t n = over_all([&](int length) { return static_cast<int64_t>(pieces_of(length, tokens)); });
    if (n <= most) return p;
    p.tokens = rounded(p.tokens / 64 * n / most + 1);
  }
  // (at most one more a sequence than all the tokens / tokens)
  p.tokens = rounded((sum + a.slots - 1) / a.slots);
  return p;
}

// x / y of numbers from 0 to 2^30, if less than 2^20 (more is then nearly right).
__device__ __forceinline__ int quotient(int x, int y) {
  const int q = static_cast<int>(static_cast<float>(x) * __builtin_amdgcn_rcpf(static_cast<float>(y)));
  const int64_t left = x - static_cast<int64_t>(q) * y;
  return left < 0 ? q - 1 : left >= y ? q + 1 : q;
}

// Many queries: the length of pieces that costs least, in tokens of a tile: rounds of work-groups that have queries, each a
// piece and what it begins and ends with; and what they leave to the join, for as many as the chip holds.  Lengths are
// parts of the longest sequence.  (The sequences differ in queries and lengths, and a ragged last round idles most
// of the chip: one or two full rounds by the sums alone took, of calls with 2 or 3 ragged causal sequences, 4% longer in bf16 and
// 9% in fp32; 2 x 2,300 queries over 16,464 tokens of 128 channels, 288 work-groups of which 256 fit, whole 901 us, so 649.
// kRound, kJoin of 64 to 512, 300 to 1,200: within 2% up to 192, 450.)
constexpr float kRound = 192.0f, kJoin = 300.0f;
__device__ __forceinline__ Pieces many_pieces(const Attend& a) {
  const int lane = lane_id();
  Pieces p{lane < a.batch ? length_of(a, lane) : 0, INT32_MAX};
  if (a.slots == 0) return p;
  // Causal prompts, whose tiles see from nothing to everything, fill the chip evenly with the longest first: whole.
  int busy = 0, steep = 0, longest = 0;
  for (int64_t b = lane; b < a.batch; b += 64) {
    const int length = length_of(a, b), tiles = busy_tiles(a, b);
    busy += tiles, longest = max(longest, length);
    if (a.causal && count_of(a, b) > length / 2) steep += tiles;
  }
  busy = static_cast<int>(wave_sum(static_cast<uint32_t>(busy))) * a.pages.kv_heads;
  steep = static_cast<int>(wave_sum(static_cast<uint32_t>(steep))) * a.pages.kv_heads;
  longest = wave_max(longest);
  if (2 * static_cast<int64_t>(steep) > busy && 10 * static_cast<int64_t>(busy) >= 9 * static_cast<int64_t>(a.held)) return p;
  const int64_t most = a.slots + a.batch;
  const auto cost = [&](int tokens, int64_t n, int64_t tiles) {
    const int groups = static_cast<int>(min(tiles * a.pages.kv_heads, int64_t{1} << 29));  // (the grid holds fewer than 2^23)
    const int rounds = quotient(groups + a.held - 1, a.held);
    const float join = tokens < longest ? kJoin * static_cast<float>(groups) / static_cast<float>(a.held) : 0.0f;
    return n > most ? INFINITY : static_cast<float>(rounds) * (static_cast<float>(tokens) + kRound) + join;
  };
  const auto part = [&](int parts) { return max((quotient(longest, parts) + 64) & ~63, a.least); };
  int taken = longest;
  if (a.batch <= 64) {
    // A lane looks at one: 1 .. 32 parts, then eight a doubling.
    const int tokens = part(lane < 32 ? lane + 1 : static_cast<int>(32.0f * __builtin_amdgcn_exp2f((lane - 31) * 0.125f)));
    const int mine = lane < a.batch ? busy_tiles(a, lane) : 0;
    int n = 0, tiles = 0;
    for (int b = 0; b < a.batch; ++b) {
      const int one = quotient(max(0, __builtin_amdgcn_readlane(p.mine, b) - 1), tokens) + 1;
      n += one, tiles += one * __builtin_amdgcn_readlane(mine, b);
    }
    const int order = -static_cast<int>(__float_as_uint(cost(tokens, n, tiles)));
    const uint64_t best = __ballot(order == wave_max(order));
    taken = __builtin_amdgcn_readlane(tokens, __ffsll(static_cast<unsigned long long>(best)) - 1);
  } else {
    // One after the other, a lane a sequence: 1 .. 4 parts, then two a doubling.  (500 sequences of up to 80 queries over
    // 1,000 tokens, a lane a length 250 us, so 120.)
    float least_cost = INFINITY;
    for (int c = 0; c < 16; ++c) {
      const int tokens = part(c < 4 ? c + 1 : (c & 1 ? 4 : 3) << ((c - 2) / 2));
      int n = 0, tiles = 0;
      for (int64_t b = lane; b < a.batch; b += 64) {
        const int one = quotient(max(0, length_of(a, b) - 1), tokens) + 1;
        n += one, tiles += one * busy_tiles(a, b);
      }
      const float mine = cost(tokens, wave_sum(static_cast<uint32_t>(n)), wave_sum(static_cast<uint32_t>(tiles)));
      if (mine < least_cost) least_cost = mine, taken = tokens;
    }
  }
  if (taken < longest) p.tokens = taken;
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

// A row's reference maximum moves where a score passes it by more than this, in powers of two.
constexpr float kLazy = 8.0f;

// Exponents are z scale - reference in one instruction, whose product is not rounded while the reference's was: they are off by
// its rounding, the same for all of a row, which normalising takes out.  From references of this size on, where that could
// pass what an exponential holds (a row of a type's lowest values, say), the difference is taken before the scale.  Whether a
// reference moves always goes by the difference before the scale: of neighbouring fp32 scores past 2^27 the products
// with it may be one number, and the larger one's exponential past every number.
constexpr float kFar = 0x1p20f;
// What sums are multiplied by where a row's reference moves.
__device__ __forceinline__ float shrink_of(float from, float to, float scale) {
  const float top = to * scale;
  return top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(fabsf(top) > kFar ? (from - to) * scale : from * scale - top);
}

// A mass as the kernels take it: a type's lowest value is a number, and with the scales that are allowed it stays one.  (NaN is
// neither below nor above.)
constexpr float kMostMass = 1e30f;
__device__ __forceinline__ float mass_of(float mass) {
  return mass < -kMostMass ? (mass == -INFINITY ? mass : -kMostMass) : mass > kMostMass ? kMostMass : mass;
}

// A channel of a query, infinities as NaN: such a query's scores are infinite or NaN, all of them, and NaN is what its row is.
__device__ __forceinline__ float channel_of(float x) { return fmaf(x, 0.0f, x); }

// Whether a row attends to nothing: no score has moved its maximum, and it has no sum either.  (Scores of NaN do not move the
// maximum, but they are in the sum.)
__device__ __forceinline__ bool sees_nothing(float top, float sum) { return top == -INFINITY && sum == 0.0f; }

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
// Those with the bits of `out`, one a token, as zero: what a mass of -infinity keeps out may be anything, too.
__device__ __forceinline__ uint2 scales_without(uint2 s, uint32_t out) {
  const auto bytes = [](uint32_t four) { return (((four & 15) * 0x00204081u) & 0x01010101u) * 0xffu; };
  return {s.x & ~bytes(out), s.y & ~bytes(out >> 4)};
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
// (48 and 64 rows of 8 x 16,384 tokens take the many's kernel 8 to 50% longer, 96 and 128 the few's 5 to 40%.)
constexpr int kFewRows = 64, kFewTile = 16;
int launch_few(const Attend& a, int64_t pieces, int head_dim, int dtype, hipStream_t s);
struct ManyShape {
  int tile_rows, resident;  // rows of a work-group, work-groups that a CU holds
};
template <typename T>
ManyShape many_shape(int head_dim, bool causal, int64_t group);
template <typename T>
int launch_many(const Attend& a, int64_t pieces, int head_dim, hipStream_t s);

}  // namespace paged
}  // namespace vgo
