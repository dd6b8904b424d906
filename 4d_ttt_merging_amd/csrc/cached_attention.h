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
// each work-group cuts the sequences' tokens into pieces of one length (split_of): about slots of
// them in all, at least one a sequence, whatever the lengths are.  Sequences of one piece are written at once, the
// others' pieces leave their sums in the workspace for merge_kernel.
#pragma once

#include "paged_cache.h"

namespace vgo {
namespace paged {

struct Attend {
  Pages pages;
  const void* q;
  void* out;
  float* sums;   // [piece][key head][row tile][rows of a tile] of D sums of values, then as many (maximum, sum) pairs
  float2* ends;
  int64_t q_stride[3], out_stride[3];
  const int32_t* lengths;
  const int32_t* counts;
  int64_t batch;
  int32_t n_query, heads, group;
  int32_t tiles, tile_rows;   // row tiles of a key head, rows of one
  int32_t slots, least;       // pieces beside one a sequence (0: no splitting), tokens of a piece at least
  int32_t causal;
  float scale;                // times log2(e)
};

__device__ __forceinline__ int64_t capacity_of(const Attend& a) { return a.pages.width << a.pages.shift; }
__device__ __forceinline__ int length_of(const Attend& a, int64_t b) {
  return static_cast<int>(min(max(static_cast<int64_t>(a.lengths[b]), int64_t{0}), capacity_of(a)));
}
__device__ __forceinline__ int count_of(const Attend& a, int64_t b) {
  return a.counts ? min(max(a.counts[b], 0), a.n_query) : a.n_query;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Tokens of a piece: a multiple of 64.
__device__ __forceinline__ int piece_tokens(const Attend& a) {
  if (a.slots == 0) return INT32_MAX;
  int64_t sum = 0;
  for (int64_t b = lane_id(); b < a.batch; b += 64) sum += length_of(a, b);
  sum = wave_sum(sum);
  const int64_t each = (sum + a.slots - 1) / a.slots;
  return static_cast<int>(max((each + 63) / 64 * 64, static_cast<int64_t>(a.least)));
}
__device__ __forceinline__ int pieces_of(int length, int tokens) {
  return tokens == INT32_MAX ? 1 : max(1, (length + tokens - 1) / tokens);
}

struct Piece {
  int64_t b;           // -1: there is no such piece
  int begin, end;      // its tokens
  int length;          // of the sequence
  bool whole;          // the only one of its sequence
};

// Piece x of all sequences' pieces in a row.  All lanes of a wave together; the same in each.
__device__ __forceinline__ Piece piece_of(const Attend& a, int64_t x) {
  const int tokens = piece_tokens(a);
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < a.batch; b0 += 64) {
    const int64_t b = b0 + lane_id();
    const int length = b < a.batch ? length_of(a, b) : 0;
    const int n = b < a.batch ? pieces_of(length, tokens) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int other = __shfl_up(upto, o);
      if (lane_id() >= o) upto += other;
    }
    const uint64_t past = __ballot(x < before + upto);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      const int mine = static_cast<int>(x - before) - (__shfl(upto, at) - __shfl(n, at));
      Piece p;
      p.b = b0 + __builtin_amdgcn_readfirstlane(at);
      p.length = __builtin_amdgcn_readfirstlane(__shfl(length, at));
      const int begin = __builtin_amdgcn_readfirstlane(mine) * (tokens == INT32_MAX ? 0 : tokens);
      p.begin = begin;
      p.end = tokens == INT32_MAX ? p.length : min(p.length, begin + min(tokens, INT32_MAX - begin));
      p.whole = __builtin_amdgcn_readfirstlane(__shfl(n, at)) == 1;
      return p;
    }
    before += __shfl(upto, 63);
  }
  return {-1, 0, 0, 0, true};
}

// bf16 terms that a query, and a probability, is split into.
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
  uint32_t w[4];
  bf16x2 p[4];
};

// Eight channels of a key: a word of codes, one scale.
__device__ __forceinline__ bf16x8 key_operand(uint32_t word, float scale) {
  Operand o;
  o.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
  o.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
  o.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
  o.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
  return o.v;
}
// A channel pair of eight tokens, a scale each: the even channel's operand and the odd one's.
__device__ __forceinline__ void value_operands(uint2 codes, uint2 scales, bf16x8& even, bf16x8& odd) {
  const auto at = [](uint32_t word, uint32_t scale, auto i) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale_of<decltype(i)::value>(scale),
                                                                                 decltype(i)::value));
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  const uint32_t t[8] = {at(codes.x, scales.x, I0()), at(codes.x, scales.x, I1()), at(codes.x, scales.x, I2()),
                         at(codes.x, scales.x, I3()), at(codes.y, scales.y, I0()), at(codes.y, scales.y, I1()),
                         at(codes.y, scales.y, I2()), at(codes.y, scales.y, I3())};
  Operand e, o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.w[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100);
    o.w[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302);
  }
  even = e.v, odd = o.v;
}
// Scale bytes of eight tokens with those from `valid` on as zero: what lies past a length may be anything, and a scale of
// 255 would make a probability of zero NaN.
__device__ __forceinline__ uint2 kept_scales(uint2 s, int valid) {
  const uint64_t keep = valid >= 8 ? ~uint64_t{0} : valid <= 0 ? 0 : (uint64_t{1} << (8 * valid)) - 1;
  return {s.x & static_cast<uint32_t>(keep), s.y & static_cast<uint32_t>(keep >> 32)};
}
// x as kTerms bf16 terms, the first ones rounded to nearest: exact but for what the last one leaves.
template <int kTerms>
__device__ __forceinline__ void split(float x, bf16_t (&t)[kTerms]) {
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    t[i] = static_cast<bf16_t>(x);
    x -= static_cast<float>(t[i]);
  }
}

int launch_few(const Attend& a, int64_t pieces, int head_dim, int dtype, hipStream_t s);
int few_rows(int64_t rows);  // rows of a tile

}  // namespace paged
}  // namespace vgo
