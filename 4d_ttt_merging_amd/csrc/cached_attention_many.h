// Attention over the paged cache for many queries (chunks and prompts).
//
// kWaves waves of 32 rows each share 64 tokens at a time: the codes come into registers two tiles ahead, are
// converted once for all waves into operands of the 32 x 32 matrix instructions and written to LDS in the order in which
// their lanes read them (16 bytes a lane), double-buffered, one barrier a tile or two:
//   scores^T = K Q^T; row m of a block of 32 tokens holds token 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so
//     that a lane's sixteen scores are two operands of the next product as they stand
//   out^T += V^T P^T, a lane having converted two channels of eight tokens, operands of two tiles
// One reference maximum a row, moved only where a score passes it by 2^8.  (Told to the compiler as seldom: 2% of calls with 128
// channels.)
//
// Bound by matrix and vector instructions in turn: a wave's products wait for its conversions and softmax, which other waves'
// products cover in part (64 channels: MFMA busy 0.40 of the time, VALU 0.62; 128: 0.43, 0.43).  bf16, 16 heads of 8,192 x 8,192:
// 64 channels 301 us, 913 TFLOP/s; 128 494, 1,112; a product of 8,192^3 reaches 1,141.
//
// f16: where a piece's scales let keys and values be f16 numbers, and they nearly always do, the products are f16 ones
// (16 heads, 8,192 x 8,192, 64 channels: two bf16 terms of q and of p 529 us, so 334; 4,096 x 8,192, 128 channels: 419, 282).
// Else, and in fp32, bf16 terms.
#pragma once

#include <type_traits>

#include "cached_attention.h"

namespace vgo {
namespace paged {
namespace {

template <typename T>
struct ManyTerms {
  static constexpr int kQuery = Terms<T>::kQuery, kWeight = Terms<T>::kWeight;
};
template <>
struct ManyTerms<bf16_t> {
  static constexpr int kQuery = 1, kWeight = 1;
};

// sum + x[0] + x[1]
__device__ __forceinline__ float pair_sum(bf16x2 x, float sum) {
  constexpr bf16x2 one = {static_cast<bf16_t>(1.0f), static_cast<bf16_t>(1.0f)};
  return __builtin_amdgcn_fdot2_f32_bf16(x, one, sum, false);
}

// How a type and width are run: waves of a work-group, waves that a SIMD is to hold.  More waves share what is converted and
// read from LDS; fewer (kSharp) leave less idle where a causal tile ends: with few heads beside a key head its rows are many
// tokens.  16 heads, us (in a graph) with 4 waves (2 a SIMD), 4 (3), 8 (2), 8 (4):
//   64 channels, 8,192 x 8,192         bf16  359 359 351 301   f16  386 386 364 334     causal  185 185 191 199   196 196 199 228
//   3 causal prompts over 4 key heads  bf16  148 148 164 135   f16  159 159 172 153     (of 4,096)
//                                            127 127 137 127         139 139 145 143     (of up to 4,116)
//   128 channels, over 8,192           bf16  560     496       f16  320     282         (8,192; 4,096)
//   128, causal, 4,096                 bf16  119     118       f16  127     128
//   fp32  2,048 x 2,048, 64 and 128 channels  72, 112  71, 109;   8 heads of 261 x 1,044  17  20
template <typename T, int D, bool kSharp>
struct Many {
  static constexpr bool kFull = std::is_same_v<T, float>;
  static constexpr int kWaves = kSharp || (D == 64 && kFull) ? 4 : 8, kResident = kSharp || D == 128 || kFull ? 2 : 4;
};
template <typename T, int D>
constexpr bool sharp(bool causal, int64_t group) {
  return causal && (group < 4 || (D == 64 && std::is_same_v<T, f16_t>));
}

// The operands of a product in its type.
template <bool kHalf>
struct Number {
  using type = bf16_t;
  using vec = bf16x8;
  static __device__ __forceinline__ f32x16 product(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Number<true> {
  using type = f16_t;
  using vec = f16x8;
  static __device__ __forceinline__ f32x16 product(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// Whether tokens [begin, end) are f16 numbers: keys exactly (scales from 2^-23, whose halves are f16's smallest numbers, to 2^13;
// or below 2^-87, where zero is as good: scores of them are below 2^-34 at the largest scale), values to f16's smallest number
// (to 2^13), as far as their sums are rounded in any case.  `end` is where what is converted ends: a probability of zero
// times a value that has become an infinity is NaN.  All threads of a work-group together.
template <int D, int kThreads>
__device__ __forceinline__ bool all_half(const Attend& a, int64_t b, int hk, int begin, int end) {
  using L = Layout<D>;
  constexpr int kWords = 2 * D / 16;  // of 16 bytes, keys' scales first
  bool fit = true;
  const int blocks = (end - begin + kBlock - 1) / kBlock;
  for (int i = threadIdx.x; i < blocks * kWords; i += kThreads) {
    const int t0 = begin + i / kWords * kBlock, at = i % kWords;
    const int page = page_of(a.pages, b, t0);
    if (page < 0) continue;
    const i32x4 word = *reinterpret_cast<const i32x4*>(a.pages.data + block_of<D>(a.pages, page, hk, t0) + L::kKeyScales + 16 * at);
    const bool key = at < kWords / 2;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int byte = 16 * at + e;
      const int token = key ? byte / L::kParts : (byte - D) / L::kScaleGroup * 8 + byte % 8;
      const uint32_t scale = (static_cast<uint32_t>(word[e / 4]) >> (e % 4 * 8)) & 0xff;
      const bool fine = scale <= 140 && (!key || scale >= 104 || scale <= 40);
      fit &= fine || t0 + token >= end;
    }
  }
  return __syncthreads_and(fit);
}

template <typename T, int D, int kWaves, int kResident>
__global__ __launch_bounds__(kWaves * 64, kResident) void many_kernel(const Attend a) {
  using L = Layout<D>;
  constexpr int kSteps = D / 16;        // products over a row's channels
  constexpr int kOut = D / 32;          // tiles of 32 channels
  constexpr bool kApart = kWaves == 8;  // half the waves convert keys, half values
  // Tiles from one barrier to the next, as many as of which twice fit LDS beside other work-groups (2 x 2,058 ragged causal queries
  // over 16,464 tokens of 128 channels: bf16 230 us with one, 218 with two, f16 242, 236, fp32 444, 451; 64 channels within 2%).
  constexpr int kSpan = kApart && !std::is_same_v<T, float> ? 2 : 1, kSlots = 2 * kSpan;
  // [slot][block of 32 tokens][step][lane], [slot][block][tile][step of 16 tokens][lane]: operands of 16 bytes
  __shared__ u32x4 keys[kSlots][2][kSteps][64];
  __shared__ u32x4 values[kSlots][2][kOut][2][64];
  __shared__ uint2 bias[kSlots][64];  // three bf16 terms of what is added to a token's scores, before the scale
  const int lane = lane_id(), m = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = a.pages.kv_heads;
  const int hk = blockIdx.x % kv;
  const int rest = blockIdx.x / kv;
  // The tiles of a piece one after the other, so that they find its tokens in the cache, and the longest of a causal call first.
  // Where sequences are whole, the longest of all sequences first (3 causal prompts of up to 4,116 tokens, f16, 16 heads of 64
  // channels: 129 us, so 112; cut ones in this order 265, 290: 2 x 2,058 queries over 16,464).
  const Pieces all = many_pieces(a);
  int tile = a.tiles - 1 - rest % a.tiles, x = rest / a.tiles;
  if (a.causal && all.tokens == INT32_MAX) {
    const int n = pieces_in_all(a, all);
    tile = a.tiles - 1 - rest / n, x = rest % n;
    if (tile < 0) return;
  }
  const Piece piece = piece_of(a, all, x);
  if (piece.b < 0) return;
  leave(a, piece, x, threadIdx.x == 0 && hk == 0 && tile == 0);
  const int64_t b = piece.b;
  const int count = count_of(a, b);
  const int tile0 = a.first_row + tile * a.tile_rows;
  const int place0 = first_place(a, b, count), stop = stop_of(a, piece.length, count, place0, tile0);
  const int end = min(piece.end, stop);
  if (piece.begin > 0 && piece.begin >= stop) return;  // (the join does not ask for it)
  const bool whole = piece.begin == 0 && stop <= piece.end;

  const int row0 = tile0 + wave * 32, row = row0 + m;
  const int place = row >= count * a.group ? -1 : a.causal ? place0 + row / a.group : INT32_MAX;
  // Channels 16 s + 8 h .. of the lane's row (zeros where there is no query).
  const T* query = static_cast<const T*>(a.q) + b * a.q_stride[0] + (hk * a.group + row % a.group) * a.q_stride[1] +
                   row / a.group * a.q_stride[2] + 8 * h;
  // The first place of the wave's rows: tiles up to it need no causal mask.
  const int least = a.causal ? place0 + row0 / a.group : INT32_MAX;
  const bool idle = row0 >= count * a.group;

  // What this thread converts, all of one block of the tile's two: a quarter of a key's channels; a channel pair of
  // eight tokens, D / 64 times.
  const int ww = wave & 3, block = ww >> 1;
  const bool does_keys = !kApart || wave < 4, does_values = !kApart || wave >= 4;
  const int key = lane & 31, part = 2 * (ww & 1) + h, group = part, pair = lane & 31;
  const uint32_t key_from = key * L::kKeyBytes + part * (D / 8);
  const uint32_t key_scale_from = L::kKeyScales + key * L::kParts + part * L::kParts / 4;
  const uint32_t value_from = L::kValues + group * L::kGroup + pair * 8;
  const uint32_t value_scale_from = L::kValueScales + group * L::kScaleGroup + pair / 16 * 8;
  const int key_row = ((key >> 4) & 1) * 16 + ((key >> 2) & 1) * 8 + ((key >> 3) & 1) * 4 + (key & 3);
  uint2 key_codes[D / 64] = {}, value_codes[D / 64] = {}, value_scales[D / 64] = {};
  uint32_t key_scale = 0;
  float key_mass = 0.0f;
  // The page of this wave's block of a tile, looked up a tile before it is read and looked at then.  (Tokens before `end` are
  // within the table.)
  typedef const __attribute__((address_space(4))) int32_t* constant;
  const constant table = reinterpret_cast<constant>(reinterpret_cast<uintptr_t>(a.pages.table + b * a.pages.width));
  const int shift = a.pages.shift, pages = static_cast<int>(a.pages.pages), in_page = (1 << shift) - 1;
  const uint32_t page_blocks = static_cast<uint32_t>(kv) << (shift - 5);
  const uint8_t* head_data = a.pages.data + static_cast<int64_t>(hk << (shift - 5)) * L::kBytes;
  const float* masses = a.pages.mass;
  int first_found = -1, second_found = -1;
  int page = -1;
  bool gap_read = false;  // whether the tile has tokens that have no page, or lie past the end
  const auto find = [&](int n) {
    const int t0 = piece.begin + 64 * n;
    if (t0 >= end) return;
    first_found = table[t0 >> shift];
    second_found = shift == 5 && t0 + 32 < end ? table[(t0 >> 5) + 1] : first_found;
  };
  // Reads the wave's block of tile n.  Without a page nothing is read: scales of zero keep what is left finite, and the
  // bias keeps it out.
  const auto read = [&](int n) {
    const int t0 = piece.begin + 64 * n + 32 * block;
    const bool first = static_cast<uint32_t>(first_found) < static_cast<uint32_t>(pages);
    const bool second = static_cast<uint32_t>(second_found) < static_cast<uint32_t>(pages) && t0 - 32 * block + 32 < end;
    page = block == 0 ? (first ? first_found : -1) : second ? second_found : -1;
    gap_read = !first || !second || t0 - 32 * block + 64 > piece.length;
    if (page >= 0) {
      const uint8_t* base = head_data + (static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_blocks + ((t0 & in_page) >> 5)) * L::kBytes;
      if (does_keys) {
#pragma unroll
        for (int e = 0; e < D / 64; ++e) key_codes[e] = reinterpret_cast<const uint2*>(base + key_from)[e];
        key_scale = base[key_scale_from];
      }
      if (masses) key_mass = masses[(static_cast<int64_t>(page) << shift) + (t0 & in_page) + key];
      if (does_values) {
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
          value_codes[e] = *reinterpret_cast<const uint2*>(base + value_from + 256 * e);
          value_scales[e] = *reinterpret_cast<const uint2*>(base + value_scale_from + 16 * e);
        }
      }
    }
    if (gap_read) {
      const int kept = page < 0 ? 0 : piece.length - t0;
      if (key >= kept) key_scale = 0;
      key_mass = key >= kept ? -INFINITY : masses ? key_mass : 0.0f;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) value_scales[e] = kept_scales(value_scales[e], kept - 8 * group);
    }
  };
  const auto convert = [&](int slot, auto half) {
    constexpr bool kHalf = decltype(half)::value;
    if (masses) {
      // Tokens that their masses keep out, a bit each: as zeros, of which no product is NaN.
      const uint32_t out = static_cast<uint32_t>(__ballot(key_mass == -INFINITY));
      if (out != 0) {
        if (key_mass == -INFINITY) key_scale = 0;
#pragma unroll
        for (int e = 0; e < D / 64; ++e) value_scales[e] = scales_without(value_scales[e], out >> (8 * group));
      }
    }
    if (does_keys) {
      const float scale = scale_of<0>(key_scale);
      u32x4* to = &keys[slot][block][0][0] + key_row;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        // chunk c of 8 channels: step c / 2, lanes' half c % 2
        const int c = part * (D / 32) + 2 * e;
        to[c / 2 * 64] = key_operand<kHalf>(key_codes[e].x, scale);
        to[c / 2 * 64 + 32] = key_operand<kHalf>(key_codes[e].y, scale);
      }
      if (part == 0 && (gap_read || masses)) {
        const float raw = mass_of(key_mass) * a.per_scale;
        bf16_t t[3];
        split<3>(raw, t);
        if (raw == -INFINITY) t[1] = t[2] = static_cast<bf16_t>(0.0f);
        const bf16x2 first = {t[0], t[1]}, second = {t[2], static_cast<bf16_t>(0.0f)};
        bias[slot][32 * block + key_row] = {__builtin_bit_cast(uint32_t, first), __builtin_bit_cast(uint32_t, second)};
      }
    }
    if (does_values) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        u32x4 even, odd;
        value_operands<kHalf>(value_codes[e], value_scales[e], even, odd);
        values[slot][block][2 * e][group >> 1][(group & 1) * 32 + pair] = even;
        values[slot][block][2 * e + 1][group >> 1][(group & 1) * 32 + pair] = odd;
      }
    }
  };

  f32x16 acc[kOut] = {};
  float raw = -INFINITY, top = -INFINITY, total = 0.0f;  // the reference maximum, before and after the scale
  const int tiles = (end - piece.begin + 63) / 64;  // (none where end is before begin)

  const auto run = [&](auto half) {
    constexpr bool kHalf = decltype(half)::value;
    using N = Number<kHalf>;
    using vec = typename N::vec;
    constexpr int kQ = kHalf ? 1 : ManyTerms<T>::kQuery, kP = kHalf ? 1 : ManyTerms<T>::kWeight;
    // f16 probabilities are taken times 2^7, up to 2^15, which leaves them all their bits down to 2^-21.
    constexpr float kLift = kHalf ? 7.0f : 0.0f;
    vec q[kSteps][kQ];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float v[8] = {};
      if (row < count * a.group) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 four = load4(query + 16 * s + 4 * e);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * e + i] = channel_of(four[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        typename N::type t[kQ];
        split<kQ>(v[i], t);
#pragma unroll
        for (int n = 0; n < kQ; ++n) q[s][n][i] = t[n];
      }
    }
    // (Else the first product of every tile waits for whatever is outstanding, in case it is these.)
    wait_vmem<0>();
    bool gaps[kSpan] = {};  // of tiles n, ..
    if (tiles > 0) {
      find(0);
#pragma unroll
      for (int i = 0; i < kSpan; ++i)
        if (i < tiles) {
          read(i);
          find(i + 1);
          convert(i, half);
          gaps[i] = gap_read;
        }
      if (tiles > kSpan) read(kSpan);
      find(kSpan + 1);
    }
    for (int n = 0; n < tiles; ++n) {
      const int slot = n % kSlots;
      if (n % kSpan == 0) __syncthreads();
      const bool uneven = gaps[0] || masses != nullptr;
#pragma unroll
      for (int i = 0; i + 1 < kSpan; ++i) gaps[i] = gaps[i + 1];
      if (n + kSpan < tiles) {
        convert((n + kSpan) % kSlots, half);
        gaps[kSpan - 1] = gap_read;
      }
      if (n + kSpan + 1 < tiles) read(n + kSpan + 1);
      find(n + kSpan + 2);
      const int t0 = piece.begin + 64 * n;
      if (idle || (a.causal && t0 > place0 + (row0 + 31) / a.group)) continue;
      f32x16 z[2] = {};
      vec key_parts[2][kSteps];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) key_parts[k][s] = __builtin_bit_cast(vec, keys[slot][k][s][lane]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int t = kQ - 1; t >= 0; --t) z[k] = N::product(key_parts[k][s], q[s][t], z[k]);
      if (uneven) {
        // What is added to a token's scores, and what has no place: one more step of the product, by ones.
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint2 t = bias[slot][32 * k + m];
          Operand o, one;
          o.w[0] = h == 0 ? t.x : 0, o.w[1] = h == 0 ? t.y : 0, o.w[2] = o.w[3] = 0;
          one.w[0] = h == 0 ? 0x3f803f80u : 0, one.w[1] = h == 0 ? 0x00003f80u : 0, one.w[2] = one.w[3] = 0;
          z[k] = Number<false>::product(o.v, one.v, z[k]);
        }
      }
      if (t0 + 63 > least) {
        // Bits of the tokens that are seen, a word for 32 (comparisons would keep 64 scalar registers).
        const int most = place - t0 - 8 * h;
        const uint64_t seen = most < 0 ? 0 : most >= 63 ? ~uint64_t{0} : (uint64_t{2} << most) - 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int word = static_cast<int>(seen >> (32 * k));
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(word, 16 * (i >> 3) + (i & 7), 1));
            z[k][i] = __uint_as_float((__float_as_uint(z[k][i]) & keep) | (0xff800000u & ~keep));
          }
        }
      }
      float local = z[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) local = fmaxf(local, z[i >> 4][i & 15]);
      if (__builtin_expect(__any(local - raw > a.lazy), 0)) {
        local = half_max(local);
        const float shrink = shrink_of(raw, fmaxf(raw, local), a.scale);
        raw = fmaxf(raw, local), top = raw * a.scale;
        total *= shrink;
#pragma unroll
        for (int c = 0; c < kOut; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c][e] *= shrink;
      }
      float from = top == -INFINITY ? 0.0f : top - kLift;
      if (__builtin_expect(__any(fabsf(from) > kFar), 0)) {  // (see kFar)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) z[k][i] -= raw == -INFINITY ? 0.0f : raw;
        from = -kLift;
      }
      vec weights[2][2][kP];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(z[k][i], a.scale, -from));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(z[k][i + 1], a.scale, -from));
          typename N::type t0[kP], t1[kP];
          split<kP>(p0, t0), split<kP>(p1, t1);
          if constexpr (kP == 1 && !kHalf) {
            total = pair_sum(bf16x2{t0[0], t1[0]}, total);  // of the rounded ones, as the product takes them
          } else {
            total += p0 + p1;
          }
#pragma unroll
          for (int w = 0; w < kP; ++w) weights[k][i >> 3][w][i & 7] = t0[w], weights[k][i >> 3][w][(i & 7) + 1] = t1[w];
        }
      vec value_parts[2][kOut][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int c = 0; c < kOut; ++c)
#pragma unroll
          for (int t = 0; t < 2; ++t) value_parts[k][c][t] = __builtin_bit_cast(vec, values[slot][k][c][t][lane]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int c = 0; c < kOut; ++c)
#pragma unroll
            for (int w = kP - 1; w >= 0; --w) acc[c] = N::product(value_parts[k][c][t], weights[k][t][w], acc[c]);
    }
    top -= kLift;
  };
  if constexpr (std::is_same_v<T, f16_t>) {
    // (Blocks are converted whole, the last one past what a causal tile sees.)
    const int converted = min((end + kBlock - 1) & -kBlock, piece.length);
    if (all_half<D, kWaves * 64>(a, b, hk, piece.begin, converted)) run(std::true_type());
    else run(std::false_type());
  } else {
    run(std::false_type());
  }

  // A lane has, for its row, channels 64 c + 16 j + 8 h .. + 7 of tiles 2 c and 2 c + 1.
  total = half_sum(total);
  if (row >= min(tile0 + a.tile_rows, a.last_row)) return;
  const bool none = row >= count * a.group || sees_nothing(top, total);
  const float share = whole ? (none ? 0.0f : 1.0f / total) : 1.0f;
  const int64_t place_of = ((static_cast<int64_t>(x) * kv + hk) * a.tiles + tile) * a.tile_rows + row - tile0;
  T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + (hk * a.group + row % a.group) * a.out_stride[1] +
           row / a.group * a.out_stride[2];
  float* sums = a.sums + place_of * D;
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int channel = 64 * c + 16 * j + 8 * h;
      f32x4 v[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = none && whole ? 0.0f : acc[2 * c + (i & 1)][4 * j + i / 2] * share;
      if (whole) {
        store4(out + channel, v[0]);
        store4(out + channel + 4, v[1]);
      } else {
        store4(sums + channel, v[0]);
        store4(sums + channel + 4, v[1]);
      }
    }
  if (!whole && h == 0) a.ends[place_of] = {top, total};
}

// (What a CU holds, asked once: registers may leave room for more than the bound asked of the compiler.)
template <typename T, int D, typename M>
ManyShape shape_of() {
  static const int resident = [] {
    int n = 0;
    const bool known = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, many_kernel<T, D, M::kWaves, M::kResident>, M::kWaves * 64,
                                                                    0) == hipSuccess;
    if (!known) (void)hipGetLastError();  // (no device: nothing is launched either)
    return known && n > 0 ? n : 4 * M::kResident / M::kWaves;
  }();
  return {32 * M::kWaves, resident};
}
template <typename T, int D>
ManyShape shape_of(bool causal, int64_t group) {
  return sharp<T, D>(causal, group) ? shape_of<T, D, Many<T, D, true>>() : shape_of<T, D, Many<T, D, false>>();
}
template <typename T, int D>
int run_many(const Attend& a, int64_t pieces, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(pieces * a.tiles * a.pages.kv_heads);
  const auto run = [&](auto shape) {
    using M = Many<T, D, decltype(shape)::value>;
    many_kernel<T, D, M::kWaves, M::kResident><<<grid, M::kWaves * 64, 0, s>>>(a);
  };
  if (sharp<T, D>(a.causal, a.group)) run(std::true_type());
  else run(std::false_type());
  return check_launch("cached_attn");
}

}  // namespace
}  // namespace paged
}  // namespace vgo
