// Attention over the paged cache for many queries (chunks and prompts).
//
// kWaves waves of 32 MT rows each share 64 tokens at a time: the codes come into registers two tiles ahead, are
// converted once for all waves into operands of the 32 x 32 matrix instructions and written to LDS in the order in which
// their lanes read them (16 bytes a lane, no bank conflicts), double-buffered, one barrier a tile:
//   scores^T = K Q^T; row m of a block of 32 tokens holds token 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so
//     that a lane's sixteen scores are two operands of the next product as they stand
//   out^T += V^T P^T, a lane having converted two channels of eight tokens, operands of two tiles
// One reference maximum a row, moved only where a score passes it by 2^8.
#pragma once

#include "cached_attention.h"

namespace vgo {
namespace paged {
namespace {

constexpr float kLazyMany = 8.0f;

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

// How a type and width are run: waves of a work-group, 32-row tiles of a wave, waves that a SIMD is to hold.
template <typename T, int D>
struct Many {
  static constexpr int kWaves = 4, kTiles = 1, kResident = 2;
};
template <>
struct Many<bf16_t, 64> {
  static constexpr int kWaves = 8, kTiles = 1, kResident = 4;
};
template <>
struct Many<bf16_t, 128> {
  static constexpr int kWaves = 8, kTiles = 1, kResident = 2;
};

template <typename T, int D, int kWaves, int MT, int kResident>
__global__ __launch_bounds__(kWaves * 64, kResident) void many_kernel(const Attend a) {
  using L = Layout<D>;
  constexpr int kQ = ManyTerms<T>::kQuery, kP = ManyTerms<T>::kWeight;
  constexpr int kSteps = D / 16;        // products over a row's channels
  constexpr int kOut = D / 32;          // tiles of 32 channels
  constexpr bool kApart = kWaves == 8;  // half the waves convert keys, half values
  // [buffer][block of 32 tokens][step][lane], [buffer][block][tile][step of 16 tokens][lane]
  __shared__ bf16x8 keys[2][2][kSteps][64];
  __shared__ bf16x8 values[2][2][kOut][2][64];
  __shared__ uint2 bias[2][64];  // three bf16 terms of what is added to a token's scores, before the scale
  const int lane = lane_id(), m = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = a.pages.kv_heads;
  const int hk = blockIdx.x % kv;
  const int rest = blockIdx.x / kv;
  const int tile = tile_at(a, rest % a.tiles);
  const int x = rest / a.tiles;
  const Piece piece = piece_of(a, x);
  if (piece.b < 0) return;
  leave(a, piece, x, threadIdx.x == 0 && hk == 0 && rest % a.tiles == 0);
  const int64_t b = piece.b;
  const int count = count_of(a, b);
  const int tile0 = a.first_row + tile * a.tile_rows;
  const int place0 = a.lengths[b] - count, stop = stop_of(a, piece.length, count, place0, tile0);
  const int end = min(piece.end, stop);
  if (piece.begin > 0 && piece.begin >= stop) return;  // (merge_kernel does not ask for it)
  const bool whole = piece.begin == 0 && stop <= piece.end;

  const int row0 = tile0 + wave * 32 * MT;
  bf16x8 q[MT][kSteps][kQ];
  int place[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 32 * mt + m, token = row / a.group;
    const bool real = row < count * a.group;
    place[mt] = !real ? -1 : a.causal ? place0 + token : INT32_MAX;
    const T* from = static_cast<const T*>(a.q) + b * a.q_stride[0] + (hk * a.group + row % a.group) * a.q_stride[1] +
                    token * a.q_stride[2] + 8 * h;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float v[8] = {};
      if (real) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 four = load4(from + 16 * s + 4 * e);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * e + i] = four[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bf16_t t[kQ];
        split<kQ>(v[i], t);
#pragma unroll
        for (int n = 0; n < kQ; ++n) q[mt][s][n][i] = t[n];
      }
    }
  }
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
  // The page of this wave's block of a tile, known a tile before it is read.
  int page = -1;
  bool gap_read = false;  // whether the tile has tokens that have no page, or lie past the end
  bool gap_found = false;
  const auto find = [&](int n) {
    const int t0 = piece.begin + 64 * n;
    const int first = t0 < end ? page_of(a.pages, b, t0) : -1;
    const int second = t0 + 32 < end ? a.pages.shift > 5 ? first : page_of(a.pages, b, t0 + 32) : -1;
    page = __builtin_amdgcn_readfirstlane(block == 0 ? first : second);
    gap_found = first < 0 || second < 0 || t0 + 64 > piece.length;
  };
  // Reads the wave's block of tile n.  Without a page nothing is read: scales of zero keep what is left finite, and the
  // bias keeps it out.
  const auto read = [&](int n) {
    const int t0 = piece.begin + 64 * n + 32 * block;
    gap_read = gap_found;
    if (page >= 0) {
      const uint8_t* base = a.pages.data + block_of<D>(a.pages, page, hk, t0);
      if (does_keys) {
#pragma unroll
        for (int e = 0; e < D / 64; ++e) key_codes[e] = reinterpret_cast<const uint2*>(base + key_from)[e];
        key_scale = base[key_scale_from];
        if (part == 0 && a.pages.mass)
          key_mass = a.pages.mass[(static_cast<int64_t>(page) << a.pages.shift) + (t0 & ((1 << a.pages.shift) - 1)) + key];
      }
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
      key_mass = key >= kept ? -INFINITY : a.pages.mass ? key_mass : 0.0f;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) value_scales[e] = kept_scales(value_scales[e], kept - 8 * group);
    }
  };
  const auto convert = [&](int buffer) {
    if (does_keys) {
      const float scale = scale_of<0>(key_scale);
      bf16x8* to = &keys[buffer][block][0][0] + key_row;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        // chunk c of 8 channels: step c / 2, lanes' half c % 2
        const int c = part * (D / 32) + 2 * e;
        to[c / 2 * 64] = key_operand(key_codes[e].x, scale);
        to[c / 2 * 64 + 32] = key_operand(key_codes[e].y, scale);
      }
      if (part == 0 && (gap_read || a.pages.mass)) {
        const float raw = mass_of(key_mass) * a.per_scale;
        bf16_t t[3];
        split<3>(raw, t);
        if (raw == -INFINITY) t[1] = t[2] = static_cast<bf16_t>(0.0f);
        const bf16x2 first = {t[0], t[1]}, second = {t[2], static_cast<bf16_t>(0.0f)};
        bias[buffer][32 * block + key_row] = {__builtin_bit_cast(uint32_t, first), __builtin_bit_cast(uint32_t, second)};
      }
    }
    if (does_values) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        bf16x8 even, odd;
        value_operands(value_codes[e], value_scales[e], even, odd);
        values[buffer][block][2 * e][group >> 1][(group & 1) * 32 + pair] = even;
        values[buffer][block][2 * e + 1][group >> 1][(group & 1) * 32 + pair] = odd;
      }
    }
  };

  f32x16 acc[MT][kOut] = {};
  float top[MT], total[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) top[mt] = -INFINITY, total[mt] = 0.0f;
  const int tiles = (end - piece.begin + 63) / 64;  // (none where end is before begin)
  bool gap = false;
  if (tiles > 0) {
    find(0);
    read(0);
    find(1);
    convert(0);
    gap = gap_read;
    if (tiles > 1) read(1);
    find(2);
  }
  for (int n = 0; n < tiles; ++n) {
    const int buffer = n & 1;
    __syncthreads();
    const bool uneven = gap || a.pages.mass != nullptr;
    if (n + 1 < tiles) {
      convert(buffer ^ 1);
      gap = gap_read;
    }
    if (n + 2 < tiles) read(n + 2);
    find(n + 3);
    const int t0 = piece.begin + 64 * n;
    if (idle || (a.causal && t0 > place0 + (row0 + 32 * MT - 1) / a.group)) continue;
    f32x16 z[MT][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) z[mt][k] = f32x16{};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 key_part = keys[buffer][k][s][lane];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int t = kQ - 1; t >= 0; --t)
            z[mt][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_part, q[mt][s][t], z[mt][k], 0, 0, 0);
      }
    }
    const bool diagonal = t0 + 63 > least;
    if (uneven) {
      // What is added to a token's scores, and what has no place: one more step of the product, by ones.
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 t = bias[buffer][32 * k + m];
        Operand o, one;
        o.w[0] = h == 0 ? t.x : 0, o.w[1] = h == 0 ? t.y : 0, o.w[2] = o.w[3] = 0;
        one.w[0] = h == 0 ? 0x3f803f80u : 0, one.w[1] = h == 0 ? 0x00003f80u : 0, one.w[2] = one.w[3] = 0;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) z[mt][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.v, one.v, z[mt][k], 0, 0, 0);
      }
    }
    if (diagonal) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int most = place[mt] - t0 - 8 * h;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * k + 16 * (i >> 3) + (i & 7) > most) z[mt][k][i] = -INFINITY;
      }
    }
    bf16x8 weights[MT][2][2][kP];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float local = z[mt][0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) local = fmaxf(local, z[mt][i >> 4][i & 15]);
      local *= a.scale;
      if (__any(local > top[mt] + kLazyMany)) {
        local = half_max(local);
        const float to = fmaxf(top[mt], local);
        const float shrink = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[mt] - to);
        top[mt] = to;
        total[mt] *= shrink;
#pragma unroll
        for (int c = 0; c < kOut; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[mt][c][e] *= shrink;
      }
      const float from = top[mt] == -INFINITY ? 0.0f : top[mt];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(z[mt][k][i], a.scale, -from));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(z[mt][k][i + 1], a.scale, -from));
          if constexpr (kP == 1) {
            // The sum of the rounded probabilities, as the product takes them.
            const bf16x2 pair = {static_cast<bf16_t>(p0), static_cast<bf16_t>(p1)};
            total[mt] = pair_sum(pair, total[mt]);
            weights[mt][k][i >> 3][0][i & 7] = pair[0], weights[mt][k][i >> 3][0][(i & 7) + 1] = pair[1];
          } else {
            total[mt] += p0 + p1;
            bf16_t t0[kP], t1[kP];
            split<kP>(p0, t0), split<kP>(p1, t1);
#pragma unroll
            for (int w = 0; w < kP; ++w) weights[mt][k][i >> 3][w][i & 7] = t0[w], weights[mt][k][i >> 3][w][(i & 7) + 1] = t1[w];
          }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < kOut; ++c)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bf16x8 value = values[buffer][k][c][t][lane];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int w = kP - 1; w >= 0; --w)
              acc[mt][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value, weights[mt][k][t][w], acc[mt][c], 0, 0, 0);
        }
  }

  // A lane has, for its row, channels 64 c + 16 j + 8 h .. + 7 of tiles 2 c and 2 c + 1.
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 32 * mt + m;
    total[mt] = half_sum(total[mt]);
    if (row >= min(tile0 + a.tile_rows, a.last_row)) continue;
    const bool none = row >= count * a.group || top[mt] == -INFINITY;
    const float share = whole ? (none ? 0.0f : 1.0f / total[mt]) : 1.0f;
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
        for (int i = 0; i < 8; ++i)
          v[i >> 2][i & 3] = none && whole ? 0.0f : acc[mt][2 * c + (i & 1)][4 * j + i / 2] * share;
        if (whole) {
          store4(out + channel, v[0]);
          store4(out + channel + 4, v[1]);
        } else {
          store4(sums + channel, v[0]);
          store4(sums + channel + 4, v[1]);
        }
      }
    if (!whole && h == 0) a.ends[place_of] = {top[mt], total[mt]};
  }
}

template <typename T, int D>
int run_many(const Attend& a, int64_t pieces, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(pieces * a.tiles * a.pages.kv_heads);
  using M = Many<T, D>;
  many_kernel<T, D, M::kWaves, M::kTiles, M::kResident><<<grid, M::kWaves * 64, 0, s>>>(a);
  return check_launch("cached_attn");
}

}  // namespace
}  // namespace paged
}  // namespace vgo
