// Attention over the paged cache for few queries (decoding steps): up to 64 rows beside a key head.
//
// Bound by the cache's bytes, 17/16 D a token and key head, which are read once, and, with 64 channels, nearly as much by the
// vector units (a conversion makes two numbers of a byte, and a token of 64 channels needs 64 of them): one query of 16 heads
// over 4 key heads, 32 sequences of 32,768 tokens, codes from memory, with the join: 64 channels 66 us, 4.3 TB/s
// (f16 67, fp32 78); 128 114, 5.0 (115, 126); a copy reaches 5.1.  A wave takes
// blocks of 32 tokens on its own, the next two's codes on their way meanwhile:
//   scores^T = K Q^T, two 16 x 16 tiles; row m of tile i holds token 8 (m / 4) + 4 i + m % 4, so that the
//     lane that gets rows 4 g .. 4 g + 3 of both has tokens 8 g .. 8 g + 7 -- as the next product's operand wants them
//   out^T += V^T P^T; a lane has converted two channels of eight tokens, operands of two tiles
// Maxima are kept in common by the wave and moved only where a score exceeds them by 2^8; sums stay in their lanes.
// Eight waves share a piece of a sequence and join their sums in LDS.  Rows go by 16, whose further tiles find the codes in the
// caches; 32 at a time spill registers with 128 channels (32 rows of 8 x 16,384 tokens with masses, us: f16 91, so 45; fp32 139,
// 50; bf16 52, 43) and are as fast as this with 64 (bf16 30, 32 with masses; 64 rows without 38, 36).
#include "cached_attention.h"

namespace vgo {
namespace paged {
namespace {

constexpr int kWaves = 8;

// Four floats anywhere: masses are aligned as floats are (one load of 16 bytes all the same).
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// What a lane reads of a block of 32 tokens.
template <int D, bool kMass>
struct Codes {
  uint2 k[2][D / 64], v[D / 32], vs[D / 32];
  uint32_t ks[2];
  f32x4 mass[kMass ? 2 : 1];
};

// Where in a block (and, for masses, in a page's) a lane reads: 32-bit offsets, so that a read takes its block's address
// from scalar registers.
template <int D>
struct Offsets {
  uint32_t k[2], ks[2], v, vs, mass;
  __device__ __forceinline__ Offsets(int lane) {
    using L = Layout<D>;
    const uint32_t m = lane & 15, g = lane >> 4;
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t token = 8 * (m >> 2) + 4 * i + (m & 3);
      k[i] = token * L::kKeyBytes + g * (D / 8);
      ks[i] = L::kKeyScales + token * L::kParts + g * L::kParts / 4;
    }
    v = L::kValues + g * L::kGroup + m * 8;
    vs = L::kValueScales + g * L::kScaleGroup;
    mass = 32 * g;
  }
};

template <int D, bool kMass>
__device__ __forceinline__ void read_codes(Codes<D, kMass>& c, const uint8_t* block, const float* mass, const Offsets<D>& o) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < D / 64; ++e) c.k[i][e] = *reinterpret_cast<const uint2*>(block + o.k[i] + 8 * e);
    c.ks[i] = block[o.ks[i]];
  }
#pragma unroll
  for (int u = 0; u < D / 32; ++u) {
    c.v[u] = *reinterpret_cast<const uint2*>(block + o.v + 128 * u);
    c.vs[u] = *reinterpret_cast<const uint2*>(block + o.vs + 8 * u);
  }
  if constexpr (kMass) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      c.mass[i] = *reinterpret_cast<const f32x4_any*>(reinterpret_cast<const uint8_t*>(mass) + o.mass + 16 * i);
  }
}

// Two numbers as kTerms bf16 terms each, in pairs.
template <int kTerms>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&t)[kTerms]) {
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    const bf16x2 pair = {static_cast<bf16_t>(x), static_cast<bf16_t>(y)};
    t[i] = __builtin_bit_cast(uint32_t, pair);
    asm("" : "+v"(t[i]));  // (else the first of the pair is converted a second time)
    if (i + 1 < kTerms) {
      x -= __uint_as_float(t[i] << 16);
      y -= __uint_as_float(t[i] & 0xffff0000u);
    }
  }
}

template <typename T, int D, bool kMass>
__global__ __launch_bounds__(kWaves * 64, 2) void few_kernel(const Attend a) {
  using L = Layout<D>;
  constexpr int kQ = Terms<T>::kQuery, kP = Terms<T>::kWeight;
  constexpr int kSteps = D / 32;
  __shared__ float joined[kWaves][16][D + 4];
  __shared__ float tops[kWaves][16], totals[kWaves][16];
  const int lane = lane_id(), m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = a.pages.kv_heads;
  const int hk = blockIdx.x % kv;
  const int rest = blockIdx.x / kv;
  const int tile = rest % a.tiles;
  const int x = rest / a.tiles;
  const Piece piece = piece_of(a, few_pieces(a), x);
  if (piece.b < 0) return;
  leave(a, piece, x, threadIdx.x == 0 && hk == 0 && rest % a.tiles == 0);
  const int64_t b = piece.b;
  const int count = count_of(a, b);
  const int row0 = a.first_row + tile * a.tile_rows;
  const int place0 = first_place(a, b, count), stop = stop_of(a, piece.length, count, place0, row0);
  const int end = min(piece.end, stop);
  if (piece.begin > 0 && piece.begin >= stop) return;  // (the join does not ask for it)
  const bool whole = piece.begin == 0 && stop <= piece.end;

  // Queries: row m of the tile, channels 8 s .. of this lane's D / 4.
  bf16x8 q[kSteps][kQ];
  const int mine = row0 + m, token = mine / a.group;
  const bool real = mine < count * a.group;
  const int place = !real ? -1 : a.causal ? place0 + token : INT32_MAX;
  const T* query = static_cast<const T*>(a.q) + b * a.q_stride[0] + (hk * a.group + mine % a.group) * a.q_stride[1] +
                   token * a.q_stride[2] + g * (D / 4);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    float v[8] = {};
    if (real) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 four = load4(query + 8 * s + 4 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * e + i] = channel_of(four[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16_t t[kQ];
      split<kQ>(v[i], t);
#pragma unroll
      for (int n = 0; n < kQ; ++n) q[s][n][i] = t[n];
    }
  }
  f32x4 acc[D / 16] = {};
  float raw = -INFINITY, top = -INFINITY, total = 0.0f;  // the reference maximum, before and after the scale

  // A ring of blocks on their way.  Reads are not conditional, so that the compiler knows how many are outstanding: what has
  // no page, or lies past the end, reads the start of the cache instead and is left out.
  constexpr int kRing = 3;
  const Offsets<D> offsets(lane);
  Codes<D, kMass> ring[kRing];
  bool there[kRing];
  const int first = piece.begin / kBlock, blocks = a.pages.pages > 0 ? (end + kBlock - 1) / kBlock : 0;
  // (Looked up a step before it is looked at.  Tokens before `end` are within the table.)
  typedef const __attribute__((address_space(4))) int32_t* constant;
  const constant table = reinterpret_cast<constant>(reinterpret_cast<uintptr_t>(a.pages.table + b * a.pages.width));
  const int shift = a.pages.shift - 5, in_page = (1 << shift) - 1;  // in blocks
  const uint32_t pages = static_cast<uint32_t>(a.pages.pages), page_blocks = static_cast<uint32_t>(kv) << shift;
  const uint8_t* head_data = a.pages.data + static_cast<int64_t>(hk << shift) * L::kBytes;
  const auto page_at = [&](int block) { return block < blocks ? table[block >> shift] : -1; };
  const auto read = [&](int slot, int block, int page) {
    there[slot] = static_cast<uint32_t>(page) < pages;
    const uint8_t* from = a.pages.data;
    const float* mass = a.pages.mass;
    if (there[slot]) {
      from = head_data + (static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_blocks + (block & in_page)) * L::kBytes;
      if (kMass) mass += ((static_cast<int64_t>(page) << shift) + (block & in_page)) * kBlock;
    }
    read_codes(ring[slot], from, mass, offsets);
  };
  const auto compute = [&](const Codes<D, kMass>& codes, int block) {
    const int t0 = block * kBlock;
    const bool inside = t0 + kBlock <= piece.length;
    bf16x8 keys[2][kSteps];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float scale = scale_of<0>(codes.ks[i]);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        keys[i][s] = __builtin_bit_cast(bf16x8, key_operand(s % 2 ? codes.k[i][s / 2].y : codes.k[i][s / 2].x, scale));
    }
    Operand weights[kP];
    float z[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 c = {};
#pragma unroll
      for (int n = kQ - 1; n >= 0; --n)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys[i][s], q[s][n], c, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[4 * i + e] = c[e];
    }
    uint2 value_scales[D / 32];
#pragma unroll
    for (int u = 0; u < D / 32; ++u) value_scales[u] = codes.vs[u];
    if constexpr (kMass) {
      const auto mass = [&](int i) { return codes.mass[i / 4][i % 4]; };
      float largest = 0.0f;  // (NaN in any is kept)
#pragma unroll
      for (int i = 0; i < 8; ++i) largest = __builtin_elementwise_maximum(largest, fabsf(mass(i)));
      if (!__any(!(largest <= kMostMass))) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = fmaf(z[i], a.scale, mass(i) * 1.4426950408889634f);
      } else {
        uint32_t out = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool gone = mass(i) == -INFINITY;
          z[i] = gone ? -INFINITY : fmaf(z[i], a.scale, mass_of(mass(i)) * 1.4426950408889634f);
          out |= gone ? 1u << i : 0u;
        }
#pragma unroll
        for (int u = 0; u < D / 32; ++u) value_scales[u] = scales_without(value_scales[u], out);
      }
    }
    const float scale = kMass ? 1.0f : a.scale;  // still to be applied
    if (a.causal || !inside) {
      const int most = min(place, piece.length - 1) - t0 - 8 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = i <= most ? z[i] : -INFINITY;
    }
    float local = z[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) local = fmaxf(local, z[i]);
    if (__any(local - raw > (kMass ? kLazy : a.lazy))) {
      local = fmaxf(local, __shfl_xor(local, 16));
      local = half_max(local);
      const float shrink = shrink_of(raw, fmaxf(raw, local), scale);
      raw = fmaxf(raw, local), top = raw * scale;
      total *= shrink;
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][e] *= shrink;
    }
    float from = top == -INFINITY ? 0.0f : top;
    if (__any(fabsf(from) > kFar)) {  // (see kFar)
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] -= raw == -INFINITY ? 0.0f : raw;
      from = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(z[2 * i], scale, -from));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(z[2 * i + 1], scale, -from));
      total += p0 + p1;
      uint32_t t[kP];
      split_pair<kP>(p0, p1, t);
#pragma unroll
      for (int n = 0; n < kP; ++n) weights[n].w[i] = t[n];
    }
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      uint2 scales = value_scales[u];
      if (!inside) scales = kept_scales(scales, piece.length - t0 - 8 * g);
      u32x4 two[2];
      value_operands(codes.v[u], scales, two[0], two[1]);
      const bf16x8 even = __builtin_bit_cast(bf16x8, two[0]), odd = __builtin_bit_cast(bf16x8, two[1]);
#pragma unroll
      for (int n = kP - 1; n >= 0; --n) {
        acc[2 * u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, weights[n].v, acc[2 * u], 0, 0, 0);
        acc[2 * u + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, weights[n].v, acc[2 * u + 1], 0, 0, 0);
      }
    }
  };
  int block = first + wave;
  if (block < blocks) {
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) read(i, block + i * kWaves, page_at(block + i * kWaves));
    int page = page_at(block + (kRing - 1) * kWaves);
    while (block < blocks) {
#pragma unroll
      for (int i = 0; i < kRing; ++i) {
        read((i + kRing - 1) % kRing, block + (kRing - 1) * kWaves, page);
        page = page_at(block + kRing * kWaves);
        if (there[i]) compute(ring[i], block);
        block += kWaves;
      }
    }
  }

  // The waves' sums.
  total += __shfl_xor(total, 16);
  total = half_sum(total);
  if (g == 0) tops[wave][m] = top, totals[wave][m] = total;
#pragma unroll
  for (int u = 0; u < D / 32; ++u) {
    const f32x4 e = acc[2 * u], o = acc[2 * u + 1];
    f32x4* to = reinterpret_cast<f32x4*>(&joined[wave][m][32 * u + 8 * g]);
    to[0] = f32x4{e[0], o[0], e[1], o[1]};
    to[1] = f32x4{e[2], o[2], e[3], o[3]};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * D / 4; i += kWaves * 64) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    const int row = row0 + r;
    if (row >= a.last_row) continue;
    float most = tops[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, tops[w][r]);
    const float from = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float share = __builtin_amdgcn_exp2f(tops[w][r] - from);
      const f32x4 part = *reinterpret_cast<const f32x4*>(&joined[w][r][c]);
      sum = fmaf(totals[w][r], share, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(part[e], share, v[e]);
    }
    if (whole) {
      const bool none = row >= count * a.group || sees_nothing(most, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : v[e] / sum;
      store4(static_cast<T*>(a.out) + b * a.out_stride[0] + (hk * a.group + row % a.group) * a.out_stride[1] +
                 row / a.group * a.out_stride[2] + c, v);
    } else {
      const int64_t to = ((static_cast<int64_t>(x) * kv + hk) * a.tiles + tile) * a.tile_rows + r;
      store4(a.sums + to * D + c, v);
      if (c == 0) a.ends[to] = {most, sum};
    }
  }
}

template <typename T, int D>
int launch(const Attend& a, int64_t pieces, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(pieces * a.tiles * a.pages.kv_heads);
  if (a.pages.mass) few_kernel<T, D, true><<<grid, kWaves * 64, 0, s>>>(a);
  else few_kernel<T, D, false><<<grid, kWaves * 64, 0, s>>>(a);
  return check_launch("cached_attn");
}

}  // namespace

int launch_few(const Attend& a, int64_t pieces, int head_dim, int dtype, hipStream_t s) {
  if (head_dim == 64) {
    if (dtype == VGO_BF16) return launch<bf16_t, 64>(a, pieces, s);
    if (dtype == VGO_F16) return launch<f16_t, 64>(a, pieces, s);
    return launch<float, 64>(a, pieces, s);
  }
  if (dtype == VGO_BF16) return launch<bf16_t, 128>(a, pieces, s);
  if (dtype == VGO_F16) return launch<f16_t, 128>(a, pieces, s);
  return launch<float, 128>(a, pieces, s);
}

}  // namespace paged
}  // namespace vgo
