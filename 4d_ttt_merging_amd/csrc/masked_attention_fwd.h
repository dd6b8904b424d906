// Masked attention, forward (rules and layouts: masked_attention.h).
//
// A task is kWaves x 32 rows of one (batch, head), or, where a head has few queries and shares
// its keys, of all heads of one key head (rows r = head g, query i: r = g n_query + i); it runs over
// the key tiles in which any pair of its rows attends, found 64 tiles at a time by one ballot, in
// which each lane judges one tile.  K and V tiles come into LDS by DMA, row-major, double-buffered,
// one barrier per tile; V's columns are read by transposing LDS reads.
//
// Softmax: online, one reference maximum per row, moved (and the sums rescaled) only when a logit
// passes it by 8 powers of 2; P is rounded to the inputs' type for P V as the products take it,
// sums and outputs are kept in fp32.  In bf16 the row sums take the rounded P, two per instruction: where one key
// has most of a row its rounding then cancels (sums of the unrounded ones are as fast, within 1%).
//
// Bound: with a cap the issue of vector instructions (busy 0.87 of the time at 16 x 16,464 x 64 causal, 0.90 where
// scores come near the cap; the matrix pipes 0.30 and 0.23).  Else neither pipe is full (matrix and vector, which may be
// busy at once: 0.36 and 0.63 at 16 x 8,232 x 64 causal, 0.43 and 0.42 with 128 channels): a work-group's waves are in
// products, or in the softmax (exponential, FMA, conversion, maximum per score), together, between barriers a tile.
// 32 rows a wave, so that three waves (64 channels) overlap, where 64 rows at two were as fast on long rows and slower
// on short ones (8,232 causal: 294 us, 240).  16 heads of 8,232 x 8,232: 390 us with 64 channels (0.71 PFLOP/s; a
// library product 1.2), 687 with 128 (0.81), 16,464 causal 660 (0.84), capped 842, and 990 where scores come near
// the cap; fp32 2,058 x 2,058 191 us (91 of 140 TFLOP/s; matrix pipes busy 0.72, then the join).
// Single tokens: HBM, 32 of 32,928 keys with 4 key heads 140 to 152 us capped and ragged (0.9 of a copy's rate).
#pragma once

#include <type_traits>

#include "masked_attention.h"

namespace vgo {
namespace masked {

// How a problem is cut into tasks.
struct ForwardPlan {
  int pack, rows, row_blocks, splits, tiles;
  int64_t tasks;
};

ForwardPlan forward_plan(const vgo_masked_attn* p, int dtype);
size_t forward_bytes(const vgo_masked_attn* p, const ForwardPlan& plan);
inline size_t align16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// The launches of one type (instantiated in masked_attention_bf16.hip and its like).
template <typename T>
int run_forward(const vgo_masked_attn* p, const ForwardPlan& plan, void* out, const int64_t out_stride[3], float* lse,
                void* rest, char* ws, hipStream_t stream);
extern template int run_forward<bf16_t>(const vgo_masked_attn*, const ForwardPlan&, void*, const int64_t[3], float*,
                                        void*, char*, hipStream_t);
extern template int run_forward<f16_t>(const vgo_masked_attn*, const ForwardPlan&, void*, const int64_t[3], float*,
                                       void*, char*, hipStream_t);
extern template int run_forward<float>(const vgo_masked_attn*, const ForwardPlan&, void*, const int64_t[3], float*,
                                       void*, char*, hipStream_t);

namespace {

// What rounding to T takes from x.
template <typename T>
__device__ __forceinline__ f32x4 rounding(f32x4 x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] -= to_f32(from_f32<T>(x[e]));
  return x;
}

// log2 of a row's sum of e^z, l 2^m, as two numbers: beside a large m, the same for all of a row's scores, log2(l)
// would be rounded away, and with it what makes the gradients' probabilities add up to one (fp32 keys that share a
// mass of -1e6: off by a sixteenth).
__device__ __forceinline__ void store_lse(float* lse, int64_t rows, int64_t at, float m, float l) {
  const float log = __builtin_amdgcn_logf(l), sum = m + log;
  lse[at] = l == 0.0f ? kInf : sum;
  lse[rows + at] = l == 0.0f ? 0.0f : log - (sum - m);
}

// What a launch adds to the problem.
template <typename T>
struct Forward {
  Args<T> a;
  T* out;
  float* lse;     // or null: two planes [batch, heads, n_query], what the sum of the first rounds and that rest
  T* rest;        // or null: what rounding took from out, [batch, heads, n_query, D]
  float* part_o;  // splits > 1: [splits, batch * virtual heads, rows, D] unnormalised sums
  float* part_ml; // and [.., rows, 3] their reference maxima (log2) and row sums (rounded, unrounded)
  int pack;       // heads per task (1, or heads / kv_heads)
  int rows;       // pack * n_query
  int row_blocks, splits, tiles, tasks, joiners;
};

// The key tiles of one task that its work-group (`wg`) and this wave (`w`) take part in, of every `step`-th from
// `first` on: splits take turns, so that each gets its share of what masks and lengths leave.
template <typename T>
struct Walk {
  const Args<T>& a;
  Range wg, w;
  int b, limit, prefix, end, first, step, base, tile;
  uint64_t todo, mine, full, whole;  // of the 64 tiles first + step * (base ..)
  bool in_mine, in_full, in_whole;   // of `tile`
  const bool rows_here;              // the wave has rows

  __device__ __forceinline__ Walk(const Args<T>& args, const Range& group, const Range& wave, bool rows, int batch,
                                  int split, int splits, int tiles)
      : a(args), wg(group), w(wave), b(batch), end(tiles), first(split), step(splits), base(-64), tile(0), todo(0),
        rows_here(rows) {
    limit = key_limit(a, b);
    prefix = prefix_of(a, b);
    end = min(end, (limit + kTile - 1) / kTile);
  }
  __device__ __forceinline__ bool next() {
    while (todo == 0) {
      base += 64;
      if (first + step * base >= end) return false;
      const int t = first + step * (base + lane_id());
      bool any = t < end, all_w = false, any_w = false, whole_t = false;
      if (any) {
        Range k{};
        if (a.key_doc) k = info_range(a.key_info[static_cast<int64_t>(b) * ((a.n_key + kTile - 1) / kTile) + t]);
        k.lo = t * kTile, k.hi = min(k.lo + kTile, limit) - 1;
        bool all;
        judge(a, wg, k, prefix, any, all);
        judge(a, w, k, prefix, any_w, all_w);
        const bool inside = k.lo + kTile <= limit;
        any_w = any_w && rows_here;
        all_w = all_w && inside;
        whole_t = inside && (!a.key_doc || k.docs_whole);
      }
      todo = __ballot(any), mine = __ballot(any && any_w), full = __ballot(all_w), whole = __ballot(whole_t);
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    tile = first + step * (base + bit);
    in_mine = mine >> bit & 1, in_full = full >> bit & 1, in_whole = whole >> bit & 1;
    return true;
  }
};

constexpr int kWaves = 4, kRowsPerWave = 32, kRows = kRowsPerWave * kWaves;  // of a work-group

template <typename T, int D>
struct Layout {
  static constexpr int kTiles = 4 * Tile<T, D>::kBytes;  // K and V, two buffers
  static constexpr int kMass = kTiles, kDocs = kMass + 2 * kTile * 4, kRange = kDocs + 2 * kTile * 4;
  static constexpr int kDistances = kRange + kWaves * 16;
};

// A row's reference moves when a logit passes it by more than this many powers of 2 (f16: and those by which it is
// lower): probabilities stay below 2^8, 2^15 of f16.
constexpr float kSlack = 8.0f;

// kTrain: 1 where gradients follow, whose probabilities are those of the unrounded row sum; 2 with slopes, too.
// D = dO . O then has to be the mean of dP under the very probabilities that the gradients compute again: the
// slopes' weigh what it is off by with the distances, and from rounded probabilities they were off by 0.2 to
// 0.5% in bf16.  A second product takes what the rounding left out (1e-5).
template <typename T, int D, bool kCap, int kBias, int kTrain>
__global__ __launch_bounds__(64 * kWaves, D * sizeof(T) > 256 ? 1 : D * sizeof(T) > 128 ? 2 : 3) void forward_kernel(
    const Forward<T> f) {
  typedef Tile<T, D> TL;
  typedef Layout<T, D> LO;
  typedef typename Op<T>::op8 op8;
  extern __shared__ __align__(16) char lds[];
  const Args<T>& a = f.a;
  const int lane = lane_id(), l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Heads, then key splits, then row blocks.
  int task = xcd_remap(blockIdx.x, f.tasks);
  const int block = f.row_blocks - 1 - zigzag(task % f.row_blocks, f.row_blocks, task / f.row_blocks, f.tasks / f.row_blocks);
  task /= f.row_blocks;
  const int split = task % f.splits;
  task /= f.splits;
  const int vheads = a.heads / f.pack, vh = task % vheads, b = task / vheads;
  const int kvh = vh * f.pack / (a.heads / a.kv_heads);
  const int row0 = block * kRows + wave * kRowsPerWave;
  const int start = first_position(a, b);

  // The wave's rows: operands, positions, documents.
  const int row = row0 + l31, rc = min(row, f.rows - 1);
  const bool stored = row < f.rows;
  const int of_group = f.pack == 1 ? 0 : rc / a.n_query;
  const int index = rc - of_group * a.n_query, head = vh * f.pack + of_group, pos = start + index;
  const int doc = a.query_doc ? a.query_doc[static_cast<int64_t>(b) * a.n_query + index] : 0;
  const float slope = slope2(a, head);
  const float* distance = reinterpret_cast<const float*>(lds + LO::kDistances) +
                          of_group * distance_words(a.buckets.reach);
  op8 q[TL::kSteps];
  const T* src = a.q + b * a.qs[0] + head * a.qs[1] + index * a.qs[2] + 8 * h;
#pragma unroll
  for (int t = 0; t < TL::kSteps; ++t) q[t] = *reinterpret_cast<const op8*>(src + 16 * t);
  // Positions of rows first .. first + n: contiguous within a head, everything across heads.
  const auto positions = [&](int first, int n, Range& r) {
    const int last = min(first + n, f.rows) - 1;
    first = min(first, f.rows - 1);
    const bool one = f.pack == 1 || first / a.n_query == last / a.n_query;
    r.lo = start + (one ? first % a.n_query : 0);
    r.hi = start + (one ? last % a.n_query : a.n_query - 1);
  };
  Range rw{}, rg{};
  positions(row0, kRowsPerWave, rw);
  positions(block * kRows, kRows, rg);
  if (a.query_doc) {
    const bool of = stored && doc >= 0;
    int lo = of ? doc : INT_MAX, hi = of ? doc : -1;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
    rw.doc_lo = __builtin_amdgcn_readfirstlane(lo), rw.doc_hi = __builtin_amdgcn_readfirstlane(hi);
    rw.docs_whole = __all(!stored || doc >= 0);
    int* slot = reinterpret_cast<int*>(lds + LO::kRange);
    if (lane == 0) slot[4 * wave] = lo, slot[4 * wave + 1] = hi;
    __syncthreads();
    rg.doc_lo = INT_MAX, rg.doc_hi = -1, rg.docs_whole = false;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      rg.doc_lo = min(rg.doc_lo, __builtin_amdgcn_readfirstlane(slot[4 * i]));
      rg.doc_hi = max(rg.doc_hi, __builtin_amdgcn_readfirstlane(slot[4 * i + 1]));
    }
  }
  if (a.table)
    for (int g = 0; g < f.pack; ++g)
      fill_distances(a, reinterpret_cast<float*>(lds + LO::kDistances) + g * distance_words(a.buckets.reach), vh * f.pack + g,
                     64 * kWaves);

  // Reference maxima (exponents of 2; -inf until something attends) and row sums.
  float mref = -kInf, lsum = 0.0f, lsum32 = 0.0f;
  f32x16 o[TL::kCols];
#pragma unroll
  for (int dt = 0; dt < TL::kCols; ++dt) o[dt] = f32x16{};

  const T* kbase = a.k + b * a.ks[0] + kvh * a.ks[1];
  const T* vbase = a.v + b * a.vs[0] + kvh * a.vs[1];
  const int* kdocs = a.key_doc ? a.key_doc + static_cast<int64_t>(b) * a.n_key : nullptr;
  const uint32_t lds0 = lds_offset(lds);
  Walk<T> walk(a, rg, rw, row0 < f.rows, b, split, f.splits, f.tiles);
  const int limit = walk.limit;
  const int shift = kBias == 2 ? slope_shift(pos - index % kTile, limit) : 0;
  // Last of the keys that lengths and the causal mask leave the row.
  const int last = min(limit, a.causal ? max(pos + 1, walk.prefix) : INT_MAX) - 1;

  float next_mass = 0.0f;  // of wave 0: the loaded tile's, one key a lane
  const auto load = [&](int buf) {
    const int k0 = walk.tile * kTile;
    const auto live = [&](int j) { return kdocs == nullptr || kdocs[j] >= 0; };
    stage<T, D, kWaves>(kbase, a.ks[2], k0, limit, walk.in_whole, lds0 + (2 * buf) * TL::kBytes, live);
    stage<T, D, kWaves>(vbase, a.vs[2], k0, limit, walk.in_whole, lds0 + (2 * buf + 1) * TL::kBytes, live);
    if (wave == 0) {
      const int j = min(k0 + lane, a.n_key - 1);
      if (kdocs) lds_dma4(kdocs, j * 4u, lds0 + LO::kDocs + buf * kTile * 4);
      if (kBias && a.mass) next_mass = mass2(a, j);
    }
  };

  const float c = kBias ? 1.0f : kCap ? a.cap2 : a.scale * kLog2e;  // of x below to exponents of 2
  const auto compute = [&](bool partial, int k0, int buf) {
    const char* kt = lds + 2 * buf * TL::kBytes;
    const char* vt = kt + TL::kBytes;
    f32x16 s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      s[sub] = f32x16{};
#pragma unroll
      for (int t = 0; t < TL::kSteps; ++t) {
        const op8 ka = TL::rows_op(kt, 32 * sub, t);
        s[sub] = Op<T>::mma(ka, q[t], s[sub]);
      }
    }
    // Whether any score of the wave's tile is past the series' reach, and whether none is past the short one's.
    bool exact = false, low = false;
    if constexpr (kCap) {
      float most = fabsf(s[0][0]);
#pragma unroll
      for (int r = 1; r < 32; ++r) most = fmaxf(most, fabsf(s[r / 16][r % 16]));
      exact = __any(!(most <= a.cap_reach)), low = !__any(!(most <= a.cap_low));
    }
    // x = the scores of sub-tile sub, before the factor c, -inf where a pair does not attend.
    const auto scores = [&](int sub, float (&x)[16]) {
      const int j0 = 32 * sub + 4 * h;  // key of register r: k0 + j0 + 8 (r / 4) + r % 4
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = s[sub][r];
      if constexpr (kCap) {
        if (low) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = cap_low(a, x[r]);
        } else if (exact) {
          cap_all(a, x);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = cap_short(a, x[r]);
        }
      }
      if constexpr (kBias) {
        const float* mass = reinterpret_cast<const float*>(lds + LO::kMass) + buf * kTile + j0;
        const float to2 = kCap ? a.cap2 : a.scale * kLog2e;
        if (kBias == 1 || a.mass) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 m = *reinterpret_cast<const f32x4*>(mass + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = fmaf(x[4 * g + e], to2, m[e]);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= to2;
        }
      }
      if constexpr (kBias == 2) {
        if (a.slopes) {
          const float d0 = static_cast<float>(k0 + j0 - pos + shift);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            x[r] = fmaf(-slope, fabsf(d0 + static_cast<float>(8 * (r / 4) + r % 4)), x[r]);
        }
        if (a.table) {
          const int reach = a.buckets.reach;
          if (k0 + kTile - 1 - rw.lo <= -reach || k0 - rw.hi >= reach) {  // beyond the buckets' reach, all of it
            const float far = distance[k0 > rw.lo ? 2 * distance_zero(reach) : 0];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += far;
          } else {
            const float* near = distance + (k0 + j0 - pos + distance_zero(reach));
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += near[8 * (r / 4) + r % 4];
          }
        }
      }
      if (partial) {
        const int last_r = last - k0 - j0;  // keys past it do not attend
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 8 * (r / 4) + r % 4 <= last_r ? x[r] : -kInf;
        if (kdocs) {
          const int* tags = reinterpret_cast<const int*>(lds + LO::kDocs) + buf * kTile + j0;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const i32x4 tag = *reinterpret_cast<const i32x4*>(tags + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = tag[e] == doc ? x[4 * g + e] : -kInf;
          }
        }
      }
    };
    op8 p[4];  // probabilities as operands
    float x[2][16];
    scores(0, x[0]);
    scores(1, x[1]);
    float top = fmaxf(x[0][0], x[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(fmaxf(top, x[0][r]), x[1][r]);
    top = half_max(top) * c;
    if (__any(top > mref + kSlack + kLowerReference<T>)) {
      const float m = fmaxf(mref, top - kLowerReference<T>);
      const float alpha = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(mref - m);
      mref = m;
      lsum *= alpha, lsum32 *= alpha;
#pragma unroll
      for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    const float off = mref == -kInf ? 0.0f : -mref;
    float sum = 0.0f, sum32 = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; r += 2) {
      float& p0 = x[r / 16][r % 16] = __builtin_amdgcn_exp2f(fmaf(x[r / 16][r % 16], c, off));
      float& p1 = x[r / 16][r % 16 + 1] = __builtin_amdgcn_exp2f(fmaf(x[r / 16][r % 16 + 1], c, off));
      op8& to = p[r / 8];
      to[r % 8] = from_f32<T>(p0), to[r % 8 + 1] = from_f32<T>(p1);
      sum = add_pair<T>(sum, p0, p1, to[r % 8], to[r % 8 + 1]);
      if constexpr (kTrain) sum32 += p0 + p1;
    }
    lsum += sum, lsum32 += sum32;
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) {
      op8 left;
      if constexpr (kTrain == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          left[e] = from_f32<T>(x[kc / 2][8 * (kc % 2) + e] - to_f32(static_cast<T>(p[kc][e])));
      }
#pragma unroll
      for (int dt = 0; dt < TL::kCols; ++dt) {
        const op8 va = TL::cols_op(vt, dt, kc);
        o[dt] = Op<T>::mma(va, p[kc], o[dt]);
        if constexpr (kTrain == 2) o[dt] = Op<T>::mma(va, left, o[dt]);
      }
    }
  };

  bool more = walk.next();
  int buf = 0;
  if (more) load(0);
  while (more) {
    const int k0 = walk.tile * kTile;
    const bool mine = walk.in_mine, full = walk.in_full;
    more = walk.next();
    wait_vmem<0>();
    if (kBias && a.mass && wave == 0) reinterpret_cast<float*>(lds + LO::kMass)[buf * kTile + lane] = next_mass;
    __syncthreads();
    if (more) load(buf ^ 1);
    if (mine) compute(!full, k0, buf);
    buf ^= 1;
  }

  if (!stored) return;
  const bool dead = a.query_doc && doc < 0;
  float l = half_sum(lsum);
  // The gradients divide by the sum of the unrounded probabilities, which they compute again.
  float l32 = kTrain ? half_sum(lsum32) : l;
  if constexpr (kTrain == 2) l = l32;
  if (dead) l = l32 = 0.0f;
  if (f.splits > 1) {
    const int64_t row = (static_cast<int64_t>(split) * a.batch * vheads + b * vheads + vh) * f.rows + row0 +
                        l31;
    float* dst = f.part_o + row * D;
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g + 4 * h) =
            f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    if (h == 0) {
      f.part_ml[3 * row] = l == 0.0f ? -kInf : mref;
      f.part_ml[3 * row + 1] = l, f.part_ml[3 * row + 2] = l32;
    }
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* dst = f.out + b * a.os[0] + head * a.os[1] + index * a.os[2];
#pragma unroll
  for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0.0f : o[dt][4 * g + e] * inv;
      store4(dst + 32 * dt + 8 * g + 4 * h, y);
      if (f.rest) {
        const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.n_query + index;
        store4(f.rest + at * D + 32 * dt + 8 * g + 4 * h, rounding<T>(y));
      }
    }
  if (f.lse && h == 0)
    store_lse(f.lse, static_cast<int64_t>(a.batch) * a.heads * a.n_query,
              (static_cast<int64_t>(b) * a.heads + head) * a.n_query + index, mref, l32);
}

// Joins the splits' states of each row: D / 4 lanes a row, `f.joiners` of them that take every
// f.joiners-th split (many splits are few rows, where one lane would wait for each in turn).
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(const Forward<T> f) {
  const Args<T>& a = f.a;
  constexpr int kLanes = D / 4;
  __shared__ f32x4 sums[256];
  __shared__ f32x4 states[256];  // reference, row sums (rounded, unrounded)
  const int vheads = a.heads / f.pack, each = kLanes * f.joiners;
  const int64_t n = static_cast<int64_t>(a.batch) * vheads * f.rows;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / each) + static_cast<int>(threadIdx.x) / each;
  const int joiner = static_cast<int>(threadIdx.x) % each / kLanes, d = static_cast<int>(threadIdx.x) % kLanes * 4;
  float m = -kInf, l = 0.0f, l32 = 0.0f;
  f32x4 y{};
  const auto add = [&](float ms, float ls, float ls32, const f32x4& x) {
    if (ls == 0.0f) return;  // nothing attended there
    const float to = fmaxf(m, ms);
    const float was = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to), now = ms == to ? 1.0f : __builtin_amdgcn_exp2f(ms - to);
    m = to;
    l = fmaf(was, l, now * ls), l32 = fmaf(was, l32, now * ls32);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fmaf(was, y[e], now * x[e]);
  };
  if (row < n) {
#pragma unroll 4
    for (int s = joiner; s < f.splits; s += f.joiners) {
      const float* ml = f.part_ml + 3 * (s * n + row);
      const f32x4 x = *reinterpret_cast<const f32x4*>(f.part_o + (s * n + row) * D + d);
      add(ml[0], ml[1], ml[2], x);
    }
  }
  if (f.joiners > 1) {
    sums[threadIdx.x] = y, states[threadIdx.x] = f32x4{m, l, l32, 0.0f};
    __syncthreads();
    if (joiner > 0) return;
    for (int j = 1; j < f.joiners; ++j) {
      const f32x4 s = states[threadIdx.x + j * kLanes];
      add(s[0], s[1], s[2], sums[threadIdx.x + j * kLanes]);
    }
  }
  if (row >= n) return;
  const int vh = static_cast<int>(row / f.rows), r = static_cast<int>(row % f.rows);
  const int b = vh / vheads, head = vh % vheads * f.pack + r / a.n_query, i = r % a.n_query;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] *= inv;
  store4(f.out + b * a.os[0] + head * a.os[1] + i * a.os[2] + d, y);
  if (f.rest)
    store4(f.rest + ((static_cast<int64_t>(b) * a.heads + head) * a.n_query + i) * D + d, rounding<T>(y));
  if (f.lse && d == 0)
    store_lse(f.lse, static_cast<int64_t>(a.batch) * a.heads * a.n_query,
              (static_cast<int64_t>(b) * a.heads + head) * a.n_query + i, m, l32);
}

template <typename T, int D, bool kCap, int kBias, int kTrain>
int launch(const Forward<T>& f, hipStream_t stream) {
  typedef Layout<T, D> LO;
  const size_t bytes = LO::kDistances + (f.a.table ? static_cast<size_t>(f.pack) * distance_words(f.a.buckets.reach) * 4 : 0);
  const auto kernel = forward_kernel<T, D, kCap, kBias, kTrain>;
  const int status = allow_lds(kernel, bytes, "masked_attn");
  if (status != VGO_OK) return status;
  hipLaunchKernelGGL(kernel, dim3(f.tasks), dim3(64 * kWaves), bytes, stream, f);
  return check_launch("masked_attn");
}

// The kernel without the rules that the problem does not have: kBias 1 has masses alone, 2 slopes or a table too.
template <typename T, int D>
int choose(const Forward<T>& f, hipStream_t stream) {
  const int bias = f.a.slopes || f.a.table ? 2 : f.a.mass ? 1 : 0;
  const auto with = [&](auto cap) {
    constexpr bool kCap = decltype(cap)::value;
    if constexpr (sizeof(T) == 2)
      if (f.lse && f.a.slopes) return launch<T, D, kCap, 2, 2>(f, stream);
    if constexpr (std::is_same<T, bf16_t>::value)
      if (f.lse)
        return bias == 0   ? launch<T, D, kCap, 0, 1>(f, stream)
               : bias == 1 ? launch<T, D, kCap, 1, 1>(f, stream)
                           : launch<T, D, kCap, 2, 1>(f, stream);
    return bias == 0   ? launch<T, D, kCap, 0, 0>(f, stream)
           : bias == 1 ? launch<T, D, kCap, 1, 0>(f, stream)
                       : launch<T, D, kCap, 2, 0>(f, stream);
  };
  return f.a.cap2 != 0.0f ? with(std::true_type{}) : with(std::false_type{});
}

template <typename T, int D>
int run(const vgo_masked_attn* p, const ForwardPlan& plan, void* out, const int64_t out_stride[3], float* lse, void* rest,
        char* ws, hipStream_t stream) {
  Forward<T> f{};
  f.a = make_args<T>(p);
  for (int i = 0; i < 3; ++i) f.a.os[i] = out_stride[i];
  f.out = static_cast<T*>(out), f.lse = lse, f.rest = static_cast<T*>(rest);
  f.pack = plan.pack, f.rows = plan.rows, f.row_blocks = plan.row_blocks, f.splits = plan.splits;
  f.tiles = plan.tiles, f.tasks = static_cast<int>(plan.tasks);
  launch_info(p, f.a, ws, stream);
  const int64_t rows = p->batch * (p->heads / plan.pack) * plan.rows;
  if (plan.splits > 1) {
    f.part_o = reinterpret_cast<float*>(ws + info_bytes(p));
    f.part_ml = reinterpret_cast<float*>(ws + info_bytes(p) + align16(plan.splits * rows * p->head_dim * 4));
  }
  const int status = choose<T, D>(f, stream);
  if (status != VGO_OK || plan.splits == 1) return status;
  f.joiners = 1;
  while (f.joiners < 256 / (D / 4) && 2 * f.joiners < plan.splits && rows * (D / 4) * f.joiners < 256LL * 2 * device_cus())
    f.joiners *= 2;
  const int64_t each = 256 / (D / 4 * f.joiners);  // rows per work-group
  hipLaunchKernelGGL((join_kernel<T, D>), dim3(static_cast<unsigned>((rows + each - 1) / each)), dim3(256), 0, stream, f);
  return check_launch("masked_attn join");
}

}  // namespace

template <typename T>
int run_forward(const vgo_masked_attn* p, const ForwardPlan& plan, void* out, const int64_t out_stride[3], float* lse,
                void* rest, char* ws, hipStream_t stream) {
  return p->head_dim == 128 ? run<T, 128>(p, plan, out, out_stride, lse, rest, ws, stream)
                            : run<T, 64>(p, plan, out, out_stride, lse, rest, ws, stream);
}

}  // namespace masked
}  // namespace vgo
