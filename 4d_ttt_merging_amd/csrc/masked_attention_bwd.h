// Gradients of the masked attention (rules and layouts: masked_attention.h).
//
//   P = exp2(x - lse) exp2(-lse's rest) with the forward's row sums;  D_i = dO_i . O_i;  dZ = P (dO V^T - D)
//   dV = P^T dO;  dK = scale (dZ cap')^T Q;  dQ = scale (dZ cap') K;  cap' = 1 - tanh^2
//   d log_mass_j = sum dZ;  d slope = -sum dZ |r|;  d table[t] = sum of dZ over the pairs of bucket t
//
// Two kernels, so that every sum has one owner and a fixed order (no atomics): one holds 32 keys a
// wave and runs over the query tiles of all heads that share them (dK, dV, d log_mass), one holds 32
// queries a wave and runs over the key tiles (dQ, d slope, d table).  Both recompute the scores: seven
// products in place of five.
//
// Bound: as the forward's, no pipe full (matrix and vector busy 0.52 and 0.66 of the time in dQ, 0.42 and 0.50 in dK and
// dV with 64 channels, 0.54 and 0.40, 0.42 and 0.30 with 128).  16 heads of 8,232 x 8,232 in bf16: dQ 479 us (0.87
// PFLOP/s of its three products), dK and dV 714 (0.78 of four) with 64 channels, 883 and 1,413 (0.94 and 0.79) with
// 128; f16 504 and 781, whose dV takes P raised; fp32 2,058 x 2,058: 270 and 377 (96 and 92 of 140 TFLOP/s, matrix
// pipes busy 0.76 and 0.72).  D comes in a pass of its own, bound by HBM: 17 us for 16 x 8,232 x 128.
#pragma once

#include "masked_attention.h"

namespace vgo {
namespace masked {

constexpr int kRowWaves = 4, kRowBlock = 32 * kRowWaves;  // of the kernel that holds queries

// Of the kernel that holds keys.  LDS: Q and dO tiles (two buffers), lse, delta and documents of their rows, distance biases.
template <typename T, int D>
struct KeyLds {
  static constexpr bool kValues = sizeof(T) == 2;  // V of the wave's keys in LDS, not in registers
  static constexpr int kWaves = sizeof(T) == 2 && D == 128 ? 8 : 4, kBlock = 32 * kWaves;
  static constexpr int kV = 4 * Tile<T, D>::kBytes, kLse = kV + (kValues ? kWaves * Tile<T, D>::kBytes / 2 : 0);
  static constexpr int kDelta = kLse + 2 * kTile * 4, kDocs = kDelta + 2 * kTile * 4;
  static constexpr int kDistances = kDocs + 2 * kTile * 4;
};

struct GradPlan {
  int key_blocks, row_blocks, splits, row_splits, query_tiles, key_tiles;
  int64_t key_tasks, row_tasks;
};
GradPlan grad_plan(const vgo_masked_attn* p, int dtype);

// Workspace pieces in order; each a multiple of 16 bytes.
struct GradPieces {
  size_t delta, marks, kv, q, mass, slopes, table, bytes;
};
GradPieces grad_pieces(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, const GradPlan& plan);

// The launches of one type (instantiated in masked_attention_grad_bf16.hip and its like).
template <typename T>
int run_grad(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, const GradPlan& plan, char* ws,
             hipStream_t stream);
extern template int run_grad<bf16_t>(const vgo_masked_attn*, const vgo_masked_attn_grads*, const GradPlan&, char*,
                                 hipStream_t);
extern template int run_grad<f16_t>(const vgo_masked_attn*, const vgo_masked_attn_grads*, const GradPlan&, char*,
                                 hipStream_t);
extern template int run_grad<float>(const vgo_masked_attn*, const vgo_masked_attn_grads*, const GradPlan&, char*,
                                 hipStream_t);

namespace {

template <typename T>
struct Grad {
  Args<T> a;
  const T *o, *go, *rest;
  int64_t gos[3];
  const float *lse, *lse_rest;  // the two planes
  float* delta;          // [batch, heads, n_query], -D; 0 for rows that attend to nothing
  unsigned char* marks;  // [batch, heads, query tiles]: kEmpty and kRests of the tile's rows
  T *dq, *dk, *dv;       // dq null: not wanted; likewise dk and dv
  int64_t dqs[3], dks[3], dvs[3];
  float* part_kv;      // splits > 1: [splits, batch * kv_heads, n_key, 2 D]
  float* part_q;       // row_splits > 1: [row_splits, batch * heads, n_query, D]
  float* part_mass;    // [splits * batch * kv_heads, n_key] or null
  float* part_slopes;  // [row_splits * batch * row_blocks, heads] or null
  float* part_table;   // [row_splits * batch * row_blocks, n_buckets, heads] or null
  int query_tiles, key_tiles, splits, row_splits;
  int key_blocks, row_blocks, key_tasks, row_tasks;
};

// A tile's marks: a row attends to nothing; a row's lse left a rest past the rounding of a score of 64.  Such tiles are
// done as partly masked ones are, whose probabilities take the rest as a factor; the others are spared it (a subtraction
// in all of them, or the rests beside lse in LDS, was 1 to 3% of the keys' kernel).
constexpr unsigned char kEmpty = 1, kRests = 2;
constexpr float kRestReach = 0x1p-18f;

// delta and marks (delta from the unrounded outputs where their rest is there: what it is off by is off in every
// score of the row): a work-group per tile of one head, 16 bytes a lane, every load of a lane's rows in flight
// together.
template <typename T, int D>
__global__ __launch_bounds__(256) void delta_kernel(const Grad<T> f) {
  const Args<T>& a = f.a;
  constexpr int kEach = 16 / sizeof(T), kLanes = D / kEach, kStep = 256 / kLanes, kTimes = kTile / kStep;
  typedef T Part __attribute__((ext_vector_type(kEach)));
  const int tile = blockIdx.x % f.query_tiles, bh = blockIdx.x / f.query_tiles;
  const int b = bh / a.heads, head = bh % a.heads;
  const int part = threadIdx.x % kLanes, i0 = tile * kTile + threadIdx.x / kLanes;
  const T* o = f.o + b * a.os[0] + head * a.os[1] + part * kEach;
  const T* go = f.go + b * f.gos[0] + head * f.gos[1] + part * kEach;
  const int64_t row0 = static_cast<int64_t>(bh) * a.n_query;
  Part x[kTimes], y[kTimes], z[kTimes];
  float lse[kTimes], rest[kTimes];
#pragma unroll
  for (int t = 0; t < kTimes; ++t) {
    const int i = min(i0 + t * kStep, a.n_query - 1);
    x[t] = *reinterpret_cast<const Part*>(o + i * a.os[2]);
    y[t] = *reinterpret_cast<const Part*>(go + i * f.gos[2]);
    z[t] = f.rest ? *reinterpret_cast<const Part*>(f.rest + (row0 + i) * D + part * kEach) : Part{};
    lse[t] = f.lse[row0 + i], rest[t] = f.lse_rest[row0 + i];
  }
  bool none = false, rests = false;
#pragma unroll
  for (int t = 0; t < kTimes; ++t) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum = fmaf(to_f32(x[t][e]) + to_f32(z[t][e]), to_f32(y[t][e]), sum);
#pragma unroll
    for (int off = 1; off < kLanes; off <<= 1) sum += __shfl_xor(sum, off);
    const int i = i0 + t * kStep;
    const bool empty = lse[t] == kInf;
    none = none || (empty && i < a.n_query);
    rests = rests || fabsf(rest[t]) > kRestReach;
    if (part == 0 && i < a.n_query) f.delta[row0 + i] = empty ? 0.0f : -sum;
  }
  const bool any = __syncthreads_or(none), any_rests = __syncthreads_or(rests);
  if (threadIdx.x == 0) f.marks[blockIdx.x] = (any ? kEmpty : 0) | (any_rests ? kRests : 0);
}

// Raw products of one 32 x 32 block to what the factor returned makes exponents of 2; with a cap, to
// their tanh, and cap' in `bend`.
template <typename T, bool kCap>
__device__ __forceinline__ float rescore(const Args<T>& a, float (&x)[16], float (&bend)[16]) {
  if constexpr (!kCap) {
    return a.scale * kLog2e;
  } else {
    float most = fabsf(x[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) most = fmaxf(most, fabsf(x[r]));
    if (!__any(!(most <= a.cap_low))) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = cap_low(a, x[r]);
    } else if (__any(!(most <= a.cap_reach))) {
      cap_all(a, x);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = cap_short(a, x[r]);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) bend[r] = fmaf(-x[r], x[r], 1.0f);
    return a.cap2;
  }
}

// ------------------------------------------------------------ keys' side ----
template <typename T, int D, bool kCap, int kBias>
__global__ __launch_bounds__((64 * KeyLds<T, D>::kWaves), sizeof(T) == 4 ? 1 : D == 64 ? 3 : 2) void key_kernel(const Grad<T> f) {
  typedef Tile<T, D> TL;
  typedef KeyLds<T, D> LO;
  constexpr int kWaves = LO::kWaves, kBlock = LO::kBlock;
  typedef typename Op<T>::op8 op8;
  extern __shared__ __align__(16) char lds[];
  const Args<T>& a = f.a;
  const int lane = lane_id(), l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.heads / a.kv_heads;

  int task = xcd_remap(blockIdx.x, f.key_tasks);
  const int block = zigzag(task % f.key_blocks, f.key_blocks, task / f.key_blocks, f.key_tasks / f.key_blocks);
  task /= f.key_blocks;
  const int split = task % f.splits;
  task /= f.splits;
  const int kvh = task % a.kv_heads, b = task / a.kv_heads;
  const int start = first_position(a, b), limit = key_limit(a, b), prefix = prefix_of(a, b);
  const int key = block * kBlock + 32 * wave + l32;
  const int doc = a.key_doc && key < a.n_key ? a.key_doc[static_cast<int64_t>(b) * a.n_key + key] : 0;
  const bool taken = key < limit && doc >= 0;
  const float mass = a.mass && key < a.n_key ? mass2(a, key) : 0.0f;

  op8 k[TL::kSteps], v[LO::kValues ? 1 : TL::kSteps];
  const char* vl = lds + LO::kV + wave * (TL::kBytes / 2);
  {
    const T* kp = a.k + b * a.ks[0] + kvh * a.ks[1] + static_cast<int64_t>(min(key, a.n_key - 1)) * a.ks[2] + 8 * h;
    const T* vp = a.v + b * a.vs[0] + kvh * a.vs[1] + static_cast<int64_t>(min(key, a.n_key - 1)) * a.vs[2] + 8 * h;
#pragma unroll
    for (int t = 0; t < TL::kSteps; ++t) {
      k[t] = taken ? *reinterpret_cast<const op8*>(kp + 16 * t) : op8{};
      const op8 x = taken ? *reinterpret_cast<const op8*>(vp + 16 * t) : op8{};
      if constexpr (LO::kValues)
        *reinterpret_cast<op8*>(lds + LO::kV + wave * (TL::kBytes / 2) + TL::rows_at(0, t)) = x;
      else
        v[t] = x;
    }
  }
  // Ranges of the work-group's and the wave's keys; rows that are none's narrow only the documents.
  Range rg{}, rw{};
  rg.lo = block * kBlock, rg.hi = min(rg.lo + kBlock, limit) - 1;
  rw.lo = rg.lo + 32 * wave, rw.hi = min(rw.lo + 32, limit) - 1;
  if (a.key_doc) {
    int lo = taken ? doc : INT_MAX, hi = taken ? doc : -1;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
    rw.doc_lo = __builtin_amdgcn_readfirstlane(lo), rw.doc_hi = __builtin_amdgcn_readfirstlane(hi);
    rw.docs_whole = __all(taken);
    constexpr int kSpan = kBlock / kTile;
    const int tiles = (a.n_key + kTile - 1) / kTile, t0 = kSpan * block;
    rg.doc_lo = INT_MAX, rg.doc_hi = -1, rg.docs_whole = false;
    for (int t = t0; t < min(t0 + kSpan, tiles); ++t) {
      const Range r = info_range(a.key_info[static_cast<int64_t>(b) * tiles + t]);
      rg.doc_lo = min(rg.doc_lo, r.doc_lo), rg.doc_hi = max(rg.doc_hi, r.doc_hi);
    }
  }

  // The rows that lengths and the causal mask let attend to the lane's key: row_count from first_row on.
  const int first_row = a.causal && key >= prefix ? max(0, key - start) : 0;
  const unsigned row_count = taken && first_row < a.n_query ? a.n_query - first_row : 0;

  f32x16 dk[TL::kCols], dv[TL::kCols];
#pragma unroll
  for (int dt = 0; dt < TL::kCols; ++dt) dk[dt] = dv[dt] = f32x16{};
  LongSum mass_sums;

  // (head of the group, query tile) units of this split, every f.splits-th, 64 judged at a time.
  const int end = rg.lo < limit ? group * f.query_tiles : 0;
  int base = -64, unit = 0, unit_head = 0, unit_tile = 0;
  uint64_t todo = 0, mine = 0, full = 0, whole = 0;
  bool in_mine = false, in_full = false, in_whole = false;
  const auto next = [&]() {
    while (todo == 0) {
      base += 64;
      if (split + f.splits * base >= end) return false;
      const int u = split + f.splits * (base + lane), g = u / f.query_tiles, t = u % f.query_tiles;
      bool any = u < end, any_w = false, all_w = false, all = false, inside = false;
      if (any) {
        Range r{};
        if (a.key_doc) r = info_range(a.query_info[static_cast<int64_t>(b) * f.query_tiles + t]);
        r.lo = start + t * kTile, r.hi = start + min(t * kTile + kTile, a.n_query) - 1;
        judge(a, r, rg, prefix, any, all);
        judge(a, r, rw, prefix, any_w, all_w);
        inside = t * kTile + kTile <= a.n_query;
        all_w = all_w && inside && rw.hi == rw.lo + 31;
        any_w = any_w && rw.lo < limit;
        const int marks = f.marks[(static_cast<int64_t>(b) * a.heads + kvh * group + g) * f.query_tiles + t];
        inside = inside && !(marks & kEmpty);
        all_w = all_w && !(marks & kRests);
      }
      todo = __ballot(any), mine = __ballot(any && any_w), full = __ballot(all_w), whole = __ballot(inside);
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    unit = split + f.splits * (base + bit);
    unit_head = kvh * group + unit / f.query_tiles, unit_tile = unit % f.query_tiles;
    in_mine = mine >> bit & 1, in_full = full >> bit & 1, in_whole = whole >> bit & 1;
    return true;
  };
  const uint32_t lds0 = lds_offset(lds);
  const auto load = [&](int buf) {
    const int q0 = unit_tile * kTile;
    const float* lse = f.lse + (static_cast<int64_t>(b) * a.heads + unit_head) * a.n_query;
    const float* delta = f.delta + (static_cast<int64_t>(b) * a.heads + unit_head) * a.n_query;
    const auto live = [&](int i) { return lse[i] != kInf; };
    stage<T, D, kWaves>(a.q + b * a.qs[0] + unit_head * a.qs[1], a.qs[2], q0, a.n_query, in_whole,
                        lds0 + 2 * buf * TL::kBytes, live);
    stage<T, D, kWaves>(f.go + b * f.gos[0] + unit_head * f.gos[1], f.gos[2], q0, a.n_query, in_whole,
                        lds0 + (2 * buf + 1) * TL::kBytes, live);
    const uint32_t i = min(q0 + lane, a.n_query - 1) * 4u;
    if (wave == 0) lds_dma4(lse, i, lds0 + LO::kLse + buf * kTile * 4);
    if (wave == 1) lds_dma4(delta, i, lds0 + LO::kDelta + buf * kTile * 4);
    if (wave == 2 && a.key_doc)
      lds_dma4(a.query_doc + static_cast<int64_t>(b) * a.n_query, i, lds0 + LO::kDocs + buf * kTile * 4);
  };

  float slope = 0.0f;
  const auto compute = [&](bool partial, int q0, int head, int buf) {
    const char* qt = lds + 2 * buf * TL::kBytes;
    const char* gt = qt + TL::kBytes;
    const float* lse = reinterpret_cast<const float*>(lds + LO::kLse) + buf * kTile;
    const float* delta = reinterpret_cast<const float*>(lds + LO::kDelta) + buf * kTile;
    const int* tags = reinterpret_cast<const int*>(lds + LO::kDocs) + buf * kTile;
    const int p0 = start + q0;  // position of the tile's first row
    // S, dV, dP, dK: P becomes an operand before dP's registers are there, and dP starts from -D.
    // One 32-row half at a time, and the scheduling barriers, keep what is live within the registers
    // that two waves (64 channels: three) a SIMD leave: without them the compiler reads operands ahead and
    // spills.
#pragma unroll 1
    for (int sub = 0; sub < 2; ++sub) {
      f32x16 s{};
#pragma unroll
      for (int t = 0; t < TL::kSteps; ++t) s = Op<T>::mma(TL::rows_op(qt, 32 * sub, t), k[t], s);
      const int i0 = 32 * sub + 4 * h;  // row of register r: q0 + i0 + 8 (r / 4) + r % 4
      __builtin_amdgcn_sched_barrier(0);
      float x[16], bend[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = s[r];
      const float c = rescore<T, kCap>(a, x, bend);
      if constexpr (kBias) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], c, mass);
      }
      if constexpr (kBias == 2) {
        if (a.slopes) {
          const float d0 = static_cast<float>(key - p0 + slope_shift(p0, limit) - i0);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            x[r] = fmaf(-slope, fabsf(d0 - static_cast<float>(8 * (r / 4) + r % 4)), x[r]);
        }
        if (a.table) {
          const float* distance = reinterpret_cast<const float*>(lds + LO::kDistances);
          const int reach = a.buckets.reach;
          if (rw.lo + 31 - p0 <= -reach || rw.lo - (p0 + kTile - 1) >= reach) {
            const float far = distance[rw.lo > p0 ? 2 * distance_zero(reach) : 0];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += far;
          } else {
            const float* near = distance + (key - p0 - i0 + distance_zero(reach));
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += near[-(8 * (r / 4) + r % 4)];
          }
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse + i0 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          x[r] = __builtin_amdgcn_exp2f(kBias ? x[r] - l4[e] : fmaf(x[r], c, -l4[e]));
        }
      }
      if (partial) {
        const int64_t bh = static_cast<int64_t>(b) * a.heads + head;
        if (__builtin_expect(f.marks[bh * f.query_tiles + q0 / kTile] & kRests, 0)) {
          const float* rest = f.lse_rest + bh * a.n_query;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            x[r] *= __builtin_amdgcn_exp2f(-rest[min(q0 + i0 + 8 * (r / 4) + r % 4, a.n_query - 1)]);
        }
        const int i_first = q0 + i0 - first_row;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[r] = static_cast<unsigned>(i_first + 8 * (r / 4) + r % 4) < row_count ? x[r] : 0.0f;
        if (a.key_doc) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const i32x4 tag = *reinterpret_cast<const i32x4*>(tags + i0 + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = tag[e] == doc ? x[4 * g + e] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const op8 pb = as_op<T, kRaise<T>>(x, half);
#pragma unroll
        for (int dt = 0; dt < TL::kCols; ++dt) dv[dt] = Op<T>::mma(TL::cols_op(gt, dt, 2 * sub + half), pb, dv[dt]);
      }
      if constexpr (kCap && !kBias) {  // nothing else needs P alone
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= bend[r];
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 dp;  // starts from -D
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(delta + i0 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * g + e] = d4[e];
      }
#pragma unroll
      for (int t = 0; t < TL::kSteps; ++t)
        dp = Op<T>::mma(TL::rows_op(gt, 32 * sub, t), LO::kValues ? TL::rows_op(vl, 0, t) : v[LO::kValues ? 0 : t], dp);
      __builtin_amdgcn_sched_barrier(0);
      float dz[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) dz[r] = x[r] * dp[r];
      if constexpr (kBias) {
        if (f.part_mass) {
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += dz[r];
          mass_sums.add(sum);
        }
        if constexpr (kCap) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dz[r] *= bend[r];
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const op8 zb = as_op<T>(dz, half);
#pragma unroll
        for (int dt = 0; dt < TL::kCols; ++dt) dk[dt] = Op<T>::mma(TL::cols_op(qt, dt, 2 * sub + half), zb, dk[dt]);
      }
    }
  };

  bool more = next();
  int buf = 0, distance_head = -1;
  if (more) load(0);
  while (more) {
    const int q0 = unit_tile * kTile, head = unit_head;
    const bool run = in_mine, all = in_full;
    if (kBias == 2 && head != distance_head) {
      if (a.table) {
        __syncthreads();  // (where the last reads of the head before end)
        fill_distances(a, reinterpret_cast<float*>(lds + LO::kDistances), head, 64 * kWaves);
      }
      // Here, where no DMA but the one about to be waited for is in flight: a load's wait is a wait for all of them.
      slope = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, slope2(a, head))));
      distance_head = head;
    }
    more = next();
    wait_vmem<0>();
    __syncthreads();
    if (more) load(buf ^ 1);
    if (run) compute(!all, q0, head, buf);
    buf ^= 1;
  }

  const int64_t bk = static_cast<int64_t>(b) * a.kv_heads + kvh;
  if (f.part_mass) {
    const float mass_sum = half_sum(mass_sums.sum);
    if (h == 0 && key < a.n_key)
      f.part_mass[(static_cast<int64_t>(split) * a.batch * a.kv_heads + bk) * a.n_key + key] = mass_sum;
  }
  if (!f.dk || key >= a.n_key) return;
  constexpr float lower = 1.0f / (1 << kRaise<T>);
  if (f.splits > 1) {
    float* dst = f.part_kv + ((static_cast<int64_t>(split) * a.batch * a.kv_heads + bk) * a.n_key + key) * (2 * D);
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = dk[dt][4 * g + e] * a.scale, y[e] = dv[dt][4 * g + e] * lower;
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g + 4 * h) = x;
        *reinterpret_cast<f32x4*>(dst + D + 32 * dt + 8 * g + 4 * h) = y;
      }
    return;
  }
  T* kd = f.dk + b * f.dks[0] + kvh * f.dks[1] + key * f.dks[2];
  T* vd = f.dv + b * f.dvs[0] + kvh * f.dvs[1] + key * f.dvs[2];
#pragma unroll
  for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dk[dt][4 * g + e] * a.scale, y[e] = dv[dt][4 * g + e] * lower;
      store4(kd + 32 * dt + 8 * g + 4 * h, x);
      store4(vd + 32 * dt + 8 * g + 4 * h, y);
    }
}

// dK and dV of split work: four values a lane, the splits in order.  Bound: HBM, 14.5 us for two splits of 2 x 16 x
// 2,058 x 64.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_keys_kernel(const Grad<T> f) {
  const Args<T>& a = f.a;
  constexpr int kLanes = 2 * D / 4;
  const int64_t n = static_cast<int64_t>(a.batch) * a.kv_heads * a.n_key;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  if (row >= n) return;
  const int d = static_cast<int>(threadIdx.x) % kLanes * 4;
  f32x4 y{};
  for (int s = 0; s < f.splits; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(f.part_kv + (s * n + row) * (2 * D) + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += x[e];
  }
  const int key = static_cast<int>(row % a.n_key), bk = static_cast<int>(row / a.n_key);
  const int kvh = bk % a.kv_heads, b = bk / a.kv_heads;
  if (d < D)
    store4(f.dk + b * f.dks[0] + kvh * f.dks[1] + key * f.dks[2] + d, y);
  else
    store4(f.dv + b * f.dvs[0] + kvh * f.dvs[1] + key * f.dvs[2] + (d - D), y);
}

// --------------------------------------------------------- queries' side ----
// LDS: K and V tiles (two buffers; one where two leave no room for the rest), masses and documents of
// their keys, distance biases; for the table's gradient, per wave a sheared 32 x 32 block of dZ (rows of
// kShear words: 16-byte reads spread over the banks) and the sums by distance.
template <typename T, int D>
struct RowLds {
  static constexpr int kBuffers = sizeof(T) == 4 && D == 128 ? 1 : 2;
  static constexpr int kMass = 2 * kBuffers * Tile<T, D>::kBytes, kDocs = kMass + 2 * kTile * 4;
  static constexpr int kSums = kDocs + 2 * kTile * 4;  // the waves' slope sums
  static constexpr int kDistances = kSums + kRowWaves * 16;
};
constexpr int kShear = 36, kDiagonal = 63 * kShear;  // words
__host__ __device__ inline int sum_words(int reach) { return (2 * reach + 4) & ~3; }

// kBias 3: with the table's gradient, whose registers and LDS leave two work-groups a CU (64 channels; three without:
// 2 x 16 heads of 4,116 with slopes 277 us against 352, with a table 306 against 385).
template <typename T, int D, bool kCap, int kBias>
__global__ __launch_bounds__(64 * kRowWaves, sizeof(T) == 4 ? 1 : D == 64 && kBias < 3 ? 3 : 2) void row_kernel(const Grad<T> f) {
  typedef Tile<T, D> TL;
  typedef RowLds<T, D> LO;
  typedef typename Op<T>::op8 op8;
  extern __shared__ __align__(16) char lds[];
  const Args<T>& a = f.a;
  const int lane = lane_id(), l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int task = xcd_remap(blockIdx.x, f.row_tasks);
  const int block = f.row_blocks - 1 - zigzag(task % f.row_blocks, f.row_blocks, task / f.row_blocks, f.row_tasks / f.row_blocks);
  task /= f.row_blocks;
  const int split = task % f.row_splits;
  task /= f.row_splits;
  const int head = task % a.heads, b = task / a.heads, kvh = head / (a.heads / a.kv_heads);
  const int start = first_position(a, b), limit = key_limit(a, b), prefix = prefix_of(a, b);
  const int row0 = block * kRowBlock + 32 * wave, row = row0 + l32, rc = min(row, a.n_query - 1);
  const bool stored = row < a.n_query;
  const int pos = start + row;
  const int doc = a.query_doc ? a.query_doc[static_cast<int64_t>(b) * a.n_query + rc] : 0;
  const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.n_query + rc;
  const float lse = stored ? f.lse[at] : kInf, lse_rest = f.lse_rest[at], unrest = __builtin_amdgcn_exp2f(-lse_rest);
  const bool rests = __any(fabsf(lse_rest) > kRestReach);
  const bool live = lse != kInf;
  const float delta = live ? f.delta[at] : 0.0f;
  const float slope = slope2(a, head);
  const int shift = kBias >= 2 ? slope_shift(start + row - row % kTile, limit) : 0;

  const int last = min(limit, a.causal ? max(pos + 1, prefix) : INT_MAX) - 1;  // key that may attend

  op8 q[TL::kSteps], go[TL::kSteps];
  {
    const T* qp = a.q + b * a.qs[0] + head * a.qs[1] + rc * a.qs[2] + 8 * h;
    const T* gp = f.go + b * f.gos[0] + head * f.gos[1] + rc * f.gos[2] + 8 * h;
#pragma unroll
    for (int t = 0; t < TL::kSteps; ++t) {
      q[t] = live ? *reinterpret_cast<const op8*>(qp + 16 * t) : op8{};
      go[t] = live ? *reinterpret_cast<const op8*>(gp + 16 * t) : op8{};
    }
  }
  Range rg{}, rw{};
  rg.lo = start + block * kRowBlock, rg.hi = start + min(block * kRowBlock + kRowBlock, a.n_query) - 1;
  rw.lo = start + row0, rw.hi = start + min(row0 + 32, a.n_query) - 1;
  if (a.query_doc) {
    const bool of = stored && doc >= 0;
    int lo = of ? doc : INT_MAX, hi = of ? doc : -1;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
    rw.doc_lo = __builtin_amdgcn_readfirstlane(lo), rw.doc_hi = __builtin_amdgcn_readfirstlane(hi);
    rw.docs_whole = __all(!stored || doc >= 0);
    rg.doc_lo = INT_MAX, rg.doc_hi = -1, rg.docs_whole = false;
    for (int t = 2 * block; t < min(2 * block + 2, f.query_tiles); ++t) {
      const Range r = info_range(a.query_info[static_cast<int64_t>(b) * f.query_tiles + t]);
      rg.doc_lo = min(rg.doc_lo, r.doc_lo), rg.doc_hi = max(rg.doc_hi, r.doc_hi);
    }
  }
  float* distance = reinterpret_cast<float*>(lds + LO::kDistances);
  const int words = sum_words(a.buckets.reach);
  float* diagonal = distance + distance_words(a.buckets.reach) + wave * kDiagonal;
  float* sums = distance + distance_words(a.buckets.reach) + kRowWaves * kDiagonal + wave * words;
  if (kBias >= 2 && a.table) fill_distances(a, distance, head, 64 * kRowWaves);
  if (kBias == 3) {
    for (int i = lane; i < words; i += 64) sums[i] = 0.0f;
    for (int i = lane; i < kDiagonal; i += 64) diagonal[i] = 0.0f;
    wave_lds_order();
  }

  f32x16 dq[TL::kCols];
#pragma unroll
  for (int dt = 0; dt < TL::kCols; ++dt) dq[dt] = f32x16{};
  LongSum slope_sum, far_behind, far_ahead;

  const T* kbase = a.k + b * a.ks[0] + kvh * a.ks[1];
  const T* vbase = a.v + b * a.vs[0] + kvh * a.vs[1];
  const int* kdocs = a.key_doc ? a.key_doc + static_cast<int64_t>(b) * a.n_key : nullptr;
  const uint32_t lds0 = lds_offset(lds);

  // Key tiles of this split, every f.row_splits-th.
  const int end = min((limit + kTile - 1) / kTile, f.key_tiles);
  int base = -64, tile = 0;
  uint64_t todo = 0, mine = 0, full = 0, whole = 0;
  bool in_mine = false, in_full = false, in_whole = false;
  const auto next = [&]() {
    while (todo == 0) {
      base += 64;
      if (split + f.row_splits * base >= end) return false;
      const int t = split + f.row_splits * (base + lane);
      bool any = t < end, any_w = false, all_w = false, all = false, inside = false;
      if (any) {
        Range r{};
        if (kdocs) r = info_range(a.key_info[static_cast<int64_t>(b) * f.key_tiles + t]);
        r.lo = t * kTile, r.hi = min(r.lo + kTile, limit) - 1;
        judge(a, rg, r, prefix, any, all);
        judge(a, rw, r, prefix, any_w, all_w);
        inside = r.lo + kTile <= limit;
        all_w = all_w && inside;
        any_w = any_w && row0 < a.n_query;
        inside = inside && (!kdocs || r.docs_whole);
      }
      todo = __ballot(any), mine = __ballot(any && any_w), full = __ballot(all_w), whole = __ballot(inside);
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    tile = split + f.row_splits * (base + bit);
    in_mine = mine >> bit & 1, in_full = full >> bit & 1, in_whole = whole >> bit & 1;
    return true;
  };
  float next_mass = 0.0f;  // of wave 0: the loaded tile's, one key a lane
  const auto load = [&](int buf) {
    const int k0 = tile * kTile;
    const auto kept = [&](int j) { return kdocs == nullptr || kdocs[j] >= 0; };
    const uint32_t to = lds0 + 2 * (LO::kBuffers == 2 ? buf : 0) * TL::kBytes;
    stage<T, D, kRowWaves>(kbase, a.ks[2], k0, limit, in_whole, to, kept);
    stage<T, D, kRowWaves>(vbase, a.vs[2], k0, limit, in_whole, to + TL::kBytes, kept);
    if (wave == 0) {
      const int j = min(k0 + lane, a.n_key - 1);
      if (kdocs) lds_dma4(kdocs, j * 4u, lds0 + LO::kDocs + buf * kTile * 4);
      if (kBias && a.mass) next_mass = mass2(a, j);
    }
  };

  const auto compute = [&](bool partial, int k0, int buf) {
    const char* kt = lds + 2 * (LO::kBuffers == 2 ? buf : 0) * TL::kBytes;
    const char* vt = kt + TL::kBytes;
    const float* mass = reinterpret_cast<const float*>(lds + LO::kMass) + buf * kTile;
    const int* tags = reinterpret_cast<const int*>(lds + LO::kDocs) + buf * kTile;
    const int reach = a.buckets.reach;
    const bool behind = k0 + kTile - 1 - rw.lo <= -reach, ahead = k0 - (rw.lo + 31) >= reach;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      f32x16 s{}, dp{};
#pragma unroll
      for (int t = 0; t < TL::kSteps; ++t) s = Op<T>::mma(TL::rows_op(kt, 32 * sub, t), q[t], s);
#pragma unroll
      for (int t = 0; t < TL::kSteps; ++t) dp = Op<T>::mma(TL::rows_op(vt, 32 * sub, t), go[t], dp);
      const int j0 = 32 * sub + 4 * h;
      float x[16], bend[16], dz[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = s[r], dz[r] = dp[r];
      const float c = rescore<T, kCap>(a, x, bend);
      const float d0f = static_cast<float>(k0 + j0 - pos + shift);
      if constexpr (kBias) {
        if (kBias == 1 || a.mass) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 m = *reinterpret_cast<const f32x4*>(mass + j0 + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = fmaf(x[4 * g + e], c, m[e]);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= c;
        }
      }
      if constexpr (kBias >= 2) {
        if (a.slopes) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            x[r] = fmaf(-slope, fabsf(d0f + static_cast<float>(8 * (r / 4) + r % 4)), x[r]);
        }
        if (a.table) {
          if (behind || ahead) {
            const float far = distance[ahead ? 2 * distance_zero(reach) : 0];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += far;
          } else {
            const float* near = distance + (k0 + j0 - pos + distance_zero(reach));
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += near[8 * (r / 4) + r % 4];
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = __builtin_amdgcn_exp2f(kBias ? x[r] - lse : fmaf(x[r], c, -lse));
        dz[r] += delta;
      }
      if (partial) {
        const int last_r = last - k0 - j0;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 8 * (r / 4) + r % 4 <= last_r ? x[r] * unrest : 0.0f;
        if (kdocs) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const i32x4 tag = *reinterpret_cast<const i32x4*>(tags + j0 + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = tag[e] == doc ? x[4 * g + e] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dz[r] *= x[r];
      if constexpr (kBias >= 2) {
        if (f.part_slopes) {
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum = fmaf(-fabsf(d0f + static_cast<float>(8 * (r / 4) + r % 4)), dz[r], sum);
          slope_sum.add(sum);
        }
        if constexpr (kBias == 3) {
          if (behind || ahead) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum += dz[r];
            (ahead ? far_ahead : far_behind).add(sum);
          } else {
            // dZ sheared: row key - row + 31, column row, so that a diagonal is a row, one lane's; what no
            // pair has was cleared at the start and stays.
#pragma unroll
            for (int r = 0; r < 16; ++r)
              diagonal[(8 * (r / 4) + 4 * h + r % 4 - l32 + 31) * kShear + l32] = dz[r];
            wave_lds_order();
            const int d = lane - 31;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const f32x4 y = *reinterpret_cast<const f32x4*>(diagonal + min(lane, 62) * kShear + 4 * i);
              sum += (y[0] + y[1]) + (y[2] + y[3]);
            }
            const int r = k0 + 32 * sub - rw.lo + d;
            if (lane < 63) {
              if (r <= -reach)
                far_behind.add(sum);
              else if (r >= reach)
                far_ahead.add(sum);
              else
                sums[r + reach] += sum;
            }
            wave_lds_order();  // (the next block's diagonals, and their words of `sums`, are other lanes')
          }
        }
      }
      if constexpr (kCap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dz[r] *= bend[r];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const op8 zb = as_op<T>(dz, half);
#pragma unroll
        for (int dt = 0; dt < TL::kCols; ++dt) dq[dt] = Op<T>::mma(TL::cols_op(kt, dt, 2 * sub + half), zb, dq[dt]);
      }
    }
  };

  bool more = next();
  int buf = 0;
  if (more) load(0);
  while (more) {
    const int k0 = tile * kTile;
    const bool run = in_mine, all = in_full;
    more = next();
    wait_vmem<0>();
    if (kBias && a.mass && wave == 0) reinterpret_cast<float*>(lds + LO::kMass)[buf * kTile + lane] = next_mass;
    __syncthreads();
    if (LO::kBuffers == 2 && more) load(buf ^ 1);
    if (run) compute(!all || rests, k0, buf);
    if (LO::kBuffers == 1 && more) {
      __syncthreads();
      load(buf ^ 1);
    }
    buf ^= 1;
  }

  if (f.part_q && stored) {
    const int64_t bh = static_cast<int64_t>(b) * a.heads + head;
    float* dst = f.part_q + ((static_cast<int64_t>(split) * a.batch * a.heads + bh) * a.n_query + row) * D;
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = dq[dt][4 * g + e] * a.scale;
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g + 4 * h) = y;
      }
  } else if (f.dq && stored) {
    T* dst = f.dq + b * f.dqs[0] + head * f.dqs[1] + row * f.dqs[2];
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = dq[dt][4 * g + e] * a.scale;
        store4(dst + 32 * dt + 8 * g + 4 * h, y);
      }
  }
  const int64_t part = (static_cast<int64_t>(split) * a.batch + b) * f.row_blocks + block;
  if (kBias < 2 || (kBias == 2 && !f.part_slopes)) return;
  float slopes = slope_sum.sum, behind = far_behind.sum, ahead = far_ahead.sum;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    slopes += __shfl_xor(slopes, off), behind += __shfl_xor(behind, off), ahead += __shfl_xor(ahead, off);
  }
  float* totals = reinterpret_cast<float*>(lds + LO::kSums);
  if (lane == 0) totals[wave] = slopes;
  if (kBias == 3 && lane == 0) sums[0] = behind, sums[2 * a.buckets.reach] = ahead;
  __syncthreads();
  if (f.part_slopes && threadIdx.x == 0)
    f.part_slopes[part * a.heads + head] = ((totals[0] + totals[1]) + totals[2]) + totals[3];
  if (kBias < 3) return;
  float* by = distance + distance_words(a.buckets.reach) + kRowWaves * kDiagonal;  // all waves', into the first one's
  for (int i = threadIdx.x; i < words; i += 64 * kRowWaves)
    by[i] = ((by[i] + by[words + i]) + by[2 * words + i]) + by[3 * words + i];
  __syncthreads();
  a.buckets.template gather<64 * kRowWaves>(
      by, [&](int t, float s) { f.part_table[(part * a.buckets.count + t) * a.heads + head] = s; });
}

// dQ of split work, likewise.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_rows_kernel(const Grad<T> f) {
  const Args<T>& a = f.a;
  constexpr int kLanes = D / 4;
  const int64_t n = static_cast<int64_t>(a.batch) * a.heads * a.n_query;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  if (row >= n) return;
  const int d = static_cast<int>(threadIdx.x) % kLanes * 4;
  f32x4 y{};
#pragma unroll 4
  for (int s = 0; s < f.row_splits; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(f.part_q + (s * n + row) * D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += x[e];
  }
  const int i = static_cast<int>(row % a.n_query), bh = static_cast<int>(row / a.n_query);
  store4(f.dq + bh / a.heads * f.dqs[0] + bh % a.heads * f.dqs[1] + i * f.dqs[2] + d, y);
}

template <typename T, int D>
int run(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, const GradPlan& plan, char* ws, hipStream_t stream) {
  Grad<T> f{};
  f.a = make_args<T>(p);
  const GradPieces at = grad_pieces(p, g, plan);
  for (int i = 0; i < 3; ++i) {
    f.a.os[i] = g->out_stride[i], f.gos[i] = g->grad_out_stride[i];
    f.dqs[i] = g->dq_stride[i], f.dks[i] = g->dk_stride[i], f.dvs[i] = g->dv_stride[i];
  }
  f.o = static_cast<const T*>(g->out), f.go = static_cast<const T*>(g->grad_out), f.lse = g->lse;
  f.lse_rest = g->lse + p->batch * p->heads * p->n_query;
  f.rest = static_cast<const T*>(g->out_rest);
  f.dq = static_cast<T*>(g->dq), f.dk = static_cast<T*>(g->dk), f.dv = static_cast<T*>(g->dv);
  f.query_tiles = plan.query_tiles, f.key_tiles = plan.key_tiles, f.splits = plan.splits, f.row_splits = plan.row_splits;
  f.key_blocks = plan.key_blocks, f.row_blocks = plan.row_blocks;
  f.key_tasks = static_cast<int>(plan.key_tasks), f.row_tasks = static_cast<int>(plan.row_tasks);
  const auto piece = [&](size_t offset) { return reinterpret_cast<float*>(ws + offset); };
  f.delta = piece(at.delta), f.marks = reinterpret_cast<unsigned char*>(ws + at.marks);
  if (plan.splits > 1 && f.dk) f.part_kv = piece(at.kv);
  if (plan.row_splits > 1 && f.dq) f.part_q = piece(at.q);
  if (g->d_log_mass) f.part_mass = piece(at.mass);
  if (g->d_slopes) f.part_slopes = piece(at.slopes);
  if (g->d_table) f.part_table = piece(at.table);
  launch_info(p, f.a, ws, stream);
  int status = check_launch("masked_attn_grad documents");
  if (status != VGO_OK) return status;
  const unsigned tiles = static_cast<unsigned>(p->batch * p->heads * plan.query_tiles);
  if (tiles > 0) {
    hipLaunchKernelGGL((delta_kernel<T, D>), dim3(tiles), dim3(256), 0, stream, f);
    status = check_launch("masked_attn_grad delta");
    if (status != VGO_OK) return status;
  }
  const bool cap = f.a.cap2 != 0.0f;
  const int bias = f.a.slopes || f.a.table ? 2 : f.a.mass ? 1 : 0;  // (kBias: masses alone, or distances too)
  const size_t distances = f.a.table ? static_cast<size_t>(distance_words(f.a.buckets.reach)) * 4 : 0;
  if ((f.dk || f.part_mass) && plan.key_tasks > 0) {
    const size_t bytes = KeyLds<T, D>::kDistances + distances;
    const auto kernel = cap ? (bias == 0 ? key_kernel<T, D, true, 0> : bias == 1 ? key_kernel<T, D, true, 1> : key_kernel<T, D, true, 2>)
                            : (bias == 0 ? key_kernel<T, D, false, 0> : bias == 1 ? key_kernel<T, D, false, 1> : key_kernel<T, D, false, 2>);
    status = allow_lds(kernel, bytes, "masked_attn_grad");
    if (status != VGO_OK) return status;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.key_tasks)), dim3(64 * KeyLds<T, D>::kWaves), bytes,
                       stream, f);
    status = check_launch("masked_attn_grad keys");
    if (status != VGO_OK) return status;
    if (f.part_kv) {
      const int64_t rows = p->batch * p->kv_heads * p->n_key;
      hipLaunchKernelGGL((join_keys_kernel<T, D>), dim3(static_cast<unsigned>((rows * (2 * D / 4) + 255) / 256)),
                         dim3(256), 0, stream, f);
      status = check_launch("masked_attn_grad join");
      if (status != VGO_OK) return status;
    }
  }
  if ((f.dq || f.part_slopes || f.part_table) && plan.row_tasks > 0) {
    const size_t bytes = RowLds<T, D>::kDistances + distances +
                         (f.part_table ? static_cast<size_t>(kRowWaves) * (kDiagonal + sum_words(f.a.buckets.reach)) * 4 : 0);
    const auto of_bias = [&](auto capped) {
      constexpr bool kCap = decltype(capped)::value;
      return f.part_table ? row_kernel<T, D, kCap, 3>
             : bias == 2  ? row_kernel<T, D, kCap, 2>
             : bias == 1  ? row_kernel<T, D, kCap, 1>
                          : row_kernel<T, D, kCap, 0>;
    };
    const auto kernel = cap ? of_bias(std::true_type{}) : of_bias(std::false_type{});
    status = allow_lds(kernel, bytes, "masked_attn_grad");
    if (status != VGO_OK) return status;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.row_tasks)), dim3(64 * kRowWaves), bytes,
                       stream, f);
    status = check_launch("masked_attn_grad rows");
    if (status != VGO_OK) return status;
    if (f.part_q) {
      const int64_t rows = p->batch * p->heads * p->n_query;
      hipLaunchKernelGGL((join_rows_kernel<T, D>), dim3(static_cast<unsigned>((rows * (D / 4) + 255) / 256)), dim3(256),
                         0, stream, f);
      status = check_launch("masked_attn_grad join");
      if (status != VGO_OK) return status;
    }
  }
  if (g->d_log_mass) {
    status = sum_parts(f.part_mass, plan.key_tasks > 0 ? plan.splits * p->batch * p->kv_heads : 0, p->n_key,
                       g->d_log_mass, p->log_mass_dtype, stream);
    if (status != VGO_OK) return status;
  }
  const int64_t parts = plan.row_splits * p->batch * plan.row_blocks;
  if (g->d_slopes) {
    status = sum_parts(f.part_slopes, parts, p->heads, g->d_slopes, p->slopes_dtype, stream);
    if (status != VGO_OK) return status;
  }
  if (g->d_table)
    return sum_parts(f.part_table, parts, static_cast<int64_t>(p->n_buckets) * p->heads, g->d_table, p->table_dtype, stream);
  return VGO_OK;
}

}  // namespace

template <typename T>
int run_grad(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, const GradPlan& plan, char* ws,
             hipStream_t stream) {
  return p->head_dim == 128 ? run<T, 128>(p, g, plan, ws, stream) : run<T, 64>(p, g, plan, ws, stream);
}

}  // namespace masked
}  // namespace vgo
