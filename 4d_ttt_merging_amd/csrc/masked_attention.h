// What the masked-attention kernels share (forward: masked_attention.hip, gradients:
// masked_attention_grad.hip): the problem as the kernels see it, which pairs attend, the scores'
// rules, LDS tiles and their MFMA operands.
//
//   position of query i: p_i = query_start[b] + i;  distance r = j - p_i
//   z_ij = cap tanh(scale q_i.k_j / cap) + mass_j - slope_h |r| + table[bucket(r), h]
//   pair (i, j) attends if j < key_length[b], the documents are equal and >= 0, and, when causal,
//   r <= 0 or j < prefix[b].  P = softmax over those; a row without any gives zeros.
//
// Scores are computed transposed where a wave holds queries (S^T = K Q^T: a lane owns one query,
// its registers run over keys) and straight where it holds keys (S = Q K^T), so the accumulator of
// v_mfma_f32_32x32x16 -- register r of lane l: row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32 --
// is the next product's B operand as it stands: its k slots take rows in the order that the
// registers have them, and the A operand is read from LDS in that order (cols_op).
#pragma once

#include <algorithm>
#include <climits>
#include <string>
#include <type_traits>

#include "vgo_common.h"

namespace vgo {
namespace masked {

constexpr int kTile = 64;  // keys (or queries) per LDS tile
constexpr int kMaxStarts = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

typedef __attribute__((__vector_size__(8 * sizeof(float)))) float f32x8;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
typedef __attribute__((__vector_size__(8 * sizeof(short)))) short s16x8;

// Operands of one 16-deep product step: eight k slots per lane.  fp32 has no 16-deep instruction:
// eight 32x32x2 steps, step e with slot e of both halves, so both types share every layout.
template <typename T>
struct Op;
template <>
struct Op<bf16_t> {
  typedef bf16x8 op8;
  static __device__ __forceinline__ f32x16 mma(op8 a, op8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Op<f16_t> {
  typedef f16x8 op8;
  static __device__ __forceinline__ f32x16 mma(op8 a, op8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Op<float> {
  typedef f32x8 op8;
  static __device__ __forceinline__ f32x16 mma(op8 a, op8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// Accumulator registers 8 c .. 8 c + 7, times 2^raise, as an operand of T (bf16 / f16: rounded, as both products of
// a 16-bit attention take their probabilities).
template <typename T, int raise = 0>
__device__ __forceinline__ typename Op<T>::op8 as_op(const float (&s)[16], int c) {
  typename Op<T>::op8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = from_f32<T>(raise ? s[8 * c + e] * static_cast<float>(1 << raise) : s[8 * c + e]);
  return r;
}

// Powers of 2 by which f16 probabilities are held larger than they are, within f16's largest number, so that those
// of improbable keys keep their bits: its normal numbers end at 2^-14, all of them at 2^-25.  In the forward by a lower
// reference, which probabilities pass by 2^8; in the gradients, where 1 is the most, by a factor.
template <typename T>
constexpr int kLowerReference = std::is_same<T, f16_t>::value ? 7 : 0;
template <typename T>
constexpr int kRaise = std::is_same<T, f16_t>::value ? 14 : 0;

// ------------------------------------------------------------- LDS tiles ----
// kTile rows of D elements without padding; the 16-byte chunks of a row are permuted by XOR with a
// function of row % 16 that keeps apart, in the banks, both the 16 rows that a row-operand read
// takes at one chunk and the 4 (fp32: 2) rows x 64 (128) bytes that a column-operand read takes.
template <typename T, int D>
struct Tile {
  static constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
  static constexpr int kChunks = kRowBytes / 16;  // per row: 8, 16 or 32
  static constexpr int kBytes = kTile * kRowBytes;
  static constexpr int kSteps = D / 16;  // 16-deep steps over the channels
  static constexpr int kCols = D / 32;   // 32-channel blocks
  typedef typename Op<T>::op8 op8;

  static __device__ __forceinline__ int swz(int row) {
    if constexpr (sizeof(T) == 4) return (row & 3) | ((row >> 1) & 4) | ((row << 1) & 8);
    if constexpr (kChunks == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
    return ((row & 3) << 2) | ((row >> 2) & 3);
  }

  // Where the lane's 16 bytes of rows_op() of a 16-bit type lie in the tile.
  static __device__ __forceinline__ int rows_at(int row0, int t) {
    const int lane = lane_id();
    return (row0 + (lane & 31)) * kRowBytes + (((2 * t + (lane >> 5)) ^ swz(lane & 15)) << 4);
  }
  // A operand with rows row0 + l % 32 (row0 a multiple of 16), channels 16 t + 8 (l / 32) ..
  static __device__ __forceinline__ op8 rows_op(const char* tile, int row0, int t) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const op8*>(tile + rows_at(row0, t));
    } else {
      const int lane = lane_id(), row = row0 + (lane & 31), h = lane >> 5;
      const char* base = tile + row * kRowBytes;
      const int f = swz(lane & 15);
      const f32x4 a = *reinterpret_cast<const f32x4*>(base + (((4 * t + 2 * h) ^ f) << 4));
      const f32x4 b = *reinterpret_cast<const f32x4*>(base + (((4 * t + 2 * h + 1) ^ f) << 4));
      return op8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  // A operand of the transposed tile: row l % 32 of channels 32 dt .., k slot e = tile row
  // 16 c + 4 (l / 32) + e % 4 + 8 (e / 4).  16-bit types: two transposing reads, in each of which
  // 16 lanes take a 4 x 16 block (lane i: 4 channels of row i / 4) and keep column i of it.
  static __device__ __forceinline__ op8 cols_op(const char* tile, int dt, int c) {
    const int lane = lane_id(), h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, gg = (lane >> 4) & 1;
      s16x8 r;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = 4 * h + (i >> 2) + 8 * half;  // of 16
        const int chunk = (4 * dt + 2 * gg + ((i >> 1) & 1)) ^ swz(row);
        const char* p = tile + (16 * c + row) * kRowBytes + (chunk << 4) + ((i & 1) << 3);
        typedef __attribute__((address_space(3))) s16x4* lds_p;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p));
#pragma unroll
        for (int e = 0; e < 4; ++e) r[4 * half + e] = x[e];
      }
      return __builtin_bit_cast(op8, r);
    } else {
      op8 r;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 4 * h + (e & 3) + 8 * (e >> 2);
        const int d = 32 * dt + (lane & 31);
        r[e] = *reinterpret_cast<const float*>(tile + (16 * c + row) * kRowBytes + (((d >> 2) ^ swz(row)) << 4) +
                                               ((d & 3) << 2));
      }
      return r;
    }
  }
};

// 16 bytes that stand for every row a tile must not take: those past the end, and those that the
// masks keep from every row whatever they hold.
static __device__ __attribute__((aligned(16))) const char zero_chunk[16] = {};

// Rows row0 .. row0 + kTile of a [*, D] operand into an LDS tile by LDS DMA, wave w of `kWaves`
// taking its share of 1 KB pieces.  `whole`: every row is taken; else row r is taken if
// row0 + r < limit and live(row0 + r).
template <typename T, int D, int kWaves, typename Live>
__device__ __forceinline__ void stage(const T* base, int64_t row_stride, int row0, int limit, bool whole,
                                      uint32_t lds, Live live) {
  typedef Tile<T, D> TL;
  constexpr int kPieces = TL::kBytes / 1024 / kWaves;
  const int lane = lane_id();
  const int wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const char* first = reinterpret_cast<const char*>(base + row0 * row_stride);
  const uint32_t row_bytes = static_cast<uint32_t>(row_stride * static_cast<int64_t>(sizeof(T)));
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int piece = wave * kPieces + i, c = piece * 64 + lane;
    const int row = c / TL::kChunks;
    const uint32_t offset = row * row_bytes + (((c % TL::kChunks) ^ TL::swz(row & 15)) << 4);
    const uint32_t to = lds + piece * 1024;
    if (whole) {
      lds_dma16(first, offset, to);
    } else {
      const bool taken = row0 + row < limit && live(row0 + row);
      lds_dma16_addr(taken ? first + offset : zero_chunk, to);
    }
  }
}

// Where lanes of a wave read, or add to, LDS words that other lanes of it wrote.  The hardware keeps a wave's LDS
// operations in order; this keeps the compiler, which sees one lane's addresses, from moving them past each other.  No
// instruction.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// Buckets of distances: that of r is the number of starts <= |r|, plus half of them for r > 0
// (bidirectional), or the number <= max(-r, 0).  Distances from `reach` on share one a side.
struct Buckets {
  int count, bidirectional, n_starts, reach;
  int starts[kMaxStarts];

  __device__ __forceinline__ int of(int r) const {
    const int n = bidirectional ? abs(r) : max(-r, 0);
    int bucket = 0;
    for (int t = 0; t < n_starts; ++t) bucket += starts[t] <= n;
    return bucket + (bidirectional && r > 0 ? count / 2 : 0);
  }
  // Sums by distance (by[r + reach], r = -reach .. reach, in LDS) to the sums of the buckets: put(t, sum), by
  // the whole work-group, `kLanes` lanes a bucket.
  template <int kThreads, typename Put>
  __device__ __forceinline__ void gather(const float* by, Put put) const {
    constexpr int kLanes = 8;
    const int j = threadIdx.x % kLanes, side = bidirectional ? count / 2 : count;
    for (int t0 = 0; t0 < count; t0 += kThreads / kLanes) {
      const int t = t0 + threadIdx.x / kLanes, index = t % side;
      float s = 0.0f;
      if (t < count && index <= n_starts) {
        const int from = index == 0 ? 0 : starts[index - 1], to = index < n_starts ? starts[index] : reach + 1;
        const bool ahead = t >= side;
        for (int n = (ahead ? max(1, from) : from) + j; n < to; n += kLanes) s += by[reach + (ahead ? n : -n)];
        if (!bidirectional && index == 0)
          for (int n = 1 + j; n <= reach; n += kLanes) s += by[reach + n];
      }
#pragma unroll
      for (int off = kLanes / 2; off >= 1; off >>= 1) s += __shfl_xor(s, off);
      if (t < count && j == 0) put(t, s);
    }
  }
};

// A long sum in fp32 with what each addition lost.
struct LongSum {
  float sum = 0.0f, lost = 0.0f;
  __device__ __forceinline__ void add(float x) {
    const float y = x - lost, to = sum + y;
    lost = (to - sum) - y;
    sum = to;
  }
};

inline Buckets make_buckets(int count, const int32_t* starts, int n_starts, int bidirectional) {
  Buckets b{};
  b.count = count, b.bidirectional = bidirectional != 0, b.n_starts = n_starts;
  for (int t = 0; t < n_starts; ++t) b.starts[t] = starts[t];
  b.reach = n_starts > 0 ? starts[n_starts - 1] : 1;
  return b;
}
// VGO_OK, or the status of buckets that the kernels do not take.
int check_buckets(int64_t count, const int32_t* starts, int n_starts, int bidirectional);

// ---------------------------------------------------------- the problem ----
// Strides in elements.  Documents: query_doc [batch, n_query], key_doc [batch, n_key] or null; the
// tile_info of either: per kTile rows {smallest, largest} valid document, the smallest one's bits
// inverted where a row of the tile is none's (negative, or past the end).
template <typename T>
struct Args {
  const T *q, *k, *v;
  int64_t qs[3], ks[3], vs[3], os[3];
  int batch, heads, kv_heads, n_query, n_key;
  float scale, inv_cap, cap2;     // scale; scale / cap and cap log2(e) (0: no cap)
  float cap_reach, cap_series[5]; // kCapReach and kCapSeries for products before the scale (reach 0: not used)
  float cap_low, cap_low_series[3];  // likewise kCapLow and kCapLowSeries
  int cap_large;                  // past kCapShort: kTanhReach, kTanhLow and kTanhSeries in their places
  const void* mass;               // [n_key] or null
  const void* slopes;             // [heads] or null
  const void* table;              // [n_buckets, heads] or null
  int mass_type, slopes_type, table_type;
  Buckets buckets;                // of the table
  int causal, query_start;
  const int *prefix, *key_lengths, *query_starts;  // [batch] or null
  const int *query_doc, *key_doc;
  const int2 *query_info, *key_info;  // [batch, tiles]
};

// Element i of a parameter of any type, in units of log2.  A type's lowest value, which masks use to keep keys out,
// is a finite number, and a row of nothing else a softmax over them: what is finite stays so, here and where a mass and
// a table add up.
constexpr float kMostParameter = 0x1p126f;
__device__ __forceinline__ float parameter2(const void* p, int type, int64_t i) {
  const float x = type == VGO_F32    ? static_cast<const float*>(p)[i]
                  : type == VGO_BF16 ? to_f32(static_cast<const bf16_t*>(p)[i])
                                     : to_f32(static_cast<const f16_t*>(p)[i]);
  const float y = x * kLog2e;
  return fabsf(x) < kInf ? fmaxf(-kMostParameter, fminf(y, kMostParameter)) : y;
}
template <typename T>
__device__ __forceinline__ float mass2(const Args<T>& a, int key) { return parameter2(a.mass, a.mass_type, key); }
template <typename T>
__device__ __forceinline__ float slope2(const Args<T>& a, int head) {
  return a.slopes ? parameter2(a.slopes, a.slopes_type, head) : 0.0f;
}

// A causal mask makes one end of a head's blocks the longest: every second list of blocks runs the other
// way, so that work-groups that share a CU are long and short ones, and the last list ends with the short.
__device__ __forceinline__ int zigzag(int index, int blocks, int list, int lists) {
  return (lists - 1 - list) & 1 ? blocks - 1 - index : index;
}

template <typename T>
__device__ __forceinline__ int key_limit(const Args<T>& a, int b) {
  return a.key_lengths ? max(0, min(a.n_key, a.key_lengths[b])) : a.n_key;
}
template <typename T>
__device__ __forceinline__ int first_position(const Args<T>& a, int b) {
  constexpr int kMost = 1 << 29;  // keeps every distance in 32 bits
  return a.query_starts ? max(-kMost, min(kMost, a.query_starts[b])) : a.query_start;
}
// What the slopes take off the positions of a tile of queries (whose first is `first`): nothing, or, where the tile lies
// beyond all keys, what brings its nearer end to theirs.  A softmax leaves out what that takes off every distance of a
// row, and so does the slopes' gradient (a row's dZ add up to nothing); left on, the difference of two keys' scores was
// lost in fp32 (a position of 1e6 and a slope of 0.5: 0.03).  By tiles, so that a tile's positions stay in a row.
__device__ __forceinline__ int slope_shift(int first, int limit) {
  return max(0, first - (limit - 1)) + min(0, first + kTile - 1);
}
template <typename T>
__device__ __forceinline__ int prefix_of(const Args<T>& a, int b) {
  return a.prefix ? a.prefix[b] : 0;
}

// Rows of one side as the other side's tiles are judged by: positions (queries) or indices (keys)
// lo .. hi, the documents' smallest and largest, and whether every row is a document's.
struct Range {
  int lo, hi, doc_lo, doc_hi;
  bool docs_whole;
};

__device__ __forceinline__ Range info_range(int2 info) {
  Range r;
  r.docs_whole = info.x >= 0;
  r.doc_lo = r.docs_whole ? info.x : ~info.x;
  r.doc_hi = info.y;
  return r;
}

// Whether any pair of the two ranges attends, and whether all do.  Keys past the limit are the
// caller's to leave out of `any` and to count against `all`.
template <typename T>
__device__ __forceinline__ void judge(const Args<T>& a, const Range& q, const Range& k, int prefix, bool& any,
                                      bool& all) {
  any = all = true;
  if (a.causal) {
    any = k.lo <= q.hi || k.lo < prefix;
    all = k.hi <= q.lo || k.hi < prefix;
  }
  if (a.key_doc) {
    any = any && q.doc_lo <= k.doc_hi && k.doc_lo <= q.doc_hi;
    all = all && q.docs_whole && k.docs_whole && q.doc_lo == q.doc_hi && k.doc_lo == k.doc_hi &&
          q.doc_lo == k.doc_lo;
  }
}

// table[bucket(r), head] log2(e) by distance in LDS, r = 0 at distance_zero(): as far as a 64 x 32 block that
// touches the buckets' reach does, so that lookups need no bounds of their own.
constexpr int kMargin = 96;
__host__ __device__ inline int distance_zero(int reach) { return reach + kMargin; }
__host__ __device__ inline int distance_words(int reach) { return (2 * distance_zero(reach) + 4) & ~3; }
template <typename T>
__device__ __forceinline__ void fill_distances(const Args<T>& a, float* to, int head, int threads) {
  const int zero = distance_zero(a.buckets.reach);
  for (int i = threadIdx.x; i <= 2 * zero; i += threads)
    to[i] = parameter2(a.table, a.table_type, static_cast<int64_t>(a.buckets.of(i - zero)) * a.heads + head);
}

// out[i] = sum over parts of part[p][i], in a fixed order: 64 outputs a work-group, four runs of parts each.
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int64_t parts, int64_t n, T* out) {
  __shared__ float s[4][64];
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
  const int run = threadIdx.x >> 6;
  float x = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int64_t p = run; p < parts; p += 4) x += part[p * n + i];
  }
  s[run][threadIdx.x & 63] = x;
  __syncthreads();
  if (run == 0 && i < n)
    out[i] = from_f32<T>(((s[0][threadIdx.x] + s[1][threadIdx.x]) + s[2][threadIdx.x]) + s[3][threadIdx.x]);
}
inline int sum_parts(const float* part, int64_t parts, int64_t n, void* out, int type, hipStream_t stream) {
  if (n == 0) return VGO_OK;
  const dim3 groups(static_cast<unsigned>((n + 63) / 64));
  if (type == VGO_F32)
    hipLaunchKernelGGL(sum_parts_kernel<float>, groups, dim3(256), 0, stream, part, parts, n, static_cast<float*>(out));
  else if (type == VGO_BF16)
    hipLaunchKernelGGL(sum_parts_kernel<bf16_t>, groups, dim3(256), 0, stream, part, parts, n, static_cast<bf16_t*>(out));
  else
    hipLaunchKernelGGL(sum_parts_kernel<f16_t>, groups, dim3(256), 0, stream, part, parts, n, static_cast<f16_t*>(out));
  return check_launch("sum of parts");
}

// tanh of the capped scores.  For 16-bit inputs, where |y| stays below kCapReach, an odd polynomial (weighted least
// squares at Chebyshev points towards the least largest error: 2e-7), six full-rate instructions in
// place of two quarter-rate ones and three more; past it, and for fp32, 1 - 2 / (1 + e^2y), whose
// 1 costs a small y about 1e-7, so that fp32 takes the odd series below 0.3 (its next term is 1e-9).
// Both errors are multiplied by the cap: past a cap of kCapShort, where 2e-7 of it is 2e-5 of a score, 16-bit inputs
// take the odd series too, as far as its error is fp32's rounding: 0.3, and 0.1 of its first three terms.
constexpr float kCapShort = 100.0f;
constexpr double kTanhSeries[5] = {1.0, -1.0 / 3.0, 2.0 / 15.0, -17.0 / 315.0, 62.0 / 2835.0};
constexpr float kTanhReach = 0.3f, kTanhLow = 0.1f;
constexpr float kCapReach = 0.75f;
// tanh(y) / y in powers of y^2.
constexpr float kCapSeries[5] = {0.999997228f, -0.333230765f, 0.132260916f, -0.0492804483f, 0.0123188331f};
// Below kCapLow, where a cap well past the scores leaves nearly all, two terms less do for half of that error: the
// capped forward is bound by its vector instructions (16 x 16,464 x 64 causal: 902 us with the longer series, 842 now;
// 990 with the exponential's form, where scores come near the cap or pass it).
constexpr float kCapLow = 0.28f;
constexpr float kCapLowSeries[3] = {0.9999973373f, -0.3330590180f, 0.1262284013f};
template <typename T>
__device__ __forceinline__ float cap_low(const Args<T>& a, float s) {
  const float u = s * s;
  return s * fmaf(fmaf(u, a.cap_low_series[2], a.cap_low_series[1]), u, a.cap_low_series[0]);
}
template <typename T>
__device__ __forceinline__ float cap_short(const Args<T>& a, float s) {  // of the raw product s
  const float u = s * s;
  float x = fmaf(u, a.cap_series[4], a.cap_series[3]);
  x = fmaf(x, u, a.cap_series[2]);
  x = fmaf(x, u, a.cap_series[1]);
  return s * fmaf(x, u, a.cap_series[0]);
}
template <typename T>
__device__ __forceinline__ float cap_tanh(float y) {
  const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
  float t = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
  if constexpr (sizeof(T) == 4) {
    const float y2 = y * y;
    float s = fmaf(y2, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    s = fmaf(s, -y2, 17.0f / 315.0f);
    s = fmaf(s, -y2, 2.0f / 15.0f);
    s = fmaf(s, -y2, 1.0f / 3.0f);
    t = fabsf(y) < 0.3f ? fmaf(-y * y2, s, y) : t;
  }
  return t;
}
// tanh of 16 raw products, some past the series' reach; of a large cap, the others by the series all the same.
template <typename T>
__device__ __forceinline__ void cap_all(const Args<T>& a, float (&x)[16]) {
  if (sizeof(T) == 2 && a.cap_large) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float near = cap_short(a, x[r]), far = cap_tanh<T>(x[r] * a.inv_cap);
      x[r] = fabsf(x[r]) <= a.cap_reach ? near : far;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = cap_tanh<T>(x[r] * a.inv_cap);
  }
}

// Row sums of probabilities as the products take them: of bf16 the rounded values, two per instruction,
// so that their rounding cancels where one key has most of a row (f16 and fp32: what is not
// worth a second look, the sum of the unrounded ones; the two-value form would drop f16's subnormals).
template <typename T>
__device__ __forceinline__ float add_pair(float sum, float a, float b, T, T) {
  return sum + a + b;
}
template <>
__device__ __forceinline__ float add_pair<bf16_t>(float sum, float, float, bf16_t a, bf16_t b) {
  const bf16x2 pair = {a, b}, one = {static_cast<bf16_t>(1.0f), static_cast<bf16_t>(1.0f)};
  return __builtin_amdgcn_fdot2_f32_bf16(pair, one, sum, false);
}

constexpr size_t kLdsBytes = 163840;  // a CU's
// Lets a kernel have `bytes` of dynamic LDS.
template <typename K>
int allow_lds(K kernel, size_t bytes, const char* what) {
  if (bytes <= 65536) return VGO_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == hipSuccess) return VGO_OK;
  (void)hipGetLastError();  // (or the next launch would report it)
  return fail(VGO_ELAUNCH, std::string(what) + ": " + hipGetErrorString(e));
}

inline int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

// Document ranges of the tiles of both sides (tile_info above): key_info [batch, key tiles], query_info behind it.
void launch_doc_info(const vgo_masked_attn* p, int2* info, hipStream_t stream);

// Whether documents keep pairs apart: there are any to keep apart (arrays of no element may be null).
inline bool has_documents(const vgo_masked_attn* p) {
  return p->n_query > 0 && p->n_key > 0 && p->query_documents && p->key_documents;
}

// How many ways to split the `tiles` tiles of each of `tasks` work-groups (the rule stands at its definition).
int splits_of(const vgo_masked_attn* p, int64_t tasks, int tiles, int resident, double tile_us, double join_us);
// Whether a launch of so many work-groups is one: threads of a grid are counted in 32 bits.
inline bool fits_grid(int64_t groups, int threads) { return groups < (int64_t{1} << 32) / threads; }

// VGO_OK, or the status of a problem the kernels do not take, with its message.
int check_problem(const vgo_masked_attn* p, int dtype);
bool strides_fit(const int64_t stride[3], int64_t head_dim, int dtype);

template <typename T>
Args<T> make_args(const vgo_masked_attn* p) {
  Args<T> a{};
  a.q = static_cast<const T*>(p->q), a.k = static_cast<const T*>(p->k), a.v = static_cast<const T*>(p->v);
  for (int i = 0; i < 3; ++i) a.qs[i] = p->q_stride[i], a.ks[i] = p->k_stride[i], a.vs[i] = p->v_stride[i];
  a.batch = static_cast<int>(p->batch), a.heads = static_cast<int>(p->heads);
  a.kv_heads = static_cast<int>(p->kv_heads);
  a.n_query = static_cast<int>(p->n_query), a.n_key = static_cast<int>(p->n_key);
  a.scale = p->scale;
  if (p->score_cap > 0.0f) {
    // Caps beyond these leave scores up to 1e11 as they are, or next to nothing of any; within them the factors and the
    // series' squares are finite.
    const float cap = std::max(1e-20f, std::min(p->score_cap, 1e15f));
    a.inv_cap = p->scale / cap, a.cap2 = cap * kLog2e;
    a.cap_large = cap > kCapShort;
    if (sizeof(T) == 2 && a.inv_cap < 1e3f) {  // (below, ninth powers grow out of range)
      a.cap_reach = (a.cap_large ? kTanhReach : kCapReach) / a.inv_cap;
      a.cap_low = (a.cap_large ? kTanhLow : kCapLow) / a.inv_cap;
      double power = a.inv_cap;
      for (int i = 0; i < 5; ++i, power *= static_cast<double>(a.inv_cap) * a.inv_cap) {
        a.cap_series[i] = static_cast<float>((a.cap_large ? kTanhSeries[i] : kCapSeries[i]) * power);
        if (i < 3) a.cap_low_series[i] = static_cast<float>((a.cap_large ? kTanhSeries[i] : kCapLowSeries[i]) * power);
      }
    }
  }
  a.mass = p->log_mass, a.slopes = p->slopes, a.table = p->bucket_table;
  a.mass_type = p->log_mass_dtype, a.slopes_type = p->slopes_dtype, a.table_type = p->table_dtype;
  if (a.table) a.buckets = make_buckets(p->n_buckets, p->bucket_starts, p->n_starts, p->bidirectional);
  a.causal = p->causal != 0, a.query_start = a.n_key - a.n_query;
  a.prefix = p->prefix_lengths, a.key_lengths = p->key_lengths, a.query_starts = p->query_starts;
  if (has_documents(p)) a.query_doc = p->query_documents, a.key_doc = p->key_documents;
  return a;
}

// Document ranges of both sides' tiles: their bytes, and their launch into `ws`.
size_t info_bytes(const vgo_masked_attn* p);
template <typename T>
void launch_info(const vgo_masked_attn* p, Args<T>& a, char* ws, hipStream_t stream) {
  if (!a.key_doc) return;
  int2* key = reinterpret_cast<int2*>(ws);
  int2* query = key + static_cast<int64_t>(a.batch) * tiles_of(a.n_key);
  launch_doc_info(p, key, stream);
  a.key_info = key, a.query_info = query;
}

}  // namespace masked
}  // namespace vgo
