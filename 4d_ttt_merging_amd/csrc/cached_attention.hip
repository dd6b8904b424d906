// Attention over the paged cache of keys and values in 4 bits (paged_cache.h).
#include "cached_attention.h"

#include <algorithm>
#include <cmath>

namespace vgo {
namespace paged {
namespace {

// The sums of a row's parts, as one.
struct Joined {
  float top = -INFINITY, sum = 0.0f;
  f32x4 v = {};
};
// Parts part, part + stride, ... of n, from place `start` on by `step`: what is read does not depend on what has been read, so
// that four parts take one trip to memory.
template <int D>
__device__ __forceinline__ void join(const Attend& a, Joined& j, int part, int stride, int n, int64_t start, int64_t step, int c) {
  for (; part < n; part += 4 * stride) {
    float2 end[4];
    f32x4 values[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t place = start + min(part + i * stride, n - 1) * step;
      end[i] = a.ends[place];
      values[i] = *reinterpret_cast<const f32x4*>(a.sums + place * D + c);
      if (part + i * stride >= n) end[i] = {-INFINITY, 0.0f};
    }
    const float most = fmaxf(fmaxf(j.top, fmaxf(end[0].x, end[1].x)), fmaxf(end[2].x, end[3].x));
    const float from = most == -INFINITY ? 0.0f : most;
    const float shrink = __builtin_amdgcn_exp2f(j.top - from);
    j.top = most, j.sum *= shrink;
#pragma unroll
    for (int e = 0; e < 4; ++e) j.v[e] *= shrink;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float share = __builtin_amdgcn_exp2f(end[i].x - from);
      j.sum = fmaf(end[i].y, share, j.sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) j.v[e] = fmaf(values[i][e], share, j.v[e]);
    }
  }
}

// Joins the pieces of `kRows` rows of a tile, where there are several.  D / 4 lanes take four channels of a row each; a
// wave's others, if kApart (few rows), every second or fourth piece of the same row, else the next rows.
template <typename T, int D, int kRows, bool kApart>
__global__ __launch_bounds__(256) void join_kernel(const Attend a) {
  constexpr int kLanes = D / 4, kGroups = kApart ? 64 / kLanes : 1, kAtOnce = 256 / kLanes / kGroups;
  const int rows = a.last_row - a.first_row, kv = a.pages.kv_heads, chunks = (rows + kRows - 1) / kRows;
  const int of0 = static_cast<int>(blockIdx.x % chunks) * kRows, hk = static_cast<int>(blockIdx.x / chunks % kv);
  const int64_t b = blockIdx.x / chunks / kv;
  const int2 piece = a.firsts[b];
  const int count = count_of(a, b), tile = of0 / a.tile_rows;
  const int stop = stop_of(a, length_of(a, b), count, first_place(a, b, count), a.first_row + tile * a.tile_rows);
  const int n = stop <= 0 ? 1 : (stop - 1) / piece.y + 1;
  if (n <= 1) return;
  const int64_t step = static_cast<int64_t>(kv) * a.tiles * a.tile_rows;
  const int64_t start = piece.x * step + (static_cast<int64_t>(hk) * a.tiles + tile) * a.tile_rows - tile * a.tile_rows;
  const int c = threadIdx.x % kLanes * 4, group = kApart ? lane_id() / kLanes : 0;
  for (int r = kApart ? threadIdx.x / 64 : threadIdx.x / kLanes; r < kRows && of0 + r < rows; r += kAtOnce) {
    Joined j;
    join<D>(a, j, group, kGroups, n, start + of0 + r, step, c);
#pragma unroll
    for (int o = kLanes; o < kLanes * kGroups; o <<= 1) {
      const float other = __shfl_xor(j.top, o), most = fmaxf(j.top, other), from = most == -INFINITY ? 0.0f : most;
      const float mine = __builtin_amdgcn_exp2f(j.top - from), theirs = __builtin_amdgcn_exp2f(other - from);
      // (the same products and one sum on both sides: the same bits)
      j.sum = j.sum * mine + __shfl_xor(j.sum, o) * theirs;
#pragma unroll
      for (int e = 0; e < 4; ++e) j.v[e] = j.v[e] * mine + __shfl_xor(j.v[e], o) * theirs;
      j.top = most;
    }
    const int row = a.first_row + of0 + r;
    const bool none = row >= count * a.group || sees_nothing(j.top, j.sum);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : j.v[e] / j.sum;
    if (group == 0)
      store4(static_cast<T*>(a.out) + b * a.out_stride[0] + (hk * a.group + row % a.group) * a.out_stride[1] +
                 row / a.group * a.out_stride[2] + c, v);
  }
}

// Rows of a work-group: four, a wave each, where there are few; else 128, so that calls of which no row has several pieces
// are soon through with them (64 rows of 8 key heads over 16 pieces 42 us with the one, 52 with 32; 3 causal prompts, whole:
// 16,464 rows each 196 by 4, 154 by 32, some 9,000 rows each 73 by 32, 70 by 128; two cut chunks of 8,232 rows alike by 32 and
// 128).  Neither passes the end of a tile: of tiles of 16 a launch with pieces has fewer than 8,192 rows.
template <typename T, int D>
void join_pieces(const Attend& a, hipStream_t s) {
  const int64_t rows = a.last_row - a.first_row, all = a.batch * a.pages.kv_heads;
  const bool few = rows * all <= 16384;
  const int64_t each = few ? 4 : 128;
  const unsigned grid = static_cast<unsigned>(all * ((rows + each - 1) / each));
  if (few) join_kernel<T, D, 4, true><<<grid, 256, 0, s>>>(a);
  else join_kernel<T, D, 128, false><<<grid, 256, 0, s>>>(a);
}
template <typename T>
int join_pieces(const Attend& a, int head_dim, hipStream_t s) {
  if (head_dim == 64) join_pieces<T, 64>(a, s);
  else join_pieces<T, 128>(a, s);
  return check_launch("cached_attn");
}

}  // namespace

template <>
ManyShape many_shape<bf16_t>(int head_dim, bool causal, int64_t group);
template <>
ManyShape many_shape<f16_t>(int head_dim, bool causal, int64_t group);
template <>
ManyShape many_shape<float>(int head_dim, bool causal, int64_t group);
template <>
int launch_many<bf16_t>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s);
template <>
int launch_many<f16_t>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s);
template <>
int launch_many<float>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s);

namespace {

// Tokens of a piece at least, and (few queries) up to how many a sequence stays whole: the join is a launch of 3 us.
// One query of 16 heads over 4 key heads, us: 1,044 tokens whole 8.2, in pieces of 512 9.8; 2,048 11.1, 10.0; 32,768 in
// pieces of at least 256, 512, 1,024: 16.1, 12.1, 12.6.  Many: 8 heads of 261 queries in fp32 over 1,044 tokens in
// pieces of 64, 128, 256: 20.0, 16.3, 19.1.
constexpr int64_t kLeastFew = 512, kWholeFew = 1536, kLeastMany = 128;

// How a call's rows are run: up to two launches, the second for the few rows that would be a tile of the first.
struct Part {
  bool few;
  int64_t first_row, last_row;
  int tile_rows, slots;
  int64_t least;
  int held;
  int64_t tiles, pieces;
  size_t sums, ends, firsts;  // bytes of the workspace
  size_t bytes() const { return sums + ends + firsts; }
};
struct Plan {
  int parts;
  Part part[2];
  size_t bytes() const { return part[0].bytes() + (parts > 1 ? part[1].bytes() : 0); }
};
Part part_of(const vgo_paged_cache* c, int64_t first_row, int64_t last_row, bool few, bool ragged, const ManyShape& shape) {
  Part p{};
  const int64_t rows = last_row - first_row, capacity = c->table_width * c->page_size;
  p.few = few, p.first_row = first_row, p.last_row = last_row;
  p.tile_rows = few ? kFewTile : shape.tile_rows;
  p.least = few ? kLeastFew : kLeastMany;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  // Few queries: as many work-groups as the chip holds at once.  Many, of which some sequences may have fewer than others: more,
  // which those that have queries then share (a grid of four times as many is through with its idle ones in 8 us).  us with
  // once, twice and four times as many as it holds: ragged causal 2 x 2,058 queries over 16,464 tokens of 128 channels 269 272
  // 218, of 64 188 138 138; 5 x 1,029 over 8,232 200 188 188; of tiles below 8, 6 x 300 158 125 125 (but 3 x 300 of 8 heads 43
  // 54 56), 20 x 100 47 47 56, and 500 whole over 16,464 45 44 48.
  // None beside one a tile where all are busy and leave little of their last round idle, or rounds are many: the device would
  // mostly leave those whole, too (7, 6 and 13 sequences of 1,029 queries, by borders of 0.75, 0.85 and 0.95: within 0.2%; 8.25
  // rounds whole 2,437 us, cut 2,429, 4.1 rounds of 128 channels 1,203, 1,204), and they need neither workspace nor join.
  const int64_t held = static_cast<int64_t>(few ? 2 : shape.resident) * device_cus(), beside = c->kv_heads * p.tiles;
  const int64_t busy = c->batch * beside, last = (busy + held - 1) / held * held;
  const bool full = !few && (busy >= 8 * held || (!ragged && 20 * busy >= 17 * last));
  const int64_t rounds = few || (p.tiles == 1 && c->batch * beside <= held / 4) ? 1 : p.tiles < 8 ? 2 : 4;
  const int64_t slots = full ? 0 : rounds * held / beside - c->batch;
  p.held = static_cast<int>(held);
  // (no more pieces than the tables could hold)
  p.slots = capacity <= (few ? kWholeFew : kLeastMany) ? 0 : static_cast<int>(std::max<int64_t>(0, std::min(slots, c->batch * ((capacity - 1) / p.least))));
  p.pieces = c->batch + p.slots;
  if (p.slots > 0) {
    const size_t parts = static_cast<size_t>(p.pieces) * beside * p.tile_rows;
    p.sums = parts * c->head_dim * sizeof(float);
    p.ends = (parts * sizeof(float2) + 15) / 16 * 16;
    p.firsts = (c->batch * sizeof(int2) + 15) / 16 * 16;
  }
  return p;
}
Plan plan_of(const vgo_paged_cache* c, int64_t heads, int64_t n_query, bool causal, bool ragged, int dtype) {
  Plan p{};
  const int64_t rows = n_query * (heads / c->kv_heads);
  const int dim = static_cast<int>(c->head_dim);
  const ManyShape shape = dtype == VGO_BF16  ? many_shape<bf16_t>(dim, causal, heads / c->kv_heads)
                          : dtype == VGO_F16 ? many_shape<f16_t>(dim, causal, heads / c->kv_heads)
                                             : many_shape<float>(dim, causal, heads / c->kv_heads);
  const int64_t over = rows % shape.tile_rows;
  // Rows of the large tiles.  (A last tile of 5 rows beside 1, 2, 3, 4, 8 and 16 full ones of 256, 16 heads over 16,464 tokens, the
  // last over 8,192, us as a tile 57, 75, 91, 117, 188, 203; by the few's kernel 57, 73, 93, 111, 180, 180.  Of ragged
  // sequences few have such rows: 2 x 1,029 queries 100 as a tile, 108 so, 4 x 1,029 146, 151, which is the price.)
  const int64_t split = rows <= kFewRows ? 0 : over <= kFewRows && rows >= 4 * shape.tile_rows ? rows - over : rows;
  if (split > 0) p.part[p.parts++] = part_of(c, 0, split, false, ragged, shape);
  if (split < rows) p.part[p.parts++] = part_of(c, split, rows, true, ragged, shape);
  return p;
}

constexpr int64_t kMostThreads = int64_t{1} << 32;
int check_attend(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int dtype) {
  const int status = check_cache(cache);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "cached_attn: unsupported dtype");
  VGO_REQUIRE(n_query >= 0 && n_query <= INT32_MAX && heads >= 1 && heads <= 65535, "cached_attn: size out of range");
  VGO_REQUIRE(heads % cache->kv_heads == 0, "cached_attn: heads must be a multiple of the key heads");
  // (a grid's threads are counted in 32 bits; rows and their places among a launch's in 31)
  VGO_REQUIRE(cache->batch == 0 || n_query == 0 || cache->batch < kMostThreads / heads / n_query / 32, "cached_attn: too many rows");
  return VGO_OK;
}

}  // namespace
}  // namespace paged
}  // namespace vgo

extern "C" int vgo_cached_attn_workspace(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int causal,
                                         int ragged, int dtype, size_t* bytes) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_attend(cache, heads, n_query, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "cached_attn: null pointer");
  *bytes = 0;
  if (cache->batch == 0 || n_query == 0) return VGO_OK;
  const Plan p = plan_of(cache, heads, n_query, causal != 0, ragged != 0, dtype);
  *bytes = p.bytes();
  return VGO_OK;
}

extern "C" int vgo_cached_attn_fwd(const vgo_paged_cache* cache, const void* q, const int64_t q_stride[3], int64_t heads,
                                   int64_t n_query, const int32_t* lengths, const int32_t* counts, int causal, float scale,
                                   void* out, const int64_t out_stride[3], int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_attend(cache, heads, n_query, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(scale >= 1e-8f && scale <= 1e8f, "cached_attn: the scale must be from 1e-8 to 1e8");
  if (cache->batch == 0 || n_query == 0) return VGO_OK;
  VGO_REQUIRE(lengths, "cached_attn: null lengths");
  VGO_REQUIRE(rows_fit(q, q_stride, dtype) && rows_fit(out, out_stride, dtype),
              "cached_attn: q and out must be 16-byte aligned, with strides of whole 16 bytes");
  const Plan p = plan_of(cache, heads, n_query, causal != 0, counts != nullptr, dtype);
  for (int i = 0; i < p.parts; ++i)
    VGO_REQUIRE(p.part[i].pieces < kMostThreads / 512 / (p.part[i].tiles * cache->kv_heads), "cached_attn: too many rows");
  if (p.bytes() > 0 && (!workspace || workspace_bytes < p.bytes() || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "cached_attn: workspace of " + std::to_string(p.bytes()) + " bytes needed");
  Attend a{};
  a.pages = pages_of(cache);
  a.q = q, a.out = out, a.lengths = lengths, a.counts = counts, a.batch = cache->batch;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q_stride[i], a.out_stride[i] = out_stride[i];
  a.n_query = static_cast<int32_t>(n_query);
  a.group = static_cast<int32_t>(heads / cache->kv_heads);
  a.causal = causal != 0, a.scale = scale * 1.4426950408889634f, a.per_scale = 1.0f / scale, a.lazy = kLazy / a.scale;
  const hipStream_t s = as_stream(stream);
  const int dim = static_cast<int>(cache->head_dim);
  char* ws = static_cast<char*>(workspace);
  for (int i = 0; i < p.parts; ++i) {
    const Part& part = p.part[i];
    a.first_row = static_cast<int32_t>(part.first_row), a.last_row = static_cast<int32_t>(part.last_row);
    a.tiles = static_cast<int32_t>(part.tiles), a.tile_rows = part.tile_rows, a.slots = part.slots, a.least = static_cast<int32_t>(part.least);
    a.held = part.held;
    a.sums = reinterpret_cast<float*>(ws), a.ends = reinterpret_cast<float2*>(ws + part.sums);
    a.firsts = reinterpret_cast<int2*>(ws + part.sums + part.ends);
    ws += part.bytes();
    int run = part.few            ? launch_few(a, part.pieces, dim, dtype, s)
              : dtype == VGO_BF16 ? launch_many<bf16_t>(a, part.pieces, dim, s)
              : dtype == VGO_F16  ? launch_many<f16_t>(a, part.pieces, dim, s)
                                  : launch_many<float>(a, part.pieces, dim, s);
    if (run == VGO_OK && part.slots > 0) {
      run = dtype == VGO_BF16  ? join_pieces<bf16_t>(a, dim, s)
            : dtype == VGO_F16 ? join_pieces<f16_t>(a, dim, s)
                               : join_pieces<float>(a, dim, s);
    }
    if (run != VGO_OK) return run;
  }
  return VGO_OK;
}
