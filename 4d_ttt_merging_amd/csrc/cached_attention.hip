// Attention over the paged cache of keys and values in 4 bits (paged_cache.h).
#include "cached_attention.h"

#include <algorithm>
#include <cmath>

namespace vgo {
namespace paged {
namespace {

// Joins the pieces of the rows that have several.  A wave takes a row, D / 4 lanes four channels each of every second
// (fourth) piece: what they read does not depend on what they have read, so that up to 8 (16) pieces take one trip to memory.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const Attend a) {
  constexpr int kLanes = D / 4, kGroups = 64 / kLanes;
  const int rows = a.last_row - a.first_row, kv = a.pages.kv_heads;
  const int64_t task = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
  const int hk = static_cast<int>(task % kv), of = static_cast<int>(task / kv % rows);
  const int64_t b = task / kv / rows;
  if (b >= a.batch) return;
  const int2 first = a.firsts[b];
  const int length = length_of(a, b), count = count_of(a, b);
  const int row = a.first_row + of, tile = of / a.tile_rows, tokens = first.y;
  const int stop = stop_of(a, length, count, a.lengths[b] - count, a.first_row + tile * a.tile_rows);
  const int n = (stop - 1) / tokens + 1;
  if (stop <= 0 || n <= 1) return;
  const int group = lane_id() / kLanes, c = lane_id() % kLanes * 4;
  const int64_t step = static_cast<int64_t>(kv) * a.tiles * a.tile_rows;
  const int64_t start = first.x * step + (static_cast<int64_t>(hk) * a.tiles + tile) * a.tile_rows + of % a.tile_rows;
  float top = -INFINITY, sum = 0.0f;
  f32x4 v = {};
  for (int piece = group; piece < n; piece += 4 * kGroups) {
    float2 end[4];
    f32x4 part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t place = start + min(piece + i * kGroups, n - 1) * step;
      end[i] = a.ends[place];
      part[i] = *reinterpret_cast<const f32x4*>(a.sums + place * D + c);
      if (piece + i * kGroups >= n) end[i] = {-INFINITY, 0.0f};
    }
    const float most = fmaxf(fmaxf(top, fmaxf(end[0].x, end[1].x)), fmaxf(end[2].x, end[3].x));
    const float from = most == -INFINITY ? 0.0f : most;
    const float shrink = __builtin_amdgcn_exp2f(top - from);
    top = most, sum *= shrink;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= shrink;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float share = __builtin_amdgcn_exp2f(end[i].x - from);
      sum = fmaf(end[i].y, share, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(part[i][e], share, v[e]);
    }
  }
#pragma unroll
  for (int o = kLanes; o < 64; o <<= 1) {
    const float other = __shfl_xor(top, o), most = fmaxf(top, other), from = most == -INFINITY ? 0.0f : most;
    const float mine = __builtin_amdgcn_exp2f(top - from), theirs = __builtin_amdgcn_exp2f(other - from);
    // (the same products and one sum on both sides: the same bits)
    sum = sum * mine + __shfl_xor(sum, o) * theirs;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] * mine + __shfl_xor(v[e], o) * theirs;
    top = most;
  }
  if (group > 0) return;
  const bool none = row >= count * a.group || top == -INFINITY;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : v[e] / sum;
  store4(static_cast<T*>(a.out) + b * a.out_stride[0] + (hk * a.group + row % a.group) * a.out_stride[1] +
             row / a.group * a.out_stride[2] + c, v);
}

template <typename T>
int merge(const Attend& a, int head_dim, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((a.batch * (a.last_row - a.first_row) * a.pages.kv_heads + 3) / 4);
  if (head_dim == 64) merge_kernel<T, 64><<<grid, 256, 0, s>>>(a);
  else merge_kernel<T, 128><<<grid, 256, 0, s>>>(a);
  return check_launch("cached_attn");
}

}  // namespace

template <>
ManyShape many_shape<bf16_t>(int head_dim, bool causal);
template <>
ManyShape many_shape<f16_t>(int head_dim, bool causal);
template <>
ManyShape many_shape<float>(int head_dim, bool causal);
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
  bool fold;
  int64_t tiles, pieces;
  size_t sums, ends, firsts;  // bytes of the workspace
  size_t bytes() const { return sums + ends + firsts; }
};
struct Plan {
  int parts;
  Part part[2];
  size_t bytes() const { return part[0].bytes() + (parts > 1 ? part[1].bytes() : 0); }
};
Part part_of(const vgo_paged_cache* c, int64_t first_row, int64_t last_row, bool few, int causal, const ManyShape& shape) {
  Part p{};
  const int64_t rows = last_row - first_row, capacity = c->table_width * c->page_size;
  p.few = few, p.first_row = first_row, p.last_row = last_row;
  p.tile_rows = few ? few_tile(rows) : shape.tile_rows;
  p.least = few ? kLeastFew : kLeastMany;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  // As many work-groups as the chip holds at once; of causal calls that leave room, whose tiles differ, twice as many.
  const int64_t held = static_cast<int64_t>(few ? 2 : shape.resident) * device_cus(), beside = c->kv_heads * p.tiles;
  const bool uneven = causal && !few;
  const int64_t slots = (uneven && c->batch * beside <= held / 2 ? 2 * held : held) / beside - c->batch;
  p.fold = uneven && c->batch * beside <= held;
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
Plan plan_of(const vgo_paged_cache* c, int64_t heads, int64_t n_query, int causal, int dtype) {
  Plan p{};
  const int64_t rows = n_query * (heads / c->kv_heads);
  const int dim = static_cast<int>(c->head_dim);
  const ManyShape shape = dtype == VGO_BF16  ? many_shape<bf16_t>(dim, causal)
                          : dtype == VGO_F16 ? many_shape<f16_t>(dim, causal)
                                             : many_shape<float>(dim, causal);
  const int64_t over = rows % shape.tile_rows;
  // Rows of the large tiles.
  const int64_t split = rows <= kFewRows ? 0 : over <= kFewRows && rows >= 4 * shape.tile_rows ? rows - over : rows;
  if (split > 0) p.part[p.parts++] = part_of(c, 0, split, false, causal, shape);
  if (split < rows) p.part[p.parts++] = part_of(c, split, rows, true, causal, shape);
  return p;
}

int check_attend(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int dtype) {
  const int status = check_cache(cache);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "cached_attn: unsupported dtype");
  VGO_REQUIRE(n_query >= 0 && n_query <= INT32_MAX && heads >= 1 && heads <= 65535, "cached_attn: size out of range");
  VGO_REQUIRE(heads % cache->kv_heads == 0, "cached_attn: heads must be a multiple of the key heads");
  return VGO_OK;
}
constexpr int64_t kMostThreads = int64_t{1} << 32;

bool rows_fit(const void* p, const int64_t stride[3], int dtype) {
  const int64_t size = dtype == VGO_F32 ? 4 : 2;
  if (!p || !aligned(p, 16) || !stride) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] * size % 16 != 0) return false;
  return true;
}

}  // namespace
}  // namespace paged
}  // namespace vgo

extern "C" int vgo_cached_attn_workspace(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int causal,
                                         int dtype, size_t* bytes) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_attend(cache, heads, n_query, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "cached_attn: null pointer");
  *bytes = 0;
  if (cache->batch == 0 || n_query == 0) return VGO_OK;
  const Plan p = plan_of(cache, heads, n_query, causal, dtype);
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
  // (a grid's threads are counted in 32 bits; rows and their places among a launch's in 31)
  VGO_REQUIRE(cache->batch < kMostThreads / heads / n_query / 32, "cached_attn: too many rows");
  const Plan p = plan_of(cache, heads, n_query, causal, dtype);
  for (int i = 0; i < p.parts; ++i)
    VGO_REQUIRE(p.part[i].pieces < kMostThreads / 512 / (p.part[i].tiles * cache->kv_heads), "cached_attn: too many rows");
  if (p.bytes() > 0 && (!workspace || workspace_bytes < p.bytes() || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "cached_attn: workspace of " + std::to_string(p.bytes()) + " bytes needed");
  Attend a{};
  a.pages = pages_of(cache);
  a.q = q, a.out = out, a.lengths = lengths, a.counts = counts, a.batch = cache->batch;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q_stride[i], a.out_stride[i] = out_stride[i];
  a.n_query = static_cast<int32_t>(n_query), a.heads = static_cast<int32_t>(heads);
  a.group = static_cast<int32_t>(heads / cache->kv_heads);
  a.causal = causal != 0, a.scale = scale * 1.4426950408889634f, a.per_scale = 1.0f / scale;
  const hipStream_t s = as_stream(stream);
  const int dim = static_cast<int>(cache->head_dim);
  char* ws = static_cast<char*>(workspace);
  for (int i = 0; i < p.parts; ++i) {
    const Part& part = p.part[i];
    a.first_row = static_cast<int32_t>(part.first_row), a.last_row = static_cast<int32_t>(part.last_row);
    a.tiles = static_cast<int32_t>(part.tiles), a.tile_rows = part.tile_rows, a.slots = part.slots, a.least = static_cast<int32_t>(part.least);
    a.fold = part.fold;
    a.sums = reinterpret_cast<float*>(ws), a.ends = reinterpret_cast<float2*>(ws + part.sums);
    a.firsts = reinterpret_cast<int2*>(ws + part.sums + part.ends);
    ws += part.bytes();
    int run = part.few            ? launch_few(a, part.pieces, dim, dtype, s)
              : dtype == VGO_BF16 ? launch_many<bf16_t>(a, part.pieces, dim, s)
              : dtype == VGO_F16  ? launch_many<f16_t>(a, part.pieces, dim, s)
                                  : launch_many<float>(a, part.pieces, dim, s);
    if (run == VGO_OK && part.slots > 0) {
      run = dtype == VGO_BF16  ? merge<bf16_t>(a, dim, s)
            : dtype == VGO_F16 ? merge<f16_t>(a, dim, s)
                               : merge<float>(a, dim, s);
    }
    if (run != VGO_OK) return run;
  }
  return VGO_OK;
}
