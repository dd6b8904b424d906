// Attention over the paged cache of keys and values in 4 bits (paged_cache.h).
#include "cached_attention.h"

#include <algorithm>
#include <cmath>

namespace vgo {
namespace paged {
namespace {

// Joins the pieces of a row: a wave a row, D / 64 channels a lane.  Rows of sequences in one piece are written already.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const Attend a) {
  constexpr int kEach = D / 64;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int rows = a.n_query * a.group, lane = lane_id(), kv = a.pages.kv_heads;
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(at % rows));
  const int64_t rest = at / rows;
  const int hk = __builtin_amdgcn_readfirstlane(static_cast<int>(rest % kv));
  const int64_t b = rest / kv;
  if (b >= a.batch) return;
  const int tokens = piece_tokens(a), length = length_of(a, b);
  const int all = pieces_of(length, tokens);
  if (all == 1) return;
  int64_t first = 0;
  for (int64_t o = lane; o < b; o += 64) first += pieces_of(length_of(a, o), tokens);
  first = wave_sum(first);
  const int count = count_of(a, b), tile = row / a.tile_rows;
  const int last = min((tile + 1) * a.tile_rows, count * a.group) - 1;  // (as the tile's work-groups reckon)
  const int stop = last < tile * a.tile_rows ? 0
                   : a.causal ? max(0, min(length, a.lengths[b] - count + last / a.group + 1)) : length;
  const int n = max(1, (stop + tokens - 1) / tokens);
  const auto place = [&](int piece) {
    return (((first + piece) * kv + hk) * a.tiles + tile) * a.tile_rows + row % a.tile_rows;
  };
  float most = -INFINITY;
  for (int piece = 0; piece < n; ++piece) most = fmaxf(most, a.ends[place(piece)].x);
  const float from = most == -INFINITY ? 0.0f : most;
  float sum = 0.0f, v[kEach] = {};
  for (int piece = 0; piece < n; ++piece) {
    const float2 end = a.ends[place(piece)];
    const float share = __builtin_amdgcn_exp2f(end.x - from);
    sum = fmaf(end.y, share, sum);
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = fmaf(a.sums[place(piece) * D + lane + 64 * e], share, v[e]);
  }
  const bool none = row >= count * a.group || most == -INFINITY;
  T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + (hk * a.group + row % a.group) * a.out_stride[1] +
           row / a.group * a.out_stride[2];
#pragma unroll
  for (int e = 0; e < kEach; ++e) out[lane + 64 * e] = from_f32<T>(none ? 0.0f : v[e] / sum);
}

// How a call is cut.
struct Plan {
  int tile_rows, slots, least;
  int64_t tiles, pieces;
  size_t sums, ends;  // bytes of the workspace
};
Plan plan_of(const vgo_paged_cache* c, int64_t heads, int64_t n_query) {
  Plan p{};
  const int64_t rows = n_query * (heads / c->kv_heads), capacity = c->table_width * c->page_size;
  p.tile_rows = few_rows(rows);
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  p.least = 512;
  const int64_t groups = 2 * device_cus(), beside = c->kv_heads * p.tiles;
  const int64_t slots = groups / beside - c->batch;
  // (no more pieces than the tables could hold)
  p.slots = capacity <= p.least ? 0 : static_cast<int>(std::max<int64_t>(0, std::min(slots, c->batch * ((capacity - 1) / p.least))));
  p.pieces = c->batch + p.slots;
  if (p.slots > 0) {
    const size_t parts = static_cast<size_t>(p.pieces) * beside * p.tile_rows;
    p.sums = parts * c->head_dim * sizeof(float);
    p.ends = parts * sizeof(float2);
  }
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
// A grid's threads are counted in 32 bits; work-groups of 512.
constexpr int64_t kMostGroups = (int64_t{1} << 32) / 512;

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

extern "C" int vgo_cached_attn_workspace(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int dtype,
                                         size_t* bytes) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_attend(cache, heads, n_query, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "cached_attn: null pointer");
  *bytes = 0;
  if (cache->batch == 0 || n_query == 0) return VGO_OK;
  const Plan p = plan_of(cache, heads, n_query);
  *bytes = p.sums + p.ends;
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
  VGO_REQUIRE(scale > 0.0f && scale < INFINITY, "cached_attn: the scale must be positive and finite");
  if (cache->batch == 0 || n_query == 0) return VGO_OK;
  VGO_REQUIRE(lengths, "cached_attn: null lengths");
  VGO_REQUIRE(rows_fit(q, q_stride, dtype) && rows_fit(out, out_stride, dtype),
              "cached_attn: q and out must be 16-byte aligned, with strides of whole 16 bytes");
  const Plan p = plan_of(cache, heads, n_query);
  VGO_REQUIRE(p.pieces < kMostGroups / (p.tiles * cache->kv_heads) && cache->batch < kMostGroups * 8 / heads / n_query,
              "cached_attn: too many rows");  // (the join: four rows a work-group of 256)
  if (p.sums > 0 && (!workspace || workspace_bytes < p.sums + p.ends || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "cached_attn: workspace of " + std::to_string(p.sums + p.ends) + " bytes needed");
  Attend a{};
  a.pages = pages_of(cache);
  a.q = q, a.out = out, a.lengths = lengths, a.counts = counts, a.batch = cache->batch;
  a.sums = static_cast<float*>(workspace), a.ends = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.sums);
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q_stride[i], a.out_stride[i] = out_stride[i];
  a.n_query = static_cast<int32_t>(n_query), a.heads = static_cast<int32_t>(heads);
  a.group = static_cast<int32_t>(heads / cache->kv_heads);
  a.tiles = static_cast<int32_t>(p.tiles), a.tile_rows = p.tile_rows, a.slots = p.slots, a.least = p.least;
  a.causal = causal != 0, a.scale = scale * 1.4426950408889634f;
  const hipStream_t s = as_stream(stream);
  const int run = launch_few(a, p.pieces, static_cast<int>(cache->head_dim), dtype, s);
  if (run != VGO_OK || p.slots == 0) return run;
  const unsigned grid = static_cast<unsigned>((cache->batch * heads * n_query + 3) / 4);
  if (cache->head_dim == 64) {
    if (dtype == VGO_BF16) merge_kernel<bf16_t, 64><<<grid, 256, 0, s>>>(a);
    else if (dtype == VGO_F16) merge_kernel<f16_t, 64><<<grid, 256, 0, s>>>(a);
    else merge_kernel<float, 64><<<grid, 256, 0, s>>>(a);
  } else {
    if (dtype == VGO_BF16) merge_kernel<bf16_t, 128><<<grid, 256, 0, s>>>(a);
    else if (dtype == VGO_F16) merge_kernel<f16_t, 128><<<grid, 256, 0, s>>>(a);
    else merge_kernel<float, 128><<<grid, 256, 0, s>>>(a);
  }
  return check_launch("cached_attn");
}
