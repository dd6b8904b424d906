// Masked attention: checks, cutting into tasks and C entries of the forward (kernels:
// masked_attention_fwd.h), and the document ranges of tiles.
#include "masked_attention_fwd.h"

#include <cmath>

namespace vgo {
namespace masked {
namespace {

// The documents' range of every tile, ~ of its first where a row is of none.  One wave per tile, the keys' tiles
// first; bound by the launch (4 us).
__global__ __launch_bounds__(256) void doc_info_kernel(const int* key_docs, const int* query_docs, const int* lengths,
                                                       int n_key, int n_query, int batch, int key_tiles,
                                                       int query_tiles, int2* info) {
  const int id = blockIdx.x * 4 + (threadIdx.x >> 6), lane = lane_id();
  if (id >= batch * (key_tiles + query_tiles)) return;
  const bool key = id < batch * key_tiles;
  const int at = key ? id : id - batch * key_tiles, tiles = key ? key_tiles : query_tiles, n = key ? n_key : n_query;
  const int b = at / tiles, j = at % tiles * kTile + lane;
  const int limit = key && lengths ? max(0, min(n, lengths[b])) : n;
  const int doc = j < limit ? (key ? key_docs : query_docs)[static_cast<int64_t>(b) * n + j] : -1;
  int lo = doc < 0 ? INT_MAX : doc, hi = doc < 0 ? -1 : doc;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
  const bool whole = __all(doc >= 0);
  if (lane == 0) info[id] = int2{whole ? lo : ~lo, hi};
}

}  // namespace

// Time of a launch by splits s, in us.  `tile_us`: a CU's time per tile and work-group where `resident` of them,
// as many as fit it, keep it busy (measured for 128 rows: 0.62 of 64 channels in 16 bits, 1.1 of 128, 4.3 and
// 8.6 in fp32).  They hide each other's waits: of three, one alone takes 1.5 times its share and two 2.3 times
// it, of two one 1.3 times it, and what does not fill the last round costs as much as those few alone.
// Joining takes a launch and the partial states' way out and back (`join_us` per split).  16 heads of
// 8,232 x 8,232 x 64: 412 us unsplit (1,040 tasks, 4.06 a CU), 388 in three; 2,058 x 128: 74 and 82 (in two);
// 2,058 x 64 in fp32: 286 and 187 (in six).  All measured without biases: masses, slopes and tables have no factor here,
// and documents count as if the longest ran over all keys.
int splits_of(const vgo_masked_attn* p, int64_t tasks, int tiles, int resident, double tile_us, double join_us) {
  // A causal mask leaves the tasks half of the tiles where all keys are the queries' own, documents fewer: where
  // more follow, their ends spread and the whole work counts; where all start at once, the longest does (2 x 16
  // heads of 2,058 x 2,058, causal and capped: dQ 91 us unsplit, 79 in two).
  const bool all = !p->causal && !has_documents(p) && !p->key_lengths;
  const double share =
      p->causal ? 1.0 - 0.5 * std::min<double>(p->n_query, p->n_key) / std::max<int64_t>(1, p->n_key) : 1.0;
  const double alone[4][3] = {{}, {0.0}, {0.0, 1.3}, {0.0, 1.5, 2.3}}, one = resident == 1 ? 1.0 : alone[resident][1];
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::min(tiles, 512); s += s < 8 ? 1 : s < 32 ? 4 : 32) {
    const double run = (tiles + s - 1) / s, per_cu = tasks * s / static_cast<double>(device_cus());
    const int most = static_cast<int>(std::ceil(per_cu));
    const double beside = all ? most / resident * resident + alone[resident][most % resident]
                              : std::max(one / share, per_cu * (per_cu <= resident ? 2.0 : 1.15));
    const double us = run * share * beside * tile_us * (p->score_cap > 0.0f ? 1.5 : 1.0) + (s > 1 ? 6.0 + s * join_us : 0.0);
    if (us < least * 0.98) least = us, best = s;
  }
  return best;
}

ForwardPlan forward_plan(const vgo_masked_attn* p, int dtype) {
  ForwardPlan r{};
  const int group = static_cast<int>(p->heads / p->kv_heads);
  const int reach = p->bucket_table && p->n_starts ? p->bucket_starts[p->n_starts - 1] : 1;
  // The heads' tables beside the tiles, in 32 KB (two work-groups a CU of the 16-bit kernels) and in what LDS there is:
  // fp32 tiles of 128 channels leave 31,680 bytes.
  const bool wide = p->head_dim == 128;
  const size_t tile_bytes = dtype == VGO_F32 ? (wide ? Layout<float, 128>::kDistances : Layout<float, 64>::kDistances)
                                             : (wide ? Layout<bf16_t, 128>::kDistances : Layout<bf16_t, 64>::kDistances);
  const size_t tables = static_cast<size_t>(group) * distance_words(reach) * 4;
  const bool table_fits = !p->bucket_table || tables <= std::min<size_t>(32768, kLdsBytes - tile_bytes);
  r.pack = p->n_query < 32 && table_fits ? group : 1;
  r.rows = static_cast<int>(r.pack * p->n_query);
  r.tiles = static_cast<int>(tiles_of(p->n_key));
  const int64_t vheads = p->batch * (p->heads / r.pack);
  constexpr int kRows = 128;  // a task's
  r.row_blocks = (r.rows + kRows - 1) / kRows;
  const int64_t tasks = vheads * r.row_blocks;
  // Few rows a task only wait for their keys: two work-groups a CU at least, up to eight where each keeps four
  // tiles (lengths even out), and no more than the join takes in its stride (32 sequences of 32,928 keys, 4 key
  // heads: 554 us unsplit, 201 in 16; one of them: 541, and 22 in 64).
  if (r.rows <= 32) {
    const int64_t cus = device_cus(), n = std::max<int64_t>(1, tasks), tiles = std::max(1, r.tiles);
    const int64_t want = std::max((2 * cus + n - 1) / n, std::min((8 * cus + n - 1) / n, tiles / 4));
    r.splits = static_cast<int>(std::min<int64_t>({tiles, want, static_cast<int64_t>(std::ceil(std::sqrt(20.0 * tiles)))}));
  } else {
    const double tile_us = dtype == VGO_F32 ? (wide ? 8.6 : 4.3) : wide ? 1.1 : 0.62;
    const double bytes = 8.0 * vheads * r.rows * p->head_dim;
    r.splits = splits_of(p, tasks, r.tiles, dtype == VGO_F32 ? 1 : wide ? 2 : 3, tile_us, bytes / 7e6);
  }
  r.tasks = tasks * r.splits;
  return r;
}

size_t forward_bytes(const vgo_masked_attn* p, const ForwardPlan& plan) {
  size_t n = info_bytes(p);
  if (plan.splits > 1) {
    const size_t rows = static_cast<size_t>(plan.splits) * p->batch * (p->heads / plan.pack) * plan.rows;
    n += align16(rows * p->head_dim * 4) + align16(rows * 12);
  }
  return n;
}

void launch_doc_info(const vgo_masked_attn* p, int2* info, hipStream_t stream) {
  const int key_tiles = static_cast<int>(tiles_of(p->n_key)), query_tiles = static_cast<int>(tiles_of(p->n_query));
  const int64_t waves = p->batch * (static_cast<int64_t>(key_tiles) + query_tiles);
  if (waves == 0) return;
  hipLaunchKernelGGL(doc_info_kernel, dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, stream,
                     p->key_documents, p->query_documents, p->key_lengths, static_cast<int>(p->n_key),
                     static_cast<int>(p->n_query), static_cast<int>(p->batch), key_tiles, query_tiles, info);
}

size_t info_bytes(const vgo_masked_attn* p) {
  return has_documents(p) ? align16(static_cast<size_t>(p->batch) * (tiles_of(p->n_key) + tiles_of(p->n_query)) * 8)
                          : 0;
}

bool strides_fit(const int64_t stride[3], int64_t head_dim, int dtype) {
  const int64_t size = dtype == VGO_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] * size % 16 != 0) return false;
  return stride[2] * size * kTile < (int64_t{1} << 31);  // 32-bit offsets within a tile
}

int check_buckets(int64_t count, const int32_t* starts, int n_starts, int bidirectional) {
  VGO_REQUIRE(n_starts >= 0 && n_starts <= kMaxStarts && (n_starts == 0 || starts), "buckets: at most 128 starts");
  VGO_REQUIRE(count >= (bidirectional ? 2 : 1) * (n_starts + 1) && count <= 4096 && (!bidirectional || count % 2 == 0),
              "buckets: the table must hold every bucket, and at most 4096");
  for (int t = 0; t < n_starts; ++t)
    VGO_REQUIRE(starts[t] >= 1 && starts[t] <= 1024 && (t == 0 || starts[t] >= starts[t - 1]),
                "buckets: starts must ascend within 1 .. 1024");
  return VGO_OK;
}

int check_problem(const vgo_masked_attn* p, int dtype) {
  VGO_REQUIRE(p, "masked_attn: null problem");
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "masked_attn: unsupported dtype");
  VGO_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "masked_attn: head_dim must be 64 or 128");
  VGO_REQUIRE(p->batch >= 0 && p->heads >= 1 && p->kv_heads >= 1 && p->n_query >= 0 && p->n_key >= 0,
              "masked_attn: negative size");
  VGO_REQUIRE(p->heads % p->kv_heads == 0, "masked_attn: heads must be a multiple of the key heads");
  const int64_t most = int64_t{1} << 28;
  VGO_REQUIRE(p->n_query < most && p->n_key < most && p->batch < most && p->heads < most,
              "masked_attn: sizes are below 2^28");
  // Task counts, and rows of all heads, are 32-bit.
  VGO_REQUIRE(p->batch * p->heads < most && (p->batch * p->heads) * (p->n_query / 32 + 1) < most &&
                  p->batch * (p->heads / p->kv_heads) * 32 < most,
              "masked_attn: too many rows");
  VGO_REQUIRE(p->scale > 0.0f && p->scale < kInf, "masked_attn: the scale must be positive and finite");
  VGO_REQUIRE(p->score_cap >= 0.0f && p->score_cap < kInf, "masked_attn: the score cap must be finite and not negative");
  VGO_REQUIRE(!p->prefix_lengths || p->causal, "masked_attn: a prefix goes with a causal mask");
  VGO_REQUIRE(p->batch == 0 || p->n_query == 0 || p->n_key == 0 || !p->query_documents == !p->key_documents,
              "masked_attn: documents of queries and keys go together");
  const auto number = [](int type) { return type == VGO_F32 || type == VGO_BF16 || type == VGO_F16; };
  VGO_REQUIRE((!p->log_mass || number(p->log_mass_dtype)) && (!p->slopes || number(p->slopes_dtype)) &&
                  (!p->bucket_table || number(p->table_dtype)),
              "masked_attn: unsupported dtype of a parameter");
  VGO_REQUIRE(p->batch * (tiles_of(p->n_key) + tiles_of(p->n_query)) < (has_documents(p) ? most / 4 : most),
              "masked_attn: too many rows");  // (documents: a wave a tile)
  if (p->bucket_table) {
    const int status = check_buckets(p->n_buckets, p->bucket_starts, p->n_starts, p->bidirectional);
    if (status != VGO_OK) return status;
  }
  if (p->batch == 0 || p->n_query == 0) return VGO_OK;
  VGO_REQUIRE(p->q && aligned(p->q, 16) && strides_fit(p->q_stride, p->head_dim, dtype),
              "masked_attn: q must be 16-byte aligned, with strides of whole 16 bytes");
  if (p->n_key == 0) return VGO_OK;
  VGO_REQUIRE(p->k && p->v && aligned(p->k, 16) && aligned(p->v, 16) &&
                  strides_fit(p->k_stride, p->head_dim, dtype) && strides_fit(p->v_stride, p->head_dim, dtype),
              "masked_attn: k and v must be 16-byte aligned, with strides of whole 16 bytes");
  return VGO_OK;
}

}  // namespace masked
}  // namespace vgo

extern "C" int vgo_masked_attn_workspace(const vgo_masked_attn* problem, int dtype, size_t* bytes) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_problem(problem, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "masked_attn: null pointer");
  *bytes = 0;
  if (problem->batch == 0 || problem->n_query == 0) return VGO_OK;
  const ForwardPlan plan = forward_plan(problem, dtype);
  VGO_REQUIRE(fits_grid(plan.tasks, 256), "masked_attn: too many rows");
  *bytes = forward_bytes(problem, plan);
  return VGO_OK;
}

extern "C" int vgo_masked_attn_fwd(const vgo_masked_attn* problem, void* out, const int64_t out_stride[3], float* lse,
                                   void* rest, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_problem(problem, dtype);
  if (status != VGO_OK) return status;
  if (problem->batch == 0 || problem->n_query == 0) return VGO_OK;
  VGO_REQUIRE(out && out_stride && aligned(out, 16) && strides_fit(out_stride, problem->head_dim, dtype),
              "masked_attn: out must be 16-byte aligned, with strides of whole 16 bytes");
  VGO_REQUIRE(aligned(rest, 16) && (!rest || dtype != VGO_F32), "masked_attn: rest must be 16-byte aligned, and of a 16-bit type");
  const ForwardPlan plan = forward_plan(problem, dtype);
  VGO_REQUIRE(fits_grid(plan.tasks, 256), "masked_attn: too many rows");
  const size_t need = forward_bytes(problem, plan);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "masked_attn: workspace of " + std::to_string(need) + " bytes needed");
  char* ws = static_cast<char*>(workspace);
  const hipStream_t s = as_stream(stream);
  if (dtype == VGO_BF16) return run_forward<bf16_t>(problem, plan, out, out_stride, lse, rest, ws, s);
  if (dtype == VGO_F16) return run_forward<f16_t>(problem, plan, out, out_stride, lse, rest, ws, s);
  return run_forward<float>(problem, plan, out, out_stride, lse, rest, ws, s);
}
