// Attention over the paged cache of keys and values in 4 bits (paged_cache.h).
#include "paged_cache.h"

#include <cmath>

namespace vgo {
namespace paged {
namespace {

struct Attend {
  Pages pages;
  const void* q;
  void* out;
  int64_t q_stride[3], out_stride[3];
  const int32_t* lengths;
  const int32_t* counts;
  int64_t n_query, rows;
  int heads, causal;
  float scale;
};

// A wave takes one query of one head; its lanes 64 keys at a time for the scores, then two channels each (one
// of 64) for the values.
template <typename T, int D>
__global__ __launch_bounds__(64) void attend_kernel(const Attend a) {
  using L = Layout<D>;
  constexpr int kEach = D / 64;
  __shared__ float q[D];
  __shared__ float weight[64];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t i = row % a.n_query;
  const int h = static_cast<int>(row / a.n_query % a.heads);
  const int64_t b = row / a.n_query / a.heads;
  const int hk = h / (a.heads / a.pages.kv_heads);
  const int64_t length = min(static_cast<int64_t>(a.lengths[b]), a.pages.width << a.pages.shift);
  const int64_t count = a.counts ? min(max(static_cast<int64_t>(a.counts[b]), int64_t{0}), a.n_query) : a.n_query;
  T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[1] + i * a.out_stride[2];
  const T* from = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[1] + i * a.q_stride[2];
  for (int e = lane; e < D; e += 64) q[e] = to_f32(from[e]) * a.scale;
  __syncthreads();
  int64_t end = a.causal ? min(length, a.lengths[b] - count + i + 1) : length;
  if (i >= count) end = 0;
  float top = -INFINITY, total = 0.0f, acc[kEach] = {};
  for (int64_t j0 = 0; j0 < end; j0 += 64) {
    const int64_t j = j0 + lane;
    const int page = j < end ? page_of(a.pages, b, j) : -1;
    float z = -INFINITY;
    if (page >= 0) {
      const uint8_t* block = a.pages.data + block_of<D>(a.pages, page, hk, j);
      const int slot = static_cast<int>(j) & 31;
      z = 0.0f;
      for (int w = 0; w < D / 8; ++w) {
        const uint32_t word = reinterpret_cast<const uint32_t*>(block + slot * L::kKeyBytes)[w];
        const float s = scale_of<0>(block[L::kKeyScales + slot * L::kParts + w / 4]);
        const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 3)};
        for (int e = 0; e < 8; ++e) z = fmaf(q[8 * w + e], to_f32(p[e / 2][e % 2]), z);
      }
      if (a.pages.mass) z += a.pages.mass[(static_cast<int64_t>(page) << a.pages.shift) + (j & ((1 << a.pages.shift) - 1))];
    }
    float most = z;
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    const float next = fmaxf(top, most), safe = next == -INFINITY ? 0.0f : next;
    const float shrink = expf(top - safe), p = expf(z - safe);
    top = next;
    total = total * shrink + p;
    for (int e = 0; e < kEach; ++e) acc[e] *= shrink;
    __syncthreads();
    weight[lane] = p;
    __syncthreads();
    for (int t = 0; t < 64 && j0 + t < end; ++t) {
      const int at = page_of(a.pages, b, j0 + t);
      if (at < 0) continue;
      const uint8_t* block = a.pages.data + block_of<D>(a.pages, at, hk, j0 + t);
      const int slot = static_cast<int>(j0 + t) & 31;
      for (int e = 0; e < kEach; ++e) {
        const int ch = lane + 64 * e;
        const uint32_t byte = block[L::kValues + slot / 8 * L::kGroup + ch / 2 * 8 + slot % 8];
        const float s = scale_of<0>(block[L::kValueScales + slot / 8 * L::kScaleGroup + ch / 32 * 8 + slot % 8]);
        const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(byte, s, 0);
        acc[e] = fmaf(weight[t], to_f32(v[ch % 2]), acc[e]);
      }
    }
  }
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
  for (int e = 0; e < kEach; ++e) out[lane + 64 * e] = from_f32<T>(total > 0.0f || total != total ? acc[e] / total : 0.0f);
}

int check_attend(const vgo_paged_cache* cache, int64_t heads, int64_t n_query, int dtype) {
  const int status = check_cache(cache);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "cached_attn: unsupported dtype");
  VGO_REQUIRE(n_query >= 0 && n_query <= INT32_MAX && heads >= 1 && heads <= 65535, "cached_attn: size out of range");
  VGO_REQUIRE(heads % cache->kv_heads == 0, "cached_attn: heads must be a multiple of the key heads");
  return VGO_OK;
}
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
  Attend a{};
  a.pages = pages_of(cache);
  a.q = q, a.out = out, a.lengths = lengths, a.counts = counts, a.n_query = n_query;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q_stride[i], a.out_stride[i] = out_stride[i];
  a.heads = static_cast<int>(heads), a.causal = causal, a.scale = scale;
  VGO_REQUIRE(cache->batch < ((int64_t{1} << 32) / 64) / heads / n_query, "cached_attn: too many rows");
  a.rows = cache->batch * heads * n_query;
  const unsigned grid = static_cast<unsigned>(a.rows);
  const hipStream_t s = as_stream(stream);
  if (cache->head_dim == 64) {
    if (dtype == VGO_BF16) attend_kernel<bf16_t, 64><<<grid, 64, 0, s>>>(a);
    else if (dtype == VGO_F16) attend_kernel<f16_t, 64><<<grid, 64, 0, s>>>(a);
    else attend_kernel<float, 64><<<grid, 64, 0, s>>>(a);
  } else {
    if (dtype == VGO_BF16) attend_kernel<bf16_t, 128><<<grid, 64, 0, s>>>(a);
    else if (dtype == VGO_F16) attend_kernel<f16_t, 128><<<grid, 64, 0, s>>>(a);
    else attend_kernel<float, 128><<<grid, 64, 0, s>>>(a);
  }
  return check_launch("cached_attn");
}
