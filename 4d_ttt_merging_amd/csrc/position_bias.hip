// Relative position bias by buckets, dense: out[h, i, j] = table[bucket(j - start - i), h], and the
// gradient of the table.
//
// Bound: HBM, the one tensor [heads, n_query, n_key] written (forward) or read (gradient) once; the
// table of one head by distance sits in LDS.  A wave takes a segment of one row at a time in 16-byte
// pieces; pieces beyond the buckets' reach, most of a long row, are one value.  In the gradient such
// pieces add up in registers, and the distances within reach, one lane each, in LDS sums that belong
// to the wave: every sum has a fixed order.
//
// 16 heads of 2,058 x 2,058 in bf16 (136 MB): 29 us written (4.6 TB/s; a copy 4.9), 40 us for the gradient (3.4) and
// 4 for the join of its parts; 261 x 1,044 in fp32 (17 MB): 7.5 and 9 us.
#include "masked_attention.h"

namespace vgo {
namespace masked {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kSegment = 2048;  // elements of a row per forward unit
constexpr int kMostRows = 8;    // rows per wave of the gradient

// LDS words of the table by distance: one of padding in 64, so that lanes 8 apart, 64 words on, do
// not share a bank.
__device__ __forceinline__ int padded(int i) { return i + (i >> 6); }
inline int padded_words(int reach) { return 2 * reach + 1 + (2 * reach >> 6); }

template <typename T>
struct Piece {
  static constexpr int kN = 16 / sizeof(T);
  T x[kN] __attribute__((aligned(16)));
};

template <typename T>
struct BiasArgs {
  const T* table;
  T* out;
  int heads, n_query, n_key, start, segments, units;  // units: (row, segment) of one head
  Buckets buckets;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void bias_kernel(const BiasArgs<T> a) {
  constexpr int kN = Piece<T>::kN;
  extern __shared__ float by_distance[];
  const int reach = a.buckets.reach, lane = lane_id();
  const int groups = gridDim.x / a.heads, head = blockIdx.x / groups, first = blockIdx.x % groups;
  for (int i = threadIdx.x; i <= 2 * reach; i += kThreads)
    by_distance[padded(i)] = to_f32(a.table[static_cast<int64_t>(a.buckets.of(i - reach)) * a.heads + head]);
  __syncthreads();
  const T behind = from_f32<T>(by_distance[0]), ahead = from_f32<T>(by_distance[padded(2 * reach)]);
  const auto value = [&](int r) { return from_f32<T>(by_distance[padded(max(-reach, min(reach, r)) + reach)]); };
  for (int u = first * kWaves + (threadIdx.x >> 6); u < a.units; u += groups * kWaves) {
    const int i = u / a.segments, j0 = u % a.segments * kSegment, j1 = min(a.n_key, j0 + kSegment);
    T* row = a.out + (static_cast<int64_t>(head) * a.n_query + i) * a.n_key;
    const int pos = a.start + i;
    // Elements before the first 16-byte boundary, whole pieces, and the rest.
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(row + j0) % 16 / sizeof(T));
    const int lead = min(j1 - j0, skew == 0 ? 0 : kN - skew);
    if (lane < lead) row[j0 + lane] = value(j0 + lane - pos);
    const int body = j0 + lead, pieces = (j1 - body) / kN;
    for (int p = lane; p < pieces; p += 64) {
      const int j = body + p * kN, r = j - pos;
      Piece<T> y;
      if (r + kN - 1 <= -reach || r >= reach) {
        const T x = r > 0 ? ahead : behind;
#pragma unroll
        for (int e = 0; e < kN; ++e) y.x[e] = x;
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e) y.x[e] = value(r + e);
      }
      *reinterpret_cast<Piece<T>*>(row + j) = y;
    }
    const int tail = body + pieces * kN;
    if (tail + lane < j1) row[tail + lane] = value(tail + lane - pos);
  }
}

template <typename T>
struct BiasGradArgs {
  const T* grad;
  float* part;  // [row blocks, buckets, heads]
  int heads, n_query, n_key, start, rows, row_blocks;  // rows: a wave's
  Buckets buckets;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void bias_grad_kernel(const BiasGradArgs<T> a) {
  constexpr int kN = Piece<T>::kN;
  extern __shared__ float lds[];
  const int reach = a.buckets.reach, lane = lane_id(), wave = threadIdx.x >> 6, words = 2 * reach + 1;
  const int block = blockIdx.x % a.row_blocks, head = blockIdx.x / a.row_blocks;
  float* sums = lds + wave * words;  // by distance + reach; the two ends take everything beyond
  for (int i = lane; i < words; i += 64) sums[i] = 0.0f;
  wave_lds_order();
  float behind = 0.0f, ahead = 0.0f;
  for (int k = 0; k < a.rows; ++k) {
    const int i = (block * a.rows + k) * kWaves + wave;
    if (i >= a.n_query) break;
    const T* row = a.grad + (static_cast<int64_t>(head) * a.n_query + i) * a.n_key;
    const int pos = a.start + i;
    const auto single = [&](int j) {
      const float x = to_f32(row[j]);
      const int r = j - pos;
      if (r <= -reach)
        behind += x;
      else if (r >= reach)
        ahead += x;
      else
        sums[r + reach] += x;  // (every lane its own distance)
    };
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    const int lead = min(a.n_key, skew == 0 ? 0 : kN - skew), pieces = (a.n_key - lead) / kN;
    if (lane < lead) single(lane);
#pragma unroll 4
    for (int p = lane; p < pieces; p += 64) {
      const int j = lead + p * kN, r = j - pos;
      const Piece<T> x = *reinterpret_cast<const Piece<T>*>(row + j);
      if (r + kN - 1 <= -reach || r >= reach) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < kN; ++e) t += to_f32(x.x[e]);
        (r > 0 ? ahead : behind) += t;
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          if (r + e <= -reach)
            behind += to_f32(x.x[e]);
          else if (r + e >= reach)
            ahead += to_f32(x.x[e]);
          else
            sums[r + e + reach] += to_f32(x.x[e]);
        }
      }
    }
    const int tail = lead + pieces * kN + lane;
    if (tail < a.n_key) single(tail);
    wave_lds_order();  // (the next row's distances are other lanes')
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) behind += __shfl_xor(behind, off), ahead += __shfl_xor(ahead, off);
  if (lane == 0) sums[0] = behind, sums[2 * reach] = ahead;
  __syncthreads();
  for (int i = threadIdx.x; i < words; i += kThreads)
    lds[i] = ((lds[i] + lds[words + i]) + lds[2 * words + i]) + lds[3 * words + i];
  __syncthreads();
  a.buckets.template gather<kThreads>(
      lds, [&](int t, float s) { a.part[(static_cast<int64_t>(block) * a.buckets.count + t) * a.heads + head] = s; });
}

int check(int64_t n_buckets, int64_t heads, const int32_t* starts, int n_starts, int bidirectional, int64_t query_start,
          int64_t n_query, int64_t n_key, int dtype) {
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "position_bias: unsupported dtype");
  const int64_t most = int64_t{1} << 28;
  VGO_REQUIRE(heads >= 1 && heads < most && n_query >= 0 && n_key >= 0 && n_query < most && n_key < most,
              "position_bias: sizes are below 2^28");
  VGO_REQUIRE(query_start > -most && query_start < most, "position_bias: the first position is below 2^28");
  VGO_REQUIRE(heads * (n_query / kWaves + 1) < (int64_t{1} << 31) &&
                  n_query * ((n_key + kSegment - 1) / kSegment) < (int64_t{1} << 31),
              "position_bias: too many rows");
  VGO_REQUIRE(fits_grid(heads, kThreads), "position_bias: too many heads");
  return check_buckets(n_buckets, starts, n_starts, bidirectional);
}

template <typename T>
int run(BiasArgs<T> a, const void* table, void* out, hipStream_t stream) {
  a.table = static_cast<const T*>(table), a.out = static_cast<T*>(out);
  // Enough work-groups to fill the chip eight times over, each filling the distances once.
  const int64_t want = std::max<int64_t>(1, 8LL * device_cus() / a.heads);
  const int64_t groups = std::min<int64_t>(want, (a.units + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(bias_kernel<T>, dim3(static_cast<unsigned>(groups * a.heads)), dim3(kThreads),
                     padded_words(a.buckets.reach) * 4, stream, a);
  return check_launch("position_bias");
}

template <typename T>
int run_grad(BiasGradArgs<T> a, const void* grad, void* d_table, float* part, int dtype, hipStream_t stream) {
  a.grad = static_cast<const T*>(grad), a.part = part;
  if (a.row_blocks > 0) {
    hipLaunchKernelGGL(bias_grad_kernel<T>, dim3(static_cast<unsigned>(a.row_blocks) * a.heads), dim3(kThreads),
                       static_cast<size_t>(kWaves) * (2 * a.buckets.reach + 1) * 4, stream, a);
    const int status = check_launch("position_bias_grad");
    if (status != VGO_OK) return status;
  }
  return sum_parts(part, a.row_blocks, static_cast<int64_t>(a.buckets.count) * a.heads, d_table, dtype,
                   stream);
}

// Rows of a wave: one until the chip has 16 waves a CU, then up to eight (fewer partial sums).
int rows_of(int64_t heads, int64_t n_query) {
  const int64_t waves = 16LL * device_cus();
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostRows, (heads * n_query + waves - 1) / waves)));
}
int64_t row_blocks_of(int64_t heads, int64_t n_query) {
  const int64_t rows = static_cast<int64_t>(rows_of(heads, n_query)) * kWaves;
  return (n_query + rows - 1) / rows;
}

}  // namespace
}  // namespace masked
}  // namespace vgo

extern "C" int vgo_position_bias(const void* table, int64_t n_buckets, int64_t heads, const int32_t* bucket_starts,
                                 int32_t n_starts, int32_t bidirectional, int64_t query_start, int64_t n_query,
                                 int64_t n_key, void* out, int dtype, void* stream) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status =
      check(n_buckets, heads, bucket_starts, n_starts, bidirectional, query_start, n_query, n_key, dtype);
  if (status != VGO_OK) return status;
  if (n_query == 0 || n_key == 0) return VGO_OK;
  VGO_REQUIRE(table && out, "position_bias: null pointer");
  VGO_REQUIRE(aligned(table, dtype == VGO_F32 ? 4 : 2) && aligned(out, dtype == VGO_F32 ? 4 : 2),
              "position_bias: misaligned pointer");
  const auto fill = [&](auto a) {
    a.heads = static_cast<int>(heads), a.n_query = static_cast<int>(n_query), a.n_key = static_cast<int>(n_key);
    a.start = static_cast<int>(query_start);
    a.segments = static_cast<int>((n_key + kSegment - 1) / kSegment);
    a.units = static_cast<int>(n_query * a.segments);
    a.buckets = make_buckets(static_cast<int>(n_buckets), bucket_starts, n_starts, bidirectional);
    return a;
  };
  const hipStream_t s = as_stream(stream);
  if (dtype == VGO_BF16) return run(fill(BiasArgs<bf16_t>{}), table, out, s);
  if (dtype == VGO_F16) return run(fill(BiasArgs<f16_t>{}), table, out, s);
  return run(fill(BiasArgs<float>{}), table, out, s);
}

extern "C" int vgo_position_bias_grad_workspace(int64_t n_buckets, int64_t heads, int64_t n_query, int64_t n_key,
                                                size_t* bytes) {
  using namespace vgo;
  using namespace vgo::masked;
  VGO_REQUIRE(bytes && n_buckets >= 0 && n_buckets <= 4096 && heads >= 1 && heads < (1 << 28) && n_query >= 0 &&
                  n_query < (1 << 28) && n_key >= 0,
              "position_bias_grad: sizes");
  *bytes = n_key == 0 ? 0 : static_cast<size_t>(row_blocks_of(heads, n_query)) * n_buckets * heads * 4;
  return VGO_OK;
}

extern "C" int vgo_position_bias_grad(const void* grad, int64_t n_buckets, int64_t heads,
                                      const int32_t* bucket_starts, int32_t n_starts, int32_t bidirectional,
                                      int64_t query_start, int64_t n_query, int64_t n_key, void* d_table, int dtype,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status =
      check(n_buckets, heads, bucket_starts, n_starts, bidirectional, query_start, n_query, n_key, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(d_table && (grad || n_query == 0 || n_key == 0), "position_bias_grad: null pointer");
  VGO_REQUIRE(aligned(grad, dtype == VGO_F32 ? 4 : 2) && aligned(d_table, dtype == VGO_F32 ? 4 : 2),
              "position_bias_grad: misaligned pointer");
  const int64_t blocks = n_key == 0 ? 0 : row_blocks_of(heads, n_query);
  VGO_REQUIRE(fits_grid(blocks * heads, kThreads), "position_bias_grad: too many rows");
  const size_t need = static_cast<size_t>(blocks) * n_buckets * heads * 4;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
    return fail(VGO_EWORKSPACE, "position_bias_grad: workspace of " + std::to_string(need) + " bytes needed");
  const auto fill = [&](auto a) {
    a.heads = static_cast<int>(heads), a.n_query = static_cast<int>(n_query), a.n_key = static_cast<int>(n_key);
    a.start = static_cast<int>(query_start), a.row_blocks = static_cast<int>(blocks);
    a.rows = rows_of(heads, n_query);
    a.buckets = make_buckets(static_cast<int>(n_buckets), bucket_starts, n_starts, bidirectional);
    return a;
  };
  float* part = static_cast<float*>(workspace);
  const hipStream_t s = as_stream(stream);
  if (dtype == VGO_BF16) return run_grad(fill(BiasGradArgs<bf16_t>{}), grad, d_table, part, dtype, s);
  if (dtype == VGO_F16) return run_grad(fill(BiasGradArgs<f16_t>{}), grad, d_table, part, dtype, s);
  return run_grad(fill(BiasGradArgs<float>{}), grad, d_table, part, dtype, s);
}
