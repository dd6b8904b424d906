// Appending tokens to the paged cache of keys and values (paged_cache.h) and reading them back.
#include "paged_cache.h"

#include <algorithm>

namespace vgo {
namespace paged {

int check_cache(const vgo_paged_cache* c) {
  VGO_REQUIRE(c, "paged cache: null pointer");
  VGO_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "paged cache: head_dim must be 64 or 128");
  VGO_REQUIRE(c->page_size >= kMinPage && c->page_size <= kMaxPage && (c->page_size & (c->page_size - 1)) == 0,
              "paged cache: the page size must be a power of two from 32 to 1,024");
  VGO_REQUIRE(c->pages >= 0 && c->pages <= INT32_MAX && c->kv_heads >= 1 && c->kv_heads <= 65535 && c->batch >= 0 &&
                  c->batch <= INT32_MAX && c->table_width >= 0 && c->table_width <= (int64_t{1} << 30) / c->page_size,
              "paged cache: size out of range");
  VGO_REQUIRE(c->pages == 0 || (c->data && aligned(c->data, 16)), "paged cache: the data must be 16-byte aligned");
  VGO_REQUIRE(aligned(c->log_mass, 4), "paged cache: the masses must be aligned as floats are");
  VGO_REQUIRE(c->batch == 0 || c->table_width == 0 || c->page_table, "paged cache: null page table");
  return VGO_OK;
}

bool rows_fit(const void* p, const int64_t stride[3], int dtype) {
  const int64_t size = dtype == VGO_F32 ? 4 : 2;
  if (!p || !aligned(p, 16) || !stride) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] * size % 16 != 0) return false;
  return true;
}

Pages pages_of(const vgo_paged_cache* c) {
  int shift = 5;
  while ((int64_t{1} << shift) < c->page_size) ++shift;
  return {static_cast<uint8_t*>(c->data), c->log_mass, c->page_table, c->pages, c->table_width,
          static_cast<int>(c->kv_heads), shift};
}

namespace {

typedef __attribute__((__vector_size__(16))) uint32_t u32x4;

struct Append {
  Pages pages;
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  int64_t k_stride[3], v_stride[3], q_stride[3], out_stride[3];  // elements
  const int32_t* starts;
  const int32_t* counts;
  const float* sin;
  const float* cos;
  const int32_t* positions;
  const float* log_mass;
  int64_t rope_rows, n;
  int heads;  // of q; 0 without it
  int64_t items, groups;
  int chunks, per;  // chunks of `per` heads of k, q and v together
};

// Eight consecutive channels of a row, as they are in memory, and as fp32.
template <typename T>
struct Raw {
  u32x4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw<T> raw8(const T* p) {
  Raw<T> r;
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const u32x4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void widened(const Raw<T>& r, float (&x)[8]) {
  typedef __attribute__((__vector_size__(16))) T vec;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    constexpr int kEach = 16 / sizeof(T);
    x[i] = to_f32(__builtin_bit_cast(vec, r.w[i / kEach])[i % kEach]);
  }
}

// The channels of lane ^ kLanes, 4 or 8, by the LDS unit's crossbar.
template <int kLanes, typename T>
__device__ __forceinline__ Raw<T> across(const Raw<T>& r) {
  Raw<T> o;
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o.w[i][e] = static_cast<uint32_t>(__builtin_amdgcn_ds_swizzle(static_cast<int>(r.w[i][e]), kLanes << 10 | 0x1f));
  return o;
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) { widened(raw8(p), x); }
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    store4(p, f32x4{x[0], x[1], x[2], x[3]});
    store4(p + 4, f32x4{x[4], x[5], x[6], x[7]});
  } else {
    typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec;
    vec o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(x[i]);
    *reinterpret_cast<vec*>(p) = o;
  }
}

// The scale byte of a block whose largest magnitude has these bits (NaN counts as past infinity).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  const int e = static_cast<int>(top >> 23) - ((top & 0x7fffffu) > 0x600000u ? 1 : 2);  // 7 = 1.75 * 2^2
  return static_cast<uint32_t>(min(max(e, 2), 252));
}
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  const auto other = [](uint32_t v, auto at) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), decltype(at)::value, 0xF, 0xF, true));
  };
  x = max(x, other(x, std::integral_constant<int, 0xB1>()));  // lane ^ 1
  return max(x, other(x, std::integral_constant<int, 0x4E>()));  // lane ^ 2
}
// The largest magnitude of 32 channels, eight of this lane and its quad's, as bits.
__device__ __forceinline__ uint32_t top_of(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return quad_max(top);
}
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale) {
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[0], x[1], scale, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[2], x[3], scale, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[4], x[5], scale, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[6], x[7], scale, 3);
  return word;
}
__device__ __forceinline__ float factor_of(uint32_t byte) { return __uint_as_float(byte == 255 ? 0x3f800000u : byte << 23); }
// Codes of eight channels; `byte` gets the scale of the 32 that this lane's quad holds.
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], uint32_t& byte) {
  byte = scale_byte(top_of(x));
  return codes_of(x, factor_of(byte));
}

// fp32 of a 64-bit number, rounded to odd: what is cut off leaves the last bit set, so that a later rounding
// to fewer bits, or a comparison with a number of fewer bits, comes out as for the 64-bit number itself.
__device__ __forceinline__ float to_odd(double d) {
  const float f = static_cast<float>(d);
  uint32_t bits = __float_as_uint(f);
  const double back = static_cast<double>(f);
  if (back != d && d == d) {
    if (fabs(back) > fabs(d)) bits -= 1;
    bits |= 1;
  }
  return __uint_as_float(bits);
}

// Codes of x cos + o sin, exactly those of the 64-bit value: fp32 first, which is off by at most 2^-24 of the
// product x cos and of the sum each; where the codes, or the scale, at the two ends of four times that differ in some
// channel of the wave (about one of 500 waves), 64 bits.  The ends, and not the largest magnitude, say whether the
// scale is certain: a channel's partner is in another block, so that all of a block may cancel to far less than its parts.
// (64 bits throughout kept the vector unit busy for three times as long as
// memory takes: 4 ragged prompts of up to 8,232 tokens, 16 heads of 64 channels, 184 us, this 67.)
__device__ __forceinline__ uint32_t quantise_rotated(const float (&x)[8], const float (&o)[8], const float (&sin)[8],
                                                     const float (&cos)[8], bool real, uint32_t& byte) {
  float y[8], low[8], high[8];
  float least = 0.0f, most = 0.0f;  // what the largest magnitude is at least, and at most; NaN in any channel is kept
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float part = x[i] * cos[i];
    y[i] = fmaf(o[i], sin[i], part);
    const float off = fabsf(part) + fabsf(y[i]);
    low[i] = fmaf(off, -0x1p-22f, y[i]), high[i] = fmaf(off, 0x1p-22f, y[i]);
    least = __builtin_elementwise_maximum(__builtin_elementwise_maximum(least, low[i]), -high[i]);
    most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, high[i]), -low[i]);
  }
  const uint32_t top = quad_max(__float_as_uint(most) & 0x7fffffffu);
  byte = scale_byte(top);
  const float scale = factor_of(byte);
  const uint32_t word = codes_of(low, scale);
  // Numbers near the ends of fp32, and those that are not finite, are left to 64 bits.
  const bool plain = word == codes_of(high, scale) && byte == scale_byte(quad_max(__float_as_uint(least) & 0x7fffffffu)) &&
                     top > 0x10000000u && top < 0x7e000000u;
  if (__all(plain || !real)) return word;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = to_odd(fma(static_cast<double>(o[i]), static_cast<double>(sin[i]), static_cast<double>(x[i]) * cos[i]));
  return quantise(y, byte);
}
// Bytes of four lanes `kStep` apart as a 4 x 4 matrix, transposed: byte c of lane r goes to byte r of lane c
// (r counts in steps of kStep).  Its own inverse.
template <int kStep>
__device__ __forceinline__ uint32_t transposed_bytes(uint32_t w) {
  const int lane = lane_id();
  uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), kStep));
  // (v_perm: bytes 0-3 are the second operand's, 4-7 the first's)
  w = (lane & kStep) ? __builtin_amdgcn_perm(w, o, 0x07030501) : __builtin_amdgcn_perm(o, w, 0x06020400);
  o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), 2 * kStep));
  return (lane & (2 * kStep)) ? __builtin_amdgcn_perm(w, o, 0x07060302) : __builtin_amdgcn_perm(o, w, 0x05040100);
}

// A wave takes 512 / D tokens, all or half of those that share position / 8 (whose values of a channel pair are eight bytes
// of the format), and `per` heads of k, q and v, one after the other with the next one's channels on their way; a lane
// eight channels of a token.
template <typename T, int D>
__global__ __launch_bounds__(256, 5) void append_kernel(const Append a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;            // of a token
  constexpr int kTokens = 64 / kLanes, kParts = 8 / kTokens;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.items) return;
  const int lane = lane_id();
  const int chunk = static_cast<int>(item % a.chunks);
  const int64_t rest = item / a.chunks, group = rest / kParts % a.groups, b = rest / kParts / a.groups;
  const int64_t start = a.starts[b];
  const int64_t count = a.counts ? min(max(static_cast<int64_t>(a.counts[b]), int64_t{0}), a.n) : a.n;
  const int64_t first = (start & ~int64_t{7}) + 8 * group;
  const int c = lane % kLanes;  // its channels 8c ..
  const bool low = c < kLanes / 2;
  const int page = first >= 0 ? page_of(a.pages, b, first) : -1;
  const int kv = a.pages.kv_heads;
  const bool rotate = a.sin != nullptr;
  const int begin = chunk * a.per, end = min(begin + a.per, 2 * kv + a.heads);
  const int j = static_cast<int>(rest % kParts) * kTokens + lane / kLanes;
  const int64_t t = first + j, i = t - start;
  const bool inside = i >= 0 && i < a.n, real = i >= 0 && i < count;
  if (!__any(inside)) return;
  if (!__any(real)) {  // padding alone: nothing to read
    const float zeros[8] = {};
    for (int h = max(begin - kv, 0); h < min(end - kv, a.heads); ++h)
      if (inside) store8(static_cast<T*>(a.q_out) + b * a.out_stride[0] + h * a.out_stride[1] + i * a.out_stride[2] + 8 * c, zeros);
    return;
  }
  const int64_t at_row = min(max(i, int64_t{0}), a.n - 1);  // (padding lanes read some row of the call)
  const int slot = static_cast<int>(t) & 31;
  bool turned = false;
  float sin[8], cos[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sin[e] = 0.0f, cos[e] = 1.0f;
  if (rotate && real) {
    const int64_t row = a.positions ? a.positions[b * a.n + i] : t;
    turned = row >= 0 && row < a.rope_rows;
    if (turned) {
      load8(a.sin + row * D + 8 * c, sin);
      load8(a.cos + row * D + 8 * c, cos);
    }
  }
  if (chunk == 0 && a.pages.mass && real && page >= 0 && c == 0)
    a.pages.mass[(static_cast<int64_t>(page) << a.pages.shift) + (t & ((1 << a.pages.shift) - 1))] =
        a.log_mass ? a.log_mass[b * a.n + i] : 0.0f;
  // The channels of virtual head `at`: keys' heads, the queries', the values'.
  const int64_t k_row = at_row * a.k_stride[2] + 8 * c, q_row = at_row * a.q_stride[2] + 8 * c, v_row = at_row * a.v_stride[2] + 8 * c;
  const auto read = [&](int at, Raw<T>& x) {
    const T* from;
    if (at < kv) from = static_cast<const T*>(a.k) + b * a.k_stride[0] + at * a.k_stride[1] + k_row;
    else if (at < kv + a.heads) from = static_cast<const T*>(a.q) + b * a.q_stride[0] + (at - kv) * a.q_stride[1] + q_row;
    else from = static_cast<const T*>(a.v) + b * a.v_stride[0] + (at - kv - a.heads) * a.v_stride[1] + v_row;
    x = raw8(from);
  };
  const auto use = [&](int at, const Raw<T>& raw) {
    const bool key = at < kv, value = at >= kv + a.heads;
    float x[8], other[8];
    widened(raw, x);
    uint32_t byte = 0, word = 0;
    if (rotate && !value) {
      widened(across<kLanes / 2>(raw), other);
#pragma unroll
      for (int e = 0; e < 8; ++e) other[e] = !turned ? 0.0f : low ? -other[e] : other[e];  // (not turned: x 1 + 0 0)
    }
    if (!key && !value) {
      if (rotate) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(other[e], sin[e], x[e] * cos[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = real ? x[e] : 0.0f;
      if (inside)
        store8(static_cast<T*>(a.q_out) + b * a.out_stride[0] + (at - kv) * a.out_stride[1] + i * a.out_stride[2] + 8 * c, x);
      return;
    }
    if (rotate && key) word = quantise_rotated(x, other, sin, cos, real, byte);
    else word = quantise(x, byte);
    if (value) word = transposed_bytes<kLanes>(word);
    if (page < 0) return;
    uint8_t* block = a.pages.data + block_of<D>(a.pages, page, key ? at : at - kv - a.heads, first);
    if (key) {
      if (real) {
        *reinterpret_cast<uint32_t*>(block + static_cast<uint32_t>(slot * L::kKeyBytes + 4 * c)) = word;
        if (c % 4 == 0) block[static_cast<uint32_t>(L::kKeyScales + slot * L::kParts + c / 4)] = static_cast<uint8_t>(byte);
      }
      return;
    }
    if (real && c % 4 == 0)
      block[static_cast<uint32_t>(L::kValueScales + slot / 8 * L::kScaleGroup + c / 4 * 8 + slot % 8)] = static_cast<uint8_t>(byte);
    // Four tokens of channel pair 4c + j % 4; tokens that are not this call's keep their bytes.
    const int64_t four = i - j % 4;
    uint8_t* to = block + static_cast<uint32_t>(L::kValues + slot / 8 * L::kGroup + (4 * c + j % 4) * 8 + (slot & 4));
    if (four >= 0 && four + 3 < count) {
      *reinterpret_cast<uint32_t*>(to) = word;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (four + e >= 0 && four + e < count) to[e] = static_cast<uint8_t>(word >> (8 * e));
    }
  };
  Raw<T> x0{}, x1{};
  read(begin, x0);
  for (int at = begin; at < end; at += 2) {
    if (at + 1 < end) read(at + 1, x1);
    use(at, x0);
    if (at + 2 < end) read(at + 2, x0);
    if (at + 1 < end) use(at + 1, x1);
  }
}

struct Read {
  Pages pages;
  void* k;
  void* v;
  const int32_t* starts;
  const int32_t* counts;
  int64_t n, items, groups;
  int chunks, per;  // chunks of `per` heads of keys and values together
};

// The inverse: a wave takes eight tokens and `per` heads of keys and values, four heads' codes on their way together.
template <typename T, int D>
__global__ __launch_bounds__(256) void read_kernel(const Read a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8, kTokens = 64 / kLanes, kParts = 8 / kTokens, kAhead = 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.items) return;
  const int lane = lane_id(), kv = a.pages.kv_heads;
  const int chunk = static_cast<int>(item % a.chunks);
  const int64_t rest = item / a.chunks, group = rest / kParts % a.groups, b = rest / kParts / a.groups;
  const int64_t start = a.starts[b];
  const int64_t count = a.counts ? min(max(static_cast<int64_t>(a.counts[b]), int64_t{0}), a.n) : a.n;
  const int64_t first = (start & ~int64_t{7}) + 8 * group;
  const int c = lane % kLanes;
  const int page = first >= 0 && a.pages.pages > 0 ? page_of(a.pages, b, first) : -1;
  const int begin = chunk * a.per, end = min(begin + a.per, 2 * kv);
  const int j = static_cast<int>(rest % kParts) * kTokens + lane / kLanes;
  const int64_t t = first + j, i = t - start;
  const int slot = static_cast<int>(t) & 31;
  const bool inside = i >= 0 && i < a.n, real = inside && i < count;
  const uint32_t key_at = slot * L::kKeyBytes + 4 * c, key_scale_at = L::kKeyScales + slot * L::kParts + c / 4;
  const uint32_t value_at = L::kValues + slot / 8 * L::kGroup + (4 * c + j % 4) * 8 + (slot & 4);
  const uint32_t value_scale_at = L::kValueScales + slot / 8 * L::kScaleGroup + c / 4 * 8 + slot % 8;
  for (int at0 = begin; at0 < end; at0 += kAhead) {
    uint32_t words[kAhead] = {}, bytes[kAhead] = {};
    if (page >= 0 && __any(real)) {
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int at = min(at0 + e, end - 1);
        const bool value = at >= kv;
        const uint8_t* block = a.pages.data + block_of<D>(a.pages, page, value ? at - kv : at, first);
        words[e] = *reinterpret_cast<const uint32_t*>(block + (value ? value_at : key_at));
        bytes[e] = block[value ? value_scale_at : key_scale_at];
      }
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int at = at0 + e;
      if (at >= end) break;
      const bool value = at >= kv;
      uint32_t word = words[e];
      if (value) word = transposed_bytes<kLanes>(word);
      if (!inside) continue;
      if (!real) word = 0, bytes[e] = 0;  // beyond the sequence's tokens: zeros
      const float scale = scale_of<0>(bytes[e]);
      const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
      const bf16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
      const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
      const bf16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
      const float x[8] = {to_f32(p0[0]), to_f32(p0[1]), to_f32(p1[0]), to_f32(p1[1]),
                          to_f32(p2[0]), to_f32(p2[1]), to_f32(p3[0]), to_f32(p3[1])};
      store8(static_cast<T*>(value ? a.v : a.k) + ((b * kv + (value ? at - kv : at)) * a.n + i) * D + 8 * c, x);
    }
  }
}

template <template <typename, int> class Launch, typename Args>
int by_type(const Args& a, int64_t head_dim, int dtype, hipStream_t s) {
  if (head_dim == 64) {
    if (dtype == VGO_BF16) return Launch<bf16_t, 64>::run(a, s);
    if (dtype == VGO_F16) return Launch<f16_t, 64>::run(a, s);
    return Launch<float, 64>::run(a, s);
  }
  if (dtype == VGO_BF16) return Launch<bf16_t, 128>::run(a, s);
  if (dtype == VGO_F16) return Launch<f16_t, 128>::run(a, s);
  return Launch<float, 128>::run(a, s);
}
template <typename T, int D>
struct LaunchAppend {
  static int run(const Append& a, hipStream_t s) {
    append_kernel<T, D><<<static_cast<unsigned>((a.items + 3) / 4), 256, 0, s>>>(a);
    return check_launch("cache_append");
  }
};
template <typename T, int D>
struct LaunchRead {
  static int run(const Read& a, hipStream_t s) {
    read_kernel<T, D><<<static_cast<unsigned>((a.items + 3) / 4), 256, 0, s>>>(a);
    return check_launch("cache_read");
  }
};

bool known(int dtype) { return dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16; }
// Heads that a wave takes one after the other: more where there are waves enough without (the tables' rows, the page and
// the addresses are then fetched once for them).
int heads_of_a_wave(int64_t groups, int heads) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, groups >= (int64_t{1} << 40) ? 8 : groups * heads / 2048)));
}
// A grid's threads are counted in 32 bits; four items a work-group of 256.
constexpr int64_t kMostItems = ((int64_t{1} << 32) / 256 - 1) * 4;

}  // namespace
}  // namespace paged
}  // namespace vgo

extern "C" int vgo_cache_append(const vgo_paged_cache* cache, const vgo_cache_tokens* tokens, int dtype, void* stream) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_cache(cache);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(tokens, "cache_append: null pointer");
  VGO_REQUIRE(known(dtype), "cache_append: unsupported dtype");
  const vgo_cache_tokens& t = *tokens;
  VGO_REQUIRE(t.n_tokens >= 0 && t.n_tokens <= INT32_MAX && t.heads >= 0 && t.heads <= 65535,
              "cache_append: size out of range");
  VGO_REQUIRE(!t.rope_sin == !t.rope_cos && (!t.rope_sin || t.rope_rows >= 0),
              "cache_append: the rotation's two tables go together");
  VGO_REQUIRE(!t.positions || t.rope_sin, "cache_append: positions go with a rotation");
  VGO_REQUIRE(!t.log_mass || cache->log_mass, "cache_append: this cache holds no masses");
  VGO_REQUIRE(aligned(t.rope_sin, 16) && aligned(t.rope_cos, 16), "cache_append: the tables must be 16-byte aligned");
  if (cache->batch == 0 || t.n_tokens == 0) return VGO_OK;
  VGO_REQUIRE(t.starts, "cache_append: null starts");
  VGO_REQUIRE(rows_fit(t.k, t.k_stride, dtype) && rows_fit(t.v, t.v_stride, dtype) &&
                  (t.heads == 0 || (rows_fit(t.q, t.q_stride, dtype) && rows_fit(t.q_out, t.q_out_stride, dtype))),
              "cache_append: operands must be 16-byte aligned, with strides of whole 16 bytes");
  Append a{};
  a.pages = pages_of(cache);
  a.k = t.k, a.v = t.v, a.q = t.q, a.q_out = t.q_out;
  for (int i = 0; i < 3; ++i) {
    a.k_stride[i] = t.k_stride[i], a.v_stride[i] = t.v_stride[i];
    a.q_stride[i] = t.q_stride[i], a.out_stride[i] = t.q_out_stride[i];
  }
  a.starts = t.starts, a.counts = t.counts, a.sin = t.rope_sin, a.cos = t.rope_cos, a.positions = t.positions;
  a.log_mass = t.log_mass, a.rope_rows = t.rope_rows, a.n = t.n_tokens, a.heads = static_cast<int>(t.heads);
  a.groups = (t.n_tokens + 14) / 8;  // (a sequence may start anywhere in its first group)
  const int all = static_cast<int>(2 * cache->kv_heads) + a.heads;
  a.per = heads_of_a_wave(cache->batch * a.groups, all);
  a.chunks = (all + a.per - 1) / a.per;
  VGO_REQUIRE(cache->batch <= kMostItems / 2 / a.groups / a.chunks, "cache_append: too many tokens");
  a.items = cache->batch * a.groups * a.chunks * (cache->head_dim / 64);
  return by_type<LaunchAppend>(a, cache->head_dim, dtype, as_stream(stream));
}

extern "C" int vgo_cache_read(const vgo_paged_cache* cache, const int32_t* starts, const int32_t* counts, int64_t n_tokens,
                              void* k, void* v, int dtype, void* stream) {
  using namespace vgo;
  using namespace vgo::paged;
  const int status = check_cache(cache);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(known(dtype), "cache_read: unsupported dtype");
  VGO_REQUIRE(n_tokens >= 0 && n_tokens <= INT32_MAX, "cache_read: size out of range");
  if (cache->batch == 0 || n_tokens == 0) return VGO_OK;
  VGO_REQUIRE(starts, "cache_read: null starts");
  VGO_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16), "cache_read: outputs must be 16-byte aligned");
  Read a{};
  a.pages = pages_of(cache);
  a.k = k, a.v = v, a.starts = starts, a.counts = counts, a.n = n_tokens;
  a.groups = (n_tokens + 14) / 8;
  const int all = static_cast<int>(2 * cache->kv_heads);
  a.per = heads_of_a_wave(cache->batch * a.groups, all);
  a.chunks = (all + a.per - 1) / a.per;
  VGO_REQUIRE(cache->batch <= kMostItems / 2 / a.groups / a.chunks, "cache_read: too many tokens");
  a.items = cache->batch * a.groups * a.chunks * (cache->head_dim / 64);
  return by_type<LaunchRead>(a, cache->head_dim, dtype, as_stream(stream));
}
