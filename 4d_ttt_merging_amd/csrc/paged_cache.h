// The paged cache of keys and values in 4 bits: its format, and how kernels find a token in it.
//
// 32 channels x of one token and head share a scale 2^e, e the smallest integer of [-125, 125] with max|x| <= 7 * 2^e,
// and each is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} * 2^e (E2M1), the nearest, ties to the even code, at most 6: no
// value is off by more than the scale.  A scale byte is e + 127 (E8M0), 255 where a channel is not finite: the
// whole block then is NaN.  This is what v_cvt_scalef32_pk_{fp4_f32,bf16_fp4} convert, and a code times
// its scale is exact in bf16 (e >= -125 keeps 0.5 * 2^e a normal number, e <= 125 keeps 6 * 2^e finite).
//
// data [pages][kv_heads][page_size / 32] blocks of 32 tokens, 34 * head_dim bytes each:
//   keys' codes    [32 tokens][D / 2]        a lane's 8 (16) bytes are channels of one key, an MFMA operand's order
//   values' codes  [4][D / 2][8 tokens]      two channels of 8 tokens side by side: an operand's order for the
//                                            product with the probabilities, where tokens are the inner dimension
//   keys' scales   [32 tokens][D / 32]
//   values' scales [4][D / 32][8 tokens]
// One block is contiguous so that a tile of keys is one stream of bytes from one base address.
#pragma once

#include "vgo_common.h"

namespace vgo {
namespace paged {

constexpr int kBlock = 32;
constexpr int kMinPage = 32, kMaxPage = 1024;

template <int D>
struct Layout {
  static constexpr int kValues = 16 * D, kKeyScales = 32 * D, kValueScales = 33 * D, kBytes = 34 * D;
  static constexpr int kKeyBytes = D / 2;      // a key's codes
  static constexpr int kGroup = 4 * D;         // eight tokens' values
  static constexpr int kParts = D / 32;        // scales of a token
  static constexpr int kScaleGroup = D / 4;    // eight tokens' values' scales
};

struct Pages {
  uint8_t* data;
  float* mass;           // [pages][page_size] or null
  const int32_t* table;  // [batch][width]
  int64_t pages;
  int64_t width;
  int kv_heads;
  int shift;  // log2 of the page size
};

// Page of token t (not negative) of sequence b, or -1 where the table has none.  The table is read as constant memory, by
// the scalar unit where b and t are the wave's.
__device__ __forceinline__ int page_of(const Pages& p, int64_t b, int64_t t) {
  const int64_t at = t >> p.shift;
  if (at >= p.width) return -1;
  typedef const __attribute__((address_space(4))) int32_t* constant;
  const int id = reinterpret_cast<constant>(reinterpret_cast<uintptr_t>(p.table))[b * p.width + at];
  return id >= 0 && id < p.pages ? id : -1;
}
// The block of a page that holds token t, for one key head.
template <int D>
__device__ __forceinline__ int64_t block_of(const Pages& p, int64_t page, int head, int64_t t) {
  const int blocks = 1 << (p.shift - 5);
  return ((page * p.kv_heads + head) * blocks + ((t >> 5) & (blocks - 1))) * Layout<D>::kBytes;
}

// 2^(byte - 127) of byte kAt of a word; 255 becomes infinity, of which the conversion makes NaN.  One instruction, where
// the shifts and masks of C++ become two for the outer bytes.
template <int kAt>
__device__ __forceinline__ float scale_of(uint32_t word) {
  static_assert(kAt >= 0 && kAt < 4, "four bytes");
  uint32_t r;
  if constexpr (kAt == 0)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(23), "v"(word));
  else if constexpr (kAt == 1)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(23), "v"(word));
  else if constexpr (kAt == 2)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(23), "v"(word));
  else
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(23), "v"(word));
  return __uint_as_float(r);
}

// Checks of the host, shared by the entry points.
int check_cache(const vgo_paged_cache* c);
bool rows_fit(const void* p, const int64_t stride[3], int dtype);  // rows that are read and written by 16 bytes
Pages pages_of(const vgo_paged_cache* c);

}  // namespace paged
}  // namespace vgo
