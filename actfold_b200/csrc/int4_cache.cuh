// The 4-bit paged key/value cache: its layout and the arithmetic of its values.
//
// The tokens of a page lie in blocks of 8, per key/value head; a block is one
// run of 10 * HD bytes,
//   [codes of K: 8 rows of HD / 2] [pairs of K: 8 rows of HD / 8] [codes of V] [pairs of V],
// so whole tokens of a head, keys and values, come with one bulk copy. A pair
// is the 16-bit (scale, offset) of 32 dims, and a value is
//   T(code * scale + offset), rounded once (T: fp16 or bf16, the pair's type).
// Word w of a row of codes holds dims 8 w .. 8 w + 7: bits 4 i of its low half
// dim 8 w + 2 i, of its high half dim 8 w + 2 i + 1; so one mask takes two
// neighbours out of a word of a key, and two values of one dim out of a pair of half words of
// two tokens. With 128 dims a row is 64 bytes and the halves of rows 2, 3, 6 and 7
// are swapped: the 32 bytes that four lanes read of each of four rows then
// lie in different banks.
#pragma once

#include "common.cuh"

namespace af {
namespace kv4 {

constexpr int kGroup = 32;  // dims of a pair
constexpr int kBlockTokens = 8;

template <int HD>
struct Block {
  static constexpr int kCodes = HD / 2, kPairs = HD / 8;        // bytes of a row
  static constexpr int kPart = kBlockTokens * (kCodes + kPairs);  // keys, or values
  static constexpr int kBytes = 2 * kPart;
  static constexpr int kPairsAt = kBlockTokens * kCodes;         // within a part
  // Byte of code word w of row r.
  __host__ __device__ static constexpr int word(int r, int w) { return r * kCodes + 4 * (HD == 128 ? w ^ ((r & 2) << 2) : w); }
  __host__ __device__ static constexpr int pair(int r, int group) { return kPairsAt + r * kPairs + 4 * group; }
};

// A page's head is one run of blocks, so entries that share no memory lie at least that far apart.
inline bool runs_apart(const af_int4_cache& c, bool layers) {
  const int64_t run = c.page_size / kBlockTokens * 10 * c.head_dim;
  return (!layers || c.layers <= 1 || c.strides[0] >= run) && (c.pages <= 1 || c.strides[1] >= run) && (c.heads <= 1 || c.strides[2] >= run);
}

template <int DT>
struct Pair16;
template <>
struct Pair16<AF_DTYPE_F16> {
  using type = __half2;
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024: a code in the lowest bits adds to it exactly
  __device__ __forceinline__ static type make(uint32_t b) { return *reinterpret_cast<__half2*>(&b); }
};
template <>
struct Pair16<AF_DTYPE_BF16> {
  using type = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u;  // 128
  __device__ __forceinline__ static type make(uint32_t b) { return *reinterpret_cast<__nv_bfloat162*>(&b); }
};

template <typename H>
__device__ __forceinline__ uint32_t bits_of(H h) {
  return *reinterpret_cast<uint32_t*>(&h);
}

// Codes I of both halves of a word as two values: (x >> 4 I) & 15 each, times scale plus offset.
template <int DT, int I>
__device__ __forceinline__ uint32_t two_values(uint32_t w, uint32_t scale2, uint32_t offset2) {
  using P = Pair16<DT>;
  uint32_t c;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(c) : "r"(I ? w >> (4 * I) : w), "r"(P::kMagic));  // (w & mask) | magic
  return bits_of(__hfma2(__hsub2(P::make(c), P::make(P::kMagic)), P::make(scale2), P::make(offset2)));
}

}  // namespace kv4
}  // namespace af
