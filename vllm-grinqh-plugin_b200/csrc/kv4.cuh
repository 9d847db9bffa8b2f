// Layout of the paged KV cache held in 4 bits (include/grinqh_b200.h): one record per
// 16 tokens of a head, so that a record is one bulk copy and its words are the operand
// fragments of the attention kernel.
//
// Where a word lies follows from the m16n8k16 matrix instruction (kv4_attention.cu). As
// operand A a lane 4 g + t holds rows g and g + 8 and, of the contracted index, the
// entries of thread t; the contracted index may be numbered in any order.
//   scores  rows = tokens, contracted = channels: thread t needs a quarter of every
//           group's channels of its tokens: chunk c = t of a K row;
//   output  rows = channels, contracted = tokens: lane (g, t) needs an eighth of every
//           group's channels, of the token pairs t and t + 4: chunk c = g of two V rows.
// A chunk is D/32 words (16 or 8 bytes), one shared-memory load. The chunks of a V row
// are permuted by XOR with 2 (row mod 4): the four rows of a load start in the same
// bank, and the XOR spreads their chunks over all banks.
#pragma once

#include "common.cuh"

namespace grinqh {

constexpr int kTile = 16;  // tokens of a record

template <int D, int GS>
struct Kv4 {
  static_assert(D == 64 || D == 128, "head_dim");
  static_assert((GS == 32 || GS == 64 || GS == 128) && GS <= D, "group_size");
  static constexpr int kDim = D, kGroup = GS;
  static constexpr int NG = D / GS;             // groups of a token
  static constexpr int kWords = D / 32;         // words of a chunk
  static constexpr int kGroupWords = GS / 32;   // of them in one group
  static constexpr int kV = 8 * D;              // byte offsets in a record
  static constexpr int kKParams = 16 * D;
  static constexpr int kVParams = 16 * D + 64 * NG;
  static constexpr int kRecord = 16 * D + 128 * NG;

  // K: word (8 channels, bits 4 e) of a token's row that holds channels d .. d + 7, d % 8 == 0
  static __host__ __device__ constexpr int k_word(int d) {
    const int g = d / GS, r = d % GS;
    return (r / (GS / 4)) * kWords + g * kGroupWords + (r % (GS / 4)) / 8;
  }
  // V: word (4 channels of a token pair) of row `pair` that holds channels d .. d + 3, d % 4 == 0
  static __host__ __device__ constexpr int v_word(int pair, int d) {
    const int g = d / GS, r = d % GS;
    return ((r / (GS / 8)) ^ (2 * (pair & 3))) * kWords + g * kGroupWords + (r % (GS / 8)) / 4;
  }
};

inline bool kv4_supported(int dim, int group) {
  return (dim == 64 || dim == 128) && (group == 32 || group == 64 || group == 128) && group <= dim;
}

inline int64_t kv4_record(int dim, int group) {
  return kv4_supported(dim, group) ? 16 * (int64_t)dim + 128 * (dim / group) : 0;
}

// Calls f with the Kv4 of a supported pair.
template <typename F>
int kv4_dispatch(int dim, int group, F&& f) {
  if (dim == 128) {
    if (group == 128) return f(Kv4<128, 128>{});
    if (group == 64) return f(Kv4<128, 64>{});
    return f(Kv4<128, 32>{});
  }
  if (group == 64) return f(Kv4<64, 64>{});
  return f(Kv4<64, 32>{});
}

// Shared checks of the entry points that take a cache.
inline int kv4_check_cache(const void* cache, int64_t pages, int page_size, int kv_heads, int dim, int group) {
  if (!kv4_supported(dim, group))
    return set_error(GRINQH_ERR_UNSUPPORTED, "head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim "
                     "(got %d, %d)", dim, group);
  GRINQH_REQUIRE(kv_heads > 0 && kv_heads <= 65535, "num_kv_heads must be in 1..65535 (got %d)", kv_heads);
  GRINQH_REQUIRE(page_size > 0 && page_size % kTile == 0, "page_size must be a positive multiple of 16 (got %d)",
                 page_size);
  GRINQH_REQUIRE(pages >= 0 && pages < (1LL << 31) && pages * (page_size / kTile) < (1LL << 31),
                 "num_pages is out of range (%lld)", (long long)pages);
  GRINQH_REQUIRE(pages == 0 || (cache && aligned(cache, 16)), "cache must be a 16-byte aligned device pointer");
  return GRINQH_OK;
}

}  // namespace grinqh
