// Attention of a sequence's last tokens over the 4-bit KV cache.
#include "kv4.cuh"

namespace grinqh {
namespace {

constexpr int kMaxRows = 32;  // new tokens x query heads of a kv head

struct Kv4AttnArgs {
  const void* q;
  int64_t q_seq, q_token, q_head;  // strides in elements
  const uint8_t* cache;
  const int32_t* tables;
  const int32_t* lens;
  void* out;
  float* lse;
  int64_t table_stride;
  int64_t pages;
  int seqs, new_tokens, heads, kv_heads, group;  // group: query heads of a kv head
  int page_tiles;
  int64_t max_len;
  float scale_log2;  // softmax scale * log2(e)
};

constexpr float kLn2 = 0.69314718055994531f;

// One warp per row (new token, query head), online softmax, token by token.
template <typename T, int D, int GS>
__global__ void __launch_bounds__(128) kv4_attention_kernel(const Kv4AttnArgs a) {
  using L = Kv4<D, GS>;
  constexpr int C = D / 32;  // channels of a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, b = blockIdx.y;
  const int len = (int)max((int64_t)0, min((int64_t)a.lens[b], a.max_len));
  const int d0 = lane * C;
  for (int r = warp; r < a.new_tokens * a.group; r += 4) {
    const int j = r / a.group, head = h * a.group + r % a.group;
    const T* q = static_cast<const T*>(a.q) + b * a.q_seq + j * a.q_token + head * a.q_head;
    float qv[C], o[C];
    for (int c = 0; c < C; ++c) {
      qv[c] = Act<T>::to_f(q[d0 + c]) * a.scale_log2;
      o[c] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int seen = len - a.new_tokens + j + 1;
    for (int t = 0; t < seen; ++t) {
      const int tile = t / kTile, token = t % kTile;
      const int page = a.tables[b * a.table_stride + tile / a.page_tiles];
      if (page < 0 || page >= a.pages) continue;
      const uint8_t* rec =
          a.cache + (((int64_t)page * a.kv_heads + h) * a.page_tiles + tile % a.page_tiles) * L::kRecord;
      const uint32_t kw = reinterpret_cast<const uint32_t*>(rec + token * (D / 2))[L::k_word(d0 & ~7)];
      const T* kp = reinterpret_cast<const T*>(rec + L::kKParams) + 2 * (token * L::NG + d0 / GS);
      float s = 0.f;
      for (int c = 0; c < C; ++c)
        s = fmaf(qv[c], fmaf((float)((kw >> (4 * ((d0 & 7) + c))) & 15u), Act<T>::to_f(kp[0]), Act<T>::to_f(kp[1])), s);
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float mn = fmaxf(m, s);
      const float f = exp2f(m - mn), p = exp2f(s - mn);
      m = mn;
      l = l * f + p;
      const uint32_t vw =
          reinterpret_cast<const uint32_t*>(rec + L::kV + (token / 2) * D)[L::v_word(token / 2, d0 & ~3)] >>
          (16 * (token & 1));
      const T* vp = reinterpret_cast<const T*>(rec + L::kVParams) + 2 * (token * L::NG + d0 / GS);
      for (int c = 0; c < C; ++c)
        o[c] = o[c] * f + p * fmaf((float)((vw >> (4 * ((d0 & 3) + c))) & 15u), Act<T>::to_f(vp[0]), Act<T>::to_f(vp[1]));
    }
    const int64_t row = ((int64_t)b * a.new_tokens + j) * a.heads + head;
    for (int c = 0; c < C; ++c) static_cast<T*>(a.out)[row * D + d0 + c] = Act<T>::from_f(l > 0.f ? o[c] / l : 0.f);
    if (lane == 0) a.lse[row] = l > 0.f ? m * kLn2 + logf(l) : -INFINITY;
  }
}

}  // namespace
}  // namespace grinqh

using namespace grinqh;

extern "C" size_t grinqh_kv4_attention_workspace_size(int64_t num_seqs, int new_tokens, int num_heads,
                                                      int num_kv_heads, int head_dim) {
  return 0;
}

extern "C" int grinqh_kv4_attention(const void* q, int dtype, int64_t num_seqs, int new_tokens, int num_heads,
                                    int num_kv_heads, int head_dim, int group_size, int64_t q_seq_stride,
                                    int64_t q_token_stride, int64_t q_head_stride, const uint8_t* cache,
                                    int64_t num_pages, int page_size, const int32_t* block_tables,
                                    int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                                    float softmax_scale, void* out, float* lse, void* workspace,
                                    size_t workspace_bytes, int flags, grinqh_stream_t stream) {
  GRINQH_RETURN_IF(check_device());
  GRINQH_REQUIRE(dtype == GRINQH_BF16 || dtype == GRINQH_F16, "dtype must be GRINQH_BF16 or GRINQH_F16");
  GRINQH_RETURN_IF(kv4_check_cache(cache, num_pages, page_size, num_kv_heads, head_dim, group_size));
  GRINQH_REQUIRE(num_heads > 0 && num_heads % num_kv_heads == 0,
                 "num_heads must be a positive multiple of num_kv_heads (got %d, %d)", num_heads, num_kv_heads);
  GRINQH_REQUIRE(new_tokens > 0, "new_tokens must be positive (got %d)", new_tokens);
  if ((int64_t)new_tokens * (num_heads / num_kv_heads) > kMaxRows)
    return set_error(GRINQH_ERR_UNSUPPORTED, "new_tokens x query heads per kv head must be at most %d (got %d x %d)",
                     kMaxRows, new_tokens, num_heads / num_kv_heads);
  GRINQH_REQUIRE(num_seqs >= 0 && num_seqs <= 65535, "num_seqs out of range (%lld)", (long long)num_seqs);
  GRINQH_REQUIRE(table_width >= 0 && table_width * page_size < (1LL << 31) && (num_seqs <= 1 || table_stride >= 0),
                 "block_tables out of range");
  GRINQH_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "softmax_scale must be positive and finite");
  if (num_seqs == 0) return GRINQH_OK;
  GRINQH_REQUIRE(q && seq_lens && out && lse && (block_tables || table_width == 0), "null pointer");
  GRINQH_REQUIRE(aligned(q, 16) && q_seq_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                     aligned(out, 16),
                 "q, its strides and out must be 16-byte aligned");
  const Kv4AttnArgs a{q, q_seq_stride, q_token_stride, q_head_stride, cache, block_tables, seq_lens, out, lse,
                      table_stride, num_pages, (int)num_seqs, new_tokens, num_heads, num_kv_heads,
                      num_heads / num_kv_heads, page_size / kTile, table_width * page_size,
                      softmax_scale * 1.4426950408889634f};
  return kv4_dispatch(head_dim, group_size, [&](auto layout) {
    using L = decltype(layout);
    const dim3 grid((unsigned)num_kv_heads, (unsigned)num_seqs);
    if (dtype == GRINQH_BF16)
      kv4_attention_kernel<__nv_bfloat16, L::kDim, L::kGroup><<<grid, 128, 0, stream>>>(a);
    else
      kv4_attention_kernel<__half, L::kDim, L::kGroup><<<grid, 128, 0, stream>>>(a);
    return check_launch("kv4_attention");
  });
}
