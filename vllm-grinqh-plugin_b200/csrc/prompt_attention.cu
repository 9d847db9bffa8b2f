// Causal attention over packed prompts with grouped heads.
#include "common.cuh"

namespace grinqh {
namespace {

struct PromptArgs {
  const void *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int64_t total_q, total_k;
  int seqs, heads, group;  // group: query heads of a kv head
  float scale_log2;        // softmax scale * log2(e)
};

constexpr float kLn2 = 0.69314718055994531f;

// One warp per query row and head, online softmax, key by key.
template <typename T, int D>
__global__ void __launch_bounds__(128) prompt_attention_kernel(const PromptArgs a) {
  constexpr int C = D / 32;  // channels of a lane
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int head = blockIdx.y;
  if (row >= a.total_q) return;
  int b = 0;
  while (b < a.seqs && row >= a.cu_q[b + 1]) ++b;
  if (b == a.seqs || row < a.cu_q[b]) return;
  const int64_t k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  const int64_t seen = min(min(k1, a.total_k), k1 - (a.cu_q[b + 1] - row) + 1);
  const T* q = static_cast<const T*>(a.q) + row * a.q_token + head * a.q_head + lane * C;
  float qv[C], o[C];
  for (int c = 0; c < C; ++c) {
    qv[c] = Act<T>::to_f(q[c]) * a.scale_log2;
    o[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t t = max(k0, (int64_t)0); t < seen; ++t) {
    const T* k = static_cast<const T*>(a.k) + t * a.k_token + (head / a.group) * a.k_head + lane * C;
    const T* v = static_cast<const T*>(a.v) + t * a.v_token + (head / a.group) * a.v_head + lane * C;
    float s = 0.f;
    for (int c = 0; c < C; ++c) s = fmaf(qv[c], Act<T>::to_f(k[c]), s);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float f = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * f + p;
    for (int c = 0; c < C; ++c) o[c] = o[c] * f + p * Act<T>::to_f(v[c]);
  }
  const int64_t at = row * a.heads + head;
  for (int c = 0; c < C; ++c)
    static_cast<T*>(a.out)[at * D + lane * C + c] = Act<T>::from_f(l > 0.f ? o[c] / l : 0.f);
  if (lane == 0) a.lse[at] = l > 0.f ? m * kLn2 + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace grinqh

using namespace grinqh;

extern "C" int grinqh_prompt_attention(const void* q, const void* k, const void* v, int dtype, int64_t total_q,
                                       int64_t total_k, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                       int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                       const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, float softmax_scale,
                                       void* out, float* lse, grinqh_stream_t stream) {
  GRINQH_RETURN_IF(check_device());
  GRINQH_REQUIRE(dtype == GRINQH_BF16 || dtype == GRINQH_F16, "dtype must be GRINQH_BF16 or GRINQH_F16");
  if (head_dim != 64 && head_dim != 128)
    return set_error(GRINQH_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
  GRINQH_REQUIRE(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0 && num_heads <= 65535,
                 "num_heads must be a positive multiple of num_kv_heads (got %d, %d)", num_heads, num_kv_heads);
  GRINQH_REQUIRE(total_q >= 0 && total_q < (1LL << 31) && total_k >= 0 && total_k < (1LL << 31) && num_seqs >= 0,
                 "token counts out of range");
  if (total_q == 0 || num_seqs == 0) return GRINQH_OK;
  GRINQH_REQUIRE(q && (total_k == 0 || (k && v)) && cu_seqlens_q && cu_seqlens_k && out && lse, "null pointer");
  GRINQH_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && q_token_stride % 8 == 0 &&
                     q_head_stride % 8 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                     v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                 "q, k, v, their strides and out must be 16-byte aligned");
  const PromptArgs a{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                     v_head_stride, cu_seqlens_q, cu_seqlens_k, out, lse, total_q, total_k, num_seqs, num_heads,
                     num_heads / num_kv_heads, softmax_scale * 1.4426950408889634f};
  const dim3 grid((unsigned)((total_q + 3) / 4), (unsigned)num_heads);
  auto run = [&](auto type) {
    using T = decltype(type);
    if (head_dim == 128)
      prompt_attention_kernel<T, 128><<<grid, 128, 0, stream>>>(a);
    else
      prompt_attention_kernel<T, 64><<<grid, 128, 0, stream>>>(a);
    return check_launch("prompt_attention");
  };
  return dtype == GRINQH_BF16 ? run(__nv_bfloat16{}) : run(__half{});
}
