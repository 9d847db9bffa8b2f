// Writing tokens to the 4-bit KV cache and reading them back.
//
// Per token, head and group of GS channels, in fp32 from the model's type T:
//   zero = min x, scale = T((max x - min x) / 15), code = clamp(rint((x - zero) / scale), 0, 15)
//   value = T(scale * code + zero)
// zero is a value of x, so it is exact in T; the codes are made from the rounded scale,
// so its rounding costs at most 15 * 2^-9 of a step at the group's largest value. The
// quotient is a product with 1 / scale: a code can differ from the quotient's only where
// x lies midway between two codes, to fp32 precision.
//
// Bound by HBM: 4 D bytes of K and V in the model's type and D + 8 NG of the cache, per
// token and kv head. Measured with 8 kv heads: append of 16383 tokens, D = 128, group 128,
// 49 us, 53% of the copy bandwidth; gather of 70001, D = 64, group 32, 41 us, 71%. 64
// tokens, 13 us, and 1500 read back, 8 us, are the call on the host.
#include "kv4.cuh"

#include <algorithm>

namespace grinqh {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 2;  // tokens that a thread of the gather takes

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_f(type v) { return __bfloat1622float2(v); }
};
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 to_f(type v) { return __half22float2(v); }
};

struct CacheArgs {
  uint8_t* cache;
  const int64_t* slots;
  int64_t tokens;
  int64_t capacity;  // places in the cache
  int kv_heads;
  uint32_t page_tiles;
};

// Record of a place for head h; the place must lie in the cache.
template <int RECORD>
__device__ __forceinline__ int64_t record_at(const CacheArgs& a, int64_t slot, int h) {
  const uint32_t tile = (uint32_t)(slot >> 4);
  const uint32_t page = tile / a.page_tiles;
  return (((int64_t)page * a.kv_heads + h) * a.page_tiles + (tile - page * a.page_tiles)) * RECORD;
}

// Quantizes this lane's 8 channels of a group that GS / 8 neighbouring lanes share:
// returns the 8 codes at bits 4 e and the group's {scale, zero}.
template <typename T, int GS>
__device__ __forceinline__ uint32_t quantize8(const uint4& raw, uint32_t& params) {
  using T2 = typename Pair<T>::type;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  T2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const T2*>(&w[i]);
  // the NaN-keeping forms: a group that holds a NaN reads back as NaN
  T2 lo = __hmin2_nan(__hmin2_nan(x[0], x[1]), __hmin2_nan(x[2], x[3]));
  T2 hi = __hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3]));
#pragma unroll
  for (int o = 1; o < GS / 8; o *= 2) {
    lo = __hmin2_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = __hmax2_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const T zero = __hmin_nan(lo.x, lo.y), top = __hmax_nan(hi.x, hi.y);
  const float z = Act<T>::to_f(zero);
  float step = (Act<T>::to_f(top) - z) / 15.0f;
  step += step - step;  // an infinite one becomes NaN: so does every value of the group
  const T scale_t = Act<T>::from_f(step);
  const float scale = Act<T>::to_f(scale_t);
  const float inv = scale >= 1.17549435e-38f ? 1.0f / scale : 0.0f;  // a smaller scale's inverse overflows
  T2 both;
  both.x = scale_t;
  both.y = zero;
  params = *reinterpret_cast<uint32_t*>(&both);
  // x >= zero, so a code is rint(min(q, 15)): rounded by adding 1.5 2^23 and collected as
  // the digits of a number to base 16, four at a time, which fp32 holds exactly. (One
  // conversion to an integer per code would take the special function units 16 x 8 cycles
  // a warp.) A NaN becomes 15.
  constexpr float kRound = 12582912.0f;
  float digits[2] = {kRound, kRound};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Pair<T>::to_f(x[i]);
    const float a = fminf((f.x - z) * inv, 15.0f), b = fminf((f.y - z) * inv, 15.0f);
    digits[i / 2] = fmaf((a + kRound) - kRound, i % 2 ? 256.0f : 1.0f, digits[i / 2]);
    digits[i / 2] = fmaf((b + kRound) - kRound, i % 2 ? 4096.0f : 16.0f, digits[i / 2]);
  }
  return __byte_perm(__float_as_uint(digits[0]), __float_as_uint(digits[1]), 0x5410u);
}

// One lane per 8 channels of a token and head (blockIdx.y); the lanes of tokens 2 p and
// 2 p + 1 are neighbours, so that the pair's V words are written whole where both tokens lie in one
// pair row of the cache (else each token writes its 16-bit halves).
template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads) append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                          int64_t k_token, int64_t k_head, int64_t v_token,
                                                          int64_t v_head, CacheArgs a) {
  using L = Kv4<D, GS>;
  constexpr int kLanes = D / 8;
  const int l = threadIdx.x % kLanes, odd = threadIdx.x / kLanes & 1, h = blockIdx.y;
  const int64_t i = 2 * ((int64_t)blockIdx.x * (kThreads / (2 * kLanes)) + threadIdx.x / (2 * kLanes)) + odd;
  const bool in = i < a.tokens;
  int64_t slot = in ? a.slots[i] : -1;
  if (slot < 0 || slot >= a.capacity) slot = -1;
  const uint4 zero4 = make_uint4(0u, 0u, 0u, 0u);
  // (not waiting for the slot)
  const uint4 kr = in ? *reinterpret_cast<const uint4*>(k + i * k_token + h * k_head + 8 * l) : zero4;
  const uint4 vr = in ? *reinterpret_cast<const uint4*>(v + i * v_token + h * v_head + 8 * l) : zero4;
  uint32_t kp, vp;
  const uint32_t kc = quantize8<T, GS>(kr, kp);
  const uint32_t vc = quantize8<T, GS>(vr, vp);
  // the other token of the pair
  const uint32_t vo = __shfl_xor_sync(0xffffffffu, vc, kLanes);
  const int64_t so = __shfl_xor_sync(0xffffffffu, slot, kLanes);
  if (slot < 0) return;
  const int d = 8 * l, token = (int)(slot & 15);
  uint8_t* rec = a.cache + record_at<L::kRecord>(a, slot, h);
  reinterpret_cast<uint32_t*>(rec + token * (D / 2))[L::k_word(d)] = kc;
  uint8_t* vrow = rec + L::kV + (token >> 1) * D;
  const int w0 = L::v_word(token >> 1, d), w1 = L::v_word(token >> 1, d + 4);
  if (so == (slot ^ 1) && (token & 1) == odd) {
    // lanes of the even token write the words of channels d .. d + 3, those of the odd
    // token the words of d + 4 .. d + 7
    reinterpret_cast<uint32_t*>(vrow)[odd ? w1 : w0] = odd ? ((vo >> 16) | (vc & 0xffff0000u))
                                                           : ((vc & 0xffffu) | (vo << 16));
  } else {
    reinterpret_cast<uint16_t*>(vrow)[2 * w0 + (token & 1)] = (uint16_t)vc;
    reinterpret_cast<uint16_t*>(vrow)[2 * w1 + (token & 1)] = (uint16_t)(vc >> 16);
  }
  if (d % GS == 0) {
    reinterpret_cast<uint32_t*>(rec + L::kKParams)[token * L::NG + d / GS] = kp;
    reinterpret_cast<uint32_t*>(rec + L::kVParams)[token * L::NG + d / GS] = vp;
  }
}

template <typename T>
__device__ __forceinline__ uint4 values8(uint32_t codes, uint32_t params) {
  using T2 = typename Pair<T>::type;
  const float2 p = Pair<T>::to_f(*reinterpret_cast<const T2*>(&params));
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T2 r;
    r.x = Act<T>::from_f(fmaf((float)((codes >> (8 * i)) & 15u), p.x, p.y));
    r.y = Act<T>::from_f(fmaf((float)((codes >> (8 * i + 4)) & 15u), p.x, p.y));
    o[i] = *reinterpret_cast<uint32_t*>(&r);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// One lane per 8 channels of a token and head (blockIdx.y), the lanes of tokens 2 p and
// 2 p + 1 side by side: where they are a pair in the cache too, both read the same words of
// V. A thread takes kUnits pairs of tokens, for more loads in flight behind the slots'.
template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads) gather_kernel(CacheArgs a, T* __restrict__ k, T* __restrict__ v) {
  using L = Kv4<D, GS>;
  constexpr int kLanes = D / 8;
  constexpr int kPairs = kThreads / (2 * kLanes);  // of a block at a time
  const int d = 8 * (threadIdx.x % kLanes), h = blockIdx.y;
  const int64_t first = 2 * ((int64_t)blockIdx.x * kUnits * kPairs + threadIdx.x / (2 * kLanes)) +
                        (threadIdx.x / kLanes & 1);
  int64_t slot[kUnits];
  uint32_t kc[kUnits], v0[kUnits], v1[kUnits], kp[kUnits], vp[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t i = first + 2 * kPairs * u;
    slot[u] = i < a.tokens ? a.slots[i] : -1;
    if (slot[u] >= a.capacity) slot[u] = -1;
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    kc[u] = v0[u] = v1[u] = kp[u] = vp[u] = 0u;
    if (slot[u] < 0) continue;
    const int token = (int)(slot[u] & 15), pair = token >> 1;
    const uint8_t* rec = a.cache + record_at<L::kRecord>(a, slot[u], h);
    kc[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + token * (D / 2)) + L::k_word(d));
    v0[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + L::kV + pair * D) + L::v_word(pair, d));
    v1[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + L::kV + pair * D) + L::v_word(pair, d + 4));
    kp[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + L::kKParams) + token * L::NG + d / GS);
    vp[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + L::kVParams) + token * L::NG + d / GS);
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t i = first + 2 * kPairs * u;
    if (i >= a.tokens) continue;
    const int64_t at = (i * a.kv_heads + h) * D + d;
    const uint32_t vc = __byte_perm(v0[u], v1[u], slot[u] & 1 ? 0x7632u : 0x5410u);
    __stcs(reinterpret_cast<uint4*>(k + at), values8<T>(kc[u], kp[u]));
    __stcs(reinterpret_cast<uint4*>(v + at), values8<T>(vc, vp[u]));
  }
}

}  // namespace
}  // namespace grinqh

using namespace grinqh;

extern "C" int64_t grinqh_kv4_record_bytes(int head_dim, int group_size) { return kv4_record(head_dim, group_size); }

extern "C" int grinqh_kv4_append(const void* k, const void* v, int dtype, int64_t tokens, int num_kv_heads,
                                 int head_dim, int group_size, int64_t k_token_stride, int64_t k_head_stride,
                                 int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots, uint8_t* cache,
                                 int64_t num_pages, int page_size, grinqh_stream_t stream) {
  GRINQH_RETURN_IF(check_device());
  GRINQH_REQUIRE(dtype == GRINQH_BF16 || dtype == GRINQH_F16, "dtype must be GRINQH_BF16 or GRINQH_F16");
  GRINQH_RETURN_IF(kv4_check_cache(cache, num_pages, page_size, num_kv_heads, head_dim, group_size));
  GRINQH_REQUIRE(tokens >= 0 && tokens < (1LL << 31), "tokens out of range (%lld)", (long long)tokens);
  if (tokens == 0) return GRINQH_OK;
  GRINQH_REQUIRE(k && v && slots, "null pointer");
  GRINQH_REQUIRE(aligned(k, 16) && aligned(v, 16) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                     v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                 "k, v and their strides must be 16-byte aligned");
  const CacheArgs a{cache, slots, tokens, num_pages * page_size, num_kv_heads, (uint32_t)(page_size / kTile)};
  const int pairs = kThreads / (2 * (head_dim / 8));  // of a block
  const int64_t blocks = ((tokens + 1) / 2 + pairs - 1) / pairs;
  const dim3 grid((unsigned)blocks, (unsigned)num_kv_heads);
  return kv4_dispatch(head_dim, group_size, [&](auto layout) {
    using L = decltype(layout);
    if (dtype == GRINQH_BF16)
      append_kernel<__nv_bfloat16, L::kDim, L::kGroup><<<grid, kThreads, 0, stream>>>(
          static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), k_token_stride, k_head_stride,
          v_token_stride, v_head_stride, a);
    else
      append_kernel<__half, L::kDim, L::kGroup><<<grid, kThreads, 0, stream>>>(
          static_cast<const __half*>(k), static_cast<const __half*>(v), k_token_stride, k_head_stride, v_token_stride,
          v_head_stride, a);
    return check_launch("kv4_append");
  });
}

extern "C" int grinqh_kv4_gather(const uint8_t* cache, int dtype, int64_t num_pages, int page_size, int num_kv_heads,
                                 int head_dim, int group_size, const int64_t* slots, int64_t tokens, void* k, void* v,
                                 grinqh_stream_t stream) {
  GRINQH_RETURN_IF(check_device());
  GRINQH_REQUIRE(dtype == GRINQH_BF16 || dtype == GRINQH_F16, "dtype must be GRINQH_BF16 or GRINQH_F16");
  GRINQH_RETURN_IF(kv4_check_cache(cache, num_pages, page_size, num_kv_heads, head_dim, group_size));
  GRINQH_REQUIRE(tokens >= 0 && tokens < (1LL << 31), "tokens out of range (%lld)", (long long)tokens);
  if (tokens == 0) return GRINQH_OK;
  GRINQH_REQUIRE(k && v && slots, "null pointer");
  GRINQH_REQUIRE(aligned(k, 16) && aligned(v, 16), "k and v must be 16-byte aligned");
  const CacheArgs a{const_cast<uint8_t*>(cache), slots,        tokens,
                    num_pages * page_size,       num_kv_heads, (uint32_t)(page_size / kTile)};
  const int pairs = kUnits * (kThreads / (2 * (head_dim / 8)));  // of a block
  const int64_t blocks = ((tokens + 1) / 2 + pairs - 1) / pairs;
  const dim3 grid((unsigned)blocks, (unsigned)num_kv_heads);
  return kv4_dispatch(head_dim, group_size, [&](auto layout) {
    using L = decltype(layout);
    if (dtype == GRINQH_BF16)
      gather_kernel<__nv_bfloat16, L::kDim, L::kGroup><<<grid, kThreads, 0, stream>>>(
          a, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v));
    else
      gather_kernel<__half, L::kDim, L::kGroup><<<grid, kThreads, 0, stream>>>(a, static_cast<__half*>(k),
                                                                             static_cast<__half*>(v));
    return check_launch("kv4_gather");
  });
}
