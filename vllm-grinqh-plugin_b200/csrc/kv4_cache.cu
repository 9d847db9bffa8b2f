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
// What they cannot do without: 4 D bytes of K and V in the model's type and D + 8 NG of the
// cache, per token and kv head. Measured with 8 kv heads: 16383 tokens, D = 128, group 128,
// written 26.6 us, 3.2 TB/s, and written and read back 38.9 us, 67% of the copy bandwidth;
// 70001 tokens, D = 64, group 32, read back 40.6 us, 71%. 64 tokens written and read, 12.5 us,
// and 1500 read, 8 us, are the calls on the host. Writing is not bound by HBM: it reads its
// input once (67 MB) and its records stay in L2, with 66% of the issue slots in use, half of
// the warps and loads waited for. Reading 70001 back uses 68%, with 132 MB to and from HBM.
#include "kv4.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace grinqh {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 2;  // tokens that a thread of the gather takes

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_f(type v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ uint32_t pack(float2 f) {
    const type v = __float22bfloat162_rn(f);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 to_f(type v) { return __half22float2(v); }
  static __device__ __forceinline__ uint32_t pack(float2 f) {
    const type v = __float22half2_rn(f);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

struct CacheArgs {
  uint8_t* cache;
  const int64_t* slots;
  int64_t tokens;
  int64_t capacity;  // places in the cache
  int kv_heads;
  uint32_t page_tiles;
  uint32_t page_inv;  // (2^32 - 1) / page_tiles
};

// Record of a place for head h; the place must lie in the cache.
template <int RECORD>
__device__ __forceinline__ int64_t record_at(const CacheArgs& a, int64_t slot, int h) {
  const uint32_t tile = (uint32_t)(slot >> 4);
  // tile < 2^31, so the product with the inverse is the quotient or one less
  uint32_t page = __umulhi(tile, a.page_inv), at = tile - page * a.page_tiles;
  if (at >= a.page_tiles) ++page, at -= a.page_tiles;
  return (int64_t)((uint64_t)(page * (uint64_t)(uint32_t)a.kv_heads + h) * a.page_tiles + at) * RECORD;
}

// 1.5 2^23: an fp32 number u + kRound has the bits kRoundBits + u for a small integer u, and
// adding kRound rounds to one.
constexpr float kRound = 12582912.0f;
constexpr uint32_t kRoundBits = 0x4b400000u;

// Quantizes this lane's 16 channels of a group that GS / 16 neighbouring lanes share: the 8
// codes of a half at bits 4 e, and the group's {scale, zero}.
template <typename T, int GS>
__device__ __forceinline__ uint2 quantize16(const uint4& r0, const uint4& r1, uint32_t& params) {
  using T2 = typename Pair<T>::type;
  const uint32_t w[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
  T2 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const T2*>(&w[i]);
  // the NaN-keeping forms: a group that holds a NaN reads back as NaN
  T2 lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) lo = __hmin2_nan(lo, x[i]), hi = __hmax2_nan(hi, x[i]);
  hi = __hneg2(hi);
  T2 a, b;  // {min, -max}: one shuffle and one minimum a step
  a.x = lo.x, a.y = hi.x, b.x = lo.y, b.y = hi.y;
  a = __hmin2_nan(a, b);
#pragma unroll
  for (int o = 1; o < GS / 16; o *= 2) a = __hmin2_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const T zero = a.x;
  const float z = Act<T>::to_f(zero);
  float step = (-Act<T>::to_f(a.y) - z) / 15.0f;
  step += step - step;  // an infinite one becomes NaN: so does every value of the group
  const T scale_t = Act<T>::from_f(step);
  const float scale = Act<T>::to_f(scale_t);
  const float inv = scale >= 1.17549435e-38f ? 1.0f / scale : 0.0f;  // a smaller scale's inverse overflows
  T2 both;
  both.x = scale_t;
  both.y = zero;
  params = *reinterpret_cast<uint32_t*>(&both);
  // x >= zero, so a code is rint(min(q, 15)); its bits are added up as the digits of a number
  // to base 16, what kRoundBits adds is known. (A conversion to an integer per code would
  // take the special function units 8 cycles a warp each.) A NaN becomes 15.
  uint32_t digits[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t d = 0u - kRoundBits * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = mul2(add2(Pair<T>::to_f(x[4 * half + i]), make_float2(-z, -z)), make_float2(inv, inv));
      f.x = fminf(f.x, 15.0f), f.y = fminf(f.y, 15.0f);
      f = add2(f, make_float2(kRound, kRound));
      d += __float_as_uint(f.x) << (8 * i);
      d += __float_as_uint(f.y) << (8 * i + 4);
    }
    digits[half] = d;
  }
  return make_uint2(digits[0], digits[1]);
}

// Two words of a row of codes: side by side where a chunk has more than one of a group.
template <bool kTogether>
__device__ __forceinline__ void store2(uint8_t* row, int i, int j, uint32_t a, uint32_t b) {
  if constexpr (kTogether) {
    *reinterpret_cast<uint2*>(row + 4 * i) = make_uint2(a, b);
  } else {
    reinterpret_cast<uint32_t*>(row)[i] = a;
    reinterpret_cast<uint32_t*>(row)[j] = b;
  }
}

// One lane per 16 channels of a token and head (blockIdx.y). A group's and an address's
// instructions bound it at 8 channels a lane and one fp32 at a time: 16383 tokens x 8 heads,
// D = 128, 23.7 M warp instructions and 32.8 us, against 12.6 M and 26.6 us. The lanes of
// tokens 2 p and 2 p + 1 are neighbours, so that the pair's V words are written whole where
// both tokens lie in one pair row of the cache (else each token writes its 16-bit halves).
template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads) append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                          int64_t k_token, int64_t k_head, int64_t v_token,
                                                          int64_t v_head, CacheArgs a) {
  using L = Kv4<D, GS>;
  constexpr int kLanes = D / 16;
  const int l = threadIdx.x % kLanes, odd = threadIdx.x / kLanes & 1, h = blockIdx.y;
  const int64_t i = 2 * ((int64_t)blockIdx.x * (kThreads / (2 * kLanes)) + threadIdx.x / (2 * kLanes)) + odd;
  const bool in = i < a.tokens;
  int64_t slot = in ? a.slots[i] : -1;
  if (slot < 0 || slot >= a.capacity) slot = -1;
  uint4 kr[2], vr[2];
  kr[0] = kr[1] = vr[0] = vr[1] = make_uint4(0u, 0u, 0u, 0u);
  if (in) {  // (not waiting for the slot)
    const uint4* kp = reinterpret_cast<const uint4*>(k + i * k_token + h * k_head + 16 * l);
    const uint4* vp = reinterpret_cast<const uint4*>(v + i * v_token + h * v_head + 16 * l);
    kr[0] = kp[0], kr[1] = kp[1], vr[0] = vp[0], vr[1] = vp[1];
  }
  uint32_t kp, vp;
  const uint2 kc = quantize16<T, GS>(kr[0], kr[1], kp);
  const uint2 vc = quantize16<T, GS>(vr[0], vr[1], vp);
  // lanes of the pair's even token write the words of channels d .. d + 7, those of the odd
  // one the words of d + 8 .. d + 15: each gets the other's codes of its half
  const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? vc.x : vc.y, kLanes);
  const int64_t so = __shfl_xor_sync(0xffffffffu, slot, kLanes);
  if (slot < 0) return;
  const int d = 16 * l, token = (int)(slot & 15), pair = token >> 1;
  uint8_t* rec = a.cache + record_at<L::kRecord>(a, slot, h);
  store2<(GS > 32)>(rec + token * (D / 2), L::k_word(d), L::k_word(d + 8), kc.x, kc.y);
  uint8_t* vrow = rec + L::kV + pair * D;
  if (so == (slot ^ 1) && (token & 1) == odd) {
    const uint32_t first = odd ? other : vc.x, second = odd ? vc.y : other;
    const int at = d + 8 * odd;
    store2<(GS > 32)>(vrow, L::v_word(pair, at), L::v_word(pair, at + 4), __byte_perm(first, second, 0x5410u),
                      __byte_perm(first, second, 0x7632u));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      reinterpret_cast<uint16_t*>(vrow)[2 * L::v_word(pair, d + 4 * e) + (token & 1)] =
          (uint16_t)((e < 2 ? vc.x : vc.y) >> (16 * (e & 1)));
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
  const uint32_t even = codes & 0x0f0f0f0fu, odd = codes >> 4 & 0x0f0f0f0fu;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // u + kRound by its bits: an integer's conversion is the special function units'
    const float2 u = add2(make_float2(__uint_as_float(__byte_perm(even, kRoundBits, 0x7650u + i)),
                                      __uint_as_float(__byte_perm(odd, kRoundBits, 0x7650u + i))),
                          make_float2(-kRound, -kRound));
    o[i] = Pair<T>::pack(fma2(u, make_float2(p.x, p.x), make_float2(p.y, p.y)));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// One lane per 8 channels of a token and head (blockIdx.y), the lanes of tokens 2 p and
// 2 p + 1 side by side: where they are a pair in the cache too, both read the same words of
// V. A thread takes kUnits pairs of tokens, for more loads in flight behind the slots': 70001
// tokens, D = 64, 41.3 us with one, 40.8 with two, 40.9 with four. Nor do smaller blocks (40.7)
// or stores that stay in L2 (40.2) change much: three quarters of the bytes are writes.
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
  const CacheArgs a{cache, slots, tokens, num_pages * page_size, num_kv_heads, (uint32_t)(page_size / kTile),
                    0xffffffffu / (uint32_t)(page_size / kTile)};
  const int pairs = kThreads / (2 * (head_dim / 16));  // of a block
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
                    num_pages * page_size,       num_kv_heads, (uint32_t)(page_size / kTile),
                    0xffffffffu / (uint32_t)(page_size / kTile)};
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
