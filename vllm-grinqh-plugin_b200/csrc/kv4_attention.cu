// Attention of a sequence's last tokens over the 4-bit KV cache.
//
//   s_t = c q . k_t, p = softmax(s) over the tokens a query sees, out = sum_t p_t v_t
//   k_t = scale u + zero per group of channels, v_t likewise, u the 4-bit codes
//
// Bound by HBM: D + 8 NG bytes per token and kv head, against 4 D flops per query head.
// What has to be fast besides the loads is taking the codes apart, so nothing is ever
// dequantized: the products are made with the codes and corrected afterwards,
//   q . k_t   = sum_g scale_tg (q_g . u_tg) + zero_tg (sum of q_g)
//   sum p v_t = sum_t (p_t scale_tg) u_t  +  sum_t p_t zero_tg
// and a code is used as the f16 number with its bits: code u in the low bits is the
// subnormal u 2^-24, in bits 4..7 it is 16 u 2^-24, both exact as operands of the matrix
// instruction. An AND makes two operand values, and one shift serves eight codes. The
// factor 16 is taken out of q (exact), or of the output's channel; 2^24 of the results.
//
// mma.sync, with the roles that waste least on few query rows: rows of the instruction
// are tokens (scores) or channels (output), its 8 columns are query rows, new tokens x
// heads of the group. tcgen05 would need the codes expanded in shared memory first: 4
// times the bytes written and read there for an instruction of at least 64 rows.
//
// Work is cut evenly: the records (16 tokens) of all sequences and kv heads are numbered
// in a row, a CTA takes a run of them and its warps take turns. A warp streams its
// records through its own ring of bulk copies, across the borders of sequences. Where a
// sequence and head ends in a CTA, the warps' sums are joined in shared memory; where it
// is shared by several CTAs, each writes its sums to the workspace and the last one to
// arrive joins them in order.
#include "kv4.cuh"
#include "kv4_attention.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace grinqh {
namespace {

constexpr int kMaxRows = 32;  // new tokens x query heads of a kv head
constexpr float kSlack = 8.0f;       // weights may reach 2^kSlack before the running maximum follows
constexpr float kTopWeight = 64.0f;  // weights x V scales stay below this x 2^kSlack, in f16's range
constexpr float kLn2 = 0.69314718055994531f;
constexpr uint32_t kFull = 0xffffffffu;

struct Kv4AttnArgs {
  const void* q;
  int64_t q_seq, q_token, q_head;  // strides in elements
  const uint8_t* cache;
  const int32_t* tables;
  const int32_t* lens;
  void* out;
  float* lse;
  float* slots;       // [CTA][2][rows]{m, l, O[D]}: sums of a shared sequence and head
  unsigned* tickets;  // [CTA]: arrivals for the one that begins in this CTA and goes on
  int64_t table_stride;
  int64_t pages;
  int seqs, fresh, heads, kv_heads, group;  // fresh: new tokens; group: query heads of a kv head
  int page_tiles;
  int max_len;
  float scale_log2;  // softmax scale * log2(e)
};

template <int D, int GS, int NT>
struct Plan {
  static constexpr int kRows = 8 * NT;
  static constexpr int kWarps = NT == 1 ? 8 : 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kCtas = 2;  // per SM
  // as many as let two CTAs share an SM's 228 KB
  static constexpr int kStages = D == 64 ? 6 : (Kv4<D, GS>::NG == 4 || NT == 4 ? 3 : 4);
  static constexpr int kRow = D + 4;  // floats of a row in the join buffer
  static constexpr int kJoin = kRows * kRow + 2 * kRows;  // of a warp: O, m, l
  static constexpr int kQWords = NT == 4 ? NT * (D / 16) * 2 * 32 : 0;  // q operands in shared memory
  static constexpr uint32_t kRing = kWarps * kStages * Kv4<D, GS>::kRecord;
  static constexpr uint32_t kSmem = kRing + kWarps * kJoin * 4 + kWarps * kStages * 8 + kQWords * 4 + 128;
};

__device__ __forceinline__ int tiles_of(const Kv4AttnArgs& a, int b) {
  return (min(max(a.lens[b], 0), a.max_len) + kTile - 1) / kTile;
}

// A record's place in the numbering: sequence, kv head, tile of the sequence's nt tiles.
struct Pos {
  int b, h, t, nt;
};

// `step` records on; the record must exist.
__device__ __forceinline__ void advance(const Kv4AttnArgs& a, Pos& p, int step) {
  p.t += step;
  while (p.t >= p.nt) {
    p.t -= p.nt;
    if (++p.h == a.kv_heads) {
      p.h = 0;
      do {
        ++p.b;
        p.nt = tiles_of(a, p.b);
      } while (p.nt == 0);
    }
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (Act<T>::kBf16)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^(e - exponent of x), x > 0, as far as it is a normal number
__device__ __forceinline__ float power_for(float x, int e) {
  const int ex = (int)(__float_as_uint(x) >> 23) - 127;
  return __uint_as_float((uint32_t)(min(max(e - ex, -126), 127) + 127) << 23);
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <typename T, int D, int GS, int NT>
__global__ void __launch_bounds__(Plan<D, GS, NT>::kThreads, Plan<D, GS, NT>::kCtas)
    kv4_attention_kernel(const Kv4AttnArgs a) {
  using L = Kv4<D, GS>;
  using P = Plan<D, GS, NT>;
  constexpr int NG = L::NG, W = L::kWords, NW = P::kWarps, ST = P::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  float* s_join = reinterpret_cast<float*>(smem + P::kRing);
  uint32_t* s_q = reinterpret_cast<uint32_t*>(s_join + NW * P::kJoin);
  uint64_t* s_bars = reinterpret_cast<uint64_t*>(s_q + P::kQWords);
  int* s_start = reinterpret_cast<int*>(s_bars + NW * ST);  // [0..3] Pos, [4] per CTA, [5] total, [6] last to arrive

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rows = a.fresh * a.group;
  uint64_t* bars = s_bars + warp * ST;
  unsigned char* ring = smem + warp * ST * L::kRecord;
  if (lane == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&bars[s], 1);
    fence_mbar_init();
  }

  // ---------------------------------------------------------------- this CTA's run
  if (warp == 0) {
    int total = 0, most = 0;
    for (int b = lane; b < a.seqs; b += 32) {
      const int n = tiles_of(a, b);
      total += n;
      most = max(most, n);
    }
    total = __reduce_add_sync(kFull, total) * a.kv_heads;
    most = __reduce_max_sync(kFull, most);
    // Even shares, but no smaller than 4 records a warp: below that a CTA more saves
    // less than joining its sums costs. Few records: shares that end where the longest
    // sequence does.
    constexpr int kLeast = 4 * NW;
    int per = (total + gridDim.x - 1) / gridDim.x;
    if (per < kLeast && most > 0) {
      const int parts = (most + kLeast - 1) / kLeast;
      per = max(per, (most + parts - 1) / parts);
    }
    const int first = (int)blockIdx.x * per;
    Pos p{0, 0, 0, 0};
    if (first < total) {
      int before = 0;
      for (int b0 = 0;; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < a.seqs ? tiles_of(a, b) * a.kv_heads : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int x = __shfl_up_sync(kFull, upto, o);
          if (lane >= o) upto += x;
        }
        const unsigned hit = __ballot_sync(kFull, first < before + upto);
        if (hit) {
          const int src = __ffs(hit) - 1;
          const int inside = first - before - __shfl_sync(kFull, upto - n, src);
          p.b = b0 + src;
          p.nt = __shfl_sync(kFull, n, src) / a.kv_heads;
          p.h = inside / p.nt;
          p.t = inside % p.nt;
          break;
        }
        before += __shfl_sync(kFull, upto, 31);
      }
    }
    if (lane == 0) {
      s_start[0] = p.b;
      s_start[1] = p.h;
      s_start[2] = p.t;
      s_start[3] = p.nt;
      s_start[4] = per;
      s_start[5] = total;
    }
  } else {
    // queries of sequences without tokens
    for (int b = blockIdx.x; b < a.seqs; b += gridDim.x) {
      if (tiles_of(a, b) > 0) continue;
      const int64_t at = (int64_t)b * a.fresh * a.heads;
      for (int64_t i = threadIdx.x - 32; i < (int64_t)a.fresh * a.heads * (D / 8); i += P::kThreads - 32)
        reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      for (int i = threadIdx.x - 32; i < a.fresh * a.heads; i += P::kThreads - 32) a.lse[at + i] = -INFINITY;
    }
  }
  __syncthreads();
  Pos seg{s_start[0], s_start[1], s_start[2], s_start[3]};
  const int per = s_start[4], total = s_start[5];
  const int begin = min((int)blockIdx.x * per, total), end = min(begin + per, total);
  if (begin >= end) return;

  // ---------------------------------------------------------------- the warp's loads
  // Record `at` of the numbering is next to be loaded, into ring stage `put`; its page
  // was read one record ahead.
  int at = begin + warp, put = 0;
  Pos ld = seg;
  uint32_t skipped = 0;  // bit per stage: page outside the cache, nothing was loaded
  int page = 0;
  auto next_page = [&](int step) {  // to record `at`
    if (at >= end) return;
    advance(a, ld, step);
    page = a.tables[ld.b * a.table_stride + ld.t / a.page_tiles];
  };
  auto load = [&] {
    if (at >= end) return;
    const bool ok = page >= 0 && page < a.pages;
    if (lane == 0) {
      if (ok) {
        const uint8_t* rec =
            a.cache + (((int64_t)page * a.kv_heads + ld.h) * a.page_tiles + ld.t % a.page_tiles) * L::kRecord;
        mbar_arrive_expect_tx(&bars[put], L::kRecord);
        bulk_g2s(ring + put * L::kRecord, rec, L::kRecord, &bars[put]);
      } else {
        mbar_arrive(&bars[put]);
      }
    }
    skipped = (skipped & ~(1u << put)) | ((ok ? 0u : 1u) << put);
    put = put + 1 == ST ? 0 : put + 1;
    at += NW;
    next_page(NW);
  };
  next_page(warp);
  for (int s = 0; s < ST; ++s) load();

  int get = 0, index = begin + warp, phase = 0;  // consuming: stage, record, parity
  // ---------------------------------------------------------------- segment by segment
  for (int pos = begin; pos < end;) {
    const int left = min(seg.nt - seg.t, end - pos);  // records of this sequence and head in the run
    const int len = min(max(a.lens[seg.b], 0), a.max_len);
    const int see = len - a.fresh + 1;  // tokens that the first new token sees; token j sees j more

    // q as operand B: column g of tile nt is query row 8 nt + g; this lane's channels are
    // those of chunk t of a K row. f16 with the row's largest value near 2^13, so that the
    // fourth of them that is divided by 16 keeps its bits; below 2^-22 of the largest they
    // are rounded, which moves no score by more than 2^-24 of its largest term.
    uint32_t qf[NT == 4 ? 1 : NT][D / 16][2];
    float fac[NT][2], qsum[NT][2][NG];  // by this lane's columns 2 t, 2 t + 1 of the results
    int seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + g;
      float x[W][8];
      float top = 0.f, sum[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) sum[i] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int gi = w / L::kGroupWords, j = w % L::kGroupWords;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows)
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + seg.b * a.q_seq + (r / a.group) * a.q_token +
                                              (int64_t)(seg.h * a.group + r % a.group) * a.q_head + gi * GS +
                                              t * (GS / 4) + 8 * j);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(u[e]);
          x[w][2 * e] = f.x;
          x[w][2 * e + 1] = f.y;
          sum[gi] += f.x + f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
      const float up = top > 0.f ? power_for(top, 13) : 1.0f;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        sum[i] += __shfl_xor_sync(kFull, sum[i], 1);
        sum[i] += __shfl_xor_sync(kFull, sum[i], 2);
      }
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // two steps of 16 channels per word
          const uint32_t b0 = half2_bits(x[w][2 * k] * up, x[w][2 * k + 4] * up);
          const uint32_t b1 = half2_bits(x[w][2 * k + 1] * (up * 0.0625f), x[w][2 * k + 5] * (up * 0.0625f));
          if constexpr (NT == 4) {
            // every warp writes the same values
            uint2* to = reinterpret_cast<uint2*>(s_q) + ((n * (D / 16) + 2 * w + k) * 32 + lane);
            if (warp == 0) *to = make_uint2(b0, b1);
          } else {
            qf[n][2 * w + k][0] = b0;
            qf[n][2 * w + k][1] = b1;
          }
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int src = 4 * (2 * t + c);
        fac[n][c] = (1.0f / __shfl_sync(kFull, up, src)) * a.scale_log2 * 16777216.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) qsum[n][c][i] = __shfl_sync(kFull, sum[i], src) * a.scale_log2;
        seen[n][c] = see + min((8 * n + 2 * t + c) / a.group, a.fresh - 1);
      }
    }
    if constexpr (NT == 4) __syncthreads();

    float m[NT][2], ref[NT][2], l[NT][2], z[NT][2][NG];
    float o[2 * W][NT][4];
    float vf = 0x1p100f, back = 0x1p-100f;  // weights enter the product as p scale vf; back = 1 / vf
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = -INFINITY;
        ref[n][c] = 0.f;
        l[n][c] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) z[n][c][i] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 2 * W; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[k][n][c] = 0.f;
    }

    // ------------------------------------------------------------ this warp's records
    for (; index < pos + left; index += NW) {
      const int tile = seg.t + (index - pos);
      mbar_wait_nocall(&bars[get], phase);
      const uint8_t* rec = ring + get * L::kRecord;
      const bool skip = (skipped >> get) & 1u;
      if (!skip) {
        // scores: tokens g and g + 8 of the record, columns 2 t and 2 t + 1
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[n][c] = 0.f;
        {
          uint32_t ka[W], kb[W], pa[NG], pb[NG];
          load_words(rec + g * (D / 2) + t * (D / 8), ka);
          load_words(rec + (g + 8) * (D / 2) + t * (D / 8), kb);
          load_words(rec + L::kKParams + g * (4 * NG), pa);
          load_words(rec + L::kKParams + (g + 8) * (4 * NG), pb);
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
#pragma unroll
            for (int j = 0; j < L::kGroupWords; ++j) {
              const int w = gi * L::kGroupWords + j;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint32_t x = ka[w] >> (8 * k), y = kb[w] >> (8 * k);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  uint32_t b0, b1;
                  if constexpr (NT == 4) {
                    const uint2 v = reinterpret_cast<const uint2*>(s_q)[(n * (D / 16) + 2 * w + k) * 32 + lane];
                    b0 = v.x, b1 = v.y;
                  } else {
                    b0 = qf[n][2 * w + k][0], b1 = qf[n][2 * w + k][1];
                  }
                  mma_m16n8k16(acc[n], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, b0, b1);
                }
              }
            }
            const float2 qa = unpack2<T>(pa[gi]), qb = unpack2<T>(pb[gi]);  // scale, zero
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                s[n][c] = fmaf(qa.x * acc[n][c], fac[n][c], fmaf(qa.y, qsum[n][c][gi], s[n][c]));
                s[n][2 + c] = fmaf(qb.x * acc[n][2 + c], fac[n][c], fmaf(qb.y, qsum[n][c][gi], s[n][2 + c]));
              }
          }
        }
        const bool partly = (tile + 1) * kTile > see;  // some row does not see some token
        if (partly) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (tile * kTile + g >= seen[n][c]) s[n][c] = -INFINITY;
              if (tile * kTile + g + 8 >= seen[n][c]) s[n][2 + c] = -INFINITY;
            }
        }
        uint32_t pa[NG], pb[NG];
        load_words(rec + L::kVParams + g * (4 * NG), pa);
        load_words(rec + L::kVParams + (g + 8) * (4 * NG), pb);
        float sa[NG], sb[NG], za[NG], zb[NG];
        float wide = 0.f;
        bool grow = false;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const float2 x = unpack2<T>(pa[i]), y = unpack2<T>(pb[i]);
          sa[i] = x.x, za[i] = x.y, sb[i] = y.x, zb[i] = y.y;
          if (partly) {  // what lies behind the sequence may be anything
            if (tile * kTile + g >= len) sa[i] = za[i] = 0.f;
            if (tile * kTile + g + 8 >= len) sb[i] = zb[i] = 0.f;
          }
          wide = fmaxf(wide, fmaxf(sa[i], sb[i]));
        }
        grow = wide * vf > kTopWeight;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) grow = grow || fmaxf(s[n][c], s[n][2 + c]) > m[n][c] + kSlack;
        if (__any_sync(kFull, grow)) {
#pragma unroll
          for (int x = 4; x < 32; x *= 2) wide = fmaxf(wide, __shfl_xor_sync(kFull, wide, x));
          float turn = 1.0f;
          if (wide * vf > kTopWeight) {
            const float fresh = power_for(wide, 5);
            turn = fresh * back;
            vf = fresh;
            back = 1.0f / fresh;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float top = fmaxf(s[n][c], s[n][2 + c]);
#pragma unroll
              for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, x));
              float f = 1.0f;
              if (top > m[n][c] + kSlack) {
                f = exp2_fast(m[n][c] - top);
                m[n][c] = ref[n][c] = top;
              }
              l[n][c] *= f;
#pragma unroll
              for (int i = 0; i < NG; ++i) z[n][c][i] *= f;
#pragma unroll
              for (int k = 0; k < 2 * W; ++k) {
                o[k][n][c] *= f * turn;
                o[k][n][2 + c] *= f * turn;
              }
            }
        }
        // weights, and weights x scale as operand B of the output's product. What that loses
        // by its 11 bits is given back for a code of 7.5, the middle of the range: the
        // codes lie around it, so the error left is that of v's spread and not of its offset.
        uint32_t pf[NT][NG][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = exp2_fast(s[n][c] - ref[n][c & 1]);
          l[n][0] += p[0] + p[2];
          l[n][1] += p[1] + p[3];
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            float x[4] = {p[0] * (sa[i] * vf), p[1] * (sa[i] * vf), p[2] * (sb[i] * vf), p[3] * (sb[i] * vf)};
            float y[4] = {p[0] * za[i], p[1] * za[i], p[2] * zb[i], p[3] * zb[i]};
            if (partly) {  // a token that this row does not see may hold NaN
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (s[n][c] == -INFINITY) x[c] = y[c] = 0.f;
            }
            const uint32_t ha = half2_bits(x[0], x[1]), hb = half2_bits(x[2], x[3]);
            const float2 ra = __half22float2(*reinterpret_cast<const __half2*>(&ha));
            const float2 rb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
            z[n][0][i] += (y[0] + y[2]) + ((x[0] - ra.x) + (x[2] - rb.x)) * (7.5f * back);
            z[n][1][i] += (y[1] + y[3]) + ((x[1] - ra.y) + (x[3] - rb.y)) * (7.5f * back);
            pf[n][i][0] = transpose_8x8(ha);
            pf[n][i][1] = transpose_8x8(hb);
          }
        }
        uint32_t va[W], vb[W];
        load_words(rec + L::kV + t * D + ((g ^ (2 * t)) * W) * 4, va);
        load_words(rec + L::kV + (t + 4) * D + ((g ^ (2 * t)) * W) * 4, vb);
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t x = va[w] >> (8 * k), y = vb[w] >> (8 * k);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_m16n8k16(o[2 * w + k][n], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u,
                           pf[n][w / L::kGroupWords][0], pf[n][w / L::kGroupWords][1]);
          }
      }
      __syncwarp();
      load();
      if (++get == ST) {
        get = 0;
        phase ^= 1;
      }
    }

    // ------------------------------------------------------------ join the warps' sums
    float* mine = s_join + warp * P::kJoin;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * n + 2 * t + c;
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
          l[n][c] += __shfl_xor_sync(kFull, l[n][c], x);
#pragma unroll
          for (int i = 0; i < NG; ++i) z[n][c][i] += __shfl_xor_sync(kFull, z[n][c][i], x);
        }
        if (g == 0) {
          mine[P::kRows * P::kRow + r] = m[n][c];
          mine[P::kRows * P::kRow + P::kRows + r] = l[n][c];
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int gi = w / L::kGroupWords, j = w % L::kGroupWords;
          const float f = back * 16777216.0f;
          const float4 v = make_float4(fmaf(o[2 * w][n][c], f, z[n][c][gi]),
                                       fmaf(o[2 * w][n][2 + c], f * 0.0625f, z[n][c][gi]),
                                       fmaf(o[2 * w + 1][n][c], f, z[n][c][gi]),
                                       fmaf(o[2 * w + 1][n][2 + c], f * 0.0625f, z[n][c][gi]));
          *reinterpret_cast<float4*>(mine + r * P::kRow + gi * GS + g * (GS / 8) + 4 * j) = v;
        }
      }
    __syncthreads();
    const int seg_begin = pos - seg.t;              // the sequence and head in the numbering
    const int seg_end = seg_begin + seg.nt;
    const bool whole = seg.t == 0 && left == seg.nt;
    const int which = seg.t == 0 ? 1 : 0;           // slot: goes on in the next CTA, or came from the last
    float* slot = a.slots + ((int64_t)blockIdx.x * 2 + which) * P::kRows * (D + 2);
    // a thread takes 4 channels of a row
    auto finish = [&](int r, int d, float top, float sum, float4 v) {
      const int64_t row = ((int64_t)seg.b * a.fresh + r / a.group) * a.heads + seg.h * a.group + r % a.group;
      const bool none = sum == 0.f;
      const float inv = 1.0f / sum;
      T* out = static_cast<T*>(a.out) + row * D + d;
      const float x[4] = {v.x, v.y, v.z, v.w};
      T y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = Act<T>::from_f(none ? 0.f : x[i] * inv);
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
      if (d == 0) a.lse[row] = none ? -INFINITY : (top + log2f(sum)) * kLn2;
    };
    for (int i = threadIdx.x; i < rows * (D / 4); i += P::kThreads) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4));
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, s_join[w * P::kJoin + P::kRows * P::kRow + r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* from = s_join + w * P::kJoin;
        const float mw = from[P::kRows * P::kRow + r];
        const float lw = from[P::kRows * P::kRow + P::kRows + r];
        if (lw == 0.f) continue;  // this warp saw nothing (a NaN sum counts)
        const float f = exp2_fast(mw - top);
        const float4 x = *reinterpret_cast<const float4*>(from + r * P::kRow + d);
        sum = fmaf(lw, f, sum);
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
      }
      if (whole) {
        finish(r, d, top, sum, v);
      } else {
        __stcg(reinterpret_cast<float4*>(slot + 2 * P::kRows + r * D + d), v);
        if (d == 0) __stcg(reinterpret_cast<float2*>(slot + 2 * r), make_float2(top, sum));
      }
    }
    if (!whole) {
      const int c0 = seg_begin / per, c1 = (seg_end - 1) / per;  // the CTAs that share it
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const bool last = atomicAdd(&a.tickets[c0], 1u) == (unsigned)(c1 - c0);
        if (last) a.tickets[c0] = 0u;  // ready for the next launch
        __threadfence();
        s_start[6] = last;
      }
      __syncthreads();
      if (s_start[6]) {
        for (int i = threadIdx.x; i < rows * (D / 4); i += P::kThreads) {
          const int r = i / (D / 4), d = 4 * (i % (D / 4));
          auto part = [&](int c) {
            return a.slots + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * P::kRows * (D + 2);
          };
          float top = -INFINITY, sum = 0.f;
          for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(part(c) + 2 * r));
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c = c0; c <= c1; ++c) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(c) + 2 * r));
            if (ml.y == 0.f) continue;
            const float f = exp2_fast(ml.x - top);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part(c) + 2 * P::kRows + r * D + d));
            sum = fmaf(ml.y, f, sum);
            v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
          }
          finish(r, d, top, sum, v);
        }
      }
    }
    pos += left;
    if (pos < end) {
      advance(a, seg, left);
      __syncthreads();  // the join buffer is free again
    }
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  return sms;
}

constexpr int kCtasPerSm = 2;
constexpr size_t kTicketRegion = 16 << 10;  // where the linears keep theirs: all zero between calls
static_assert(kTicketRegion >= 4 * 2 * 1024, "a ticket per CTA");

int row_tiles(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

template <typename T, int D, int GS, int NT>
int launch(const Kv4AttnArgs& a, int sms, cudaStream_t st) {
  using P = Plan<D, GS, NT>;
  static_assert(P::kCtas == kCtasPerSm, "grid");
  auto kern = kv4_attention_kernel<T, D, GS, NT>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kSmem);
  if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  kern<<<(unsigned)(P::kCtas * sms), P::kThreads, P::kSmem, st>>>(a);
  return check_launch("kv4_attention");
}

}  // namespace

unsigned take_kv4_timeouts() {
  unsigned v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_wait_timeouts, sizeof(v)) != cudaSuccess) return 0;
  cudaMemcpyToSymbol(g_wait_timeouts, &z, sizeof(z));
  return v;
}

}  // namespace grinqh

using namespace grinqh;

extern "C" size_t grinqh_kv4_attention_workspace_size(int64_t num_seqs, int new_tokens, int num_heads,
                                                      int num_kv_heads, int head_dim) {
  if (num_seqs <= 0 || num_kv_heads <= 0) return 0;
  const int rows = 8 * row_tiles((int64_t)new_tokens * (num_heads / num_kv_heads));
  return kTicketRegion + (size_t)kCtasPerSm * sm_count() * 2 * rows * (head_dim + 2) * sizeof(float);
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
  GRINQH_REQUIRE(num_seqs >= 0 && num_seqs < (1LL << 31), "num_seqs out of range (%lld)", (long long)num_seqs);
  GRINQH_REQUIRE(table_width >= 0 && table_width * page_size < (1LL << 31) - 64 && (num_seqs <= 1 || table_stride >= 0),
                 "block_tables out of range");
  GRINQH_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "softmax_scale must be positive and finite");
  GRINQH_REQUIRE((double)num_seqs * num_kv_heads * (double)table_width * (page_size / kTile) < 2147000000.0,
                 "num_seqs x num_kv_heads x table_width x page_size / 16 must be below 2147000000");
  if (num_seqs == 0) return GRINQH_OK;
  GRINQH_REQUIRE(q && seq_lens && out && lse && (block_tables || table_width == 0), "null pointer");
  GRINQH_REQUIRE(aligned(q, 16) && q_seq_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                     aligned(out, 16),
                 "q, its strides and out must be 16-byte aligned");
  const size_t need =
      grinqh_kv4_attention_workspace_size(num_seqs, new_tokens, num_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return set_error(GRINQH_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, workspace_bytes);
  GRINQH_REQUIRE(aligned(workspace, 256), "workspace must be 256-byte aligned");
  const int sms = sm_count();
  Kv4AttnArgs a{};
  a.q = q;
  a.q_seq = q_seq_stride;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.cache = cache;
  a.tables = block_tables;
  a.lens = seq_lens;
  a.out = out;
  a.lse = lse;
  a.tickets = static_cast<unsigned*>(workspace);
  a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketRegion);
  a.table_stride = table_stride;
  a.pages = num_pages;
  a.seqs = (int)num_seqs;
  a.fresh = new_tokens;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.page_tiles = page_size / kTile;
  a.max_len = (int)(table_width * page_size);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  if (!(flags & GRINQH_WORKSPACE_ZEROED)) {
    const cudaError_t e = cudaMemsetAsync(workspace, 0, (size_t)kCtasPerSm * sms * sizeof(unsigned), stream);
    if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
  }
  const int tiles = row_tiles((int64_t)new_tokens * a.group);
  return kv4_dispatch(head_dim, group_size, [&](auto layout) {
    using L = decltype(layout);
    auto with = [&](auto type) {
      using T = decltype(type);
      if (tiles == 1) return launch<T, L::kDim, L::kGroup, 1>(a, sms, stream);
      if (tiles == 2) return launch<T, L::kDim, L::kGroup, 2>(a, sms, stream);
      return launch<T, L::kDim, L::kGroup, 4>(a, sms, stream);
    };
    return dtype == GRINQH_BF16 ? with(__nv_bfloat16{}) : with(__half{});
  });
}
