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
// in a row, and every warp takes a run of them, which streams through a ring of its own
// across the borders of sequences. One warp issues the bulk copies for all rings, a lane
// each: looking up pages would cost the computing warps a quarter more instructions and
// the registers that keep two records in flight. A sequence and head that lies in one
// run is finished by its warp; the sums of one that several warps share are joined in
// shared memory when the CTA's warps are done, and where it is shared by several CTAs,
// each writes its sums to the workspace and the last one to arrive joins them in order.
//
// Waits are bounded. A warp whose wait is lost leaves NaN sums, so that the rows which
// needed the record become NaN, and every CTA still arrives where it is waited for.
//
// Measured (bf16, D = 128, group 128, 32 / 8 heads): 5 sequences of 50001 to 131072 tokens,
// 111 us, 67% of the copy bandwidth (the loop runs at 90%; the rest is the ends, and the SMs
// whose loads take longer); 64 of 8192, 121 us, 72%; 64 of 512 to 768, group 64, 26 us, 28%;
// one of 301, 8 us, one after another: looking up pages, a record, joining. 33 of up to 9000
// with 4 new tokens (fp16, D = 64, group 32, 24 / 8 heads), 31.4 us: 12 query rows a record, in
// a kernel that spills (Plan), at 46% of the issue slots, and the same joins.
#include "kv4.cuh"
#include "kv4_attention.cuh"
#include "launch.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace grinqh {
namespace {

constexpr int kMaxRows = 32;  // new tokens x query heads of a kv head
constexpr float kSlack = 16.0f;  // a lane's weights of a step may sum to this before the maximum follows
constexpr int kTopScale = 10;    // V scales x vf stay below 2^(kTopScale + 1): weights x that within f16's range
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
  float* slots;       // [CTA][2]{m, l of the rows, O[rows][D]}: sums of a shared sequence and head
  float* sums;        // [CTA][warp]{O, m, l}: of a piece that began before the warp's run
  unsigned* tickets;  // [CTA]: arrivals for the one that begins in this CTA and goes on
  int64_t table_stride;
  int64_t pages;
  int seqs, fresh, heads, kv_heads, group;  // fresh: new tokens; group: query heads of a kv head
  int parts;                                // blocks of 8 NT query rows of a kv head, each reads the cache
  int page_tiles;
  int max_len;
  float scale_log2;  // softmax scale * log2(e)
  uint64_t wait_ns;  // the longest wait
};

template <int D, int GS, int NT>
struct Plan {
  static constexpr int kRows = 8 * NT;
  // Warps that compute, beside the one that loads: one CTA per SM, and 128 registers a
  // thread, or 255 where the sums of 16 rows x 128 channels take 128 of them. 15 rings of
  // D = 128, group 32 would not fit the shared memory, 14 do. Not all instances fit their
  // registers. Bytes of a thread's spilled stores: 16 rows, D = 64, 280 to 300 (group 32) and 100
  // (group 64); 8 rows, D = 128, 200 to 225 (group 32) and 20 to 30; the others up to 44.
  static constexpr int kWarps = NT == 2 && D == 128 ? 7 : (D == 128 && GS == 32 ? 14 : 15);
  static constexpr int kThreads = 32 * (kWarps + 1);
  // Stages of two records.
  static constexpr int kStages = D == 64 ? 5 : 3;
  static constexpr uint32_t kStage = 2 * Kv4<D, GS>::kRecord;
  static constexpr int kRow = D + 4;                     // floats of a row of sums
  static constexpr int kSums = kRows * kRow + 2 * kRows;  // O, m, l
  static constexpr uint32_t kWarpRing = kStages * kStage;
  static constexpr uint32_t kSmem = kWarps * kWarpRing;
  static_assert(kSums * 4 <= kWarpRing, "a run's last sums go where its ring was");
  static_assert(kSmem <= 225 * 1024, "shared memory");
};

// What a sequence and head costs beside its records, in records: q, finishing or joining.
// 33 sequences of up to 9000 tokens with 4 new ones, 8 kv heads: 38.2 us with 4, 31.4 with 8,
// 33.8 with 16; 64 of 512 to 768, 27.2, 26.0 and 26.5; long ones, 110.9, 111.2 and 111.8.
constexpr int kCost = 8;

__device__ __forceinline__ int tiles_of(const Kv4AttnArgs& a, int b) {
  return (min(max(a.lens[b], 0), a.max_len) + kTile - 1) / kTile;
}

// A place in the numbering: sequence, kv head (and part), place in their `stride` places,
// of which the first nt are records.
struct Pos {
  int b, h, at, nt, stride;
};

// `step` places on; the place must exist. same > 0: every stride is `same`.
__device__ __forceinline__ void advance(const Kv4AttnArgs& a, Pos& p, int step, int same) {
  p.at += step;
  while (p.at >= p.stride) {
    p.at -= p.stride;
    if (++p.h == a.kv_heads * a.parts) {
      p.h = 0;
      do {
        ++p.b;
        p.nt = tiles_of(a, p.b);
      } while (p.nt == 0);
      p.stride = same > 0 ? same : p.nt + kCost;
    }
  }
}

// What a warp leaves to join: a piece of a sequence and head that began before its run
// (kHead; kThrough if it also goes on behind it), and one that goes on behind it (kTail).
// The sums of the run's last piece are in the ring, those of a head before it in the
// workspace (kAway).
enum { kHead = 1, kThrough = 2, kTail = 4, kAway = 8 };
struct Piece {
  int b, h, first, nt;  // first: the place of its first record
};
struct Left {
  int flags;
  Piece head, tail;
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (Act<T>::kBf16)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename T>
__device__ __forceinline__ auto two(uint32_t w) {
  if constexpr (Act<T>::kBf16)
    return *reinterpret_cast<const __nv_bfloat162*>(&w);
  else
    return *reinterpret_cast<const __half2*>(&w);
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

// Adds sums l, y by the maximum m to those by `top`.
__device__ __forceinline__ void add_sums(float& top, float& sum, float4& v, float m, float l, float4 y) {
  const bool some = l != 0.f;  // (a NaN counts)
  const float now = some ? fmaxf(top, m) : top;
  const float f = now == -INFINITY ? 1.0f : exp2_fast(top - now), h = some ? exp2_fast(m - now) : 0.f;
  top = now;
  sum = fmaf(l, h, sum * f);
  v.x = some ? fmaf(y.x, h, v.x * f) : v.x;
  v.y = some ? fmaf(y.y, h, v.y * f) : v.y;
  v.z = some ? fmaf(y.z, h, v.z * f) : v.z;
  v.w = some ? fmaf(y.w, h, v.w * f) : v.w;
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
__global__ void __launch_bounds__(Plan<D, GS, NT>::kThreads, 1) kv4_attention_kernel(const Kv4AttnArgs a) {
  using L = Kv4<D, GS>;
  using P = Plan<D, GS, NT>;
  using T2 = decltype(two<T>(0u));
  constexpr int NG = L::NG, W = L::kWords, NW = P::kWarps, ST = P::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  float* heads_of = a.sums + (int64_t)blockIdx.x * NW * P::kSums;  // of the warps: pieces that began before
  __shared__ uint64_t s_full[NW][ST], s_empty[NW][ST];
  __shared__ uint32_t s_gone[NW][ST];  // bits: record of the stage that was not loaded
  __shared__ int s_pages[NW][64];
  __shared__ Pos s_start;
  __shared__ int s_plan[3];  // places of a run, the common stride (0: none), places in all
  __shared__ Left s_left[NW];
  __shared__ int s_last[2];
  __shared__ int s_lost;  // a wait of this CTA was lost

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int heads = a.kv_heads * a.parts;  // what is numbered within a sequence
  if (warp < NW && lane == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&s_full[warp][s], 1);
      mbar_init(&s_empty[warp][s], 1);
    }
    fence_mbar_init();
    s_left[warp].flags = 0;
  }

  if (threadIdx.x == 0) s_lost = lost_beforehand(a.wait_ns);

  // the next kernel's set-up may overlap this one, as this one's did its predecessor
  allow_dependent_grid();
  wait_prior_grid();

  // ---------------------------------------------------------------- the CTA's runs
  if (warp == NW) {
    int tiles = 0, most = 0, count = 0;
    for (int b = lane; b < a.seqs; b += 32) {
      const int n = tiles_of(a, b);
      tiles += n;
      most = max(most, n);
      count += n > 0;
    }
    tiles = __reduce_add_sync(kFull, tiles) * heads;
    most = __reduce_max_sync(kFull, most);
    count = __reduce_add_sync(kFull, count) * heads;
    // Even runs. Where a CTA for each sequence and head makes the runs of the longest at
    // most 2 records longer, that is taken: no sums pass between CTAs. Measured with 8 kv
    // heads, D = 128: 18 sequences of 300 tokens, 16.0 us with even runs and 12.3 so, 18 of
    // 4000, 32.8 and 28.7; 5 of 500 to 1500, 6 records longer, 16.2 and 18.4.
    const int workers = (int)gridDim.x * NW;
    int total = tiles + count * kCost;
    int per = max((total + workers - 1) / workers, 2), same = 0;
    const int alone = (most + NW - 1) / NW;
    if (count <= (int)gridDim.x && alone <= per + 2) {
      per = max(alone, 1);
      same = per * NW;
      total = count * same;
    }
    const int first = (int)blockIdx.x * NW * per;
    Pos p{0, 0, 0, 0, 1};
    if (first < total) {
      int before = 0;
      for (int b0 = 0;; b0 += 32) {
        const int b = b0 + lane;
        const int nt = b < a.seqs ? tiles_of(a, b) : 0;
        const int n = nt > 0 ? (same > 0 ? same : nt + kCost) * heads : 0;
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
          p.nt = __shfl_sync(kFull, nt, src);
          p.stride = same > 0 ? same : p.nt + kCost;
          p.h = inside / p.stride;
          p.at = inside % p.stride;
          break;
        }
        before += __shfl_sync(kFull, upto, 31);
      }
    }
    if (lane == 0) {
      s_start = p;
      s_plan[0] = per;
      s_plan[1] = same;
      s_plan[2] = total;
    }
  } else {
    // queries of sequences without tokens
    for (int b = blockIdx.x; b < a.seqs; b += gridDim.x) {
      if (tiles_of(a, b) > 0) continue;
      const int64_t at = (int64_t)b * a.fresh * a.heads;
      for (int64_t i = threadIdx.x; i < (int64_t)a.fresh * a.heads * (D / 8); i += 32 * NW)
        reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      for (int i = threadIdx.x; i < a.fresh * a.heads; i += 32 * NW) a.lse[at + i] = -INFINITY;
    }
  }
  __syncthreads();
  const int per = s_plan[0], same = s_plan[1], total = s_plan[2];
  if ((int)blockIdx.x * NW * per >= total) return;
  Pos seg = s_start;

  // One row of a finished sequence and head: 4 channels from d on.
  auto finish = [&](int b, int h, int r, int d, float top, float sum, float4 v) {
    const int j = a.fresh == 1 ? 0 : r / a.group;
    const int64_t row = ((int64_t)b * a.fresh + j) * a.heads + h * a.group + r - j * a.group;
    const bool none = sum == 0.f;
    const float inv = 1.0f / sum;
    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    T w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Act<T>::from_f(none ? 0.f : y[i]);
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * D + d) = *reinterpret_cast<const uint2*>(w);
    if (d == 0) a.lse[row] = none ? -INFINITY : (top + log2f(sum)) * kLn2;
  };

  if (warp == NW) {
    // -------------------------------------------------------------- loads: lane w for warp w
    // A stage takes the next two records of a sequence and head (the last of them alone may
    // be one): one copy where they lie in one page. Page numbers wait in shared memory, 64
    // per warp: the lanes' own loads would each wait for the one before to return, since
    // they write one register of the warp.
    int x = ((int)blockIdx.x * NW + lane) * per;
    const int end = lane < NW ? min(x + per, total) : x;
    int entry = 0, in_page = 0, filled = 0, last = 0;  // page and record in it; pages read, the last one
    auto enter = [&] {
      entry = seg.at / a.page_tiles;
      in_page = seg.at - entry * a.page_tiles;
      last = (seg.nt - 1) / a.page_tiles;
      filled = entry & ~31;
    };
    auto settle = [&] {  // to the next place that is a record
      while (x < end && seg.at >= seg.nt) {
        const int step = seg.stride - seg.at;
        x += step;
        if (x < end) advance(a, seg, step, same);
      }
      if (x < end) enter();
    };
    if (x < end) {
      advance(a, seg, lane * per, same);
      settle();
    }
    int put = 0;
    uint32_t phase = 1, idle = 0;  // the first round finds the stages empty
    uint64_t since = 0;
    while (__any_sync(kFull, x < end)) {
      for (uint32_t need; (need = __ballot_sync(kFull, x < end && filled <= min(entry + 8, last))) != 0u;) {
        // 32 page numbers for each of these warps, four loads in flight
        int got[4], who[4], base[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          who[k] = need ? __ffs(need) - 1 : -1;
          need &= need - 1u;
          const int w = max(who[k], 0);
          base[k] = __shfl_sync(kFull, filled, w) + lane;
          const int b = __shfl_sync(kFull, seg.b, w), to = __shfl_sync(kFull, last, w);
          got[k] = who[k] >= 0 ? a.tables[b * a.table_stride + min(base[k], to)] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (who[k] >= 0) s_pages[who[k]][base[k] & 63] = got[k];
          if (lane == who[k]) filled += 32;
        }
        __syncwarp();
      }
      const bool go = x < end && mbar_test(&s_empty[lane][put], phase);
      if (go) {
        const bool both = min(seg.nt - seg.at, end - x) >= 2, whole = both && in_page + 1 < a.page_tiles;
        const int page0 = s_pages[lane][entry & 63], page1 = s_pages[lane][(entry + 1) & 63];
        const bool ok0 = page0 >= 0 && page0 < a.pages;
        const bool ok1 = whole ? ok0 : both && page1 >= 0 && page1 < a.pages;
        const int h = seg.h / a.parts;
        const uint8_t* from =
            a.cache + (((int64_t)page0 * a.kv_heads + h) * a.page_tiles + in_page) * L::kRecord;
        unsigned char* to = smem + lane * P::kWarpRing + put * P::kStage;
        uint64_t* bar = &s_full[lane][put];
        s_gone[lane][put] = (ok0 ? 0u : 1u) | (ok1 ? 0u : 2u);
        const uint32_t bytes = (ok0 ? L::kRecord : 0) + (ok1 ? L::kRecord : 0);
        if (bytes > 0)
          mbar_arrive_expect_tx(bar, bytes);
        else
          mbar_arrive(bar);
        if (ok0) bulk_g2s(to, from, whole ? P::kStage : L::kRecord, bar);
        if (ok1 && !whole)
          bulk_g2s(to + L::kRecord, a.cache + ((int64_t)page1 * a.kv_heads + h) * a.page_tiles * L::kRecord, L::kRecord,
                   bar);
        const int n = both ? 2 : 1;
        x += n;
        seg.at += n;
        in_page += n;
        while (in_page >= a.page_tiles) {
          in_page -= a.page_tiles;
          ++entry;
        }
        if (seg.at >= seg.nt) settle();
        if (++put == ST) {
          put = 0;
          phase ^= 1u;
        }
      }
      if (__any_sync(kFull, go)) {
        idle = 0;
      } else {
        __nanosleep(20);
        if ((++idle & 63u) == 0u) {  // bounded, like every wait
          const uint64_t now = globaltimer_ns();
          if (idle == 64u) since = now;
          bool lost = *reinterpret_cast<volatile int*>(&s_lost) != 0;
          if (!lost && now - since >= a.wait_ns) {
            lost = true;
            if (atomicExch(&s_lost, 1) == 0) atomicAdd(&g_wait_timeouts, 1u);
          }
          if (__any_sync(kFull, lost)) break;
        }
      }
    }
    // the copies still in flight: of each stage the last, a round back behind `put`
    if (lane < NW) {
#pragma unroll 1
      for (int s = 0; s < ST; ++s)
        if (!mbar_drain(&s_full[lane][s], s < put ? phase ^ 1u : phase)) s_lost = 1;
    }
  } else {
    // -------------------------------------------------------------- a run, piece by piece
    int x = ((int)blockIdx.x * NW + warp) * per;  // places x .. end
    const int end = min(x + per, total);
    if (x < end) advance(a, seg, warp * per, same);
    unsigned char* ring = smem + warp * P::kWarpRing;
    const uint32_t k_at = g * (D / 2) + t * (D / 8), p_at = g * (4 * NG),
                   v_at = L::kV + t * D + (g ^ (2 * t)) * (4 * W);
    int get = 0;
    uint32_t phase = 0;
    bool lost = a.wait_ns == 0;  // a wait of this warp was: no record is used from there on
    while (x < end) {
      const int t0 = seg.at, t1 = min(seg.nt, seg.at + (end - x));  // this piece's records
      if (t0 < t1) {
        const int kv_head = seg.h / a.parts, row0 = (seg.h - kv_head * a.parts) * P::kRows;
        const int rows = min(a.fresh * a.group - row0, P::kRows);
        const int len = min(max(a.lens[seg.b], 0), a.max_len);
        const int see = len - a.fresh + 1 + (a.fresh == 1 ? 0 : row0 / a.group);  // tokens that the first row sees

        // q as operand B: column g of block n is query row 8 n + g; this lane's channels are
        // those of chunk t of a K row. f16 with the row's largest value near 2^13, so that the
        // half of them that is divided by 16 keeps its bits; below 2^-22 of the largest they
        // are rounded, which moves no score by more than 2^-24 of its largest term.
        const T* q = static_cast<const T*>(a.q) + seg.b * a.q_seq + t * (GS / 4);
        uint32_t raw[NT][W][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = row0 + 8 * n + g;
          const int j = a.fresh == 1 ? 0 : r / a.group;
          const T* from = q + j * a.q_token + (int64_t)(kv_head * a.group + r - j * a.group) * a.q_head;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (8 * n + g < rows)
              v = *reinterpret_cast<const uint4*>(from + w / L::kGroupWords * GS + w % L::kGroupWords * 8);
            raw[n][w][0] = v.x, raw[n][w][1] = v.y, raw[n][w][2] = v.z, raw[n][w][3] = v.w;
          }
        }
        uint32_t qf[NT][D / 16][2];
        float fac[NT][2], qsum[NT][2][NG];  // by this lane's columns 2 t, 2 t + 1 of the results
        int seen[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const T2 zero2 = two<T>(0u);
          T2 most = zero2;
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = __hmax2(most, __habs2(two<T>(raw[n][w][e])));
          float top = fmaxf(Act<T>::to_f(most.x), Act<T>::to_f(most.y));
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
          // (above 2^-103, for down; only rows of 2^116 and more come closer to f16's end)
          const float up = top > 0.f ? fmaxf(power_for(top, 13), 0x1p-103f) : 1.0f;
          float sum[NG];
#pragma unroll
          for (int i = 0; i < NG; ++i) sum[i] = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<T>(raw[n][w][e]);
              v[2 * e] = f.x, v[2 * e + 1] = f.y;
              sum[w / L::kGroupWords] += f.x + f.y;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // two steps of 16 channels per word
              qf[n][2 * w + k][0] = half2_bits(v[2 * k] * up, v[2 * k + 4] * up);
              qf[n][2 * w + k][1] = half2_bits(v[2 * k + 1] * (up * 0.0625f), v[2 * k + 5] * (up * 0.0625f));
            }
          }
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            sum[i] += __shfl_xor_sync(kFull, sum[i], 1);
            sum[i] += __shfl_xor_sync(kFull, sum[i], 2);
          }
          // 1 / up, and 2^24 for the codes' subnormals, by the exponent
          const float down = __uint_as_float((278u << 23) - __float_as_uint(up));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int src = 4 * (2 * t + c), r = row0 + 8 * n + 2 * t + c;
            fac[n][c] = __shfl_sync(kFull, down, src) * a.scale_log2;
#pragma unroll
            for (int i = 0; i < NG; ++i) qsum[n][c][i] = __shfl_sync(kFull, sum[i], src) * a.scale_log2;
            seen[n][c] = len - a.fresh + 1 + (a.fresh == 1 ? 0 : min(r / a.group, a.fresh - 1));
          }
        }

        float m[NT][2], ref[NT][2], l[NT][2], z[NT][2][NG];
        float o[2 * W][NT][4];
        // Weights enter the product as p scale vf; back = 1 / vf, scales stay below the limit.
        // vf follows the largest scale of the piece, so f16's smallest step is 2^-35 of that
        // one's weight 1: a scale 2^20 times smaller has its weights to 2^-16 of the largest. With
        // kSlack 1024 these were 2^-29 and 2^-10, for the same times; with 4, which would
        // leave 2^-37, the maximum follows too often (33 sequences with drafts, 31.4 us -> 32.5).
        float vf = 0x1p100f, back = 0x1p-100f, limit = (float)(2 << kTopScale) * back;
        bool first = true;
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

        const int clear = min(t1, see / kTile);  // records before this one are seen whole by all rows
#pragma unroll 1
        for (int tile = t0; tile < t1; tile += 2) {
          lost = lost || !__all_sync(kFull, mbar_wait_or_lose(&s_full[warp][get], phase, a.wait_ns, &s_lost));
          if (lost) break;
          const unsigned char* rec = ring + get * P::kStage;
          const uint32_t gone = s_gone[warp][get];
          const bool masked = tile + 2 > clear || gone != 0u;  // a row does not see a token, or there is none
          // scores: tokens g and g + 8 of a record, columns 2 t and 2 t + 1
          float s[2][NT][4];
          uint32_t ka[2][W], kb[2][W], pa[2][NG], pb[2][NG];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            load_words(rec + i * L::kRecord + k_at, ka[i]);
            load_words(rec + i * L::kRecord + 4 * D + k_at, kb[i]);
            load_words(rec + i * L::kRecord + L::kKParams + p_at, pa[i]);
            load_words(rec + i * L::kRecord + L::kKParams + 32 * NG + p_at, pb[i]);
          }
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            float acc[2][NT][4];
#pragma unroll
            for (int j = 0; j < L::kGroupWords; ++j) {
              const int w = gi * L::kGroupWords + j;
#pragma unroll
              for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t u = ka[i][w] >> (8 * q), v = kb[i][w] >> (8 * q);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    if (j == 0 && q == 0)
                      mma_m16n8k16_zero(acc[i][n], u & 0x000f000fu, v & 0x000f000fu, u & 0x00f000f0u, v & 0x00f000f0u,
                                        qf[n][2 * w + q][0], qf[n][2 * w + q][1]);
                    else
                      mma_m16n8k16(acc[i][n], u & 0x000f000fu, v & 0x000f000fu, u & 0x00f000f0u, v & 0x00f000f0u,
                                   qf[n][2 * w + q][0], qf[n][2 * w + q][1]);
                  }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 qa = unpack2<T>(pa[i][gi]), qb = unpack2<T>(pb[i][gi]);  // scale, zero
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float za = gi == 0 ? qa.y * qsum[n][c][gi] : fmaf(qa.y, qsum[n][c][gi], s[i][n][c]);
                  const float zb = gi == 0 ? qb.y * qsum[n][c][gi] : fmaf(qb.y, qsum[n][c][gi], s[i][n][2 + c]);
                  s[i][n][c] = fmaf(qa.x * acc[i][n][c], fac[n][c], za);
                  s[i][n][2 + c] = fmaf(qb.x * acc[i][n][2 + c], fac[n][c], zb);
                }
            }
          }
          // V's scales and zeros of the lane's tokens
          float sv[2][2][NG], zv[2][2][NG];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            load_words(rec + i * L::kRecord + L::kVParams + p_at, pa[i]);
            load_words(rec + i * L::kRecord + L::kVParams + 32 * NG + p_at, pb[i]);
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              const float2 u = unpack2<T>(pa[i][k]), v = unpack2<T>(pb[i][k]);
              sv[i][0][k] = u.x, zv[i][0][k] = u.y, sv[i][1][k] = v.x, zv[i][1][k] = v.y;
            }
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                const int at = (gone >> i) & 1u ? 0x7fffffff : (tile + i) * kTile + g + 8 * b;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int c = 0; c < 2; ++c)
                    if (at >= seen[n][c]) s[i][n][2 * b + c] = -INFINITY;
#pragma unroll
                for (int k = 0; k < NG; ++k)  // what lies behind the sequence may be anything
                  if (at >= len) sv[i][b][k] = zv[i][b][k] = 0.f;
              }
          }
          float wide = 0.f;
#pragma unroll
          for (int k = 0; k < NG; ++k)
            wide = fmaxf(fmaxf(wide, fmaxf(sv[0][0][k], sv[0][1][k])), fmaxf(sv[1][0][k], sv[1][1][k]));
          // Weights by the maximum so far. Where they sum to more than kSlack the maximum is
          // raised and they are made anew; `first` makes that so until every row has a maximum.
          float p[2][NT][4], add[NT][2];
#pragma unroll 1
          for (bool raised = false;; raised = true) {
            bool grow = first || wide > limit;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) p[i][n][c] = exp2_fast(s[i][n][c] - ref[n][c & 1]);
#pragma unroll
              for (int c = 0; c < 2; ++c) add[n][c] = (p[0][n][c] + p[0][n][2 + c]) + (p[1][n][c] + p[1][n][2 + c]);
              grow = grow || fmaxf(add[n][0], add[n][1]) > kSlack;
            }
            if (raised || !__any_sync(kFull, grow)) break;
#pragma unroll
            for (int k = 4; k < 32; k *= 2) wide = fmaxf(wide, __shfl_xor_sync(kFull, wide, k));
            float turn = 1.0f;
            if (wide > limit) {
              const float now = power_for(wide, kTopScale);
              turn = now * back;
              vf = now;
              back = 1.0f / now;
              limit = (float)(2 << kTopScale) * back;
            }
            bool unset = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float top = fmaxf(fmaxf(s[0][n][c], s[0][n][2 + c]), fmaxf(s[1][n][c], s[1][n][2 + c]));
#pragma unroll
                for (int k = 4; k < 32; k *= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, k));
                float f = 1.0f;
                if (top > m[n][c]) {
                  f = exp2_fast(m[n][c] - top);
                  m[n][c] = ref[n][c] = top;
                }
                unset = unset || m[n][c] == -INFINITY;
                l[n][c] *= f;
#pragma unroll
                for (int i = 0; i < NG; ++i) z[n][c][i] *= f;
#pragma unroll
                for (int k = 0; k < 2 * W; ++k) {
                  o[k][n][c] *= f * turn;
                  o[k][n][2 + c] *= f * turn;
                }
              }
            first = __any_sync(kFull, unset);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) l[n][c] += add[n][c];
          // weights x scale as operand B of the output's product
          uint32_t pf[2][NT][NG][2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float* w = p[i][n];
#pragma unroll
              for (int k = 0; k < NG; ++k) {
                const float sa = sv[i][0][k] * vf, sb = sv[i][1][k] * vf;
                float u[4] = {w[0] * sa, w[1] * sa, w[2] * sb, w[3] * sb};
                float y[4] = {w[0] * zv[i][0][k], w[1] * zv[i][0][k], w[2] * zv[i][1][k], w[3] * zv[i][1][k]};
                if (masked) {  // a token that this row does not see may hold NaN
#pragma unroll
                  for (int c = 0; c < 4; ++c)
                    if (s[i][n][c] == -INFINITY) u[c] = y[c] = 0.f;
                }
                const uint32_t ha = half2_bits(u[0], u[1]), hb = half2_bits(u[2], u[3]);
                z[n][0][k] += y[0] + y[2];
                z[n][1][k] += y[1] + y[3];
                if constexpr (!Act<T>::kBf16) {
                  // What the 11 bits lose is given back for a code of 7.5, the middle of the
                  // range, so that the error left is that of v's spread and not of its offset:
                  // fp16 outputs would show it (3.5e-4 relative without, 2.4e-4 with), bf16's
                  // own rounding (1.7e-3, with fp32 weights too) hides it, so bf16 goes without.
                  const float2 ra = __half22float2(*reinterpret_cast<const __half2*>(&ha));
                  const float2 rb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
                  z[n][0][k] = fmaf((u[0] - ra.x) + (u[2] - rb.x), 7.5f * back, z[n][0][k]);
                  z[n][1][k] = fmaf((u[1] - ra.y) + (u[3] - rb.y), 7.5f * back, z[n][1][k]);
                }
                pf[i][n][k][0] = transpose_8x8(ha);
                pf[i][n][k][1] = transpose_8x8(hb);
              }
            }
          }
          // The products of a step start from zero and are added to the sums here: the
          // instruction cuts its sums off instead of rounding them, and over a long sequence,
          // where the codes' sum and the zeros' all but cancel, that bias showed (1.6 % of
          // the output at 131072 tokens when the sums stayed in it and lo was the difference
          // of whole bytes and hi).
          uint32_t va[2][W], vb[2][W];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            load_words(rec + i * L::kRecord + v_at, va[i]);
            load_words(rec + i * L::kRecord + 4 * D + v_at, vb[i]);
          }
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float acc[4];
                const uint32_t u = va[0][w] >> (8 * k), y = vb[0][w] >> (8 * k);
                mma_m16n8k16_zero(acc, u & 0x000f000fu, u & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u,
                                  pf[0][n][w / L::kGroupWords][0], pf[0][n][w / L::kGroupWords][1]);
                const uint32_t u1 = va[1][w] >> (8 * k), y1 = vb[1][w] >> (8 * k);
                mma_m16n8k16(acc, u1 & 0x000f000fu, u1 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u,
                             pf[1][n][w / L::kGroupWords][0], pf[1][n][w / L::kGroupWords][1]);
#pragma unroll
                for (int c = 0; c < 4; ++c) o[2 * w + k][n][c] += acc[c];
              }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[warp][get]);
          if (++get == ST) {
            get = 0;
            phase ^= 1u;
          }
        }

        // ---------------------------------------------------------- the piece's sums
        const bool began = t0 > 0, goes = t1 < seg.nt;
        // the run's last piece leaves its sums where the ring was
        const bool last = x + (t1 - t0) >= end || (x + (seg.stride - seg.at) >= end);
        float* sums = last ? reinterpret_cast<float*>(ring) : heads_of + warp * P::kSums;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int r = 8 * n + 2 * t + c;
#pragma unroll
            for (int k = 4; k < 32; k *= 2) {
              l[n][c] += __shfl_xor_sync(kFull, l[n][c], k);
#pragma unroll
              for (int i = 0; i < NG; ++i) z[n][c][i] += __shfl_xor_sync(kFull, z[n][c][i], k);
            }
            if (lost) l[n][c] = __int_as_float(0x7fffffff);  // NaN: so is what the rows come to
            if ((began || goes) && g == 0) {
              sums[P::kRows * P::kRow + r] = m[n][c];
              sums[P::kRows * P::kRow + P::kRows + r] = l[n][c];
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const int gi = w / L::kGroupWords, j = w % L::kGroupWords;
              const int d = gi * GS + g * (GS / 8) + 4 * j;
              // in two steps: back x 2^24 may be more than fp32 holds
              const float4 v = make_float4(fmaf(o[2 * w][n][c] * back, 0x1p24f, z[n][c][gi]),
                                           fmaf(o[2 * w][n][2 + c] * back, 0x1p20f, z[n][c][gi]),
                                           fmaf(o[2 * w + 1][n][c] * back, 0x1p24f, z[n][c][gi]),
                                           fmaf(o[2 * w + 1][n][2 + c] * back, 0x1p20f, z[n][c][gi]));
              if (began || goes) {
                *reinterpret_cast<float4*>(sums + r * P::kRow + d) = v;
              } else if (r < rows) {
                finish(seg.b, kv_head, row0 + r, d, m[n][c], l[n][c], v);
              }
            }
          }
        if (lane == 0 && (began || goes)) {
          const Piece piece{seg.b, seg.h, x - seg.at, seg.nt};
          if (began) {
            s_left[warp].flags |= (goes ? kHead | kThrough : kHead) | (last ? 0 : kAway);
            s_left[warp].head = piece;
          } else {
            s_left[warp].flags |= kTail;
            s_left[warp].tail = piece;
          }
        }
      }
      const int step = min(seg.stride - seg.at, end - x);
      x += step;
      if (x < end) advance(a, seg, step, same);
    }
  }

  // ---------------------------------------------------------------- join what warps share
  __syncthreads();
  // Chain 0 is the piece that came from the CTA before, chain 1 + w the one that warp w
  // leaves open; a chain takes the heads of the warps behind it while they go through.
  // A thread takes 4 channels of a row of a chain.
  const int all = a.fresh * a.group;
  const bool lost = s_lost != 0;
  // four warps a chain, as many chains at a time as there are such; the rest of 15 have none
  constexpr int kGroups = (NW + 1) / 4;
  const bool is = lane <= NW && (s_left[max(lane - 1, 0)].flags & (lane == 0 ? kHead : kTail));
  uint32_t chains = __ballot_sync(kFull, is && warp < 4 * kGroups);
  for (int k = warp / 4; k > 0; --k) chains &= chains - 1u;
#pragma unroll 1
  while (chains != 0u) {
    const int chain = __ffs(chains) - 1;
    for (int k = 0; k < kGroups; ++k) chains &= chains - 1u;
    const Left& first = s_left[max(chain - 1, 0)];
    const Piece piece = chain == 0 ? first.head : first.tail;
    const int kv_head = piece.h / a.parts, row0 = (piece.h - kv_head * a.parts) * P::kRows;
    const int w0 = max(chain - 1, 0);
    // the chain's last warp: the first behind it whose head does not go through
    const int flags = lane < NW ? s_left[lane].flags : 0;
    const uint32_t closed = __ballot_sync(kFull, !(flags & kThrough)) & ~((1u << w0) | ((1u << w0) - 1u));
    const bool through = chain > 0 || (first.flags & kThrough);
    const int stop = through ? __ffs(closed) - 1 : w0;
    const bool open = through && stop >= NW;
    const int w1 = min(stop, NW - 1);
    const uint32_t away = __ballot_sync(kFull, flags & kAway);
    for (int i = threadIdx.x & 127; i < min(all - row0, P::kRows) * (D / 4); i += 128) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4));
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](const float* from) {
        add_sums(top, sum, v, from[P::kRows * P::kRow + r], from[P::kRows * P::kRow + P::kRows + r],
                 *reinterpret_cast<const float4*>(from + r * P::kRow + d));
      };
#pragma unroll 4
      for (int w = w0; w <= w1; ++w) {
        if (w >= chain && (away >> w & 1u))
          add(heads_of + w * P::kSums);
        else
          add(reinterpret_cast<const float*>(smem + w * P::kWarpRing));
      }
      // a copy may have come to a ring after the sums: none of this CTA's count
      if (lost) sum = __int_as_float(0x7fffffff);
      if (chain > 0 && !open) {
        finish(piece.b, kv_head, row0 + r, d, top, sum, v);
      } else {
        float* slot = a.slots + ((int64_t)blockIdx.x * 2 + (chain > 0)) * P::kRows * (D + 2);
        __stcg(reinterpret_cast<float4*>(slot + 2 * P::kRows + r * D + d), v);
        if (d == 0) __stcg(reinterpret_cast<float2*>(slot + 2 * r), make_float2(top, sum));
      }
    }
  }
  // The sequences and heads that other CTAs share: the one that came from the CTA before,
  // and the one that goes on into the next. One that does both is the first of these.
  bool after = false;
  int from = 0;
  for (int w = 0; w < NW; ++w) {
    if (s_left[w].flags & kTail)
      after = true, from = w;
    else if (!(s_left[w].flags & kThrough))
      after = false;
  }
  const bool before = s_left[0].flags & kHead;
  if (!before && !after) return;
  __syncthreads();  // the slots are written; the fence below covers them for the whole CTA
  if (threadIdx.x < 2) {
    const bool mine = threadIdx.x == 0 ? before : after;
    bool last = false;
    if (mine) {
      const Piece p = threadIdx.x == 0 ? s_left[0].head : s_left[from].tail;
      const int c0 = p.first / per / NW, c1 = (p.first + p.nt - 1) / per / NW;
      __threadfence();
      last = atomicAdd(&a.tickets[c0], 1u) == (unsigned)(c1 - c0);
      if (last) a.tickets[c0] = 0u;  // ready for the next launch
      __threadfence();
    }
    s_last[threadIdx.x] = last;
  }
  __syncthreads();
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (!s_last[which]) continue;
    const Piece p = which == 0 ? s_left[0].head : s_left[from].tail;
    const int c0 = p.first / per / NW, c1 = (p.first + p.nt - 1) / per / NW;
    const int kv_head = p.h / a.parts, row0 = (p.h - kv_head * a.parts) * P::kRows;
    for (int i = threadIdx.x; i < min(all - row0, P::kRows) * (D / 4); i += P::kThreads) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4));
      // the slots of four CTAs at a time, for the loads' latency
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = c0; c <= c1; c += 4) {
        float2 ml[4];
        float4 y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* from = a.slots + ((int64_t)min(c + k, c1) * 2 + (c + k == c0 ? 1 : 0)) * P::kRows * (D + 2);
          ml[k] = __ldcg(reinterpret_cast<const float2*>(from + 2 * r));
          y[k] = __ldcg(reinterpret_cast<const float4*>(from + 2 * P::kRows + r * D + d));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c + k <= c1) add_sums(top, sum, v, ml[k].x, ml[k].y, y[k]);
        }
      }
      finish(p.b, kv_head, row0 + r, d, top, sum, v);
    }
  }
}

constexpr size_t kTicketRegion = 16 << 10;  // where the linears keep theirs: all zero between calls
static_assert(kTicketRegion >= 4 * 1024, "a ticket per CTA, one CTA per SM");

int row_tiles(int64_t rows) { return rows <= 8 ? 1 : 2; }  // blocks of 8 query rows of a warp

template <typename T, int D, int GS, int NT>
int launch(const Kv4AttnArgs& a, int sms, cudaStream_t st) {
  using P = Plan<D, GS, NT>;
  auto kern = kv4_attention_kernel<T, D, GS, NT>;
  static std::atomic<uint64_t> ready{0};
  GRINQH_RETURN_IF(allow_smem(reinterpret_cast<const void*>(kern), ready, P::kSmem));
  return launch_dependent(kern, dim3((unsigned)sms), P::kThreads, P::kSmem, st, "kv4_attention", a);
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
  if (num_seqs <= 0 || new_tokens <= 0 || num_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  const int rows = 8 * row_tiles((int64_t)new_tokens * (num_heads / num_kv_heads));
  const size_t warps = rows == 16 && head_dim == 128 ? 7 : 15;
  return kTicketRegion + (size_t)sm_count() * (2 * rows * (head_dim + 2) + warps * rows * (head_dim + 6)) * sizeof(float);
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
  GRINQH_REQUIRE(2.0 * (double)num_seqs * num_kv_heads * ((double)table_width * (page_size / kTile) + kCost) < 2147000000.0,
                 "num_seqs x num_kv_heads x (table_width x page_size / 16 + 8) must be below 1073000000");
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
  const int tiles = row_tiles((int64_t)new_tokens * (num_heads / num_kv_heads));
  a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketRegion);
  a.sums = a.slots + (size_t)sms * 2 * 8 * tiles * (head_dim + 2);
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
  a.wait_ns = attention_wait_ns();
  if (!(flags & GRINQH_WORKSPACE_ZEROED)) {
    const cudaError_t e = cudaMemsetAsync(workspace, 0, (size_t)sms * sizeof(unsigned), stream);
    if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
  }
  a.parts = (new_tokens * a.group + 8 * tiles - 1) / (8 * tiles);
  return kv4_dispatch(head_dim, group_size, [&](auto layout) {
    using L = decltype(layout);
    auto with = [&](auto type) {
      using T = decltype(type);
      if (tiles == 1) return launch<T, L::kDim, L::kGroup, 1>(a, sms, stream);
      return launch<T, L::kDim, L::kGroup, 2>(a, sms, stream);
    };
    return dtype == GRINQH_BF16 ? with(__nv_bfloat16{}) : with(__half{});
  });
}
