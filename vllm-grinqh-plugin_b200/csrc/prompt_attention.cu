// Causal attention over packed prompts with grouped heads.
//
//   s = scale * q k^T over the keys a query sees, p = softmax(s), out = p v
//
// One pass over the keys with the running maximum m and sum l of the softmax: a block of
// 128 keys adds exp2(s' - m) v to an accumulator, s' = s log2(e). m is kept where a new
// maximum exceeds it by less than kSlack: the weights then reach at most 2^kSlack, no
// accumulator is rescaled, and the division by l in the end makes up for it.
//
// A CTA computes two tiles of 128 queries at once, so that one tile's softmax runs while
// the tensor cores work on the other's: two heads of one kv head over the same rows where
// the group is even (they share K and V and see the same keys), else two row tiles of one
// head.
//   warp 8     loads Q once and blocks of 128 keys of K and V through a ring, by TMA
//   warp 9     issues S = Q K^T (both operands in shared memory, S in TMEM) and
//              O += P V (P in TMEM, where S was)
//   warps 0-7  one thread per query row: read S, mask, softmax, write P in 16 bits, and
//              at the end read O, divide and store
// S of the next block overwrites P of this one: the tensor pipe runs the MMAs of a thread
// in order, and S of a block is complete only after the O += P V before it, which is what
// allows the softmax warps to rescale O when they hold a new S.
//
// Keys past the sequence's end belong to another sequence and may hold anything: their
// scores are masked, the O += P V steps of 16 keys past the last visible one are not
// issued, and the at most 15 rows of V behind it are cleared in shared memory.
#include "ptx.cuh"
#include "prompt_attention.cuh"
#include "tmap.cuh"

#include <type_traits>

namespace grinqh {
namespace {

constexpr int kRows = 128;    // queries of a tile
constexpr int kKeys = 128;    // keys of a block
constexpr int kThreads = 384;
constexpr float kSlack = 8.0f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;  // columns: S0 / P0 at 0, S1 / P1 at 128, O0, O1 from here

struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int total_q, total_k;
  int seqs, heads, group;  // group: query heads of a kv head
  float scale_log2;        // softmax scale * log2(e)
};

template <int D>
struct Shape {
  static constexpr int kAtoms = D / 64;                  // 64-channel (128-byte) columns of a tile
  static constexpr uint32_t kAtom = 128 * 128;           // bytes of one, 128 rows
  static constexpr uint32_t kTileBytes = kAtoms * kAtom;
  static constexpr int kStages = D == 128 ? 5 : 10;      // K / V blocks in the ring
  static constexpr uint32_t kSmem = (2 + kStages) * kTileBytes + 1024 /*align*/ + 512 /*barriers*/;
};

// What a CTA works on.
struct Item {
  int q0, n;        // first query row, queries of the sequence
  int k0, m;        // first key row, keys of the sequence
  int row;          // first row of the tiles in the sequence
  int blocks;       // key blocks the tiles see
  bool none;
};

// Finds row block `want` (counted from the last one) over all sequences; one warp.
__device__ __forceinline__ Item find_item(const PromptArgs& a, int rows, int64_t want) {
  const int lane = threadIdx.x & 31;
  Item it;
  it.none = true;
  // sequences from the last to the first, 32 at a time: their long rows, which see the
  // most keys, start first
  for (int top = a.seqs; top > 0; top -= 32) {
    const int b = top - 1 - lane;
    int q0 = 0, q1 = 0;
    if (b >= 0) {
      q0 = min(max(a.cu_q[b], 0), a.total_q);
      q1 = min(max(a.cu_q[b + 1], q0), a.total_q);
    }
    const int count = (q1 - q0 + rows - 1) / rows;
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, want < upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int first = __shfl_sync(0xffffffffu, upto - count, src);
      const int cnt = __shfl_sync(0xffffffffu, count, src);
      it.q0 = __shfl_sync(0xffffffffu, q0, src);
      it.n = __shfl_sync(0xffffffffu, q1, src) - it.q0;
      it.row = (cnt - 1 - (int)(want - first)) * rows;
      const int bb = top - 1 - src;
      it.k0 = min(max(a.cu_k[bb], 0), a.total_k);
      it.m = min(max(a.cu_k[bb + 1], it.k0), a.total_k) - it.k0;
      // the last row of the tiles sees the most keys
      const int seen = min(it.m, it.m - it.n + min(it.n, it.row + rows));
      it.blocks = seen > 0 ? (seen + kKeys - 1) / kKeys : 0;
      it.none = false;
      return it;
    }
    want -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return it;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (Act<T>::kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap tmap_q,
                                                                       const __grid_constant__ CUtensorMap tmap_k,
                                                                       const __grid_constant__ CUtensorMap tmap_v,
                                                                       const PromptArgs a) {
  using S = Shape<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* s_q = smem;
  unsigned char* s_kv = smem + 2 * S::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_kv + S::kStages * S::kTileBytes);
  uint64_t* full = bars;                      // ring stage holds its block
  uint64_t* empty = full + S::kStages;        // ring stage may be filled
  uint64_t* q_full = empty + S::kStages;
  uint64_t* s_full = q_full + 1;              // [2] S of a tile is in TMEM
  uint64_t* p_full = s_full + 2;              // [2] P of a tile is in TMEM
  uint64_t* o_full = p_full + 2;              // [2] O of a tile is final
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  Item* s_item = reinterpret_cast<Item*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool paired = (a.group & 1) == 0;  // the tiles are two heads (else two row tiles)
  const int columns = paired ? a.heads / 2 : a.heads;  // CTAs of a row block
  const int head = (int)(blockIdx.x % columns) * (paired ? 2 : 1);

  if (warp == 8) {
    const Item it = find_item(a, paired ? kRows : 2 * kRows, blockIdx.x / columns);
    if (lane == 0) *s_item = it;
  } else if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
  } else if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_full[t], 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Item it = *s_item;
  const int kv_head = head / a.group;
  const int nb = it.none ? 0 : it.blocks;
  // keys that the last row of a tile sees (tile 1 of an unpaired item is 128 rows on)
  auto tile_row = [&](int t) { return it.row + (paired ? 0 : t * kRows); };
  auto tile_keys = [&](int t) { return min(it.m, it.m - it.n + min(it.n, tile_row(t) + kRows)); };

  // The softmax warps take the registers that the others do not need:
  // 256 x 232 + 128 x 40 = 384 x 168, what the launch holds.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8 && nb > 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, 2 * S::kTileBytes);
        for (int t = 0; t < 2; ++t)
          for (int c = 0; c < S::kAtoms; ++c)
            tma_load_3d(s_q + t * S::kTileBytes + c * S::kAtom, &tmap_q, 64 * c, paired ? head + t : head,
                        it.q0 + tile_row(t), q_full);
        for (int i = 0; i < 2 * nb; ++i) {  // K of block 0, V of block 0, K of block 1, ...
          const int s = i % S::kStages;
          if (i >= S::kStages) mbar_wait_nocall(&empty[s], ((i / S::kStages) - 1) & 1);
          mbar_arrive_expect_tx(&full[s], S::kTileBytes);
          for (int c = 0; c < S::kAtoms; ++c)
            tma_load_3d(s_kv + s * S::kTileBytes + c * S::kAtom, i & 1 ? &tmap_v : &tmap_k, 64 * c, kv_head,
                        it.k0 + (i >> 1) * kKeys, &full[s]);
        }
      }
    } else if (warp == 9 && nb > 0) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t fmt = Act<T>::kBf16 ? 1 : 0;
      constexpr uint32_t id_s = instr_desc(1, fmt, fmt, 0, 0, kKeys, kRows);
      constexpr uint32_t id_o = instr_desc(1, fmt, fmt, 0, 1, D, kRows);
      auto scores = [&](int t, int stage) {  // S_t = Q_t K^T
        const uint32_t qb = smem_u32(s_q + t * S::kTileBytes), kb = smem_u32(s_kv + stage * S::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk / 4) * S::kAtom + (kk % 4) * 32;
          mma_f16_ss(tmem + t * kKeys, smem_desc(qb + off, 16, 1024, 2), smem_desc(kb + off, 16, 1024, 2), id_s, kk > 0);
        }
        mma_commit(&s_full[t]);
      };
      auto outputs = [&](int t, int j, int stage) {  // O_t += P_t V
        const uint32_t vb = smem_u32(s_kv + stage * S::kTileBytes);
        const int steps = min(kKeys / 16, (tile_keys(t) - j * kKeys + 15) / 16);
        for (int kk = 0; kk < steps; ++kk)
          mma_f16_ts(tmem + kTmemO + t * 128, tmem + t * kKeys + kk * 8, smem_desc(vb + kk * 2048, S::kAtom, 1024, 2),
                     id_o, (j > 0 || kk > 0) ? 1u : 0u);
      };
      mbar_wait_nocall(q_full, 0);
      mbar_wait_nocall(&full[0], 0);
      if (lane == 0) {
        scores(0, 0);
        scores(1, 0);
        mma_commit(&empty[0]);
      }
      __syncwarp();
      for (int j = 0; j < nb; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 2;
        const int vs = vi % S::kStages, ks = ki % S::kStages;
        mbar_wait_nocall(&full[vs], (vi / S::kStages) & 1);
        const int left = it.m - j * kKeys;  // keys of the sequence from this block on
        if (left < kKeys && (left & 15)) {
          // rows of V behind the sequence's end in its last step of 16 keys
          for (int r = left + (lane >> 3); r < ((left + 15) & ~15); r += 4)
            for (int c = 0; c < S::kAtoms; ++c)
              *reinterpret_cast<uint4*>(s_kv + vs * S::kTileBytes + c * S::kAtom + r * 128 + (lane & 7) * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
        }
        for (int t = 0; t < 2; ++t) {
          mbar_wait_nocall(&p_full[t], j & 1);
          tc_fence_after();
          if (t == 0 && j + 1 < nb) mbar_wait_nocall(&full[ks], (ki / S::kStages) & 1);
          if (lane == 0) {
            outputs(t, j, vs);
            if (j + 1 < nb) {
              scores(t, ks);
            } else {
              mma_commit(&o_full[t]);
            }
          }
          __syncwarp();
        }
        if (lane == 0) {
          mma_commit(&empty[vs]);
          if (j + 1 < nb) mma_commit(&empty[ks]);
        }
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if (!it.none) {
      // ------------------------------------------------------------ softmax, epilogue
      const int t = warp >> 2;
      const int r = (warp & 3) * 32 + lane;           // row of the tile
      const int row = tile_row(t) + r;                // of the sequence
      const int seen = min(it.m, it.m - it.n + row + 1);  // keys this row sees (<= 0: none)
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + t * kKeys, to = tmem + lanes + kTmemO + t * 128;
      const int first_seen = it.m - it.n + tile_row(t) + 1;  // keys the tile's first row sees
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nb; ++j) {
        mbar_wait_nocall(&s_full[t], j & 1);
        tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, sr[c]);
        tmem_ld_wait();
        if ((j + 1) * kKeys > min(it.m, first_seen)) {
          const int lim = seen - j * kKeys;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i >= lim) sr[c][i] = 0xff800000u;  // -inf
        }
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(sr[c][i]));
        top *= a.scale_log2;
        const bool up = top > m + kSlack || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, up)) {
          const float f = up ? exp2_fast(m - top) : 1.0f;
          if (up) m = top;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(to + 32 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(to + 32 * c, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p0 = exp2_fast(fmaf(__uint_as_float(sr[c][2 * i]), a.scale_log2, -ref));
            const float p1 = exp2_fast(fmaf(__uint_as_float(sr[c][2 * i + 1]), a.scale_log2, -ref));
            l += p0 + p1;
            pk[i] = pack2<T>(p0, p1);
          }
          tmem_st16(ts + 16 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (nb > 0) {
        mbar_wait_nocall(&o_full[t], 0);
        tc_fence_after();
      }
      const bool in = row < it.n, none = l == 0.f;
      const int64_t at = (int64_t)(it.q0 + row) * a.heads + (paired ? head + t : head);
      T* out = static_cast<T*>(a.out) + at * D;
      const float inv = 1.0f / l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (nb > 0) {
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait();
        }
        if (in) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              w[x] = none ? 0u
                          : pack2<T>(__uint_as_float(o[8 * i + 2 * x]) * inv, __uint_as_float(o[8 * i + 2 * x + 1]) * inv);
            *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
      }
      if (in) a.lse[at] = none ? -INFINITY : m * kLn2 + logf(l);
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, kTmemCols);
}

template <typename T, int D>
int launch(const PromptArgs& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  auto kern = prompt_attention_kernel<T, D>;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<D>::kSmem);
  if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const bool paired = (a.group & 1) == 0;
  const int rows = paired ? kRows : 2 * kRows;
  // every sequence's rows fill whole tiles but its last: at most this many row blocks
  const int64_t blocks = std::min<int64_t>(a.total_q / rows + a.seqs, a.total_q);
  const int64_t grid = blocks * (paired ? a.heads / 2 : a.heads);
  GRINQH_REQUIRE(grid < (1LL << 31), "too many row blocks (%lld)", (long long)blocks);
  kern<<<(unsigned)grid, kThreads, Shape<D>::kSmem, st>>>(q, k, v, a);
  return check_launch("prompt_attention");
}

}  // namespace

unsigned take_prompt_timeouts() {
  unsigned v = 0, z = 0;
  if (cudaMemcpyFromSymbol(&v, g_wait_timeouts, sizeof(v)) != cudaSuccess) return 0;
  cudaMemcpyToSymbol(g_wait_timeouts, &z, sizeof(z));
  return v;
}

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
  GRINQH_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "softmax_scale must be positive and finite");
  if (total_q == 0 || num_seqs == 0) return GRINQH_OK;
  GRINQH_REQUIRE(q && (total_k == 0 || (k && v)) && cu_seqlens_q && cu_seqlens_k && out && lse, "null pointer");
  GRINQH_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && q_token_stride % 8 == 0 &&
                     q_head_stride % 8 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                     v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                 "q, k, v, their strides and out must be 16-byte aligned");
  const PromptArgs a{cu_seqlens_q,   cu_seqlens_k, out, lse, (int)total_q, (int)total_k, num_seqs, num_heads,
                     num_heads / num_kv_heads, softmax_scale * 1.4426950408889634f};
  const bool bf16 = dtype == GRINQH_BF16;
  CUtensorMap tq, tk, tv;
  GRINQH_RETURN_IF(tmap_heads(&tq, bf16, q, total_q, num_heads, head_dim, q_token_stride, q_head_stride, 128, "q"));
  if (total_k > 0) {
    GRINQH_RETURN_IF(tmap_heads(&tk, bf16, k, total_k, num_kv_heads, head_dim, k_token_stride, k_head_stride, 128, "k"));
    GRINQH_RETURN_IF(tmap_heads(&tv, bf16, v, total_k, num_kv_heads, head_dim, v_token_stride, v_head_stride, 128, "v"));
  } else {
    tk = tv = tq;  // never read: no row sees a key
  }
  if (head_dim == 128)
    return bf16 ? launch<__nv_bfloat16, 128>(a, tq, tk, tv, stream) : launch<__half, 128>(a, tq, tk, tv, stream);
  return bf16 ? launch<__nv_bfloat16, 64>(a, tq, tk, tv, stream) : launch<__half, 64>(a, tq, tk, tv, stream);
}
