// Causal attention over packed prompts with grouped heads.
//
//   s = scale * q k^T over the keys a query sees, p = softmax(s), out = p v
//
// One pass over the keys with the running maximum m and sum l of the softmax: a block of
// keys adds exp2(s' - m) v to an accumulator, s' = s log2(e). m is kept where a new maximum
// exceeds it by less than kSlack: the weights then reach at most 2^kSlack, no accumulator
// is rescaled, and the division by l in the end makes up for it.
//
// A tile is 128 rows: as many tokens as its query heads of one kv head allow, token by
// token (which a TMA box of {64 channels, heads, tokens} lays out by itself), so a short
// prompt fills its tiles with all heads that share K and V. An item is two tiles, so that
// one tile's softmax runs while the tensor cores work on the other's. The grid has a CTA
// per item, those that see the most keys first; the CTA that an SM runs takes over the
// items of CTAs that have not started (cluster launch control) and keeps its pipeline
// going from one to the next.
//   warp 8     finds the items; loads Q and blocks of K and V through a ring, by TMA
//   warp 9     issues S = Q K^T (both operands in shared memory, S in TMEM) and
//              O += P V (P in TMEM)
//   warps 0-7  one thread per query row: read S, mask, softmax, write P in 16 bits, and
//              at the end read O, divide and store
// The softmax warps hold a block's scores, then its weights, in registers: S is free for
// the other tile as soon as it is read, and P (and O) may be in use until the next weights
// are made. So one S serves both tiles, S, P and O fit the 512 columns of TMEM, and the
// products follow one another as S0 O0 S1 O1, each with a whole round of the others to
// wait in. A 128 x 128 x 16 product takes 102 cycles with both operands in shared memory
// and 78 with A in TMEM (measured alone; 64 would be full rate), 2880 a round at head_dim
// 128; the exponentials, 8 cycles for a warp's 32 of them, 2048 a round.
//
// What bounds it, by the SMs' active cycles: a prompt of 16384 tokens at head_dim 128 takes 3080
// cycles a round, so the products 94% of them, and 5% more until the last SM ends. 14 packed
// prompts of up to 2048 tokens take 4270 a round: with 6 items an SM, half masked blocks,
// starts and epilogues count, in which one of the two pipes waits. 7 chunks after prefixes at
// head_dim 64, 3280 a round, have 1.6 items an SM that are not cut: SMs are active for 72 to 124
// thousand cycles, 94 on average, of which exponentials are 59%.
//
// Where there are few items for the SMs (a chunk after a long prefix), each item's keys are
// cut into the same number of parts, items of their own; each writes its sums to the
// workspace and a second kernel joins them in order.
//
// Waits are bounded. Once one of a CTA is lost, nothing more is loaded and no more items are
// asked for. Those that the CTA has taken over pass through as ever, their products are made
// with whatever is there, and their rows become NaN; what is in flight is waited for before
// the CTA ends. (Leaving the loops instead takes a vote at every wait: 475 us -> 553 for a
// prompt of 16384 tokens.)
//
// Measured (bf16, D = 128): a prompt of 16384 tokens, 8 / 2 heads, 475 us, 1.16 PFLOP/s or
// 69% of a library matrix product's rate (the SMs at 1.65 GHz), with the tensor pipe active in
// 66% of the cycles; 14 packed prompts of up to 2048 tokens, 32 / 8 heads, 111 us and 46%.
//
// Keys past the sequence's end belong to another sequence and may hold anything: their
// scores are masked, the O += P V steps of 16 keys past the last visible one are not
// issued, and the at most 15 rows of V behind it are cleared in shared memory.
#include "launch.cuh"
#include "ptx.cuh"
#include "prompt_attention.cuh"
#include "tmap.cuh"

#include <algorithm>

namespace grinqh {
namespace {

constexpr int kRows = 128;    // rows of a tile: tokens x query heads
constexpr int kKeys = 128;    // keys of a block
constexpr int kThreads = 384;
constexpr float kSlack = 8.0f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr uint32_t kTmemCols = 512;

struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int total_q, total_k;
  int seqs, heads, kv_heads, group;  // group: query heads of a kv head
  int tokens;                        // of a tile: 128 / group
  int parts;                         // of an item's keys
  int more;                          // whether there are more items than SMs
  float scale_log2;                  // softmax scale * log2(e)
  uint64_t wait_ns;                  // the longest wait
  float* sums;                       // [item][part][tile]{O[D / 4][row][4], {m, l}[row], token[row]}, for parts > 1
};

template <int D>
struct Shape {
  static constexpr int kAtoms = D / 64;                  // 64-channel (128-byte) columns of a tile or block
  static constexpr uint32_t kQAtom = kRows * 128;        // bytes of one
  static constexpr uint32_t kQBytes = kAtoms * kQAtom;
  static constexpr uint32_t kAtom = kKeys * 128;
  static constexpr uint32_t kBytes = kAtoms * kAtom;
  static constexpr int kStages = D == 128 ? 5 : 10;      // K / V blocks in the ring
  static constexpr uint32_t kSmem = 2 * kQBytes + kStages * kBytes + 1024 /*align*/ + 512 /*barriers*/;
  // Steps of 16 keys whose weights are handed over first, while the others are made. At
  // head_dim 64 the exponentials bound the kernel and the wait for them is worth a second
  // hand-over: chunks of prompts 69.4 -> 68.0 us with 64 keys first; at 128 the products do, and it
  // costs: a prompt of 16384 tokens 487 -> 495.
  static constexpr int kFirst = D == 64 ? kKeys / 32 : kKeys / 16;
  // TMEM columns: S, then P and O of both tiles
  static constexpr uint32_t kS = 0, kP = kKeys, kO = 2 * kKeys, kPNext = kKeys / 2, kONext = D;
  static_assert(kO + 2 * D <= kTmemCols && kSmem <= 227 * 1024, "budgets");
};

// Two tiles of a sequence and kv head.
struct Item {
  int q0, n;      // first query row, queries of the sequence
  int k0, m;      // first key row, keys of the sequence
  int token;      // first token of the tiles in the sequence
  int kv_head;    // < 0: no more items
  int begin, end;  // the key blocks of this part
  int index, part;
  __device__ __forceinline__ int first(int t, int tokens) const { return token + t * tokens; }
  // keys that the last token of tile t sees, and blocks of them
  __device__ __forceinline__ int keys(int t, int tokens) const {
    return max(0, min(m, m - n + min(n, first(t, tokens) + tokens)));
  }
  __device__ __forceinline__ int all_blocks(int t, int tokens) const {
    return first(t, tokens) < n ? (keys(t, tokens) + kKeys - 1) / kKeys : 0;
  }
  // of them, those of this part
  __device__ __forceinline__ int blocks(int t, int tokens) const {
    return max(0, min(all_blocks(t, tokens), end) - begin);
  }
};

// A sequence's rows, cut to the tensors.
struct Rows {
  int q0, n, k0, m;
};

__device__ __forceinline__ Rows rows_of(const PromptArgs& a, int b) {
  const int q0 = min(max(a.cu_q[b], 0), a.total_q), k0 = min(max(a.cu_k[b], 0), a.total_k);
  return {q0, min(max(a.cu_q[b + 1], q0), a.total_q) - q0, k0, min(max(a.cu_k[b + 1], k0), a.total_k) - k0};
}

// The sequences if there are at most 32, one a lane, those with the most keys last.
__device__ __forceinline__ Rows sorted_rows(const PromptArgs& a) {
  const int lane = threadIdx.x & 31;
  Rows mine{0, 0, 0, 0};
  if (lane < a.seqs) mine = rows_of(a, lane);
  int rank = lane;
  if (a.seqs > 1) {
    rank = lane < a.seqs ? 0 : lane;
    for (int o = 0; o < a.seqs; ++o) {
      const int other = __shfl_sync(0xffffffffu, mine.m, o);
      if (lane < a.seqs) rank += other < mine.m || (other == mine.m && o < lane);
    }
  }
  int from = lane;
  for (int o = 0; o < a.seqs; ++o)
    if (__shfl_sync(0xffffffffu, rank, o) == lane) from = o;
  return {__shfl_sync(0xffffffffu, mine.q0, from), __shfl_sync(0xffffffffu, mine.n, from),
          __shfl_sync(0xffffffffu, mine.k0, from), __shfl_sync(0xffffffffu, mine.m, from)};
}

// Finds item `at`, token blocks of `tokens` each being counted from the last one over all
// sequences; one warp. few: the sequences if there are at most 32.
__device__ __forceinline__ Item find_item(const PromptArgs& a, const Rows& few, int tokens, int at) {
  const int lane = threadIdx.x & 31;
  Item it{0, 0, 0, 0, 0, -1, 0, 0, 0, 0};
  if (at < 0) return it;
  const int kv_head = at % a.kv_heads, part = at / a.kv_heads % a.parts;
  int want = at / a.kv_heads / a.parts;
  it.index = want * a.kv_heads + kv_head;
  it.part = part;
  // sequences from the last to the first, 32 at a time, and their tokens from the last,
  // which see the most keys
  for (int top = a.seqs; top > 0; top -= 32) {
    const int b = top - 1 - lane;
    Rows rows;
    if (a.seqs <= 32) {
      const int from = max(b, 0);
      rows = {__shfl_sync(0xffffffffu, few.q0, from), __shfl_sync(0xffffffffu, few.n, from),
              __shfl_sync(0xffffffffu, few.k0, from), __shfl_sync(0xffffffffu, few.m, from)};
    } else if (b >= 0) {
      rows = rows_of(a, b);
    }
    const int count = b >= 0 ? (rows.n + tokens - 1) / tokens : 0;
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, want < upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int before = __shfl_sync(0xffffffffu, upto - count, src);
      const int cnt = __shfl_sync(0xffffffffu, count, src);
      it.q0 = __shfl_sync(0xffffffffu, rows.q0, src);
      it.n = __shfl_sync(0xffffffffu, rows.n, src);
      it.k0 = __shfl_sync(0xffffffffu, rows.k0, src);
      it.m = __shfl_sync(0xffffffffu, rows.m, src);
      it.token = (cnt - 1 - (want - before)) * tokens;
      it.kv_head = kv_head;
      const int all = max(it.all_blocks(0, tokens / 2), it.all_blocks(1, tokens / 2));
      it.begin = (int)((int64_t)all * part / a.parts);
      it.end = (int)((int64_t)all * (part + 1) / a.parts);
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

// Sums of a tile of one part, in floats.
__host__ __device__ constexpr int64_t sums_floats(int dim) { return (int64_t)kRows * (dim + 3); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap tmap_q,
                                                                       const __grid_constant__ CUtensorMap tmap_k,
                                                                       const __grid_constant__ CUtensorMap tmap_v,
                                                                       const PromptArgs a) {
  using S = Shape<D>;
  constexpr int ST = S::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* s_q = smem;
  unsigned char* s_kv = smem + 2 * S::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_kv + ST * S::kBytes);
  uint64_t* full = bars;            // ring stage holds its block
  uint64_t* empty = full + ST;      // ring stage may be filled
  uint64_t* q_full = empty + ST;    // the item's queries are there
  uint64_t* q_empty = q_full + 1;   // ... are not needed any more
  uint64_t* s_full = q_empty + 1;   // [2] S of a tile is in TMEM
  uint64_t* s_empty = s_full + 2;   // ... is in registers
  uint64_t* p_full = s_empty + 1;   // [2] P of a tile is in TMEM
  uint64_t* p_half = p_full + 2;    // [2] ... of the first kFirst steps
  uint64_t* o_full = p_half + 2;    // [2] ... has been multiplied: O holds the block, P may be written
  uint64_t* o_empty = o_full + 2;   // [2] O of an item is read
  uint64_t* i_full = o_empty + 2;   // [2] an item is known
  uint64_t* i_empty = i_full + 2;   // [2] ... is not needed any more
  uint64_t* c_full = i_empty + 2;   // the answer about a next CTA is there
  uint64_t* done = c_full + 1;      // no product is in flight
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  Item* s_item = reinterpret_cast<Item*>(tmem_slot + 2);  // [2]
  __shared__ __align__(16) uint32_t s_next[4];
  __shared__ int s_lost;  // a wait of this CTA was lost

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
  } else if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(s_empty, 128);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&p_half[t], 128);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 128);
      mbar_init(&i_full[t], 1);
      mbar_init(&i_empty[t], 9);
    }
    mbar_init(c_full, 1);
    mbar_init(done, 1);
    fence_mbar_init();
    s_lost = lost_beforehand(a.wait_ns);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // the next kernel's set-up may overlap this one, as this one's did its predecessor
  allow_dependent_grid();
  wait_prior_grid();
  const uint32_t tmem = *tmem_slot;
  const int tokens = a.tokens;
  // A wait for data. Who goes on after it was lost is followed by NaN (see the epilogue).
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or_lose(bar, parity, a.wait_ns, &s_lost); };
  // Items pass through whatever was lost: whom these wait for goes on in bounded time.
  auto wait_item = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_drain(bar, parity)); };
  // the k-th item of this CTA, for every warp but the one that finds it
  auto item = [&](int k) {
    Item it{0, 0, 0, 0, 0, -1, 0, 0, 0, 0};
    if (!wait_item(&i_full[k & 1], (k >> 1) & 1)) return it;
    it = s_item[k & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[k & 1]);
    return it;
  };

  // The softmax warps take the registers that the others do not need:
  // 256 x 232 + 128 x 40 = 384 x 168, what the launch holds.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8) {
      // ---------------------------------------------------------- items, TMA producer
      int stage = 0, round = 1, used = 0;  // ring stage and parity of its release; items so far
      // Whether memory may be loaded to: it is free, and was not passed on too soon (a load
      // still on its way would share its barrier with the next).
      bool lost = false;
      auto may_load = [&](uint64_t* bar, uint32_t parity) {
        const bool free = mbar_wait_or_lose(bar, parity, a.wait_ns, &s_lost) &&
                          *reinterpret_cast<volatile int*>(&s_lost) == 0;
        lost = lost || !__all_sync(0xffffffffu, free);
        return !lost;
      };
      // The next item is asked for when this one's last kAhead loads are left and looked up
      // kFind before its end, so that neither is waited for (a few microseconds an item) and
      // an SM that is behind still takes fewer.
      constexpr int kAhead = 12, kFind = 4;
      const Rows few = a.seqs <= 32 ? sorted_rows(a) : Rows{0, 0, 0, 0};  // the longest start first
      Item it = find_item(a, few, 2 * tokens, (int)blockIdx.x);
      for (int k = 0;; ++k) {
        if (k >= 2 && !wait_item(&i_empty[k & 1], ((k >> 1) - 1) & 1)) break;
        if (lane == 0) {
          s_item[k & 1] = it;
          mbar_arrive(&i_full[k & 1]);
        }
        __syncwarp();
        if (it.kv_head < 0) break;
        int loads = 2 * max(it.blocks(0, tokens), it.blocks(1, tokens));
        if (loads > 0 && used > 0) may_load(q_empty, (used - 1) & 1);
        if (lost) loads = 0;
        if (loads > 0) {
          ++used;
          if (lane == 0) {
            const uint32_t bytes = a.group * tokens * 128;  // of 64 channels of a tile
            mbar_arrive_expect_tx(q_full, 2 * S::kAtoms * bytes);
            for (int t = 0; t < 2; ++t)
              for (int c = 0; c < S::kAtoms; ++c)
                tma_load_3d(s_q + t * S::kQBytes + c * S::kQAtom, &tmap_q, 64 * c, it.kv_head * a.group,
                            it.q0 + it.first(t, tokens), q_full);
          }
        }
        Item following = it;
        following.kv_head = -1;
        bool asked = false;
        auto ask = [&] {
          asked = a.more && !lost;
          if (lane == 0 && asked) {
            fence_proxy_async_smem();  // the last answer has been read
            mbar_arrive_expect_tx(c_full, 16);
            next_cta_ask(s_next, c_full);
          }
          __syncwarp();
        };
        auto find = [&] {
          const bool answered = asked && wait_item(c_full, k & 1);
          following = find_item(a, few, 2 * tokens, answered ? (int)next_cta_answer(s_next) : -1);
        };
        const int when_ask = max(0, loads - kAhead), when_find = max(0, loads - kFind);
        bool found = false;
        for (int n = 0; n < loads; ++n) {  // K of block 0, V of block 0, K of block 1, ...
          if (n == when_ask) ask();
          if (n == when_find) found = true, find();
          if (!may_load(&empty[stage], round)) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[stage], S::kBytes);
            for (int c = 0; c < S::kAtoms; ++c)
              tma_load_3d(s_kv + stage * S::kBytes + c * S::kAtom, n & 1 ? &tmap_v : &tmap_k, 64 * c, it.kv_head,
                          it.k0 + (it.begin + (n >> 1)) * kKeys, &full[stage]);
          }
          __syncwarp();
          if (++stage == ST) {
            stage = 0;
            round ^= 1;
          }
        }
        if (!found) {
          if (loads == 0) ask();
          find();
        }
        it = following;
      }
      // the loads still in flight: of each stage the last, a round back behind `stage`
      if (used > 0) mbar_drain(q_full, (used - 1) & 1);
#pragma unroll 1
      for (int s = 0; s < ST; ++s) mbar_drain(&full[s], s < stage ? round ^ 1 : round);
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t fmt = Act<T>::kBf16 ? 1 : 0;
      constexpr uint32_t id_s = instr_desc(1, fmt, fmt, 0, 0, kKeys, kRows);
      constexpr uint32_t id_o = instr_desc(1, fmt, fmt, 0, 1, D, kRows);
      const uint32_t tm = uniform(tmem);
      // descriptors by their first one: an address is 16 bytes a unit, in the low bits
      const uint64_t q_desc = smem_desc(smem_u32(s_q), 16, 1024, 2);
      const uint64_t k_desc = smem_desc(smem_u32(s_kv), 16, 1024, 2);
      const uint64_t v_desc = smem_desc(smem_u32(s_kv), S::kAtom, 1024, 2);
      int ns = 0, np[2] = {0, 0}, no[2] = {0, 0};  // uses of S, weights and outputs of each tile so far
      bool free = true;  // no wait for O to be read was lost; once one was, O is not written any more
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      auto scores = [&](int t, int at) {  // S = Q_t K^T
        if (ns > 0) wait(s_empty, (ns - 1) & 1);
        ++ns;
        tc_fence_after();
        const uint64_t qd = q_desc + t * (S::kQBytes >> 4), kd = k_desc + at * (S::kBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_f16_ss(tm + S::kS, qd + (kk / 4) * (S::kQAtom >> 4) + (kk % 4) * 2,
                       kd + (kk / 4) * (S::kAtom >> 4) + (kk % 4) * 2, id_s, kk > 0);
          mma_commit(&s_full[t]);
        }
        __syncwarp();
      };
      auto outputs = [&](int t, int at, int steps, bool more) {  // O_t += P_t V, steps of 16 keys
        const uint64_t vd = v_desc + at * (S::kBytes >> 4);
        const uint32_t o = tm + S::kO + t * S::kONext, p = tm + S::kP + t * S::kPNext;
        constexpr int kSteps = kKeys / 16, kFirst = S::kFirst;
        wait(kFirst < kSteps ? &p_half[t] : &p_full[t], np[t] & 1);
        tc_fence_after();
        if (elect_one() && free) {
          if (steps >= kFirst) {
#pragma unroll
            for (int kk = 0; kk < kFirst; ++kk)
              mma_f16_ts(o, p + kk * 8, vd + kk * 128, id_o, more || kk > 0 ? 1u : 0u);
          } else {
            for (int kk = 0; kk < steps; ++kk)
              mma_f16_ts(o, p + kk * 8, vd + kk * 128, id_o, more || kk > 0 ? 1u : 0u);
          }
          if constexpr (kFirst == kSteps) mma_commit(&o_full[t]);
        }
        __syncwarp();
        if constexpr (kFirst < kSteps) {
          wait(&p_full[t], np[t] & 1);
          tc_fence_after();
          if (elect_one() && free) {
            if (steps == kSteps) {
#pragma unroll
              for (int kk = kFirst; kk < kSteps; ++kk) mma_f16_ts(o, p + kk * 8, vd + kk * 128, id_o, 1u);
            } else {
              for (int kk = kFirst; kk < steps; ++kk) mma_f16_ts(o, p + kk * 8, vd + kk * 128, id_o, 1u);
            }
            mma_commit(&o_full[t]);
          }
          __syncwarp();
        }
        ++np[t];
      };
      int stage = 0, round = 0, used = 0;  // ring stage of the next block and its parity; items so far
      auto next = [&] {
        wait(&full[stage], round);
        const int at = stage;
        if (++stage == ST) {
          stage = 0;
          round ^= 1;
        }
        return at;
      };
      for (int k = 0;; ++k) {
        const Item it = item(k);
        if (uniform(it.kv_head) < 0) break;
        const int nbt[2] = {uniform(it.blocks(0, tokens)), uniform(it.blocks(1, tokens))};
        const int keys[2] = {uniform(it.keys(0, tokens)), uniform(it.keys(1, tokens))};
        const int nb = max(nbt[0], nbt[1]), begin = uniform(it.begin), m = uniform(it.m);
        if (nb == 0) continue;
        wait(q_full, used & 1);
        ++used;
        const int first = next();
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (nbt[t] > 0) scores(t, first);
        commit(&empty[first]);
        if (nb == 1) commit(q_empty);
        for (int j = 0; j < nb; ++j) {
          const int vs = next();
          const int left = m - (begin + j) * kKeys;  // keys of the sequence from this block on
          if (left < kKeys && (left & 15)) {
            // rows of V behind the sequence's end in its last step of 16 keys
            for (int r = left + (lane >> 3); r < ((left + 15) & ~15); r += 4)
              for (int c = 0; c < S::kAtoms; ++c)
                *reinterpret_cast<uint4*>(s_kv + vs * S::kBytes + c * S::kAtom + r * 128 + (lane & 7) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
          }
          const int ks = j + 1 < nb ? next() : 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j + 1 < nbt[t]) scores(t, ks);  // of the next block, while this one's weights are made
            if (j >= nbt[t]) continue;
            if (j == 0) {
              if (no[t] > 0) free = wait(&o_empty[t], (no[t] - 1) & 1) && free;
              ++no[t];
            }
            outputs(t, vs, min(kKeys / 16, (keys[t] - (begin + j) * kKeys + 15) / 16), j > 0);
          }
          if (j + 1 < nb) commit(&empty[ks]);
          if (j + 2 == nb) commit(q_empty);
          commit(&empty[vs]);
        }
      }
      if (elect_one()) mma_commit(done);
      __syncwarp();
      mbar_drain(done, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ------------------------------------------------------------ softmax, epilogue
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile
    const int r_token = r / a.group, r_head = r - r_token * a.group;
    const uint32_t base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = base + S::kS, tp = base + S::kP + t * S::kPNext,
                   to = base + S::kO + t * S::kONext;
    constexpr int kCols = 16, kChunks = kKeys / kCols;
    int ns = 0;  // blocks so far
    for (int k = 0;; ++k) {
      const Item it = item(k);
      if (it.kv_head < 0) break;
      const int nb = it.blocks(t, tokens);
      const int token = it.first(t, tokens) + r_token;         // of the sequence
      const int seen = min(it.m, it.m - it.n + token + 1);      // keys this row sees (<= 0: none)
      const int all_see = min(it.m, it.m - it.n + it.first(t, tokens) + 1);  // keys that every row sees
      float m = -INFINITY, ref = 0.f;
      float2 l0 = make_float2(0.f, 0.f), l1 = l0;
      for (int j = 0; j < nb; ++j, ++ns) {
        wait(&s_full[t], ns & 1);
        tc_fence_after();
        uint32_t sr[kChunks][kCols];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) tmem_ld16(ts + kCols * c, sr[c]);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(s_empty);
        if ((it.begin + j + 1) * kKeys > all_see) {
          const int lim = seen - (it.begin + j) * kKeys;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < kCols; ++i)
              if (kCols * c + i >= lim) sr[c][i] = 0xff800000u;  // -inf
        }
        float mx[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          mx[c] = __uint_as_float(sr[c][0]);
#pragma unroll
          for (int i = 1; i < kCols - 1; i += 2)
            mx[c] = fmaxf(fmaxf(mx[c], __uint_as_float(sr[c][i])), __uint_as_float(sr[c][i + 1]));
          mx[c] = fmaxf(mx[c], __uint_as_float(sr[c][kCols - 1]));
        }
#pragma unroll
        for (int c = 1; c < kChunks; ++c) mx[0] = fmaxf(mx[0], mx[c]);
        const float top = mx[0] * a.scale_log2;
        const bool up = top > m + kSlack || (m == -INFINITY && top > m);
        const float f = up ? exp2_fast(m - top) : 1.0f;
        if (up) m = ref = top;
        const bool rescale = __any_sync(0xffffffffu, up);
        if (rescale) l0.x *= f, l0.y *= f, l1.x *= f, l1.y *= f;
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), ref2 = make_float2(-ref, -ref);
        // Weights are rounded to the type of V, since a product's operands have one: each by
        // up to 2^-9 (bf16) or 2^-12 of itself, either way, and l sums them before. Outputs are off
        // by 1.9e-3 (bf16) and 2.9e-4 (fp16) in the 2-norm, against 1.6e-3 and 2.1e-4 with fp32
        // weights, where only their own rounding is left; V and P in fp32 would take twice the
        // products. The exponential's own error is 2^-22.
        auto weights = [&](int c, uint32_t (&pk)[kCols / 2]) {
#pragma unroll
          for (int i = 0; i < kCols / 2; ++i) {
            const float2 x = __ffma2_rn(
                make_float2(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), scale2, ref2);
            const float2 p = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            if (i & 1)
              l1 = __fadd2_rn(l1, p);
            else
              l0 = __fadd2_rn(l0, p);
            pk[i] = pack2<T>(p.x, p.y);
          }
        };
        uint32_t pk[kChunks][kCols / 2];
#pragma unroll
        for (int c = 0; c < S::kFirst; ++c) weights(c, pk[c]);
        // the weights stay in registers until the block before has been multiplied: P is
        // free then, and O whole
        if (ns > 0) wait(&o_full[t], (ns - 1) & 1);
        tc_fence_after();
        if (rescale && j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(to + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(to + 16 * c, o);
          }
        }
#pragma unroll
        for (int c = 0; c < S::kFirst; ++c) tmem_st8(tp + kCols / 2 * c, pk[c]);
        if constexpr (S::kFirst < kChunks) {  // their product may begin while the others are made
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&p_half[t]);
#pragma unroll
          for (int c = S::kFirst; c < kChunks; ++c) weights(c, pk[c]);
#pragma unroll
          for (int c = S::kFirst; c < kChunks; ++c) tmem_st8(tp + kCols / 2 * c, pk[c]);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      float l = (l0.x + l0.y) + (l1.x + l1.y);
      const bool in = token < it.n && r_token < tokens;
      const int64_t at = (int64_t)(it.q0 + token) * a.heads + it.kv_head * a.group + r_head;
      // The rows of a pair of lanes; their lanes store 64 bytes of one row, then of the other.
      // (A row a lane, 16 bytes at a time, a store touched 32 lines: 2 us for two tiles.)
      const int odd = lane & 1;
      const int64_t other = __shfl_xor_sync(0xffffffffu, at, 1);
      const bool other_in = __shfl_xor_sync(0xffffffffu, (int)in, 1);
      T* row0 = static_cast<T*>(a.out) + (odd ? other : at) * D + 16 * odd;
      T* row1 = static_cast<T*>(a.out) + (odd ? at : other) * D + 16 * odd;
      const bool in0 = odd ? other_in : in, in1 = odd ? in : other_in;
      if (nb > 0) {
        wait(&o_full[t], (ns - 1) & 1);
        tc_fence_after();
        // Whoever passed on what was not there had lost a wait before, and this read follows
        // what was passed on: the row comes to NaN.
        if (*reinterpret_cast<volatile int*>(&s_lost)) l = __int_as_float(0x7fffffff);
      }
      const bool none = m == -INFINITY && l == l;  // no score but -inf
      const float inv = 1.0f / l;
      float* sums = a.sums + (((int64_t)it.index * a.parts + it.part) * 2 + t) * sums_floats(D);
      // 32 channels of O at once: with more, the loop above loses registers
#pragma unroll 1
      for (int h = 0; h < D; h += 32) {
        uint32_t o[32];
        if (nb > 0) {
          tmem_ld32(to + h, o);
          tmem_ld_wait();
          if (h + 32 == D) {
            tc_fence_before();
            mbar_arrive(&o_empty[t]);
          }
        }
        if (a.parts > 1) {
          if (nb > 0) {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              __stcg(reinterpret_cast<uint4*>(sums) + (h + d) / 4 * kRows + r,
                     make_uint4(o[d], o[d + 1], o[d + 2], o[d + 3]));
          }
        } else {
          uint32_t w0[8], w1[8];  // what this lane stores of the two rows
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float f = none ? 0.f : inv;
            const uint32_t lo = none ? 0u : pack2<T>(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f);
            const uint32_t hi =
                none ? 0u : pack2<T>(__uint_as_float(o[16 + 2 * i]) * f, __uint_as_float(o[17 + 2 * i]) * f);
            const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
            w0[i] = odd ? x : lo;
            w1[i] = odd ? hi : x;
          }
          if (in0) st_32(row0 + h, w0);
          if (in1) st_32(row1 + h, w1);
        }
        __syncwarp();
      }
      if (a.parts == 1) {
        if (in) a.lse[at] = none ? -INFINITY : m * kLn2 + logf(l);
        continue;
      }
      // a part of an item
      __stcg(reinterpret_cast<float2*>(sums + kRows * D) + r, make_float2(nb > 0 ? m : -INFINITY, nb > 0 ? l : 0.f));
      __stcg(reinterpret_cast<int*>(sums + kRows * (D + 2)) + r, in ? it.q0 + token : -1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, kTmemCols);
}

// Joins the parts of an item: blockIdx.x is item and tile, blockIdx.y 32 of the channels; a
// thread takes a row.
template <typename T, int D>
__global__ void __launch_bounds__(kRows) join_kernel(const PromptArgs a) {
  const int index = blockIdx.x >> 1, t = blockIdx.x & 1, r = threadIdx.x, d0 = 32 * blockIdx.y;
  allow_dependent_grid();
  wait_prior_grid();
  // how many items there are
  int count = 0;
  for (int b = threadIdx.x & 31; b < a.seqs; b += 32) {
    const int q0 = min(max(a.cu_q[b], 0), a.total_q), q1 = min(max(a.cu_q[b + 1], q0), a.total_q);
    count += (q1 - q0 + 2 * a.tokens - 1) / (2 * a.tokens);
  }
  if (index >= __reduce_add_sync(0xffffffffu, count) * a.kv_heads) return;
  const float* sums = a.sums + ((int64_t)index * a.parts * 2 + t) * sums_floats(D);
  const int token = __ldcg(reinterpret_cast<const int*>(sums + kRows * (D + 2)) + r);
  if (token < 0) return;
  float top = -INFINITY, all = 0.f, v[32];
#pragma unroll
  for (int d = 0; d < 32; ++d) v[d] = 0.f;
#pragma unroll 2
  for (int p = 0; p < a.parts; ++p, sums += 2 * sums_floats(D)) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(sums + kRows * D) + r);
    float4 x[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = __ldcg(reinterpret_cast<const float4*>(sums) + (d0 / 4 + d) * kRows + r);
    if (ml.y == 0.f) continue;  // it saw nothing, and wrote no sums (a NaN counts)
    const float now = fmaxf(top, ml.x);
    const float f = now == -INFINITY ? 1.0f : exp2_fast(top - now), g = exp2_fast(ml.x - now);
    top = now;
    all = fmaf(ml.y, g, all * f);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      v[4 * d] = fmaf(x[d].x, g, v[4 * d] * f), v[4 * d + 1] = fmaf(x[d].y, g, v[4 * d + 1] * f);
      v[4 * d + 2] = fmaf(x[d].z, g, v[4 * d + 2] * f), v[4 * d + 3] = fmaf(x[d].w, g, v[4 * d + 3] * f);
    }
  }
  const bool none = top == -INFINITY && all == all;
  const float inv = 1.0f / all;
  const int64_t at = (int64_t)token * a.heads + index % a.kv_heads * a.group + r % a.group;
  T* out = static_cast<T*>(a.out) + at * D + d0;
#pragma unroll
  for (int d = 0; d < 32; d += 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = none ? 0u : pack2<T>(v[d + 2 * i] * inv, v[d + 2 * i + 1] * inv);
    *reinterpret_cast<uint4*>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (d0 == 0) a.lse[at] = none ? -INFINITY : top * kLn2 + logf(all);
}

// Every sequence's tokens fill whole items but its last: at most this many.
int64_t most_items(int64_t total_q, int64_t seqs, int tokens, int kv_heads) {
  return std::min<int64_t>(total_q / (2 * tokens) + seqs, total_q) * kv_heads;
}

// Parts of an item's keys. The lengths are on the device, so this goes by what the host
// knows: as many parts as give each SM one, of 4 blocks or more on average. Whole items
// against parts, 32 / 8 heads, D = 128: 200 tokens after 7800, 32 items, 111 us -> 47 with
// 4 parts (54 with two parts' items per SM, 67 with three); 512 after 1536, 72 items, 34 -> 31.
// With about an item per SM or more, parts gain nothing, and their sums (8 D bytes a row,
// written and read) cost: 7 chunks of 24 / 8 heads, D = 64, 264 items, 69.3 -> 71.5 with two parts; a prompt of 16384,
// 514 items, 481 -> 532.
int parts_for(int64_t items, int64_t total_k, int64_t seqs, int sms) {
  const int64_t blocks = total_k / std::max<int64_t>(seqs, 1) / kKeys;
  if (items <= 0 || 2 * items > sms || blocks < 8) return 1;
  return (int)std::min<int64_t>({sms / items, blocks / 4, 16});
}

constexpr size_t kTicketRegion = 16 << 10;  // the workspace's start is kept zero for the linears' tickets

template <typename T, int D>
int launch(const PromptArgs& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
           cudaStream_t st) {
  auto kern = prompt_attention_kernel<T, D>;
  static std::atomic<uint64_t> ready{0};
  GRINQH_RETURN_IF(allow_smem(reinterpret_cast<const void*>(kern), ready, Shape<D>::kSmem));
  const int64_t items = most_items(a.total_q, a.seqs, a.tokens, a.kv_heads) * a.parts;
  GRINQH_REQUIRE(items < (1LL << 31), "too many row blocks (%lld)", (long long)items);
  GRINQH_RETURN_IF(launch_dependent(kern, dim3((unsigned)items), kThreads, Shape<D>::kSmem, st, "prompt_attention", q,
                                    k, v, a));
  if (a.parts == 1) return GRINQH_OK;
  return launch_dependent(join_kernel<T, D>, dim3((unsigned)(items / a.parts * 2), D / 32), kRows, 0, st,
                          "prompt_attention (join)", a);
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

extern "C" size_t grinqh_prompt_attention_workspace_size(int64_t total_q, int64_t total_k, int num_seqs, int num_heads,
                                                         int num_kv_heads, int head_dim) {
  if (total_q <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      num_heads / num_kv_heads > kRows || num_heads <= 0)
    return 0;
  const int64_t items = most_items(total_q, num_seqs, kRows / (num_heads / num_kv_heads), num_kv_heads);
  const int parts = parts_for(items, total_k, num_seqs, sm_count());
  return parts == 1 ? 0 : kTicketRegion + (size_t)items * parts * 2 * sums_floats(head_dim) * sizeof(float);
}

extern "C" int grinqh_prompt_attention(const void* q, const void* k, const void* v, int dtype, int64_t total_q,
                                       int64_t total_k, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                       int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                       const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, float softmax_scale,
                                       void* out, float* lse, void* workspace, size_t workspace_bytes,
                                       grinqh_stream_t stream) {
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
  GRINQH_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 32) && q_token_stride % 8 == 0 &&
                     q_head_stride % 8 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                     v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                 "q, k, v and their strides must be 16-byte, out 32-byte aligned");
  const int group = num_heads / num_kv_heads;
  if (group > kRows)
    return set_error(GRINQH_ERR_UNSUPPORTED, "at most %d query heads per kv head (got %d)", kRows, group);
  PromptArgs a{};
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.out = out;
  a.lse = lse;
  a.total_q = (int)total_q;
  a.total_k = (int)total_k;
  a.seqs = num_seqs;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = group;
  a.tokens = kRows / group;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.wait_ns = attention_wait_ns();
  const int64_t items = most_items(total_q, num_seqs, a.tokens, num_kv_heads);
  a.parts = parts_for(items, total_k, num_seqs, sm_count());
  a.more = items * a.parts > sm_count();
  if (a.parts > 1) {
    const size_t need = grinqh_prompt_attention_workspace_size(total_q, total_k, num_seqs, num_heads, num_kv_heads,
                                                               head_dim);
    if (!workspace || workspace_bytes < need)
      return set_error(GRINQH_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, workspace_bytes);
    GRINQH_REQUIRE(aligned(workspace, 256), "workspace must be 256-byte aligned");
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketRegion);
  }
  const bool bf16 = dtype == GRINQH_BF16;
  CUtensorMap tq, tk, tv;
  GRINQH_RETURN_IF(tmap_heads(&tq, bf16, q, total_q, num_heads, head_dim, q_token_stride, q_head_stride, group,
                              a.tokens, "q"));
  if (total_k > 0) {
    GRINQH_RETURN_IF(tmap_heads(&tk, bf16, k, total_k, num_kv_heads, head_dim, k_token_stride, k_head_stride, 1, kKeys,
                                "k"));
    GRINQH_RETURN_IF(tmap_heads(&tv, bf16, v, total_k, num_kv_heads, head_dim, v_token_stride, v_head_stride, 1, kKeys,
                                "v"));
  } else {
    tk = tv = tq;  // never read: no row sees a key
  }
  if (head_dim == 128)
    return bf16 ? launch<__nv_bfloat16, 128>(a, tq, tk, tv, stream)
                : launch<__half, 128>(a, tq, tk, tv, stream);
  return bf16 ? launch<__nv_bfloat16, 64>(a, tq, tk, tv, stream) : launch<__half, 64>(a, tq, tk, tv, stream);
}
