// Attention of packed prompts of different lengths (sm_100a), keys and values packed or in pages.
//
// For query row t of a sequence with n new tokens and len keys, at position len - n + t:
//   s_j = scale q k_j over the keys it sees, p_j = 2^((s_j - m) log2 e), o = sum p_j v_j / sum p_j
// in one pass over tiles of 128 keys with a running reference m and sum per row.
//
// A work item is one key head and two query tiles of 128 rows: the rep = nq / nkv query heads of
// 128 / rep tokens ride side by side in a tile (row = token * rep + head), so the group's heads share
// every K and V tile and the causal edge cuts off 128 / rep tokens at a time, not 128. Warps of a CTA:
//   0-3, 4-7  softmax of query tile 0 and 1, one thread a row
//   8         one lane issues the tcgen05.mma: S_i = Q_i K^T (both in shared memory) and
//             O_i += P_i V (P in TMEM). A product of 128 x 128 x 16 runs for 64 cycles and is issued in 22
//             (66 where a branch around it keeps the operands out of uniform registers)
//   9         loads Q, and K and V tiles through a ring, by TMA with the 128-byte swizzle
//   10        zeroes the rows behind a sequence's last value
//   11        asks for the next item
// TMEM: S_0 | S_1 | O_0 | O_1; P_i overwrites S_i (16-bit, half its columns) as that is read. While one
// tile's softmax runs, the tensor core works for the other.
//
// A step (128 keys, both tiles) needs 2048 cycles of the tensor core at head_dim 128 and 2048 of the
// special-function unit, one exponential a score; it takes 3270, for each tile goes round a chain that
// nothing shortens: scores seen 300 cycles after their product, weights 1840, seen by the issuing lane 250
// to 400, products 790. Measured, bf16, 32 query and 8 key heads of 128, in a graph: 8191 causal tokens
// 422 us (1.30 PFLOP/s; 490 us under the power cap of minutes of it), 16 prompts of 1 to 1024 tokens 85 us,
// 48 tokens behind 16001 keys 33 us; fp16 541, 106 and 40 us, for its weights go out all at once. Tried and slower: two issuing warps (545 us: the tiles fall into step
// and meet at either unit), sixteen softmax warps with two threads a row (441), a part of the exponentials
// by polynomial (470: packed fp32 instructions take two issue slots), the output turned through shared
// memory (16 prompts 96 us), all weights announced at once (432 against 426), the maximum of every
// step (451).
#include <type_traits>  // integral_constant

#include "paged.cuh"
#include "tensor_core.cuh"

namespace mt {
namespace prompt {

using namespace tcore;
using paged::add2;
using paged::Elem;
using paged::fma2;
using paged::Pages;
using pipe::mbar_arrive;
using pipe::mbar_expect_tx;
using pipe::mbar_init;
using pipe::mbar_try_wait;

__device__ int g_prompt_error;  // set when a bounded wait expired (read through mt_read_error_word)

constexpr int kTile = 128;      // query rows of a tile and keys of a step
constexpr int kMmaWarp = 8, kLoadWarp = 9, kZeroWarp = 10, kFeedWarp = 11, kThreads = 384;
constexpr int kWalkers = 11;    // warps that take an item from the feed
constexpr int kTmemCols = 512;
// Far above a step's microseconds; the time that a warp spends on the slow path (row_again) does not count.
constexpr unsigned long long kDeadlineNs = 4000ull * 1000 * 1000;
// Softmax weights round to the values' type for the tensor core, by 2^-9 of themselves on average for bf16:
// with the rounding of the output that makes an error sqrt(2) times the output's alone. Calls of up to
// kFineRows rows (tokens_q * nq, rows of no sequence counted), single tokens for most, are as exact as the
// decode kernel (FINE): a weight is the sum of two 16-bit numbers, the second in the other half of the scores'
// columns. Measured in a graph, 32 heads, one number and two, bf16 (fp16): 16 tokens (512 rows) 7.0 and 8.2 us
// (7.5, 9.4), 24 tokens 7.4 and 8.6 (7.7, 9.6), one token of 16 sequences of 2000 keys 30 and 43 (37, 65), of 24
// sequences 55 and 78 (66, 122), 48 tokens behind 16001 keys 30 and 37 (33, 49). Single tokens have the decode
// kernel for speed; larger calls are not made to pay a sixth to four fifths more.
//
// The reference m that a row's exponentials are taken against need not be the largest score: weights far
// above 1 lose nothing in fp32 sums and 16-bit floating weights. It begins at the row's first score and
// moves when a step's weights add up to more than `most`, for the next step, which rescales the
// accumulator (seldom: the largest of many scores is rarely far above the first). No maximum is looked for.
//   bf16 weights have the range of fp32: scores that rise by 2^97 within one step leave an infinity, and
//   the item is taken once more, with the maximum of every step (kCareful).
//   fp16 weights end at 2^16: a step whose weights add up to more than `fits` is taken again with its
//   maximum, before the weights go out; they go out all at once.
// A move goes 2^kFarthest at the most, and the next step's the rest: ex2 makes a factor below 2^-126 zero, and a sum
// of 2^127, which is finite, would be lost with the accumulator.
constexpr float kSlack = 8.f, kFarthest = 120.f;
constexpr int kFineRows = 512;
template <typename T>
struct Reference {
  static constexpr bool kChecked = __is_same(T, __half);
  static constexpr float most = kChecked ? 256.f : 1073741824.f, fits = 32768.f;
};

struct Joined;
struct PromptArgs {
  const char* q;     // [tokens_q][nq][D]
  const char *k, *v; // [tokens_k][nkv][D] (packed form)
  char* out;         // [tokens_q][nq][D], contiguous
  const int *cu_q, *cu_k;
  int* status;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  int tokens_q, tokens_k, batch, nq, nkv, rep, causal;
  int tok;           // tokens of a query tile: 128 / rep
  float scale;       // scale * log2 e
  // where items may be cut along their keys: the most pieces there may be; per piece unnormalised outputs
  // [D / 8][256 rows][8] (a warp's 32 rows store whole lines), [256] references, [256] sums; and every
  // item's place for the join
  int units;
  float* parts;
  Joined* joined;
};

// Rows [first, first + n) of sequence b in a packed buffer of `tokens` rows; offsets outside the
// buffer or out of order leave an empty or a shorter sequence.
__device__ __forceinline__ void span_of(const int* cu, int b, int tokens, int& first, int& n) {
  first = min(max(cu[b], 0), tokens);
  n = max(min(cu[b + 1], tokens) - first, 0);
}

// What a warp is to do with what the feed lays out: an item; an item once more, now with the largest score of
// every step; nothing, there is no further one.
enum Mode { kItem, kCareful, kNone };

struct __align__(16) Item {
  int b, kh, q0, lq, k0, len;  // sequence, key head, its rows
  int t0;                      // first token of query tile 0
  int seen[2];                 // keys that query tile i's last row sees
  int j0, j1;                  // key tiles of this piece of the item: [j0, j1), as far as a query tile reads
  int mode;
};
// Key tiles of a query tile, and the keys that step j of them works on: 128, or 64 where the last
// tile holds no more.
__device__ __forceinline__ int tiles_of(int seen) { return (seen + kTile - 1) / kTile; }
__device__ __forceinline__ bool half_step(int seen, int j) { return seen - j * kTile <= kTile / 2; }

__device__ __forceinline__ int keys_seen(const PromptArgs& a, const Item& it, int t) {
  return a.causal ? min(max(it.len - it.lq + t + 1, 0), it.len) : it.len;
}

struct __align__(16) Joined {  // an item and the pieces it is cut into; 0 pieces: no such item
  Item it;
  int cut, pad[3];
};

// Tile pairs of a sequence of lq new tokens.
__device__ __forceinline__ int pairs_of(const PromptArgs& a, int lq) { return (lq + 2 * a.tok - 1) / (2 * a.tok); }

// The most items that a call can have, whatever its sequences' lengths: each of n that are not empty has a
// pair for its first row and one for every 2 tok of the others.
__host__ __device__ __forceinline__ long long items_most(const PromptArgs& a) {
  const int n = a.batch < a.tokens_q ? a.batch : a.tokens_q;
  return ((long long)(a.tokens_q - n) / (2 * a.tok) + n) * a.nkv;
}

// Finds flat item w = (query tile pair, key head); pairs in order of the sequences and, inside one,
// from its end, where a causal row sees most. By a converged warp; rising indices are found without a new
// start.
struct Finder {
  int first = 0;    // 32 sequences from here on are scanned next
  long before = 0;  // tile pairs of the sequences before `first`

  template <bool PAGED>
  __device__ bool find(const PromptArgs& a, const Pages& p, int lane, int w, Item& it) {
    const int pair = w / a.nkv;
    it.kh = w - pair * a.nkv;
    if (pair < before) first = 0, before = 0;
    for (; first < a.batch; first += 32) {
      int q0 = 0, lq = 0;
      if (first + lane < a.batch) span_of(a.cu_q, first + lane, a.tokens_q, q0, lq);
      int upto = pairs_of(a, lq);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > pair);
      if (past) {
        const int src = __ffs(past) - 1;
        it.b = first + src;
        it.q0 = __shfl_sync(0xffffffffu, q0, src);
        it.lq = __shfl_sync(0xffffffffu, lq, src);
        it.t0 = (int)(before + __shfl_sync(0xffffffffu, upto, src) - 1 - pair) * 2 * a.tok;
        it.k0 = 0;
        if (PAGED)
          it.len = paged::clamped_len(p, it.b, lane == 0 ? a.status : nullptr);
        else
          span_of(a.cu_k, it.b, a.tokens_k, it.k0, it.len);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = it.t0 + i * a.tok;
          it.seen[i] = t < it.lq ? keys_seen(a, it, min(t + a.tok, it.lq) - 1) : 0;
        }
        it.j0 = 0;
        it.j1 = tiles_of(max(it.seen[0], it.seen[1]));
        return true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
  }
};

// Pieces that every item is cut into along its keys, where there are fewer items than half the CTAs: as
// many as there are CTAs for, of three key tiles or more (a piece costs its accumulator's way through
// the workspace and a join, about two tiles). By a converged warp.
template <bool PAGED>
__device__ int pieces(const PromptArgs& a, const Pages& p, int lane) {
  int pairs = 0, longest = 0;  // pieces are cut where there are few pairs: 32 bits hold everything here
  for (int b = lane; b < a.batch; b += 32) {
    int first, lq, len;
    span_of(a.cu_q, b, a.tokens_q, first, lq);
    if (PAGED)
      len = paged::clamped_len(p, b, nullptr);
    else
      span_of(a.cu_k, b, a.tokens_k, first, len);
    pairs += pairs_of(a, lq);
    if (lq) longest = max(longest, len);
  }
  pairs = __reduce_add_sync(0xffffffffu, pairs);
  longest = __reduce_max_sync(0xffffffffu, longest);
  return max(1, min(a.units / max(pairs * a.nkv, 1), tiles_of(longest) / 3));
}

// Waits for a phase. Where that does not come, the kernel gives up: `dead` ends this and every later
// wait at once, and the warps run through what is left of their work, to no use but within bounds.
// dead[1] counts the warps on the slow path: half a second for 32 rows of 65536 keys, and it ends by itself.
// The clock is read in a function of its own: the waits of 20 places stay short (16 prompts 87.9 us with it
// in line, 85.9 without).
__device__ __noinline__ unsigned long long waited_long(unsigned long long since, volatile int* dead) {
  const unsigned long long now = globaltimer_ns();
  if (since == 0 || dead[1]) return now;
  if (now - since > kDeadlineNs) *dead = 1;
  return since;
}
__device__ __forceinline__ void wait_for(uint64_t* bar, unsigned parity, volatile int* dead) {
  unsigned long long since = 0;
  for (unsigned tries = 0; !mbar_try_wait(bar, parity); ++tries) {
    if (*dead) return;
    if (tries % 64 == 63) since = waited_long(since, dead);
  }
}
// For copies and matrix products in flight when the kernel gives up: bounded, whatever `dead` says.
__device__ __forceinline__ void drain(uint64_t* bar, unsigned parity) { (void)pipe::mbar_wait_bounded(bar, parity); }

// A tile multiplies masked weights (zeros) with values too: a value row that is not finite makes
// rows that must not see it NaN. A row that comes out non-finite from its item's second pass too is computed
// again, by one warp, from its own keys alone, so that it holds what its keys say.
template <typename T, int D, bool PAGED>
__device__ __noinline__ void row_again(const PromptArgs* args, const Pages* pages, int b, int kh, int k0, int seen,
                                       int row, int h) {
  constexpr int E = D / 32;
  const PromptArgs& a = *args;
  const Pages& p = *pages;
  const int lane = threadIdx.x & 31;
  const uint32_t* qp = reinterpret_cast<const uint32_t*>(a.q + (row * a.q_row + h * a.q_head) * 2) + lane * (E / 2);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const float2 f = Elem<T>::unpack(qp[e]);
    q[2 * e] = f.x * a.scale, q[2 * e + 1] = f.y * a.scale;
  }
  paged::row_attention<T, D>(q, seen, lane, [&](int j, const T*& k, const T*& v) {
    if (PAGED) {
      const long long page = paged::page_of(p, p.table + b * p.table_row, j, nullptr);
      const int slot = j & ((1 << p.shift) - 1);
      k = page < 0 ? nullptr : (const T*)p.k + page * p.k_page + kh * p.k_head + slot * p.k_row;
      v = page < 0 ? nullptr : (const T*)p.v + page * p.v_page + kh * p.v_head + slot * p.v_row;
    } else {
      k = (const T*)a.k + (k0 + j) * a.k_row + kh * a.k_head;
      v = (const T*)a.v + (k0 + j) * a.v_row + kh * a.v_head;
    }
  }, o);
  uint32_t* op = reinterpret_cast<uint32_t*>(a.out + ((long long)row * a.nq + h) * D * 2) + lane * (E / 2);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) op[e] = Elem<T>::pack(o[2 * e], o[2 * e + 1]);
}

// The warp's rows of a mask, a lane a row; `busy` counts the warps at it.
template <typename T, int D, bool PAGED>
__device__ __noinline__ void rows_again(const PromptArgs* args, const Pages* pages, int b, int kh, int k0, unsigned again,
                                        int seen, int row, int h, int* busy) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) atomicAdd(busy, 1);
  for (; again; again &= again - 1) {
    const int src = __ffs(again) - 1;
    row_again<T, D, PAGED>(args, pages, b, kh, k0, __shfl_sync(0xffffffffu, seen, src), __shfl_sync(0xffffffffu, row, src),
                           __shfl_sync(0xffffffffu, h, src));
  }
  if (lane == 0) atomicSub(busy, 1);
}

template <int N>
__device__ __forceinline__ void scale_columns(uint32_t at, float f) {
#pragma unroll
  for (int c = 0; c < N; c += 32) {
    uint32_t w[32];
    ld32(at + c, w);
    wait_ld();
    hold<32>(w);
#pragma unroll
    for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
    st32(at + c, w);
  }
}
// What is needed seldom, as functions of their own: in line they cost the loops around them registers (16
// prompts 88.6 us and 48 rows behind 16001 keys 36.6 with all three in line, 85.7 and 34.1 so). fp16, whose
// reference moves sooner, scales in line (12 windows 57.2 us
// otherwise, 56.1 so).
template <int N>
__device__ __noinline__ void scale_columns_seldom(uint32_t at, float f) {
  scale_columns<N>(at, f);
}
// The largest of this lane's scores in `cols` columns, of which the first `left` count.
__device__ __noinline__ float largest(uint32_t at, int cols, int left, float scale) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < cols; c += 32) {
    uint32_t w[32];
    ld32(at + c, w);
    wait_ld();
    hold<32>(w);
#pragma unroll
    for (int e = 0; e < 32; ++e) top = fmaxf(top, c + e < left ? __uint_as_float(w[e]) * scale : -INFINITY);
  }
  return top;
}

// All warps of a CTA, at the end: whether the last item is to be taken again.
__device__ __noinline__ bool goes_again(volatile int* dead, volatile int* flagged) {
  __syncwarp();
  pipe::named_sync(1, kThreads);
  return !*dead && *flagged;
}

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;                  // a tile is `halves` boxes of 64 elements a row
  static constexpr uint32_t kBox = kTile * 128;           // bytes of a box
  static constexpr uint32_t kTileBytes = kHalves * kBox;
  static constexpr int kStages = D == 128 ? 5 : 10;       // ring of K and V tiles
  static constexpr uint32_t kBytes = (2 + kStages) * kTileBytes + 1024;
};

template <typename T, int D, bool PAGED, bool SPLIT, bool FINE>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tiles(const __grid_constant__ PromptArgs a, const __grid_constant__ Pages p, const __grid_constant__ CUtensorMap qmap,
                 const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D>;
  constexpr int NS = L::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], s_full[2], p_most[2], p_full[2], o_full[2], o_free[2];
  __shared__ __align__(8) uint64_t kv_full[NS], kv_empty[NS], v_tail[NS], v_clean[NS], drained;
  __shared__ uint4 answer;  // which block's item comes next
  __shared__ Item item_s;
  __shared__ __align__(8) uint64_t answered, item_full, item_empty;
  __shared__ uint32_t tmem_s;
  __shared__ int dead_s[2], flagged_s[2];
  volatile int *dead = dead_s, *flagged = flagged_s;  // flagged: rows of item n & 1 came out infinite or NaN
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;  // Q_0, Q_1, then the ring
  const uint32_t ring = smem + 2 * L::kTileBytes;

  if (warp == kLoadWarp && lane < 3) prefetch_map(lane == 0 ? &qmap : lane == 1 ? &kmap : &vmap);
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                 "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 1);
        mbar_init(&s_full[i], 1);
        mbar_init(&p_most[i], 4);  // a lane of each softmax warp
        mbar_init(&p_full[i], 4);
        mbar_init(&o_full[i], 1);
        mbar_init(&o_free[i], 4);
      }
      for (int i = 0; i < NS; ++i) {
        mbar_init(&kv_full[i], 1);
        mbar_init(&kv_empty[i], 1);
        mbar_init(&v_tail[i], 1);
        mbar_init(&v_clean[i], 1);
      }
      mbar_init(&answered, 1);
      mbar_init(&item_full, 1);
      mbar_init(&item_empty, kWalkers);
      mbar_init(&drained, 1);
      dead_s[0] = dead_s[1] = flagged_s[0] = flagged_s[1] = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_s;
  pdl_wait();
  pdl_trigger();

  // 168 registers a thread at launch, three warpgroups: the softmax's two take from the third
  constexpr int kSoftmaxRegs = 200, kOtherRegs = 3 * 168 - 2 * kSoftmaxRegs;
  if (warp < kMmaWarp)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  Item it;
  unsigned taken = 0;  // items of this CTA so far
  // An item of which rows came out infinite or NaN is taken once more, with the largest score of every step as
  // its reference (kCareful): finite scores, however far they rise, then cost no more than a second pass. All
  // warps are done with item n - 2 when they have taken item n - 1, which the feed waits for before it lays out
  // item n. Only for the last one all wait, once each, before they leave.
  bool waited = false;
  auto last_flagged = [&](unsigned n) {  // whether item n goes round again, behind which there is no other
    waited = true;
    return goes_again(dead, &flagged[n & 1]);
  };
  // The next item, as the feed warp has laid it out; `leaving` runs where there may be none.
  auto next = [&](auto leaving) -> bool {
    while (true) {
      wait_for(&item_full, taken++ & 1, dead);
      const int4 *from = reinterpret_cast<const int4*>(&item_s);
      int4 *to = reinterpret_cast<int4*>(&it);
#pragma unroll
      for (int x = 0; x < 3; ++x) to[x] = from[x];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty);
      if (!*dead && it.mode != kNone) return true;
      leaving();
      if (waited || !last_flagged(taken - 2)) return false;
    }
  };
  if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ softmax, one thread a row
    const int i = warp >> 2, row = threadIdx.x & 127;
    const int rtok = row / a.rep, rhead = row - rtok * a.rep;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes (lane << 16)
    const uint32_t s_at = tmem + lanes + i * kTile, o_at = tmem + lanes + 2 * kTile + i * D;
    unsigned steps = 0, items = 0;
    // 2^(s k - m): a scale that is not positive is multiplied in first, so that the largest product
    // belongs to the largest score
    const bool plain = a.scale > 0.f;
    const float k = plain ? a.scale : 1.f;
    while (next([] {})) {
      const int t = it.t0 + i * a.tok + rtok;  // this row's token
      const bool live = rtok < a.tok && t < it.lq;
      const int n = min(tiles_of(it.seen[i]), it.j1), seen = live ? keys_seen(a, it, t) : 0;  // key tiles [j0, n)
      // tiles that end before the first row's last key need no mask (rows without a token never count)
      const int clear = it.seen[i] ? keys_seen(a, it, it.t0 + i * a.tok) / kTile : 0;
      float m = -INFINITY, l = 0.f;
      float last = 0.f;  // the sum of the last step's weights
      // One step: a tile of scores to weights. COLS of its keys, MASKED where a row sees fewer.
      auto step = [&](int j, auto cols, auto masked) {
        constexpr int COLS = decltype(cols)::value, NC = COLS / 32;
        constexpr bool MASKED = decltype(masked)::value;
        const int left = seen - j * kTile;  // this row's keys from this tile's first on
        auto score = [&](uint32_t w, int c) {
          float s = __uint_as_float(w);
          if (!plain) s *= a.scale;
          if constexpr (MASKED) s = c < left ? s : -INFINITY;
          return s;
        };
        auto move = [&](bool moves, float to) {  // of the rows that do, to another reference
          const float f = moves ? ex2(m - to) : 1.f;
          if (moves) m = to;
          l *= f;
          if (j == it.j0) return;
          // S of this step is there, so the product of the last one is done
          if constexpr (Reference<T>::kChecked)
            scale_columns<D>(o_at, f);
          else
            scale_columns_seldom<D>(o_at, f);
        };
        auto maximum = [&]() {
          return largest(s_at, COLS, MASKED ? left : kTile, plain ? 1.f : a.scale) * k;
        };
        const float2 k2 = make_float2(k, k);
        float2 sum[2];
        uint32_t sw[2][32];  // a chunk of scores and the next
        auto load = [&](int c) { ld32(s_at + 32 * c, sw[c & 1]); };
        auto arrived = [&](int c) {
          wait_ld();
          hold<32>(sw[c & 1]);
        };
        auto weights = [&](int c, float ref, uint32_t* pw, uint32_t* low) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int x = 32 * c + 2 * e;
            float2 v = fma2(make_float2(score(sw[c & 1][2 * e], x), score(sw[c & 1][2 * e + 1], x + 1)), k2,
                            make_float2(-ref, -ref));
            v.x = ex2(v.x);
            v.y = ex2(v.y);
            sum[e & 1] = add2(sum[e & 1], v);
            // the weights round to the values' type, as the tensor core wants them; the sum does not
            pw[e] = Elem<T>::pack(v.x, v.y);
            if constexpr (FINE) {
              const float2 hi = Elem<T>::unpack(pw[e]);
              low[e] = Elem<T>::pack(v.x - hi.x, v.y - hi.y);
            }
          }
        };
        auto announce = [&](uint64_t* bar) {
          wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
        auto total = [&]() { return (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y); };

        const bool far = live && last > Reference<T>::most;  // rows without a token hold anything
        if (__any_sync(0xffffffffu, far)) move(far, m + fminf(__log2f(last), kFarthest));
        load(0);
        arrived(0);
        if (j == it.j0) m = score(sw[0][0], 0) * k;
        // no key seen yet, or infinitely low ones: no reference to weigh the others against, this step's neither
        const bool careful = it.mode == kCareful;
        if (careful || __any_sync(0xffffffffu, live && left > 0 && m == -INFINITY)) {
          const float to = maximum();
          move((careful || m == -INFINITY) && to > m, to);
          load(0);
          arrived(0);
        }
        sum[0] = sum[1] = make_float2(0.f, 0.f);
        if constexpr (FINE) {
          if constexpr (Reference<T>::kChecked) {  // fp16: the maximum first, as there is time for it
            const float to = maximum();
            if (__any_sync(0xffffffffu, live && to - m > kSlack)) move(to - m > kSlack, to);
            load(0);
            arrived(0);
          }
          const float ref = m == -INFINITY ? 0.f : m;
          uint32_t low[NC][16];
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (c + 1 < NC) load(c + 1);
            uint32_t pw[16];
            weights(c, ref, pw, low[c]);
            st16(s_at + 16 * c, pw);  // over scores that are read
            if (c + 1 < NC) arrived(c + 1);
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) st16(s_at + kTile / 2 + 16 * c, low[c]);  // now all of them are
          announce(&p_most[i]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[i]);
        } else if constexpr (Reference<T>::kChecked) {
          uint32_t pw[COLS / 2];
#pragma unroll 1
          for (int taken_again = 0;; taken_again = 1) {
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              if (c + 1 < NC) load(c + 1);  // on its way meanwhile
              weights(c, ref, pw + 16 * c, nullptr);
              if (c + 1 < NC) arrived(c + 1);
            }
            if (taken_again || !__any_sync(0xffffffffu, live && total() > Reference<T>::fits)) break;
            const float to = maximum();
            move(to > m, to);
            sum[0] = sum[1] = make_float2(0.f, 0.f);
            load(0);
            arrived(0);
          }
#pragma unroll
          for (int c = 0; c < NC / 2; ++c) st32(s_at + 32 * c, pw + 32 * c);
          announce(&p_most[i]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[i]);
        } else {
          const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (c + 1 < NC) load(c + 1);  // on its way meanwhile
            uint32_t pw[16];
            weights(c, ref, pw, nullptr);
            // the first 64 keys' weights are announced a chunk late, when their store has long finished
            if (c == 2) announce(&p_most[i]);
            st16(s_at + 16 * c, pw);  // over scores that are read
            if (c + 1 < NC) {
              arrived(c + 1);
            } else {
              if (NC < 3) announce(&p_most[i]);
              announce(&p_full[i]);
            }
          }
        }
        last = total();
        l += last;
      };
      for (int j = it.j0; j < n; ++j, ++steps) {
        wait_for(&s_full[i], steps & 1, dead);
        fence_after();
        if (j < clear)
          step(j, std::integral_constant<int, kTile>{}, std::false_type{});
        else if (half_step(it.seen[i], j))
          step(j, std::integral_constant<int, kTile / 2>{}, std::true_type{});
        else
          step(j, std::integral_constant<int, kTile>{}, std::true_type{});
      }
      const int h = it.kh * a.rep + rhead;
      if constexpr (SPLIT) {
        // A piece: the accumulator, the reference and the sum. The join weighs pieces by their references, so a
        // power of two near the sum goes over to it: the largest weight may lie 2^127 above the reference.
        const int up = min(max((__float_as_int(l) >> 23 & 255) - 127, 0), (int)kFarthest);
        const float f = __int_as_float((127 - up) << 23);
        float* part = a.parts + (long long)blockIdx.x * (2 * kTile) * (D + 2);
        const int r = i * kTile + row;
        const bool none = n <= it.j0 || l == 0.f;  // nothing to add; -inf says so
        part[2 * kTile * D + r] = none ? -INFINITY : (m == -INFINITY ? 0.f : m) + up;
        part[2 * kTile * (D + 1) + r] = none ? 0.f : l * f;
        if (n <= it.j0) continue;
        wait_for(&o_full[i], items++ & 1, dead);
        fence_after();
        float2 odd2 = make_float2(l * 0.f, 0.f);  // as below
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t ow[32];
          ld32(o_at + 32 * c, ow);
          wait_ld();
          hold<32>(ow);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 zero = make_float2(0.f, 0.f);
            const float2 o = fma2(make_float2(__uint_as_float(ow[e]), __uint_as_float(ow[e + 1])), make_float2(f, f), zero);
            odd2 = fma2(o, zero, odd2);
            ow[e] = __float_as_uint(o.x), ow[e + 1] = __float_as_uint(o.y);
          }
          if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              store32(part + ((4 * c + e) * (2 * kTile) + r) * 8, reinterpret_cast<const uint32_t(&)[8]>(ow[8 * e]));
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[i]);
        // what is not finite even then is the join's to compute again
        if (__any_sync(0xffffffffu, live && !none && !(odd2.x + odd2.y == 0.f)) && it.mode == kItem && lane == 0)
          flagged[(taken - 1) & 1] = 1;
        continue;
      }
      char* dst = a.out + ((long long)(it.q0 + t) * a.nq + h) * D * 2;
      if (n == 0) {  // no key for any row of the tile
        if (live) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) store32(dst + 32 * c, {0, 0, 0, 0, 0, 0, 0, 0});
        }
        continue;
      }
      wait_for(&o_full[i], items++ & 1, dead);
      fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // not zero once an element, or the sum, is infinite or NaN; four chains
      float2 odd2[2] = {make_float2(l * 0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t ow[32];
        ld32(o_at + 32 * c, ow);
        wait_ld();
        hold<32>(ow);
        if (live) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // 32 bytes a store, the most there is: rows lie apart
            uint32_t w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float2 zero = make_float2(0.f, 0.f);
              const float2 f = fma2(make_float2(__uint_as_float(ow[16 * e + 2 * x]), __uint_as_float(ow[16 * e + 2 * x + 1])),
                                    make_float2(inv, inv), zero);
              odd2[x & 1] = fma2(f, zero, odd2[x & 1]);
              w[x] = Elem<T>::pack(f.x, f.y);
            }
            store32(dst + 64 * c + 32 * e, w);
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[i]);
      const float odd = (odd2[0].x + odd2[0].y) + (odd2[1].x + odd2[1].y);
      const unsigned again = __ballot_sync(0xffffffffu, live && !(odd == 0.f));
      if (again && it.mode == kCareful)
        rows_again<T, D, PAGED>(&a, &p, it.b, it.kh, it.k0, again, seen, it.q0 + t, h, &dead_s[1]);
      else if (again && lane == 0)
        flagged[(taken - 1) & 1] = 1;
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ tensor core
    constexpr uint32_t kType = __is_same(T, __half) ? 0u : 1u;
    constexpr uint32_t kScores = (1u << 4) | (kType << 7) | (kType << 10) | ((kTile >> 4) << 24);  // K as stored
    constexpr uint32_t kValues = kScores | (1u << 16) | ((D >> 3) << 17);  // V transposed: its rows run along N
    const bool leader = elect_one();
    const uint32_t tm = uniform(tmem);
    unsigned loads = 0, steps[2] = {0, 0}, items[2] = {0, 0}, tails = 0;  // `tails`: a bit a stage, v_clean's parity
    auto landed = [&](unsigned x) { wait_for(&kv_full[x % NS], (x / NS) & 1, dead); };
    auto scores = [&](int i, unsigned x, bool half) {
      const uint32_t idesc = kScores | ((half ? kTile / 2 : kTile) >> 3) << 17;
      const uint64_t qd = operand(smem + i * L::kTileBytes, 16), kd = operand(ring + (x % NS) * L::kTileBytes, 16);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const uint32_t at = ((d >> 2) * L::kBox + (d & 3) * 32) >> 4;
        mma_ss(leader, tm + i * kTile, qd + at, kd + at, idesc, d > 0);
      }
      commit(leader, &s_full[i]);
    };
    // the products' arrivals at the barriers end before the CTA does, and its TMEM is given back; the softmax
    // warps are at the last item's outputs meanwhile
    unsigned drains = 0;
    auto settle = [&]() {
      commit(leader, &drained);
      drain(&drained, drains++ & 1);
      __syncwarp();
    };
    while (next(settle)) {
      const int seen[2] = {uniform(it.seen[0]), uniform(it.seen[1])}, len = uniform(it.len);
      const int j0 = uniform(it.j0), j1 = uniform(it.j1);
      const int tiles[2] = {min(tiles_of(seen[0]), j1), min(tiles_of(seen[1]), j1)};  // key tiles [j0, tiles[i])
      if (j1 <= j0) continue;
      const unsigned base = loads;  // K, V, K, V, ... of the item
      loads += 2 * (j1 - j0);
      landed(base);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (tiles[i] <= j0) continue;
        wait_for(&q_full[i], items[i] & 1, dead);
        scores(i, base, half_step(seen[i], j0));
        if (tiles[i] == j0 + 1) commit(leader, &q_empty[i]);
      }
      commit(leader, &kv_empty[base % NS]);
      for (int j = j0; j < j1; ++j) {
        const unsigned vx = base + 2 * (j - j0) + 1, kx = vx + 1;
        landed(vx);
        if (j + 1 < j1) landed(kx);
        if (len - j * kTile < kTile) {
          wait_for(&v_clean[vx % NS], tails >> (vx % NS) & 1, dead);
          tails ^= 1u << (vx % NS);
        }
        const uint64_t vd = operand(ring + (vx % NS) * L::kTileBytes, L::kBox);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (j >= tiles[i]) continue;
          const uint32_t p_at = tm + i * kTile, o_at = tm + 2 * kTile + i * D;
          const bool more = j + 1 < tiles[i];
          auto values = [&](int x) {  // 16 keys
            mma_ts(leader, o_at, p_at + 8 * x, vd + x * (2048 >> 4), kValues, j > j0 || x > 0);
            if constexpr (FINE) mma_ts(leader, o_at, p_at + kTile / 2 + 8 * x, vd + x * (2048 >> 4), kValues, true);
          };
          const bool half = half_step(seen[i], j);
          if (j == j0) wait_for(&o_free[i], (items[i]++ & 1) ^ 1, dead);
          wait_for(&p_most[i], steps[i] & 1, dead);
          fence_after();
#pragma unroll
          for (int x = 0; x < 4; ++x) values(x);
          wait_for(&p_full[i], steps[i]++ & 1, dead);
          fence_after();
          if (!half) {
#pragma unroll
            for (int x = 4; x < 8; ++x) values(x);
          }
          if (more) {
            scores(i, kx, half_step(seen[i], j + 1));
            if (j + 2 == tiles[i]) commit(leader, &q_empty[i]);
          } else {
            commit(leader, &o_full[i]);
          }
        }
        commit(leader, &kv_empty[vx % NS]);
        if (j + 1 < j1) commit(leader, &kv_empty[kx % NS]);
      }
    }
  } else if (warp == kZeroWarp) {
    // ------------------------------------------------------------------ behind the last value
    // What lies there is not this sequence's: zero, or its weight of zero would make NaN of a NaN.
    // v_tail says that the load of such a tile is under way (kv_full alone would not say which of the
    // stage's loads it speaks of), v_clean that it is ready; the stage is not loaded again before that.
    unsigned loads = 0, tails = 0;
    while (next([] {})) {
      const int rows = it.len - (it.j1 - 1) * kTile;
      if (it.j1 <= it.j0) continue;
      loads += 2 * (it.j1 - it.j0);
      if (rows >= kTile) continue;
      const unsigned vx = loads - 1, st = vx % NS;
      wait_for(&v_tail[st], tails >> st & 1, dead);
      wait_for(&kv_full[st], (vx / NS) & 1, dead);
      tails ^= 1u << st;
      for (int x = rows * 8 + lane; x < kTile * 8; x += 32)
#pragma unroll
        for (int hf = 0; hf < L::kHalves; ++hf)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + st * L::kTileBytes + hf * L::kBox + x * 16),
                       "r"(0) : "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_clean[st]);
    }
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ loads
    unsigned loads = 0, items[2] = {0, 0};
    const int rows_q = a.tok * a.rep;
    while (next([] {})) {
      const int* table = PAGED ? p.table + it.b * p.table_row : nullptr;
      for (int j = it.j0; j < it.j1; ++j) {
        for (int kv = 0; kv < 2; ++kv, ++loads) {
          if (j == it.j0) {  // Q_0, K, Q_1, V: in the order of their use
            if (tiles_of(it.seen[kv]) > it.j0) {
              wait_for(&q_empty[kv], (items[kv]++ & 1) ^ 1, dead);
              if (elect_one()) {
                mbar_expect_tx(&q_full[kv], rows_q * 128 * L::kHalves);
#pragma unroll
                for (int hf = 0; hf < L::kHalves; ++hf)
                  tma_3d(smem + kv * L::kTileBytes + hf * L::kBox, &qmap, hf * 64, it.kh * a.rep,
                         it.q0 + it.t0 + kv * a.tok, &q_full[kv]);
              }
              __syncwarp();
            }
          }
          const unsigned st = loads % NS;
          wait_for(&kv_empty[st], ((loads / NS) & 1) ^ 1, dead);
          const CUtensorMap* map = kv ? &vmap : &kmap;
          const uint32_t dst = ring + st * L::kTileBytes;
          if (PAGED) {
            // one lane a box: the pages that hold keys of this tile, their halves
            const int per = min(1 << p.shift, kTile), left = min(kTile, it.len - j * kTile);
            const int boxes = (left + per - 1) / per;
            if (lane == 0) mbar_expect_tx(&kv_full[st], boxes * per * 128 * L::kHalves);
            __syncwarp();
            if (lane < boxes * L::kHalves) {
              const int box = lane / L::kHalves, hf = lane - box * L::kHalves, key = j * kTile + box * per;
              int page = paged::page_of(p, table, key, a.status);
              if (page < 0) page = p.pages;  // out of range: the box reads as zeros
              tma_4d(dst + hf * L::kBox + box * per * 128, map, hf * 64, key & ((1 << p.shift) - 1), it.kh, page,
                     &kv_full[st]);
            }
          } else if (elect_one()) {
            mbar_expect_tx(&kv_full[st], L::kTileBytes);
#pragma unroll
            for (int hf = 0; hf < L::kHalves; ++hf)
              tma_3d(dst + hf * L::kBox, map, hf * 64, it.kh, it.k0 + j * kTile, &kv_full[st]);
          }
          __syncwarp();
          if (kv && it.len - j * kTile < kTile && lane == 0) mbar_arrive(&v_tail[st]);
        }
      }
    }
    if (*dead) {  // copies in flight end before this CTA's shared memory does
      for (unsigned x = loads > NS ? loads - NS : 0; x < loads; ++x) drain(&kv_full[x % NS], (x / NS) & 1);
      for (int i = 0; i < 2; ++i)
        if (items[i]) drain(&q_full[i], (items[i] - 1) & 1);
    }
  } else {
    // ------------------------------------------------------------------ feed
    // The first item is this block's own. Each further one belongs to a block that then never starts:
    // a CTA that is done early takes more, with no counter in memory. It is asked for when all warps
    // have begun the last one, not sooner: what is taken early is work that no idle CTA can take.
    Finder finder;
    unsigned asked = 0;
    auto take = [&]() {  // a block that has not started, or -1, after which there is no asking again
      if (*dead) return -1;
      __syncwarp();  // all lanes have read the last answer
      if (lane == 0) {
        mbar_expect_tx(&answered, 16);
        take_block(&answer, &answered);
      }
      __syncwarp();
      wait_for(&answered, asked++ & 1, dead);
      const int block = *dead ? -1 : taken_block(&answer);
      // this lane's read comes before the next answer, which the asynchronous proxy writes to the same place
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      return block;
    };
    int w1 = -1, w2 = -1;  // the blocks of items n - 1 and n - 2
    bool ended = SPLIT;    // there is no block to ask for
    for (unsigned n = 0;; ++n) {
      int w = -1, cut = 1;
      if constexpr (SPLIT) cut = pieces<PAGED>(a, p, lane);
      it.mode = kItem;
      if (n == 0) {
        w = blockIdx.x / cut;
      } else {
        wait_for(&item_empty, (n - 1) & 1, dead);
        if (flagged[n & 1]) {
          w = w2;
          it.mode = kCareful;
          __syncwarp();
          if (lane == 0 && !waited) flagged[n & 1] = 0;  // (behind last_flagged others may still have to read it)
        }
      }
      bool none = w < 0 || !finder.find<PAGED>(a, p, lane, w, it);
      // Blocks without an item (sequences that are empty or fill their tiles leave some): taken too, each
      // would begin as a CTA of its own only to end. Measured: 16 prompts and 1008 empty sequences 623 us
      // without.
      while (none && !ended) {
        w = take();
        ended = w < 0;
        none = ended || !finder.find<PAGED>(a, p, lane, w, it);
      }
      if (none) it.mode = kNone;
      w2 = w1, w1 = w;
      if constexpr (SPLIT) {
        const int piece = blockIdx.x - w * cut, tiles = it.j1;
        it.j0 = (int)((unsigned)tiles * piece / (unsigned)cut);  // at most 2^24 tiles x 148 pieces
        it.j1 = (int)((unsigned)tiles * (piece + 1) / (unsigned)cut);
      }
      if (lane == 0) {
        item_s = it;
        mbar_arrive(&item_full);
      }
      if (SPLIT && n == 0 && blockIdx.x < items_most(a)) {  // beside it, this block's share of the list for the join
        Finder all;
        Joined* j = a.joined + blockIdx.x;
        Item listed;
        const bool there = all.find<PAGED>(a, p, lane, blockIdx.x, listed);
        if (lane == 0) {
          if (there) j->it = listed;
          j->cut = there ? cut : 0;
        }
      }
      if (none && (waited || !last_flagged(n - 1))) break;
    }
    if (*dead) drain(&answered, 0), drain(&answered, 1);
  }
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    if (dead_s[0] && lane == 0) atomicExch(&g_prompt_error, 1);
  }
}

// Joins the pieces of the items, a warp a row; D/8 lanes (32 bytes each) take one piece, the other lanes
// the next:  m = max m_i,
// o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.
constexpr int kJoinRows = 8;  // of a block
template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(32 * kJoinRows) prompt_join(const __grid_constant__ PromptArgs a, const __grid_constant__ Pages p) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kAtOnce = 8;
  pdl_wait();
  const int lane = threadIdx.x & 31, r = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
  const int cut = a.joined[blockIdx.x].cut;
  const Item it = a.joined[blockIdx.x].it;
  const int tile = r / kTile, rtok = (r % kTile) / a.rep, rhead = r % kTile - rtok * a.rep;
  const int t = it.t0 + tile * a.tok + rtok;
  if (cut == 0 || rtok >= a.tok || t >= it.lq) return;
  const int h = it.kh * a.rep + rhead, seen = keys_seen(a, it, t);
  const float* part = a.parts + (long long)blockIdx.x * cut * (2 * kTile) * (D + 2);
  const int sub = lane / kLanes, d8 = lane - sub * kLanes;
  // eight pieces at a time and group of lanes, all their loads under way at once
  float m = -INFINITY, l = 0.f, o[8] = {};
  for (int i0 = sub; i0 < cut; i0 += kAtOnce * kGroups) {
    float pm[kAtOnce], pl[kAtOnce], top = m;
    float4 po[kAtOnce][2];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      pm[n] = -INFINITY;
      if (i0 + n * kGroups < cut) {
        const float* x = part + (long long)(i0 + n * kGroups) * (2 * kTile) * (D + 2);
        const float4* y = reinterpret_cast<const float4*>(x + (d8 * (2 * kTile) + r) * 8);
        pm[n] = x[2 * kTile * D + r], pl[n] = x[2 * kTile * (D + 1) + r];
        po[n][0] = y[0], po[n][1] = y[1];
      }
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) top = fmaxf(top, pm[n]);
    const float ref = top == -INFINITY ? 0.f : top, keep = ex2(m - ref);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= keep;
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      if (pm[n] == -INFINITY) continue;  // no key there: nothing was written
      const float f = ex2(pm[n] - ref);
      const float* v = reinterpret_cast<const float*>(po[n]);
      l = fmaf(f, pl[n], l);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(f, v[e], o[e]);
    }
  }
#pragma unroll
  for (int x = kLanes; x < 32; x <<= 1) {  // the groups of lanes
    const float om = __shfl_xor_sync(0xffffffffu, m, x), top = fmaxf(m, om), ref = top == -INFINITY ? 0.f : top;
    const float f = ex2(m - ref), of = ex2(om - ref);
    l = l * f + __shfl_xor_sync(0xffffffffu, l, x) * of;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f + __shfl_xor_sync(0xffffffffu, o[e], x) * of;
    m = top;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float odd = l * 0.f;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = o[2 * e] * inv, y = o[2 * e + 1] * inv;
    odd = fmaf(x, 0.f, fmaf(y, 0.f, odd));
    w[e] = Elem<T>::pack(x, y);
  }
  if (__any_sync(0xffffffffu, !(odd == 0.f))) {
    row_again<T, D, PAGED>(&a, &p, it.b, it.kh, it.k0, seen, it.q0 + t, h);
    return;
  }
  if (sub == 0)
    *reinterpret_cast<uint4*>(a.out + (((long long)(it.q0 + t) * a.nq + h) * D + d8 * 8) * 2) =
        make_uint4(w[0], w[1], w[2], w[3]);
}

// Query map: boxes of 64 elements x rep heads x 128 / rep tokens. Keys and values: 64 elements x up to
// 128 rows of one head, of a page or of the packed rows.
template <typename T, int D, bool PAGED>
static cudaError_t launch_tiles(const PromptArgs& a, const Pages& p, cudaStream_t s, int flags) {
  using L = Layout<D>;
  constexpr bool fp16 = __is_same(T, __half);
  CUtensorMap qm, km, vm;
  const cuuint64_t qd[3] = {D, (cuuint64_t)a.nq, (cuuint64_t)a.tokens_q};
  const cuuint64_t qs[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_row * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)a.rep, (cuuint32_t)a.tok};
  bool ok = tensor_map(&qm, fp16, 3, a.q, qd, qs, qb);
  if (PAGED) {
    const cuuint64_t page = 1ull << p.shift;
    const cuuint64_t d[4] = {D, page, (cuuint64_t)p.heads, (cuuint64_t)p.pages};
    const cuuint64_t ks[3] = {(cuuint64_t)p.k_row * 2, (cuuint64_t)p.k_head * 2, (cuuint64_t)p.k_page * 2};
    const cuuint64_t vs[3] = {(cuuint64_t)p.v_row * 2, (cuuint64_t)p.v_head * 2, (cuuint64_t)p.v_page * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page < kTile ? page : kTile), 1, 1};
    ok = ok && tensor_map(&km, fp16, 4, p.k, d, ks, box) && tensor_map(&vm, fp16, 4, p.v, d, vs, box);
  } else {
    const cuuint64_t d[3] = {D, (cuuint64_t)a.nkv, (cuuint64_t)a.tokens_k};
    const cuuint64_t ks[2] = {(cuuint64_t)a.k_head * 2, (cuuint64_t)a.k_row * 2};
    const cuuint64_t vs[2] = {(cuuint64_t)a.v_head * 2, (cuuint64_t)a.v_row * 2};
    const cuuint32_t box[3] = {64, 1, kTile};
    ok = ok && tensor_map(&km, fp16, 3, a.k, d, ks, box) && tensor_map(&vm, fp16, 3, a.v, d, vs, box);
  }
  if (!ok) return cudaErrorInvalidValue;
  const bool fine = (long long)a.tokens_q * a.nq <= kFineRows;
  const auto kernel = a.parts ? (fine ? prompt_tiles<T, D, PAGED, true, true> : prompt_tiles<T, D, PAGED, true, false>)
                              : (fine ? prompt_tiles<T, D, PAGED, false, true> : prompt_tiles<T, D, PAGED, false, false>);
  const unsigned items = (unsigned)items_most(a);
  const cudaError_t e = launch(kernel, dim3(a.parts ? (unsigned)a.units : items), dim3(kThreads), L::kBytes, s, flags, a, p,
                               qm, km, vm);
  if (e != cudaSuccess || !a.parts) return e;
  return launch(prompt_join<T, D, PAGED>, dim3(items, 2 * kTile / kJoinRows), dim3(32 * kJoinRows), 0, s, flags | kFlagPdl,
                a, p);
}

template <bool PAGED>
static cudaError_t launch_prompt(const PromptArgs& a, const Pages& p, int d, int type, cudaStream_t s, int flags) {
  if (items_most(a) > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (type == 0)
    return d == 128 ? launch_tiles<__nv_bfloat16, 128, PAGED>(a, p, s, flags)
                    : launch_tiles<__nv_bfloat16, 64, PAGED>(a, p, s, flags);
  return d == 128 ? launch_tiles<__half, 128, PAGED>(a, p, s, flags) : launch_tiles<__half, 64, PAGED>(a, p, s, flags);
}

// Workspace bytes: pieces may be cut where there can be no more items than half the SMs, and keys
// enough for two pieces (six tiles).
static long long workspace_of(const PromptArgs& a, long long keys, int d) {
  if (2 * items_most(a) > sm_count() || keys <= 5 * kTile) return 0;
  return (long long)sm_count() * ((2 * kTile) * (d + 2) * sizeof(float) + sizeof(Joined));
}

static void cut_items(PromptArgs* a, void* workspace, int d) {
  if (!workspace) return;
  a->parts = (float*)workspace;
  a->joined = (Joined*)(a->parts + (long long)a->units * (2 * kTile) * (d + 2));
}

static bool query_ok(const void* q, int q_row, int q_head, const void* cu, int tokens, int nq, int nkv, const void* out) {
  return q && cu && out && tokens >= 1 && nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= 64 && q_row > 0 &&
         q_head > 0 && q_row % 8 == 0 && q_head % 8 == 0 && aligned(q, 16) && aligned(out, 32) && aligned(cu, 4);
}

}  // namespace prompt

cudaError_t prompt_error_word(int* value, bool clear) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, prompt::g_prompt_error, sizeof(int));
  if (e != cudaSuccess) return e;
  *value |= v;
  if (clear) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(prompt::g_prompt_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace mt

using namespace mt;

// Workspace bytes of the two calls below: of `batch` sequences with `tokens` query rows in all and up to
// `keys` keys each.
MT_API int mt_prompt_attention_workspace(int tokens, int batch, int keys, int nq, int nkv, int head_dim, long long* bytes) {
  if (!bytes || tokens < 0 || batch < 1 || keys < 0 || nkv < 1 || nq < 1 || nq % nkv || nq / nkv > 64) return kBadArgument;
  prompt::PromptArgs a = {};
  a.tokens_q = tokens, a.batch = batch, a.nkv = nkv, a.tok = prompt::kTile / (nq / nkv);
  *bytes = prompt::workspace_of(a, keys, head_dim);
  return 0;
}

// Attention of packed prompts over packed keys and values (see the header).
MT_API int mt_packed_attention(const void* q, int q_row, int q_head, const void* k, int k_row, int k_head, const void* v,
                               int v_row, int v_head, const void* cu_q, const void* cu_k, int batch, int tokens_q,
                               int tokens_k, int nq, int nkv, int head_dim, int type, int causal, float scale, void* out,
                               void* workspace, int flags, void* stream) {
  if (!prompt::query_ok(q, q_row, q_head, cu_q, tokens_q, nq, nkv, out) || !k || !v || !cu_k) return kBadArgument;
  if (batch < 1 || tokens_k < 1 || (head_dim != 64 && head_dim != 128) || (type != 0 && type != 1)) return kBadArgument;
  if (k_row < 1 || k_head < 1 || v_row < 1 || v_head < 1 || k_row % 8 || k_head % 8 || v_row % 8 || v_head % 8 ||
      !aligned(k, 16) || !aligned(v, 16) || !aligned(cu_k, 4) || !aligned(workspace, 32))
    return kBadArgument;
  if (!paged::apart(paged::span_of_rows(out, tokens_q, (long long)nq * head_dim, nq, head_dim, head_dim),
                    {paged::span_of_rows(q, tokens_q, q_row, nq, q_head, head_dim),
                     paged::span_of_rows(k, tokens_k, k_row, nkv, k_head, head_dim),
                     paged::span_of_rows(v, tokens_k, v_row, nkv, v_head, head_dim),
                     paged::span_of_ints(cu_q, batch + 1LL), paged::span_of_ints(cu_k, batch + 1LL)}))
    return kBadArgument;
  const int rep = nq / nkv;
  prompt::PromptArgs a{(const char*)q, (const char*)k, (const char*)v, (char*)out, (const int*)cu_q,
                       (const int*)cu_k, nullptr, q_row, q_head, k_row, k_head, v_row, v_head,
                       tokens_q, tokens_k, batch, nq, nkv, rep, causal != 0, prompt::kTile / rep,
                       scale * paged::kLog2e, sm_count(), nullptr, nullptr};
  if (prompt::workspace_of(a, tokens_k, head_dim)) prompt::cut_items(&a, workspace, head_dim);
  return prompt::launch_prompt<false>(a, paged::Pages{}, head_dim, type, (cudaStream_t)stream, flags);
}

// Causal attention of packed prompts over a paged cache (see the header).
MT_API int mt_paged_attention_prompt(const void* q, int q_row, int q_head, const mt_paged_kv* kv, const void* cu_seqlens,
                                     int tokens, int nq, float scale, void* out, void* workspace, void* status, int flags,
                                     void* stream) {
  paged::Pages p;
  if (!paged::pages_of(kv, &p) || !prompt::query_ok(q, q_row, q_head, cu_seqlens, tokens, nq, kv->heads, out) ||
      !aligned(workspace, 32))
    return kBadArgument;
  const int d = kv->head_dim;
  if (!paged::apart(paged::span_of_rows(out, tokens, (long long)nq * d, nq, d, d),
                    {paged::span_of_rows(q, tokens, q_row, nq, q_head, d), paged::span_of_pages(kv, false),
                     paged::span_of_pages(kv, true), paged::span_of_table(kv), paged::span_of_ints(kv->kv_lens, kv->batch),
                     paged::span_of_ints(cu_seqlens, kv->batch + 1LL)}))
    return kBadArgument;
  const int rep = nq / kv->heads;
  prompt::PromptArgs a{(const char*)q, nullptr, nullptr, (char*)out, (const int*)cu_seqlens, nullptr, (int*)status,
                       q_row, q_head, 0, 0, 0, 0, tokens, 0, kv->batch, nq, kv->heads, rep, 1,
                       prompt::kTile / rep, scale * paged::kLog2e, sm_count(), nullptr, nullptr};
  if (prompt::workspace_of(a, (long long)kv->max_pages * kv->page_size, kv->head_dim))
    prompt::cut_items(&a, workspace, kv->head_dim);
  return prompt::launch_prompt<true>(a, p, kv->head_dim, kv->type, (cudaStream_t)stream, flags);
}
