// Attention of one new token per sequence over a paged key-value cache (sm_100a).
//
//   s_j = scale q k_j,  p_j = 2^((s_j - m) log2 e),  o = sum p_j v_j / sum p_j      over all keys j
//
// Bound by HBM: every key and value row is read once, 4 D bytes for 4 D flops a query head. The work is
// cut into chunks of 64 keys of one key head (and up to 8 of its query heads), laid out one after the
// other over the sequences, and every CTA takes a run of chunks, wherever sequences begin and end: a
// batch of ragged sequences and one long sequence both load all SMs alike. A run that covers a
// sequence's head only in part leaves (m, l, o) in the workspace; a second kernel joins the parts,
//   m = max m_i,  o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i,
// in the order of the keys, so the same inputs give the same bits.
//
// Measured in a graph, bf16, pages of 64: 128 sequences of 256 to 4096 tokens, 8 key heads, 182 us
// (6.25 TB/s, 0.96 of the copy's rate); one of 32749 32 us (4.2 TB/s: 6 us until all SMs stream, 5 for
// the merge and the join); one of 2048 9.9 us, all of it latency (setup 2, first chunk 1.4, merge 1.6, join
// 3). With one CTA of eight warps an SM and runs of one length the same took 190, 36 and 14 us.
#include "paged.cuh"
#include "tensor_core.cuh"

namespace mt {
namespace paged {

using namespace tcore;
using pipe::mbar_arrive;
using pipe::mbar_expect_tx;
using pipe::mbar_init;
using pipe::mbar_wait_bounded;

__device__ int g_paged_error;  // set when a bounded wait expired (read through mt_read_error_word)

constexpr int kChunk = 64;      // keys of a chunk
constexpr int kHeads = 8;       // query heads of an item: rows 0-7 of the mma's 16 (8-15 take the
                                // low halves of the weights)
constexpr int kConsumers = 4;   // warps, 16 keys of a chunk each
constexpr int kDecodeThreads = (kConsumers + 1) * 32;
constexpr int kCtasPerSm = 2;   // one streams while the other begins or ends a run
// SMs do not get equal shares of HBM: with runs of one length the slowest of 148 ended 16% after the
// median. Large calls therefore have kRounds runs for every resident CTA, of falling length (shares of 64
// of the work), which the hardware hands out as CTAs end.
constexpr int kRounds = 6;
__constant__ int kShares[kRounds + 1] = {0, 28, 44, 53, 58, 61, 64};

// How `work` chunks are laid out in runs: `rounds` x `width`, none empty.
struct Plan {
  long work;
  int width, rounds;
  __device__ __forceinline__ Plan(long work, int runs, int rounds_most) : work(work) {
    width = runs / rounds_most;
    // the shortest round has 3/64 of the work
    rounds = rounds_most > 1 && work * 3 >= 64L * (width + 1) ? rounds_most : 1;
    if (work < width) width = (int)work;
  }
  __device__ __forceinline__ int runs() const { return rounds * width; }
  __device__ __forceinline__ long base(int round) const { return rounds == 1 ? (round ? work : 0) : work * kShares[round] / 64; }
  __device__ __forceinline__ long divide(long a, long b) const {  // both positive; 32 bits are much quicker
    return (unsigned long)a >> 32 ? a / b : (long)((unsigned)a / (unsigned)b);
  }
  __device__ __forceinline__ long start(int run) const {
    const int round = run / width, j = run - round * width;
    const long b = base(round);
    if (round == rounds) return work;
    const long n = base(round + 1) - b, per = divide(n, width);
    return b + j * per + min((long)j, n - per * width);
  }
  __device__ __forceinline__ int run_of(long chunk) const {
    int round = 0;
    while (round + 1 < rounds && base(round + 1) <= chunk) ++round;
    const long b = base(round), n = base(round + 1) - b, per = divide(n, width), longer = n - per * width;
    const long in = chunk - b, edge = longer * (per + 1);
    return round * width + (int)(in < edge ? divide(in, per + 1) : longer + divide(in - edge, per));
  }
};

struct DecodeArgs {
  const char* q;     // [batch][nq][D]
  char* out;         // [batch][nq][D], contiguous
  int* status;
  float* parts;      // [runs][2][kHeads][D + 2]: o, m, l
  int4* joins;       // [runs]: {first output row, heads, parts, -}: the item that starts in this run
                     // and ends in a later one; 0 parts where there is none
  long long q_row, q_head;
  int nq, rep, groups;  // groups of up to 8 query heads of a key head
  int rounds;           // at the most
  float scale;          // scale * log2 e
};

template <int D>
struct Ring {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kBox = kChunk * 128;  // 64 elements of a chunk's rows
  static constexpr uint32_t kStage = 2 * kHalves * kBox;  // K and V
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kRow = D + 8;  // floats of a merge row: the eight heads on banks of their own
  static constexpr uint32_t kMerge = (kConsumers - 1) * kHeads * kRow * 4;
  static constexpr uint32_t kBytes = kStages * kStage + kMerge + 1024;
};

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte piece `piece` of row r in a chunk: the 128-byte swizzle of its box.
__device__ __forceinline__ uint32_t swizzled(int r, int piece) {
  return (uint32_t)((piece >> 3) * (kChunk * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
}

// Chunks of a sequence; one even where it is empty, so that its rows get their zeros.
__device__ __forceinline__ int chunks_of(int len) { return len > kChunk ? (len + kChunk - 1) / kChunk : 1; }

// An item in a run: chunks [c0, c1) of sequence b for key head kh, query heads of `group`.
struct Run {
  int b, kh, group, len, chunks, c0, c1;
};

template <typename T, int D>
__global__ void __launch_bounds__(kDecodeThreads, kCtasPerSm)
    paged_decode(const __grid_constant__ DecodeArgs a, const __grid_constant__ Pages p,
                 const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using R = Ring<D>;
  constexpr int NS = R::kStages, NK = D / 16;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t full[NS], empty[NS];
  __shared__ long wsum[kConsumers + 1];
  __shared__ float wm[kConsumers][kHeads], wl[kConsumers][kHeads];
  __shared__ int dead_s;
  volatile int* dead = &dead_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
  float* merge = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)) + NS * R::kStage);  // [warp - 1][head][kRow]
  long* slab = reinterpret_cast<long*>(merge);  // chunks (of one head) of the sequences before thread t's slab

  if (warp == kConsumers && lane < 2) prefetch_map(lane ? &vmap : &kmap);
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    dead_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  // prefix sums of the sequences' chunks: a slab of consecutive sequences a thread
  const int per = (p.batch + kDecodeThreads - 1) / kDecodeThreads;
  long mine = 0;
  for (int b = tid * per; b < min((tid + 1) * per, p.batch); ++b)
    mine += chunks_of(clamped_len(p, b, blockIdx.x == 0 ? a.status : nullptr));
  long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) wsum[warp] = upto;
  __syncthreads();
  long total = 0;
#pragma unroll
  for (int w = 0; w <= kConsumers; ++w) {
    if (w < warp) upto += wsum[w];
    total += wsum[w];
  }
  slab[tid] = upto - mine;
  __syncthreads();

  const int per_seq = p.heads * a.groups;  // items of a sequence
  const Plan plan(total * per_seq, gridDim.x, a.rounds);
  const int run = blockIdx.x;
  if (run >= plan.runs()) {
    if (tid == 0) a.joins[run] = make_int4(0, 0, 0, 0);
    return;
  }
  const long w0 = plan.start(run), w1 = plan.start(run + 1);
  // the sequence and item of chunk w0: every warp by itself
  Run r;
  long at = w0;  // the run's position in the flat order
  {
    int t = 0;  // the last slab that starts at or before w0 and holds something
    for (int s = 0; s < kDecodeThreads; s += 32) {
      const int n = __popc(__ballot_sync(0xffffffffu, slab[s + lane] * per_seq <= w0));
      if (n) t = s + n - 1;
      if (n < 32) break;
    }
    long before = slab[t] * per_seq;
    int b = t * per;
    while (true) {
      r.len = clamped_len(p, b, nullptr);
      r.chunks = chunks_of(r.len);
      if (w0 < before + (long)r.chunks * per_seq || b + 1 >= p.batch) break;
      before += (long)r.chunks * per_seq;
      ++b;
    }
    r.b = b;
    const long in = w0 - before;
    const int item = (int)plan.divide(in, r.chunks);
    r.kh = item / a.groups;
    r.group = item - r.kh * a.groups;
    r.c0 = (int)(in - (long)item * r.chunks);
    r.c1 = (int)min((long)r.chunks, r.c0 + (w1 - w0));
  }
  __syncthreads();  // `merge` takes the slabs' place
  auto advance = [&]() {  // the next item, from its first chunk; false past the run's end
    at += r.c1 - r.c0;
    if (at >= w1 || (r.b + 1 >= p.batch && r.kh + 1 >= p.heads && r.group + 1 >= a.groups)) return false;
    if (++r.group == a.groups) {
      r.group = 0;
      if (++r.kh == p.heads) {
        r.kh = 0;
        ++r.b;
        r.len = clamped_len(p, r.b, nullptr);
        r.chunks = chunks_of(r.len);
      }
    }
    r.c0 = 0;
    r.c1 = (int)min((long)r.chunks, w1 - at);
    return true;
  };

  unsigned idx = 0;  // chunks of this run so far: stage idx % NS
  if (warp == kConsumers) {
    // -------------------------------------------------------------------- loads
    bool ok = true;
    const int rows = min(1 << p.shift, kChunk);           // of a box
    const int per_chunk = kChunk / rows;                  // boxes of a chunk, for either half of K and of V
    const int box = lane / (2 * R::kHalves), what = lane - box * 2 * R::kHalves;  // page, then half, K or V
    do {
      if (r.len == 0) continue;
      const int* table = p.table + r.b * p.table_row;
      int ids = 0, first = 1 << 30;  // a lane a box: the page ids of the 32 boxes from `first` on
      for (int c = r.c0; c < r.c1; ++c, ++idx) {
        const unsigned st = idx % NS;
        const int left = min(kChunk, r.len - c * kChunk), boxes = (left + rows - 1) / rows;
        if (c * per_chunk < first || (c + 1) * per_chunk > first + 32) {
          first = c * per_chunk;
          const int key = (first + lane) * rows;
          ids = key < r.len ? page_of(p, table, key, a.status) : 0;
          if (ids < 0) ids = p.pages;  // out of range: the box reads as zeros
        }
        const int page = __shfl_sync(0xffffffffu, ids, (c * per_chunk - first + box) & 31);
        if (!(ok = !*dead && mbar_wait_bounded(&empty[st], ((idx / NS) & 1) ^ 1))) break;
        if (lane == 0) mbar_expect_tx(&full[st], boxes * rows * 128 * 2 * R::kHalves);
        __syncwarp();
        if (box < boxes) {
          const int key = c * kChunk + box * rows, hf = what % R::kHalves, v = what / R::kHalves;
          tma_4d(ring + st * R::kStage + what * R::kBox + box * rows * 128, v ? &vmap : &kmap, hf * 64,
                 key & ((1 << p.shift) - 1), r.kh, page, &full[st]);
        }
        __syncwarp();
      }
    } while (ok && advance());
    if (!ok) {
      if (lane == 0) *dead = 1;
      for (unsigned x = idx > NS ? idx - NS : 0; x < idx; ++x) mbar_wait_bounded(&full[x % NS], (x / NS) & 1);
      if (lane == 0) atomicExch(&g_paged_error, 1);
    }
    return;
  }

  // ---------------------------------------------------------------------- attention
  const int g = lane >> 2, t4 = lane & 3;  // this lane's query head, and its keys 2 t4 (+1) of 8
  const int tok0 = 16 * warp;
  do {
    const int heads = min(kHeads, a.rep - r.group * kHeads), row0 = r.b * a.nq + r.kh * a.rep + r.group * kHeads;
    if (r.len == 0) {  // one chunk of nothing, always whole: zeros
      for (int x = tid; x < heads * D / 8; x += kConsumers * 32)
        reinterpret_cast<uint4*>(a.out + (long long)row0 * D * 2)[x] = make_uint4(0, 0, 0, 0);
      if (tid == 0 && at + 1 >= w1) a.joins[run] = make_int4(0, 0, 0, 0);
      continue;
    }
    uint32_t qa[NK][2];
    const char* qp = a.q + (r.b * a.q_row + (long long)(r.kh * a.rep + r.group * kHeads + g) * a.q_head) * 2;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      qa[kk][0] = g < heads ? *reinterpret_cast<const uint32_t*>(qp + 32 * kk + 4 * t4) : 0u;
      qa[kk][1] = g < heads ? *reinterpret_cast<const uint32_t*>(qp + 32 * kk + 4 * t4 + 16) : 0u;
    }
    float o[2 * NK][4] = {};
    float m = -INFINITY, l = 0.f;  // of head g; l over this lane's keys
    for (int c = r.c0; c < r.c1; ++c, ++idx) {
      const unsigned st = idx % NS;
      const int left = r.len - c * kChunk - tok0;  // keys of this warp's 16 and behind
      const bool got = !*dead && mbar_wait_bounded(&full[st], (idx / NS) & 1);
      if (!__all_sync(0xffffffffu, got)) {
        if (lane == 0) *dead = 1, atomicExch(&g_paged_error, 1);
      } else if (left > 0) {
        const uint32_t kb = ring + st * R::kStage, vb = kb + R::kHalves * R::kBox;
        if (left < 16) {
          // rows past the last key are not the sequence's: zero, or their weight of zero would make
          // NaN of a NaN
          for (int x = lane; x < (16 - left) * 8 * R::kHalves; x += 32) {
            const int hf = x / ((16 - left) * 8), rest = x - hf * (16 - left) * 8;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vb + hf * R::kBox + (tok0 + left) * 128 + rest * 16),
                         "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next load
          __syncwarp();
        }
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          uint32_t b[4];
          ldsm(b, kb + swizzled(tok0 + (lane & 7) + 8 * (lane >> 4), 2 * kk + ((lane >> 3) & 1)));
          mma16<T>(s[0], qa[kk][0], 0u, qa[kk][1], 0u, b[0], b[1]);
          mma16<T>(s[1], qa[kk][0], 0u, qa[kk][1], 0u, b[2], b[3]);
        }
        float x[4], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // keys 8 (e / 2) + 2 t4 + e % 2
          x[e] = 8 * (e >> 1) + 2 * t4 + (e & 1) < left ? s[e >> 1][e & 1] * a.scale : -INFINITY;
          mx = fmaxf(mx, x[e]);
        }
        // the reference follows the maximum when that is 2^8 above it (the sums are fp32)
        if (__any_sync(0xffffffffu, mx - m > 8.f)) {
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float to = fmaxf(m, mx), f = to == -INFINITY ? 1.f : ex2(m - to);
          m = to;
          l *= f;
#pragma unroll
          for (int jd = 0; jd < 2 * NK; ++jd)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[jd][e] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int jn = 0; jn < 2; ++jn) {
          const float p0 = ex2(x[2 * jn] - ref), p1 = ex2(x[2 * jn + 1] - ref);
          l += p0 + p1;
          // a weight as the sum of two 16-bit numbers, rows g and g + 8 of one product
          hi[jn] = Elem<T>::pack(p0, p1);
          const float2 h = Elem<T>::unpack(hi[jn]);
          lo[jn] = Elem<T>::pack(p0 - h.x, p1 - h.y);
        }
#pragma unroll
        for (int jp = 0; jp < NK; ++jp) {
          uint32_t b[4];
          ldsm_t(b, vb + swizzled(tok0 + (lane & 7) + 8 * ((lane >> 3) & 1), 2 * jp + (lane >> 4)));
          mma16<T>(o[2 * jp], hi[0], lo[0], hi[1], lo[1], b[0], b[1]);
          mma16<T>(o[2 * jp + 1], hi[0], lo[0], hi[1], lo[1], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    // the warps' parts of the item: each brings its own to the common reference, warp 0 adds up
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t4 == 0) wm[warp][g] = m, wl[warp][g] = l;
    pipe::named_sync(1, kConsumers * 32);
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) mm = fmaxf(mm, wm[w][g]);
    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) ll = fmaf(ex2(wm[w][g] - ref), wl[w][g], ll);
    const float f = ex2(m - ref);
    if (warp) {
      float* mine_o = merge + ((warp - 1) * kHeads + g) * R::kRow;
#pragma unroll
      for (int jd = 0; jd < 2 * NK; ++jd)
        *reinterpret_cast<float2*>(mine_o + 8 * jd + 2 * t4) =
            make_float2((o[jd][0] + o[jd][2]) * f, (o[jd][1] + o[jd][3]) * f);
    }
    pipe::named_sync(1, kConsumers * 32);
    if (warp == 0) {
      const bool whole = r.c0 == 0 && r.c1 == r.chunks;
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      float* part = a.parts + ((long long)run * 2 + (r.c0 == 0 ? 1 : 0)) * kHeads * (D + 2);
#pragma unroll
      for (int jd = 0; jd < 2 * NK; ++jd) {
        const int d = 8 * jd + 2 * t4;
        float x0 = (o[jd][0] + o[jd][2]) * f, x1 = (o[jd][1] + o[jd][3]) * f;
#pragma unroll
        for (int w = 0; w < kConsumers - 1; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(merge + (w * kHeads + g) * R::kRow + d);
          x0 += v.x;
          x1 += v.y;
        }
        if (g < heads) {
          if (whole)
            *reinterpret_cast<uint32_t*>(a.out + ((long long)(row0 + g) * D + d) * 2) = Elem<T>::pack(x0 * inv, x1 * inv);
          else
            *reinterpret_cast<float2*>(part + g * D + d) = make_float2(x0, x1);
        }
      }
      if (!whole && t4 == 0) part[kHeads * D + g] = mm, part[kHeads * D + kHeads + g] = ll;
      if (lane == 0 && at + (r.c1 - r.c0) >= w1)  // the run's last item: does it go on in the next ones?
        a.joins[run] = make_int4(row0, heads,
                                 r.c0 == 0 && r.c1 < r.chunks ? plan.run_of(at + r.chunks - 1) - run + 1 : 0, 0);
    }
    pipe::named_sync(1, kConsumers * 32);
  } while (advance());
}

// Joins the parts of the items that more than one run worked on: block column c the item that starts in
// run c. With a block row a query head, the block's warps take a share of the parts each (few items of
// many parts); with one row they take a head each (many items of two parts).
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_decode_join(const __grid_constant__ DecodeArgs a) {
  constexpr int E = D / 32;
  __shared__ float om[kJoinWarps], ol[kJoinWarps], oo[kJoinWarps][D];
  static_assert(kJoinWarps == 4, "the maximum below");
  pdl_wait();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 j = a.joins[c];
  if (j.z == 0) return;
  const bool shared = gridDim.y > 1;
  const int first = shared ? warp : 0, stride = shared ? kJoinWarps : 1;
  auto part = [&](int i) {  // the first in slot 1 of run c, the others in slot 0 of the next ones
    return a.parts + ((long long)(c + i) * 2 + (i == 0 ? 1 : 0)) * kHeads * (D + 2);
  };
  for (int h = shared ? blockIdx.y : warp; h < j.y; h += shared ? gridDim.y : kJoinWarps) {
    // eight parts at a time, all their loads under way at once
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int i0 = first; i0 < j.z; i0 += 8 * stride) {
      float pm[8], pl[8], po[8][E], top = m;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int i = i0 + n * stride;
        pm[n] = -INFINITY;
        if (i < j.z) {
          const float* x = part(i);
          pm[n] = x[kHeads * D + h], pl[n] = x[kHeads * D + kHeads + h];
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float2 v = *reinterpret_cast<const float2*>(x + h * D + lane * E + e);
            po[n][e] = v.x, po[n][e + 1] = v.y;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) top = fmaxf(top, pm[n]);
      const float ref = top == -INFINITY ? 0.f : top, keep = ex2(m - ref);
      m = top;
      l *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= keep;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (i0 + n * stride >= j.z) continue;
        const float f = ex2(pm[n] - ref);
        l = fmaf(f, pl[n], l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(f, po[n][e], o[e]);
      }
    }
    if (shared) {
      if (lane == 0) om[warp] = m, ol[warp] = l;
#pragma unroll
      for (int e = 0; e < E; ++e) oo[warp][lane * E + e] = o[e];
      __syncthreads();
      if (warp) return;
      const float top = fmaxf(fmaxf(om[0], om[1]), fmaxf(om[2], om[3])), ref = top == -INFINITY ? 0.f : top;
      l = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float f = ex2(om[w] - ref);
        l = fmaf(f, ol[w], l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(f, oo[w][lane * E + e], o[e]);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* op = reinterpret_cast<uint32_t*>(a.out + ((long long)(j.x + h) * D + lane * E) * 2);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) op[e] = Elem<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
  }
}

template <typename T, int D>
static cudaError_t launch_decode(const DecodeArgs& a, const Pages& p, int runs, cudaStream_t s, int flags) {
  constexpr bool fp16 = __is_same(T, __half);
  CUtensorMap km, vm;
  const cuuint64_t page = 1ull << p.shift;
  const cuuint64_t d[4] = {D, page, (cuuint64_t)p.heads, (cuuint64_t)p.pages};
  const cuuint64_t ks[3] = {(cuuint64_t)p.k_row * 2, (cuuint64_t)p.k_head * 2, (cuuint64_t)p.k_page * 2};
  const cuuint64_t vs[3] = {(cuuint64_t)p.v_row * 2, (cuuint64_t)p.v_head * 2, (cuuint64_t)p.v_page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)(page < kChunk ? page : kChunk), 1, 1};
  if (!tensor_map(&km, fp16, 4, p.k, d, ks, box) || !tensor_map(&vm, fp16, 4, p.v, d, vs, box))
    return cudaErrorInvalidValue;
  cudaError_t e = launch(paged_decode<T, D>, dim3(runs), dim3(kDecodeThreads), Ring<D>::kBytes, s, flags, a, p, km, vm);
  if (e != cudaSuccess) return e;
  return launch(paged_decode_join<T, D>, dim3(runs, a.rounds > 1 ? 1 : kHeads), dim3(32 * kJoinWarps), 0, s,
                flags | kFlagPdl, a);
}

// Rounds of a call: more than one where the items alone, or the lengths that the page table allows, give
// every resident CTA plenty to do.
static int rounds_of(long long items, long long most_chunks) {
  const long long resident = (long long)kCtasPerSm * sm_count();
  return items >= 2 * resident || most_chunks >= 64 * resident ? kRounds : 1;
}

}  // namespace paged

cudaError_t paged_error_word(int* value, bool clear) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, paged::g_paged_error, sizeof(int));
  if (e != cudaSuccess) return e;
  *value |= v;
  if (clear) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(paged::g_paged_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace mt

using namespace mt;

// Workspace bytes of mt_paged_attention_decode on the current device, whatever the sizes.
MT_API int mt_paged_attention_decode_workspace(long long* bytes) {
  if (!bytes) return kBadArgument;
  const long long runs = (long long)paged::kRounds * paged::kCtasPerSm * sm_count();
  *bytes = runs * (2 * paged::kHeads * (128 + 2) * sizeof(float) + sizeof(int4));
  return 0;
}

// Decode attention over pages (see the header).
MT_API int mt_paged_attention_decode(const void* q, int q_row, int q_head, const mt_paged_kv* kv, int nq, float scale,
                                     void* out, void* workspace, void* status, int flags, void* stream) {
  paged::Pages p;
  if (!q || !out || !workspace || !paged::pages_of(kv, &p) || nq < 1 || nq % kv->heads || nq / kv->heads > 64)
    return kBadArgument;
  if (q_row < 1 || q_head < 1 || q_row % 8 || q_head % 8 || !aligned(q, 16) || !aligned(out, 16) ||
      !aligned(workspace, 16))
    return kBadArgument;
  const int d = kv->head_dim;
  if (!paged::apart(paged::span_of_rows(out, kv->batch, (long long)nq * d, nq, d, d),
                    {paged::span_of_rows(q, kv->batch, q_row, nq, q_head, d), paged::span_of_pages(kv, false),
                     paged::span_of_pages(kv, true), paged::span_of_table(kv), paged::span_of_ints(kv->kv_lens, kv->batch)}))
    return kBadArgument;
  const int rep = nq / kv->heads, groups = (rep + paged::kHeads - 1) / paged::kHeads;
  const long long items = (long long)kv->batch * kv->heads * groups;
  const long long most = items * (((long long)kv->max_pages * kv->page_size + paged::kChunk - 1) / paged::kChunk);
  const long long resident = (long long)paged::kCtasPerSm * sm_count();
  const int rounds = paged::rounds_of(items, most), runs = (int)(rounds > 1 ? rounds * resident : most < resident ? most : resident);
  int4* joins = (int4*)workspace;
  const paged::DecodeArgs a{(const char*)q, (char*)out, (int*)status, (float*)(joins + paged::kRounds * resident), joins,
                            q_row, q_head, nq, rep, groups, rounds, scale * paged::kLog2e};
  const cudaStream_t s = (cudaStream_t)stream;
  if (kv->type == 0)
    return kv->head_dim == 128 ? paged::launch_decode<__nv_bfloat16, 128>(a, p, runs, s, flags)
                               : paged::launch_decode<__nv_bfloat16, 64>(a, p, runs, s, flags);
  return kv->head_dim == 128 ? paged::launch_decode<__half, 128>(a, p, runs, s, flags)
                             : paged::launch_decode<__half, 64>(a, p, runs, s, flags);
}
