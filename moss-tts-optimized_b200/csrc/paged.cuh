// Shared pieces of the paged key-value cache's kernels (sm_100a): 16-bit element types, where a
// key's row lies (in pages or packed), which sequence a packed token belongs to, packed fp32 arithmetic, and the attention
// of one query row by one warp.
#pragma once
#include <cuda_fp16.h>

#include <initializer_list>

#include "common.cuh"

namespace mt {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;  // softmax in powers of two: e^x = 2^(x log2 e)
constexpr int kStatusPosition = 1;  // a length or position outside the page table or the rope tables
constexpr int kStatusPage = 3;      // a page id outside the cache

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(bf16_lo(w), bf16_hi(w)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// One layer's pages, as mt_paged_kv with the element strides of a page, a head and a row.
struct Pages {
  char* k;
  char* v;
  long long k_page, k_head, k_row, v_page, v_head, v_row;
  const int* table;    // [batch][table_row]
  const int* lens;     // [batch]
  long long table_row;
  int pages, heads, shift, max_pages, batch;  // page size 1 << shift
};

// Tokens of sequence b that the page table can hold, at most its length.
__device__ __forceinline__ int clamped_len(const Pages& p, int b, int* status) {
  const int len = p.lens[b];
  const long long cap = (long long)p.max_pages << p.shift;
  if (len < 0 || len > cap) {
    if (status) atomicExch(status, kStatusPosition);
    return len < 0 ? 0 : (int)cap;
  }
  return len;
}

// The page of key j of a sequence whose row of the page table is `row`; -1 where the table names
// no page of the cache.
__device__ __forceinline__ int page_of(const Pages& p, const int* row, int j, int* status) {
  const int id = row[j >> p.shift];
  if ((unsigned)id >= (unsigned)p.pages) {
    if (status) atomicExch(status, kStatusPage);
    return -1;
  }
  return id;
}

// The sequence that holds packed token t: the first b with cu[b + 1] > t, or `batch` past the last
// one. 32 probes a round by the lanes of a (converged) warp, so 2 rounds up to 1024 sequences.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int t, int lane) {
  int lo = 0, n = batch;  // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step + step - 1;  // the last sequence of this lane's share
    const bool past = at < lo + n && cu[at + 1] <= t;
    const int whole = __popc(__ballot_sync(0xffffffffu, past));
    const int next = lo + whole * step;
    n = min(step - 1, lo + n - next);
    lo = next;
  }
  return lo;
}

// softmax(scale q k^T) v of one query row over keys 0..n-1 by one warp, lane l holding elements
// [l D/32, (l + 1) D/32) of q (scaled by scale * log2 e), k, v and the result. Keys past n are not
// read, nor keys behind one that leaves nothing but NaN. `rows(j, k, v)` gives key j's rows, null for a page
// that is not there (zeros).
template <typename T, int D, typename Rows>
__device__ __forceinline__ void row_attention(const float (&q)[D / 32], int n, int lane, Rows rows,
                                              float (&o)[D / 32]) {
  constexpr int E = D / 32;
  constexpr int kAtOnce = 4;  // keys whose rows are on their way at once
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int j0 = 0; j0 < n; j0 += kAtOnce) {
    uint32_t kw[kAtOnce][E / 2], vw[kAtOnce][E / 2];
    float s[kAtOnce], mn = m;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const T *kr = nullptr, *vr = nullptr;
      if (j0 + x < n) rows(j0 + x, kr, vr);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        kw[x][e] = kr ? reinterpret_cast<const uint32_t*>(kr)[lane * (E / 2) + e] : 0u;
        vw[x][e] = vr ? reinterpret_cast<const uint32_t*>(vr)[lane * (E / 2) + e] : 0u;
      }
    }
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      s[x] = 0.f;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float2 kf = Elem<T>::unpack(kw[x][e]);
        s[x] = fmaf(q[2 * e], kf.x, fmaf(q[2 * e + 1], kf.y, s[x]));
      }
      s[x] = warp_sum(s[x]);
      if (j0 + x >= n) s[x] = -INFINITY;
      mn = fmaxf(mn, s[x]);
    }
    const float ref = mn == -INFINITY ? 0.f : mn, keep = exp2f(m - ref);
    m = mn;
    l *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= keep;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const float p = exp2f(s[x] - ref);
      l += p;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float2 vf = Elem<T>::unpack(vw[x][e]);
        o[2 * e] = fmaf(p, vf.x, o[2 * e]);
        o[2 * e + 1] = fmaf(p, vf.y, o[2 * e + 1]);
      }
    }
    bool settled = true;  // once all is NaN it stays so
#pragma unroll
    for (int e = 0; e < E; ++e) settled = settled && o[e] != o[e];
    if (__all_sync(0xffffffffu, settled || l != l)) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] *= inv;
}

// Host: the kernels' form of a caller's mt_paged_kv; false where a field is not supported.
static inline bool pages_of(const mt_paged_kv* kv, Pages* p) {
  if (!kv || !kv->k_pages || !kv->v_pages || !kv->page_table || !kv->kv_lens) return false;
  if (kv->pages < 1 || kv->heads < 1 || kv->max_pages < 1 || kv->batch < 1) return false;
  if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1))) return false;
  if (kv->head_dim != 64 && kv->head_dim != 128) return false;
  if (kv->type != 0 && kv->type != 1) return false;
  if ((long long)kv->max_pages * kv->page_size > (1LL << 30)) return false;
  const long long strides[6] = {kv->k_page_stride, kv->k_head_stride, kv->k_row_stride,
                                kv->v_page_stride, kv->v_head_stride, kv->v_row_stride};
  for (long long s : strides)
    if (s < 1 || s % 8 || s >= (1LL << 39)) return false;
  if (!aligned(kv->k_pages, 16) || !aligned(kv->v_pages, 16) || !aligned(kv->page_table, 4) ||
      !aligned(kv->kv_lens, 4) || kv->table_stride < 0)
    return false;
  p->k = (char*)kv->k_pages;
  p->v = (char*)kv->v_pages;
  p->k_page = kv->k_page_stride;
  p->k_head = kv->k_head_stride;
  p->k_row = kv->k_row_stride;
  p->v_page = kv->v_page_stride;
  p->v_head = kv->v_head_stride;
  p->v_row = kv->v_row_stride;
  p->table = (const int*)kv->page_table;
  p->lens = (const int*)kv->kv_lens;
  p->table_row = kv->table_stride;
  p->pages = kv->pages;
  p->heads = kv->heads;
  p->shift = __builtin_ctz((unsigned)kv->page_size);
  p->max_pages = kv->max_pages;
  p->batch = kv->batch;
  return true;
}

// Host: the bytes from an operand's first element to its last.
struct Span {
  const char *first, *past;
};
static inline Span span_of_bytes(const void* p, long long bytes) { return {(const char*)p, (const char*)p + (p ? bytes : 0)}; }
// Rows of heads of d 16-bit elements.
static inline Span span_of_rows(const void* p, long long rows, long long row, long long heads, long long head, int d) {
  return span_of_bytes(p, 2 * ((rows - 1) * row + (heads - 1) * head + d));
}
static inline Span span_of_pages(const mt_paged_kv* kv, bool values) {
  const long long last = values ? (kv->pages - 1) * kv->v_page_stride + (kv->heads - 1) * kv->v_head_stride +
                                      (kv->page_size - 1) * kv->v_row_stride
                                : (kv->pages - 1) * kv->k_page_stride + (kv->heads - 1) * kv->k_head_stride +
                                      (kv->page_size - 1) * kv->k_row_stride;
  return span_of_bytes(values ? kv->v_pages : kv->k_pages, 2 * (last + kv->head_dim));
}
static inline Span span_of_table(const mt_paged_kv* kv) {
  return span_of_bytes(kv->page_table, 4 * ((kv->batch - 1) * kv->table_stride + kv->max_pages));
}
static inline Span span_of_ints(const void* p, long long n) { return span_of_bytes(p, 4 * n); }
// Whether what is written lies apart from all that is read: rows are read by other blocks than the one that
// writes them, and some a second time.
static inline bool apart(Span written, std::initializer_list<Span> read) {
  for (const Span& r : read)
    if (r.first < written.past && written.first < r.past) return false;
  return true;
}

}  // namespace paged
}  // namespace mt
