// Write of new tokens into a paged key-value cache (sm_100a): per head RMSNorm, rotate-half rotary
// position, the query rows out and the key and value rows into their pages, for packed tokens of
// sequences of different lengths.
//
//   y = x / sqrt(mean(x^2) + eps) * w        r_i = y_i cos_i -+ y_(i +- D/2) sin_i
//
// Everything between the 16-bit input and output is fp32 and rounds once, at the store.
#include "paged.cuh"

namespace mt {
namespace paged {

struct WriteArgs {
  const char* qkv;      // [tokens][(nq + 2 nkv) D], rows qkv_row elements apart
  const char *qw, *kw;  // [D]
  const char *cos_tab, *sin_tab;  // [table_rows][D]
  const int* cu;        // [batch + 1], or null: token t is sequence t's only one
  char* q_out;          // [tokens][nq][D]
  int* status;
  long long qkv_row;
  int tokens, nq, table_rows;
  float eps;
};

constexpr int kThreads = 128;
// Heads that a thread has on their way at once. Measured in a graph, 3357 rows of 48 heads and 4 rows: with 6
// 18.4 and 3.4 us, with 3 18.8 and 2.7, with 2 20.9 and 2.6 (64 threads: the same). What bounds the many rows
// is the chain of look-ups and the instructions of a head (issue slots 68% full), at 4.4 TB/s.
constexpr int kAhead = 3;

// Bound by HBM. A CTA has one token's kAhead x kGroups heads: D/8 lanes hold one head (16 bytes each), so the mean of squares is
// a shuffle inside the group and the rotation's partner element, D/2 away, is in the lane (D/8)/2
// away. The heads' loads are issued before the token's sequence, position and page are looked up (four
// loads, one after the other).
template <typename T, typename Tab, int D>
__global__ void __launch_bounds__(kThreads) qk_rope_paged(WriteArgs a, Pages p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int group = threadIdx.x / kLanes, sub = threadIdx.x % kLanes;
  const int heads = a.nq + 2 * p.heads;
  pdl_wait();
  pdl_trigger();
  const char* src = a.qkv + ((long long)t * a.qkv_row + sub * 8) * 2;
  uint4 raw[kAhead];
  auto load = [&](int h0) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int h = h0 + n * kGroups + group;
      raw[n] = h < heads ? *reinterpret_cast<const uint4*>(src + (long long)h * D * 2) : make_uint4(0, 0, 0, 0);
    }
  };
  const int h0 = blockIdx.y * (kAhead * kGroups);
  load(h0);
  const uint4 qv = *reinterpret_cast<const uint4*>(a.qw + sub * 16), kv = *reinterpret_cast<const uint4*>(a.kw + sub * 16);
  const int b = a.cu ? sequence_of(a.cu, p.batch, t, lane) : t;
  if (b >= p.batch || (a.cu && a.cu[b] > t)) return;  // behind the last sequence
  const int len = p.lens[b];
  char* qo = a.q_out + ((long long)t * a.nq * D + sub * 8) * 2;
  if (!a.cu && len == 0) {  // an empty slot of a step: no token, so zeros for its query and nothing in the pages
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int h = h0 + n * kGroups + group;
      if (h < a.nq) *reinterpret_cast<uint4*>(qo + (long long)h * D * 2) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int pos = a.cu ? len - a.cu[b + 1] + t : len - 1;
  if (pos < 0 || pos >= a.table_rows || (pos >> p.shift) >= p.max_pages) {
    if (a.status && threadIdx.x == 0) atomicExch(a.status, kStatusPosition);
    return;
  }
  const int page = page_of(p, p.table + (long long)b * p.table_row, pos, threadIdx.x == 0 ? a.status : nullptr);
  const int slot = pos & ((1 << p.shift) - 1);

  float c[8], s[8];
  if constexpr (sizeof(Tab) == 4) {
    const float4* cp = reinterpret_cast<const float4*>(a.cos_tab + ((long long)pos * D + sub * 8) * 4);
    const float4* sp = reinterpret_cast<const float4*>(a.sin_tab + ((long long)pos * D + sub * 8) * 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 cv = cp[i], sv = sp[i];
      c[4 * i] = cv.x, c[4 * i + 1] = cv.y, c[4 * i + 2] = cv.z, c[4 * i + 3] = cv.w;
      s[4 * i] = sv.x, s[4 * i + 1] = sv.y, s[4 * i + 2] = sv.z, s[4 * i + 3] = sv.w;
    }
  } else {
    const uint4 cv = *reinterpret_cast<const uint4*>(a.cos_tab + ((long long)pos * D + sub * 8) * 2);
    const uint4 sv = *reinterpret_cast<const uint4*>(a.sin_tab + ((long long)pos * D + sub * 8) * 2);
    const uint32_t cw[4] = {cv.x, cv.y, cv.z, cv.w}, sw[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 cf = Elem<T>::unpack(cw[i]), sf = Elem<T>::unpack(sw[i]);
      c[2 * i] = cf.x, c[2 * i + 1] = cf.y, s[2 * i] = sf.x, s[2 * i + 1] = sf.y;
    }
  }
  const float sign = sub < kLanes / 2 ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] *= sign;
  char* ko = p.k + (page * p.k_page + slot * p.k_row + sub * 8) * 2;
  char* vo = p.v + (page * p.v_page + slot * p.v_row + sub * 8) * 2;
#pragma unroll
  for (int n = 0; n < kAhead; ++n) {
    const int h = h0 + n * kGroups + group;
    if (h0 + n * kGroups + group / (32 / kLanes) * (32 / kLanes) >= a.nq + p.heads) {  // the warp holds values only
      if (page >= 0 && h < heads) *reinterpret_cast<uint4*>(vo + (h - a.nq - p.heads) * p.v_head * 2) = raw[n];
      continue;
    }
    // every lane takes part in the shuffles
    const uint32_t w[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
    float2 x[4], ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = Elem<T>::unpack(w[i]);
      ss = fma2(x[i], x[i], ss);
    }
    float sq = ss.x + ss.y;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float inv = rsqrtf(fmaf(sq, 1.f / D, a.eps));
    const uint4 nv = h < a.nq ? qv : kv;
    const uint32_t nw[4] = {nv.x, nv.y, nv.z, nv.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack(nw[i]), zero = make_float2(0.f, 0.f);
      x[i] = fma2(fma2(x[i], make_float2(inv, inv), zero), f, zero);
      const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, x[i].x, kLanes / 2),
                                   __shfl_xor_sync(0xffffffffu, x[i].y, kLanes / 2));
      const float2 z = fma2(x[i], make_float2(c[2 * i], c[2 * i + 1]),
                            fma2(y, make_float2(s[2 * i], s[2 * i + 1]), zero));
      r[i] = Elem<T>::pack(z.x, z.y);
    }
    const uint4 out = make_uint4(r[0], r[1], r[2], r[3]);
    if (h < a.nq)
      *reinterpret_cast<uint4*>(qo + (long long)h * D * 2) = out;
    else if (page >= 0 && h < a.nq + p.heads)
      *reinterpret_cast<uint4*>(ko + (h - a.nq) * p.k_head * 2) = out;
    else if (page >= 0 && h < heads)  // values as they are
      *reinterpret_cast<uint4*>(vo + (h - a.nq - p.heads) * p.v_head * 2) = raw[n];
  }
}

template <typename T, typename Tab>
static cudaError_t launch_write(const WriteArgs& a, const Pages& p, int d, cudaStream_t s, int flags) {
  const int heads = a.nq + 2 * p.heads, of_block = kAhead * kThreads * 8 / d;
  const dim3 grid(a.tokens, (heads + of_block - 1) / of_block);
  return d == 128 ? launch(qk_rope_paged<T, Tab, 128>, grid, dim3(kThreads), 0, s, flags, a, p)
                  : launch(qk_rope_paged<T, Tab, 64>, grid, dim3(kThreads), 0, s, flags, a, p);
}

}  // namespace paged
}  // namespace mt

using namespace mt;

// Head norm, rotary position and page write of packed new tokens (see the header).
MT_API int mt_qk_rope_paged(const void* qkv, const void* q_norm, const void* k_norm, const void* cos_tab,
                            const void* sin_tab, int table_rows, int table_fp32, const mt_paged_kv* kv,
                            const void* cu_seqlens, int tokens, int nq, int qkv_row, void* q_out, float eps,
                            void* status, int flags, void* stream) {
  paged::Pages p;
  if (!qkv || !q_norm || !k_norm || !cos_tab || !sin_tab || !q_out || !paged::pages_of(kv, &p)) return kBadArgument;
  if (table_rows < 1 || tokens < 1 || nq < 1 || qkv_row % 8 || (!cu_seqlens && tokens != kv->batch))
    return kBadArgument;
  if (qkv_row < (long long)(nq + 2LL * kv->heads) * kv->head_dim || nq + 2LL * kv->heads > (1 << 20)) return kBadArgument;
  const void* wide[6] = {qkv, q_norm, k_norm, cos_tab, sin_tab, q_out};
  for (const void* x : wide)
    if (!aligned(x, 16)) return kBadArgument;
  const int d = kv->head_dim;
  const long long table = (long long)table_rows * d * (table_fp32 ? 4 : 2);
  const paged::Span pages[2] = {paged::span_of_pages(kv, false), paged::span_of_pages(kv, true)};
  const paged::Span rows = paged::span_of_rows(q_out, tokens, (long long)nq * d, nq, d, d);
  for (const paged::Span& written : {rows, pages[0], pages[1]})
    if (!paged::apart(written, {paged::span_of_bytes(qkv, 2 * ((tokens - 1LL) * qkv_row + (nq + 2LL * kv->heads) * d)),
                                paged::span_of_bytes(q_norm, 2 * d), paged::span_of_bytes(k_norm, 2 * d),
                                paged::span_of_bytes(cos_tab, table), paged::span_of_bytes(sin_tab, table),
                                paged::span_of_table(kv), paged::span_of_ints(kv->kv_lens, kv->batch),
                                paged::span_of_ints(cu_seqlens, kv->batch + 1LL)}))
      return kBadArgument;
  if (!paged::apart(rows, {pages[0], pages[1]})) return kBadArgument;
  const paged::WriteArgs a{(const char*)qkv,     (const char*)q_norm, (const char*)k_norm, (const char*)cos_tab,
                           (const char*)sin_tab, (const int*)cu_seqlens, (char*)q_out,   (int*)status,
                           qkv_row,              tokens,              nq,                  table_rows,
                           eps};
  const cudaStream_t s = (cudaStream_t)stream;
  if (kv->type == 0)
    return table_fp32 ? paged::launch_write<__nv_bfloat16, float>(a, p, kv->head_dim, s, flags)
                      : paged::launch_write<__nv_bfloat16, __nv_bfloat16>(a, p, kv->head_dim, s, flags);
  return table_fp32 ? paged::launch_write<__half, float>(a, p, kv->head_dim, s, flags)
                    : paged::launch_write<__half, __half>(a, p, kv->head_dim, s, flags);
}
