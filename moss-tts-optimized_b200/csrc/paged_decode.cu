// Attention of one new token per sequence over a paged key-value cache (sm_100a).
#include "paged.cuh"

namespace mt {
namespace paged {

struct DecodeArgs {
  const char* q;  // [batch][nq][D]
  char* out;      // [batch][nq][D], contiguous
  int* status;
  long long q_row, q_head;
  int nq, rep;
  float scale;    // scale * log2 e
};

// One warp a query head.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_decode_rows(DecodeArgs a, Pages p) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, b = blockIdx.y, h = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (h >= a.nq) return;
  const int kh = h / a.rep, len = clamped_len(p, b, lane == 0 ? a.status : nullptr);
  const int* row = p.table + b * p.table_row;
  const uint32_t* qp = reinterpret_cast<const uint32_t*>(a.q + (b * a.q_row + h * a.q_head) * 2) + lane * (E / 2);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const float2 f = Elem<T>::unpack(qp[e]);
    q[2 * e] = f.x * a.scale, q[2 * e + 1] = f.y * a.scale;
  }
  row_attention<T, D>(q, len, lane, [&](int j, const T*& k, const T*& v) {
    const long long page = page_of(p, row, j, lane == 0 ? a.status : nullptr);
    const int slot = j & ((1 << p.shift) - 1);
    k = page < 0 ? nullptr : (const T*)p.k + page * p.k_page + kh * p.k_head + slot * p.k_row;
    v = page < 0 ? nullptr : (const T*)p.v + page * p.v_page + kh * p.v_head + slot * p.v_row;
  }, o);
  uint32_t* op = reinterpret_cast<uint32_t*>(a.out + ((long long)b * a.nq + h) * D * 2) + lane * (E / 2);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) op[e] = Elem<T>::pack(o[2 * e], o[2 * e + 1]);
}

}  // namespace paged
}  // namespace mt

using namespace mt;

// Decode attention over pages (see the header).
MT_API int mt_paged_attention_decode(const void* q, int q_row, int q_head, const mt_paged_kv* kv, int nq, float scale,
                                     void* out, void* status, int flags, void* stream) {
  paged::Pages p;
  if (!q || !out || !paged::pages_of(kv, &p) || nq < 1 || nq % kv->heads || nq / kv->heads > 64) return kBadArgument;
  if (q_row < 1 || q_head < 1 || q_row % 8 || q_head % 8 || !aligned(q, 16) || !aligned(out, 16)) return kBadArgument;
  const paged::DecodeArgs a{(const char*)q, (char*)out, (int*)status, q_row, q_head, nq, nq / kv->heads,
                            scale * paged::kLog2e};
  const dim3 grid((unsigned)((nq + 3) / 4), (unsigned)kv->batch);
  if (kv->batch > 65535) return kBadArgument;
  auto k = kv->type == 0 ? (kv->head_dim == 128 ? paged::paged_decode_rows<__nv_bfloat16, 128>
                                                : paged::paged_decode_rows<__nv_bfloat16, 64>)
                         : (kv->head_dim == 128 ? paged::paged_decode_rows<__half, 128>
                                                : paged::paged_decode_rows<__half, 64>);
  return launch(k, grid, dim3(128), 0, (cudaStream_t)stream, flags, a, p);
}
