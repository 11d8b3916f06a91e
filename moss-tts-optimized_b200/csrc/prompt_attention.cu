// Attention of packed prompts of different lengths (sm_100a), keys and values packed or in pages.
#include "paged.cuh"

namespace mt {
namespace prompt {

using paged::Elem;
using paged::Pages;

struct PromptArgs {
  const char* q;     // [tokens_q][nq][D]
  const char *k, *v; // [tokens_k][nkv][D] (packed form)
  char* out;         // [tokens_q][nq][D], contiguous
  const int *cu_q, *cu_k;
  int* status;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  int tokens_q, tokens_k, batch, nq, rep, causal;
  float scale;       // scale * log2 e
};

// Rows [first, first + n) of sequence b in a packed buffer of `tokens` rows; offsets outside the
// buffer or out of order leave an empty or a shorter sequence.
__device__ __forceinline__ void span_of(const int* cu, int b, int tokens, int& first, int& n) {
  first = min(max(cu[b], 0), tokens);
  n = max(min(cu[b + 1], tokens) - first, 0);
}

// One warp a (token, query head).
template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(128) prompt_rows(PromptArgs a, Pages p) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.nq) return;
  const int b = paged::sequence_of(a.cu_q, a.batch, t, lane);
  if (b >= a.batch) return;
  int q0, nq_rows, k0 = 0, len;
  span_of(a.cu_q, b, a.tokens_q, q0, nq_rows);
  if (t < q0) return;
  int* status = lane == 0 ? a.status : nullptr;
  if (PAGED)
    len = paged::clamped_len(p, b, status);
  else
    span_of(a.cu_k, b, a.tokens_k, k0, len);
  const int keys = a.causal ? min(max(len - nq_rows + (t - q0) + 1, 0), len) : len;
  const int kh = h / a.rep;
  const uint32_t* qp = reinterpret_cast<const uint32_t*>(a.q + (t * a.q_row + h * a.q_head) * 2) + lane * (E / 2);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const float2 f = Elem<T>::unpack(qp[e]);
    q[2 * e] = f.x * a.scale, q[2 * e + 1] = f.y * a.scale;
  }
  paged::row_attention<T, D>(q, keys, lane, [&](int j, const T*& k, const T*& v) {
    if (PAGED) {
      const long long page = paged::page_of(p, p.table + b * p.table_row, j, status);
      const int slot = j & ((1 << p.shift) - 1);
      k = page < 0 ? nullptr : (const T*)p.k + page * p.k_page + kh * p.k_head + slot * p.k_row;
      v = page < 0 ? nullptr : (const T*)p.v + page * p.v_page + kh * p.v_head + slot * p.v_row;
    } else {
      k = (const T*)a.k + (k0 + j) * a.k_row + kh * a.k_head;
      v = (const T*)a.v + (k0 + j) * a.v_row + kh * a.v_head;
    }
  }, o);
  uint32_t* op = reinterpret_cast<uint32_t*>(a.out + ((long long)t * a.nq + h) * D * 2) + lane * (E / 2);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) op[e] = Elem<T>::pack(o[2 * e], o[2 * e + 1]);
}

template <typename T, bool PAGED>
static cudaError_t launch_prompt(const PromptArgs& a, const Pages& p, int d, cudaStream_t s, int flags) {
  const dim3 grid((unsigned)a.tokens_q, (unsigned)((a.nq + 3) / 4));
  return d == 128 ? launch(prompt_rows<T, 128, PAGED>, grid, dim3(128), 0, s, flags, a, p)
                  : launch(prompt_rows<T, 64, PAGED>, grid, dim3(128), 0, s, flags, a, p);
}

static bool query_ok(const void* q, int q_row, int q_head, const void* cu, int tokens, int nq, int nkv, const void* out) {
  return q && cu && out && tokens >= 1 && nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= 64 && q_row > 0 &&
         q_head > 0 && q_row % 8 == 0 && q_head % 8 == 0 && aligned(q, 16) && aligned(out, 16) && aligned(cu, 4);
}

}  // namespace prompt
}  // namespace mt

using namespace mt;

// Attention of packed prompts over packed keys and values (see the header).
MT_API int mt_packed_attention(const void* q, int q_row, int q_head, const void* k, int k_row, int k_head, const void* v,
                               int v_row, int v_head, const void* cu_q, const void* cu_k, int batch, int tokens_q,
                               int tokens_k, int nq, int nkv, int head_dim, int type, int causal, float scale, void* out,
                               int flags, void* stream) {
  if (!prompt::query_ok(q, q_row, q_head, cu_q, tokens_q, nq, nkv, out) || !k || !v || !cu_k) return kBadArgument;
  if (batch < 1 || tokens_k < 1 || (head_dim != 64 && head_dim != 128) || (type != 0 && type != 1)) return kBadArgument;
  if (k_row < 1 || k_head < 1 || v_row < 1 || v_head < 1 || k_row % 8 || k_head % 8 || v_row % 8 || v_head % 8 ||
      !aligned(k, 16) || !aligned(v, 16) || !aligned(cu_k, 4))
    return kBadArgument;
  const prompt::PromptArgs a{(const char*)q, (const char*)k, (const char*)v, (char*)out, (const int*)cu_q,
                             (const int*)cu_k, nullptr, q_row, q_head, k_row, k_head, v_row, v_head,
                             tokens_q, tokens_k, batch, nq, nq / nkv, causal != 0, scale * paged::kLog2e};
  const paged::Pages none = {};
  const cudaStream_t s = (cudaStream_t)stream;
  return type == 0 ? prompt::launch_prompt<__nv_bfloat16, false>(a, none, head_dim, s, flags)
                   : prompt::launch_prompt<__half, false>(a, none, head_dim, s, flags);
}

// Causal attention of packed prompts over a paged cache (see the header).
MT_API int mt_paged_attention_prompt(const void* q, int q_row, int q_head, const mt_paged_kv* kv, const void* cu_seqlens,
                                     int tokens, int nq, float scale, void* out, void* status, int flags, void* stream) {
  paged::Pages p;
  if (!paged::pages_of(kv, &p) || !prompt::query_ok(q, q_row, q_head, cu_seqlens, tokens, nq, kv->heads, out))
    return kBadArgument;
  const prompt::PromptArgs a{(const char*)q, nullptr, nullptr, (char*)out, (const int*)cu_seqlens, nullptr, (int*)status,
                             q_row, q_head, 0, 0, 0, 0, tokens, 0, kv->batch, nq, nq / kv->heads, 1,
                             scale * paged::kLog2e};
  const cudaStream_t s = (cudaStream_t)stream;
  return kv->type == 0 ? prompt::launch_prompt<__nv_bfloat16, true>(a, p, kv->head_dim, s, flags)
                       : prompt::launch_prompt<__half, true>(a, p, kv->head_dim, s, flags);
}
