// Attention of a chunk of new tokens over a paged cache: prompt chunks,
// drafted tokens to verify and single tokens, ragged in one batch.
//
// O_i = sum_j softmax_j(q_i . k_j s) v_j over the keys j that row i sees; row i
// of sequence b stands at position len_b - n_b + i.  First form: one warp per
// (token, query head) walks the keys with the running maximum and sum of the
// softmax in fp32.
#include "common.cuh"
#include "profile.cuh"

#include <string>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

struct ChunkParams {
  const char* q;
  int64_t q_tok, q_head;  // bytes
  const int32_t* q_indptr;
  int64_t num_tokens;
  const char* kv;
  int64_t s_page, s_kv, s_head, s_tok;  // bytes
  int64_t num_pages, num_page_entries;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last;
  char* out;
  int64_t o_tok, o_head;  // bytes
  float* lse;
  int64_t l_tok, l_head;  // elements
  int B, Hq, Hkv, group, P, causal;
  float scale_log2;
};

constexpr int kWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) chunk_rows_kernel(const ChunkParams p) {
  constexpr int N = D / 32;  // values of a row per lane
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= p.num_tokens * p.Hq) return;
  const int64_t tok = row / p.Hq;
  const int h = (int)(row - tok * p.Hq), kvh = h / p.group;
  int lo = 0, hi = p.B - 1;  // the last b with q_indptr[b] <= tok
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(p.q_indptr + mid) <= tok) lo = mid; else hi = mid - 1;
  }
  const int64_t a0 = __ldg(p.q_indptr + lo), a1 = __ldg(p.q_indptr + lo + 1);
  const int s = __ldg(p.indptr + lo), e = __ldg(p.indptr + lo + 1);
  int64_t keys = 0;
  if (tok < __ldg(p.q_indptr) || tok >= __ldg(p.q_indptr + p.B)) {
    // padding: no sequence
  } else if (a0 < 0 || tok < a0 || tok >= a1 || a1 > p.num_tokens || s < 0 || e < s || e > p.num_page_entries) {
    if (lane == 0) record_status(kStatusBadIndptr);
  } else if (e > s) {
    const int64_t len = (int64_t)(e - s - 1) * p.P + min(max(__ldg(p.last + lo), 0), p.P);
    keys = p.causal ? max((int64_t)0, len - (a1 - a0) + (tok - a0) + 1) : len;
  }
  float q[N], o[N];
  const T* qr = reinterpret_cast<const T*>(p.q + tok * p.q_tok + h * p.q_head);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = Elem<T>::to_float(qr[lane + 32 * i]) * p.scale_log2;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j0 = 0; j0 < keys; j0 += p.P) {
    const int page = __ldg(p.indices + s + j0 / p.P);
    const bool bad = page < 0 || page >= p.num_pages;  // reads as zeros
    if (bad && lane == 0) record_status(kStatusBadPage);
    const char* k = p.kv + (bad ? 0 : (int64_t)page * p.s_page + kvh * p.s_head);
    const int n = (int)min((int64_t)p.P, keys - j0);
    for (int t = 0; t < n; ++t, k += bad ? 0 : p.s_tok) {
      const T* kr = reinterpret_cast<const T*>(k);
      const T* vr = reinterpret_cast<const T*>(k + p.s_kv);
      float x = 0.f;
      if (!bad) {
#pragma unroll
        for (int i = 0; i < N; ++i) x = fmaf(q[i], Elem<T>::to_float(kr[lane + 32 * i]), x);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const float m2 = fmaxf(m, x), a = fast_exp2(m - m2), w = fast_exp2(x - m2);
      m = m2;
      l = l * a + w;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = bad ? o[i] * a : fmaf(w, Elem<T>::to_float(vr[lane + 32 * i]), o[i] * a);
    }
  }
  T* orow = reinterpret_cast<T*>(p.out + tok * p.o_tok + h * p.o_head);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) orow[lane + 32 * i] = Elem<T>::from_float(o[i] * inv);
  if (p.lse && lane == 0) p.lse[tok * p.l_tok + h * p.l_head] = l > 0.f ? (m + __log2f(l)) * kLn2 : -INFINITY;
}

int check_args(const akt_chunk_paged_args* a) {
  if (a->batch < 0 || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->page_size <= 0 || a->num_tokens < 0 ||
      a->num_pages < 0 || a->num_page_entries < 0)
    return set_error(AKT_ERR_INVALID, "chunk_paged: bad sizes");
  if (a->num_qo_heads % a->num_kv_heads)
    return set_error(AKT_ERR_INVALID, "num_qo_heads must be a multiple of num_kv_heads");
  if (a->dtype != AKT_FLOAT16 && a->dtype != AKT_BFLOAT16) return set_error(AKT_ERR_INVALID, "dtype");
  if (a->head_dim != 64 && a->head_dim != 128)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: head_dim must be 64 or 128");
  if (!(a->softmax_scale > 0.f) || a->softmax_scale == INFINITY)
    return set_error(AKT_ERR_INVALID, "chunk_paged: softmax_scale must be positive and finite");
  if (a->num_tokens > 0x7fffffff / a->num_qo_heads || a->num_page_entries > 0x7fffffff / a->page_size)
    return set_error(AKT_ERR_INVALID, "chunk_paged: too many tokens");
  if (a->num_tokens == 0) return AKT_OK;
  if (!a->q || !a->out || !a->q_indptr || !a->kv_page_indptr || !a->kv_last_page_len ||
      (a->num_page_entries > 0 && (!a->kv_page_indices || !a->kv_cache)))
    return set_error(AKT_ERR_INVALID, "chunk_paged: missing tensor");
  if (a->batch == 0) return set_error(AKT_ERR_INVALID, "chunk_paged: tokens without sequences");
  if (a->q_stride_dim != 1 || a->kv_stride_dim != 1 || a->out_stride_dim != 1)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: unit dim stride required");
  return AKT_OK;
}

template <typename T>
int launch(const ChunkParams& p, int D, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.num_tokens * p.Hq + kWarps - 1) / kWarps);
  {
    ProfileScope prof(st);
    if (D == 64) chunk_rows_kernel<T, 64><<<grid, kWarps * 32, 0, st>>>(p);
    else chunk_rows_kernel<T, 128><<<grid, kWarps * 32, 0, st>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : set_error(AKT_ERR_CUDA, std::string("chunk_paged: ") + cudaGetErrorString(e));
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" size_t akt_chunk_paged_workspace_size(const akt_chunk_paged_args* a) { return 0; }

extern "C" int akt_chunk_paged(const akt_chunk_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  const int rc = check_args(a);
  if (rc || a->num_tokens == 0) return rc;
  ChunkParams p{};
  p.q = static_cast<const char*>(a->q);
  p.q_tok = a->q_stride_token * 2;
  p.q_head = a->q_stride_head * 2;
  p.q_indptr = a->q_indptr;
  p.num_tokens = a->num_tokens;
  p.kv = static_cast<const char*>(a->kv_cache);
  p.s_page = a->kv_stride_page * 2;
  p.s_kv = a->kv_stride_kv * 2;
  p.s_head = a->kv_stride_head * 2;
  p.s_tok = a->kv_stride_token * 2;
  p.num_pages = a->num_pages;
  p.num_page_entries = a->num_page_entries;
  p.indptr = a->kv_page_indptr;
  p.indices = a->kv_page_indices;
  p.last = a->kv_last_page_len;
  p.out = static_cast<char*>(a->out);
  p.o_tok = a->out_stride_token * 2;
  p.o_head = a->out_stride_head * 2;
  p.lse = a->lse;
  p.l_tok = a->lse_stride_token;
  p.l_head = a->lse_stride_head;
  p.B = a->batch;
  p.Hq = a->num_qo_heads;
  p.Hkv = a->num_kv_heads;
  p.group = p.Hq / p.Hkv;
  p.P = a->page_size;
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->softmax_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->dtype == AKT_FLOAT16 ? launch<__half>(p, a->head_dim, st) : launch<__nv_bfloat16>(p, a->head_dim, st);
}
