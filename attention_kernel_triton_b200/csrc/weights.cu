// Accumulated attention weights over a paged cache: for each key the sum of the
// softmax weights that it gets from the new tokens' queries.  No reference
// counterpart.
//
// W[b, h, j] += sum_{heads g of h} sum_{rows i that see j} exp(s q_ig . k_j - lse_ig)
// with the rows' final log-sum-exps, so nothing is rescaled and each key's sum is
// its own: a thread per key.
#include "common.cuh"
#include "profile.cuh"

#include <algorithm>
#include <string>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

constexpr int BN = 128;

struct WeightsParams {
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
  const float* lse;
  int64_t l_tok, l_head;
  const float* w;
  int64_t w_batch, w_head;
  float* out;
  int64_t o_batch, o_head;
  int B, Hq, Hkv, group, P, causal, width;
  float scale_log2;
};

template <typename T, int D>
__global__ void __launch_bounds__(BN) weights_simple_kernel(const WeightsParams p) {
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int a0 = __ldg(p.q_indptr + b), a1 = __ldg(p.q_indptr + b + 1);
  const int s = __ldg(p.indptr + b), e = __ldg(p.indptr + b + 1);
  int n = a1 - a0, len = 0;
  if (a0 < 0 || a1 < a0 || a1 > p.num_tokens) {
    record_status(kStatusBadIndptr);
    n = 0;
  }
  if (s < 0 || e < s || e > p.num_page_entries) record_status(kStatusBadIndptr);
  else if (e > s) len = (e - s - 1) * p.P + min(max(__ldg(p.last + b), 0), p.P);
  if (len > p.width) record_status(kStatusBadToken);
  __shared__ T qs[D];
  for (int j0 = blockIdx.z * BN; j0 < min(len, p.width); j0 += gridDim.z * BN) {
    const int j = j0 + threadIdx.x;
    const bool mine = j < min(len, p.width);
    uint4 k[D / 8];
    for (int i = 0; i < D / 8; ++i) k[i] = make_uint4(0, 0, 0, 0);
    if (mine) {
      const int page = __ldg(p.indices + s + j / p.P);
      if (page >= 0 && page < p.num_pages) {
        const uint4* row = reinterpret_cast<const uint4*>(p.kv + page * p.s_page + kvh * p.s_head + (j % p.P) * p.s_tok);
        for (int i = 0; i < D / 8; ++i) k[i] = __ldg(row + i);
      } else {
        record_status(kStatusBadPage);
      }
    }
    float sum = 0.f;
    for (int i = 0; i < n; ++i)
      for (int g = 0; g < p.group; ++g) {
        const int head = kvh * p.group + g;
        __syncthreads();
        if (threadIdx.x < D)
          qs[threadIdx.x] = reinterpret_cast<const T*>(p.q + (int64_t)(a0 + i) * p.q_tok + head * p.q_head)[threadIdx.x];
        __syncthreads();
        const float lse = __ldg(p.lse + (int64_t)(a0 + i) * p.l_tok + head * p.l_head);
        float x = 0.f;
        const uint32_t* q2 = reinterpret_cast<const uint32_t*>(qs);
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          const uint32_t kk[4] = {k[d].x, k[d].y, k[d].z, k[d].w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 a = Elem<T>::to_float2(q2[d * 4 + u]), c = Elem<T>::to_float2(kk[u]);
            x = fmaf(a.x, c.x, fmaf(a.y, c.y, x));
          }
        }
        const bool seen = mine && (!p.causal || j <= len - n + i) && lse != -INFINITY;
        if (seen) sum += fast_exp2(fmaf(x, p.scale_log2, -lse * kLog2e));
      }
    if (mine)
      p.out[b * p.o_batch + kvh * p.o_head + j] = (p.w ? p.w[b * p.w_batch + kvh * p.w_head + j] : 0.f) + sum;
  }
}

bool al16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

int check_args(const akt_attention_weights_args* a) {
  if (a->batch < 0 || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->page_size <= 0 || a->num_tokens < 0 ||
      a->num_pages < 0 || a->num_page_entries < 0 || a->width < 0)
    return set_error(AKT_ERR_INVALID, "attention_weights: bad sizes");
  if (a->num_qo_heads % a->num_kv_heads)
    return set_error(AKT_ERR_INVALID, "num_qo_heads must be a multiple of num_kv_heads");
  if (a->dtype != AKT_FLOAT16 && a->dtype != AKT_BFLOAT16) return set_error(AKT_ERR_INVALID, "dtype");
  if (a->head_dim != 64 && a->head_dim != 128)
    return set_error(AKT_ERR_UNSUPPORTED, "attention_weights: head_dim must be 64 or 128");
  if (a->num_qo_heads / a->num_kv_heads > 128)
    return set_error(AKT_ERR_UNSUPPORTED, "attention_weights: at most 128 query heads per kv head");
  if (!(a->softmax_scale > 0.f) || a->softmax_scale == INFINITY)
    return set_error(AKT_ERR_INVALID, "attention_weights: softmax_scale must be positive and finite");
  // positions, rows and pages are 32-bit in the kernels (addresses are 64-bit)
  if (a->num_tokens > 0x3fffffff / a->num_qo_heads || a->num_page_entries > 0x3fffffff / a->page_size ||
      a->num_pages > 0x7ffffff0 || a->width > 0x3fffffff)
    return set_error(AKT_ERR_INVALID, "attention_weights: too many tokens");
  if (a->batch == 0) return AKT_OK;
  if ((a->num_tokens > 0 && (!a->q || !a->lse)) || !a->q_indptr || !a->kv_page_indptr || !a->kv_last_page_len ||
      (a->width > 0 && !a->out) ||
      (a->num_page_entries > 0 && (!a->kv_page_indices || (!a->kv_cache && a->num_pages > 0))))
    return set_error(AKT_ERR_INVALID, "attention_weights: missing tensor");
  if (a->q_stride_dim != 1 || a->kv_stride_dim != 1)
    return set_error(AKT_ERR_UNSUPPORTED, "attention_weights: unit dim stride required");
  const int64_t strides[] = {a->q_stride_token, a->q_stride_head, a->kv_stride_page,
                             a->kv_stride_kv,   a->kv_stride_head, a->kv_stride_token};
  for (int64_t s : strides)
    if (s % 8) return set_error(AKT_ERR_UNSUPPORTED, "attention_weights: strides must be multiples of 16 bytes");
  if (!al16(a->q) || !al16(a->kv_cache))
    return set_error(AKT_ERR_UNSUPPORTED, "attention_weights: 16-byte alignment required");
  return AKT_OK;
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" size_t akt_attention_weights_workspace_size(const akt_attention_weights_args* a) {
  (void)a;
  return 0;
}

extern "C" int akt_attention_weights(const akt_attention_weights_args* a, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  const int rc = check_args(a);
  if (rc || a->batch == 0) return rc;
  WeightsParams p{};
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
  p.lse = a->lse;
  p.l_tok = a->lse_stride_token;
  p.l_head = a->lse_stride_head;
  p.w = a->weights;
  p.w_batch = a->weights_stride_batch;
  p.w_head = a->weights_stride_head;
  p.out = a->out;
  p.o_batch = a->out_stride_batch;
  p.o_head = a->out_stride_head;
  p.B = a->batch;
  p.Hq = a->num_qo_heads;
  p.Hkv = a->num_kv_heads;
  p.group = p.Hq / p.Hkv;
  p.P = a->page_size;
  p.causal = a->causal ? 1 : 0;
  p.width = (int)a->width;
  p.scale_log2 = a->softmax_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.Hkv, p.B, 32);
  {
    ProfileScope prof(st);
    if (a->dtype == AKT_FLOAT16)
      a->head_dim == 64 ? weights_simple_kernel<__half, 64><<<grid, BN, 0, st>>>(p)
                        : weights_simple_kernel<__half, 128><<<grid, BN, 0, st>>>(p);
    else
      a->head_dim == 64 ? weights_simple_kernel<__nv_bfloat16, 64><<<grid, BN, 0, st>>>(p)
                        : weights_simple_kernel<__nv_bfloat16, 128><<<grid, BN, 0, st>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : set_error(AKT_ERR_CUDA, std::string("attention_weights: ") + cudaGetErrorString(e));
}
