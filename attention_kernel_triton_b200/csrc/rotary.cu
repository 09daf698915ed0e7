// Rotary positions on query and key rows, on plain tensors and fused with the
// append to a paged KV cache.  No reference counterpart (its inputs come
// rotated); the pool and page table are those of the paged decodes.
//
// Pair i of a head's first R values, (a, b) = (x[i], x[i + R/2]) or
// (x[2i], x[2i+1]), becomes (a c - b s, b c + a s) with c, s the table's cosine
// and sine of angle i at the token's position; the values past R are copied.
// The products and the sum are in fp32, rounded once to the type.  The
// rotation is orthogonal, so its gradient is the turn by -s (inverse).
//
// Byte work: each value is read once and written once.  A head is cut into
// pieces of W values (half layout: W values and their W partners), a thread
// takes one piece, and the pieces of a token's q, k (and v) rows are numbered
// one after the other so that neighbouring threads touch neighbouring bytes.
// The table's values come through L1 (a token's heads share its row).  W is
// the widest of 8 (16-byte accesses), 4, 2 and 1 that divides the pair count,
// the copied part and every stride.
#include "common.cuh"
#include "profile.cuh"

#include <string>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

struct RotaryParams {
  const char* q;
  const char* k;
  const char* v;
  char* q_out;
  char* k_out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // bytes
  int64_t qo_tok, qo_head, ko_tok, ko_head;             // bytes
  const float* cos_sin;
  int64_t cs_stride, max_positions;
  const int32_t* positions;
  // append: pool and page table
  char* cache;
  int64_t s_page, s_kv, s_head, s_tok;  // bytes
  int64_t num_pages, num_page_entries;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last;
  const int32_t* app_indptr;
  int B, P;
  int64_t num_tokens;
  int Hq, Hkv, R, D;
  float sign;         // +1, or -1 for the inverse
  FastDiv div_head;   // pieces of one rotated head
  FastDiv div_vrow;   // pieces of one copied v row
  int turned;         // rotating pieces per head; the head's remaining pieces are copied
  int n_rot;          // pieces of the q and k heads of a token
  int n_tok;          // pieces of a token in all (append: with v)
  int tokens_per_cta;
};

template <typename T, int W>
struct Vec;
template <typename T>
struct Vec<T, 8> { using type = uint4; };
template <typename T>
struct Vec<T, 4> { using type = uint2; };
template <typename T>
struct Vec<T, 2> { using type = uint32_t; };
template <typename T>
struct Vec<T, 1> { using type = uint16_t; };

// W values at p (aligned to W values) as floats, and back
template <typename T, int W>
__device__ __forceinline__ void load_row(const char* p, float (&x)[W]) {
  union {
    typename Vec<T, W>::type v;
    T e[W];
  } u;
  u.v = *reinterpret_cast<const typename Vec<T, W>::type*>(p);
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = Elem<T>::to_float(u.e[i]);
}

template <typename T, int W>
__device__ __forceinline__ void store_row(char* p, const float (&x)[W]) {
  union {
    typename Vec<T, W>::type v;
    T e[W];
  } u;
#pragma unroll
  for (int i = 0; i < W; ++i) u.e[i] = Elem<T>::from_float(x[i]);
  *reinterpret_cast<typename Vec<T, W>::type*>(p) = u.v;
}

// N consecutive floats of the table; 16-byte loads when N is a multiple of 4
// (the host has checked the alignment)
template <int N>
__device__ __forceinline__ void load_angles(const float* p, float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
      x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __ldg(p + i);
  }
}

// One rotating piece: pairs of `src` turned into `dst` (the same row offsets);
// cs is the token's table row.  INTER with W == 1 takes one pair in two scalar
// accesses, so a piece holds max(W / 2, 1) pairs there and W pairs otherwise.
template <typename T, int W, bool INTER>
__device__ __forceinline__ void turn_piece(const char* src, char* dst, int c, int R, const float* cs, float sign) {
  if constexpr (INTER) {
    constexpr int NP = W >= 2 ? W / 2 : 1;
    constexpr int NV = 2 * NP;
    float x[NV], y[NV], co[NP], si[NP];
    const int64_t at = (int64_t)c * NV * 2;
    if constexpr (W >= 2) {
      load_row<T, NV>(src + at, x);
    } else {
      float t[1];
      load_row<T, 1>(src + at, t); x[0] = t[0];
      load_row<T, 1>(src + at + 2, t); x[1] = t[0];
    }
    load_angles<NP>(cs + c * NP, co);
    load_angles<NP>(cs + R / 2 + c * NP, si);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float s = sign * si[i];
      y[2 * i] = x[2 * i] * co[i] - x[2 * i + 1] * s;
      y[2 * i + 1] = x[2 * i + 1] * co[i] + x[2 * i] * s;
    }
    if constexpr (W >= 2) {
      store_row<T, NV>(dst + at, y);
    } else {
      const float y0[1] = {y[0]}, y1[1] = {y[1]};
      store_row<T, 1>(dst + at, y0);
      store_row<T, 1>(dst + at + 2, y1);
    }
  } else {
    float a[W], b[W], ya[W], yb[W], co[W], si[W];
    const int64_t at = (int64_t)c * W * 2, half = (int64_t)R;  // R/2 values of two bytes
    load_row<T, W>(src + at, a);
    load_row<T, W>(src + at + half, b);
    load_angles<W>(cs + c * W, co);
    load_angles<W>(cs + R / 2 + c * W, si);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float s = sign * si[i];
      ya[i] = a[i] * co[i] - b[i] * s;
      yb[i] = b[i] * co[i] + a[i] * s;
    }
    store_row<T, W>(dst + at, ya);
    store_row<T, W>(dst + at + half, yb);
  }
}

template <typename T, int W>
__device__ __forceinline__ void copy_piece(const char* src, char* dst) {
  *reinterpret_cast<typename Vec<T, W>::type*>(dst) = *reinterpret_cast<const typename Vec<T, W>::type*>(src);
}

// Position and pool row (K half) of appended token `tok`, by one warp: a
// search with 32 pivots a round for the sequence (two rounds up to 1024
// sequences, where a binary search takes ten dependent loads), then its four
// bounds loaded by four lanes at once.  pos is -1 and the status recorded when
// the page table does not place the token.
__device__ __forceinline__ void place_token(const RotaryParams& p, int64_t tok, int lane, int64_t& pos, char*& dst) {
  int lo = 0, n = p.B;  // the last b in [lo, lo + n) with app_indptr[b] <= tok
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int b = lo + lane * step;
    const bool in = lane * step < n && __ldg(p.app_indptr + b) <= tok;
    const unsigned m = __ballot_sync(0xffffffffu, in);
    const int at = m ? 31 - __clz(m) : 0;
    lo += at * step;
    n = min(step, n - at * step);
  }
  const int b = lo;
  int v = 0;
  if (lane < 2) v = __ldg(p.app_indptr + b + lane);
  else if (lane < 4) v = __ldg(p.indptr + b + lane - 2);
  else if (lane == 4) v = __ldg(p.last + b);
  const int a0 = __shfl_sync(0xffffffffu, v, 0), a1 = __shfl_sync(0xffffffffu, v, 1);
  const int s = __shfl_sync(0xffffffffu, v, 2), e = __shfl_sync(0xffffffffu, v, 3);
  const int last = __shfl_sync(0xffffffffu, v, 4);
  pos = -1;
  dst = nullptr;
  if (lane) return;
  if (a0 > tok || tok >= a1 || s < 0 || e <= s || e > p.num_page_entries) {
    record_status(kStatusBadIndptr);
    return;
  }
  const int64_t len = (int64_t)(e - s - 1) * p.P + last;
  const int64_t at = len - (a1 - a0) + (tok - a0);
  if (last < 1 || last > p.P || at < 0 || at >= len || at >= p.max_positions) {
    record_status(kStatusBadToken);
    return;
  }
  const int page = __ldg(p.indices + s + at / p.P);
  if (page < 0 || page >= p.num_pages) {
    record_status(kStatusBadPage);
    return;
  }
  pos = at;
  dst = p.cache + (int64_t)page * p.s_page + (at % p.P) * p.s_tok;
}

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // tokens of one CTA, one warp each while they are placed

template <typename T, int W, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  __shared__ int64_t pos_s[kMaxTokens];
  __shared__ char* dst_s[kMaxTokens];
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int nt = (int)min((int64_t)p.tokens_per_cta, p.num_tokens - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < nt) {
    int64_t pos;
    char* dst = nullptr;
    if constexpr (APPEND) {
      place_token(p, t0 + warp, lane, pos, dst);
    } else {
      pos = __ldg(p.positions + t0 + warp);
      if (pos < 0 || pos >= p.max_positions) {
        if (lane == 0) record_status(kStatusBadToken);
        pos = -1;
      }
    }
    if (lane == 0) {
      pos_s[warp] = pos;
      dst_s[warp] = dst;
    }
  }
  __syncthreads();
  for (int i = 0; i < nt; ++i) {
    const int64_t tok = t0 + i, pos = pos_s[i];
    char* row = dst_s[i];
    const float* cs = p.cos_sin + pos * p.cs_stride;
    for (int w = threadIdx.x; w < p.n_tok; w += kThreads) {
      if (APPEND && w >= p.n_rot) {  // v rows: copied
        if (pos < 0) continue;
        const int r = w - p.n_rot, h = (int)fdiv((uint32_t)r, p.div_vrow), c = r - h * (int)p.div_vrow.d;
        copy_piece<T, W>(p.v + tok * p.v_tok + h * p.v_head + (int64_t)c * W * 2,
                         row + p.s_kv + h * p.s_head + (int64_t)c * W * 2);
        continue;
      }
      const int h = (int)fdiv((uint32_t)w, p.div_head);
      int c = w - h * (int)p.div_head.d;
      const bool is_q = h < p.Hq;
      const int hk = h - p.Hq;
      const char* src = is_q ? p.q + tok * p.q_tok + h * p.q_head : p.k + tok * p.k_tok + hk * p.k_head;
      char* dst = is_q ? p.q_out + tok * p.qo_tok + h * p.qo_head
                       : (APPEND ? row + hk * p.s_head : p.k_out + tok * p.ko_tok + hk * p.ko_head);
      if (pos < 0) {
        if (APPEND && !is_q) continue;
        // no position: a row of zeros (every piece clears what it would write)
        const float z[W] = {};
        if (c >= p.turned) {
          store_row<T, W>(dst + (int64_t)p.R * 2 + (int64_t)(c - p.turned) * W * 2, z);
        } else if (INTER) {
          constexpr int NV = W >= 2 ? W : 2;
#pragma unroll
          for (int o = 0; o < NV; o += W) store_row<T, W>(dst + (int64_t)c * NV * 2 + o * 2, z);
        } else {
          store_row<T, W>(dst + (int64_t)c * W * 2, z);
          store_row<T, W>(dst + (int64_t)c * W * 2 + p.R, z);
        }
        continue;
      }
      if (c < p.turned) {
        turn_piece<T, W, INTER>(src, dst, c, p.R, cs, p.sign);
      } else {
        const int64_t at = (int64_t)p.R * 2 + (int64_t)(c - p.turned) * W * 2;
        copy_piece<T, W>(src + at, dst + at);
      }
    }
  }
}

// Pieces per token for width W, and the launch.
template <typename T, int W, bool INTER, bool APPEND>
int launch_rotary(RotaryParams p, cudaStream_t st) {
  const int pairs = INTER ? (W >= 2 ? W / 2 : 1) : W;  // pairs of one piece
  p.turned = p.R / 2 / pairs;
  const int per_head = p.turned + (p.D - p.R) / W;
  const int64_t n_rot = (int64_t)(p.Hq + p.Hkv) * per_head;
  const int64_t n_tok = n_rot + (APPEND ? (int64_t)p.Hkv * (p.D / W) : 0);
  if (n_tok > 0x3fffffff) return set_error(AKT_ERR_UNSUPPORTED, "rotary: token rows too large");
  p.n_rot = (int)n_rot;
  p.n_tok = (int)n_tok;
  p.div_head = make_fastdiv((uint32_t)per_head);
  p.div_vrow = make_fastdiv((uint32_t)(p.D / W));
  p.tokens_per_cta = 1;
  const int64_t ctas = (p.num_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (ctas > 0x7fffffff) return set_error(AKT_ERR_INVALID, "rotary: too many tokens");
  {
    ProfileScope prof(st);
    rotary_kernel<T, W, INTER, APPEND><<<(unsigned)ctas, kThreads, 0, st>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(AKT_ERR_CUDA, std::string("rotary: ") + cudaGetErrorString(e));
  return AKT_OK;
}

template <typename T, bool APPEND>
int dispatch_rotary(const RotaryParams& p, int W, bool inter, cudaStream_t st) {
#define AKT_W(N) \
  case N: return inter ? launch_rotary<T, N, true, APPEND>(p, st) : launch_rotary<T, N, false, APPEND>(p, st);
  switch (W) {
    AKT_W(8)
    AKT_W(4)
    AKT_W(2)
    AKT_W(1)
  }
#undef AKT_W
  return set_error(AKT_ERR_INVALID, "rotary: width");
}

// The widest piece (8, 4, 2 or 1 values) that every row and the rotated part
// can take: `bits` is the OR of the pointers and byte strides involved.
int piece_width(uint64_t bits, int D, int R, bool inter, const float* cs, int64_t cs_stride) {
  for (int W = 8; W > 1; W >>= 1) {
    const int pairs = inter ? W / 2 : W;
    // the table is read in 16-byte loads from 4 pairs per piece on
    const bool table = pairs % 4 || (!((uint64_t)(uintptr_t)cs & 15u) && !(cs_stride % 4) && !((R / 2) % 4));
    if (!(bits & (uint64_t)(2 * W - 1)) && !(D % W) && !(R % W) && !((R / 2) % pairs) && table) return W;
  }
  return 1;
}

uint64_t addr_bits(const void* p) { return (uint64_t)(uintptr_t)p; }

int check_rotary(int64_t tokens, int Hq, int Hkv, int D, int R, int dtype, const void* cs, int64_t cs_stride,
                 int64_t max_positions) {
  if (tokens < 0 || Hq < 0 || Hkv < 0 || D <= 0 || max_positions < 0)
    return set_error(AKT_ERR_INVALID, "rotary: bad sizes");
  if (R < 0 || R > D || (R & 1)) return set_error(AKT_ERR_INVALID, "rotary: rotary_dim must be even and at most head_dim");
  if (dtype != AKT_FLOAT16 && dtype != AKT_BFLOAT16) return set_error(AKT_ERR_INVALID, "dtype");
  if (tokens > 0x7fffffff) return set_error(AKT_ERR_INVALID, "rotary: too many tokens");
  if (R > 0 && tokens > 0 && (!cs || cs_stride < R))
    return set_error(AKT_ERR_INVALID, "rotary: cos_sin must hold rows of rotary_dim values");
  return AKT_OK;
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_rotary(const akt_rotary_args* a, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_rotary(a->num_tokens, a->num_qo_heads, a->num_kv_heads, a->head_dim, a->rotary_dim, a->dtype,
                        a->cos_sin, a->cos_sin_stride, a->max_positions);
  if (rc) return rc;
  const bool has_q = a->num_qo_heads > 0, has_k = a->num_kv_heads > 0;
  if (a->num_tokens == 0 || (!has_q && !has_k)) return AKT_OK;
  if ((has_q && (!a->q || !a->q_out)) || (has_k && (!a->k || !a->k_out)) || !a->positions)
    return set_error(AKT_ERR_INVALID, "rotary: missing tensor");
  if ((has_q && (a->q_stride_dim != 1 || a->q_out_stride_dim != 1)) ||
      (has_k && (a->k_stride_dim != 1 || a->k_out_stride_dim != 1)))
    return set_error(AKT_ERR_UNSUPPORTED, "rotary: unit dim stride required");
  RotaryParams p{};
  uint64_t bits = 0;
  if (has_q) {
    p.q = static_cast<const char*>(a->q);
    p.q_out = static_cast<char*>(a->q_out);
    p.q_tok = a->q_stride_token * 2;
    p.q_head = a->q_stride_head * 2;
    p.qo_tok = a->q_out_stride_token * 2;
    p.qo_head = a->q_out_stride_head * 2;
    bits |= addr_bits(a->q) | addr_bits(a->q_out) | p.q_tok | p.q_head | p.qo_tok | p.qo_head;
  }
  if (has_k) {
    p.k = static_cast<const char*>(a->k);
    p.k_out = static_cast<char*>(a->k_out);
    p.k_tok = a->k_stride_token * 2;
    p.k_head = a->k_stride_head * 2;
    p.ko_tok = a->k_out_stride_token * 2;
    p.ko_head = a->k_out_stride_head * 2;
    bits |= addr_bits(a->k) | addr_bits(a->k_out) | p.k_tok | p.k_head | p.ko_tok | p.ko_head;
  }
  p.cos_sin = a->cos_sin;
  p.cs_stride = a->cos_sin_stride;
  p.max_positions = a->max_positions;
  p.positions = a->positions;
  p.num_tokens = a->num_tokens;
  p.Hq = a->num_qo_heads;
  p.Hkv = a->num_kv_heads;
  p.R = a->rotary_dim;
  p.D = a->head_dim;
  p.sign = a->inverse ? -1.f : 1.f;
  const bool inter = a->interleaved != 0;
  const int W = piece_width(bits, p.D, p.R, inter, a->cos_sin, a->cos_sin_stride);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->dtype == AKT_FLOAT16 ? dispatch_rotary<__half, false>(p, W, inter, st)
                                 : dispatch_rotary<__nv_bfloat16, false>(p, W, inter, st);
}

extern "C" int akt_append_rotary_paged_kv(const akt_append_rotary_args* x, void* stream) {
  if (!x) return set_error(AKT_ERR_INVALID, "null args");
  const akt_append_paged_args* a = &x->append;
  int rc = check_rotary(a->num_append, x->num_qo_heads, a->num_kv_heads, a->head_dim, x->rotary_dim, a->dtype,
                        x->cos_sin, x->cos_sin_stride, x->max_positions);
  if (rc) return rc;
  if (a->batch < 0 || a->num_kv_heads <= 0 || a->page_size <= 0)
    return set_error(AKT_ERR_INVALID, "append_rotary_paged_kv: bad sizes");
  if (a->num_append == 0) return AKT_OK;
  if (a->batch == 0) return set_error(AKT_ERR_INVALID, "append_rotary_paged_kv: tokens without sequences");
  const bool has_q = x->num_qo_heads > 0;
  if (!a->kv_cache || !a->append_k || !a->append_v || !a->kv_page_indptr || !a->kv_last_page_len ||
      !a->append_indptr || (!a->kv_page_indices && a->num_page_entries > 0) || (has_q && (!x->q || !x->q_out)))
    return set_error(AKT_ERR_INVALID, "append_rotary_paged_kv: missing tensor");
  if (a->kv_stride_dim != 1 || a->k_stride_dim != 1 || a->v_stride_dim != 1 ||
      (has_q && (x->q_stride_dim != 1 || x->q_out_stride_dim != 1)))
    return set_error(AKT_ERR_UNSUPPORTED, "append_rotary_paged_kv: unit dim stride required");
  RotaryParams p{};
  p.q = static_cast<const char*>(x->q);
  p.q_out = static_cast<char*>(x->q_out);
  p.q_tok = x->q_stride_token * 2;
  p.q_head = x->q_stride_head * 2;
  p.qo_tok = x->q_out_stride_token * 2;
  p.qo_head = x->q_out_stride_head * 2;
  p.k = static_cast<const char*>(a->append_k);
  p.v = static_cast<const char*>(a->append_v);
  p.k_tok = a->k_stride_token * 2;
  p.k_head = a->k_stride_head * 2;
  p.v_tok = a->v_stride_token * 2;
  p.v_head = a->v_stride_head * 2;
  p.cos_sin = x->cos_sin;
  p.cs_stride = x->cos_sin_stride;
  p.max_positions = x->max_positions;
  p.cache = static_cast<char*>(a->kv_cache);
  p.s_page = a->kv_stride_page * 2;
  p.s_kv = a->kv_stride_kv * 2;
  p.s_head = a->kv_stride_head * 2;
  p.s_tok = a->kv_stride_token * 2;
  p.num_pages = a->num_pages;
  p.num_page_entries = a->num_page_entries;
  p.indptr = a->kv_page_indptr;
  p.indices = a->kv_page_indices;
  p.last = a->kv_last_page_len;
  p.app_indptr = a->append_indptr;
  p.B = a->batch;
  p.P = a->page_size;
  p.num_tokens = a->num_append;
  p.Hq = x->num_qo_heads;
  p.Hkv = a->num_kv_heads;
  p.R = x->rotary_dim;
  p.D = a->head_dim;
  p.sign = 1.f;
  uint64_t bits = addr_bits(a->append_k) | addr_bits(a->append_v) | addr_bits(a->kv_cache) | p.k_tok | p.k_head |
                  p.v_tok | p.v_head | p.s_page | p.s_kv | p.s_head | p.s_tok;
  if (has_q) bits |= addr_bits(x->q) | addr_bits(x->q_out) | p.q_tok | p.q_head | p.qo_tok | p.qo_head;
  const bool inter = x->interleaved != 0;
  const int W = piece_width(bits, p.D, p.R, inter, x->cos_sin, x->cos_sin_stride);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->dtype == AKT_FLOAT16 ? dispatch_rotary<__half, true>(p, W, inter, st)
                                 : dispatch_rotary<__nv_bfloat16, true>(p, W, inter, st);
}
