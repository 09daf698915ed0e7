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
// pieces of W values (half layout: W values and their W partners); a lane keeps
// one piece number, so it loads that piece's cosines and sines once per token and
// walks the heads by adding a stride.  (Numbering all pieces and dividing for each
// took 150 instructions a piece and was bound by them: 75 us against 64 for an
// append of 13K tokens, whose bytes need 49 at the measured copy rate.)  W is the
// widest of 8 (16-byte accesses), 4, 2 and 1 that divides the pair count, the
// copied part and every stride.
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
  int warps_per_token;
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

// A piece as loaded: W values, and for a rotating piece of the half layout (or a
// single interleaved pair) W more.
template <typename T, int W>
struct Raw {
  typename Vec<T, W>::type a, b;
};

template <typename T, int W, bool INTER>
struct PieceOp {
  using V = typename Vec<T, W>::type;
  static constexpr int NP = INTER ? (W >= 2 ? W / 2 : 1) : W;  // pairs
  static constexpr bool TWO = !INTER || W == 1;                // a rotating piece takes two accesses
  // byte offsets of the two accesses of rotating piece c
  static __device__ __forceinline__ int64_t at_a(int c) { return (int64_t)c * (INTER ? 2 * NP : W) * 2; }
  static __device__ __forceinline__ int64_t gap(int R) { return INTER ? 2 : (int64_t)R; }  // R / 2 values of two bytes

  static __device__ __forceinline__ V load(const char* p) { return *reinterpret_cast<const V*>(p); }
  static __device__ __forceinline__ void store(char* p, V v) { *reinterpret_cast<V*>(p) = v; }

  union Words {  // a vector as its 32-bit words (W >= 2) or its value
    V v;
    uint32_t w[W >= 2 ? W / 2 : 1];
    T e[W];
    __device__ __forceinline__ Words() {}
  };

  // The piece's pairs turned by the angles' cosines and (signed) sines, a word at
  // a time and in place.
  static __device__ __forceinline__ void turn(Raw<T, W>& r, const float (&co)[NP], const float (&si)[NP]) {
    Words a, b;
    a.v = r.a;
    if constexpr (TWO) b.v = r.b;
    if constexpr (W == 1) {
      const float x = Elem<T>::to_float(a.e[0]), y = Elem<T>::to_float(b.e[0]);
      a.e[0] = Elem<T>::from_float(x * co[0] - y * si[0]);
      b.e[0] = Elem<T>::from_float(y * co[0] + x * si[0]);
    } else {
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        const float2 x = Elem<T>::to_float2(a.w[i]);
        if constexpr (TWO) {
          const float2 y = Elem<T>::to_float2(b.w[i]);
          a.w[i] = Elem<T>::pack2(x.x * co[2 * i] - y.x * si[2 * i], x.y * co[2 * i + 1] - y.y * si[2 * i + 1]);
          b.w[i] = Elem<T>::pack2(y.x * co[2 * i] + x.x * si[2 * i], y.y * co[2 * i + 1] + x.y * si[2 * i + 1]);
        } else {
          a.w[i] = Elem<T>::pack2(x.x * co[i] - x.y * si[i], x.y * co[i] + x.x * si[i]);
        }
      }
    }
    r.a = a.v;
    if constexpr (TWO) r.b = b.v;
  }
};

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
  unsigned bad = 0;
  if (a0 > tok || tok >= a1 || s < 0 || e <= s || e > p.num_page_entries) {
    bad = kStatusBadIndptr;
  } else {
    const int64_t len = (int64_t)(e - s - 1) * p.P + last;
    const int64_t at = len - (a1 - a0) + (tok - a0);
    if (last < 1 || last > p.P || at < 0 || at >= len || at >= p.max_positions) {
      bad = kStatusBadToken;
    } else {
      const int entry = (int)(at / p.P), page = __ldg(p.indices + s + entry);
      if (page < 0 || page >= p.num_pages) {
        bad = kStatusBadPage;
      } else {
        pos = at;
        dst = p.cache + (int64_t)page * p.s_page + (at - (int64_t)entry * p.P) * p.s_tok;
      }
    }
  }
  if (bad && lane == 0) record_status(bad);
}

constexpr int kThreads = 128, kWarps = kThreads / 32;

// How a warp's lanes share rows of n pieces: lane's piece and first row, and the
// steps (n <= 32: several rows at a time; more: the pieces of one row in turns).
struct Lanes {
  int c, row, c_step, rows;
  __device__ __forceinline__ Lanes(int n, int lane) {
    if (n <= 32) {
      rows = 32 / n;
      row = lane / n;
      c = row < rows ? lane - row * n : n;  // the last lanes may have none
      c_step = n;
    } else {
      rows = 1;
      row = 0;
      c = lane;
      c_step = 32;
    }
  }
};

// CTAs per SM that the registers are cut for.  More warps cover more of the loads'
// latency until the angles and rows in flight spill: interleaved pieces (half the
// values) take 8 (append of 13K tokens 60 us against 64, plain rows of 8192 tokens
// of 80 heads 134 against 146), half pieces 6 with the append's lookups (62 against
// 68) and no cut on plain rows (132 us a training step's q and k and their
// gradients; 226 at 6, 328 at 8).
constexpr int min_ctas(bool inter, bool append) { return inter ? 8 : append ? 6 : 1; }

// One or several warps per token, each with every warps_per_token-th group of
// rows.  The first rows are asked for before the token is placed (a chain of four
// dependent lookups) and its angles are read, since they need neither.
template <typename T, int W, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads, min_ctas(INTER, APPEND)) rotary_kernel(const RotaryParams p) {
  using Op = PieceOp<T, W, INTER>;
  constexpr int U = 2;  // rows in flight per lane, and as many on their way (1: 74 us, 2: 64, 4: 74)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * (kWarps / p.warps_per_token) + warp / p.warps_per_token;
  if (tok >= p.num_tokens) return;
  const int part = warp % p.warps_per_token, heads = p.Hq + p.Hkv, turned = p.R / 2 / Op::NP;
  const char* q = p.q + tok * p.q_tok;
  const char* k = p.k + tok * p.k_tok;
  auto src_of = [&](int h) { return h < p.Hq ? q + h * p.q_head : k + (h - p.Hq) * p.k_head; };
  Raw<T, W> raw[U];
  const Lanes lt(max(turned, 1), lane);
  const int h0 = part * lt.rows + lt.row, h_step = p.warps_per_token * lt.rows;
  auto fetch = [&](int h, int c) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u * h_step < heads) {
        const char* src = src_of(h + u * h_step) + Op::at_a(c);
        raw[u].a = Op::load(src);
        if constexpr (Op::TWO) raw[u].b = Op::load(src + Op::gap(p.R));
      }
  };
  const bool some = lt.c < turned;
  if (some) fetch(h0, lt.c);
  int64_t pos;
  char* row = nullptr;
  if constexpr (APPEND) {
    place_token(p, tok, lane, pos, row);
  } else {
    pos = __ldg(p.positions + tok);
    if (pos < 0 || pos >= p.max_positions) {
      if (lane == 0) record_status(kStatusBadToken);
      pos = -1;
    }
  }
  const bool placed = pos >= 0;
  char* qo = p.q_out + tok * p.qo_tok;
  char* ko = APPEND ? row : p.k_out + tok * p.ko_tok;
  const int64_t ko_head = APPEND ? p.s_head : p.ko_head;
  // null: not written (a key of a token without a place)
  auto dst_of = [&](int h) -> char* {
    return h < p.Hq ? qo + h * p.qo_head : (APPEND && !placed ? nullptr : ko + (h - p.Hq) * ko_head);
  };
  const float* cs = p.cos_sin + pos * p.cs_stride;
  for (int c = lt.c; c < turned; c += lt.c_step) {
    float co[Op::NP] = {}, si[Op::NP] = {};
    if (placed) {
      load_angles<Op::NP>(cs + c * Op::NP, co);
      load_angles<Op::NP>(cs + p.R / 2 + c * Op::NP, si);
#pragma unroll
      for (int i = 0; i < Op::NP; ++i) si[i] *= p.sign;
    }
    if (c != lt.c) fetch(h0, c);
    for (int h = h0; h < heads; h += U * h_step) {
      Raw<T, W> now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = raw[u];
      fetch(h + U * h_step, c);  // the next rows while these are turned
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u * h_step >= heads) continue;
        char* dst = dst_of(h + u * h_step);
        if (!dst) continue;
        if (placed) Op::turn(now[u], co, si);
        else now[u] = Raw<T, W>{};  // no position: a row of zeros
        Op::store(dst + Op::at_a(c), now[u].a);
        if constexpr (Op::TWO) Op::store(dst + Op::at_a(c) + Op::gap(p.R), now[u].b);
      }
    }
  }
  // the rest of the heads, and v: copied
  auto copy_rows = [&](int n, int rows, int64_t first, auto from, auto to, bool zero) {
    const Lanes lc(n, lane);
    const int step = p.warps_per_token * lc.rows;
    for (int c = lc.c; c < n; c += lc.c_step) {
      constexpr int V = 4;
      for (int h = part * lc.rows + lc.row; h < rows; h += V * step) {
        typename Op::V v[V];
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (h + u * step < rows) v[u] = zero ? typename Op::V{} : Op::load(from(h + u * step) + first + (int64_t)c * W * 2);
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (h + u * step < rows) {
            char* dst = to(h + u * step);
            if (dst) Op::store(dst + first + (int64_t)c * W * 2, v[u]);
          }
      }
    }
  };
  if (p.R < p.D) copy_rows((p.D - p.R) / W, heads, (int64_t)p.R * 2, src_of, dst_of, !placed);
  if (APPEND && placed) {
    const char* v = p.v + tok * p.v_tok;
    copy_rows(p.D / W, p.Hkv, 0, [&](int h) { return v + h * p.v_head; },
              [&](int h) { return row + p.s_kv + h * p.s_head; }, false);
  }
}

// Few tokens do not fill the GPU with a warp each: up to 512 a CTA's four warps
// share one (64 tokens of 40 heads appended in 10.3 us against 12.3, 256 in 10.2
// against 12.3); above, the lookups and angles that each warp repeats cost more
// (2048 tokens in 16.4 us with one warp each, 22.6 with four).
int warps_per_token(int64_t tokens) { return tokens <= 512 ? kWarps : 1; }

template <typename T, int W, bool INTER, bool APPEND>
int launch_rotary(RotaryParams p, cudaStream_t st) {
  p.warps_per_token = warps_per_token(p.num_tokens);
  const int per_cta = kWarps / p.warps_per_token;
  const int64_t ctas = (p.num_tokens + per_cta - 1) / per_cta;
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
