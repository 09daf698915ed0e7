// Accumulated attention weights over a paged cache, on the 5th-generation tensor
// cores (tcgen05 + TMEM): for each key the sum of the softmax weights that it gets
// from the new tokens' queries.  No reference counterpart.
//
// W[b, h, j] += sum_{heads g of h} sum_{rows i that see j} exp(s q_ig . k_j - lse_ig)
// with the rows' final log-sum-exps, so nothing is rescaled, V is not read, and each
// key's sum is its own.  S^T = K Q^T puts the keys on the TMEM lanes: a thread owns a
// key and adds up its row of S^T, no value crosses a thread.
//
// Tiles.  The G query heads of a kv head share K, so the columns of S^T are
// tokens x heads: a row tile is 2 TQ tokens (TQ = floor(128 / G)) in two halves of 128
// columns.  A unit is (sequence, kv head, 256 keys = two K tiles) with all row tiles
// that see one of its keys: the two K tiles stay in shared memory while the row tiles
// pass (64 KB of Q for 2 x 256 x 128 x D products).  Where a sequence has one row tile
// (decoding, verification) Q stays instead and the K tiles pass.
//
// Work split.  The units' costs (row tiles, and one more per unit where there are
// several) stand on a line, (sequence, kv head, unit), which is cut evenly over the
// CTAs (one per SM).  A unit of several row tiles may be cut: its parts leave their
// sums in the workspace and weights_merge_kernel adds them, in the line's order, so
// results depend on the sizes alone.
//
// Warps of a CTA (20):
//   0-15   the exponentials: four warps each for K tile 0 and 1 of the unit (S buffer 0
//          and 1) and the left and right half of its columns
//   16 / 19  loaders of K / of Q and the log-sum-exps: tensor-map boxes inside the
//          pages, or 16-byte cp.async rows where no box fits a page (TMA template)
//   17     issuer of the MMAs (one elected lane)
//   18     scheduler: the CTA's segments, a few ahead, through shared memory
// TMEM (512 columns): two S buffers of 256.  A buffer is free once its last columns
// are in registers, so the tensor pipe works on while the exponentials run.
//
// Exponentials.  The special-function unit gives 16 a cycle and SM, half of what the
// tensor pipe delivers at D = 128; so a share of them is computed on the FMA pipe:
// 2^v = 2^n 2^f, n = round(v), f in [-1/2, 1/2], 2^f by a polynomial of degree 5
// (a minimax fit of the relative error, constant term 1; largest error 1.7e-7 in fp32).
//
// What lies behind the mask.  Scores of hidden pairs are replaced before they are
// used, and K rows past a sequence only reach their own lane, which writes nothing.
//
// Built without -rdc (one status word of its own, as the chunk attention).
#define AKT_WHOLE_PROGRAM 1
#include "common.cuh"
#include "profile.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <string>
#include <type_traits>

namespace akt {

namespace {

constexpr int BK = 128;            // keys of a tile
constexpr int BR = 256;            // rows (tokens x heads) of a tile
constexpr int kExpWarps = 16;
constexpr int kLoadWarp = kExpWarps;  // K
constexpr int kMmaWarp = kExpWarps + 1;
constexpr int kSchedWarp = kExpWarps + 2;
constexpr int kLoadQWarp = kExpWarps + 3;
constexpr int kThreads = 32 * (kExpWarps + 4);
constexpr int kSegs = 4;           // segments in flight between the scheduler and the others
constexpr int kSegReaders = kExpWarps + 3;  // and the 2 loaders and the issuer
constexpr int QS = 2;              // Q tiles in shared memory

struct WeightsParams {
  const char* q;
  const int32_t* q_indptr;
  int64_t num_tokens;
  const char* kv;
  int64_t s_page, s_head, s_tok;  // bytes
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
  int B, Hkv, group, P, causal, width;
  float scale_log2;
  int TQ;
  FastDiv div_group, div_page;
  int box_rows, linear;
  int grid;
  // workspace
  struct Part* parts;  // [grid][2]
  float* part_sum;     // [grid][2][2 BK]
};

// A unit's part that one CTA left in the workspace.
struct Part {
  int used, first, last;  // whether it is one; the unit's first / last row tiles
  int b, kvh, unit;
};

// Row tiles [r0, r1) of units [u0, u1) of a sequence and kv head.
struct Seg {
  int b;       // -1: no more segments
  int q0, n;   // the sequence's first row of q, its new tokens
  int kvh;
  int page0, len;  // first entry of the index array, keys
  int u0, u1, r0, r1;
  int part;    // -1: whole units; else the place of the partial sums
  int pad;
};

template <int D>
struct Cfg {
  static constexpr int DB = D / 64;  // 64-column (128-byte) swizzle blocks of a row
  static constexpr uint32_t Q_BYTES = BR * D * 2, K_BYTES = BK * D * 2;
  // a K tile: per 8 keys, per 64 columns, 8 rows of 128 bytes (swizzled); a Q tile: per 64 columns, 256 rows
  static constexpr uint32_t HALF = 1024, GROUP = DB * 1024;
  static constexpr int KS = D == 64 ? 8 : 3;  // K tiles in shared memory
  static constexpr uint32_t OFF_Q = 0, OFF_K = QS * Q_BYTES, OFF_LSE = OFF_K + KS * K_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_LSE + QS * BR * 4;
  // k_full, k_empty [KS]; q_full, lse_full, q_empty [QS]; s_full, s_free [2]; seg_full, seg_empty [kSegs]; red_full,
  // red_empty [2]; mma_idle
  static constexpr int N_BARS = 2 * KS + 3 * QS + 4 + 2 * kSegs + 5;
  static constexpr uint32_t OFF_MISC = OFF_BAR + (N_BARS * 8 + 15) / 16 * 16;  // TMEM address, abort flag
  static constexpr uint32_t OFF_SEG = OFF_MISC + 16;
  static constexpr uint32_t OFF_RED = OFF_SEG + kSegs * sizeof(Seg);  // sums of a K tile's right half
  static constexpr uint32_t OFF_NONE = (OFF_RED + BK * 4 + 15) / 16 * 16;  // rows of Q that add nothing
  static constexpr uint32_t SMEM = OFF_NONE + QS * (BR / 32) * 4;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// -------------------------------------------------------------------------
// the sequences and their units
// -------------------------------------------------------------------------
struct Seq {
  int a0, n, page0, len;  // first row of q, new tokens, first index entry, keys
  int units, tiles;       // units of a kv head (keys past the width have none), row tiles
};

// Sequence b's bounds; a malformed one is empty, one with malformed rows has none.
__device__ __forceinline__ Seq load_seq(const WeightsParams& p, int b, bool record) {
  Seq s;
  const int a1 = __ldg(p.q_indptr + b + 1), e = __ldg(p.indptr + b + 1), last = __ldg(p.last + b);
  s.a0 = __ldg(p.q_indptr + b);
  s.page0 = __ldg(p.indptr + b);
  s.n = a1 - s.a0;
  s.len = 0;
  if (s.a0 < 0 || a1 < s.a0 || a1 > p.num_tokens) {
    if (record) record_status(kStatusBadIndptr);
    s.n = 0;
  }
  if (s.page0 < 0 || e < s.page0 || e > p.num_page_entries) {
    if (record) record_status(kStatusBadIndptr);
  } else if (e > s.page0) {
    s.len = (e - s.page0 - 1) * p.P + min(max(last, 0), p.P);
  }
  if (record && s.len > p.width) record_status(kStatusBadToken);
  s.units = (min(s.len, p.width) + 2 * BK - 1) / (2 * BK);
  s.tiles = (s.n + 2 * p.TQ - 1) / (2 * p.TQ);
  return s;
}

// First row tile that sees a key of unit u.
__device__ __forceinline__ int first_tile(const WeightsParams& p, const Seq& s, int u) {
  return p.causal ? max(0, 2 * BK * u - (s.len - s.n)) / (2 * p.TQ) : 0;
}

// sum of floor((a i + b) / m) over 0 <= i < n: whole multiples of m are taken out of a
// and b, and what is left counts the lattice points below a line, which are counted
// along the other axis.
__device__ int64_t floor_sum(int64_t n, int64_t a, int64_t b, int64_t m) {
  int64_t sum = 0;
  while (n > 0) {
    sum += (n - 1) * n / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const int64_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const int64_t t = a;
    a = m;
    m = t;
  }
  return sum;
}

// Cost of the first u units of a kv head.
__device__ __forceinline__ int64_t cost_before(const WeightsParams& p, const Seq& s, int u) {
  if (s.tiles <= 1) return u;
  int64_t c = (int64_t)u * (1 + s.tiles);
  if (p.causal) {
    const int d = s.len - s.n, i0 = d > 0 ? (d + 2 * BK - 1) / (2 * BK) : 0;
    c -= floor_sum(u - i0, 2 * BK, 2 * BK * i0 - d, 2 * p.TQ);
  }
  return c;
}

// -------------------------------------------------------------------------
// exponentials
// -------------------------------------------------------------------------
// Whether the FMA pipe computes the exponentials of this pair of columns: one of four
// (8192 tokens on top of 24576: 2.02 ms, none 2.08, three of eight 2.12, all 3.02).
constexpr bool on_fma_pipe(int pair) { return pair % 4 == 0; }

// bits below n
__device__ __forceinline__ unsigned below(int n) { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u; }

// 2^v of two values on the FMA pipe, as mantissas and scales.  The shift puts
// n + 127 into the low bits of t; v below -127 gives a scale of 0, from 127.5 on one of
// infinity (only with a log-sum-exp that is not the row's own), NaN stays NaN.
__device__ __forceinline__ void poly_exp2(float2 v, float2& mant, float2& scale) {
  constexpr float kShift = 12582912.f + 127.f;  // 1.5 * 2^23 + 127
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v.x) : "f"(v.x), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v.y) : "f"(v.y), "f"(-127.f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(v.x) : "f"(v.x), "f"(128.f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(v.y) : "f"(v.y), "f"(128.f));
  const float2 t = __fadd2_rn(v, make_float2(kShift, kShift));
  const float2 n = __fadd2_rn(t, make_float2(-kShift, -kShift));
  const float2 f = __fadd2_rn(v, make_float2(-n.x, -n.y));
  auto c = [](float x) { return make_float2(x, x); };
  float2 r = ffma2(c(0.0013264715f), f, c(0.009671509f));
  r = ffma2(r, f, c(0.055507336f));
  r = ffma2(r, f, c(0.24022242f));
  r = ffma2(r, f, c(0.693147f));
  mant = ffma2(r, f, c(1.f));
  uint32_t sx, sy;  // (a shift on the ALU; a plain one may become a multiplication on the FMA pipe)
  asm("shf.l.clamp.b32 %0, 0, %1, 23;" : "=r"(sx) : "r"(__float_as_uint(t.x)));
  asm("shf.l.clamp.b32 %0, 0, %1, 23;" : "=r"(sy) : "r"(__float_as_uint(t.y)));
  scale = make_float2(__uint_as_float(sx), __uint_as_float(sy));
}

// -------------------------------------------------------------------------
// main kernel
// -------------------------------------------------------------------------
template <typename T, int D, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
    weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ WeightsParams p) {
  using C = Cfg<D>;
  constexpr int KS = C::KS;
  constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;

  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_empty = k_full + KS;
  uint64_t* q_full = k_empty + KS;
  uint64_t* lse_full = q_full + QS;
  uint64_t* q_empty = lse_full + QS;  // the MMAs and the exponentials are done with the slot
  uint64_t* s_full = q_empty + QS;
  uint64_t* s_free = s_full + 2;
  uint64_t* seg_full = s_free + 2;
  uint64_t* seg_empty = seg_full + kSegs;
  uint64_t* red_full = seg_empty + kSegs;  // [K tile of the unit] the right half's sums are there
  uint64_t* red_empty = red_full + 2;      // and read
  uint64_t* mma_idle = red_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Seg* segs = reinterpret_cast<Seg*>(smem + C::OFF_SEG);
  float* lse_s = reinterpret_cast<float*>(smem + C::OFF_LSE);  // [QS][BR]: -lse log2 e, -inf: no such row

  unsigned* none_s = reinterpret_cast<unsigned*>(smem + C::OFF_NONE);  // [QS][BR / 32] bits: rows whose lse is -inf

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], TMA ? 1 : 32);  // cp.async: every lane of the loader
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&lse_full[s], 1);
      mbar_init(&q_empty[s], 1 + kExpWarps);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], kExpWarps / 2);
    }
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], kSegReaders);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&red_full[t], 4);
      mbar_init(&red_empty[t], 4);
    }
    mbar_init(mma_idle, 1);
    *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;  // swizzled tiles need a 1024-byte aligned base
    if (*abort_flag) record_status(kStatusWaitTimeout);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "n"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // ---- this CTA's range of the line, and the sequence that it starts in (scratch where Q goes later)
  int64_t* sums = reinterpret_cast<int64_t*>(smem + C::OFF_Q);  // of the warps
  int64_t* found = sums + kThreads / 32;                        // [2] start of the sequence, its number
  auto scan = [&](int64_t x, int64_t& total) -> int64_t {       // sum over the threads before this one
    int64_t v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      before += w < warp ? sums[w] : 0;
      total += sums[w];
    }
    __syncthreads();
    return before + v - x;
  };
  auto seq_cost = [&](int b, bool record) -> int64_t {
    if (b >= p.B) return 0;
    const Seq s = load_seq(p, b, record);
    return cost_before(p, s, s.units) * p.Hkv;
  };
  int64_t W = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    int64_t total;
    scan(seq_cost(b0 + threadIdx.x, blockIdx.x == 0), total);
    W += total;
  }
  const int64_t per = W / p.grid, left = W - per * p.grid;
  const int64_t begin = per * blockIdx.x + min((int64_t)blockIdx.x, left);
  const int64_t end = begin + per + ((int64_t)blockIdx.x < left ? 1 : 0);
  for (int64_t b0 = 0, at = 0; b0 < p.B && at <= begin && begin < end; b0 += kThreads) {
    const int64_t c = seq_cost((int)b0 + threadIdx.x, false);
    int64_t total;
    const int64_t x = at + scan(c, total);
    if (x <= begin && begin < x + c) {
      found[0] = x;
      found[1] = b0 + threadIdx.x;
    }
    at += total;
  }
  __syncthreads();
  const int64_t start_x = begin < end ? found[0] : 0;
  const int start_b = begin < end ? (int)found[1] : 0;
  __syncthreads();
  // rows of the Q tiles that no box fills
  const int used = p.TQ * p.group;
  if (used < BK)
    for (int i = threadIdx.x; i < QS * C::DB * 2 * (BK - used) * 8; i += kThreads) {
      const int piece = i & 7, r = (i >> 3) % (BK - used), part = (i >> 3) / (BK - used);  // (slot, 64 columns, half)
      *reinterpret_cast<uint4*>(smem + C::OFF_Q + (uint32_t)part * (BK * 128) + (used + r) * 128 + piece * 16) =
          make_uint4(0, 0, 0, 0);
    }
  fence_async_smem();  // generic writes and reads before the async proxy's
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // the same answer in every lane, so a warp gives up as a whole
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || wait_or_abort_call(bar, parity, abort_flag));
  };
  if (warp == kSchedWarp) {
    // ============================ scheduler ============================
    int64_t x = begin;
    int b = start_b, kvh = -1;
    Seq s{};
    int64_t head_x = 0, per_head = 0;  // where the current kv head starts, its cost
    if (begin < end) {
      s = load_seq(p, b, false);
      per_head = cost_before(p, s, s.units);
      kvh = (int)((begin - start_x) / per_head);
      head_x = start_x + kvh * per_head;
    }
    int n_parts = 0;
    if (lane < 2) p.parts[2 * blockIdx.x + lane].used = 0;
    __syncwarp();
    for (int k = 0;; ++k) {
      Seg sg{};
      sg.b = -1;
      while (x < end) {
        const int64_t rel = x - head_x;
        sg.q0 = s.a0;
        sg.n = s.n;
        sg.kvh = kvh;
        sg.page0 = s.page0;
        sg.len = s.len;
        sg.part = -1;
        bool some = true;
        if (s.tiles <= 1) {  // a run of units
          sg.u0 = (int)rel;
          sg.u1 = (int)min((int64_t)s.units, rel + (end - x));
          sg.r0 = 0;
          sg.r1 = s.tiles;
          x += sg.u1 - sg.u0;
        } else {
          // the unit that holds x: 32 places at a time
          int lo = 0, hi = s.units;  // cost_before(lo) <= rel < cost_before(hi)
          while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, at = lo + lane * step;
            const unsigned m = __ballot_sync(0xffffffffu, at < hi && cost_before(p, s, at) <= rel);
            lo += (31 - __clz(m)) * step;  // (lane 0 always holds)
            hi = min(hi, lo + step);
          }
          const int64_t unit_x = cost_before(p, s, lo), cost = cost_before(p, s, lo + 1) - unit_x;
          const int64_t from = rel - unit_x, to = min(cost, rel + (end - x) - unit_x);
          const int first = first_tile(p, s, lo);
          sg.u0 = lo;
          sg.u1 = lo + 1;
          sg.r0 = first + (int)max((int64_t)0, from - 1);
          sg.r1 = first + (int)(to - 1);
          some = sg.r0 < sg.r1;  // a range with none of the unit's tiles leaves it to the others
          if (some && sg.r1 - sg.r0 < s.tiles - first) {
            sg.part = n_parts++;
            if (lane == 0) p.parts[2 * blockIdx.x + sg.part] = Part{1, sg.r0 == first, sg.r1 == s.tiles, b, kvh, lo};
          }
          x += to - from;
        }
        sg.b = b;
        if (x == head_x + per_head && x < end) {  // on to the next kv head with any cost
          head_x = x;
          if (++kvh == p.Hkv) {
            kvh = 0;
            do {
              s = load_seq(p, ++b, false);
              per_head = cost_before(p, s, s.units);
            } while (per_head == 0);
          }
        }
        if (some) break;
        sg.b = -1;
      }
      const int e = k % kSegs;
      if (k >= kSegs && !wait(&seg_empty[e], ((k / kSegs) - 1) & 1)) break;
      if (lane == 0) {
        segs[e] = sg;
        mbar_arrive(&seg_full[e]);
      }
      __syncwarp();
      if (sg.b < 0) break;
    }
  } else if (warp == kLoadWarp) {
    // ============================ K loader ============================
    uint32_t g = 0;       // tiles asked for
    uint32_t loaded = 0;  // stages this warp has loaded (bits 0 ..) and the parity of the last load (16 ..)
    bool ok = true;
    const int boxes = TMA ? BK / p.box_rows : 0;  // of one tile, at most 16
    for (int k = 0; ok; ++k) {
      if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
      const Seg sg = segs[k % kSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
      if (sg.b < 0) break;
      if (sg.r0 == sg.r1) continue;
      const int t0 = 2 * sg.u0, t1 = 2 * sg.u1;
      if constexpr (TMA) {
        // lane l loads box l of each tile: keys [rb, rb + box_rows) of the tile
        const int rb = lane * p.box_rows;
        const bool mine = lane < boxes;
        // the index entry of the box's page, a tile ahead of its use
        auto entry = [&](int j) -> int {
          const int key = j * BK + rb;
          return mine && key < sg.len ? __ldg(p.indices + sg.page0 + (int)fdiv((uint32_t)key, p.div_page)) : -1;
        };
        int id_next = entry(t0);
        for (int j = t0; j < t1; ++j, ++g) {
          const int id = id_next, key = j * BK + rb;
          if (j + 1 < t1) id_next = entry(j + 1);
          const uint32_t st = g % KS;
          if (g >= KS && !wait(&k_empty[st], ((g / KS) - 1) & 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&k_full[st], C::K_BYTES);
          loaded = (loaded & ~(0x10001u << st)) | 1u << st | ((g / KS) & 1u) << (16 + st);
          __syncwarp();
          if (mine) {
            // boxes past the sequence, and of bad ids, are asked for past the pool: zeros
            const bool there = id >= 0 && id < p.num_pages;
            const int row = there ? key - (int)fdiv((uint32_t)key, p.div_page) * p.P : 0;
            const int page = there ? id : (int)p.num_pages;
            unsigned char* dst = smem + C::OFF_K + st * C::K_BYTES + (rb >> 3) * C::GROUP;
            if (p.linear)  // [block of a page, kv and head][8-row group][64 columns][row]
              tma_load_5d(dst, &tmK, 0, 0, row >> 3, page * 2 * p.Hkv + sg.kvh, &k_full[st]);
            else  // [page][head][64 columns][row]
              tma_load_5d(dst, &tmK, row, 0, sg.kvh, page, &k_full[st]);
            if (!there && key < sg.len) record_status(kStatusBadPage);
          }
          __syncwarp();
        }
      } else {
        // every half warp (D = 128) or quarter (D = 64) copies whole rows in 16-byte pieces
        constexpr int CH = D / 8, RW = 32 / CH;  // pieces of a row; rows a step
        const int ch = lane % CH, rl = lane / CH;
        int id_next[BK / 32];  // the index entries of a tile's rows lane, lane + 32, ..., a tile ahead of their use
        auto entries = [&](int j) {
#pragma unroll
          for (int i = 0; i < BK / 32; ++i) {
            const int key = j * BK + i * 32 + lane;
            id_next[i] = key < sg.len ? __ldg(p.indices + sg.page0 + (int)fdiv((uint32_t)key, p.div_page)) : -1;
          }
        };
        entries(t0);
        for (int j = t0; j < t1; ++j, ++g) {
          const char* src[BK / 32];  // the rows' addresses (null: zeros)
#pragma unroll
          for (int i = 0; i < BK / 32; ++i) {
            const int key = j * BK + i * 32 + lane, id = id_next[i];
            src[i] = nullptr;
            if (id >= 0 && id < p.num_pages)
              src[i] = p.kv + (int64_t)id * p.s_page + (int64_t)sg.kvh * p.s_head +
                       (int64_t)(key - (int)fdiv((uint32_t)key, p.div_page) * p.P) * p.s_tok;
            else if (key < sg.len) record_status(kStatusBadPage);
          }
          if (j + 1 < t1) entries(j + 1);
          __syncwarp();
          const uint32_t st = g % KS;
          if (g >= KS && !wait(&k_empty[st], ((g / KS) - 1) & 1)) {
            ok = false;
            break;
          }
          __syncwarp();
          const uint32_t tile = smem_u32(smem + C::OFF_K + st * C::K_BYTES);
#pragma unroll
          for (int i = 0; i < BK / 32; ++i) {
#pragma unroll 8
            for (int r0 = 0; r0 < 32; r0 += RW) {
              const int r = r0 + rl;
              const char* row =
                  reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src[i]), r));
              const uint32_t dst = tile + (uint32_t)(i * 4 + (r >> 3)) * C::GROUP + (ch >> 3) * C::HALF + (r & 7) * 128 +
                                   (((ch & 7) ^ (r & 7)) << 4);
              cp_async16(dst, row ? row + ch * 16 : p.q, row ? 16u : 0u);
            }
          }
          cp_async_arrive(&k_full[st]);  // each lane's arrival, once its copies have landed
        }
      }
    }
    if (TMA && *abort_flag && lane == 0)  // loads still in flight into this CTA's shared memory
      for (int st = 0; st < KS; ++st)  // whichever phase a stage is in, its load (if any) ends it
        if (loaded >> st & 1u) mbar_wait(&k_full[st], loaded >> (16 + st) & 1u);
    if (!TMA) cp_async_wait_all();
  } else if (warp == kLoadQWarp) {
    // ============================ loader of Q and the log-sum-exps ============================
    uint32_t g = 0;  // tiles asked for
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
      const Seg sg = segs[k % kSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
      if (sg.b < 0) break;
      for (int r = sg.r0; r < sg.r1; ++r, ++g) {  // (once for all units of a run)
        const int slot = g % QS, tok = r * 2 * p.TQ;
        if (g >= QS && !wait(&q_empty[slot], ((g / QS) - 1) & 1)) {
          ok = false;
          break;
        }
        const int halves = sg.n - tok > p.TQ ? 2 : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[slot], (uint32_t)(halves * used * 128 * C::DB));
          for (int hf = 0; hf < halves; ++hf)
#pragma unroll
            for (int db = 0; db < C::DB; ++db)
              tma_load_4d(smem + C::OFF_Q + slot * C::Q_BYTES + db * (BR * 128) + hf * (BK * 128), &tmQ, db * 64, 0,
                          sg.kvh, sg.q0 + tok + hf * p.TQ, &q_full[slot]);
        }
        __syncwarp();
        float v[BR / 32];
#pragma unroll
        for (int i = 0; i < BR / 32; ++i) {
          const int c = i * 32 + lane, rr = c & (BK - 1), rt = (int)fdiv((uint32_t)rr, p.div_group);
          const int t = tok + (c >> 7) * p.TQ + rt;
          v[i] = -INFINITY;
          if (rt < p.TQ && t < sg.n)
            v[i] = -__ldg(p.lse + (int64_t)(sg.q0 + t) * p.l_tok +
                          (int64_t)(sg.kvh * p.group + rr - rt * p.group) * p.l_head) * kLog2e;
        }
#pragma unroll
        for (int i = 0; i < BR / 32; ++i) {  // lse = -inf: the row adds nothing
          const unsigned nothing = __ballot_sync(0xffffffffu, v[i] == INFINITY);
          if (lane == 0) none_s[slot * (BR / 32) + i] = nothing;
          lse_s[slot * BR + i * 32 + lane] = v[i] == INFINITY ? -INFINITY : v[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&lse_full[slot]);
      }
    }
    if (*abort_flag && lane == 0)
      for (uint32_t i = g > QS ? g - QS : 0; i < g; ++i) mbar_wait(&q_full[i % QS], (i / QS) & 1);
  } else if (warp == kMmaWarp) {
    // ============================ MMA issuer ============================
    auto uni = [&](int v) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)v); };
    const uint64_t dk = desc_sw128(smem_u32(smem + C::OFF_K), 16, C::GROUP);
    const uint64_t dq = desc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
    const uint32_t tmem_u = uni(tmem);
    uint32_t gk = 0, gq = 0, gs = 0;  // K tiles, Q tiles, turns of the S buffers
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
      const Seg* sp = &segs[k % kSegs];
      const int more = uni(sp->b >= 0), u0 = uni(sp->u0), u1 = uni(sp->u1), r0 = uni(sp->r0), r1 = uni(sp->r1), n = uni(sp->n);
      if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
      if (!more) break;
      if (r0 == r1) continue;
      const bool stays = u1 - u0 > 1;  // one Q tile for all units
      for (int u = u0; ok && u < u1; ++u) {
        for (int r = r0; r < r1; ++r) {
          const int slot = gq % QS, toks = n - r * 2 * p.TQ;
          // columns that the tile's rows fill, in steps of 16; a half that is full of tokens is read
          // whole and without a mask, so all of its columns are written (by rows of zeros, if it must be)
          const int cols = toks > p.TQ ? BR : (toks == p.TQ ? BK : (toks * p.group + 15) / 16 * 16);
          const uint32_t idesc = idesc_f16(fmt, BK, 0, 0) | (uint32_t)(cols >> 3) << 17;
          if (!wait(&q_full[slot], (gq / QS) & 1)) { ok = false; break; }
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            const uint32_t st = (gk + t) % KS;
            if (!wait(&k_full[st], ((gk + t) / KS) & 1) || (gs && !wait(&s_free[t], (gs - 1) & 1))) {
              ok = false;
              break;
            }
            if (!TMA) fence_async_smem();  // what the copies wrote, before the MMAs' reads
            tc_fence_after();
            if (elect_one()) {
              const uint64_t a = dk + st * (C::K_BYTES >> 4), q = dq + slot * (C::Q_BYTES >> 4);
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                const uint32_t in = (i & 3) * 32;  // inside a row's 128 bytes
                mma_ss(tmem_u + t * BR, a + (((i >> 2) * C::HALF + in) >> 4), q + (((i >> 2) * (BR * 128) + in) >> 4),
                       idesc, i > 0);
              }
              mma_commit(&s_full[t]);
              if (r + 1 == r1) mma_commit(&k_empty[st]);
              if (t && (!stays || u + 1 == u1)) mma_commit(&q_empty[slot]);
            }
            __syncwarp();
          }
          if (!ok) break;
          ++gs;
          if (!stays || u + 1 == u1) ++gq;
        }
        gk += 2;
      }
    }
    // every MMA issued by this thread has finished before the CTA can exit
    if (elect_one()) mma_commit(mma_idle);
    __syncwarp();
    mbar_wait(mma_idle, 0);
  } else {
    // ============================ exponentials ============================
    const int t = warp >> 2 & 1, half = warp >> 3, row = threadIdx.x & (BK - 1);
    const bool ragged = used % 32;  // a full half reads columns of cleared rows of Q
    const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * BR + half * BK;
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
    uint32_t gq = 0, gs = 0, joins = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
      const Seg sg = segs[k % kSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
      if (sg.b < 0) break;
      const bool stays = sg.u1 - sg.u0 > 1;
      const bool wide = sg.n - sg.r0 * 2 * p.TQ > p.TQ;  // the right halves have columns
      for (int u = sg.u0; ok && u < sg.u1; ++u) {
        const int key0 = (2 * u + t) * BK, key = key0 + row;
        const bool mine = key < min(sg.len, p.width);
        float before = 0.f;
        if (mine && half == 0 && sg.part < 0 && p.w) before = __ldg(p.w + sg.b * p.w_batch + sg.kvh * p.w_head + key);
        float2 acc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = make_float2(0.f, 0.f);
        for (int r = sg.r0; r < sg.r1; ++r) {
          // the half's first token, and its tokens
          const int slot = gq % QS, tok = r * 2 * p.TQ + half * p.TQ, toks = min(sg.n - tok, p.TQ);
          if (!wait(&lse_full[slot], (gq / QS) & 1) || !wait(&s_full[t], gs & 1)) {
            ok = false;
            break;
          }
          ++gs;
          tc_fence_after();
          // tokens of the half that do not see this key yet, and whether any pair of the half is hidden
          const int skip = p.causal ? key - (sg.len - sg.n) - tok : 0;
          const bool masked = toks < p.TQ || (p.causal && key0 + BK - 1 - (sg.len - sg.n) - tok > 0);
          const int chunks = (max(toks, 0) * p.group + 31) / 32;
          // In a full half the last chunk ends in columns of cleared rows, which an infinite key makes NaN.  They are
          // looked at first (2048 tokens on top of 6144 of four sequences, 28 heads on 4, D = 64: 421 us; hidden
          // without a look 437).
          const int cleared_in = ragged ? chunks - 1 : -1;
          const float4* nl = reinterpret_cast<const float4*>(lse_s + slot * BR + half * BK);
          const unsigned* none = none_s + slot * (BR / 32) + half * (BK / 32);
          const uint4 n4 = *reinterpret_cast<const uint4*>(none);
          const bool hides = masked || (n4.x | n4.y | n4.z | n4.w);
          if (!chunks) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[t]);
          }
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            float x[32];
            {
              uint32_t rr[32];
              tmem_ld32(tS + c * 32, rr);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(rr[e]);
            }
            if (c + 1 == chunks) {  // the buffer is free for the next MMAs
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_free[t]);
            }
            if (hides || (c == cleared_in && __any_sync(0xffffffffu, x[31] != x[31]))) {
              const int lo = min(max(skip, 0), p.TQ) * p.group - c * 32, hi = toks * p.group - c * 32;
              const unsigned hidden = none[c] | below(lo) | ~below(hi);
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = hidden >> e & 1u ? -INFINITY : x[e];
            }
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 l4 = nl[c * 8 + e / 4];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int pair = e / 2 + i;
                const float2 v = ffma2(make_float2(x[e + 2 * i], x[e + 2 * i + 1]), sl2,
                                       i ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y));
                if (on_fma_pipe(pair)) {
                  float2 mant, scale;
                  poly_exp2(v, mant, scale);
                  acc[pair & 3] = ffma2(mant, scale, acc[pair & 3]);
                } else {
                  acc[pair & 3] = __fadd2_rn(acc[pair & 3], make_float2(fast_exp2(v.x), fast_exp2(v.y)));
                }
              }
            }
          }
          if (!stays || u + 1 == sg.u1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[slot]);
            ++gq;
          }
        }
        const float2 a01 = __fadd2_rn(acc[0], acc[1]), a23 = __fadd2_rn(acc[2], acc[3]), a = __fadd2_rn(a01, a23);
        float sum = a.x + a.y;
        if (wide && ok) {  // left half + right half; one buffer, the unit's two K tiles in turn
          if (half) {
            ok = t ? wait(&red_empty[0], joins & 1) : !joins || wait(&red_empty[1], (joins - 1) & 1);
            if (ok) red[row] = sum;
          } else {
            ok = wait(&red_full[t], joins & 1);
            if (ok) sum += red[row];
          }
          __syncwarp();
          if (ok && lane == 0) mbar_arrive(half ? &red_full[t] : &red_empty[t]);
          ++joins;
        }
        if (!ok) break;
        if (half) continue;
        if (sg.part >= 0) p.part_sum[((int64_t)(2 * blockIdx.x) + sg.part) * (2 * BK) + t * BK + row] = sum;
        else if (mine) p.out[sg.b * p.o_batch + sg.kvh * p.o_head + key] = before + sum;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
  }
}

// -------------------------------------------------------------------------
// merge of units in parts
// -------------------------------------------------------------------------
// The unit's parts are the one with its first row tiles and then place 0 of the CTAs
// after it, up to the one with its last (CTAs without a part of it in between had
// none of its tiles).  CTA x: place x; a thread per key.
__global__ void __launch_bounds__(2 * BK) weights_merge_kernel(const WeightsParams p) {
  grid_dep_wait();
  const Part me = p.parts[blockIdx.x];
  if (!me.used || !me.first) return;
  const int key = me.unit * 2 * BK + threadIdx.x;
  float sum = p.part_sum[(int64_t)blockIdx.x * (2 * BK) + threadIdx.x];
  bool last = me.last;
  for (int c = (blockIdx.x >> 1) + 1; !last && c < p.grid; ++c) {
    const Part next = p.parts[2 * c];
    if (!next.used) continue;
    sum += p.part_sum[(int64_t)(2 * c) * (2 * BK) + threadIdx.x];
    last = next.last;
  }
  const int s = __ldg(p.indptr + me.b), e = __ldg(p.indptr + me.b + 1);
  const int len = (e - s - 1) * p.P + min(max(__ldg(p.last + me.b), 0), p.P);
  if (key >= min(len, p.width)) return;
  const float before = p.w ? p.w[me.b * p.w_batch + me.kvh * p.w_head + key] : 0.f;
  p.out[me.b * p.o_batch + me.kvh * p.o_head + key] = before + sum;
}

// -------------------------------------------------------------------------
// host
// -------------------------------------------------------------------------
struct Layout {
  int grid;
  size_t parts, sums, bytes;
};

// One CTA per SM, or one per unit where the table's bounds show that there are fewer.
Layout make_layout(const akt_attention_weights_args* a) {
  Layout y{};
  const int64_t units = (a->num_page_entries * a->page_size / (2 * BK) + a->batch) * a->num_kv_heads;
  const int64_t tiles = a->num_tokens / (2 * (BK / (a->num_qo_heads / a->num_kv_heads))) + 1;
  y.grid = (int)std::max<int64_t>(1, std::min<int64_t>(sm_count(), units * tiles));
  y.sums = round256((size_t)y.grid * 2 * sizeof(Part));
  y.bytes = y.sums + (size_t)y.grid * 2 * 2 * BK * 4;
  return y;
}

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

template <typename T, int D, bool TMA>
int launch_weights(const CUtensorMap& mq, const CUtensorMap& mk, const WeightsParams& p, bool parts, cudaStream_t st) {
  auto kern = weights_kernel<T, D, TMA>;
  constexpr int smem = (int)Cfg<D>::SMEM;
  cudaError_t e = ensure_smem_limit<weights_kernel<T, D, TMA>>((size_t)smem);
  if (e != cudaSuccess) return set_error(AKT_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  {
    ProfileScope prof(st);
    kern<<<p.grid, kThreads, smem, st>>>(mq, mk, p);
  }
  if (parts) e = launch_dependent(weights_merge_kernel, dim3(2 * p.grid), dim3(2 * BK), 0, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : set_error(AKT_ERR_CUDA, std::string("attention_weights: ") + cudaGetErrorString(e));
}

template <typename T, int D>
int dispatch_weights(const CUtensorMap& mq, const CUtensorMap& mk, const WeightsParams& p, bool parts, cudaStream_t st) {
  return p.box_rows ? launch_weights<T, D, true>(mq, mk, p, parts, st) : launch_weights<T, D, false>(mq, mk, p, parts, st);
}

}  // namespace

cudaError_t weights_status_read(unsigned int* v) { return cudaMemcpyFromSymbol(v, g_device_status_local, sizeof(*v)); }

cudaError_t weights_status_clear() {
  const unsigned int z = 0;
  return cudaMemcpyToSymbol(g_device_status_local, &z, sizeof(z));
}

}  // namespace akt

using namespace akt;

extern "C" size_t akt_attention_weights_workspace_size(const akt_attention_weights_args* a) {
  if (!a || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->num_qo_heads % a->num_kv_heads || a->batch <= 0 ||
      a->num_qo_heads / a->num_kv_heads > BK || a->page_size <= 0 || a->num_page_entries < 0 || a->num_tokens < 0)
    return 0;
  return make_layout(a).bytes;
}

extern "C" int akt_attention_weights(const akt_attention_weights_args* a, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_args(a);
  if (rc || a->batch == 0) return rc;
  const Layout y = make_layout(a);
  if (!workspace || workspace_bytes < y.bytes)
    return set_error(AKT_ERR_WORKSPACE, "attention_weights: workspace of " + std::to_string(y.bytes) + " bytes required");
  WeightsParams p{};
  p.q = static_cast<const char*>(a->q);
  p.q_indptr = a->q_indptr;
  p.num_tokens = a->num_tokens;
  p.kv = static_cast<const char*>(a->kv_cache);
  p.s_page = a->kv_stride_page * 2;
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
  p.Hkv = a->num_kv_heads;
  p.group = a->num_qo_heads / a->num_kv_heads;
  p.P = a->page_size;
  p.causal = a->causal ? 1 : 0;
  p.width = (int)a->width;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.TQ = BK / p.group;
  p.div_group = make_fastdiv((uint32_t)p.group);
  p.div_page = make_fastdiv((uint32_t)p.P);
  p.grid = y.grid;
  p.parts = static_cast<Part*>(workspace);
  p.part_sum = reinterpret_cast<float*>(static_cast<char*>(workspace) + y.sums);
  // a box holds keys of one page: the largest power of two from 8 (the swizzle's
  // row period) to 128 that divides the page size
  p.box_rows = 0;
  for (int r = 128; r >= 8 && !p.box_rows; r >>= 1)
    if (p.P % r == 0) p.box_rows = r;
  if (p.num_pages == 0) p.box_rows = 0;
  CUtensorMap mq{}, mk{};
  if (a->num_tokens > 0) {
    const cuuint64_t qd[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)p.group, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_tokens};
    const int64_t qs[3] = {a->q_stride_head * 2, a->q_stride_head * 2 * p.group, a->q_stride_token * 2};
    const cuuint32_t qb[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)p.TQ};
    rc = make_map(&mq, a->q, a->dtype, 4, qd, qs, qb);
  }
  if (!rc && p.box_rows) {
    const cuuint64_t halves = (cuuint64_t)(a->head_dim / 64);
    // Heads, K and V, and pages in one run (a contiguous pool): one dimension counts them, and a box takes all
    // 8-row groups of its keys.  Other strides take two dimensions and a box 8 rows.
    const int64_t s_kv = a->kv_stride_kv * 2;
    p.linear = s_kv == p.s_head * p.Hkv && p.s_page == 2 * s_kv && p.num_pages * 2 * p.Hkv < 0x7fff0000;
    if (p.linear) {
      const cuuint64_t kd[5] = {64, 8, halves, (cuuint64_t)(p.P / 8), (cuuint64_t)(p.num_pages * 2 * p.Hkv)};
      const int64_t ks[4] = {p.s_tok, 128, 8 * p.s_tok, p.s_head};
      const cuuint32_t kb[5] = {64, 8, (cuuint32_t)halves, (cuuint32_t)(p.box_rows / 8), 1};
      rc = make_map(&mk, p.kv, a->dtype, 5, kd, ks, kb);
    } else {
      p.box_rows = 8;
      const cuuint64_t kd[5] = {64, (cuuint64_t)p.P, halves, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_pages};
      const int64_t ks[4] = {p.s_tok, 128, p.s_head, p.s_page};
      const cuuint32_t kb[5] = {64, 8, (cuuint32_t)halves, 1, 1};
      rc = make_map(&mk, p.kv, a->dtype, 5, kd, ks, kb);
    }
  }
  if (rc) return rc;
  // only a sequence of several row tiles can have units in parts
  const bool parts = a->num_tokens > 2 * p.TQ;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == AKT_FLOAT16)
    return a->head_dim == 64 ? dispatch_weights<__half, 64>(mq, mk, p, parts, st)
                             : dispatch_weights<__half, 128>(mq, mk, p, parts, st);
  return a->head_dim == 64 ? dispatch_weights<__nv_bfloat16, 64>(mq, mk, p, parts, st)
                           : dispatch_weights<__nv_bfloat16, 128>(mq, mk, p, parts, st);
}
