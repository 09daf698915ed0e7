// Attention of a chunk of new tokens over a paged cache, on the 5th-generation
// tensor cores (tcgen05 + TMEM): prompt chunks, drafted tokens to verify and
// single tokens, ragged in one batch.  The reference has the one-token form only
// (decode_flash_attention_redundant_var_len_paged.py:228-274).
//
// O_i = sum_j softmax_j(q_i . k_j s) v_j over the keys j that row i sees; row i
// of sequence b stands at position len_b - n_b + i.  One pass over the keys with
// the softmax's running maximum and sum in fp32; P is rounded to the input type
// before P.V, as in the reference's decode (DP:39-57).
//
// Rows and units.  The G query heads of a kv head share K and V, so a 128-row
// tile holds TQ = floor(128 / G) tokens x G heads (row = token * G + head) and
// each K/V row is read once for all of them.  A unit is (sequence, kv head, 2 TQ
// consecutive tokens): two tiles ("slots") that share every K/V tile of 128
// keys.  A unit whose rows fit one tile (decoding, verification) puts the same
// rows in both slots and gives slot t every other key tile: the two slots'
// (O, max, sum) are joined from TMEM at its end.
//
// Work split.  The units' key tiles stand on a line, (sequence, kv head, unit).
// Whole units are dealt to the CTAs (one per SM) round by round while no CTA
// gets more than its share of all tiles; the rest of the line is cut so that
// every CTA ends with the same count, also inside a unit.  A unit in parts
// leaves its normalised fp32 partial outputs and log-sum-exps in the workspace
// (at most two parts per CTA), which chunk_merge_kernel joins.  So one long
// sequence of one token fills the GPU and a batch of prompts has no tail.
//
// Warps of a CTA (12):
//   0-3 / 4-7  softmax of slot 0 / 1: thread i owns row i = TMEM lane i
//   8 / 11     loaders of K / of V and Q into a ring of tiles: tensor-map boxes inside
//              the pages, or 16-byte cp.async rows where no box fits a page (TMA template);
//              a unit's few rows of Q come by plain loads, the rest of their tile cleared
//   9          issuer of both slots' MMAs (one elected lane)
//   10         scheduler: the CTA's segments, a few ahead, through shared memory;
//              and the V tiles at the mask's edge (below)
// TMEM (512 columns): S[2] (128 each), O[2] (D each).  P_t overwrites S_t: a
// slot's MMAs are issued in the order S_j, P.V_j, S_j+1, and while one slot's
// softmax runs the tensor pipe works for the other.
//
// What lies behind the mask.  Scores are masked by selection, so K may hold
// anything there.  A masked weight is 0, but 0 x NaN is NaN in P.V, so in V tiles
// that a mask crosses the rows past the sequence are cleared, and values that are
// not finite are cleared and their tokens noted; a row that does see such a token
// gets the value added to its output at the end.
//
// Bounds and measured rates (fp16, 32 query heads on 8, pages of 16 keys, full clock).
// Long prompts: the tensor pipe and the exponentials, 60 % busy each; 8192 tokens on top
// of 24576, D = 128, 3.01 ms = 1280 TFLOP/s (D = 64: 2.53 ms).  Short prompts also their
// units' ends and the causal edge: 8 of 2048 tokens, 295 us.  Few tokens: HBM; 5 in each
// of 64 sequences of 512 to 32768 keys, 655 us = 6.66 TB/s.
//
// Built without -rdc (setmaxnreg needs whole-program device code).
#define AKT_WHOLE_PROGRAM 1
#include "common.cuh"
#include "profile.cuh"
#include "tensor_map.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

constexpr int BM = 128;            // rows of a slot
constexpr int BN = 128;            // keys of a tile
constexpr int kThreads = 384;
constexpr int kLoadWarp = 8;       // K
constexpr int kMmaWarp = 9;
constexpr int kSchedWarp = 10;
constexpr int kLoadVWarp = 11;     // V and Q
// 2 * 128 * 208 + 128 * 80 <= 384 * 168 registers (no spills; 216 and 64 spill a little)
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kControlRegs = 80;
static_assert(256 * kSoftmaxRegs + 128 * kControlRegs <= kThreads * kLaunchRegs, "register split");
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kSegs = 4;           // segments in flight between the scheduler and the others
constexpr int kSegReaders = 12;    // 2 loaders, issuer, 8 softmax warps, scheduler (its V duty)
// A unit's start and end (Q, the first tile's chain, the output), in key tiles:
// of one tile of rows, of two.  A verification of 5 tokens in 64 sequences of 512
// to 32768: without it the CTAs with the short sequences were last, 1025 us; with
// 2 and 2 787, 6 and 1 682, 6 and 3 680, 8 and 3 686.  Eight prompts of 2048 tokens:
// 451, then 400, 414, 398, 390.  (All before the later steps; see the rates above.)
constexpr int kUnitCost1 = 6, kUnitCost2 = 3;
// A unit with at most this many rows gets the rest of its Q tiles cleared; the
// tensor map would fill it with the following sequences' rows, whose products nobody
// reads but which draw power.  n tokens of 4 heads in each of 64 sequences of 512 to
// 32768 keys, first calls / repeated for a second under the power cap: n = 1 644 / 695 us
// (map: 652 / 736), 5 659 / 710 (667 / 780), 12 (48 rows) 673 / 758 (686 / 800); 16 rows
// more take a warp's copy too long at a unit's start: 718 / 765 (685 / 810), n = 32
// 920 / 969 (718 / 852).
constexpr int kFewRows = 48;
constexpr int kTableSeqs = 96;     // sequences whose table fits the CTA's shared memory
constexpr int kMaxCtas = kThreads; // of the main kernel (one per SM)

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
  int B, Hq, Hkv, group, P, causal, D;
  float scale_log2;
  int TQ;             // tokens of a slot
  FastDiv div_group;  // row -> (token, head)
  FastDiv div_page;   // key -> (page, row)
  int box_rows;       // keys of one tensor-map box (divides the page size), TMA loads
  int linear;         // pages, K and V, and heads follow one another with one stride
  int grid;           // CTAs of the main kernel
  // workspace
  struct Part* parts;  // [grid][2]
  float* part_o;       // [grid][2][part_rows][D]
  float* part_lse;     // [grid][2][part_rows] natural log, -inf: no key
  int part_rows;
  int merge_rows;      // rows of a CTA of the merge
  // tables in the workspace, for more than kTableSeqs sequences
  int64_t* plan_cost;  // [B + 1]
  int* plan_units;     // [B + 1]
  struct Plan* plan;
  int64_t* plan_share; // [grid + 1]
};

// A unit's part that one CTA left in the workspace (written for both of a
// CTA's places; keys == 0: none).
struct Part {
  int used, first, last;  // whether it is one; the unit's first / last keys
  int q0, ntok, kvh, single, pad;
};

// How the line of units is dealt: rounds of whole units, then the cuts.
struct Plan {
  int64_t base;  // tiles of the dealt units: where the cut part of the line starts
  int rounds;
};

// A run of key tiles of one unit for one CTA.
struct Seg {
  int q0;      // the unit's first row of q (token); -1: no more segments
  int ntok;    // its tokens
  int vis0;    // keys that the first token sees
  int kvh;
  int page0;   // the sequence's first entry of the index array
  int len;     // its keys
  int t0, t1;  // key tiles
  int n0, n1;  // how many of them slot 0 and slot 1 take
  int single;  // one tile of rows: the slots take turns at the key tiles
  int part;    // -1: the whole unit; else the place of the partial result
  int noted;   // tokens in `bad`
  int pad[3];
  uint32_t bad[3][BN / 32];  // tokens from tile vis0 / BN on whose V row is not finite
};

template <int D>
struct Cfg {
  static constexpr int DB = D / 64;  // 64-column (128-byte) swizzle blocks of a row
  static constexpr int COL_S = 0, COL_O = 2 * BN, TMEM_COLS = 512;
  static_assert(COL_O + 2 * D <= TMEM_COLS, "TMEM budget");
  static constexpr uint32_t Q_BYTES = BM * D * 2, KV_BYTES = BN * D * 2;
  // a K or V tile: per 8 keys, per 64 columns, 8 rows of 128 bytes (swizzled)
  static constexpr uint32_t HALF = 1024, GROUP = DB * 1024;
  static constexpr int NS = D == 64 ? 11 : 5;  // ring stages
  static constexpr uint32_t OFF_Q = 0, OFF_KV = 2 * Q_BYTES, OFF_BAR = OFF_KV + NS * KV_BYTES;
  // full, empty, ready [NS]; q_full, q_empty, s_full, p_full, o_full [slot]; seg_full,
  // seg_empty [kSegs]; join (slot 1 done), joined; mma_idle
  static constexpr int N_BARS = 3 * NS + 10 + 2 * kSegs + 3;
  static constexpr uint32_t OFF_MISC = OFF_BAR + (N_BARS * 8 + 15) / 16 * 16;  // TMEM address, abort flag
  static constexpr uint32_t OFF_SEG = OFF_MISC + 16;
  static constexpr uint32_t OFF_TABLE = OFF_SEG + kSegs * sizeof(Seg);
  static constexpr uint32_t SMEM = OFF_TABLE + (kTableSeqs + 1) * 12 + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  // slot 1's maxima and sums for the join, in the ring's place of nothing else
  static constexpr uint32_t OFF_STAT = (SMEM + 15) / 16 * 16;
  static constexpr uint32_t SMEM_ALL = OFF_STAT + 2 * BM * 4;
  static_assert(SMEM_ALL <= 227 * 1024, "shared memory budget");
};

// -------------------------------------------------------------------------
// the sequences and their units
// -------------------------------------------------------------------------
struct Seq {
  int a0, n, page0, len;  // first row of q, queries, first index entry, keys
};

// Sequence b's bounds; a malformed one is empty (recorded by the planner).
__device__ __forceinline__ Seq load_seq(const ChunkParams& p, int b, bool record) {
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
  return s;
}

__device__ __forceinline__ int num_units(const ChunkParams& p, const Seq& s) {
  return s.n ? (s.n - 1) / (2 * p.TQ) + 1 : 0;
}

// Key tiles of unit u, and what it costs on the line
__device__ __forceinline__ int unit_tiles(const ChunkParams& p, const Seq& s, int u) {
  const int vis = p.causal ? s.len - s.n + min((u + 1) * 2 * p.TQ, s.n) : s.len;
  return vis > 0 ? (vis - 1) / BN + 1 : 0;
}
__device__ __forceinline__ int unit_extra(const ChunkParams& p, const Seq& s, int u) {
  return s.n - u * 2 * p.TQ <= p.TQ ? kUnitCost1 : kUnitCost2;
}
__device__ __forceinline__ int unit_cost(const ChunkParams& p, const Seq& s, int u) {
  return unit_extra(p, s, u) + unit_tiles(p, s, u);
}

// Tables: cost[b] and units[b] count the tiles and units before sequence b; seqs
// (or null) holds the sequences while the plan is made.
struct Tables {
  const int64_t* cost;
  const int* units;
  const Seq* seqs;
};

// Largest b in [0, B) with t[b] <= x (the entry that holds x; empty ones are passed over).
template <typename V>
__device__ __forceinline__ int find_seq(const V* t, int B, V x) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Unit i of the line: its sequence, kv head and number (a sequence's units run
// from the last, longest one down).
__device__ __forceinline__ void unit_at(const ChunkParams& p, const Tables& t, int i, int& b, Seq& s, int& kvh, int& u) {
  b = find_seq(t.units, p.B, i);
  s = load_seq(p, b, false);
  const int U = num_units(p, s), r = i - t.units[b];
  kvh = r / U;
  u = U - 1 - (r - kvh * U);
}

// Fills the tables (threads of one CTA, `nthreads` of them; cost and units in
// shared or global memory), and the costliest unit's cost, no less, into
// *most_cost (shared memory).
__device__ void build_tables(const ChunkParams& p, int64_t* cost, int* units, Seq* seqs, int* most_cost, int nthreads) {
  if (threadIdx.x == 0) *most_cost = 1;
  __syncthreads();
  // a team of threads per sequence sums its units' costs
  int team = 32;
  while (team > 1 && (nthreads / team) < p.B) team >>= 1;
  const int lane = threadIdx.x % team;
  for (int b0 = 0; b0 < p.B; b0 += nthreads / team) {
    const int b = b0 + threadIdx.x / team;
    int U = 0;
    int64_t c = 0;
    Seq s{};
    if (b < p.B) {
      s = load_seq(p, b, lane == 0);
      U = num_units(p, s);
      for (int u = lane; u < U; u += team) c += unit_cost(p, s, u);
    }
    for (int o = team >> 1; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if (b < p.B && lane == 0) {
      cost[b + 1] = c * p.Hkv;
      units[b + 1] = U * p.Hkv;
      if (seqs) seqs[b] = s;
      if (U) atomicMax(most_cost, unit_tiles(p, s, U - 1) + max(kUnitCost1, kUnitCost2));
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // running sums
    int64_t c0 = 0;
    int u0 = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + threadIdx.x;
      int64_t c = b < p.B ? cost[b + 1] : 0;
      int u = b < p.B ? units[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t cy = __shfl_up_sync(0xffffffffu, c, o);
        const int uy = __shfl_up_sync(0xffffffffu, u, o);
        if (threadIdx.x >= o) {
          c += cy;
          u += uy;
        }
      }
      if (b < p.B) {
        cost[b + 1] = c0 + c;
        units[b + 1] = u0 + u;
      }
      c0 += __shfl_sync(0xffffffffu, c, 31);
      u0 += __shfl_sync(0xffffffffu, u, 31);
    }
    if (threadIdx.x == 0) {
      cost[0] = 0;
      units[0] = 0;
    }
  }
  __syncthreads();
}

// The unit that CTA c gets in round r of whole units: rounds run left to right
// and right to left in turn, which evens out costs that fall along the line.
__device__ __forceinline__ int dealt_unit(const ChunkParams& p, int r, int c) {
  return r * p.grid + ((r & 1) ? p.grid - 1 - c : c);
}

// a / b, by the short division where both fit 32 bits
__device__ __forceinline__ int64_t div_small(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Deals whole units and cuts the rest (at least p.grid threads of one CTA, all
// call it).  share[c] .. share[c + 1] is CTA c's range of the cut part, in tiles
// from plan.base.  scratch: an int64 per 32 CTAs.
__device__ Plan make_plan(const ChunkParams& p, const Tables& t, int most_cost, int64_t* share, int* scratch) {
  const int64_t W = t.cost[p.B];
  const int N = t.units[p.B], c = threadIdx.x;
  const int64_t per = div_small(W, p.grid), left = W - per * p.grid;
  const int64_t target = per + (left ? 1 : 0);
  Plan pl{0, 0};
  int64_t mine = 0;
  // Dealing pays by the CTAs of a round sharing K/V tiles in L2 and by fewer
  // parts; with one unit per (sequence, kv head) there is nothing to share.
  // Rounds that cannot pass the target (all units as dear as the dearest) take no
  // barrier; a thread's units run up the line, so it walks the sequences once.
  const int most = N > (int64_t)p.B * p.Hkv ? N / p.grid : 0;
  const int safe = (int)min((int64_t)most, div_small(target, most_cost));
  int end = 0, start = 0, U = 1;
  Seq s{};
  auto cost_in_round = [&](int r) -> int {
    const int i = dealt_unit(p, r, c);
    if (i >= end) {
      const int b = find_seq(t.units, p.B, i);
      start = t.units[b];
      end = t.units[b + 1];
      s = t.seqs ? t.seqs[b] : load_seq(p, b, false);
      U = num_units(p, s);
    }
    return unit_cost(p, s, U - 1 - (i - start) % U);
  };
  if (c < p.grid)
    for (int r = 0; r < safe; ++r) mine += cost_in_round(r);
  for (pl.rounds = safe; pl.rounds < most; ++pl.rounds) {
    const int cost = c < p.grid ? cost_in_round(pl.rounds) : 0;
    if (__syncthreads_or(mine + cost > target)) break;
    mine += cost;
  }
  if (!pl.rounds) {  // everything is cut: c W / grid, to the tile
    if (c <= p.grid) share[c] = c * per + (int64_t)((uint32_t)(c * left) / (uint32_t)p.grid);
    __syncthreads();
    return pl;
  }
  // each CTA's range is what it lacks of the target (the sums of the lacks are
  // below W; the rounding of the target, less than a tile a CTA, is the last ones' gain)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = c < p.grid ? target - mine : 0;
  const int64_t lack = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  int64_t* sums = reinterpret_cast<int64_t*>(scratch);  // of the first warps
  const int warps = (p.grid + 31) / 32;
  if (lane == 31 && warp < warps) sums[warp] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    before += w < warp ? sums[w] : 0;
    all += sums[w];
  }
  pl.base = p.grid * target - all;
  const int64_t rest = W - pl.base;
  if (c < p.grid) share[c] = min(before + x - lack, rest);
  if (c == p.grid) share[c] = rest;
  __syncthreads();
  return pl;
}

// Order of a segment's n tiles in the ring: K0, K1, V0, K2, V1, ... V(n-1).  V
// comes a tile after its K (it is needed a softmax later), so stages hold what
// is wanted soon.  Load of tile i's K and V:
__device__ __forceinline__ uint32_t ring_k(int i) { return i ? 2 * i - 1 : 0; }
__device__ __forceinline__ uint32_t ring_v(int i, int n) { return i + 1 < n ? 2 * i + 2 : 2 * i + 1; }

// -------------------------------------------------------------------------
// PTX helpers
// -------------------------------------------------------------------------
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version for sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

__host__ __device__ constexpr uint32_t idesc_f16(int fmt, int M, int N, int b_mn_major) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)b_mn_major << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int y, int z, int w, int v, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}

// 16 bytes global -> shared, or zeros when src_bytes is 0
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// an arrival on bar when this thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// generic-proxy writes to shared memory before later async-proxy reads (the MMAs)
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// whether the phase with this parity has completed, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Slow path of a bounded mbarrier wait: every 256 polls it gives up if another
// role of the CTA has, or, after kWaitLimitNs, records kStatusWaitTimeout and
// raises the abort flag itself.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 255u) == 0u) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        record_status(kStatusWaitTimeout);
        *abort_flag = 1;
        return false;
      }
    }
  }
}

__device__ __noinline__ bool wait_or_abort_call(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return wait_or_abort(bar, parity, abort_flag);
}

// Values of w that are not finite: bit 15 of each half, whose exponent is all ones
// exactly when adding one to it carries out
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((w & e) + one) & 0x80008000u;
}
// w without them
template <typename T>
__device__ __forceinline__ uint32_t without_not_finite2(uint32_t w) {
  const uint32_t m = not_finite2<T>(w) >> 15;
  return w & ~(m * 0xffffu);
}

// The rare end of a row that sees tokens whose V row is not finite (their
// values were cleared for the MMAs): each such value added to the output.
template <typename T, int D, typename O>
__device__ __forceinline__ void add_not_finite(const ChunkParams& p, const Seg& sg, int vis, O* row) {
  const int first = max(sg.vis0, 0) / BN * BN;
#pragma unroll 1
  for (int i = 0; i < 3 * BN; ++i) {
    if (!(sg.bad[i / BN][(i / 32) % (BN / 32)] >> (i & 31) & 1u)) continue;
    const int key = first + i;
    if (key >= vis) continue;
    const int pg = (int)fdiv((uint32_t)key, p.div_page);
    const int page = __ldg(p.indices + sg.page0 + pg);
    if (page < 0 || page >= p.num_pages) continue;
    const T* v = reinterpret_cast<const T*>(p.kv + (int64_t)page * p.s_page + p.s_kv + (int64_t)sg.kvh * p.s_head +
                                            (int64_t)(key - pg * p.P) * p.s_tok);
#pragma unroll 1
    for (int d = 0; d < D; ++d) {
      const float x = Elem<T>::to_float(v[d]);
      if (!isfinite(x)) {
        if constexpr (std::is_same<O, float>::value) row[d] += x;
        else row[d] = Elem<T>::from_float(Elem<T>::to_float(row[d]) + x);
      }
    }
  }
}

// A warp's fill of the slots' Q tiles with a unit's rows and zeros up to row
// `clear`, in the tiles' swizzled layout.
template <int D>
__device__ __forceinline__ void load_few_rows(const ChunkParams& p, unsigned char* tiles, int q0, int kvh, int rows,
                                              int clear, bool slot0, bool slot1) {
  constexpr int PIECES = D / 8, U = 4;
  const char* q = p.q + (int64_t)q0 * p.q_tok + (int64_t)kvh * p.group * p.q_head;
  for (int i0 = threadIdx.x & 31; i0 < clear * PIECES; i0 += 32 * U) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 32 * u, row = i / PIECES, tok = (int)fdiv((uint32_t)row, p.div_group);
      v[u] = make_uint4(0, 0, 0, 0);
      if (row < rows)
        v[u] = __ldg(reinterpret_cast<const uint4*>(q + tok * p.q_tok + (row - tok * p.group) * p.q_head) + i % PIECES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 32 * u, row = i / PIECES, c = i % PIECES;
      if (row >= clear) continue;
      unsigned char* dst = tiles + (c >> 3) * (BM * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
      if (slot0) *reinterpret_cast<uint4*>(dst) = v[u];
      if (slot1) *reinterpret_cast<uint4*>(dst + BM * D * 2) = v[u];
    }
  }
  fence_async_smem();
}

// 4 x 4 pieces of 16 bytes turned over four lanes: v[i] is piece i of this lane's
// row and becomes piece (lane % 4) of row i of its four lanes.
__device__ __forceinline__ void turn_pieces(uint4 (&v)[4]) {
  const int lane = threadIdx.x & 31;
  auto swap = [&](uint4& keep_low, uint4& keep_high, bool high, int o) {
    // the lane with the bit set gives its low piece for the other's high one
    uint4 x = high ? keep_low : keep_high;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, o);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, o);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, o);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, o);
    if (high) keep_low = x; else keep_high = x;
  };
  swap(v[0], v[1], lane & 1, 1);
  swap(v[2], v[3], lane & 1, 1);
  swap(v[0], v[2], lane & 2, 2);
  swap(v[1], v[3], lane & 2, 2);
}

// The end of a softmax warp's rows of a segment: O = w0 O_t (+ w1 O_1 where the
// slots are joined), normalised, to the output or to the segment's partial
// result.  flags: 1 the slot has an output of its own, 2 slot 1's is added.  A
// function of its own: what it needs is read again from the segment, so the key
// loop has its registers.  A thread holds a row; four lanes exchange 16-byte
// pieces so that a store covers 64 bytes of each of 8 rows (each thread storing
// its own row, 16 bytes of 32 rows at a time, took 6.8K cycles at D = 128).
template <typename T, int D>
__device__ __forceinline__ void finish_rows(const ChunkParams& p, const Seg* sg, uint32_t tO, int t, float w0, float w1,
                                         float row_lse, int flags) {
  const int r = threadIdx.x & (BM - 1), rtok = (int)fdiv((uint32_t)r, p.div_group);
  const bool single = sg->single;
  const int tok = (single ? 0 : t * p.TQ) + rtok, part = sg->part, head = sg->kvh * p.group + r - rtok * p.group;
  const bool valid = rtok < p.TQ && tok < sg->ntok;
  const int64_t grow = (int64_t)sg->q0 + tok;
  const int64_t pidx = ((int64_t)(2 * blockIdx.x) + max(part, 0)) * p.part_rows + (single ? 0 : t * BM) + r;
  char* mine = valid ? (part < 0 ? p.out + grow * p.o_tok + (int64_t)head * p.o_head
                                 : reinterpret_cast<char*>(p.part_o + pidx * D))
                     : nullptr;
  char* row[4];  // the four lanes' rows, at this lane's piece
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    row[i] = reinterpret_cast<char*>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), (threadIdx.x & 28) + i));
    if (row[i]) row[i] += (threadIdx.x & 3) * 16;
  }
  const bool take0 = __any_sync(0xffffffffu, flags & 1), take1 = __any_sync(0xffffffffu, flags & 2);
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t a[32];
    float o[32];
    if (take0) {
      tmem_ld32(tO + t * D + c * 32, a);
      tmem_wait_ld();
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = flags & 1 ? __uint_as_float(a[e]) * w0 : 0.f;
    if (take1) {
      tmem_ld32(tO + D + c * 32, a);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = flags & 2 ? fmaf(__uint_as_float(a[e]), w1, o[e]) : o[e];
    }
    uint4 v[4];
    if (part < 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = make_uint4(Elem<T>::pack2(o[8 * e], o[8 * e + 1]), Elem<T>::pack2(o[8 * e + 2], o[8 * e + 3]),
                          Elem<T>::pack2(o[8 * e + 4], o[8 * e + 5]), Elem<T>::pack2(o[8 * e + 6], o[8 * e + 7]));
      turn_pieces(v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row[i]) *reinterpret_cast<uint4*>(row[i] + c * 64) = v[i];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = make_uint4(__float_as_uint(o[16 * h + 4 * e]), __float_as_uint(o[16 * h + 4 * e + 1]),
                            __float_as_uint(o[16 * h + 4 * e + 2]), __float_as_uint(o[16 * h + 4 * e + 3]));
        turn_pieces(v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row[i]) *reinterpret_cast<uint4*>(row[i] + c * 128 + h * 64) = v[i];
      }
    }
  }
  if (valid) {
    if (part >= 0) p.part_lse[pidx] = row_lse;
    else if (p.lse) p.lse[grow * p.l_tok + (int64_t)head * p.l_head] = row_lse;
  }
  if (sg->noted) {
    __syncwarp();  // the row was stored by four lanes
    const int vis = sg->vis0 + tok;
    if (valid && part < 0) add_not_finite<T, D, T>(p, *sg, vis, reinterpret_cast<T*>(mine));
    if (valid && part >= 0) add_not_finite<T, D, float>(p, *sg, vis, reinterpret_cast<float*>(mine));
  }
}

// -------------------------------------------------------------------------
// the planner of batches past the CTA's own table
// -------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) chunk_plan_kernel(const ChunkParams p) {
  __shared__ __align__(8) int scratch[64];
  __shared__ int most_cost;
  build_tables(p, p.plan_cost, p.plan_units, nullptr, &most_cost, 1024);
  const Plan pl = make_plan(p, Tables{p.plan_cost, p.plan_units, nullptr}, most_cost, p.plan_share, scratch);
  if (threadIdx.x == 0) *p.plan = pl;
}

// -------------------------------------------------------------------------
// main kernel
// -------------------------------------------------------------------------
template <typename T, int D, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ ChunkParams p) {
  using C = Cfg<D>;
  constexpr int NS = C::NS;
  constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
  constexpr uint32_t IDESC_S = idesc_f16(fmt, BM, BN, 0);
  constexpr uint32_t IDESC_PV = idesc_f16(fmt, BM, D, 1);

  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;             // [NS] loaded
  uint64_t* empty = full + NS;       // [NS] the issuer and the scheduler warp done with it
  uint64_t* ready = empty + NS;      // [NS] seen (and, for V at a mask's edge, cleaned) by the scheduler warp
  uint64_t* q_full = ready + NS;     // [slot]
  uint64_t* q_empty = q_full + 2;    // [slot]
  uint64_t* s_full = q_empty + 2;    // [slot]
  uint64_t* p_full = s_full + 2;     // [slot]
  uint64_t* o_full = p_full + 2;     // [slot] the segment's last P.V is done
  uint64_t* seg_full = o_full + 2;   // [kSegs]
  uint64_t* seg_empty = seg_full + kSegs;
  uint64_t* join = seg_empty + kSegs;  // slot 1's statistics are in shared memory
  uint64_t* joined = join + 1;         // slot 0 has read slot 1's output
  uint64_t* mma_idle = joined + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Seg* segs = reinterpret_cast<Seg*>(smem + C::OFF_SEG);
  float* stat = reinterpret_cast<float*>(smem + C::OFF_STAT);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], TMA ? 1 : 32);  // cp.async: every lane of the loader
      mbar_init(&empty[s], 2);
      mbar_init(&ready[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], kSegReaders);
    }
    mbar_init(join, 4);
    mbar_init(joined, 4);
    mbar_init(mma_idle, 1);
    *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;  // swizzled tiles need a 1024-byte aligned base
    if (*abort_flag) record_status(kStatusWaitTimeout);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "n"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the tables and the plan: built by every CTA for itself, or read from the planner's
  int64_t begin, end;
  Plan plan;
  Tables tab;
  if (p.B <= kTableSeqs) {
    int64_t* cost = reinterpret_cast<int64_t*>(smem + C::OFF_TABLE);
    int* units = reinterpret_cast<int*>(cost + p.B + 1);
    // the shares live where slot 0's Q tile goes later
    int64_t* share = reinterpret_cast<int64_t*>(smem + C::OFF_Q);
    int* scratch = reinterpret_cast<int*>(share + p.grid + 1);
    Seq* seqs = reinterpret_cast<Seq*>(smem + C::OFF_Q + 8192);
    build_tables(p, cost, units, seqs, scratch + 63, kThreads);
    tab = Tables{cost, units, seqs};
    plan = make_plan(p, tab, scratch[63], share, scratch);
    begin = share[blockIdx.x];
    end = share[blockIdx.x + 1];
    // generic reads before the async-proxy writes of the Q tile
    fence_async_smem();
  } else {
    grid_dep_wait();
    tab = Tables{p.plan_cost, p.plan_units, nullptr};
    plan = *p.plan;
    begin = p.plan_share[blockIdx.x];
    end = p.plan_share[blockIdx.x + 1];
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    return wait_or_abort(bar, parity, abort_flag);
  };
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      if (mbar_try_wait(bar, parity)) return true;
      return wait_or_abort_call(bar, parity, abort_flag);
    };
    if (warp == kSchedWarp) {
      // ===================== scheduler, and V at the mask's edge =====================
      int round = 0;               // rounds of whole units done
      int64_t x = plan.base + begin;
      const int64_t x_end = plan.base + end;
      int b = -1, kvh = 0, u = 0, U = 0, stream = 0;  // the line's current unit
      int64_t unit_x = 0;          // where it starts
      Seq s{};
      int n_pub = 0;
      bool ok = true, more = true;
      // the next segment into ring place n_pub; false when there was none left
      auto publish = [&]() -> void {
        Seg sg{};
        sg.q0 = -1;
        if (round < plan.rounds) {
          int bb, k, uu;
          Seq q;
          unit_at(p, tab, dealt_unit(p, round, blockIdx.x), bb, q, k, uu);
          ++round;
          const int X = 2 * p.TQ;
          sg.q0 = q.a0 + uu * X;
          sg.ntok = min(X, q.n - uu * X);
          sg.vis0 = p.causal ? q.len - q.n + uu * X + 1 : q.len;
          sg.kvh = k;
          sg.page0 = q.page0;
          sg.len = q.len;
          sg.t0 = 0;
          sg.t1 = unit_tiles(p, q, uu);
          sg.part = -1;
        } else {
          while (x < x_end) {
            if (b < 0) {  // the unit that holds x
              b = find_seq(tab.cost, p.B, x);
              s = load_seq(p, b, false);
              U = num_units(p, s);
              const int64_t per_head = div_small(tab.cost[b + 1] - tab.cost[b], p.Hkv);
              const int64_t rel = x - tab.cost[b];
              kvh = (int)div_small(rel, per_head);
              unit_x = tab.cost[b] + kvh * per_head;
              for (int i0 = 0;; i0 += 32) {  // 32 units at a time
                const int i = i0 + lane;
                int64_t c = i < U ? unit_cost(p, s, U - 1 - i) : 0, run = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                  const int64_t y = __shfl_up_sync(0xffffffffu, run, o);
                  if (lane >= o) run += y;
                }
                const unsigned m = __ballot_sync(0xffffffffu, i < U && unit_x + run > x);
                if (m || i0 + 32 >= U) {
                  const int at = m ? __ffs(m) - 1 : 31;
                  u = U - 1 - min(i0 + at, U - 1);
                  unit_x += __shfl_sync(0xffffffffu, run - c, at);
                  break;
                }
                unit_x += __shfl_sync(0xffffffffu, run, 31);
              }
            }
            const int X = 2 * p.TQ, nt = unit_tiles(p, s, u), extra = unit_extra(p, s, u), cost = extra + nt;
            const int to = (int)min(x_end - unit_x, (int64_t)cost);
            sg.t0 = max(0, (int)(x - unit_x) - extra);
            sg.t1 = max(0, to - extra);
            // a range with none of the unit's tiles leaves it to the others (a unit without
            // any is the last one's, which writes zeros)
            const bool some = nt ? sg.t0 < sg.t1 : to == cost;
            if (some) {
              sg.q0 = s.a0 + u * X;
              sg.ntok = min(X, s.n - u * X);
              sg.vis0 = p.causal ? s.len - s.n + u * X + 1 : s.len;
              sg.kvh = kvh;
              sg.page0 = s.page0;
              sg.len = s.len;
              const bool whole = sg.t1 - sg.t0 == nt;
              sg.part = whole ? -1 : (stream ? 1 : 0);
              if (!whole && lane == 0) {
                Part& pt = p.parts[2 * blockIdx.x + sg.part];
                pt.used = 1;
                pt.first = sg.t0 == 0;
                pt.last = sg.t1 == nt;
                pt.q0 = sg.q0;
                pt.ntok = sg.ntok;
                pt.kvh = kvh;
                pt.single = sg.ntok <= p.TQ;
              }
              ++stream;
            }
            x = unit_x + to;
            if (to == cost) {  // on to the next unit of the line
              unit_x = x;
              if (u > 0) {
                --u;
              } else if (kvh + 1 < p.Hkv) {
                ++kvh;
                u = U - 1;
              } else {
                b = -1;
              }
            }
            if (some) break;
          }
        }
        sg.single = sg.ntok <= p.TQ;
        const int n = sg.t1 - sg.t0;
        if (sg.single) {
          sg.n0 = (n + 1) >> 1;
          sg.n1 = n >> 1;
        } else {  // slot 1 holds the unit's last token, slot 0's may see fewer keys
          const int vis = p.causal ? sg.vis0 + p.TQ - 1 : sg.len;
          sg.n0 = max(0, min(sg.t1, vis > 0 ? (vis - 1) / BN + 1 : 0) - sg.t0);
          sg.n1 = n;
        }
        more = sg.q0 >= 0;
        if (!more) sg.n1 = -1;
        const int e = n_pub % kSegs;
        if (n_pub >= kSegs && !wait(&seg_empty[e], ((n_pub / kSegs) - 1) & 1)) {
          ok = false;
          return;
        }
        if (lane == 0) {
          segs[e] = sg;
          mbar_arrive(&seg_full[e]);
        }
        __syncwarp();
        ++n_pub;
      };
      if (lane < 2) p.parts[2 * blockIdx.x + lane].used = 0;
      __syncwarp();
      uint32_t st = 0, ph = 0;
      publish();
      for (int k = 0; ok && k < n_pub; ++k) {
        if (more) publish();  // one ahead of the segment whose V tiles are looked at
        if (!ok) break;
        Seg* sg = &segs[k % kSegs];
        const int t0 = sg->t0, t1 = sg->t1, vis0 = sg->vis0, len = sg->len, j_edge = max(vis0, 0) / BN;
        if (sg->q0 < 0) break;
        const int loads = 2 * (t1 - t0);
#pragma unroll 1
        for (int i = 0; i < loads; ++i) {
          if (!wait(&full[st], ph)) {
            ok = false;
            break;
          }
          if (!TMA) {  // what the copies wrote, before the MMAs' reads
            fence_async_smem();
            __syncwarp();
          }
          // V tiles are the even loads from the third on, and the last one
          const int j = t0 + (i + 1 == loads ? (i >> 1) : (i >> 1) - 1);
          const bool is_v = i + 1 == loads || (i >= 2 && !(i & 1));
          if (is_v && ((p.causal && (j + 1) * BN > vis0) || (j + 1) * BN > len)) {
            // rows that every row of the unit sees stay as they are
            unsigned char* v = smem + C::OFF_KV + st * C::KV_BYTES;
            const int rows = len - j * BN;  // the others are past the sequence
            const int r0 = min(max(p.causal ? vis0 - j * BN : rows, 0), BN);
            constexpr int PR = D / 8, RS = 32 / PR;  // 16-byte pieces of a row, rows a step
            const int ch = lane % PR;
            unsigned char* vc = v + (ch >> 3) * C::HALF + (ch & 7) * 16;  // (the swizzle stays inside a row)
            auto at = [&](int r) { return reinterpret_cast<uint4*>(vc + (r >> 3) * C::GROUP + (r & 7) * 128); };
            const int top = min(rows, BN), mid = max(r0, top);
            for (int r = mid + lane / PR; r < BN; r += RS) *at(r) = make_uint4(0, 0, 0, 0);
            constexpr int U = 8;  // pieces at a time, one look (8 prompts of 2048 tokens, D = 128: 2 310 us, 4 301, 8 299, 16 299)
            for (int r = r0 + lane / PR; r < top; r += U * RS) {
              uint32_t any = 0;
#pragma unroll
              for (int u = 0; u < U; ++u) {  // (the last row again where there are no more)
                const uint4 y = *at(min(r + u * RS, top - 1));
                any |= not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w);
              }
              if (!any) continue;
#pragma unroll 1
              for (int q = r; q < min(r + U * RS, top); q += RS) {
                const uint4 y = *at(q);
                if (!(not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w))) continue;
                *at(q) = make_uint4(without_not_finite2<T>(y.x), without_not_finite2<T>(y.y),
                                    without_not_finite2<T>(y.z), without_not_finite2<T>(y.w));
                atomicOr(&sg->bad[j - j_edge][q >> 5], 1u << (q & 31));
                sg->noted = 1;
              }
            }
            fence_async_smem();
            __syncwarp();
          }
          if (lane == 0) {
            mbar_arrive(&ready[st]);
            // K too is refilled only once this warp has seen it: its view of the
            // barriers' phases must not fall a whole turn of the ring behind
            mbar_arrive(&empty[st]);
          }
          if (++st == NS) {
            st = 0;
            ph ^= 1u;
          }
        }
        if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
      }
    } else if (warp == kLoadWarp || warp == kLoadVWarp) {
      // ============================ K loader, V (and Q) loader ============================
      // A warp each: one warp's boxes (72 cycles apiece) took as long as a tile's whole turn.
      const int op = warp == kLoadVWarp;
      uint32_t base = 0, qn0 = 0, qn1 = 0;  // ring loads before the segment; Q loads
      int dirty = BM | BM << 8;             // rows of each slot's Q tile that are not zeros
      bool ok = true;
      const int boxes = TMA ? BN / p.box_rows : 0;  // of one tile, at most 16
      uint32_t loaded = 0;  // stages this warp has loaded (bits 0 ..) and the parity of the last load (16 ..)
      for (int k = 0; ok; ++k) {
        if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
        const Seg* sg = &segs[k % kSegs];
        const int q0 = sg->q0, t0 = sg->t0, t1 = sg->t1, kvh = sg->kvh, page0 = sg->page0, len = sg->len;
        const int single = sg->single, n0 = sg->n0, n1 = sg->n1, rows = sg->ntok * p.group;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
        if (q0 < 0) break;
        if (op && single && rows <= kFewRows) {  // the same few rows for both slots
          if ((n0 && qn0 && !wait(&q_empty[0], (qn0 - 1) & 1)) || (n1 && qn1 && !wait(&q_empty[1], (qn1 - 1) & 1))) break;
          load_few_rows<D>(p, smem + C::OFF_Q, q0, kvh, rows, max(rows, max(n0 ? dirty & 255 : 0, n1 ? dirty >> 8 : 0)),
                           n0, n1);
          __syncwarp();
          if (n0) {
            ++qn0;
            dirty = (dirty & ~255) | rows;
            if (lane == 0) mbar_arrive(&q_full[0]);
          }
          if (n1) {
            ++qn1;
            dirty = (dirty & 255) | rows << 8;
            if (lane == 0) mbar_arrive(&q_full[1]);
          }
        } else if (op) {  // Q of both slots: the buffer is free once the slot's last S before is done
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint32_t& qn = t ? qn1 : qn0;
            if (!(t ? n1 : n0)) continue;
            if (qn && !wait(&q_empty[t], (qn - 1) & 1)) {
              ok = false;
              break;
            }
            ++qn;
            dirty = t ? (dirty & 255) | BM << 8 : (dirty & ~255) | BM;
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[t], (uint32_t)(p.TQ * p.group * 128 * C::DB));
#pragma unroll
              for (int db = 0; db < C::DB; ++db)
                tma_load_4d(smem + C::OFF_Q + t * C::Q_BYTES + db * (BM * 128), &tmQ, db * 64, 0, kvh,
                            q0 + (single ? 0 : t * p.TQ), &q_full[t]);
            }
          }
        }
        if constexpr (TMA) {
          // lane l loads box l of each tile: keys [rb, rb + box_rows) of the tile
          const int rb = lane * p.box_rows;
          const bool mine = lane < boxes;
          // the index entry of the box's page, a tile ahead of its use (the id is looked at then)
          auto entry = [&](int j) -> int {
            const int key = j * BN + rb;
            return mine && key < len ? __ldg(p.indices + page0 + (int)fdiv((uint32_t)key, p.div_page)) : -1;
          };
          int id_next = t0 < t1 ? entry(t0) : -1;
          for (int j = t0; ok && j < t1; ++j) {
            const int id = id_next, key = j * BN + rb;
            if (j + 1 < t1) id_next = entry(j + 1);
            const uint32_t g = base + (op ? ring_v(j - t0, t1 - t0) : ring_k(j - t0)), st = g % NS;
            if (g >= NS && !wait(&empty[st], ((g / NS) - 1) & 1)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&full[st], C::KV_BYTES);
            loaded = (loaded & ~(0x10001u << st)) | 1u << st | ((g / NS) & 1u) << (16 + st);
            __syncwarp();
            if (mine) {
              // boxes past the sequence, and of bad ids, are asked for past the pool: zeros
              const bool there = id >= 0 && id < p.num_pages;
              const int row = there ? key - (int)fdiv((uint32_t)key, p.div_page) * p.P : 0;
              const int page = there ? id : (int)p.num_pages;
              unsigned char* dst = smem + C::OFF_KV + st * C::KV_BYTES + (rb >> 3) * C::GROUP;
              if (p.linear)  // [block of a page, kv and head][8-row group][64 columns][row]
                tma_load_5d(dst, &tmK, 0, 0, row >> 3, (page * 2 + op) * p.Hkv + kvh, &full[st]);
              else  // [page][head][64 columns][row]
                tma_load_5d(dst, op ? &tmV : &tmK, row, 0, kvh, page, &full[st]);
              if (!there && key < len) record_status(kStatusBadPage);
            }
            __syncwarp();
          }
        } else {
          // every half warp (D = 128) or quarter (D = 64) copies whole rows in 16-byte pieces
          constexpr int CH = D / 8, RW = 32 / CH;  // pieces of a row; rows a step
          const int ch = lane % CH, rl = lane / CH;
          // the index entries of a tile's rows lane, lane + 32, ..., a tile ahead of their use
          int id_next[BN / 32];
          auto entries = [&](int j) {
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
              const int key = j * BN + i * 32 + lane;
              id_next[i] = key < len ? __ldg(p.indices + page0 + (int)fdiv((uint32_t)key, p.div_page)) : -1;
            }
          };
          if (t0 < t1) entries(t0);
          for (int j = t0; ok && j < t1; ++j) {
            const char* src[BN / 32];  // the rows' addresses (null: zeros)
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
              const int key = j * BN + i * 32 + lane, id = id_next[i];
              src[i] = nullptr;
              if (id >= 0 && id < p.num_pages)
                src[i] = p.kv + (op ? p.s_kv : 0) + (int64_t)id * p.s_page + (int64_t)kvh * p.s_head +
                         (int64_t)(key - (int)fdiv((uint32_t)key, p.div_page) * p.P) * p.s_tok;
              else if (key < len) record_status(kStatusBadPage);
            }
            if (j + 1 < t1) entries(j + 1);
            __syncwarp();
            const uint32_t g = base + (op ? ring_v(j - t0, t1 - t0) : ring_k(j - t0)), st = g % NS;
            if (g >= NS && !wait(&empty[st], ((g / NS) - 1) & 1)) {
              ok = false;
              break;
            }
            __syncwarp();
            const uint32_t tile = smem_u32(smem + C::OFF_KV + st * C::KV_BYTES);
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
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
            cp_async_arrive(&full[st]);  // each lane's arrival, once its copies have landed
          }
        }
        base += 2 * (t1 - t0);
      }
      if (*abort_flag && lane == 0) {  // loads still in flight into this CTA's shared memory
        if (TMA)
          for (int st = 0; st < NS; ++st)  // whichever phase a stage is in, its load (if any) ends it
            if (loaded >> st & 1u) mbar_wait(&full[st], loaded >> (16 + st) & 1u);
        if (qn0) mbar_wait(&q_full[0], (qn0 - 1) & 1);
        if (qn1) mbar_wait(&q_full[1], (qn1 - 1) & 1);
      }
      if (!TMA) cp_async_wait_all();
    } else {
      // ============================ MMA issuer ============================
      // One warp issues both slots' MMAs, the slots in turn: P.V of slot t's tile,
      // then S of its next tile (which overwrites that P).  So the slots' softmaxes
      // run half a period apart: with an issuer per slot their MMAs mixed in the pipe,
      // both waited for S at the same time and then fought for the exponentials
      // (5.1K cycles a tile pair).  The whole warp runs the control flow on values that
      // are the same in every lane (a reduction's result is a uniform register, which is
      // what the MMA takes its descriptors from) and an elected lane issues: 50 cycles
      // an MMA, against 117 from a branch of one lane.  A wait that is over already
      // costs 150 cycles, so the ring is asked once per load: `ready` comes in the order
      // of the loads, and what a later load has answered is known of the earlier ones.
      auto uni = [&](int v) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)v); };
      auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(bar, parity));
      };
      const uint64_t dk = desc_sw128(smem_u32(smem + C::OFF_KV), 16, C::GROUP);
      const uint64_t dq = desc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
      const uint64_t dv = desc_sw128(smem_u32(smem + C::OFF_KV), C::HALF, C::GROUP);
      const uint32_t tmem_u = uni(tmem);
      uint32_t par = 0;    // parities of the next p_full (bits 0, 1) and q_full (bits 2, 3) by slot
      uint32_t begun = 0;  // bit t: slot t's first S of the segment is out already
      uint32_t base = 0;   // ring loads before the current segment
      uint32_t seen = 0;   // ring loads known to be ready
      bool ok = true;
      auto ring_wait = [&](uint32_t g) -> bool {
        if (g < seen) return true;
        seen = g + 1;
        return wait_all(&ready[g % NS], (g / NS) & 1);
      };
      // S of slot t from the K tile that is ring load g
      auto issue_s = [&](int t, uint32_t g, bool last, bool release) {
        const uint32_t st = g % NS;
        const uint64_t k = dk + st * (C::KV_BYTES >> 4), q = dq + t * (C::Q_BYTES >> 4);
        const uint32_t d = tmem_u + C::COL_S + t * BN;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint32_t in = (i & 3) * 32;  // inside a row's 128 bytes
            mma_ss(d, q + (((i >> 2) * (BM * 128) + in) >> 4), k + (((i >> 2) * C::HALF + in) >> 4), IDESC_S, i > 0);
          }
          mma_commit(&s_full[t]);
          if (release) mma_commit(&empty[st]);
          if (last) mma_commit(&q_empty[t]);
        }
        __syncwarp();
      };
      for (int k = 0; ok; ++k) {
        if (!wait_all(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
        const Seg* sg = &segs[k % kSegs];
        const int w0 = uni(sg->n0 * 2 + sg->single), n1 = uni(sg->n1);
        if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
        if (n1 < 0) break;
        const int single = w0 & 1, n0 = w0 >> 1, tiles = single ? n0 + n1 : n1;
        // both slots' first S, unless it went out at the end of the last segment
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          const int nt = t ? n1 : n0;
          if (!nt || (begun >> t & 1u)) continue;
          const uint32_t g = base + ring_k(single ? t : 0);
          if (!wait_all(&q_full[t], par >> (2 + t) & 1u) || !ring_wait(g)) {
            ok = false;
            break;
          }
          par ^= 4u << t;
          issue_s(t, g, nt == 1, single || t);
        }
        begun = 0;
        // one slot's turn: P.V of its tile r, then S of its next one
        auto turn_of = [&](int t, int r) -> bool {
          const int nt = t ? n1 : n0;
          if (r >= nt) return true;
          const bool last = r + 1 == nt;
          const int j = single ? 2 * r + t : r;  // the tile's number in the segment
          const uint32_t g = base + ring_v(j, tiles), st = g % NS;
          const uint64_t v = dv + st * (C::KV_BYTES >> 4);
          // (with two slots on a tile, this is the only wait for the ring: the next K comes before this V)
          if (!ring_wait(g) || !wait_all(&p_full[t], par >> t & 1u)) return false;
          par ^= 1u << t;
          // ---- O += P V
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int e = 0; e < BN / 16; ++e)
              mma_ts(tmem_u + C::COL_O + t * D, tmem_u + C::COL_S + t * BN + e * 8, v + e * (2 * C::GROUP >> 4), IDESC_PV,
                     e > 0 ? 1u : (uint32_t)(r > 0));
            if (single || t) mma_commit(&empty[st]);
            if (last) mma_commit(&o_full[t]);
          }
          __syncwarp();
          if (!last) {
            const uint32_t gs = base + ring_k(single ? j + 2 : j + 1);
            if (!ring_wait(gs)) return false;
            issue_s(t, gs, r + 2 == nt, single || t);
            return true;
          }
          // or S of its first tile of the next segment, if its Q and K are there.  Two slots
          // share a K tile and slot 1's S releases it, so slot 1 never goes first.
          if (!uni(mbar_test(&seg_full[(k + 1) % kSegs], ((k + 1) / kSegs) & 1))) return true;
          const Seg* s2 = &segs[(k + 1) % kSegs];
          const bool turn = s2->n1 >= 0 && (s2->single || t == 0 || (begun & 1u) || s2->n0 == 0);
          const int w2 = uni(turn ? (t ? s2->n1 : s2->n0) * 2 + s2->single : 0), nt2 = w2 >> 1, single2 = w2 & 1;
          const uint32_t gs = base + 2 * tiles + ring_k(single2 ? t : 0);
          if (nt2 && uni(mbar_test(&q_full[t], par >> (2 + t) & 1u) &&
                         (gs < seen || mbar_test(&ready[gs % NS], (gs / NS) & 1)))) {
            seen = max(seen, gs + 1);
            par ^= 4u << t;
            issue_s(t, gs, nt2 == 1, single2 || t);
            begun |= 1u << t;
          }
          return true;
        };
        const int turns = 2 * max(n0, n1);
#pragma unroll 1
        for (int i = 0; ok && i < turns; ++i) ok = turn_of(i & 1, i >> 1);  // (unrolled by slot it spills)
        base += 2 * tiles;
      }
      // every MMA issued by this thread has finished before the CTA can exit
      if (elect_one()) mma_commit(mma_idle);
      __syncwarp();
      mbar_wait(mma_idle, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ============================ softmax ============================
    const int t = warp >> 2;
    const int r = threadIdx.x & (BM - 1);  // row = TMEM lane
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_addr + C::COL_S + t * BN;
    const uint32_t tO = tmem + lane_addr + C::COL_O;
    const int rtok = (int)fdiv((uint32_t)r, p.div_group);
    uint32_t sc = 0, oc0 = 0, oc1 = 0, nj = 0;  // S tiles, finished outputs of slots 0 and 1, joins
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&seg_full[k % kSegs], (k / kSegs) & 1)) break;
      const Seg* sg = &segs[k % kSegs];
      if (sg->q0 < 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
        break;
      }
      const bool single = sg->single;
      const int n = t ? sg->n1 : sg->n0;                             // the slot's key tiles
      const bool mine = n > 0;
      const int tok0 = single ? 0 : t * p.TQ;                        // the slot's first token of the unit
      // keys past the slot's first tile that every row of the slot sees, and that this row sees more
      const int key0 = (sg->t0 + (single ? t : 0)) * BN, key_step = single ? 2 * BN : BN;
      int vis_min = (p.causal ? sg->vis0 + tok0 : sg->len) - key0;
      const int more = p.causal ? rtok : 0;
      const bool valid = rtok < p.TQ && tok0 + rtok < sg->ntok;
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      float m_use = -INFINITY, l = 0.f;
      for (int i = 0; i < n; ++i, vis_min -= key_step) {
        if (!wait(&s_full[t], sc & 1)) { ok = false; break; }
        ++sc;
        if (warp_valid) {
          tc_fence_after();
          float x[BN];
          {
            uint32_t rr[BN / 32][32];
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) tmem_ld32(tS + c * 32, rr[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e) x[c * 32 + e] = __uint_as_float(rr[c][e]);
          }
          if (vis_min < BN) {
            const int lim = vis_min + more;  // columns from lim on are hidden
#pragma unroll
            for (int c = 0; c < BN; ++c) x[c] = c >= lim ? -INFINITY : x[c];
          }
          // row maximum of the raw scores (the scale is positive): 4 chains of 3-input maxima
          float mx;
          {
            float a0 = fmaxf(x[0], x[4]), a1 = fmaxf(x[1], x[5]), a2 = fmaxf(x[2], x[6]), a3 = fmaxf(x[3], x[7]);
#pragma unroll
            for (int c = 8; c < BN; c += 8) {
              a0 = max3f(a0, x[c + 0], x[c + 1]);
              a1 = max3f(a1, x[c + 2], x[c + 3]);
              a2 = max3f(a2, x[c + 4], x[c + 5]);
              a3 = max3f(a3, x[c + 6], x[c + 7]);
            }
            mx = max3f(a0, a1, fmaxf(a2, a3)) * p.scale_log2;
          }
          // the maximum in use only moves when it grows by more than 8 (log2), so O is rescaled
          // rarely; P <= 2^8 stays as exact and the quotient O / l is the same
          const float m_new = fmaxf(m_use, mx);
          const bool need = m_new > m_use + kRescaleThreshold || (m_use == -INFINITY && m_new != -INFINITY);
          float alpha = 1.f;
          if (need) {
            alpha = fast_exp2(m_use - m_new);
            m_use = m_new;
          }
          const float m_sub = m_use == -INFINITY ? 0.f : m_use;
          const float2 sl2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(-m_sub, -m_sub);
          float2 rs2[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) rs2[e] = make_float2(0.f, 0.f);
          // 32 columns at a time: P goes out as it is made (columns of S already read)
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 v = ffma2(make_float2(x[c * 32 + 2 * e], x[c * 32 + 2 * e + 1]), sl2, nm2);
              const float2 ev = make_float2(fast_exp2(v.x), fast_exp2(v.y));
              rs2[e & 3] = __fadd2_rn(rs2[e & 3], ev);
              pk[e] = Elem<T>::pack2(ev.x, ev.y);
            }
            tmem_st16(tS + c * 16, pk);
          }
          const float2 rs01 = __fadd2_rn(rs2[0], rs2[1]), rs23 = __fadd2_rn(rs2[2], rs2[3]);
          const float2 rsum = __fadd2_rn(rs01, rs23);
          l = l * alpha + (rsum.x + rsum.y);
          // S_j's commit covered P.V_j-1, so O may be rescaled here
          if (i > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t rr[32];
              tmem_ld32(tO + t * D + c * 32, rr);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) rr[e] = __float_as_uint(__uint_as_float(rr[e]) * alpha);
              tmem_st32(tO + t * D + c * 32, rr);
            }
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // ---- the segment's output: the whole row, or its partial result
      float w0 = 0.f, w1 = 0.f, total = l, m_row = m_use;
      bool other = false;
      if (mine) {
        if (!wait(&o_full[t], (t ? oc1 : oc0) & 1)) break;
        if (t) ++oc1; else ++oc0;
        tc_fence_after();
      }
      if (single) {
        if (t == 1) {  // hand the statistics over; slot 0 reads O from TMEM
          stat[r] = m_use;
          stat[BM + r] = mine ? l : 0.f;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(join);
          if (!wait(joined, nj & 1)) break;
          ++nj;
          __syncwarp();
          if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
          continue;
        }
        if (!wait(join, nj & 1)) break;
        ++nj;
        tc_fence_after();
        const float m1 = stat[r], l1 = stat[BM + r];
        other = l1 > 0.f || l1 != l1;
        m_row = fmaxf(m_use, other ? m1 : -INFINITY);
        const float m_sub = m_row == -INFINITY ? 0.f : m_row;
        w0 = fast_exp2(m_use - m_sub);
        w1 = other ? fast_exp2(m1 - m_sub) : 0.f;
        total = l * w0 + (other ? l1 * w1 : 0.f);
      } else {
        w0 = 1.f;
      }
      const bool any = total > 0.f || total != total;  // a row that sees no key: zeros
      const float inv = any ? 1.f / total : 0.f;
      w0 *= inv;
      w1 *= inv;
      if (warp_valid)
        finish_rows<T, D>(p, sg, tO, t, w0, w1, any ? (m_row + __log2f(total)) * kLn2 : -INFINITY,
                          (mine && any ? 1 : 0) | (other ? 2 : 0));
      tc_fence_before();
      __syncwarp();
      if (single && lane == 0) mbar_arrive(joined);
      if (lane == 0) mbar_arrive(&seg_empty[k % kSegs]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::TMEM_COLS));
  }
}

// -------------------------------------------------------------------------
// merge of units in parts, and zeros for rows of no sequence
// -------------------------------------------------------------------------
// O = sum_i e^{lse_i - M} O_i / sum_i e^{lse_i - M}.  The unit's parts are the one
// with its first keys and then place 0 of the CTAs after it, up to the one with
// its last keys; the ones without keys for the row (lse_i = -inf) are left out.  CTA (x, y): place x, rows [R y, R y + R), R = merge_rows; a warp per row.
constexpr int kMergeThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const ChunkParams p) {
  grid_dep_wait();
  constexpr int N = D / 32;  // columns per lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // rows of no sequence: padding before and after all of them, and the rows of sequences with bad query bounds
  if (blockIdx.y == 0) {
    const int64_t lo = min(max((int64_t)__ldg(p.q_indptr), (int64_t)0), p.num_tokens);
    const int64_t hi = min(max((int64_t)__ldg(p.q_indptr + p.B), lo), p.num_tokens);
    const int64_t none = (lo + p.num_tokens - hi) * p.Hq;
    const int64_t w0 = (int64_t)blockIdx.x * (kMergeThreads / 32) + warp, ws = (int64_t)gridDim.x * (kMergeThreads / 32);
    auto clear = [&](int64_t tok, int h) {
      T* row = reinterpret_cast<T*>(p.out + tok * p.o_tok + (int64_t)h * p.o_head);
#pragma unroll
      for (int e = 0; e < N; ++e) row[lane + 32 * e] = Elem<T>::from_float(0.f);
      if (p.lse && lane == 0) p.lse[tok * p.l_tok + (int64_t)h * p.l_head] = -INFINITY;
    };
    for (int64_t i = w0; i < none; i += ws) {
      const int64_t tok = i / p.Hq;
      clear(tok >= lo ? tok + hi - lo : tok, (int)(i - tok * p.Hq));
    }
    for (int64_t b0 = w0 * 32; b0 < p.B; b0 += ws * 32) {  // 32 sequences a look
      const int64_t b = b0 + lane;
      const int a0 = b < p.B ? __ldg(p.q_indptr + b) : 0, a1 = b < p.B ? __ldg(p.q_indptr + b + 1) : 0;
      const int64_t r0 = max(a0, 0), r1 = min((int64_t)a1, p.num_tokens);
      for (unsigned m = __ballot_sync(0xffffffffu, (a0 < 0 || a1 > p.num_tokens) && r0 < r1); m; m &= m - 1) {
        const int64_t first = __shfl_sync(0xffffffffu, r0, __ffs(m) - 1);
        const int64_t rows = (__shfl_sync(0xffffffffu, r1, __ffs(m) - 1) - first) * p.Hq;
        for (int64_t i = 0; i < rows; ++i) clear(first + i / p.Hq, (int)(i % p.Hq));
      }
    }
  }
  const int c0 = blockIdx.x >> 1;
  const Part me = p.parts[blockIdx.x];
  if (!me.used || !me.first) return;
  const int rows = me.single ? me.ntok * p.group : BM + (me.ntok - p.TQ) * p.group;
  if ((int)blockIdx.y * p.merge_rows >= rows) return;
  // how many CTAs follow with parts of this unit (those without one are passed over)
  int last = c0;
  for (int base = c0 + 1; base < p.grid; base += 32) {
    const int c = base + lane;
    const bool ends = c < p.grid && p.parts[2 * c].used && p.parts[2 * c].last;
    const unsigned m = __ballot_sync(0xffffffffu, ends);
    if (m) {
      last = base + __ffs(m) - 1;
      break;
    }
  }
  const int count = last - c0 + 1;
  for (int r = blockIdx.y * p.merge_rows + warp; r < min(rows, (int)(blockIdx.y + 1) * p.merge_rows); r += kMergeThreads / 32) {
    const int slot = me.single ? 0 : r >> 7, rr = r & (BM - 1);
    const int rtok = (int)fdiv((uint32_t)rr, p.div_group), tok = slot * p.TQ + rtok;
    if (rtok >= p.TQ || tok >= me.ntok) continue;
    const int head = me.kvh * p.group + rr - rtok * p.group;
    auto place = [&](int i) -> int64_t {
      return ((int64_t)(i ? 2 * (c0 + i) : (int)blockIdx.x)) * p.part_rows + r;
    };
    auto lse_of = [&](int i) -> float {
      return i < count && (i == 0 || p.parts[2 * (c0 + i)].used) ? p.part_lse[place(i)] : -INFINITY;
    };
    float M = -INFINITY;
    for (int i = lane; i < count; i += 32) M = fmaxf(M, lse_of(i));
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float Ms = M == -INFINITY ? 0.f : M;
    float acc[N] = {}, den = 0.f;
    for (int i0 = 0; i0 < count; i0 += 32) {
      const float part = lse_of(i0 + lane);
      const float mine = fast_exp2((part - Ms) * kLog2e);  // NaN stays NaN
      // A part without keys for the row is left out.  One whose weight is 0 is not: a value of it that is not
      // finite is the row's, as it is where the unit is in one part.
      const unsigned holds = __ballot_sync(0xffffffffu, part != -INFINITY);
      const int n = min(32, count - i0);
      for (int i1 = 0; i1 < n; i1 += 8) {  // eight parts' rows asked for at once
        float w[8];
        float v[8][N];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          w[u] = __shfl_sync(0xffffffffu, mine, i1 + u);  // (0 past the count)
#pragma unroll
          for (int e = 0; e < N; ++e) v[u][e] = 0.f;
          if (!(holds >> (i1 + u) & 1u)) continue;
          const float* o = p.part_o + place(i0 + i1 + u) * D + lane * N;
          if constexpr (N == 4) *reinterpret_cast<float4*>(v[u]) = *reinterpret_cast<const float4*>(o);
          else *reinterpret_cast<float2*>(v[u]) = *reinterpret_cast<const float2*>(o);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          den += w[u];
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] = fmaf(w[u], v[u][e], acc[e]);
        }
      }
    }
    const bool any = den > 0.f || den != den;
    const float inv = any ? 1.f / den : 0.f;
    const int64_t grow = (int64_t)me.q0 + tok;
    T* row = reinterpret_cast<T*>(p.out + grow * p.o_tok + (int64_t)head * p.o_head) + lane * N;
    if constexpr (N == 4)
      *reinterpret_cast<uint2*>(row) = make_uint2(Elem<T>::pack2(acc[0] * inv, acc[1] * inv), Elem<T>::pack2(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(row) = Elem<T>::pack2(acc[0] * inv, acc[1] * inv);
    if (p.lse && lane == 0)
      p.lse[grow * p.l_tok + (int64_t)head * p.l_head] = any ? Ms + __log2f(den) * kLn2 : -INFINITY;
  }
}

// -------------------------------------------------------------------------
// host
// -------------------------------------------------------------------------
bool al16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

int sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = counts[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

struct Layout {
  int grid, part_rows, TQ;
  size_t parts, lse, o, cost, units, plan, share, bytes;
};

// The grid is one CTA per SM, or less where the tables' bounds show that there
// are fewer tiles: a sequence has at most one unit more per head than its rows
// fill, and a unit at most as many tiles as all pages hold.
Layout make_layout(const akt_chunk_paged_args* a) {
  Layout y{};
  const int G = a->num_qo_heads / a->num_kv_heads;
  y.TQ = BM / G;
  const int64_t units = ((int64_t)a->num_tokens / (2 * y.TQ) + std::min<int64_t>(a->batch, a->num_tokens)) * a->num_kv_heads;
  const int64_t tiles = a->num_page_entries * a->page_size / BN + 1;
  y.grid = std::min(sm_count(), kMaxCtas - 1);  // (the planning threads are one more)
  if (units < y.grid && units * tiles < y.grid) y.grid = (int)std::max<int64_t>(1, units * tiles);
  y.part_rows = (int)std::min<int64_t>(2 * BM, a->num_tokens * G <= BM ? a->num_tokens * G : 2 * BM);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t p = at;
    at += round256(n);
    return p;
  };
  y.parts = take((size_t)y.grid * 2 * sizeof(Part));
  y.lse = take((size_t)y.grid * 2 * y.part_rows * 4);
  y.o = take((size_t)y.grid * 2 * y.part_rows * a->head_dim * 4);
  if (a->batch > kTableSeqs) {
    y.cost = take(((size_t)a->batch + 1) * 8);
    y.units = take(((size_t)a->batch + 1) * 4);
    y.plan = take(sizeof(Plan));
    y.share = take(((size_t)y.grid + 1) * 8);
  }
  y.bytes = at;
  return y;
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
  if (a->num_qo_heads / a->num_kv_heads > BM)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: at most 128 query heads per kv head");
  if (!(a->softmax_scale > 0.f) || a->softmax_scale == INFINITY)
    return set_error(AKT_ERR_INVALID, "chunk_paged: softmax_scale must be positive and finite");
  // positions, rows and pages are 32-bit in the kernels (addresses are 64-bit)
  if (a->num_tokens > 0x3fffffff / a->num_qo_heads || a->num_page_entries > 0x3fffffff / a->page_size ||
      a->num_pages > 0x7ffffff0)
    return set_error(AKT_ERR_INVALID, "chunk_paged: too many tokens");
  if (a->num_tokens == 0) return AKT_OK;
  if (!a->q || !a->out || !a->q_indptr || !a->kv_page_indptr || !a->kv_last_page_len ||
      (a->num_page_entries > 0 && (!a->kv_page_indices || (!a->kv_cache && a->num_pages > 0))))
    return set_error(AKT_ERR_INVALID, "chunk_paged: missing tensor");
  if (a->batch == 0) return set_error(AKT_ERR_INVALID, "chunk_paged: tokens without sequences");
  if (a->q_stride_dim != 1 || a->kv_stride_dim != 1 || a->out_stride_dim != 1)
    return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: unit dim stride required");
  const int64_t strides[] = {a->q_stride_token,  a->q_stride_head,  a->kv_stride_page,   a->kv_stride_kv,
                             a->kv_stride_head,  a->kv_stride_token, a->out_stride_token, a->out_stride_head};
  for (int64_t s : strides)
    if (s % 8) return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: strides must be multiples of 16 bytes");
  if (!al16(a->q) || !al16(a->kv_cache) || !al16(a->out))
    return set_error(AKT_ERR_UNSUPPORTED, "chunk_paged: 16-byte alignment required");
  return AKT_OK;
}

int make_map(CUtensorMap* m, const void* base, int dtype, int rank, const cuuint64_t* dims, const int64_t* strides,
             const cuuint32_t* box) {
  auto fn = tensor_map_encoder();
  if (!fn) return set_error(AKT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  // an extent of one has no stride of its own (torch gives any)
  cuuint64_t st[4];
  for (int i = 0; i + 1 < rank; ++i) st[i] = (cuuint64_t)(dims[i + 1] > 1 ? strides[i] : 16);
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      fn(m, dtype == AKT_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
         const_cast<void*>(base), dims, st, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(AKT_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return AKT_OK;
}

template <typename T, int D, bool TMA>
int launch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkParams& p,
                 cudaStream_t st) {
  auto kern = chunk_fwd_kernel<T, D, TMA>;
  constexpr int smem = (int)Cfg<D>::SMEM_ALL;
  // the register split in the kernel is only valid at the compiled count
  static const int regs = [&] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs != kLaunchRegs)
    return set_error(AKT_ERR_CUDA, "chunk kernel compiled with " + std::to_string(regs) + " registers, expected " +
                                       std::to_string(kLaunchRegs));
  cudaError_t e = ensure_smem_limit<chunk_fwd_kernel<T, D, TMA>>((size_t)smem);
  if (e != cudaSuccess) return set_error(AKT_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  const bool planned = p.B > kTableSeqs;
  if (planned) chunk_plan_kernel<<<1, 1024, 0, st>>>(p);
  {
    ProfileScope prof(st);
    if (planned) e = launch_dependent(kern, dim3(p.grid), dim3(kThreads), smem, st, mq, mk, mv, p);
    else kern<<<p.grid, kThreads, smem, st>>>(mq, mk, mv, p);
  }
  if (e == cudaSuccess)
    e = launch_dependent(chunk_merge_kernel<T, D>, dim3(2 * p.grid, (p.part_rows + p.merge_rows - 1) / p.merge_rows),
                         dim3(kMergeThreads), 0, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : set_error(AKT_ERR_CUDA, std::string("chunk_paged: ") + cudaGetErrorString(e));
}

template <typename T, int D>
int dispatch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkParams& p,
                   cudaStream_t st) {
  return p.box_rows ? launch_chunk<T, D, true>(mq, mk, mv, p, st) : launch_chunk<T, D, false>(mq, mk, mv, p, st);
}

}  // namespace

cudaError_t chunk_status_read(unsigned int* v) { return cudaMemcpyFromSymbol(v, g_device_status_local, sizeof(*v)); }

cudaError_t chunk_status_clear() {
  const unsigned int z = 0;
  return cudaMemcpyToSymbol(g_device_status_local, &z, sizeof(z));
}

}  // namespace akt

using namespace akt;

extern "C" size_t akt_chunk_paged_workspace_size(const akt_chunk_paged_args* a) {
  if (!a || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->num_qo_heads % a->num_kv_heads || a->num_tokens <= 0 ||
      a->batch <= 0 || a->num_qo_heads / a->num_kv_heads > BM || a->page_size <= 0 || a->head_dim <= 0 ||
      a->num_page_entries < 0)
    return 0;
  return make_layout(a).bytes;
}

extern "C" int akt_chunk_paged(const akt_chunk_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_args(a);
  if (rc || a->num_tokens == 0) return rc;
  const Layout y = make_layout(a);
  if (!workspace || workspace_bytes < y.bytes)
    return set_error(AKT_ERR_WORKSPACE, "chunk_paged: workspace of " + std::to_string(y.bytes) + " bytes required");
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
  p.D = a->head_dim;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.TQ = y.TQ;
  p.div_group = make_fastdiv((uint32_t)p.group);
  p.div_page = make_fastdiv((uint32_t)p.P);
  p.grid = y.grid;
  char* ws = static_cast<char*>(workspace);
  p.parts = reinterpret_cast<Part*>(ws + y.parts);
  p.part_lse = reinterpret_cast<float*>(ws + y.lse);
  p.part_o = reinterpret_cast<float*>(ws + y.o);
  p.part_rows = y.part_rows;
  // A row of a merge is a chain of lookups, so few rows get a warp each (4 tokens on 2048
  // keys, whole call in a graph 20.6 us, 22.5 with four rows a warp; on 32768 keys 43.7, 47.8);
  // many rows would be many CTAs that mostly find nothing to join (8 prompts of 2048
  // tokens: 305 us, 316 with a row a warp).
  p.merge_rows = y.part_rows <= 64 ? 8 : 32;
  if (p.B > kTableSeqs) {
    p.plan_cost = reinterpret_cast<int64_t*>(ws + y.cost);
    p.plan_units = reinterpret_cast<int*>(ws + y.units);
    p.plan = reinterpret_cast<Plan*>(ws + y.plan);
    p.plan_share = reinterpret_cast<int64_t*>(ws + y.share);
  }
  // a box holds keys of one page: the largest power of two from 8 (the swizzle's
  // row period) to 128 that divides the page size
  p.box_rows = 0;
  for (int r = 128; r >= 8 && !p.box_rows; r >>= 1)
    if (p.P % r == 0) p.box_rows = r;
  if (p.num_pages == 0) p.box_rows = 0;
  CUtensorMap mq, mk, mv;
  const cuuint64_t qd[4] = {(cuuint64_t)p.D, (cuuint64_t)p.group, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_tokens};
  const int64_t qs[3] = {a->q_stride_head * 2, a->q_stride_head * 2 * p.group, a->q_stride_token * 2};
  const cuuint32_t qb[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)p.TQ};
  rc = make_map(&mq, a->q, a->dtype, 4, qd, qs, qb);
  mk = mv = mq;
  if (!rc && p.box_rows) {
    const cuuint64_t halves = (cuuint64_t)(p.D / 64);
    // Heads, K and V, and pages in one run (a contiguous pool): one dimension counts
    // them, and a box takes all 8-row groups of its keys, 4 KB at 16 keys of 128
    // values.  Other strides take two dimensions and a box 8 rows.
    p.linear = p.s_kv == p.s_head * p.Hkv && p.s_page == 2 * p.s_kv && p.num_pages * 2 * p.Hkv < 0x7fff0000;
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
      if (!rc) rc = make_map(&mv, p.kv + p.s_kv, a->dtype, 5, kd, ks, kb);
    }
  }
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == AKT_FLOAT16)
    return p.D == 64 ? dispatch_chunk<__half, 64>(mq, mk, mv, p, st) : dispatch_chunk<__half, 128>(mq, mk, mv, p, st);
  return p.D == 64 ? dispatch_chunk<__nv_bfloat16, 64>(mq, mk, mv, p, st)
                   : dispatch_chunk<__nv_bfloat16, 128>(mq, mk, mv, p, st);
}
