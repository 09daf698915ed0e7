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
// Shared prefixes (the SHARED template).  Groups of neighbouring sequences have their
// first pages in common.  A planner turns the batch into virtual sequences: for each
// group its sequences' rows on the shared keys, all visible, and for each sequence its
// rows on its own keys behind them.  Both are cut into units as above, so the prefix's
// K/V are read once for a group and the rows of all its sequences fill the tiles.  A
// row of a sequence with a prefix leaves two partial results (or the parts of them),
// which chunk_join_kernel joins; other rows go straight to the output.
//
// Bounds and measured rates (fp16, 32 query heads on 8, pages of 16 keys, full clock).
// Long prompts: the tensor pipe and the exponentials, 60 % busy each; 8192 tokens on top
// of 24576, D = 128, 3.01 ms = 1280 TFLOP/s (D = 64: 2.53 ms).  Short prompts also their
// units' ends and the causal edge: 8 of 2048 tokens, 295 us.  Few tokens: HBM; 5 in each
// of 64 sequences of 512 to 32768 keys, 655 us = 6.66 TB/s.
//
// Built without -rdc (setmaxnreg needs whole-program device code).
#define AKT_WHOLE_PROGRAM 1
#include "attn_mma.cuh"
#include "common.cuh"
#include "profile.cuh"
#include "tcgen05.cuh"
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
// Units of a sequence's own keys behind a prefix that take the warp-level kernel: a
// unit's chain of steps here (Q, S, the exponentials, P.V, the output) takes 4 us however
// few its rows and tiles are.  One token in each of 64 sequences of 64 to 1024 own keys
// behind 8192, 4 rows a unit: 74 us, all units here 151; five tokens in each of 64 behind
// eight prefixes, 20 rows: 160, here 216.  So too where few units leave SMs without one,
// n sequences of 2048 own keys behind 2048 on eight kv heads, n = 2 45 / 67, 8 48 / 66, 16
// 60 / 93, 64 122 / 190.  Past 2048 it depends on n: 4096 own keys, n = 2 70 / 66, 16
// 87 / 106, 64 198 / 314; 8192, n = 2 128 / 72, 16 140 / 149, 64 351 / 449.  (More rows take
// a multiple of the warp-level products.)
constexpr int kSmallRows = 32, kSmallKeys = 2048;
// The planner gives that kernel the longest first up to so many sequences (a quadratic count).  One token in each of n
// sequences of up to 1024 own keys behind 2048, eight kv heads, in order / as they come: n = 16 32.8 / 35.6 us, 64
// 66.0 / 67.0, 128 98 / 90, 256 168 / 143, 1024 536 / 459; one kv head, 1024 160 / 120.
constexpr int kOrderSeqs = 64;
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
  // shared prefixes: B counts the virtual sequences, `groups` prefixes and then the batch's
  int groups, batch;
  const int32_t* group_indptr;
  const int32_t* shared_pages;
  struct Seq* seqs;    // [B]
  struct Seq* own;     // [batch] the sequences on their own keys; those with few have no rows in `seqs`
  int* prefix_len;     // [batch] shared keys of each sequence
  int* order;          // [batch] the sequences, those with the most own keys first
  float* row_o;        // [2][rows][D] (none without groups) normalised outputs of a row on the prefix, on its own keys
  float* row_lse;      // [2][rows] (none without groups)
  int2* row_at;        // [2][rows] kWhole, kDone, or the place of the first part and the row there
};

constexpr int kWhole = -1;  // the row's result is in row_o
constexpr int kDone = -2;   // the row is in the output

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
  int causal;
  int prefix;  // shared prefixes: 0 a sequence without one, 1 a prefix, 2 a sequence's own keys behind one
  int pad;
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
  int causal, prefix;
};

// Sequence b's bounds; a malformed one is empty (recorded by the planner).
template <bool SHARED = false>
__device__ __forceinline__ Seq load_seq(const ChunkParams& p, int b, bool record) {
  if constexpr (SHARED) return p.seqs[b];
  Seq s;
  s.causal = p.causal;
  s.prefix = 0;
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
  const int vis = s.causal ? s.len - s.n + min((u + 1) * 2 * p.TQ, s.n) : s.len;
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
template <bool SHARED>
__device__ __forceinline__ void unit_at(const ChunkParams& p, const Tables& t, int i, int& b, Seq& s, int& kvh, int& u) {
  b = find_seq(t.units, p.B, i);
  s = load_seq<SHARED>(p, b, false);
  const int U = num_units(p, s), r = i - t.units[b];
  kvh = r / U;
  u = U - 1 - (r - kvh * U);
}

// Fills the tables (threads of one CTA, `nthreads` of them; cost and units in
// shared or global memory), and the costliest unit's cost, no less, into
// *most_cost (shared memory).
template <bool SHARED>
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
      s = load_seq<SHARED>(p, b, lane == 0);
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
template <bool SHARED>
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
      s = t.seqs ? t.seqs[b] : load_seq<SHARED>(p, b, false);
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
template <typename T, int D, bool SHARED>
__device__ __forceinline__ void finish_rows(const ChunkParams& p, const Seg* sg, uint32_t tO, int t, float w0, float w1,
                                         float row_lse, int flags) {
  const int r = threadIdx.x & (BM - 1), rtok = (int)fdiv((uint32_t)r, p.div_group);
  const bool single = sg->single;
  const int tok = (single ? 0 : t * p.TQ) + rtok, part = sg->part, head = sg->kvh * p.group + r - rtok * p.group;
  const bool valid = rtok < p.TQ && tok < sg->ntok;
  const int64_t grow = (int64_t)sg->q0 + tok;
  const int64_t pidx = ((int64_t)(2 * blockIdx.x) + max(part, 0)) * p.part_rows + (single ? 0 : t * BM) + r;
  const bool done = part < 0 && (!SHARED || sg->prefix == 0);  // the row's final result
  const int64_t ridx = SHARED ? (sg->prefix == 1 ? 0 : p.num_tokens * p.Hq) + grow * p.Hq + head : 0;
  char* mine = valid ? (done ? p.out + grow * p.o_tok + (int64_t)head * p.o_head
                             : reinterpret_cast<char*>(part < 0 ? p.row_o + ridx * D : p.part_o + pidx * D))
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
    if (done) {
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
  if (SHARED && valid) {
    if (part >= 0 && sg->t0 == 0) p.row_at[ridx] = make_int2(2 * blockIdx.x + part, (single ? 0 : t * BM) + r);
    else if (part < 0) p.row_at[ridx] = make_int2(done ? kDone : kWhole, 0);
    if (part < 0 && !done) p.row_lse[ridx] = row_lse;
  }
  if (valid) {
    if (part >= 0) p.part_lse[pidx] = row_lse;
    else if (done && p.lse) p.lse[grow * p.l_tok + (int64_t)head * p.l_head] = row_lse;
  }
  if (sg->noted) {
    __syncwarp();  // the row was stored by four lanes
    const int vis = sg->vis0 + tok;
    if (valid && done) add_not_finite<T, D, T>(p, *sg, vis, reinterpret_cast<T*>(mine));
    if (valid && !done) add_not_finite<T, D, float>(p, *sg, vis, reinterpret_cast<float*>(mine));
  }
}

// -------------------------------------------------------------------------
// the planner of batches past the CTA's own table
// -------------------------------------------------------------------------
// Sequences with so few rows and own keys are left to chunk_small_kernel.
__device__ __forceinline__ bool is_small(const ChunkParams& p, const Seq& s) {
  return s.n > 0 && s.n <= kSmallRows / p.group && s.len <= kSmallKeys;
}

// The virtual sequences of a batch with shared prefixes.  A group's prefix is as many
// whole pages as it is said to share, as all its sequences with rows have and (causal)
// as their first rows see; none where fewer than two have rows or one has bad bounds.
__device__ void build_shared(const ChunkParams& p, int* bad) {
  if (threadIdx.x == 0) *bad = 0;
  __syncthreads();
  for (int g = threadIdx.x; p.groups && g <= p.groups; g += 1024) {  // (no groups need no bounds)
    const int x = __ldg(p.group_indptr + g);
    if (x < 0 || x > p.batch || (g && __ldg(p.group_indptr + g - 1) > x)) *bad = 1;
  }
  __syncthreads();
  if (*bad && threadIdx.x == 0) record_status(kStatusBadIndptr);
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < p.groups; g += 32) {  // a warp per group
    const int b0 = *bad ? 0 : __ldg(p.group_indptr + g), b1 = *bad ? 0 : __ldg(p.group_indptr + g + 1);
    int keys = min(max(__ldg(p.shared_pages + g), 0), 0x3fffffff / p.P) * p.P, rows = 0, first = 0x7fffffff;
    for (int b = b0 + lane; b < b1; b += 32) {
      const Seq s = load_seq(p, b, false);
      const int a0 = __ldg(p.q_indptr + b), a1 = __ldg(p.q_indptr + b + 1);
      if (a0 < 0 || a1 < a0 || a1 > p.num_tokens) keys = 0;
      if (s.n == 0) continue;
      ++rows;
      first = min(first, b);
      keys = min(keys, max(p.causal ? s.len - s.n : s.len, 0));
    }
    keys = __reduce_min_sync(0xffffffffu, keys) / p.P * p.P;
    rows = __reduce_add_sync(0xffffffffu, rows);
    first = __reduce_min_sync(0xffffffffu, first);
    Seq v{};
    if (keys > 0 && rows > 1) {
      v.a0 = __ldg(p.q_indptr + b0);
      v.n = __ldg(p.q_indptr + b1) - v.a0;
      v.page0 = __ldg(p.indptr + first);
      v.len = keys;
      v.prefix = 1;
    }
    if (lane == 0) p.seqs[g] = v;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.batch; b += 1024) {
    Seq s = load_seq(p, b, true);
    int keys = 0;
    if (p.groups && !*bad) {
      const int g = find_seq(p.group_indptr, p.groups, b);
      if (b >= __ldg(p.group_indptr + g) && b < __ldg(p.group_indptr + g + 1) && s.n) keys = p.seqs[g].len;
    }
    if (keys) {
      s.page0 += keys / p.P;
      s.len -= keys;
      s.prefix = 2;
    }
    p.own[b] = s;
    if (is_small(p, s)) s.n = 0;
    p.seqs[p.groups + b] = s;
    p.prefix_len[b] = keys;
    p.order[b] = b;
  }
  __syncthreads();
  // long ones first, so that none of them begins last
  if (p.batch <= kOrderSeqs)
    for (int b = threadIdx.x; b < p.batch; b += 1024) {
      const int len = p.own[b].len;
      int before = 0;
      for (int e = 0; e < p.batch; ++e) {
        const int other = p.own[e].len;
        before += other > len || (other == len && e < b);
      }
      p.order[before] = b;
    }
  __syncthreads();
}

template <bool SHARED>
__global__ void __launch_bounds__(1024) chunk_plan_kernel(const ChunkParams p) {
  __shared__ __align__(8) int scratch[64];
  __shared__ int most_cost;
  if (SHARED) build_shared(p, &most_cost);
  build_tables<SHARED>(p, p.plan_cost, p.plan_units, nullptr, &most_cost, 1024);
  const Plan pl = make_plan<SHARED>(p, Tables{p.plan_cost, p.plan_units, nullptr}, most_cost, p.plan_share, scratch);
  if (threadIdx.x == 0) *p.plan = pl;
}

// -------------------------------------------------------------------------
// main kernel
// -------------------------------------------------------------------------
template <typename T, int D, bool TMA, bool SHARED>
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

  if (SHARED && threadIdx.x == 32) {  // (in the form without shared prefixes it spills at D = 64)
    prefetch_tensor_map(&tmQ);
    prefetch_tensor_map(&tmK);
    prefetch_tensor_map(&tmV);
  }
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
  if (!SHARED && p.B <= kTableSeqs) {
    int64_t* cost = reinterpret_cast<int64_t*>(smem + C::OFF_TABLE);
    int* units = reinterpret_cast<int*>(cost + p.B + 1);
    // the shares live where slot 0's Q tile goes later
    int64_t* share = reinterpret_cast<int64_t*>(smem + C::OFF_Q);
    int* scratch = reinterpret_cast<int*>(share + p.grid + 1);
    Seq* seqs = reinterpret_cast<Seq*>(smem + C::OFF_Q + 8192);
    build_tables<SHARED>(p, cost, units, seqs, scratch + 63, kThreads);
    tab = Tables{cost, units, seqs};
    plan = make_plan<SHARED>(p, tab, scratch[63], share, scratch);
    begin = share[blockIdx.x];
    end = share[blockIdx.x + 1];
    // generic reads before the async-proxy writes of the Q tile
    fence_async_smem();
  } else {
    grid_dep_wait();
    if (SHARED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the planner is done)
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
          unit_at<SHARED>(p, tab, dealt_unit(p, round, blockIdx.x), bb, q, k, uu);
          ++round;
          const int X = 2 * p.TQ;
          sg.q0 = q.a0 + uu * X;
          sg.ntok = min(X, q.n - uu * X);
          sg.vis0 = q.causal ? q.len - q.n + uu * X + 1 : q.len;
          sg.causal = q.causal;
          sg.prefix = q.prefix;
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
              s = load_seq<SHARED>(p, b, false);
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
              sg.vis0 = s.causal ? s.len - s.n + u * X + 1 : s.len;
              sg.causal = s.causal;
              sg.prefix = s.prefix;
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
          const int vis = sg.causal ? sg.vis0 + p.TQ - 1 : sg.len;
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
        const bool causal = SHARED ? sg->causal : p.causal;
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
          if (is_v && ((causal && (j + 1) * BN > vis0) || (j + 1) * BN > len)) {
            // rows that every row of the unit sees stay as they are
            unsigned char* v = smem + C::OFF_KV + st * C::KV_BYTES;
            const int rows = len - j * BN;  // the others are past the sequence
            const int r0 = min(max(causal ? vis0 - j * BN : rows, 0), BN);
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
      const bool causal = SHARED ? sg->causal : p.causal;
      int vis_min = (causal ? sg->vis0 + tok0 : sg->len) - key0;
      const int more = causal ? rtok : 0;
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
        finish_rows<T, D, SHARED>(p, sg, tO, t, w0, w1, any ? (m_row + __log2f(total)) * kLn2 : -INFINITY,
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
// join of a row's results on a shared prefix and on its own keys
// -------------------------------------------------------------------------
// Results of a row in unit kind k (0 the prefix, 1 its own keys), whose entry of row_at is
// w: whole, or parts as chunk_merge_kernel finds them.  The whole warp calls it.
struct RowParts {
  int count;  // 0: none
  int first;  // place of the first part, kWhole, or kDone
  int r;      // the row there
};

// Entry i of row_at.  Where a wait ran out (recorded) it may never have been written: no place outside the workspace.
__device__ __forceinline__ int2 row_place(const ChunkParams& p, int64_t i) {
  const int2 w = p.row_at[i];
  const bool nowhere = w.x < 0 ? !p.groups : w.x >= 2 * p.grid || (unsigned)w.y >= (unsigned)p.part_rows;
  return nowhere ? make_int2(kDone, 0) : w;
}

__device__ __forceinline__ RowParts row_parts(const ChunkParams& p, int2 w) {
  RowParts x{1, w.x, w.y};
  if (w.x < 0 || p.parts[w.x].last) return x;
  const int lane = threadIdx.x & 31, c0 = w.x >> 1;
  for (int base = c0 + 1; base < p.grid; base += 32) {  // the CTA with the last part
    const int c = base + lane;
    const bool ends = c < p.grid && p.parts[2 * c].used && p.parts[2 * c].last;
    const unsigned m = __ballot_sync(0xffffffffu, ends);
    if (m) {
      x.count = base + __ffs(m) - c0;
      break;
    }
  }
  return x;
}

// Result i of these: its log-sum-exp (-inf: nothing) and its row.
template <int D>
__device__ __forceinline__ float row_result(const ChunkParams& p, int k, int64_t row, const RowParts& x, int i,
                                            const float*& o) {
  const int64_t rows = p.num_tokens * p.Hq;
  o = nullptr;
  if (i >= x.count) return -INFINITY;
  if (x.first < 0) {
    o = p.row_o + (k * rows + row) * D;
    return p.row_lse[k * rows + row];
  }
  const int place = i ? 2 * ((x.first >> 1) + i) : x.first;
  if (i && !p.parts[place].used) return -INFINITY;
  const int64_t at = (int64_t)place * p.part_rows + x.r;
  o = p.part_o + at * D;
  return p.part_lse[at];
}

// n results of a row, result i's log-sum-exp `part` and row `o` with lane i; lane columns
// [N lane, N lane + N).  Ms is the largest log-sum-exp, den and acc the sums in its scale.
template <int N, int U>
__device__ __forceinline__ void add_weighted(int n, float part, const float* o, float Ms, float& den, float (&acc)[N]) {
  const int lane = threadIdx.x & 31;
  const float mine = fast_exp2((part - Ms) * kLog2e);  // NaN stays NaN
  const unsigned holds = __ballot_sync(0xffffffffu, part != -INFINITY);  // (a weight of 0 is not left out)
  for (int i1 = 0; i1 < n; i1 += U) {  // U rows asked for at once
    float w[U];
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = __shfl_sync(0xffffffffu, mine, i1 + u);
      const float* src = reinterpret_cast<const float*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), i1 + u));
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] = 0.f;
      if (i1 + u >= n || !(holds >> (i1 + u) & 1u)) continue;
      if constexpr (N == 4) *reinterpret_cast<float4*>(v[u]) = *reinterpret_cast<const float4*>(src + lane * N);
      else *reinterpret_cast<float2*>(v[u]) = *reinterpret_cast<const float2*>(src + lane * N);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i1 + u >= n) continue;
      den += w[u];
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(w[u], v[u][e], acc[e]);
    }
  }
}

// All results of a row.
template <int D, int N>
__device__ __forceinline__ void add_results(const ChunkParams& p, int k, int64_t row, const RowParts& x, float Ms,
                                            float& den, float (&acc)[N]) {
  for (int i0 = 0; i0 < x.count; i0 += 32) {
    const float* o;
    const float part = row_result<D>(p, k, row, x, i0 + (int)(threadIdx.x & 31), o);
    add_weighted<N, 4>(min(32, x.count - i0), part, o, Ms, den, acc);
  }
}

template <int D>
__device__ __forceinline__ float largest_result(const ChunkParams& p, int k, int64_t row, const RowParts& x) {
  const float* o;
  float M = -INFINITY;
  for (int i = threadIdx.x & 31; i < x.count; i += 32) M = fmaxf(M, row_result<D>(p, k, row, x, i, o));
#pragma unroll
  for (int s = 16; s; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
  return M;
}

// The joined row: sum of the weighted results over the sum of the weights.
template <typename T, int N>
__device__ __forceinline__ void store_row(const ChunkParams& p, int64_t tok, int head, float Ms, float den,
                                          const float (&acc)[N]) {
  const int lane = threadIdx.x & 31;
  const bool any = den > 0.f || den != den;
  const float inv = any ? 1.f / den : 0.f;
  T* out = reinterpret_cast<T*>(p.out + tok * p.o_tok + (int64_t)head * p.o_head) + lane * N;
  if constexpr (N == 4)
    *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack2(acc[0] * inv, acc[1] * inv), Elem<T>::pack2(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(out) = Elem<T>::pack2(acc[0] * inv, acc[1] * inv);
  if (p.lse && lane == 0) p.lse[tok * p.l_tok + (int64_t)head * p.l_head] = any ? Ms + __log2f(den) * kLn2 : -INFINITY;
}

constexpr int kJoinRows = 8;  // of a warp
constexpr int64_t kFoldRows = 32768;  // up to so many rows CTAs of the kernel of small units join them

// Warps of kJoinRows rows (token, head) each.  Rows of no sequence are zeros.
template <typename T, int D>
__device__ void join_rows(const ChunkParams& p, int64_t warp) {
  constexpr int N = D / 32;  // columns per lane
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.num_tokens * p.Hq, row0 = warp * kJoinRows;
  // a lane looks a row up
  int2 w0 = make_int2(kDone, 0), w1 = make_int2(kDone, 0);
  float lse0 = -INFINITY, lse1 = -INFINITY;
  int none = 0;
  if (lane < kJoinRows && row0 + lane < rows) {
    const int64_t row = row0 + lane;
    const int tok = (int)(row / p.Hq), b = find_seq(p.q_indptr, p.batch, tok);
    const int a0 = __ldg(p.q_indptr + b), a1 = __ldg(p.q_indptr + b + 1);
    none = !(a0 >= 0 && tok >= a0 && tok < a1 && a1 <= p.num_tokens);
    if (!none && !is_small(p, p.own[b])) {
      w1 = row_place(p, rows + row);
      if (w1.x == kWhole) lse1 = p.row_lse[rows + row];
      if (p.prefix_len[b]) {
        w0 = row_place(p, row);
        if (w0.x == kWhole) lse0 = p.row_lse[row];
      }
    }
  }
#pragma unroll
  for (int i0 = 0; i0 < kJoinRows; i0 += 4) {
    // rows that are whole in both places, four at a time
    float v[4][2][N];
    unsigned simple = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at0 = __shfl_sync(0xffffffffu, w0.x, i0 + u), at1 = __shfl_sync(0xffffffffu, w1.x, i0 + u);
      if (at0 != kWhole || at1 != kWhole) continue;
      simple |= 1u << u;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float* o = p.row_o + (k * rows + row0 + i0 + u) * D + lane * N;
        if constexpr (N == 4) *reinterpret_cast<float4*>(v[u][k]) = *reinterpret_cast<const float4*>(o);
        else *reinterpret_cast<float2*>(v[u][k]) = *reinterpret_cast<const float2*>(o);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t row = row0 + i0 + u;
      const int64_t tok = row / p.Hq;
      const int head = (int)(row - tok * p.Hq);
      const float x0 = __shfl_sync(0xffffffffu, lse0, i0 + u), x1 = __shfl_sync(0xffffffffu, lse1, i0 + u);
      const int at1 = __shfl_sync(0xffffffffu, w1.x, i0 + u), nobody = __shfl_sync(0xffffffffu, none, i0 + u);
      const bool prefixed = __shfl_sync(0xffffffffu, w0.x, i0 + u) != kDone;
      float acc[N] = {}, den = 0.f, M;
      if (simple >> u & 1u) {
        M = fmaxf(x0, x1);
        const float Ms = M == -INFINITY ? 0.f : M;
        const float e[2] = {fast_exp2((x0 - Ms) * kLog2e), fast_exp2((x1 - Ms) * kLog2e)};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if ((k ? x1 : x0) == -INFINITY) continue;
          den += e[k];
#pragma unroll
          for (int c = 0; c < N; ++c) acc[c] = fmaf(e[k], v[u][k][c], acc[c]);
        }
      } else if (nobody) {
        M = -INFINITY;
      } else {
        if (at1 == kDone) continue;
        const RowParts own = row_parts(p, row_place(p, rows + row));
        const RowParts front = prefixed ? row_parts(p, row_place(p, row)) : RowParts{0, kWhole, 0};
        M = fmaxf(largest_result<D>(p, 1, row, own), largest_result<D>(p, 0, row, front));
        const float Ms = M == -INFINITY ? 0.f : M;
        add_results<D, N>(p, 0, row, front, Ms, den, acc);
        add_results<D, N>(p, 1, row, own, Ms, den, acc);
      }
      store_row<T, N>(p, tok, head, M == -INFINITY ? 0.f : M, den, acc);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_join_kernel(const ChunkParams p) {
  grid_dep_wait();
  join_rows<T, D>(p, (int64_t)blockIdx.x * (kMergeThreads / 32) + (threadIdx.x >> 5));
}

// -------------------------------------------------------------------------
// few rows on few own keys, at warp level
// -------------------------------------------------------------------------
// A CTA per (sequence, kv head).  Its four warps take 16 keys at a time in turn, each
// with a ring of its own that cp.async fills (no barrier in the loop):
//   S^T[16 keys x 8 NT rows] = K . q^T,   O^T[D x 8 NT rows] += V^T . P^T
// in warp-level products, the softmax's running maximum and sum in fp32 per row.  The
// warps' results and the ones on the prefix are joined at the end, so the row is written
// once and the loop runs beside the end of the kernel that works on the prefixes.
constexpr int kSmallThreads = 128;
constexpr int kSmallStages = 3;

template <int D>
struct SmallCfg {
  static constexpr int TILE = 16 * D * 2;               // bytes of K (or V) of a step
  static constexpr int WARP = kSmallStages * 2 * TILE;  // a warp's ring
  static constexpr int RING = kSmallThreads / 32 * WARP;
  // after the loop: each warp's [rows][D] sums
  static constexpr int SUMS = kSmallThreads / 32 * kSmallRows * D * 4;
  static constexpr int SMEM = RING > SUMS ? RING : SUMS;
};

// byte offset of 16-byte piece c of row r of a tile: rows of D values, pieces exchanged within 128 bytes
template <int D>
__device__ __forceinline__ uint32_t small_at(int r, int c) {
  return (uint32_t)(r * D * 2 + ((c & ~7) | ((c & 7) ^ (r & 7))) * 16);
}

template <typename T, int D, int NT>
__device__ void small_unit(const ChunkParams& p, const Seq& s, int b, int kvh, unsigned char* smem, float* stat,
                           uint32_t* bad) {
  constexpr int KS = D / 16, PIECES = D / 8;
  using C = SmallCfg<D>;
  constexpr int warps = kSmallThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = s.n * p.group;
  // this lane's rows of each 8: columns 2 (lane % 4) and the next of the products
  int vis[NT][2];
  uint32_t qb[NT][KS][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = t * 8 + 2 * (lane & 3) + i;
      vis[t][i] = r >= rows ? 0 : (s.causal ? s.len - s.n + (int)fdiv((uint32_t)r, p.div_group) + 1 : s.len);
    }
    const int r = t * 8 + (lane >> 2), tok = (int)fdiv((uint32_t)r, p.div_group);
    const T* q = reinterpret_cast<const T*>(p.q + (int64_t)(s.a0 + tok) * p.q_tok +
                                            (int64_t)(kvh * p.group + r - tok * p.group) * p.q_head) + 2 * (lane & 3);
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      qb[t][e][0] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * e)) : 0u;
      qb[t][e][1] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * e + 8)) : 0u;
    }
  }
  const int all_see = s.causal ? max(s.len - s.n + 1, 0) : s.len;  // keys that every row sees
  const int steps = (s.len + 15) / 16;
  const uint32_t ring = smem_u32(smem) + warp * C::WARP;
  const char* kv = p.kv + (int64_t)kvh * p.s_head;
  // lane r < 16: key r of a step; its index entry is asked for a step ahead
  auto entry = [&](int j) -> int {
    const int key = j * 16 + (lane & 15);
    return j < steps && key < s.len ? __ldg(p.indices + s.page0 + (int)fdiv((uint32_t)key, p.div_page)) : -1;
  };
  int id_next = entry(warp);
  auto load = [&](int j, int st) {  // step j's K and V into stage st (an empty group past the end)
    if (j < steps) {
      const int key = j * 16 + (lane & 15), id = id_next;
      const char* src = nullptr;
      if (id >= 0 && id < p.num_pages)
        src = kv + (int64_t)id * p.s_page + (int64_t)(key - (int)fdiv((uint32_t)key, p.div_page) * p.P) * p.s_tok;
      else if (key < s.len && lane < 16) record_status(kStatusBadPage);
      id_next = entry(j + warps);
      const uint32_t dst = ring + st * 2 * C::TILE;
#pragma unroll
      for (int i = 0; i < PIECES / 2; ++i) {
        const int x = i * 32 + lane, r = x / PIECES, c = x % PIECES;
        const char* row =
            reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), r));
        cp_async16(dst + small_at<D>(r, c), row ? row + c * 16 : p.q, row ? 16u : 0u);
        cp_async16(dst + C::TILE + small_at<D>(r, c), row ? row + p.s_kv + c * 16 : p.q, row ? 16u : 0u);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int st = 0; st < kSmallStages - 1; ++st) load(warp + st * warps, st);
  float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int e = 0; e < KS; ++e) o[t][e][0] = o[t][e][1] = o[t][e][2] = o[t][e][3] = 0.f;
  }
  int st = 0, to = kSmallStages - 1;
#pragma unroll 1
  for (int j = warp; j < steps; j += warps) {
    load(j + (kSmallStages - 1) * warps, to);  // (the stage of the step before, which the warp is done with)
    asm volatile("cp.async.wait_group %0;" ::"n"(kSmallStages - 1) : "memory");
    __syncwarp();
    const uint32_t kt = ring + st * 2 * C::TILE, vt = kt + C::TILE;
    const int base = j * 16;
    if (base + 16 > all_see) {
      // values that some rows do not see must be finite (0 x NaN is NaN): others are cleared and noted
      unsigned char* v = smem + (vt - smem_u32(smem));
      for (int x = lane; x < 16 * PIECES; x += 32) {
        const int r = x / PIECES, key = base + r;
        if (key < all_see || key >= s.len) continue;
        uint4* piece = reinterpret_cast<uint4*>(v + small_at<D>(r, x % PIECES));
        const uint4 y = *piece;
        if (!(not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w))) continue;
        *piece = make_uint4(without_not_finite2<T>(y.x), without_not_finite2<T>(y.y), without_not_finite2<T>(y.z),
                            without_not_finite2<T>(y.w));
        atomicOr(bad, 1u << (key - all_see));  // (fewer than kSmallRows keys)
      }
      __syncwarp();
    }
    // ---- S^T = K q^T
    float x[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0.f;
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      uint32_t a[4];  // keys 0-7 | 8-15 of dims 0-7, then of dims 8-15
      ldsm_x4(a, kt + small_at<D>(lane & 15, 2 * e + (lane >> 4)));
#pragma unroll
      for (int t = 0; t < NT; ++t) MmaOp<T>::run(x[t], a, qb[t][e][0], qb[t][e][1]);
    }
    const bool edge = base + 16 > all_see;  // (columns past the rows are nobody's)
    const int k0 = base + (lane >> 2);
    uint32_t pb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (edge) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] = k0 + (e >> 1) * 8 < vis[t][e & 1] ? x[t][e] : -INFINITY;
      }
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(x[t][i], x[t][2 + i]);
#pragma unroll
        for (int w = 4; w <= 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float m_new = fmaxf(m[t][i], mx * p.scale_log2), m_sub = m_new == -INFINITY ? 0.f : m_new;
        alpha[i] = fast_exp2(m[t][i] - m_sub);
        m[t][i] = m_new;
        x[t][i] = fast_exp2(fmaf(x[t][i], p.scale_log2, -m_sub));
        x[t][2 + i] = fast_exp2(fmaf(x[t][2 + i], p.scale_log2, -m_sub));
        l[t][i] = fmaf(l[t][i], alpha[i], x[t][i] + x[t][2 + i]);
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          o[t][e][0] *= alpha[0];
          o[t][e][1] *= alpha[1];
          o[t][e][2] *= alpha[0];
          o[t][e][3] *= alpha[1];
        }
      }
      pb[t][0] = movmatrix_trans(Elem<T>::pack2(x[t][0], x[t][1]));
      pb[t][1] = movmatrix_trans(Elem<T>::pack2(x[t][2], x[t][3]));
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      uint32_t a[4];  // dims 0-7 | 8-15 of keys 0-7, then of keys 8-15
      ldsm_x4_trans(a, vt + small_at<D>((lane & 7) + (lane >> 4) * 8, 2 * e + (lane >> 3 & 1)));
#pragma unroll
      for (int t = 0; t < NT; ++t) MmaOp<T>::run(o[t][e], a, pb[t][0], pb[t][1]);
    }
    __syncwarp();  // the stage may be filled again
    st = st + 1 == kSmallStages ? 0 : st + 1;
    to = to + 1 == kSmallStages ? 0 : to + 1;
  }
  cp_async_wait_all();
  __syncthreads();
  // ---- the warps' results, a row at a time
  float* sums = reinterpret_cast<float*>(smem) + warp * (kSmallRows * D);  // [row][D]
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = t * 8 + 2 * (lane & 3) + i;
#pragma unroll
      for (int w = 4; w <= 16; w <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], w);
      if (lane < 4) {
        stat[(warp * kSmallRows + r) * 2] = m[t][i];
        stat[(warp * kSmallRows + r) * 2 + 1] = l[t][i];
      }
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        sums[r * D + 16 * e + (lane >> 2)] = o[t][e][i];
        sums[r * D + 16 * e + 8 + (lane >> 2)] = o[t][e][2 + i];
      }
    }
  }
  __syncthreads();
  grid_dep_wait();
  constexpr int N = D / 32, RW = NT * 8 / warps;  // rows of a warp
  // where the prefix's results of the warp's rows are: a lane per row, and the parts' log-sum-exps of all rows at once
  auto row_of = [&](int r) -> int64_t {
    const int tok = (int)fdiv((uint32_t)r, p.div_group);
    return (int64_t)(s.a0 + tok) * p.Hq + kvh * p.group + r - tok * p.group;
  };
  int2 at = make_int2(kDone, 0);
  if (s.prefix && lane < RW && warp + lane * warps < rows) at = row_place(p, row_of(warp + lane * warps));
  RowParts parts[RW];
  float largest[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int2 w = make_int2(__shfl_sync(0xffffffffu, at.x, i), __shfl_sync(0xffffffffu, at.y, i));
    if (w.x == kDone) parts[i] = RowParts{0, kWhole, 0};
    else if (i && w.x == parts[i - 1].first && parts[i - 1].count) parts[i] = RowParts{parts[i - 1].count, w.x, w.y};
    else parts[i] = row_parts(p, w);
    const float* o;  // (the first 32 of them)
    largest[i] = row_result<D>(p, 0, row_of(warp + i * warps), parts[i], lane, o);
  }
#pragma unroll 1
  for (int i = 0; i < RW; ++i) {
    const int r = warp + i * warps;
    if (r >= rows) break;
    RowParts front = parts[0];
    float big = largest[0];
#pragma unroll
    for (int e = 1; e < RW; ++e)
      if (e == i) {
        front = parts[e];
        big = largest[e];
      }
    const int tok = (int)fdiv((uint32_t)r, p.div_group), head = kvh * p.group + r - tok * p.group;
    const int64_t row = row_of(r);
    float ml = -INFINITY;  // log2 units
#pragma unroll
    for (int w = 0; w < warps; ++w) ml = fmaxf(ml, stat[(w * kSmallRows + r) * 2]);
    const float part = big;
    if (front.count > 32) {
      big = largest_result<D>(p, 0, row, front);
    } else {
#pragma unroll
      for (int w = 16; w; w >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, w));
    }
    const float M = fmaxf(ml * kLn2, big), Ms = M == -INFINITY ? 0.f : M;
    float acc[N] = {}, den = 0.f;
    if (front.count > 32) {
      add_results<D, N>(p, 0, row, front, Ms, den, acc);
    } else if (front.count) {
      const int place = lane ? 2 * ((front.first >> 1) + lane) : front.first;
      const float* o = front.first < 0 ? p.row_o + row * D : p.part_o + ((int64_t)place * p.part_rows + front.r) * D;
      if (front.count <= 4) add_weighted<N, 4>(front.count, part, o, Ms, den, acc);
      else add_weighted<N, 16>(front.count, part, o, Ms, den, acc);
    }
#pragma unroll
    for (int w = 0; w < warps; ++w) {
      const float mw = stat[(w * kSmallRows + r) * 2], lw = stat[(w * kSmallRows + r) * 2 + 1];
      if (!(lw > 0.f || lw != lw)) continue;  // no key of the warp's is seen
      const float e = fast_exp2(mw - Ms * kLog2e);
      den = fmaf(e, lw, den);
      const float* src = reinterpret_cast<const float*>(smem) + (w * kSmallRows + r) * D + lane * N;
#pragma unroll
      for (int c = 0; c < N; ++c) acc[c] = fmaf(e, src[c], acc[c]);
    }
    if (*bad) {  // the values that were cleared, where the row sees them
      const int sees = s.causal ? s.len - s.n + tok + 1 : s.len;
      for (uint32_t left = *bad; left; left &= left - 1) {
        const int key = all_see + __ffs(left) - 1;
        if (key >= sees) break;
        const int pg = (int)fdiv((uint32_t)key, p.div_page), page = __ldg(p.indices + s.page0 + pg);
        if (page < 0 || page >= p.num_pages) continue;
        const T* v = reinterpret_cast<const T*>(kv + p.s_kv + (int64_t)page * p.s_page + (int64_t)(key - pg * p.P) * p.s_tok);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const float y = Elem<T>::to_float(v[lane * N + c]);
          if (!isfinite(y)) acc[c] += y;
        }
      }
    }
    store_row<T, N>(p, s.a0 + tok, head, Ms, den, acc);
  }
}

// CTAs past the units join the other rows (launched that way where they are few).
template <typename T, int D>
__global__ void __launch_bounds__(kSmallThreads) chunk_small_kernel(const ChunkParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float stat[kSmallThreads / 32 * kSmallRows * 2];
  __shared__ uint32_t bad;
  const int unit = blockIdx.x;
  if (unit >= p.batch * p.Hkv) {
    grid_dep_wait();
    join_rows<T, D>(p, (int64_t)(unit - p.batch * p.Hkv) * (kSmallThreads / 32) + (threadIdx.x >> 5));
    return;
  }
  const int b = p.order[unit / p.Hkv], kvh = unit % p.Hkv;
  const Seq s = p.own[b];
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (!is_small(p, s)) {
    grid_dep_wait();  // (a kernel after this one relies on the one before it)
    return;
  }
  const int rows = s.n * p.group;
  if (rows <= 8) small_unit<T, D, 1>(p, s, b, kvh, smem, stat, &bad);
  else if (rows <= 16) small_unit<T, D, 2>(p, s, b, kvh, smem, stat, &bad);
  else if (rows <= 24) small_unit<T, D, 3>(p, s, b, kvh, smem, stat, &bad);
  else small_unit<T, D, 4>(p, s, b, kvh, smem, stat, &bad);
}

// -------------------------------------------------------------------------
// host
// -------------------------------------------------------------------------
struct Layout {
  int grid, part_rows, TQ;
  size_t parts, lse, o, cost, units, plan, share, seqs, own, prefix, order, row_o, row_lse, row_at, bytes;
};

// The grid is one CTA per SM, or less where the tables' bounds show that there
// are fewer tiles: a sequence has at most one unit more per head than its rows
// fill, and a unit at most as many tiles as all pages hold.
Layout make_layout(const akt_chunk_paged_args* a, int groups, bool shared) {
  Layout y{};
  const int G = a->num_qo_heads / a->num_kv_heads;
  y.TQ = BM / G;
  int64_t units = (int64_t)a->num_tokens / (2 * y.TQ) + std::min<int64_t>(a->batch, a->num_tokens);
  if (shared) units += (int64_t)a->num_tokens / (2 * y.TQ) + std::min<int64_t>(groups, a->num_tokens);
  units *= a->num_kv_heads;
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
  const size_t seqs = (size_t)a->batch + (size_t)groups;
  if (shared || a->batch > kTableSeqs) {
    y.cost = take((seqs + 1) * 8);
    y.units = take((seqs + 1) * 4);
    y.plan = take(sizeof(Plan));
    y.share = take(((size_t)y.grid + 1) * 8);
  }
  if (shared) {
    const size_t rows = (size_t)a->num_tokens * a->num_qo_heads;
    y.seqs = take(seqs * sizeof(Seq));
    y.own = take((size_t)a->batch * sizeof(Seq));
    y.prefix = take((size_t)a->batch * 4);
    y.order = take((size_t)a->batch * 4);
    const size_t results = groups ? 2 * rows : 0;  // (rows without a prefix have theirs in the output or in parts)
    y.row_o = take(results * a->head_dim * 4);
    y.row_lse = take(results * 4);
    y.row_at = take(2 * rows * sizeof(int2));
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

template <typename T, int D, bool TMA, bool SHARED>
int launch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkParams& p,
                 cudaStream_t st) {
  auto kern = chunk_fwd_kernel<T, D, TMA, SHARED>;
  constexpr int smem = (int)Cfg<D>::SMEM_ALL;
  // the register split in the kernel is only valid at the compiled count
  static const int regs = [&] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs != kLaunchRegs)
    return set_error(AKT_ERR_CUDA, "chunk kernel compiled with " + std::to_string(regs) + " registers, expected " +
                                       std::to_string(kLaunchRegs));
  cudaError_t e = ensure_smem_limit<chunk_fwd_kernel<T, D, TMA, SHARED>>((size_t)smem);
  if (e != cudaSuccess) return set_error(AKT_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  const bool planned = SHARED || p.B > kTableSeqs;
  if (planned) chunk_plan_kernel<SHARED><<<1, 1024, 0, st>>>(p);
  {
    ProfileScope prof(st);
    if (planned) e = launch_dependent(kern, dim3(p.grid), dim3(kThreads), smem, st, mq, mk, mv, p);
    else kern<<<p.grid, kThreads, smem, st>>>(mq, mk, mv, p);
  }
  if (SHARED && e == cudaSuccess) {
    constexpr int per = kMergeThreads / 32 * kJoinRows, per_small = kSmallThreads / 32 * kJoinRows;
    const int64_t rows = p.num_tokens * p.Hq;
    const bool fold = rows <= kFoldRows;
    const int64_t units = (int64_t)p.batch * p.Hkv;
    constexpr size_t smem_small = SmallCfg<D>::SMEM;
    e = ensure_smem_limit<chunk_small_kernel<T, D>>(smem_small);
    if (e == cudaSuccess)
      e = launch_dependent(chunk_small_kernel<T, D>, dim3((unsigned)(units + (fold ? (rows + per_small - 1) / per_small : 0))),
                           dim3(kSmallThreads), smem_small, st, p);
    if (e == cudaSuccess && !fold)
      e = launch_dependent(chunk_join_kernel<T, D>, dim3((unsigned)((rows + per - 1) / per)), dim3(kMergeThreads), 0, st, p);
  } else if (e == cudaSuccess)
    e = launch_dependent(chunk_merge_kernel<T, D>, dim3(2 * p.grid, (p.part_rows + p.merge_rows - 1) / p.merge_rows),
                         dim3(kMergeThreads), 0, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : set_error(AKT_ERR_CUDA, std::string("chunk_paged: ") + cudaGetErrorString(e));
}

template <typename T, int D>
int dispatch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkParams& p,
                   cudaStream_t st) {
  if (p.row_at)
    return p.box_rows ? launch_chunk<T, D, true, true>(mq, mk, mv, p, st) : launch_chunk<T, D, false, true>(mq, mk, mv, p, st);
  return p.box_rows ? launch_chunk<T, D, true, false>(mq, mk, mv, p, st) : launch_chunk<T, D, false, false>(mq, mk, mv, p, st);
}

}  // namespace

cudaError_t chunk_status_read(unsigned int* v) { return cudaMemcpyFromSymbol(v, g_device_status_local, sizeof(*v)); }

cudaError_t chunk_status_clear() {
  const unsigned int z = 0;
  return cudaMemcpyToSymbol(g_device_status_local, &z, sizeof(z));
}

}  // namespace akt

using namespace akt;

namespace {

size_t workspace_size(const akt_chunk_paged_args* a, int groups, bool shared) {
  if (a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->num_qo_heads % a->num_kv_heads || a->num_tokens <= 0 ||
      a->batch <= 0 || a->num_qo_heads / a->num_kv_heads > BM || a->page_size <= 0 || a->head_dim <= 0 ||
      a->num_page_entries < 0)
    return 0;
  return make_layout(a, groups, shared).bytes;
}

// shared: the groups of a batch with shared prefixes, or null
int run_chunk(const akt_chunk_paged_args* a, const akt_prefix_paged_args* shared, void* workspace, size_t workspace_bytes,
              void* stream) {
  int rc = check_args(a);
  if (rc || a->num_tokens == 0) return rc;
  const int groups = shared ? shared->num_groups : 0;
  const Layout y = make_layout(a, groups, shared != nullptr);
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
  p.batch = a->batch;
  p.groups = groups;
  p.B = a->batch + groups;
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
  if (shared) {
    p.group_indptr = shared->group_indptr;
    p.shared_pages = shared->shared_pages;
    p.seqs = reinterpret_cast<Seq*>(ws + y.seqs);
    p.own = reinterpret_cast<Seq*>(ws + y.own);
    p.prefix_len = reinterpret_cast<int*>(ws + y.prefix);
    p.order = reinterpret_cast<int*>(ws + y.order);
    p.row_o = reinterpret_cast<float*>(ws + y.row_o);
    p.row_lse = reinterpret_cast<float*>(ws + y.row_lse);
    p.row_at = reinterpret_cast<int2*>(ws + y.row_at);
  }
  if (shared || p.B > kTableSeqs) {
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

}  // namespace

extern "C" size_t akt_chunk_paged_workspace_size(const akt_chunk_paged_args* a) {
  return a ? workspace_size(a, 0, false) : 0;
}

extern "C" int akt_chunk_paged(const akt_chunk_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  return run_chunk(a, nullptr, workspace, workspace_bytes, stream);
}

extern "C" size_t akt_prefix_paged_workspace_size(const akt_prefix_paged_args* a) {
  return a && a->num_groups >= 0 ? workspace_size(&a->chunk, a->num_groups, true) : 0;
}

extern "C" int akt_prefix_paged(const akt_prefix_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  if (a->num_groups < 0 || (int64_t)a->num_groups + std::max(a->chunk.batch, 0) > 0x3fffffff)
    return set_error(AKT_ERR_INVALID, "prefix_paged: bad number of groups");
  if ((int64_t)std::max(a->chunk.batch, 0) * std::max(a->chunk.num_kv_heads, 0) > 0x3fffffff)
    return set_error(AKT_ERR_INVALID, "prefix_paged: too many sequences");
  if (a->num_groups > 0 && (!a->group_indptr || !a->shared_pages))
    return set_error(AKT_ERR_INVALID, "prefix_paged: missing groups");
  return run_chunk(&a->chunk, a, workspace, workspace_bytes, stream);
}
