// Eviction from a paged KV cache: which tokens of each head stay, and the pool
// with only those.  No reference counterpart (its sparse decodes take lists of
// kept tokens, SD:7-66, that its drivers draw at random).
//
// Choice.  Of a head's n tokens the first `sinks`, the last `recent` and the k
// heaviest of the others stay.  The k-th largest weight is found by a radix
// select over an order-preserving map of fp32 to 32-bit keys (digits of 11, 11
// and 10 bits from the top, a histogram each), then the list is written in
// ascending order by ballots and prefix sums, the lowest of equal weights first.
// A first histogram, of the largest keys of groups of tokens, leaves few more than k
// of them, which go into lists in shared memory.  A cluster of CTAs shares a head where
// there are few; its histograms and counts are summed over distributed shared memory.
//
// Eviction.  Slot i of a head takes the row of token keep[i].  Lists ascend, so
// keep[i] >= i: rows only move down and a sequence can stay in its own pages.  A
// cluster walks a head's rows in order, a chunk in registers at a time: all of a
// chunk is read before any of it is written (the cluster's barrier), and no later
// chunk's source lies below a slot that is written by then.  So a chunk's reads
// run ahead of the stores of the one before it.
//
// Pages that others have too (named twice by the table, or reserved) are never
// written: one that keeps all its rows in place and is full stays shared, any
// other is replaced by a dead page, in ascending order.  The plan is integer work
// of one cluster on two bits per page.
#include "cluster.cuh"
#include "common.cuh"
#include "profile.cuh"
#include "scan.cuh"

#include <algorithm>
#include <string>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

int cuda_error(const char* what, cudaError_t e) {
  return set_error(AKT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// ---------------------------------------------------------------------------
// choice of the kept tokens
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;  // tokens of a warp's list

struct SelectParams {
  const float* w;
  int64_t w_layer, w_batch, w_head;
  const int32_t* lens;
  int32_t* ind;
  int64_t i_layer, i_batch, i_head;
  int32_t* kept;
  int B, H, width, budget, sinks, recent;
};

// Larger floats have larger keys; -0 is 0, NaN comes below everything, and 0 is no float's key.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 1u;
  const uint32_t u = __float_as_uint(f + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The least float with at least this key (no less than the one of -infinity).
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

// Sum of x over the threads before this one; `sums` holds a value per warp (of one call
// in two: a call's writes follow a barrier after the reads of the one before last).
__device__ __forceinline__ int select_scan(int x, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int y = lane < kSelectWarps ? sums[lane] : 0;
  total = __reduce_add_sync(0xffffffffu, y);
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
  return before + v - x;
}

__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const SelectParams p) {
  extern __shared__ uint32_t lists[];  // each warp's [kList] keys, then each warp's [kList] places in its segment
  __shared__ __align__(16) int hist[4][kBins];
  __shared__ int sums[2][kSelectWarps];
  __shared__ int found[3];      // digit, how many are wanted of it, how many have it
  __shared__ int cta_count[2];  // tokens that stay for sure, tokens at the threshold
  const int C = (int)cluster_size(), rank = (int)cluster_rank(), row = blockIdx.x / C;
  const int h = row % p.H, b = row / p.H % p.B, l = row / p.H / p.B;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int asked = __ldg(p.lens + b), n = min(max(asked, 0), p.width);
  if (asked != n && tid == 0) record_status(kStatusBadToken);
  int32_t* ind = p.ind + l * p.i_layer + b * p.i_batch + h * p.i_head;
  if (l == 0 && h == 0 && rank == 0 && tid == 0) p.kept[b] = min(n, p.budget);
  if (n <= p.budget) {  // all stay
    for (int i = rank * kSelectThreads + tid; i < p.budget; i += C * kSelectThreads) ind[i] = i < n ? i : 0;
    return;
  }
  const float* w = p.w + l * p.w_layer + b * p.w_batch + h * p.w_head;
  // a CTA's slice of the tokens, a warp's segment of it (both multiples of 32)
  const int seg = (((n + C - 1) / C + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32, slice = seg * kSelectWarps;
  const int lo = min(rank * slice, n), hi = min(lo + slice, n);
  const int s0 = min(lo + warp * seg, hi), s1 = min(s0 + seg, hi);
  const int k = p.budget - p.sinks - p.recent, c0 = p.sinks, c1 = n - p.recent;  // candidates [c0, c1)
  uint32_t* list_key = lists + warp * kList;
  int32_t* list_at = reinterpret_cast<int32_t*>(lists + kSelectWarps * kList) + warp * kList;
  for (int i = tid; i < 4 * kBins / 4; i += kSelectThreads) reinterpret_cast<int4*>(&hist[0][0])[i] = make_int4(0, 0, 0, 0);
  if (tid == 0) found[0] = -1;
  if (C > 1) cluster_sync(); else __syncthreads();
  // f(first token of a block of 32 U, whether all are candidates, the lanes' weights of it: NaN where there is none)
  constexpr int U = 8;
  auto blocks = [&](auto&& f) {
    for (int j0 = s0; j0 < s1; j0 += 32 * U) {
      float x[U];
      const bool inside = j0 >= c0 && j0 + 32 * U <= min(s1, c1);
      if (inside) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = __ldg(w + j0 + 32 * u + lane);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = j0 + 32 * u + lane;
          x[u] = j < s1 && j >= c0 && j < c1 ? __ldg(w + j) : __int_as_float(0x7fffffff);
        }
      }
      f(j0, inside, x);
    }
  };
  // The digit at which the sum of histogram d over the cluster, from the top, reaches
  // `want`; how many are wanted of it and how many have it.  False: there are fewer.
  // Rank 0 gets the others' counts.
  auto find = [&](int d, int want) -> bool {
    __syncthreads();
    constexpr int E = kBins / kSelectThreads;
    static_assert(E == 4, "a thread's bins");
    const int at = kBins - E * (tid + 1);  // this thread's bins, from the top down
    int4 own = *reinterpret_cast<const int4*>(&hist[d][at]);
    if (C > 1) {
      if (rank) {
        if (own.x) cluster_add(&hist[d][at], 0, own.x);
        if (own.y) cluster_add(&hist[d][at + 1], 0, own.y);
        if (own.z) cluster_add(&hist[d][at + 2], 0, own.z);
        if (own.w) cluster_add(&hist[d][at + 3], 0, own.w);
      }
      cluster_sync();
      own = cluster_read4(&hist[d][at], 0);
    }
    const int sum = own.x + own.y + own.z + own.w;
    int all;
    int before = select_scan(sum, sums[d & 1], all);
    if (before < want && want <= before + sum) {
      const int c[E] = {own.w, own.z, own.y, own.x};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (before < want && want <= before + c[e]) {
          found[0] = at + E - 1 - e;
          found[1] = want - before;
          found[2] = c[e];
        }
        before += c[e];
      }
    }
    __syncthreads();
    return found[0] >= 0;
  };
  uint32_t least = 1;  // no key below it is one of the k largest
  // The k-th largest of the largest keys of groups is no more than the k-th largest of all.
  // So a histogram of those, of groups of 8 tokens or 2, leaves few more than k keys to
  // look at (k of n: 3 % of 32768 leaves 3 %, 24 % of 131072 leaves 28 %).
  const int group = (int64_t)16 * k <= n ? 8 : ((int64_t)3 * k <= n ? 2 : 0);
  if (k > 0 && group) {
    blocks([&](int, bool, const float (&x)[U]) {
      float m[U / 2];  // (NaN is passed over)
#pragma unroll
      for (int u = 0; u < U / 2; ++u) m[u] = fmaxf(x[2 * u], x[2 * u + 1]);
      if (group == 8) {
        m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        if (m[0] == m[0]) atomicAdd(&hist[3][order_key(m[0]) >> 21], 1);
      } else {
#pragma unroll
        for (int u = 0; u < U / 2; ++u)
          if (m[u] == m[u]) atomicAdd(&hist[3][order_key(m[u]) >> 21], 1);
      }
    });
    if (find(3, k)) least = (uint32_t)found[0] << 21;
    if (least <= order_key(-INFINITY)) least = 1;  // (NaN alone has a key below it)
  }
  // ---- each warp's candidates that are left, in order; where they are more than its list
  // holds they are read again for every pass
  int count = 0;
  const float bound = key_value(least);
  const bool all_left = least == 1;
  blocks([&](int j0, bool inside, const float (&x)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + 32 * u + lane;
      bool left = all_left || x[u] >= bound;
      if (!inside) left = left && j < s1 && j >= c0 && j < c1;
      const unsigned m = __ballot_sync(0xffffffffu, left);
      if (!m) continue;
      const int at = count + __popc(m & ((1u << lane) - 1u));
      if (left && at < kList) {
        list_key[at] = order_key(x[u]);
        list_at[at] = j;
      }
      count += __popc(m);
    }
  });
  __syncwarp();
  // f(token, its key) in order, 32 at a time; key 0: none
  auto each = [&](auto&& f) {
    if (count <= kList) {
      for (int i0 = 0; i0 < count; i0 += 128) {
        int at[4];
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + 32 * e + lane;
          at[e] = i < count ? list_at[i] : 0;
          x[e] = i < count ? list_key[i] : 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i0 + 32 * e < count) f(at[e], x[e]);
      }
    } else {
      blocks([&](int j0, bool inside, const float (&x)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = j0 + 32 * u + lane;
          f(j, inside || (j < s1 && j >= c0 && j < c1) ? order_key(x[u]) : 0u);
        }
      });
    }
  };
  uint32_t top = 0, mask = 0;  // the threshold's digits so far
  int want = k, have = 0;
  if (k > 0) {
#pragma unroll 1
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
      const uint32_t digit_mask = d == 2 ? 0x3ffu : 0x7ffu;
      each([&](int, uint32_t x) {
        if (x >= least && (x & mask) == top) atomicAdd(&hist[d][(x >> shift) & digit_mask], 1);
      });
      find(d, want);
      top |= (uint32_t)found[0] << shift;
      mask |= digit_mask << shift;
      want = found[1];
      have = found[2];
    }
  }
  // ---- Which candidates stay: the ones above the threshold and `want` of the `have` at it
  // (the first ones; where they are all, their order does not matter).
  const bool ties = want < have;
  auto sure = [&](uint32_t x) { return x && k > 0 && (ties ? x > top : x >= top); };
  int n_sure = 0, n_equal = 0;
  each([&](int, uint32_t x) {
    n_sure += sure(x);
    n_equal += ties && x == top;
  });
  int all;
  int sure_before = select_scan(n_sure, sums[1], all);
  if (tid == 0) cta_count[0] = all;
  int equal_before = 0;
  if (ties) {
    equal_before = select_scan(n_equal, sums[0], all);
    if (tid == 0) cta_count[1] = all;
  }
  sure_before = __shfl_sync(0xffffffffu, sure_before, 0);  // before the warp
  equal_before = __shfl_sync(0xffffffffu, equal_before, 0);
  if (C > 1) {
    cluster_sync();
    // a lane per rank
    sure_before += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_read(&cta_count[0], lane) : 0);
    if (ties) equal_before += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_read(&cta_count[1], lane) : 0);
  }
  // the tokens that always stay stand before and after them
  for (int i = rank * kSelectThreads + tid; i < p.sinks + p.recent; i += C * kSelectThreads)
    ind[i < p.sinks ? i : p.budget - p.recent + i - p.sinks] = i < p.sinks ? i : c1 + i - p.sinks;
  const unsigned below = (1u << lane) - 1u;
  sure_before += p.sinks;
  each([&](int j, uint32_t x) {
    const bool stays = sure(x), equal = ties && x == top;
    const unsigned ms = __ballot_sync(0xffffffffu, stays), me = ties ? __ballot_sync(0xffffffffu, equal) : 0u;
    const int eq = equal_before + __popc(me & below);
    if (stays || (equal && eq < want)) ind[sure_before + __popc(ms & below) + min(eq, want)] = j;
    sure_before += __popc(ms);
    equal_before += __popc(me);
  });
  if (C > 1) cluster_sync();  // the others' reads of this CTA's counts
}

// ---------------------------------------------------------------------------
// eviction: the plan
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanBounds = 4096;  // sequences whose bounds are looked up in shared memory

struct EvictParams {
  char* kv;
  int64_t s_layer, s_page, s_kv, s_head, s_tok;  // bytes
  int64_t num_pages, num_entries, max_entries;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last;
  const int32_t* keep;
  int64_t k_layer, k_batch, k_head;
  const int32_t* kept;
  const uint8_t* reserved;
  float* w;
  int64_t w_layer, w_batch, w_head;
  int32_t* out_indptr;
  int32_t* out_indices;
  int32_t* out_last;
  int layers, B, H, P, M, width;
  FastDiv div_page, div_piece;
  int pieces;  // of a row
  int rows;    // of a CTA's chunk
  // workspace
  uint32_t* seen;   // [words] live pages
  uint32_t* again;  // [words] pages of more than one holder
  int32_t* dead;    // [max_entries] the dead pages that are given out
  int32_t* lens;    // [B] tokens before
  int32_t* count;   // [B] tokens after
  int32_t* moved;   // [B] first page that is replaced, or one past all
};

// The token that a list has for slot i, after `before`; -1 where it is no good (behind
// the sequence, below its slot, or not above the one before it).
__device__ __forceinline__ int checked_token(int i, int j, int before, int len) {
  if (j >= i && j < len && j > before) return j;
  record_status(kStatusBadToken);
  return -1;
}

__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const EvictParams p) {
  __shared__ int64_t sums64[33];
  __shared__ int sums[33];
  __shared__ int n_fresh, n_dead;
  __shared__ int bounds[kPlanBounds + 1];  // the new table's
  const int C = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x;
  const int64_t words = (p.num_pages + 31) / 32;
  const int64_t w0 = words * rank / C, w1 = words * (rank + 1) / C;
  for (int64_t w = w0 + tid; w < w1; w += kPlanThreads) p.seen[w] = p.again[w] = 0;
  cluster_sync();
  if (rank == 0) {  // the new table's bounds (while the others begin to count)
    int64_t at = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
      const int b = b0 + tid;
      int len = 0, n = 0;
      if (b < p.B) {
        const int s = __ldg(p.indptr + b), e = __ldg(p.indptr + b + 1);
        if (s < 0 || e < s || e > p.num_entries) record_status(kStatusBadIndptr);
        else if (e > s) len = (e - s - 1) * p.P + min(max(__ldg(p.last + b), 0), p.P);
        const int asked = __ldg(p.kept + b);
        n = min(max(asked, 0), min(len, p.M));
        if (n != asked) record_status(kStatusBadToken);
      }
      const int pages = (n + p.P - 1) / p.P;
      int64_t total;
      const int64_t begin = at + block_scan<int64_t>(pages, sums64, total);
      const int64_t room = max((int64_t)0, p.max_entries - begin);
      if (b < p.B) {
        if (pages > room) {
          record_status(kStatusListOverflow);
          n = (int)room * p.P;
        }
        const int mine = (n + p.P - 1) / p.P;
        p.out_indptr[b] = (int)min(begin, p.max_entries);
        p.out_last[b] = mine ? n - (mine - 1) * p.P : 0;
        p.lens[b] = len;
        p.count[b] = n;
        p.moved[b] = mine;
      }
      at += total;
    }
    if (tid == 0) p.out_indptr[p.B] = (int)min(at, p.max_entries);
  }
  // pages by how many hold them
  constexpr int U = 4;
  const int counters = max(C - 1, 1), turn = C > 1 ? rank - 1 : 0;  // rank 0 only where it is alone
  for (int64_t i = (int64_t)turn * kPlanThreads + tid; turn >= 0 && i < p.num_entries;
       i += (int64_t)U * counters * kPlanThreads) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = i + (int64_t)u * counters * kPlanThreads;
      id[u] = at < p.num_entries ? __ldg(p.indices + at) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] < 0 || id[u] >= p.num_pages) {
        if (id[u] >= 0) record_status(kStatusBadPage);
        continue;
      }
      const uint32_t bit = 1u << (id[u] & 31);
      if (atomicOr(p.seen + (id[u] >> 5), bit) & bit) atomicOr(p.again + (id[u] >> 5), bit);
    }
  }
  if (p.reserved)
    for (int64_t w = w0 + tid; w < w1; w += kPlanThreads) {
      uint32_t m = 0;
      for (int i = 0; i < 32 && w * 32 + i < p.num_pages; ++i) m |= (p.reserved[w * 32 + i] ? 1u : 0u) << i;
      if (m) {
        atomicOr(p.seen + w, m);
        atomicOr(p.again + w, m);
      }
    }
  cluster_sync();
  // the new table's pages; one that has to be replaced is noted by its number among those
  const int N = __ldcg(p.out_indptr + p.B);
  const bool bounds_here = p.B <= kPlanBounds;
  if (bounds_here)
    for (int i = tid; i <= p.B; i += kPlanThreads) bounds[i] = __ldcg(p.out_indptr + i);
  __syncthreads();
  auto bound = [&](int b) { return bounds_here ? bounds[b] : __ldcg(p.out_indptr + b); };
  const int g0 = (int)((int64_t)N * rank / C), g1 = (int)((int64_t)N * (rank + 1) / C);
  int fresh = 0;
  for (int t0 = g0; t0 < g1; t0 += kPlanThreads) {
    const int g = t0 + tid;
    int page = -1, replace = 0;
    if (g < g1) {
      int b = 0, hi = p.B - 1;
      while (b < hi) {
        const int mid = (b + hi + 1) >> 1;
        if (bound(mid) <= g) b = mid; else hi = mid - 1;
      }
      const int e = g - bound(b), n = __ldcg(p.count + b);
      page = __ldg(p.indices + __ldg(p.indptr + b) + e);
      if (page >= 0 && page < p.num_pages && (__ldcg(p.again + (page >> 5)) >> (page & 31) & 1u)) {
        const int end = min((e + 1) * p.P, n) - 1;  // the page's last row: in its place only if all are
        replace = end + 1 < (e + 1) * p.P;
        for (int l = 0; l < p.layers && !replace; ++l)
#pragma unroll 8
          for (int h = 0; h < p.H; ++h)
            replace |= __ldg(p.keep + l * p.k_layer + b * p.k_batch + h * p.k_head + end) != end;
        if (replace) atomicMin(p.moved + b, e);
      }
    }
    int here;
    const int r = fresh + block_scan<int>(replace, sums, here);
    if (g < g1) p.out_indices[g] = replace ? -2 - r : max(page, -1);
    fresh += here;
  }
  for (int64_t g = (int64_t)N + rank * kPlanThreads + tid; g < p.max_entries; g += (int64_t)C * kPlanThreads)
    p.out_indices[g] = -1;
  if (tid == 0) n_fresh = fresh;
  cluster_sync();
  // over the ranks before this one, and over all: a lane per rank (at most 8)
  const int lane = tid & 31;
  auto over_ranks = [&](const int* count, int& total) -> int {
    const int x = lane < C ? cluster_read(count, lane) : 0;
    total = __reduce_add_sync(0xffffffffu, x);
    return __reduce_add_sync(0xffffffffu, lane < rank ? x : 0);
  };
  int all;
  const int first = over_ranks(&n_fresh, all);
  if (all) {  // the same in every CTA
    // the lowest dead pages, in ascending order
    int mine = 0, dead_here;
    for (int64_t w = w0 + tid; w < w1; w += kPlanThreads) {
      const int64_t left = p.num_pages - w * 32;
      mine += __popc(~__ldcg(p.seen + w) & (left >= 32 ? 0xffffffffu : (1u << left) - 1u));
    }
    block_scan<int>(mine, sums, dead_here);
    if (tid == 0) n_dead = dead_here;
    cluster_sync();
    int found;
    int r0 = over_ranks(&n_dead, found);
    for (int64_t v0 = w0; v0 < w1 && r0 < all; v0 += kPlanThreads) {
      const int64_t w = v0 + tid, left = p.num_pages - w * 32;
      uint32_t d = w < w1 ? ~__ldcg(p.seen + w) & (left >= 32 ? 0xffffffffu : (1u << left) - 1u) : 0u;
      int total;
      int r = r0 + block_scan<int>(__popc(d), sums, total);
      for (; d && r < all; d &= d - 1) p.dead[r++] = (int)(w * 32) + __ffs(d) - 1;
      r0 += total;
    }
    cluster_sync();
    for (int g = g0 + tid; g < g1; g += kPlanThreads) {
      const int v = p.out_indices[g];
      if (v > -2) continue;
      const int r = first + (-2 - v);
      if (r >= found) record_status(kStatusNoDeadPage);
      p.out_indices[g] = r < found ? __ldcg(p.dead + r) : -1;
    }
  }
  cluster_sync();  // the others' reads of this CTA's counts
}

// ---------------------------------------------------------------------------
// eviction: the rows
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 512;
constexpr int kMovePieces = 4;    // of a thread in a chunk
constexpr int kMaxRows = 256;     // of a CTA's chunk

template <int W>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<2> { using type = uint16_t; };

// Cluster (layer, sequence, head, part): part 0 is K, 1 is V, 2 the weights.
template <int W>
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const EvictParams p) {
  using V = typename Piece<W>::type;
  constexpr int U = kMovePieces;
  // Addresses of the rows of several chunks, a row a thread, in three turns: those that
  // are moved, the next ones, and those before, which a warp may still store.  In bytes;
  // from < 0: nothing moves.
  __shared__ int64_t from[3][kMoveThreads], to[3][kMoveThreads];
  __shared__ int in_place[kMoveThreads / 32];
  const int C = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x, parts = p.w ? 3 : 2;
  int unit = blockIdx.x / C;
  const int part = unit % parts;
  unit /= parts;
  const int h = unit % p.H, b = unit / p.H % p.B, l = unit / p.H / p.B;
  grid_dep_wait();
  const int n = p.count[b], len = p.lens[b];
  const int s = __ldg(p.indptr + b), os = p.out_indptr[b];
  const int32_t* keep = p.keep + l * p.k_layer + b * p.k_batch + h * p.k_head;
  // the rows that stay in place are the first ones: as many as stand before the first entry looked at that is not its slot
  const int step = (n + kMoveThreads - 1) / kMoveThreads;
  int start = 0;
  if (n) {
    const int i = min((tid + 1) * step, n) - 1;
    const unsigned moves = __ballot_sync(0xffffffffu, __ldg(keep + i) != i);
    if ((tid & 31) == 0) in_place[tid >> 5] = moves ? (tid + __ffs(moves) - 1) * step : n;
    __syncthreads();
    start = __reduce_min_sync(0xffffffffu, min(in_place[tid & (kMoveThreads / 32 - 1)], n));
  }
  if (part == 2) {
    float* w = p.w + l * p.w_layer + b * p.w_batch + h * p.w_head;
    constexpr int U = 8;
    const int per = U * kMoveThreads, turns = (n - start + C * per - 1) / (C * per);
    for (int it = 0; it < turns; ++it) {
      const int i0 = start + (it * C + rank) * per + tid;
      float v[U];
      int ok = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kMoveThreads;
        const int j = i < n ? checked_token(i, __ldg(keep + i), i ? __ldg(keep + i - 1) : -1, len) : -1;
        v[u] = j >= 0 && j < p.width ? w[j] : 0.f;
        ok |= (j >= 0 && i < p.width) << u;
      }
      cluster_sync();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (ok >> u & 1) w[i0 + u * kMoveThreads] = v[u];
    }
    for (int i = n + rank * kMoveThreads + tid; i < min(len, p.width); i += C * kMoveThreads) w[i] = 0.f;
    return;
  }
  // a page that is replaced takes its rows along even if they stay in their places
  start = (int)min((int64_t)start, (int64_t)p.moved[b] * p.P);
  const int R = p.rows, turns = (n - start + C * R - 1) / (C * R);
  char* base = p.kv + l * p.s_layer + part * p.s_kv + h * p.s_head;
  const int span = kMoveThreads / R;  // chunks whose addresses are made at once (at least 2)
  const int mine = tid / R, r_mine = tid - mine * R;
  auto slot = [&](int q) { return start + ((q * span + mine) * C + rank) * R + r_mine; };
  int2 next;  // the list's entry for this thread's row of the next span, and the one before it
  auto ask = [&](int q) {
    const int i = slot(q);
    next = mine < span && i < n ? make_int2(__ldg(keep + i), i ? __ldg(keep + i - 1) : -1) : make_int2(-1, -1);
  };
  auto address = [&](int q) {
    const int i = slot(q);
    int64_t f = -1, t = 0;
    if (mine < span && i < n) {
      const int j = checked_token(i, next.x, next.y, len);
      if (j >= 0) {
        const int pj = (int)fdiv((uint32_t)j, p.div_page), pi = (int)fdiv((uint32_t)i, p.div_page);
        const int src = __ldg(p.indices + s + pj), dst = p.out_indices[os + pi];
        if (src >= 0 && src < p.num_pages && dst >= 0 && dst < p.num_pages && (src != dst || i != j)) {
          // a page of several holders that was not replaced: the list does not ascend
          if (p.again[dst >> 5] >> (dst & 31) & 1u) {
            record_status(kStatusBadToken);
          } else {
            f = src * p.s_page + (j - pj * p.P) * p.s_tok;
            t = dst * p.s_page + (i - pi * p.P) * p.s_tok;
          }
        }
      }
    }
    from[q % 3][tid] = f;
    to[q % 3][tid] = t;
  };
  V val[2][U];
  auto load = [&](int at, V (&v)[U]) {
    const int64_t* f = &from[0][0] + at;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t x = u * kMoveThreads + tid, r = fdiv(x, p.div_piece);
      if (r < R && f[r] >= 0) v[u] = *reinterpret_cast<const V*>(base + f[r] + (x - r * p.pieces) * W);
    }
  };
  if (!turns) return;
  ask(0);
  address(0);
  ask(1);
  __syncthreads();
  load(0, val[0]);
  if (C > 1) cluster_arrive();
  int here = 0, ahead_at = R, in_span = 0, q = 0;  // this chunk's and the next one's place in the addresses
  // Chunk `it` is stored once all of it has been loaded, and the one after it is on its
  // way by then.  Inside a CTA a barrier orders the accesses; in a cluster the arrival
  // for a chunk waits for its loads and for stores of a turn ago.
  auto turn = [&](int it, V (&cur)[U], V (&ahead)[U]) {
    if (it + 1 < turns) load(ahead_at, ahead);
    if (in_span == 0 && it + span < turns) {
      address(q + 1);
      ask(q + 2);
    }
    if (C > 1) {
      cluster_wait();
      if (it + 1 < turns) cluster_arrive();
    }
    __syncthreads();
    const int64_t *f = &from[0][0] + here, *t = &to[0][0] + here;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t x = u * kMoveThreads + tid, r = fdiv(x, p.div_piece);
      if (r < R && f[r] >= 0) *reinterpret_cast<V*>(base + t[r] + (x - r * p.pieces) * W) = cur[u];
    }
    here = ahead_at;
    if (++in_span == span) {
      in_span = 0;
      ++q;
    }
    ahead_at = in_span + 1 < span ? here + R : (q + 1) % 3 * kMoveThreads;
  };
#pragma unroll 1
  for (int it = 0; it < turns; it += 2) {
    turn(it, val[0], val[1]);
    if (it + 1 < turns) turn(it + 1, val[1], val[0]);
  }
}

size_t round16(size_t n) { return (n + 15) & ~size_t(15); }

struct EvictLayout {
  size_t seen, again, dead, lens, count, moved, bytes;
};

EvictLayout evict_layout(const akt_evict_paged_args* a) {
  EvictLayout y{};
  const size_t words = ((size_t)std::max<int64_t>(a->pool.num_pages, 0) + 31) / 32;
  const size_t batch = (size_t)std::max(a->batch, 0), most = (size_t)std::max<int64_t>(a->max_entries, 0);
  y.again = round16(words * 4);
  y.dead = 2 * y.again;
  y.lens = y.dead + round16(most * 4);
  y.count = y.lens + round16(batch * 4);
  y.moved = y.count + round16(batch * 4);
  y.bytes = y.moved + round16(batch * 4) + 16;
  return y;
}

}  // namespace
}  // namespace akt

using namespace akt;

extern "C" int akt_select_tokens(const akt_select_tokens_args* a, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  if (a->layers < 0 || a->batch < 0 || a->num_heads < 0 || a->width < 0 || a->budget < 0 || a->sinks < 0 || a->recent < 0)
    return set_error(AKT_ERR_INVALID, "select_tokens: bad sizes");
  if ((int64_t)a->sinks + a->recent > a->budget)
    return set_error(AKT_ERR_INVALID, "select_tokens: sinks and recent together must not exceed the budget");
  const int64_t rows = (int64_t)a->layers * a->batch * a->num_heads;
  if (a->width > 0x3fffffff || a->budget > 0x3fffffff || rows > 0x7ffffff)
    return set_error(AKT_ERR_INVALID, "select_tokens: too many tokens");
  if (a->batch > 0 && (!a->seq_lens || !a->keep_len)) return set_error(AKT_ERR_INVALID, "select_tokens: missing tensor");
  if (a->batch == 0) return AKT_OK;
  if (rows == 0) return set_error(AKT_ERR_INVALID, "select_tokens: sequences without heads");
  if ((a->width > 0 && !a->weights) || (a->budget > 0 && !a->keep_ind))
    return set_error(AKT_ERR_INVALID, "select_tokens: missing tensor");
  SelectParams p{};
  p.w = a->weights;
  p.w_layer = a->weights_stride_layer;
  p.w_batch = a->weights_stride_batch;
  p.w_head = a->weights_stride_head;
  p.lens = a->seq_lens;
  p.ind = a->keep_ind;
  p.i_layer = a->keep_stride_layer;
  p.i_batch = a->keep_stride_batch;
  p.i_head = a->keep_stride_head;
  p.kept = a->keep_len;
  p.B = a->batch;
  p.H = a->num_heads;
  p.width = (int)a->width;
  p.budget = a->budget;
  p.sinks = a->sinks;
  p.recent = a->recent;
  // more CTAs to a head while there are SMs without one (512 heads of up to 32768 tokens:
  // one CTA 33 us, two 59, whose exchanges cost more than they save)
  int C = 1;
  while (C < 8 && rows * C < sm_count() && p.width > C * 2048) C *= 2;
  constexpr size_t smem = (size_t)kSelectWarps * kList * 8;
  cudaError_t e = ensure_smem_limit<select_kernel>(smem);
  if (e != cudaSuccess) return cuda_error("select_tokens", e);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    ProfileScope prof(st);
    e = launch_cluster(select_kernel, dim3((unsigned)(rows * C)), dim3(kSelectThreads), C, false, smem, st, p);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("select_tokens", e);
}

extern "C" size_t akt_evict_paged_workspace_size(const akt_evict_paged_args* a) { return a ? evict_layout(a).bytes : 0; }

extern "C" int akt_evict_paged(const akt_evict_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  const akt_page_pool& q = a->pool;
  if (q.num_layers <= 0 || q.num_kv_heads <= 0 || q.page_size <= 0 || q.head_dim <= 0 || q.num_pages < 0)
    return set_error(AKT_ERR_INVALID, "evict_paged: bad pool sizes");
  if (a->batch < 0 || a->num_page_entries < 0 || a->max_entries < 0 || a->max_kept < 0 || a->width < 0)
    return set_error(AKT_ERR_INVALID, "evict_paged: bad sizes");
  if (q.num_pages > 0x7fffff00 || a->num_page_entries > 0x3fffffff / q.page_size || a->max_entries > 0x3fffffff ||
      a->max_kept > 0x3fffffff || a->width > 0x3fffffff)
    return set_error(AKT_ERR_INVALID, "evict_paged: too many tokens");
  if (!q.kv_cache && q.num_pages > 0) return set_error(AKT_ERR_INVALID, "evict_paged: missing pool");
  if (!a->out_indptr || (a->max_entries > 0 && !a->out_indices) ||
      (a->batch > 0 && (!a->kv_page_indptr || !a->kv_last_page_len || !a->out_last_page_len || !a->keep_len)) ||
      (a->batch > 0 && a->max_kept > 0 && !a->keep_ind) || (a->num_page_entries > 0 && !a->kv_page_indices))
    return set_error(AKT_ERR_INVALID, "evict_paged: missing table");
  if (q.stride_dim != 1) return set_error(AKT_ERR_UNSUPPORTED, "evict_paged: unit dim stride required");
  const int64_t row = (int64_t)q.head_dim * 2;
  EvictParams p{};
  p.kv = static_cast<char*>(q.kv_cache);
  p.s_layer = q.num_layers > 1 ? q.stride_layer * 2 : 0;
  p.s_page = q.stride_page * 2;
  p.s_kv = q.stride_kv * 2;
  p.s_head = q.stride_head * 2;
  p.s_tok = q.stride_token * 2;
  // 16-byte pieces where every row and stride allows them, else single values
  const uint64_t bits = (uint64_t)(uintptr_t)q.kv_cache |
                        (uint64_t)(p.s_layer | p.s_page | p.s_kv | (q.num_kv_heads > 1 ? p.s_head : 0) |
                                   (q.page_size > 1 ? p.s_tok : 0) | row);
  const int W = (bits & 15u) ? 2 : 16;
  if (row / W > kMoveThreads * kMovePieces) return set_error(AKT_ERR_UNSUPPORTED, "evict_paged: head_dim too large");
  const int64_t units = (int64_t)q.num_layers * a->batch * q.num_kv_heads;
  if (units > 0x3ffffff) return set_error(AKT_ERR_INVALID, "evict_paged: too many heads");
  const EvictLayout y = evict_layout(a);
  if (!workspace || workspace_bytes < y.bytes)
    return set_error(AKT_ERR_WORKSPACE, "evict_paged: workspace of " + std::to_string(y.bytes) + " bytes required");
  p.num_pages = q.num_pages;
  p.num_entries = a->num_page_entries;
  p.max_entries = a->max_entries;
  p.indptr = a->kv_page_indptr;
  p.indices = a->kv_page_indices;
  p.last = a->kv_last_page_len;
  p.keep = a->keep_ind;
  p.k_layer = a->keep_stride_layer;
  p.k_batch = a->keep_stride_batch;
  p.k_head = a->keep_stride_head;
  p.kept = a->keep_len;
  p.reserved = a->reserved;
  p.w = a->weights;
  p.w_layer = a->weights_stride_layer;
  p.w_batch = a->weights_stride_batch;
  p.w_head = a->weights_stride_head;
  p.out_indptr = a->out_indptr;
  p.out_indices = a->out_indices;
  p.out_last = a->out_last_page_len;
  p.layers = q.num_layers;
  p.B = a->batch;
  p.H = q.num_kv_heads;
  p.P = q.page_size;
  p.M = (int)a->max_kept;
  p.width = (int)a->width;
  p.div_page = make_fastdiv((uint32_t)p.P);
  p.pieces = (int)(row / W);
  p.div_piece = make_fastdiv((uint32_t)p.pieces);
  p.rows = std::min(kMaxRows, kMoveThreads * kMovePieces / p.pieces);
  char* ws = static_cast<char*>(workspace);
  p.seen = reinterpret_cast<uint32_t*>(ws);
  p.again = reinterpret_cast<uint32_t*>(ws + y.again);
  p.dead = reinterpret_cast<int32_t*>(ws + y.dead);
  p.lens = reinterpret_cast<int32_t*>(ws + y.lens);
  p.count = reinterpret_cast<int32_t*>(ws + y.count);
  p.moved = reinterpret_cast<int32_t*>(ws + y.moved);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned planners = p.num_entries > 4 * kPlanThreads ? 8 : 1;
  cudaError_t e = launch_cluster(evict_plan_kernel, dim3(planners), dim3(kPlanThreads), planners, false, 0, st, p);
  if (e == cudaSuccess && units > 0) {
    ProfileScope prof(st);
    const int64_t all = units * (p.w ? 3 : 2);
    int C = 8;
    while (C > 1 && (all * C > 2 * sm_count() || p.M / C < p.rows)) C /= 2;
    const dim3 grid((unsigned)(all * C));
    e = launch_cluster(W == 16 ? evict_move_kernel<16> : evict_move_kernel<2>, grid, dim3(kMoveThreads), C, true, 0, st, p);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("evict_paged", e);
}
