// Pages of a paged KV cache: copied, forked with copy on write, compacted and
// listed as free.  No reference counterpart (its drivers build one fixed table).
//
// The page table is the only record: a page is live when the table names it
// (or a caller's `reserved` byte marks it), so there are no reference counts
// to keep in step, a dropped sequence frees its pages by not being named, and
// every call gives the same result when it is repeated on the same table.
//
// Each call is a plan by one CTA and then, where pages are copied, a grid that
// applies it.  The plan is integer work on a bit or two per page, held in shared
// memory up to kSmemPages pages: mark the live pages, then walk the words with
// block-wide prefix sums of their popcounts, which hands out dead pages in
// ascending order.  Writes go to dead pages only and reads come from live
// ones, so the copies of one call never meet.
#include "common.cuh"
#include "profile.cuh"

#include <algorithm>
#include <string>

namespace akt {
int set_error(int code, const std::string& msg);

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int64_t kSmemPages = 768 * 1024;  // two bitmaps of 96 KB

// ---------------------------------------------------------------------------
// the pool as pieces of W bytes: piece -> byte offset inside a page
// ---------------------------------------------------------------------------
struct PoolView {
  char* base;
  int64_t s_layer, s_page, s_kv, s_head, s_tok;  // bytes
  int64_t num_pages;
  int layers;
  FastDiv div_row, div_tok, div_head;  // pieces of a row; rows of a head; heads of K (or V)
  uint32_t pieces;                     // pieces of one page and layer
  int contiguous;                      // the page is one run of bytes (the kernels' RUN)
};

template <int W>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<2> { using type = uint16_t; };

template <int W, bool RUN>
__device__ __forceinline__ int64_t piece_offset(const PoolView& v, uint32_t i) {
  if (RUN) return (int64_t)i * W;
  uint32_t r = fdiv(i, v.div_row);
  const uint32_t c = i - r * v.div_row.d;
  uint32_t h = fdiv(r, v.div_tok);
  const uint32_t t = r - h * v.div_tok.d;
  const uint32_t kv = fdiv(h, v.div_head);
  h -= kv * v.div_head.d;
  return (int64_t)kv * v.s_kv + (int64_t)h * v.s_head + (int64_t)t * v.s_tok + (int64_t)c * W;
}

// Pieces [i0, i1) of page `src` to page `dst` of one layer by one CTA; U
// independent loads in flight per thread.  RUN: the page is one run of bytes.
template <int W, bool RUN>
__device__ __forceinline__ void copy_pieces(const PoolView& v, int layer, int64_t src, int64_t dst, uint32_t i0,
                                            uint32_t i1) {
  using V = typename Piece<W>::type;
  const char* s = v.base + layer * v.s_layer + src * v.s_page;
  char* d = v.base + layer * v.s_layer + dst * v.s_page;
  constexpr int U = 8;
  for (uint32_t i = i0 + threadIdx.x; i < i1; i += U * kCopyThreads) {
    V val[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kCopyThreads < i1)
        val[u] = *reinterpret_cast<const V*>(s + piece_offset<W, RUN>(v, i + u * kCopyThreads));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kCopyThreads < i1)
        *reinterpret_cast<V*>(d + piece_offset<W, RUN>(v, i + u * kCopyThreads)) = val[u];
  }
}

// ---------------------------------------------------------------------------
// block-wide helpers of the plans (kPlanThreads threads)
// ---------------------------------------------------------------------------
// Exclusive prefix sum of x over the block; total through `total`.  sums: 33 of them.
template <typename S>
__device__ __forceinline__ S block_scan(S x, S* sums, S& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  S v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const S y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    S w = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const S y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sums[lane] = w;
  }
  __syncthreads();
  total = sums[31];
  const S before = warp ? sums[warp - 1] : 0;
  __syncthreads();
  return before + v - x;
}

__device__ __forceinline__ uint32_t word_mask(int64_t num_pages, int64_t w) {  // the pages that word w stands for
  const int64_t left = num_pages - w * 32;
  return left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
}

// Words of `reserved` (a byte per page) or-ed into bits (the caller syncs).
__device__ void mark_reserved(uint32_t* bits, const uint8_t* reserved, int64_t num_pages) {
  const int64_t words = (num_pages + 31) / 32;
  for (int64_t w = threadIdx.x; w < words; w += blockDim.x) {
    uint32_t m = 0;
    for (int i = 0; i < 32 && w * 32 + i < num_pages; ++i) m |= (reserved[w * 32 + i] ? 1u : 0u) << i;
    bits[w] |= m;
  }
}

// Pages idx[0, n) marked by the block's threads; ids past the pool are recorded, negative ones passed over.
__device__ __forceinline__ void mark_entries(uint32_t* bits, const int32_t* idx, int64_t n, int64_t num_pages) {
  constexpr int U = 4, step = kPlanThreads;
  for (int64_t i = threadIdx.x; i < n; i += (int64_t)U * step) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = i + (int64_t)u * step < n ? __ldg(idx + i + (int64_t)u * step) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] < 0 || id[u] >= num_pages) {
        if (id[u] >= 0) record_status(kStatusBadPage);
        continue;
      }
      atomicOr(bits + (id[u] >> 5), 1u << (id[u] & 31));
    }
  }
}

// ---------------------------------------------------------------------------
// copy
// ---------------------------------------------------------------------------
template <int W, bool RUN>
__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(const PoolView v, const int32_t* src, const int32_t* dst, int slices, uint32_t per_slice) {
  const int64_t i = blockIdx.x / slices;
  const uint32_t sl = blockIdx.x - (uint32_t)i * slices;
  const int s = __ldg(src + i), d = __ldg(dst + i);
  if (s < 0 || s >= v.num_pages || d < 0 || d >= v.num_pages) {
    if (threadIdx.x == 0) record_status(kStatusBadPage);
    return;
  }
  if (s == d) return;
  const uint32_t i0 = sl * per_slice, i1 = min(i0 + per_slice, v.pieces);
  for (int l = blockIdx.y; l < v.layers; l += gridDim.y) copy_pieces<W, RUN>(v, l, s, d, i0, i1);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
struct ForkParams {
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last;
  const int32_t* parents;
  const uint8_t* reserved;
  int32_t* out_indptr;
  int32_t* out_indices;
  int32_t* out_last;
  int64_t num_entries, max_entries, num_pages;
  int B, F, P;
  // workspace
  uint32_t* bits;   // [2 * words] when the bitmaps are past shared memory
  int32_t* first;   // [B] first child of each parent, then the child that keeps its partly filled last page
  int32_t* owner;   // [num_pages] first child with the page as its partly filled last one (where parents share it)
  int32_t* start;   // [F] the parent's first entry
  int32_t* rank;    // [F] which copy, -1: none
  int32_t* dead;    // [F] dead pages for the copies, ascending; -1: none left
  int bits_in_smem;
};

// A parent's entries [s, s + n), its last page's tokens; n = 0 for a bad one.
__device__ __forceinline__ bool fork_parent(const ForkParams& p, int c, int& b, int& s, int& n, int& last) {
  b = __ldg(p.parents + c);
  s = n = last = 0;
  if (b < 0 || b >= p.B) return false;
  s = __ldg(p.indptr + b);
  const int e = __ldg(p.indptr + b + 1);
  if (s < 0 || e < s || e > p.num_entries) {
    s = 0;
    return false;
  }
  n = e - s;
  last = __ldg(p.last + b);
  return true;
}

constexpr int kNoChild = 0x7fffffff;

// The partly filled last page of a named parent (its bounds are good); -1: it has none, -2: one outside the pool.
__device__ __forceinline__ int partial_page(const ForkParams& p, int b) {
  const int s = __ldg(p.indptr + b), e = __ldg(p.indptr + b + 1);
  if (e <= s || __ldg(p.last + b) >= p.P) return -1;
  const int id = __ldg(p.indices + e - 1);
  return id >= 0 && id < p.num_pages ? id : -2;
}

// Two bits per page: `held`, a whole page of a named parent or reserved, which nobody may write; and `partial`, a
// partly filled last page.  A partial page that is not held goes over to the first child that ends in it, whichever
// parent's; all others get copies, since each child appends to its last page.  A page with neither bit is dead.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkParams p) {
  extern __shared__ uint32_t bits_s[];
  __shared__ int sums[33];
  __shared__ int64_t entry_sums[33];
  __shared__ int again_s;
  const int64_t words = (p.num_pages + 31) / 32;
  uint32_t* held = p.bits_in_smem ? bits_s : p.bits;
  uint32_t* partial = held + words;
  for (int64_t w = threadIdx.x; w < 2 * words; w += kPlanThreads) held[w] = 0;
  for (int b = threadIdx.x; b < p.B; b += kPlanThreads) p.first[b] = kNoChild;
  if (threadIdx.x == 0) again_s = 0;
  __syncthreads();
  for (int c = threadIdx.x; c < p.F; c += kPlanThreads) {
    int b, s, n, last;
    if (fork_parent(p, c, b, s, n, last)) atomicMin(p.first + b, c);
    else record_status(kStatusBadIndptr);
  }
  if (p.reserved) mark_reserved(held, p.reserved, p.num_pages);
  __syncthreads();
  // live pages: a team of threads per parent that has a child
  int team = kPlanThreads;
  while (team > 32 && (int64_t)(kPlanThreads / team) < p.B) team >>= 1;
  int again = 0;      // partial pages marked, less those marked once
  bool look = false;  // whether the keepers have to be looked up
  constexpr int U = 4;
  for (int b = threadIdx.x / team; b < p.B; b += kPlanThreads / team) {
    // (asked for together; the bounds of a parent without children may be anything)
    const int child = p.first[b], s = __ldg(p.indptr + b), e = __ldg(p.indptr + b + 1), last = __ldg(p.last + b);
    if (child == kNoChild) continue;
    const int n = e - s, whole = last < p.P ? n - 1 : n;  // the entries before it are whole pages
    for (int64_t i0 = threadIdx.x % team; i0 < n; i0 += (int64_t)U * team) {
      int id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = i0 + (int64_t)u * team < n ? __ldg(p.indices + s + i0 + (int64_t)u * team) : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + (int64_t)u * team;
        if (i >= n) continue;
        if (id[u] < 0 || id[u] >= p.num_pages) {
          record_status(kStatusBadPage);
          look |= i >= whole;
          continue;
        }
        atomicOr((i < whole ? held : partial) + (id[u] >> 5), 1u << (id[u] & 31));
        again += i >= whole;
      }
    }
  }
  // Who keeps a partial page: first[b] stays where b's first child does, and becomes -1 where every child copies and
  // kNoChild where there is nothing to copy.  Only where two parents end in the same page, or one ends in a page that
  // is held or outside the pool, does it change; the other batches pay for the look (fork of 16 beams 8.5 us in a
  // graph against 7.6 without it, of 1024 children of 300 parents 23.0 against 20.1).
  __syncthreads();
  for (int64_t w = threadIdx.x; w < words; w += kPlanThreads) {
    look |= (held[w] & partial[w]) != 0;
    again -= __popc(partial[w]);
  }
  again = __reduce_add_sync(0xffffffffu, again);
  if ((threadIdx.x & 31) == 0 && again) atomicAdd(&again_s, again);
  look = __syncthreads_or(look);
  const bool shared = again_s != 0;
  if (shared) {
    for (int b = threadIdx.x; b < p.B; b += kPlanThreads) {
      const int id = p.first[b] == kNoChild ? -1 : partial_page(p, b);
      if (id >= 0) p.owner[id] = kNoChild;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.B; b += kPlanThreads) {
      const int id = p.first[b] == kNoChild ? -1 : partial_page(p, b);
      if (id >= 0) atomicMin(p.owner + id, p.first[b]);
    }
    __syncthreads();
  }
  if (shared || look) {
    for (int b = threadIdx.x; b < p.B; b += kPlanThreads) {
      const int id = p.first[b] == kNoChild ? -1 : partial_page(p, b);
      if (id == -2) p.first[b] = kNoChild;
      else if (id >= 0 && ((held[id >> 5] >> (id & 31) & 1u) || (shared && p.owner[id] != p.first[b]))) p.first[b] = -1;
    }
  }
  // the children's table bounds, and which of them need a page of their own
  int64_t at = 0;
  int copies = 0;
  for (int c0 = 0; c0 < p.F; c0 += kPlanThreads) {
    const int c = c0 + threadIdx.x;
    int b = 0, s = 0, n = 0, last = 0;
    if (c < p.F) fork_parent(p, c, b, s, n, last);
    // (64 bits: the children may name far more entries than max_entries holds)
    int64_t total;
    const int64_t begin = at + block_scan<int64_t>(n, entry_sums, total);
    const int64_t room = max((int64_t)0, p.max_entries - begin);
    const bool cut = n > room;
    const int kept = cut ? (int)room : n;
    const int keeper = c < p.F && n > 0 ? p.first[b] : kNoChild;
    const int own = !cut && last < p.P && keeper != c && keeper != kNoChild;
    int n_own;
    const int r = copies + block_scan<int>(own, sums, n_own);
    if (c < p.F) {
      if (cut) record_status(kStatusListOverflow);
      p.out_indptr[c] = (int)min(begin, p.max_entries);
      p.out_last[c] = cut ? (kept ? p.P : 0) : last;
      p.start[c] = s;
      p.rank[c] = own ? r : -1;
    }
    at += total;
    copies += n_own;
  }
  if (threadIdx.x == 0) p.out_indptr[p.F] = (int)min(at, p.max_entries);
  __syncthreads();
  // the lowest dead pages, in ascending order
  int found = 0;
  for (int64_t w0 = 0; w0 < words && found < copies; w0 += kPlanThreads) {
    const int64_t w = w0 + threadIdx.x;
    uint32_t d = w < words ? ~(held[w] | partial[w]) & word_mask(p.num_pages, w) : 0u;
    int total;
    int r = found + block_scan(__popc(d), sums, total);
    while (d && r < copies) {
      const int bit = __ffs(d) - 1;
      p.dead[r++] = (int)(w * 32) + bit;
      d &= d - 1;
    }
    found += total;
  }
  for (int r = found + threadIdx.x; r < copies; r += kPlanThreads) {
    p.dead[r] = -1;
    record_status(kStatusNoDeadPage);
  }
}

// One CTA per (child, slice): slice 0 also writes the child's index entries.
template <int W, bool RUN>
__global__ void __launch_bounds__(kCopyThreads)
    fork_apply_kernel(const PoolView v, const ForkParams p, int slices, uint32_t per_slice) {
  grid_dep_wait();
  const int c = blockIdx.x / slices;
  const uint32_t sl = blockIdx.x - (uint32_t)c * slices;
  const int end = p.out_indptr[p.F];
  if (c == p.F) {  // past the table's end
    if (sl == 0)
      for (int64_t e = end + threadIdx.x; e < p.max_entries; e += kCopyThreads) p.out_indices[e] = -1;
    return;
  }
  const int e0 = p.out_indptr[c], n = p.out_indptr[c + 1] - e0, s = p.start[c], r = p.rank[c];
  const int to = r >= 0 ? p.dead[r] : -1;
  if (sl == 0 && blockIdx.y == 0)
    for (int e = threadIdx.x; e < n; e += kCopyThreads)
      p.out_indices[e0 + e] = (r >= 0 && e == n - 1) ? to : __ldg(p.indices + s + e);
  if (to < 0) return;
  const int from = __ldg(p.indices + s + n - 1);
  if (from < 0 || from >= p.num_pages) return;  // recorded by the plan
  const uint32_t i0 = sl * per_slice, i1 = min(i0 + per_slice, v.pieces);
  for (int l = blockIdx.y; l < v.layers; l += gridDim.y) copy_pieces<W, RUN>(v, l, from, to, i0, i1);
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
struct CompactParams {
  const int32_t* indices;
  const uint8_t* reserved;
  int32_t* out_indices;
  int32_t* pages_used;
  int64_t num_entries, num_pages;
  // workspace
  uint32_t* bits;   // [2 * words] when the bitmaps are past shared memory
  int32_t* head;    // [2] moves, first page number past the targets
  int32_t* src;     // [num_pages]
  int32_t* dst;     // [num_pages]
  int32_t* map;     // [num_pages] where a page past the targets goes
  int bits_in_smem;
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
  extern __shared__ uint32_t bits_s[];
  __shared__ int sums[33];
  __shared__ int cut_s, top_s;
  const int64_t words = (p.num_pages + 31) / 32;
  uint32_t* live = p.bits_in_smem ? bits_s : p.bits;
  uint32_t* kept = live + words;  // reserved
  for (int64_t w = threadIdx.x; w < 2 * words; w += kPlanThreads) live[w] = 0;
  if (threadIdx.x == 0) cut_s = top_s = 0;
  __syncthreads();
  mark_entries(live, p.indices, p.num_entries, p.num_pages);
  if (p.reserved) mark_reserved(kept, p.reserved, p.num_pages);
  __syncthreads();
  // pages that may move
  int n = 0;
  for (int64_t w = threadIdx.x; w < words; w += kPlanThreads) {
    live[w] &= ~kept[w];
    n += __popc(live[w]);
    if (kept[w]) atomicMax(&top_s, (int)(w * 32) + 32 - __clz(kept[w]));
  }
  int total;
  block_scan(n, sums, total);
  n = total;
  // Targets are the n lowest pages that are not reserved: the pages below the
  // cut.  The empty ones among them, in order, are the moves' destinations.
  int open = 0, holes = 0;
  for (int64_t w0 = 0; w0 < words && open < n; w0 += kPlanThreads) {
    const int64_t w = w0 + threadIdx.x;
    uint32_t m = w < words ? ~kept[w] & word_mask(p.num_pages, w) : 0u;
    int in_block;
    const int before = open + block_scan(__popc(m), sums, in_block);
    if (before >= n) {
      m = 0;
    } else if (before + __popc(m) >= n) {  // the last target is in this word
      uint32_t rest = m;
      for (int i = 0; i < n - before - 1; ++i) rest &= rest - 1;
      const int bit = __ffs(rest) - 1;
      cut_s = (int)(w * 32) + bit + 1;
      m &= bit == 31 ? 0xffffffffu : (1u << (bit + 1)) - 1u;
    }
    uint32_t h = w < words ? m & ~live[w] : 0u;
    int holes_here;
    int r = holes + block_scan(__popc(h), sums, holes_here);
    for (; h; h &= h - 1) p.dst[r++] = (int)(w * 32) + __ffs(h) - 1;
    open += in_block;
    holes += holes_here;
  }
  __syncthreads();
  const int cut = cut_s;
  // live pages past the cut move, in order
  int moves = 0;
  for (int64_t w0 = cut / 32; w0 < words; w0 += kPlanThreads) {
    const int64_t w = w0 + threadIdx.x;
    const uint32_t past = w == cut / 32 ? ~((1u << (cut & 31)) - 1u) : 0xffffffffu;
    uint32_t m = w < words ? live[w] & past : 0u;
    int here;
    int r = moves + block_scan(__popc(m), sums, here);
    for (; m; m &= m - 1) {
      const int page = (int)(w * 32) + __ffs(m) - 1;
      p.src[r] = page;
      p.map[page] = p.dst[r];
      ++r;
    }
    for (uint32_t k = w < words ? kept[w] & past : 0u; k; k &= k - 1) {
      const int page = (int)(w * 32) + __ffs(k) - 1;
      p.map[page] = page;
    }
    moves += here;
  }
  if (threadIdx.x == 0) {
    p.head[0] = moves;
    p.head[1] = cut;
    p.pages_used[0] = max(cut, top_s);
  }
}

// Persistent: the grid walks (move, slice) pairs of every layer, then rewrites
// its share of the index array.
template <int W, bool RUN>
__global__ void __launch_bounds__(kCopyThreads)
    compact_apply_kernel(const PoolView v, const CompactParams p, int slices, uint32_t per_slice) {
  grid_dep_wait();
  const int moves = p.head[0], cut = p.head[1];
  for (int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < p.num_entries;
       e += (int64_t)gridDim.x * kCopyThreads) {
    const int page = __ldg(p.indices + e);
    p.out_indices[e] = page >= cut && page < p.num_pages ? p.map[page] : page;
  }
  const int64_t jobs = (int64_t)moves * slices * v.layers;
  for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
    const int64_t m = j / slices;
    const uint32_t sl = (uint32_t)(j - m * slices);
    const int l = (int)(m / moves), i = (int)(m - (int64_t)l * moves);
    const uint32_t i0 = sl * per_slice, i1 = min(i0 + per_slice, v.pieces);
    copy_pieces<W, RUN>(v, l, p.src[i], p.dst[i], i0, i1);
  }
}

// ---------------------------------------------------------------------------
// free list
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads)
    free_pages_kernel(const int32_t* indices, int64_t num_entries, const uint8_t* reserved, int64_t num_pages,
                      int32_t* free_pages, int32_t* num_free, uint32_t* bits_g, int bits_in_smem) {
  extern __shared__ uint32_t bits_s[];
  __shared__ int sums[33];
  uint32_t* bits = bits_in_smem ? bits_s : bits_g;
  const int64_t words = (num_pages + 31) / 32;
  for (int64_t w = threadIdx.x; w < words; w += kPlanThreads) bits[w] = 0;
  __syncthreads();
  if (reserved) mark_reserved(bits, reserved, num_pages);
  __syncthreads();
  mark_entries(bits, indices, num_entries, num_pages);
  __syncthreads();
  int n = 0;
  for (int64_t w0 = 0; w0 < words; w0 += kPlanThreads) {
    const int64_t w = w0 + threadIdx.x;
    uint32_t d = w < words ? ~bits[w] & word_mask(num_pages, w) : 0u;
    int total;
    int r = n + block_scan(__popc(d), sums, total);
    for (; d; d &= d - 1) free_pages[r++] = (int)(w * 32) + __ffs(d) - 1;
    n += total;
  }
  for (int64_t i = n + threadIdx.x; i < num_pages; i += kPlanThreads) free_pages[i] = -1;
  if (threadIdx.x == 0) *num_free = n;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
size_t round16(size_t n) { return (n + 15) & ~size_t(15); }

size_t bitmap_bytes(int64_t num_pages) { return round16((size_t)((num_pages + 31) / 32) * 4); }

int check_pool(const akt_page_pool& q) {
  if (q.num_layers <= 0 || q.num_kv_heads <= 0 || q.page_size <= 0 || q.head_dim <= 0 || q.num_pages < 0)
    return set_error(AKT_ERR_INVALID, "pages: bad pool sizes");
  if (q.num_pages > 0x7fffff00) return set_error(AKT_ERR_INVALID, "pages: too many pages");
  if (!q.kv_cache && q.num_pages > 0) return set_error(AKT_ERR_INVALID, "pages: missing pool");
  if (q.stride_dim != 1) return set_error(AKT_ERR_UNSUPPORTED, "pages: unit dim stride required");
  if ((int64_t)2 * q.num_kv_heads * q.page_size * q.head_dim > 0x7fffffff)
    return set_error(AKT_ERR_UNSUPPORTED, "pages: page too large");
  return AKT_OK;
}

// 16-byte pieces where every row and stride allows them, else single values.
int make_view(const akt_page_pool& q, PoolView& v) {
  v.base = static_cast<char*>(q.kv_cache);
  v.s_layer = q.num_layers > 1 ? q.stride_layer * 2 : 0;
  v.s_page = q.stride_page * 2;
  v.s_kv = q.stride_kv * 2;
  v.s_head = q.stride_head * 2;
  v.s_tok = q.stride_token * 2;
  v.num_pages = q.num_pages;
  v.layers = q.num_layers;
  const int64_t row = (int64_t)q.head_dim * 2;
  v.contiguous = (q.page_size == 1 || v.s_tok == row) && (q.num_kv_heads == 1 || v.s_head == row * q.page_size) &&
                 v.s_kv == row * q.page_size * q.num_kv_heads;
  const int64_t page_bytes = 2 * row * q.page_size * q.num_kv_heads;
  uint64_t bits = (uint64_t)(uintptr_t)q.kv_cache | (uint64_t)v.s_page | (uint64_t)v.s_layer;
  bits |= v.contiguous ? (uint64_t)page_bytes : (uint64_t)(v.s_kv | v.s_head | v.s_tok | row);
  const int W = (bits & 15u) ? 2 : 16;
  v.pieces = (uint32_t)(page_bytes / W);
  v.div_row = make_fastdiv((uint32_t)(row / W > 0 ? row / W : 1));
  v.div_tok = make_fastdiv((uint32_t)q.page_size);
  v.div_head = make_fastdiv((uint32_t)q.num_kv_heads);
  return W;
}

// Slices of a page for one CTA each: 32 KB of 16-byte pieces, one turn of a CTA's
// eight loads a thread (compaction of 2300 pages of 64 KB: 54 us, with 16 KB
// slices 63, with 64 KB 55; 302 MB at the measured copy rate take 46)
constexpr uint32_t kSlicePieces = 2048;

int slices_of(const PoolView& v) { return std::max(1, (int)((v.pieces + kSlicePieces - 1) / kSlicePieces)); }


int cuda_error(const char* what, cudaError_t e) {
  return set_error(AKT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

}  // namespace
}  // namespace akt

using namespace akt;

// the kernel for the pool's piece width and layout
#define AKT_PAGES(kern) (W == 16 ? (v.contiguous ? kern<16, true> : kern<16, false>) \
                                 : (v.contiguous ? kern<2, true> : kern<2, false>))

extern "C" int akt_copy_kv_pages(const akt_page_pool* pool, const int32_t* src, const int32_t* dst, int64_t n,
                                 void* stream) {
  if (!pool) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_pool(*pool);
  if (rc) return rc;
  if (n < 0) return set_error(AKT_ERR_INVALID, "copy_kv_pages: bad count");
  if (n == 0) return AKT_OK;
  if (!src || !dst) return set_error(AKT_ERR_INVALID, "copy_kv_pages: missing page lists");
  PoolView v{};
  const int W = make_view(*pool, v);
  const int slices = slices_of(v);
  if (n * slices > 0x7fffffff) return set_error(AKT_ERR_INVALID, "copy_kv_pages: too many copies");
  const dim3 grid((unsigned)(n * slices), (unsigned)std::min(v.layers, 65535));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    ProfileScope prof(st);
    auto kern = AKT_PAGES(copy_pages_kernel);
    kern<<<grid, kCopyThreads, 0, st>>>(v, src, dst, slices, kSlicePieces);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("copy_kv_pages", e);
}

static size_t fork_workspace(const akt_fork_paged_args* a) {
  const int64_t pages = std::max<int64_t>(a->pool.num_pages, 0);
  const size_t bits = pages > kSmemPages ? 2 * bitmap_bytes(pages) : 0;
  return bits + round16((size_t)std::max(a->batch, 0) * 4) + 3 * round16((size_t)std::max(a->num_children, 0) * 4) +
         round16((size_t)pages * 4) + 16;
}

extern "C" size_t akt_fork_paged_workspace_size(const akt_fork_paged_args* a) { return a ? fork_workspace(a) : 0; }

extern "C" int akt_fork_paged(const akt_fork_paged_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_pool(a->pool);
  if (rc) return rc;
  if (a->batch < 0 || a->num_children < 0 || a->num_page_entries < 0 || a->max_entries < 0)
    return set_error(AKT_ERR_INVALID, "fork_paged: bad sizes");
  if (a->num_page_entries > 0x7fffffff || a->max_entries > 0x7fffffff)
    return set_error(AKT_ERR_INVALID, "fork_paged: too many entries");
  if (!a->out_indptr || (a->num_children > 0 && (!a->out_last_page_len || !a->parents)) ||
      (a->max_entries > 0 && !a->out_indices) ||
      (a->batch > 0 && (!a->kv_page_indptr || !a->kv_last_page_len)) || (a->num_page_entries > 0 && !a->kv_page_indices))
    return set_error(AKT_ERR_INVALID, "fork_paged: missing table");
  if (!workspace || workspace_bytes < fork_workspace(a))
    return set_error(AKT_ERR_WORKSPACE, "fork_paged: workspace of " + std::to_string(fork_workspace(a)) + " bytes required");
  PoolView v{};
  const int W = make_view(a->pool, v);
  ForkParams p{};
  p.indptr = a->kv_page_indptr;
  p.indices = a->kv_page_indices;
  p.last = a->kv_last_page_len;
  p.parents = a->parents;
  p.reserved = a->reserved;
  p.out_indptr = a->out_indptr;
  p.out_indices = a->out_indices;
  p.out_last = a->out_last_page_len;
  p.num_entries = a->num_page_entries;
  p.max_entries = a->max_entries;
  p.num_pages = a->pool.num_pages;
  p.B = a->batch;
  p.F = a->num_children;
  p.P = a->pool.page_size;
  p.bits_in_smem = p.num_pages <= kSmemPages;
  char* ws = static_cast<char*>(workspace);
  if (!p.bits_in_smem) {
    p.bits = reinterpret_cast<uint32_t*>(ws);
    ws += 2 * bitmap_bytes(p.num_pages);
  }
  p.first = reinterpret_cast<int32_t*>(ws);
  ws += round16((size_t)p.B * 4);
  const size_t per_child = round16((size_t)p.F * 4);
  p.start = reinterpret_cast<int32_t*>(ws);
  p.rank = reinterpret_cast<int32_t*>(ws + per_child);
  p.dead = reinterpret_cast<int32_t*>(ws + 2 * per_child);
  p.owner = reinterpret_cast<int32_t*>(ws + 3 * per_child);
  const size_t smem = p.bits_in_smem ? 2 * bitmap_bytes(p.num_pages) : 0;
  cudaError_t e = ensure_smem_limit<fork_plan_kernel>(smem);
  if (e != cudaSuccess) return cuda_error("fork_paged", e);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int slices = slices_of(v);
  const int64_t ctas = (int64_t)(p.F + 1) * slices;
  if (ctas > 0x7fffffff) return set_error(AKT_ERR_INVALID, "fork_paged: too many children");
  fork_plan_kernel<<<1, kPlanThreads, smem, st>>>(p);
  {
    ProfileScope prof(st);
    const dim3 grid((unsigned)ctas, (unsigned)std::min(v.layers, 65535));
    e = launch_dependent(AKT_PAGES(fork_apply_kernel), grid, dim3(kCopyThreads), 0, st, v, p, slices, kSlicePieces);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("fork_paged", e);
}

static size_t compact_workspace(const akt_compact_paged_args* a) {
  const int64_t n = std::max<int64_t>(a->pool.num_pages, 0);
  const size_t bits = n > kSmemPages ? 2 * bitmap_bytes(n) : 0;
  return bits + 16 + 3 * round16((size_t)n * 4);
}

extern "C" size_t akt_compact_paged_workspace_size(const akt_compact_paged_args* a) {
  return a ? compact_workspace(a) : 0;
}

extern "C" int akt_compact_paged(const akt_compact_paged_args* a, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!a) return set_error(AKT_ERR_INVALID, "null args");
  int rc = check_pool(a->pool);
  if (rc) return rc;
  if (a->num_page_entries < 0) return set_error(AKT_ERR_INVALID, "compact_paged: bad sizes");
  if (!a->pages_used || (a->num_page_entries > 0 && (!a->kv_page_indices || !a->out_indices)))
    return set_error(AKT_ERR_INVALID, "compact_paged: missing table");
  if (!workspace || workspace_bytes < compact_workspace(a))
    return set_error(AKT_ERR_WORKSPACE,
                     "compact_paged: workspace of " + std::to_string(compact_workspace(a)) + " bytes required");
  PoolView v{};
  const int W = make_view(a->pool, v);
  CompactParams p{};
  p.indices = a->kv_page_indices;
  p.reserved = a->reserved;
  p.out_indices = a->out_indices;
  p.pages_used = a->pages_used;
  p.num_entries = a->num_page_entries;
  p.num_pages = a->pool.num_pages;
  p.bits_in_smem = p.num_pages <= kSmemPages;
  char* ws = static_cast<char*>(workspace);
  if (!p.bits_in_smem) {
    p.bits = reinterpret_cast<uint32_t*>(ws);
    ws += 2 * bitmap_bytes(p.num_pages);
  }
  p.head = reinterpret_cast<int32_t*>(ws);
  ws += 16;
  const size_t per_page = round16((size_t)p.num_pages * 4);
  p.src = reinterpret_cast<int32_t*>(ws);
  p.dst = reinterpret_cast<int32_t*>(ws + per_page);
  p.map = reinterpret_cast<int32_t*>(ws + 2 * per_page);
  const size_t smem = p.bits_in_smem ? 2 * bitmap_bytes(p.num_pages) : 0;
  cudaError_t e = ensure_smem_limit<compact_plan_kernel>(smem);
  if (e != cudaSuccess) return cuda_error("compact_paged", e);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<1, kPlanThreads, smem, st>>>(p);
  {
    ProfileScope prof(st);
    const dim3 grid((unsigned)(sm_count() * 8));
    const int slices = slices_of(v);
    e = launch_dependent(AKT_PAGES(compact_apply_kernel), grid, dim3(kCopyThreads), 0, st, v, p, slices, kSlicePieces);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("compact_paged", e);
}

extern "C" size_t akt_free_kv_pages_workspace_size(int64_t num_pages) {
  return num_pages > kSmemPages ? bitmap_bytes(num_pages) : 0;
}

extern "C" int akt_free_kv_pages(const int32_t* indices, int64_t num_entries, const uint8_t* reserved,
                                 int64_t num_pages, int32_t* free_pages, int32_t* num_free, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (num_entries < 0 || num_pages < 0 || num_pages > 0x7fffff00)
    return set_error(AKT_ERR_INVALID, "free_kv_pages: bad sizes");
  if (!num_free || (num_pages > 0 && !free_pages) || (num_entries > 0 && !indices))
    return set_error(AKT_ERR_INVALID, "free_kv_pages: missing list");
  const size_t need = akt_free_kv_pages_workspace_size(num_pages);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(AKT_ERR_WORKSPACE, "free_kv_pages: workspace of " + std::to_string(need) + " bytes required");
  const int in_smem = num_pages <= kSmemPages;
  const size_t smem = in_smem ? bitmap_bytes(num_pages) : 0;
  cudaError_t e = ensure_smem_limit<free_pages_kernel>(smem);
  if (e != cudaSuccess) return cuda_error("free_kv_pages", e);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    ProfileScope prof(st);
    free_pages_kernel<<<1, kPlanThreads, smem, st>>>(indices, num_entries, reserved, num_pages, free_pages, num_free,
                                                     static_cast<uint32_t*>(workspace), in_smem);
  }
  e = cudaGetLastError();
  return e == cudaSuccess ? AKT_OK : cuda_error("free_kv_pages", e);
}
