// Forking and compacting the pages of a cache: several sequences may name one page in their block tables (a common prompt, beams
// of one request), and what the tables name is all there is to know: a page that no sequence's cached positions lie on is free.
//
// Fork: new sequence i goes on from sequence parents[i] with its first keep[i] positions and wants pages up to need[i].
//   * full pages are shared, by their number; a page that is partly filled is copied, its filled positions only, unless it can stay
//     with one that goes on in it: when every new sequence that names it would write into it, it stays with the first of them;
//   * fresh pages are the free ones in ascending order, dealt out sequence by sequence. What this call lets go is free for the next
//     one: so no copy reads what another one writes.
// Compact: of U held pages those numbered U and up move into the holes below U, both in ascending order.
//
// The numbers are found in a few steps (mark, look through, deal out): latency; the copies are bound by memory. Up to 32768 pages and table
// entries a call is one kernel, in which every block of threads finds all the numbers for itself, in shared memory, then writes its share of
// the table and copies its share of the pages: 32 beams over 320 pages 4.2 us, with the numbers found by one block and the copies in a
// second kernel 6.3; 112 partly filled pages of 1 MiB, 112 MB moved, 17.9 us, 6.3 TB/s, and 21.0; a compaction of 256 sequences over 4200
// pages 15.7 and 17.4. Larger ones take a cluster of blocks of threads with cluster barriers between the steps, the workspace for what is
// kept, and a second kernel that copies (10.5 us for the beams), and so do compactions in place, whose table one block cannot read while
// another writes it.
#pragma once

#include "rows.cuh"

namespace shahd {

constexpr int kPagesThreads = 1024;
constexpr int kPagesCluster = 8;
constexpr int kCopyThreads = 256;

struct PageCopy {
  int from, to, lines;  // lines: positions of the page; 0: nothing to copy (to = -1: there was no page for it)
};

struct PagesArgs {
  const int *table, *lengths, *parents, *keep, *need;
  int *new_table, *missing, *used;
  int n, new_n, max_blocks, pages, words;
  // workspace
  uint32_t *held, *read;  // bits of pages
  int* first;             // [pages] fork: the first new sequence that would write into a page; compact: where a page goes
  int* order;             // [pages] fork: free pages in order; compact: the holes
  int* start;             // [new_n] fork: number of the first fresh page of a new sequence, in `order`
  int* count;             // [2] fork: free pages; compact: held pages, pages that move
  PageCopy* copies;       // [new_n], or [pages]
};

__device__ __forceinline__ int Blocks(int positions) { return (positions >> 6) + ((positions & 63) != 0); }

// What a new sequence is made of.
struct Fork {
  int parent, keep, kept, upto, beyond;  // kept blocks, blocks that it is to have, and those that its table has no place for
  bool writes;                           // goes on in a page that is partly filled
  __device__ __forceinline__ Fork(const PagesArgs& a, int i) {
    const int most = a.max_blocks * kOpsPage;
    parent = a.parents[i];
    const bool there = (unsigned)parent < (unsigned)a.n;
    keep = there ? min(max(a.keep[i], 0), min(max(a.lengths[parent], 0), most)) : 0;
    if (!there) parent = 0;
    kept = Blocks(keep);
    const int want = max(a.need[i], keep);
    upto = min(Blocks(want), a.max_blocks);
    beyond = Blocks(want) - upto;
    writes = keep % kOpsPage != 0 && want > keep;
  }
};

// Exclusive sums of `v` over a block of threads, and the total.
__device__ __forceinline__ int BlockScan(int v, int* warps, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, count = blockDim.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 31) warps[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = lane < count ? warps[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    warps[lane] = w;
  }
  __syncthreads();
  total = warps[31];
  return incl - v + (warp > 0 ? warps[warp - 1] : 0);
}

// Whether new sequence i has a page to copy.
__device__ __forceinline__ bool Copies(const PagesArgs& a, int i, const Fork& f) {
  if (!f.writes) return false;
  const int page = a.table[(long long)f.parent * a.max_blocks + f.kept - 1];
  if ((unsigned)page >= (unsigned)a.pages) return false;
  return (__ldcg(&a.read[page >> 5]) >> (page & 31) & 1) != 0 || __ldcg(&a.first[page]) != i;
}

template <bool FORK>
__global__ void __launch_bounds__(kPagesThreads) PlanPagesKernel(const __grid_constant__ PagesArgs a) {
  __shared__ int warps[32];
  GridDepWait();
  const int all = kPagesCluster * kPagesThreads, t = (int)blockIdx.x * kPagesThreads + (int)threadIdx.x, rank = blockIdx.x;
  for (int w = t; w < a.words; w += all) {
    a.held[w] = 0;
    if (FORK) a.read[w] = 0;
  }
  if (FORK)
    for (int p = t; p < a.pages; p += all) a.first[p] = 0x7fffffff;
  ClusterSync();
  // ---- which pages are held, and which of them somebody reads without writing ----
  const long long old_entries = (long long)a.n * a.max_blocks, new_entries = (long long)a.new_n * a.max_blocks;
  for (long long e = t; e < old_entries; e += all) {
    const int s = (int)(e / a.max_blocks), b = (int)(e - (long long)s * a.max_blocks);
    if (b >= Blocks(min(max(a.lengths[s], 0), a.max_blocks * kOpsPage))) continue;
    const int page = a.table[e];
    if ((unsigned)page < (unsigned)a.pages) atomicOr(&a.held[page >> 5], 1u << (page & 31));
  }
  if constexpr (FORK) {
    for (long long e = t; e < new_entries; e += all) {
      const int i = (int)(e / a.max_blocks), b = (int)(e - (long long)i * a.max_blocks);
      const Fork f(a, i);
      if (b >= f.kept) continue;
      const int page = a.table[(long long)f.parent * a.max_blocks + b];
      if ((unsigned)page >= (unsigned)a.pages) continue;
      if (f.writes && b == f.kept - 1) atomicMin(&a.first[page], i);
      else atomicOr(&a.read[page >> 5], 1u << (page & 31));
    }
  }
  ClusterSync();
  // ---- sums in order: one block of threads over the pages, another over the new sequences ----
  if (rank == 0) {
    int before = 0, total = 0;
    if constexpr (!FORK) {  // held pages in all
      for (int w0 = 0; w0 < a.words; w0 += kPagesThreads) {
        const int w = w0 + (int)threadIdx.x;
        BlockScan(w < a.words ? __popc(__ldcg(&a.held[w])) : 0, warps, total);
        before += total;
      }
    }
    const int used = before;
    before = 0;
    int moved = 0;
    for (int w0 = 0; w0 < a.words; w0 += kPagesThreads) {
      const int w = w0 + (int)threadIdx.x, base = w * 32;
      const uint32_t bits = w < a.words ? __ldcg(&a.held[w]) : 0;
      uint32_t there = w < a.words ? 0xffffffffu : 0;  // pages of this word that exist
      if (w < a.words && a.pages - base < 32) there = (1u << (a.pages - base)) - 1;
      uint32_t front = there;
      if (!FORK) front = used <= base ? 0 : used - base < 32 ? there & ((1u << (used - base)) - 1) : there;
      uint32_t holes = ~bits & front;
      int at = before + BlockScan(__popc(holes), warps, total);
      before += total;
      for (; holes != 0; holes &= holes - 1) a.order[at++] = base + __ffs(holes) - 1;
      if constexpr (!FORK) {
        uint32_t behind = bits & there & ~front;
        int m = moved + BlockScan(__popc(behind), warps, total);
        moved += total;
        for (; behind != 0; behind &= behind - 1) a.copies[m++] = {base + __ffs(behind) - 1, 0, kOpsPage};
      }
    }
    if (threadIdx.x == 0) {
      a.count[0] = FORK ? before : used;
      if (!FORK) {
        a.count[1] = moved;
        *a.used = used;
      }
    }
  }
  if constexpr (FORK) {
    if (rank == 1) {
      int before = 0, total = 0;
      for (int i0 = 0; i0 < a.new_n; i0 += kPagesThreads) {
        const int i = i0 + (int)threadIdx.x;
        int wants = 0;
        if (i < a.new_n) {
          const Fork f(a, i);
          wants = f.upto - f.kept + (Copies(a, i, f) ? 1 : 0);
        }
        const int at = before + BlockScan(wants, warps, total);
        before += total;
        if (i < a.new_n) a.start[i] = at;
      }
    }
  }
  ClusterSync();
  GridDepLaunch();
  // ---- what is to be copied ----
  if constexpr (FORK) {
    const int free = __ldcg(a.count);
    for (int i = t; i < a.new_n; i += all) {
      const Fork f(a, i);
      const bool copies = Copies(a, i, f);
      const int start = __ldcg(&a.start[i]), wants = f.upto - f.kept + (copies ? 1 : 0);
      a.missing[i] = wants - min(max(free - start, 0), wants) + f.beyond;
      PageCopy c = {0, 0, 0};
      if (copies) {
        if (start < free) c = {a.table[(long long)f.parent * a.max_blocks + f.kept - 1], __ldcg(&a.order[start]), f.keep % kOpsPage};
        else c.to = -1;
      }
      a.copies[i] = c;
    }
  } else {
    const int moved = __ldcg(&a.count[1]);
    for (int m = t; m < moved; m += all) {
      const int to = __ldcg(&a.order[m]), from = __ldcg(&a.copies[m].from);
      a.copies[m].to = to;
      a.first[from] = to;
    }
  }
}

constexpr int kPagesSmall = 32768;  // pages, and entries of either table, that one block of threads sees to
constexpr int kPagesSmallRows = 1024;
constexpr int kNoCopy = -2;

// What one block of threads holds in shared memory.
struct PagesShared {
  uint32_t held[kPagesSmall / 32], read[kPagesSmall / 32];
  int ahead[kPagesSmall / 32];  // free pages before a word's; compact: holes below U
  int4 rows[kPagesSmallRows];   // fork: of the new sequences the parent's place in the table, whether it goes on in a page, kept blocks, blocks to have
  int start[kPagesSmall / 32];  // compact: rank of a word's first held page among those that move; fork: number of a new sequence's first fresh page
  int to[kPagesSmallRows];      // fork: where a new sequence's page is copied to; -1: there is none for it, kNoCopy: nothing to copy
  int from[kPagesSmallRows];    // fork: that page
  int copying[kPagesSmallRows];  // fork: the new sequences that copy
  int warps[32];
  int first[1];                 // [pages] fork: the first new sequence that would write into a page; compact: what moves, and where it goes
};

// The k-th (from 0) set bit of `bits`.
__device__ __forceinline__ int NthBit(uint32_t bits, int k) {
  int at = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const int below = __popc(bits & ((1u << o) - 1));
    if (k >= below) {
      k -= below;
      bits >>= o;
      at += o;
    }
  }
  return at;
}

// The k-th free page; there is one. ahead: of `words` words of pages.
__device__ __forceinline__ int NthFree(const PagesShared& s, int words, int k) {
  int lo = 0, hi = words;  // ahead[lo] <= k
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.ahead[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo * 32 + NthBit(~s.held[lo], k - s.ahead[lo]);
}

// e / blocks, exact for e below 2^21: (e + 1/2) / blocks is further from whole numbers than its rounding.
struct RowOf {
  float per;
  __device__ __forceinline__ RowOf(int blocks) : per(1.f / (float)blocks) {}
  __device__ __forceinline__ int operator()(int e) const { return (int)(((float)e + 0.5f) * per); }
};

struct CopyArgs {
  uint16_t* pool;
  long long page_stride, layer_stride;  // values
  int layers, parts, d;                 // parts: blocks of 64 positions of a layer (K and V of each head)
  const PageCopy* copies;
  const int* count;  // copies in all, or null: `most`
  int most, split;   // split: blocks of threads that share a layer of a copy
};

// This block's share of `copies` copies, which copy_of numbers; a part (64 positions of a layer's head) a warp.
template <class F>
__device__ __forceinline__ void CopyParts(const CopyArgs& c, int copies, const F& copy_of) {
  const uint32_t row16 = c.d / 8, warps = gridDim.x * (blockDim.x / 32);  // row16: 16-byte pieces of a position
  const uint32_t parts = c.parts, all = (uint32_t)copies * c.layers * parts;
  uint32_t split = 1;  // warps that share a part, where there are more of them
  while (split < 4 && 2 * split * all <= warps) split *= 2;
  for (uint32_t u = (threadIdx.x >> 5) * gridDim.x + blockIdx.x; u < all * split; u += warps) {
    const uint32_t share = u % split, whole = u / split, part = whole % parts, rest = whole / parts, which = rest / c.layers;
    const PageCopy copy = copy_of(which);
    if (copy.to < 0) continue;
    const long long in_page = (rest - which * c.layers) * c.layer_stride + (long long)part * kOpsPage * c.d;
    const uint4* in = reinterpret_cast<const uint4*>(c.pool + copy.from * c.page_stride + in_page);
    uint4* out = reinterpret_cast<uint4*>(c.pool + copy.to * c.page_stride + in_page);
    const uint32_t run = copy.lines * row16;
    for (uint32_t j = share * 128 + (threadIdx.x & 31); j < run; j += 128 * split) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j + 32 * k < run) v[k] = in[j + 32 * k];
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j + 32 * k < run) out[j + 32 * k] = v[k];
    }
  }
}

// A fork that one block of threads can plan: every block plans all of it for itself, then writes its share of the table and copies its share
// of the pages, a part (64 positions of a layer's head) a warp. Nothing passes between blocks of threads.
__global__ void __launch_bounds__(kPagesThreads) ForkPagesSmallKernel(const __grid_constant__ CopyArgs c, const __grid_constant__ PagesArgs a) {
  extern __shared__ __align__(16) uint8_t pages_raw[];
  PagesShared& s = *reinterpret_cast<PagesShared*>(pages_raw);
  const int t = threadIdx.x, most = a.max_blocks * kOpsPage, old_entries = a.n * a.max_blocks, new_entries = a.new_n * a.max_blocks;
  const RowOf row_of(a.max_blocks);
  for (int w = t; w < a.words; w += kPagesThreads) s.held[w] = s.read[w] = 0;
  for (int p = t; p < a.pages; p += kPagesThreads) s.first[p] = 0x7fffffff;
  GridDepWait();
  int4 mine = make_int4(0, 0, 0, 0);  // of new sequence t
  bool writes = false;
  int keep = 0, beyond = 0;
  if (t < a.new_n) {
    const Fork f(a, t);
    writes = f.writes;
    keep = f.keep;
    beyond = f.beyond;
    mine = make_int4(f.parent * a.max_blocks, writes, f.kept, f.upto);
    s.rows[t] = mine;
  }
  __syncthreads();
  // ---- which pages are held, and which of them somebody reads without writing ----
#pragma unroll 4
  for (int e = t; e < old_entries; e += kPagesThreads) {
    const int q = row_of(e), b = e - q * a.max_blocks, page = a.table[e];
    if (b < Blocks(min(max(a.lengths[q], 0), most)) && (unsigned)page < (unsigned)a.pages) atomicOr(&s.held[page >> 5], 1u << (page & 31));
  }
#pragma unroll 4
  for (int e = t; e < new_entries; e += kPagesThreads) {
    const int i = row_of(e), b = e - i * a.max_blocks;
    const int4 f = s.rows[i];
    if (b >= f.z) continue;
    const int page = a.table[f.x + b];
    if ((unsigned)page >= (unsigned)a.pages) continue;
    if (f.y && b == f.z - 1) atomicMin(&s.first[page], i);
    else atomicOr(&s.read[page >> 5], 1u << (page & 31));
  }
  __syncthreads();
  // ---- free pages in order; what the new sequences want of them, and what is to be copied ----
  uint32_t bits = 0, there = 0;
  if (t < a.words) {
    bits = s.held[t];
    there = a.pages - 32 * t < 32 ? (1u << (a.pages - 32 * t)) - 1 : 0xffffffffu;
  }
  int free = 0, total = 0;
  const int ahead = BlockScan(__popc(~bits & there), s.warps, free);
  if (t < a.words) s.ahead[t] = ahead;
  int page = -1;
  if (writes) page = a.table[mine.x + mine.z - 1];
  const bool copy = writes && (unsigned)page < (unsigned)a.pages && ((s.read[page >> 5] >> (page & 31) & 1) != 0 || s.first[page] != t);
  const int wants = mine.w - mine.z + (copy ? 1 : 0);
  constexpr int kOne = 1 << 20;  // more than all that is wanted: 32768 entries and 1024 copies
  const int before = BlockScan(wants + (copy ? kOne : 0), s.warps, total), start = before % kOne, copies = total / kOne;
  GridDepLaunch();
  if (t < a.new_n) {
    s.start[t] = start;
    s.to[t] = !copy ? kNoCopy : start < free ? NthFree(s, a.words, start) : -1;
    s.from[t] = page;
    if (copy) s.copying[before / kOne] = t;
    if (blockIdx.x == 0) a.missing[t] = wants - min(max(free - start, 0), wants) + beyond;
    s.rows[t].y = keep % kOpsPage;
  }
  __syncthreads();
  // ---- this block's share of the table, and of the copies ----
  for (int e = (int)blockIdx.x * kPagesThreads + t; e < new_entries; e += (int)gridDim.x * kPagesThreads) {
    const int i = row_of(e), b = e - i * a.max_blocks, to = s.to[i], copied = to != kNoCopy;
    const int4 f = s.rows[i];
    int entry = -1;
    if (b < f.z - copied) entry = a.table[f.x + b];
    else if (b < f.z) entry = to;
    else if (b < f.w) {
      const int k = s.start[i] + copied + b - f.z;
      if (k < free) entry = NthFree(s, a.words, k);
    }
    a.new_table[e] = entry;
  }
  CopyParts(c, copies, [&](uint32_t which) {
    const int i = s.copying[which];
    return PageCopy{s.from[i], s.to[i], s.rows[i].y};
  });
}

// A compaction that one block of threads can plan, into another table, in the same manner.
__global__ void __launch_bounds__(kPagesThreads) CompactPagesSmallKernel(const __grid_constant__ CopyArgs c, const __grid_constant__ PagesArgs a) {
  extern __shared__ __align__(16) uint8_t pages_raw[];
  PagesShared& s = *reinterpret_cast<PagesShared*>(pages_raw);
  const int t = threadIdx.x, most = a.max_blocks * kOpsPage, entries = a.n * a.max_blocks;
  const RowOf row_of(a.max_blocks);
  for (int w = t; w < a.words; w += kPagesThreads) s.held[w] = 0;
  GridDepWait();
  __syncthreads();
  // ---- which pages are held ----
#pragma unroll 4
  for (int e = t; e < entries; e += kPagesThreads) {
    const int q = row_of(e), b = e - q * a.max_blocks, page = a.table[e];
    if (b < Blocks(min(max(a.lengths[q], 0), most)) && (unsigned)page < (unsigned)a.pages) atomicOr(&s.held[page >> 5], 1u << (page & 31));
  }
  __syncthreads();
  // ---- holes below U in order, and the held pages that go there ----
  uint32_t bits = 0, there = 0;
  if (t < a.words) {
    bits = s.held[t];
    there = a.pages - 32 * t < 32 ? (1u << (a.pages - 32 * t)) - 1 : 0xffffffffu;
  }
  int free = 0, used = 0;
  BlockScan(__popc(bits), s.warps, used);
  const int base = 32 * t;  // holes: free pages below U
  there = used <= base ? 0 : used - base < 32 ? there & ((1u << (used - base)) - 1) : there;
  const int ahead = BlockScan(__popc(~bits & there), s.warps, free);
  if (t < a.words) s.ahead[t] = ahead;
  // held pages from U on, by their rank among them: those in front of each word (the word that U lies in has some below U, too)
  const uint32_t behind = t < a.words ? bits & ~there : 0;
  int all = 0;
  const int rank = BlockScan(__popc(behind), s.warps, all);
  if (t < a.words) s.start[t] = rank - __popc(bits & there);
  __syncthreads();
  GridDepLaunch();
  if (blockIdx.x == 0 && t == 0) *a.used = used;
  // as many pages move as there are holes: from s.first[m], to s.first[free + m]; both lists together name pages once
  const auto rank_of = [&](int p) { return s.start[p >> 5] + __popc(s.held[p >> 5] & ((1u << (p & 31)) - 1)); };
  for (int p = used + t; p < a.pages; p += kPagesThreads) {
    if (!(s.held[p >> 5] >> (p & 31) & 1)) continue;
    const int m = rank_of(p);
    s.first[m] = p;
    s.first[free + m] = NthFree(s, a.words, m);
  }
  __syncthreads();
  // ---- this block's share of the table, and of the copies ----
  for (int e = (int)blockIdx.x * kPagesThreads + t; e < entries; e += (int)gridDim.x * kPagesThreads) {
    const int q = row_of(e), b = e - q * a.max_blocks;
    int page = b < Blocks(min(max(a.lengths[q], 0), most)) ? a.table[e] : -1;
    if ((unsigned)page >= (unsigned)a.pages) page = -1;
    else if (page >= used) page = s.first[free + rank_of(page)];
    a.new_table[e] = page;
  }
  CopyParts(c, free, [&](uint32_t m) { return PageCopy{s.first[m], s.first[free + m], kOpsPage}; });
}

// The entries of the new tables, and copies of the first `lines` positions of every part of a page.
template <bool FORK>
__global__ void __launch_bounds__(kCopyThreads) CopyPagesKernel(const __grid_constant__ CopyArgs a, const __grid_constant__ PagesArgs p) {
  GridDepWait();
  GridDepLaunch();
  const long long entries = (long long)(FORK ? p.new_n : p.n) * p.max_blocks;
  for (long long e = (long long)blockIdx.x * kCopyThreads + threadIdx.x; e < entries; e += (long long)gridDim.x * kCopyThreads) {
    const int i = (int)(e / p.max_blocks), b = (int)(e - (long long)i * p.max_blocks);
    int page = -1;
    if constexpr (FORK) {
      const Fork f(p, i);
      const PageCopy c = p.copies[i];
      const int copies = c.lines != 0 || c.to < 0;
      if (b < f.kept - copies) page = p.table[(long long)f.parent * p.max_blocks + b];
      else if (b < f.kept) page = c.to;
      else if (b < f.upto) {
        const int k = p.start[i] + copies + b - f.kept;
        if (k < p.count[0]) page = p.order[k];
      }
    } else if (b < Blocks(min(max(p.lengths[i], 0), p.max_blocks * kOpsPage))) {
      page = p.table[e];
      if ((unsigned)page >= (unsigned)p.pages) page = -1;
      else if (page >= p.count[0]) page = p.first[page];
    }
    p.new_table[e] = page;
  }
  const long long items = (long long)(a.count ? *a.count : a.most) * a.layers * a.split;
  const int row16 = a.d / 8;  // 16-byte pieces of a position
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int share = (int)(item % a.split);
    const long long rest = item / a.split;
    const int layer = (int)(rest % a.layers);
    const PageCopy c = a.copies[rest / a.layers];
    if (c.lines == 0) continue;
    const uint4* from = reinterpret_cast<const uint4*>(a.pool + c.from * a.page_stride + layer * a.layer_stride);
    uint4* to = reinterpret_cast<uint4*>(a.pool + c.to * a.page_stride + layer * a.layer_stride);
    const int run = c.lines * row16, whole = kOpsPage * row16, total = a.parts * run;  // pieces of a part that are copied, that it has
    const int per = CeilDiv(total, a.split), end = min(total, (share + 1) * per);
    for (int i = share * per + (int)threadIdx.x; i < end; i += 4 * kCopyThreads) {
      uint4 v[4];
      int at[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int j = i + k * kCopyThreads, part = j / run;
        at[k] = part * whole + j - part * run;
        if (j < end) v[k] = from[at[k]];
      }
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (i + k * kCopyThreads < end) to[at[k]] = v[k];
    }
  }
}

struct PagesLayout {
  int words;
  int64_t held, read, first, order, start, count, copies, bytes;
};

inline PagesLayout LayPages(int pages, int new_n) {
  PagesLayout l;
  l.words = CeilDiv(pages, 32);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at = (at + bytes + 255) / 256 * 256;
    return here;
  };
  l.held = take(4LL * l.words);
  l.read = take(4LL * l.words);
  l.first = take(4LL * pages);
  l.order = take(4LL * pages);
  l.start = take(4LL * new_n);
  l.count = take(8);
  l.copies = take((int64_t)sizeof(PageCopy) * std::max(pages, new_n));
  l.bytes = at;
  return l;
}

inline bool CheckPagesSizes(const char* op, int pages, int n, int new_n, int max_blocks) {
  if (pages < 1 || pages > (1 << 24) || n < 0 || n > (1 << 20) || new_n < 0 || new_n > (1 << 20) || max_blocks < 1 || max_blocks > (1 << 24) ||
      (long long)std::max(n, new_n) * max_blocks > (1LL << 30)) {
    SetError("%s: need 1 .. 2^24 pages, 0 .. 2^20 sequences, max_blocks in 1 .. 2^24 and at most 2^30 table entries (got pages=%d n=%d new_n=%d max_blocks=%d)", op,
             pages, n, new_n, max_blocks);
    return false;
  }
  return true;
}

inline bool CheckPool(const char* op, const ShahdPagePool& p) {
  const int64_t one = (int64_t)p.kv_heads * 2 * kOpsPage * p.head_dim;
  const bool sizes = p.layers >= 1 && p.layers <= (1 << 16) && p.kv_heads >= 1 && p.kv_heads <= (1 << 12) && p.head_dim >= 8 && p.head_dim <= 256 && p.head_dim % 8 == 0;
  // the layers of a page lie together, or the pages of a layer
  if (!sizes || p.page_stride < one || p.page_stride % 8 != 0 || p.page_stride > (1LL << 36) ||
      (p.layers > 1 && (p.layer_stride < one || p.layer_stride % 8 != 0 || p.layer_stride > (1LL << 40) ||
                        (p.page_stride < (p.layers - 1) * p.layer_stride + one && p.layer_stride < (p.pages - 1) * p.page_stride + one)))) {
    SetError("%s: the pool needs head_dim a multiple of 8 up to 256, kv_heads in 1 .. 4096, layers in 1 .. 65536 and strides, multiples of 8, that keep pages and layers "
             "apart (got layers=%d kv_heads=%d head_dim=%d page_stride=%lld layer_stride=%lld)",
             op, p.layers, p.kv_heads, p.head_dim, (long long)p.page_stride, (long long)p.layer_stride);
    return false;
  }
  return true;
}

// One kernel for what blocks of threads can plan each for itself; else the numbers, then the copies.
template <bool FORK>
int LaunchPages(const char* op, const ShahdPagePool& pool, PagesArgs a, void* workspace, int sms, cudaStream_t st) {
  const PagesLayout l = LayPages(a.pages, a.new_n);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.words = l.words;
  a.held = reinterpret_cast<uint32_t*>(ws + l.held);
  a.read = reinterpret_cast<uint32_t*>(ws + l.read);
  a.first = reinterpret_cast<int*>(ws + l.first);
  a.order = reinterpret_cast<int*>(ws + l.order);
  a.start = reinterpret_cast<int*>(ws + l.start);
  a.count = reinterpret_cast<int*>(ws + l.count);
  a.copies = reinterpret_cast<PageCopy*>(ws + l.copies);
  CopyArgs c = {};
  c.pool = static_cast<uint16_t*>(pool.data);
  c.page_stride = pool.page_stride;
  c.layer_stride = pool.layers > 1 ? pool.layer_stride : 0;
  c.layers = pool.layers;
  c.parts = pool.kv_heads * 2;
  c.d = pool.head_dim;
  c.copies = a.copies;
  c.count = FORK ? nullptr : a.count + 1;
  c.most = FORK ? a.new_n : a.pages;
  c.split = 1;  // a layer of a page is shared by blocks of threads down to 16 KiB, while there are few
  while (c.split * 1024 < c.parts * c.d * 8 && (long long)c.most * c.layers * c.split < 4 * sms) c.split *= 2;
  TakeLaunchError(nullptr);
  const long long entries = (long long)(FORK ? a.new_n : a.n) * a.max_blocks;
  const long long units = (long long)c.most * c.layers * c.parts;  // of the copies, at most
  const bool small = a.pages <= kPagesSmall && std::max(a.n, a.new_n) * (long long)a.max_blocks <= kPagesSmall && a.new_n <= kPagesSmallRows && units < (1 << 28);
  // eight units, four warps each, or a thousand entries a block of threads, and no more blocks than multiprocessors
  if (small && (FORK || a.table != a.new_table)) {
    const int smem = (int)sizeof(PagesShared) + 4 * a.pages;
    const int blocks = (int)std::min<long long>(std::max(units / 8 + 1, (entries + kPagesThreads - 1) / kPagesThreads), sms);
    const auto kernel = FORK ? ForkPagesSmallKernel : CompactPagesSmallKernel;
    if (EnsureKernelAttrs((const void*)kernel, smem)) LaunchPdl(kernel, dim3(blocks), dim3(kPagesThreads), (size_t)smem, st, c, a);
    return LaunchStatus(op);
  }
  LaunchPdlCluster(PlanPagesKernel<FORK>, dim3(kPagesCluster), dim3(kPagesThreads), 0, dim3(kPagesCluster), st, a);
  const long long items = (long long)c.most * c.layers * c.split;
  LaunchPdl(CopyPagesKernel<FORK>, dim3((unsigned)std::min<long long>(std::max(items, entries / kCopyThreads + 1), 8LL * sms)), dim3(kCopyThreads), 0, st, c, a);
  return LaunchStatus(op);
}

}  // namespace shahd

extern "C" {

int64_t shahd_pages_workspace(int32_t pages, int32_t new_n) {
  using namespace shahd;
  const char* op = "shahd_pages_workspace";
  ClearError();
  if (!CheckPagesSizes(op, pages, 0, new_n, 1)) return SHAHD_EINVAL;
  return LayPages(pages, new_n).bytes;
}

int shahd_pages_fork(const ShahdForkCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_pages_fork";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (!CheckPagesSizes(op, c->pool.pages, c->n, c->new_n, c->max_blocks) || !CheckPool(op, c->pool)) return SHAHD_EINVAL;
  const PagesLayout l = LayPages(c->pool.pages, c->new_n);
  if (c->workspace_bytes < l.bytes) {
    SetError("%s: needs %lld bytes of workspace, got %lld", op, (long long)l.bytes, (long long)c->workspace_bytes);
    return SHAHD_EINVAL;
  }
  const int32_t *old_end = c->table + (int64_t)c->n * c->max_blocks, *new_end = c->new_table + (int64_t)c->new_n * c->max_blocks;
  if (c->table < new_end && c->new_table < old_end) {
    SetError("%s: table and new_table overlap", op);
    return SHAHD_EINVAL;
  }
  if (c->new_n == 0) return SHAHD_OK;
  BufferCheck b(op);
  b.Add("pool.data", c->pool.data, 16);
  if (c->n > 0) {
    b.Add("table", c->table, 4);
    b.Add("lengths", c->lengths, 4);
  }
  b.Add("parents", c->parents, 4);
  b.Add("keep", c->keep, 4);
  b.Add("need", c->need, 4);
  b.Add("new_table", c->new_table, 4);
  b.Add("missing", c->missing, 4);
  b.Add("workspace", c->workspace, 16);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  PagesArgs a = {};
  a.table = c->table;
  a.lengths = c->lengths;
  a.parents = c->parents;
  a.keep = c->keep;
  a.need = c->need;
  a.new_table = c->new_table;
  a.missing = c->missing;
  a.n = c->n;
  a.new_n = c->new_n;
  a.max_blocks = c->max_blocks;
  a.pages = c->pool.pages;
  return LaunchPages<true>(op, c->pool, a, c->workspace, info.sms, static_cast<cudaStream_t>(stream));
}

int shahd_pages_compact(const ShahdCompactCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_pages_compact";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (!CheckPagesSizes(op, c->pool.pages, c->n, 0, c->max_blocks) || !CheckPool(op, c->pool)) return SHAHD_EINVAL;
  const PagesLayout l = LayPages(c->pool.pages, 0);
  if (c->workspace_bytes < l.bytes) {
    SetError("%s: needs %lld bytes of workspace, got %lld", op, (long long)l.bytes, (long long)c->workspace_bytes);
    return SHAHD_EINVAL;
  }
  const int64_t entries = (int64_t)c->n * c->max_blocks;
  if (c->table != c->new_table && c->table < c->new_table + entries && c->new_table < c->table + entries) {
    SetError("%s: table and new_table overlap; they may be one", op);
    return SHAHD_EINVAL;
  }
  BufferCheck b(op);
  b.Add("pool.data", c->pool.data, 16);
  if (c->n > 0) {
    b.Add("table", c->table, 4);
    b.Add("lengths", c->lengths, 4);
    b.Add("new_table", c->new_table, 4);
  }
  b.Add("used", c->used, 4);
  b.Add("workspace", c->workspace, 16);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  PagesArgs a = {};
  a.table = c->table;
  a.lengths = c->lengths;
  a.new_table = c->new_table;
  a.used = c->used;
  a.n = c->n;
  a.max_blocks = c->max_blocks;
  a.pages = c->pool.pages;
  return LaunchPages<false>(op, c->pool, a, c->workspace, info.sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
