// Pages of paged caches: reserving, forking, freeing, compacting and copying them.
//
// A pool is three int32 arrays on the device: the page table [rows][per_row] (-1: no page), a reference count per page and
// the mapped entries per row. Pages are always taken lowest first and moved lowest to lowest, found with prefix sums, so
// the outcome does not depend on timing; reference counts change by integer atomics, whose sum does not either.
//
// A state change is one CTA's work (a scan of the counts, 4 bytes a page); it leaves a list of page moves that the copy
// kernel, launched behind it as a programmatic dependent, applies to every cache: bound by reading and writing the moved
// pages once.
#pragma once
#include "palu_common.cuh"

namespace palu {
namespace pg {

constexpr int kPlanThreads = 1024;
constexpr int kMaxPairs = 256;    // fork pairs, rows to reserve or free of one launch
constexpr int kMaxCaches = 128;   // caches of one copy launch
constexpr int kMaxCopies = 480;   // host-given page copies of one launch
constexpr int kCopyThreads = 256;
constexpr int kPart = 16384;      // bytes of a page that a CTA copies at a time
// CTAs an SM over all caches, at most: small ones that the scheduler deals out as SMs come free. 126 of 512 pages in 64 caches
// (1.06 GB moved), us, with 8 / 16 / 64 / 128 / 512: 192, 179, 172, 169, 167 (161 at the measured copy rate).
constexpr int kCopyCtas = 128;

enum : int { kErrFull = 1, kErrParent = 2, kErrChild = 4 };

struct Pool {
  int32_t* table;
  int32_t* refs;
  int32_t* mapped;
  int32_t* status;
  int rows, per_row, n_pages, page_size;
};
// Moves of whole pages, and where compaction sends a page.
struct Moves {
  int32_t* count;   // [1]
  int2* list;       // [n_pages] (from, to); `to` < 0: none
};

// Exclusive prefix sum of v over the block; the total in `total`.
PALU_DEVINL int block_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = s_warp[31];
  const int before = (warp ? s_warp[warp - 1] : 0) + x - v;
  __syncthreads();
  return before;
}

// The lowest free pages in order: take(rank, page) for ranks 0 .. want - 1. Returns how many there were (at most want).
template <class Take>
PALU_DEVINL int take_free(const Pool& p, int want, int* s_warp, Take take) {
  int found = 0;
  for (int b0 = 0; b0 < p.n_pages && found < want; b0 += 4 * kPlanThreads) {
    const int b = b0 + 4 * threadIdx.x;
    int f[4], n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = b + i < p.n_pages && p.refs[b + i] == 0;
      n += f[i];
    }
    int total, at = found + block_scan(n, s_warp, total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f[i]) {
        if (at < want) take(at, b + i);
        ++at;
      }
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

// Pages of `len` positions (len + size - 1 need not fit 32 bits).
PALU_DEVINL int pages_of(int len, int size) { return len / size + (len % size != 0); }

struct RowLens {
  int n;
  int32_t row[kMaxPairs], len[kMaxPairs];
};
// Rows get pages for `len` positions, in the order given; a row that has them keeps what it has.
__global__ void __launch_bounds__(kPlanThreads) palu_reserve_pages_kernel(const Pool p, const __grid_constant__ RowLens a) {
  __shared__ int s_warp[32], s_at[kMaxPairs + 1], s_have[kMaxPairs];
  int need = 0;
  if (threadIdx.x < a.n) {
    const int have = p.mapped[a.row[threadIdx.x]];
    s_have[threadIdx.x] = have;
    need = max(0, pages_of(a.len[threadIdx.x], p.page_size) - have);
  }
  int total;
  const int at = block_scan(need, s_warp, total);
  if (threadIdx.x < a.n) s_at[threadIdx.x] = at;
  if (threadIdx.x == 0) s_at[a.n] = total;
  __syncthreads();
  const int got = take_free(p, total, s_warp, [&](int rank, int page) {
    int lo = 0, hi = a.n - 1;  // the last row whose first rank is <= rank
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_at[mid] <= rank) lo = mid;
      else hi = mid - 1;
    }
    p.table[(int64_t)a.row[lo] * p.per_row + s_have[lo] + rank - s_at[lo]] = page;
    p.refs[page] = 1;
  });
  if (threadIdx.x < a.n) {  // ranks from `got` on found no page
    const int mine = max(0, min(need, got - at));
    p.mapped[a.row[threadIdx.x]] = s_have[threadIdx.x] + mine;
    if (mine < need) atomicOr(p.status, kErrFull);
  }
}

struct ForkList {
  int n;
  int32_t parent[kMaxPairs], child[kMaxPairs], len[kMaxPairs];
};
// Child rows share their parent's pages of the first `len` positions; a page that these positions fill only partly is
// copied into a page of the child's own.
__global__ void __launch_bounds__(kPlanThreads) palu_fork_pages_kernel(const Pool p, const Moves mv, const __grid_constant__ ForkList a) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  __shared__ int s_warp[32], s_new[kMaxPairs], s_rank[kMaxPairs];
  const int i = threadIdx.x;
  int need = 0;
  bool ok = false;
  if (i < a.n) {
    const int full = a.len[i] / p.page_size, count = pages_of(a.len[i], p.page_size);
    ok = true;
    if (p.mapped[a.parent[i]] < count) {
      atomicOr(p.status, kErrParent);
      ok = false;
    } else if (p.mapped[a.child[i]] != 0) {
      atomicOr(p.status, kErrChild);
      ok = false;
    }
    need = ok && count > full;
  }
  int total;
  const int at = block_scan(need, s_warp, total);
  if (i < kMaxPairs) s_new[i] = -1;
  if (i < a.n) s_rank[i] = ok ? (need ? at : -1) : -2;  // -1: nothing to copy, -2: refused
  __syncthreads();
  const int got = take_free(p, total, s_warp, [&](int rank, int page) { s_new[rank] = page; });
  if (i < a.n && need && at >= got) {
    atomicOr(p.status, kErrFull);
    s_rank[i] = -2;
  }
  if (i == 0) *mv.count = got;
  __syncthreads();
  for (int x = threadIdx.x >> 5; x < a.n; x += kPlanThreads / 32) {  // one warp per pair
    const int rank = s_rank[x];
    if (rank == -2) continue;
    const int full = a.len[x] / p.page_size;
    const int32_t* from = p.table + (int64_t)a.parent[x] * p.per_row;
    int32_t* to = p.table + (int64_t)a.child[x] * p.per_row;
    for (int j = threadIdx.x & 31; j < full; j += 32) {
      const int b = from[j];
      to[j] = b;
      if ((unsigned)b < (unsigned)p.n_pages) atomicAdd(p.refs + b, 1);
    }
    if ((threadIdx.x & 31) == 0) {
      if (rank >= 0) {
        const int b = from[full], page = s_new[rank];
        to[full] = page;
        p.refs[page] = 1;
        mv.list[rank] = make_int2(b, (unsigned)b < (unsigned)p.n_pages ? page : -1);
      }
      p.mapped[a.child[x]] = full + (rank >= 0);
    }
  }
}

struct RowList {
  int n;
  int32_t row[kMaxPairs];
};
// Rows give up their pages; one CTA per row.
__global__ void __launch_bounds__(256) palu_free_pages_kernel(const Pool p, const __grid_constant__ RowList a) {
  const int row = a.row[blockIdx.x], n = p.mapped[row];
  for (int j = threadIdx.x; j < n; j += 256) {
    int32_t* at = p.table + (int64_t)row * p.per_row + j;
    const int b = *at;
    *at = -1;
    if ((unsigned)b < (unsigned)p.n_pages) atomicSub(p.refs + b, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) p.mapped[row] = 0;
}

// Used pages move to the lowest places: with n pages in use, the i-th used page at or above n goes to the i-th free page
// below n. The moves carry the reference counts along.
__global__ void __launch_bounds__(kPlanThreads) palu_compact_pages_kernel(const Pool p, const Moves mv, int32_t* target) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  __shared__ int s_warp[32];
  int mine = 0, used;
  for (int b = threadIdx.x; b < p.n_pages; b += kPlanThreads) mine += p.refs[b] > 0;
  block_scan(mine, s_warp, used);
  int holes = 0, moved = 0;
  for (int b0 = 0; b0 < p.n_pages; b0 += 4 * kPlanThreads) {
    int hole[4], move[4], nh = 0, nm = 0, th, tm;
    const int b = b0 + 4 * threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = b + i < p.n_pages, live = in && p.refs[b + i] > 0;
      hole[i] = in && !live && b + i < used;
      move[i] = live && b + i >= used;
      nh += hole[i];
      nm += move[i];
    }
    int ah = holes + block_scan(nh, s_warp, th), am = moved + block_scan(nm, s_warp, tm);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (hole[i]) mv.list[ah++].y = b + i;
      if (move[i]) mv.list[am++].x = b + i;
    }
    holes += th;
    moved += tm;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
    const int2 m = mv.list[i];
    target[m.x] = m.y;
    p.refs[m.y] = p.refs[m.x];
    p.refs[m.x] = 0;
  }
  if (threadIdx.x == 0) {
    mv.count[0] = moved;
    mv.count[1] = used;
  }
}

struct Caches {
  int n;
  struct {
    unsigned char* base;
    int64_t stride, bytes;  // from page to page, and of a page
  } c[kMaxCaches];
};

template <typename V>
PALU_DEVINL void copy_part(unsigned char* to, const unsigned char* from, int bytes) {
  const V* s = reinterpret_cast<const V*>(from);
  V* d = reinterpret_cast<V*>(to);
  const int n = bytes / (int)sizeof(V);
  for (int i = threadIdx.x; i < n; i += 4 * kCopyThreads) {
    V v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (i + x * kCopyThreads < n) v[x] = s[i + x * kCopyThreads];
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (i + x * kCopyThreads < n) d[i + x * kCopyThreads] = v[x];
  }
}

template <typename V>
PALU_DEVINL void copy_moves(const Caches& a, const int2* list, int count, int n_pages) {
  const auto& c = a.c[blockIdx.y];
  const int parts = (int)((c.bytes + kPart - 1) / kPart);
  const int64_t units = (int64_t)count * parts;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int m = (int)(u / parts), part = (int)(u - (int64_t)m * parts);
    const int2 mv = list[m];
    if ((unsigned)mv.x >= (unsigned)n_pages || (unsigned)mv.y >= (unsigned)n_pages || mv.x == mv.y) continue;
    const int64_t off = (int64_t)part * kPart;
    copy_part<V>(c.base + mv.y * c.stride + off, c.base + mv.x * c.stride + off, (int)min((int64_t)kPart, c.bytes - off));
  }
}

// Applies a device list of moves to every cache (blockIdx.y); with `target`, page table entries at or above the used
// pages follow their pages.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) palu_move_pages_kernel(const Pool p, const Moves mv, const int32_t* target, const __grid_constant__ Caches a) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int count = mv.count[0];
  if (target && count > 0 && blockIdx.y == 0) {
    const int used = mv.count[1];
    for (int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < (int64_t)p.rows * p.per_row; e += (int64_t)gridDim.x * kCopyThreads) {
      const int b = p.table[e];
      if (b >= used && b < p.n_pages) p.table[e] = target[b];
    }
  }
  if (a.n > 0) copy_moves<V>(a, mv.list, count, p.n_pages);
}

struct CopyList {
  int n;
  int2 move[kMaxCopies];
};
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) palu_copy_pages_kernel(int n_pages, const __grid_constant__ CopyList l, const __grid_constant__ Caches a) {
  copy_moves<V>(a, l.move, l.n, n_pages);
}

}  // namespace pg
}  // namespace palu
