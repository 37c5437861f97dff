// Tables of pages and maps of slots, made on the device from the sequences' lengths.
//
// Sequence s of length L holds pages(L) = ceil(L / P) pages, P rows each; table[s][i] is the page of its rows
// i P .. i P + P - 1.  Pages that nobody holds lie in free_pages[0 .. n_free - 1], a stack.  A map changes the length of each
// of its entries by delta: entries that shrink push their last pages, entries that grow take pages from the top, and
// every row gained gets its slot, page * P + row in the page.  With G pages pushed and T taken in all, the pushed ones in
// the order (last entry first, last page first) and the taken ones in the order (first entry first, first page first), the
// j-th page taken is the stack's entry n_free + G - 1 - j: a pushed one for j < G.  So a map followed by its inverse leaves
// the stack as it was, and no step of this needs an atomic operation: where a page comes from follows from prefix sums.
//
// All or nothing: an entry out of range or named twice, a length below 0 or beyond the table's width, too few pages or
// too little room for the rows leave everything as it was, with every slot -1 and the reason in *error.
#include "paged.hpp"

namespace shainet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kEach = kMaxPagedSeqs / kThreads;  // entries of a thread

// What the entries look like once their sums are known; in LDS, and in scratch memory where a second kernel goes on.
struct MapSums {
  int ok, n, rows, gone, taken, top;  // top: n_free before
  int old_len[kMaxPagedSeqs], seq[kMaxPagedSeqs];
  int row_start[kMaxPagedSeqs];   // rows gained by the entries before
  int taken_start[kMaxPagedSeqs]; // pages taken by the entries before
  int gone_behind[kMaxPagedSeqs]; // pages pushed by the entries behind
};

__device__ __forceinline__ int pages_of(int len, int shift) { return (int)(((long long)len + (1 << shift) - 1) >> shift); }

// The last entry whose start is not above x (starts ascend; entries without any share their successor's).
__device__ __forceinline__ int entry_of(const int *start, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
// The same where starts descend: the first entry whose number behind is not above x.
__device__ __forceinline__ int entry_behind(const int *behind, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (behind[mid] <= x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int pushed_page(const MapArgs &a, const MapSums &m, int i) {
  const int e = entry_behind(m.gone_behind, m.n, i);
  return a.table[(long long)m.seq[e] * a.seq_pages + pages_of(m.old_len[e], a.shift) - 1 - (i - m.gone_behind[e])];
}
__device__ __forceinline__ int taken_page(const MapArgs &a, const MapSums &m, int j) {
  return j < m.gone ? pushed_page(a, m, m.gone - 1 - j) : a.free_pages[m.top - 1 - (j - m.gone)];
}

// Items first, first + step, ...: the pushed pages, the taken ones, the rows.  What is read here (lower stack entries,
// table entries of pages held) is written by nobody: pushes go above the old top, taken pages into entries beyond the old
// lengths of other sequences.
__device__ void move_pages(const MapArgs &a, const MapSums &m, int first, int step) {
  if (m.ok) {
    for (int i = first; i < m.gone; i += step) a.free_pages[m.top + i] = pushed_page(a, m, i);
    for (int j = first; j < m.taken; j += step) {
      const int e = entry_of(m.taken_start, m.n, j);
      a.table[(long long)m.seq[e] * a.seq_pages + pages_of(m.old_len[e], a.shift) + (j - m.taken_start[e])] = taken_page(a, m, j);
    }
  }
  for (int r = first; r < a.max_rows; r += step) {
    int slot = -1, pos = -1, seq = -1;
    if (m.ok && r < m.rows) {
      const int e = entry_of(m.row_start, m.n, r);
      seq = m.seq[e];
      pos = m.old_len[e] + (r - m.row_start[e]);
      const int p = pos >> a.shift, had = pages_of(m.old_len[e], a.shift);
      const int page = p < had ? a.table[(long long)seq * a.seq_pages + p] : taken_page(a, m, m.taken_start[e] + (p - had));
      // (a table or a stack that somebody else filled may hold anything: such a page has no slots)
      if ((unsigned)page < (unsigned)a.n_pages) slot = (page << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
    a.row_seqs[r] = seq;
  }
}

// Sum over the threads before this one; *total: over all.  sums: kWaves entries of LDS.
__device__ __forceinline__ long long scan_threads(long long x, long long *sums, long long *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long inclusive = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long y = __shfl_up(inclusive, d);
    if (lane >= d) inclusive += y;
  }
  __syncthreads();  // sums of the scan before
  if (lane == 63) sums[wave] = inclusive;
  __syncthreads();
  long long before = 0, all = 0;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  *total = all;
  return before + inclusive - x;
}

// One workgroup: checks the entries, makes their sums, writes the new lengths.  MOVE: and does all the rest.
template <bool MOVE>
__global__ __launch_bounds__(kThreads) void page_map_kernel(MapArgs a) {
  __shared__ MapSums m;
  __shared__ long long sums[kWaves];
  __shared__ unsigned named[kMaxPagedSeqs / 32];
  __shared__ int bad;
  const int t = threadIdx.x, each = (a.n + kThreads - 1) / kThreads;
  if (t < kMaxPagedSeqs / 32) named[t] = 0;
  if (t == 0) bad = 0;
  __syncthreads();
  const int top = *a.n_free;
  const long long most = (long long)a.seq_pages << a.shift;
  int id[kEach], old_len[kEach], new_len[kEach];
  long long rows = 0, gone = 0, taken = 0;
  bool wrong = top < 0 || top > a.n_pages, full = false;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int e = t * each + u;
    id[u] = -1;
    if (u >= each || e >= a.n) continue;
    const int s = a.inlined ? a.id[e] : a.ids ? a.ids[e] : e;
    const int d = a.inlined ? a.change[e] : a.delta ? a.delta[e] : 1;
    if ((unsigned)s >= (unsigned)a.n_seqs) {
      wrong = true;
      continue;
    }
    if (atomicOr(&named[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) wrong = true;
    const int len = a.lens[s];
    const long long now = (long long)len + d;
    if (len < 0 || len > most || now < 0) {
      wrong = true;
      continue;
    }
    if (now > most) {
      full = true;
      continue;
    }
    id[u] = s;
    old_len[u] = len;
    new_len[u] = (int)now;
    const int pages = pages_of((int)now, a.shift) - pages_of(len, a.shift);
    rows += d > 0 ? d : 0;
    taken += pages > 0 ? pages : 0;
    gone += pages < 0 ? -pages : 0;
  }
  if (wrong) atomicOr(&bad, 1);
  if (full) atomicOr(&bad, 2);
  long long all_rows, all_gone, all_taken;
  long long row_start = scan_threads(rows, sums, &all_rows);
  long long gone_start = scan_threads(gone, sums, &all_gone);
  long long taken_start = scan_threads(taken, sums, &all_taken);
  const bool room = all_taken <= top + all_gone && top + all_gone - all_taken <= a.n_pages && top + all_gone <= a.n_pages &&
                    all_rows <= a.max_rows;
  const bool ok = !bad && room;  // (the same in every thread: `bad` was last written before a barrier of the scans)
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int e = t * each + u;
    if (u >= each || e >= a.n || !ok) continue;
    const int pages = pages_of(new_len[u], a.shift) - pages_of(old_len[u], a.shift);
    m.old_len[e] = old_len[u];
    m.seq[e] = id[u];
    m.row_start[e] = (int)row_start;
    m.taken_start[e] = (int)taken_start;
    gone_start += pages < 0 ? -pages : 0;
    m.gone_behind[e] = (int)(all_gone - gone_start);
    row_start += new_len[u] > old_len[u] ? new_len[u] - old_len[u] : 0;
    taken_start += pages > 0 ? pages : 0;
    a.lens[id[u]] = new_len[u];
  }
  if (t == 0) {
    m.ok = ok;
    m.n = a.n;
    m.rows = (int)all_rows;
    m.gone = (int)all_gone;
    m.taken = (int)all_taken;
    m.top = top;
    if (ok)
      *a.n_free = (int)(top + all_gone - all_taken);
    else
      *(volatile int *)a.error = bad & 1 ? kMapBadEntry : kMapNoRoom;
  }
  __syncthreads();
  if (MOVE) {
    move_pages(a, m, t, kThreads);
  } else {
    MapSums *out = (MapSums *)a.scratch;
    if (t == 0) {
      out->ok = m.ok;
      out->n = m.n;
      out->rows = m.rows;
      out->gone = m.gone;
      out->taken = m.taken;
      out->top = m.top;
    }
    if (ok)
      for (int e = t; e < a.n; e += kThreads) {
        out->old_len[e] = m.old_len[e];
        out->seq[e] = m.seq[e];
        out->row_start[e] = m.row_start[e];
        out->taken_start[e] = m.taken_start[e];
        out->gone_behind[e] = m.gone_behind[e];
      }
  }
}

__global__ __launch_bounds__(256) void page_move_kernel(MapArgs a) {
  move_pages(a, *(const MapSums *)a.scratch, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

__global__ __launch_bounds__(256) void page_reset_kernel(int *lens, int n_seqs, int *free_pages, int *n_free, int n_pages) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n_seqs) lens[i] = 0;
  if (i < n_pages) free_pages[i] = n_pages - 1 - i;
  if (i == 0) *n_free = n_pages;
}

}  // namespace

size_t map_scratch_ints() { return sizeof(MapSums) / sizeof(int); }

hipError_t launch_page_map(const MapArgs &a, hipStream_t stream) {
  if (a.n < 1 || a.n > kMaxPagedSeqs || a.n_seqs > kMaxPagedSeqs || (a.inlined && a.n > kMaxSeqs) || a.max_rows < 0 ||
      (a.max_rows && (!a.slots || !a.positions || !a.row_seqs)))
    return hipErrorInvalidValue;
  // a workgroup by itself moves what a decode step moves; many rows, or pages by the ten thousand, are shared out
  if (a.max_rows <= 8192 && a.n_pages <= 16384) {
    hipLaunchKernelGGL(page_map_kernel<true>, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(page_map_kernel<false>, dim3(1), dim3(kThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int items = a.max_rows > a.n_pages ? a.max_rows : a.n_pages;
  const int blocks = (items + 255) / 256;
  hipLaunchKernelGGL(page_move_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_page_reset(int *lens, int n_seqs, int *free_pages, int *n_free, int n_pages, hipStream_t stream) {
  const int items = n_seqs > n_pages ? n_seqs : n_pages;
  hipLaunchKernelGGL(page_reset_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, lens, n_seqs, free_pages,
                     n_free, n_pages);
  return hipGetLastError();
}

}  // namespace shainet
