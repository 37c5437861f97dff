// Tables of pages and maps of slots, made on the device from the sequences' lengths.
//
// Sequence s of length L holds pages(L) = ceil(L / P) pages, P rows each; table[s][i] is the page of its rows
// i P .. i P + P - 1.  Pages that nobody holds lie in free_pages[0 .. n_free - 1], a stack.  A map changes the length of each
// of its entries by delta: entries that shrink push their last pages, entries that grow take pages from the top, and
// every row gained gets its slot, page * P + row in the page.  With G pages pushed and T taken in all, the pushed ones in
// the order (last entry first, last page first) and the taken ones in the order (first entry first, first page first), the
// j-th page taken is the stack's entry n_free + G - 1 - j: a pushed one for j < G.  So a map followed by its inverse leaves
// the stack as it was, and where a page comes from follows from prefix sums: the order in which threads run decides nothing.
//
// Bound by latency: a launch, the entries, their lengths, a table entry or a free page, one after the other.  A step of 16
// sequences takes 3.3 to 4.0 us on the device (8.7 as one workgroup of 1024 threads that scanned 64-bit sums by shuffles), 582054 rows
// of 300 prompts 9.3 us (7 MB of lists; as two launches, one for the sums and one for the rows, 15), of which 5.6 without any rows.
//
// All or nothing: an entry out of range or named twice, a length below 0 or beyond the table's width, too few pages or
// too little room for the rows leave everything as it was, with every slot -1 and the reason in *error.  Launches that change something
// are counted: rows are placed layer by layer, and a layer behind the first asks by the count whether they are still its sequences'.
#include "paged.hpp"
#include "lane_sums.hpp"

#include <stdint.h>

namespace shainet {

namespace {

// What the entries look like once their sums are known, in LDS.
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

// Items first, first + step, ... of the rows, the pages pushed behind them and the pages taken behind those, so that a thread
// has one of the three where there are threads enough (1000 sequences, 127644 rows gained and others lost, and the inverse 16.5 us
// a pair of calls | 20.4 with the three one after the other).  What is read here (lower stack entries, table entries of pages
// held) is written by nobody: pushes go above the old top, taken pages into entries beyond the old lengths of other sequences.
template <int EACH>
__device__ void move_pages(const MapArgs &a, const MapSums &m, int first, int step) {
  // Of more rows than threads each takes four neighbours, of which one is searched for and most are of one page: 300 prompts of 582054 rows
  // and their inverse 15.1 us a pair of calls | 16.4.
  const bool fours = EACH > 1 && a.max_rows > step && (((uintptr_t)a.slots | (uintptr_t)a.positions | (uintptr_t)a.row_seqs) & 15) == 0;
  if (m.ok) {
    const unsigned row_items = fours ? (a.max_rows + 3u) / 4 : a.max_rows;
    auto behind = [&](unsigned items) { return first - (int)(items % (unsigned)step) + (first < (int)(items % (unsigned)step) ? step : 0); };
    for (int i = behind(row_items); i < m.gone; i += step) a.free_pages[m.top + i] = pushed_page(a, m, i);
    for (int j = behind(row_items + m.gone); j < m.taken; j += step) {
      const int e = entry_of(m.taken_start, m.n, j);
      a.table[(long long)m.seq[e] * a.seq_pages + pages_of(m.old_len[e], a.shift) + (j - m.taken_start[e])] = taken_page(a, m, j);
    }
  }
  // (a table or a stack that somebody else filled may hold anything: such a page has no slots)
  auto slot_in = [&](int page, int pos) { return (unsigned)page < (unsigned)a.n_pages ? (page << a.shift) + (pos & ((1 << a.shift) - 1)) : -1; };
  auto page_at = [&](int e, int p) {
    const int had = pages_of(m.old_len[e], a.shift);
    return p < had ? a.table[(long long)m.seq[e] * a.seq_pages + p] : taken_page(a, m, m.taken_start[e] + (p - had));
  };
  if (fours) {
    for (long long r = 4LL * first; r < a.max_rows; r += 4LL * step) {
      int slot[4], pos[4], seq[4], e = -1, of = -1, page = -1;  // (page `of` of entry e)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        slot[u] = pos[u] = seq[u] = -1;
        if (!m.ok || r + u >= m.rows) continue;
        const int row = (int)r + u;
        if (e < 0) e = entry_of(m.row_start, m.n, row);
        for (; e + 1 < m.n && m.row_start[e + 1] <= row; ++e) of = -1;
        seq[u] = m.seq[e];
        pos[u] = m.old_len[e] + (row - m.row_start[e]);
        if (pos[u] >> a.shift != of) {
          of = pos[u] >> a.shift;
          page = page_at(e, of);
        }
        slot[u] = slot_in(page, pos[u]);
      }
      if (r + 4 <= a.max_rows) {
        *(int4 *)(a.slots + r) = int4{slot[0], slot[1], slot[2], slot[3]};
        *(int4 *)(a.positions + r) = int4{pos[0], pos[1], pos[2], pos[3]};
        *(int4 *)(a.row_seqs + r) = int4{seq[0], seq[1], seq[2], seq[3]};
      } else {
        for (int u = 0; u < 4 && r + u < a.max_rows; ++u) {
          a.slots[r + u] = slot[u];
          a.positions[r + u] = pos[u];
          a.row_seqs[r + u] = seq[u];
        }
      }
    }
    return;
  }
  for (unsigned at = first; at < (unsigned)a.max_rows; at += step) {
    const int r = (int)at;
    int slot = -1, pos = -1, seq = -1;
    if (m.ok && r < m.rows) {
      const int e = entry_of(m.row_start, m.n, r);
      seq = m.seq[e];
      pos = m.old_len[e] + (r - m.row_start[e]);
      slot = slot_in(page_at(e, pos >> a.shift), pos);
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
    a.row_seqs[r] = seq;
  }
}

// Every workgroup checks the entries and makes their sums for itself (nothing that they are made of is written before all have
// read it), moves its share of the pages and writes its share of the rows; the one that is done last writes the new lengths.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void page_map_kernel(MapArgs a) {
  constexpr int WAVES = THREADS / 64, EACH = THREADS == 1024 ? kMaxPagedSeqs / THREADS : 1;
  __shared__ MapSums m;
  __shared__ int sums[3][WAVES];
  __shared__ float many[WAVES];
  __shared__ unsigned named[kMaxPagedSeqs / 32];
  __shared__ int bad, last;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, each = EACH == 1 ? 1 : (a.n + THREADS - 1) / THREADS;
  const int2 words = *(const int2 *)a.n_free;
  const int top = words.x;
  int epoch = words.y;
  int *rows_epoch = a.rows_epoch;
  const long long most = (long long)a.seq_pages << a.shift;
  int id[EACH], change[EACH], old_len[EACH], new_len[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int e = t * each + u;
    id[u] = -1;
    change[u] = 0;
    if (u >= each || e >= a.n) continue;
    id[u] = a.inlined ? a.id[e] : a.ids ? a.ids[e] : e;
    change[u] = a.inlined ? a.change[e] : a.delta ? a.delta[e] : 1;
  }
  for (int i = t; i < kMaxPagedSeqs / 32; i += THREADS) named[i] = 0;
  if (t == 0) bad = 0;
  __syncthreads();
  int rows = 0, gone = 0, taken = 0;
  float rows_about = 0.0f;
  bool wrong = top < 0 || top > a.n_pages, full = false;
  asm volatile("" : "+s"(epoch), "+s"(rows_epoch));  // (not fetched at the end, behind everything)
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int s = id[u], d = change[u];
    if (u >= each || t * each + u >= a.n) continue;
    id[u] = -1;
    if ((unsigned)s >= (unsigned)a.n_seqs) {
      wrong = true;
      continue;
    }
    if (atomicOr(&named[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) wrong = true;
    const int len = a.lens[s];
    const long long now = (long long)len + d;
    if (len < 0 || len > most || now < 0 || (a.inlined && len != a.was[t * each + u])) {
      wrong = true;
      continue;
    }
    if (now > most || d > a.max_rows || (d > 0 && now > a.reach)) {
      full = true;
      continue;
    }
    id[u] = s;
    old_len[u] = len;
    new_len[u] = (int)now;
    const int pages = pages_of((int)now, a.shift) - pages_of(len, a.shift);
    rows += d > 0 ? d : 0;
    rows_about += d > 0 ? (float)d : 0.0f;
    taken += pages > 0 ? pages : 0;
    gone += pages < 0 ? -pages : 0;
  }
  if (wrong) atomicOr(&bad, 1);
  if (full) atomicOr(&bad, 2);
  const int upto[3] = {sum_lanes(rows), sum_lanes(gone), sum_lanes(taken)};
#pragma unroll
  for (int d = 32; d; d >>= 1) rows_about += __shfl_xor(rows_about, d);
  if (lane == 63) {
#pragma unroll
    for (int i = 0; i < 3; ++i) sums[i][wave] = upto[i];
    many[wave] = rows_about;
  }
  __syncthreads();
  int start[3], all[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    start[i] = upto[i] - (i == 0 ? rows : i == 1 ? gone : taken);
    all[i] = 0;
  }
  rows_about = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int x = sums[i][w];
      start[i] += w < wave ? x : 0;
      all[i] += x;
    }
    rows_about += many[w];
  }
  // (a sum of rows that is too long for 32 bits is found by the one in floats: both are good to a millionth.  Pages taken and given back
  // are no more than the table has entries, which 32 bits count.)
  const bool room = rows_about < 2.1e9f && all[0] <= a.max_rows && (long long)top + all[1] <= a.n_pages && all[2] <= top + all[1];
  const bool ok = !bad && room;
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int e = t * each + u;
    if (u >= each || e >= a.n || !ok) continue;
    const int pages = pages_of(new_len[u], a.shift) - pages_of(old_len[u], a.shift);
    m.old_len[e] = old_len[u];
    m.seq[e] = id[u];
    m.row_start[e] = start[0];
    m.taken_start[e] = start[2];
    start[0] += new_len[u] > old_len[u] ? new_len[u] - old_len[u] : 0;
    start[1] += pages < 0 ? -pages : 0;
    start[2] += pages > 0 ? pages : 0;
    m.gone_behind[e] = all[1] - start[1];
  }
  if (t == 0) {
    m.ok = ok;
    m.n = a.n;
    m.rows = all[0];
    m.gone = all[1];
    m.taken = all[2];
    m.top = top;
  }
  __syncthreads();
  move_pages<EACH>(a, m, blockIdx.x * THREADS + t, gridDim.x * THREADS);
  if (gridDim.x > 1) {
    // (the barrier: this workgroup's reads of the lengths and of the number of free pages are done)
    if (t == 0) last = __hip_atomic_fetch_add(a.scratch, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (t == 0) __hip_atomic_store(a.scratch, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
#pragma unroll
  for (int u = 0; u < EACH; ++u)
    if (u < each && t * each + u < a.n && ok) a.lens[id[u]] = new_len[u];
  if (t == 0) {
    if (ok) {
      *(int2 *)a.n_free = int2{top + all[1] - all[2], epoch + 1};
    } else {
      *(volatile int *)a.error = bad & 1 ? kMapBadEntry : kMapNoRoom;
    }
    if (rows_epoch) *rows_epoch = ok ? epoch + 1 : epoch;
  }
}

__global__ __launch_bounds__(1024) void page_report_kernel(MapArgs a, int *host, int words) {
  const long long most = (long long)a.seq_pages << a.shift;
  const int in_page = (1 << a.shift) - 1;
  int gone = 0;
  for (long long i = blockIdx.x * 1024 + threadIdx.x; i < a.max_rows; i += gridDim.x * 1024) {
    const int r = (int)i;
    const int seq = a.row_seqs[r], pos = a.positions[r], slot = a.slots[r];
    if ((unsigned)seq >= (unsigned)a.n_seqs || pos < 0 || pos >= most) {
      gone = 1;
      continue;
    }
    // (a sequence's rows follow each other, and the last is its last)
    const bool ends = r + 1 == a.max_rows || a.row_seqs[r + 1] != seq;
    if (slot >> a.shift != a.table[(long long)seq * a.seq_pages + (pos >> a.shift)] || (slot & in_page) != (pos & in_page) ||
        (ends ? a.lens[seq] : a.positions[r + 1]) != pos + 1)
      gone = 1;
  }
  gone = __syncthreads_or(gone);
  if (threadIdx.x == 0 && gone) atomicAdd(&a.n_free[1], 1);
  if (!host) return;
  __syncthreads();
  for (int i = threadIdx.x; i < a.n_seqs + words; i += 1024) host[i] = i < a.n_seqs ? a.lens[i] : a.n_free[i - a.n_seqs];
}

__global__ __launch_bounds__(256) void page_reset_kernel(int *lens, int n_seqs, int *free_pages, int *n_free, int n_pages) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n_seqs) lens[i] = 0;
  if (i < n_pages) free_pages[i] = n_pages - 1 - i;
  if (i == 0) {
    *n_free = n_pages;
    n_free[1] += 1;
  }
}

}  // namespace

hipError_t launch_page_map(const MapArgs &a, hipStream_t stream) {
  if (a.n < 1 || a.n > kMaxPagedSeqs || a.n_seqs > kMaxPagedSeqs || (a.inlined && a.n > kMaxSeqs) || a.max_rows < 0 ||
      (a.max_rows && (!a.slots || !a.positions || !a.row_seqs)))
    return hipErrorInvalidValue;
  // A decode step's rows are mapped by one workgroup of four wavefronts, whose barriers take less: 16 sequences and their inverse 8.9 us a
  // pair of calls where the pool has 60000 pages | 10.9 us by 1024 threads on each of up to 256 compute units (15.4 where it has a
  // million).  Pages by the ten thousand, which an entry may give back, want those: 8192 in one call 10.6 us | 3.0, 32768 37 | 4.
  // (The many are as fast as one of them where two would do: 1500 rows of 300 sequences 5.3 us | 5.6, 8000 5.3 | 10.9.)
  const long long of_entries = a.delta || a.inlined ? (long long)a.n * a.seq_pages : a.n;  // pages that can move, at most
  const int pages = (int)(of_entries < a.n_pages ? of_entries : a.n_pages);
  if (a.n <= 256 && a.max_rows <= 1024 && pages <= 1 << 16) {
    hipLaunchKernelGGL(page_map_kernel<256>, dim3(1), dim3(256), 0, stream, a);
  } else {
    const long long blocks = ((long long)a.max_rows + pages + 1023) / 1024;
    hipLaunchKernelGGL(page_map_kernel<1024>, dim3((unsigned)(blocks < 1 ? 1 : blocks < 256 ? blocks : 256)), dim3(1024), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_page_report(const MapArgs &a, int *host, int words, hipStream_t stream) {
  // Rows by the ten thousand, of prompts, are looked at by a launch of their own: 60000 and the report 16 us | 43 by one workgroup.
  MapArgs rest = a;
  if (a.max_rows > 8192) {
    const int blocks = (a.max_rows - 1) / 1024 + 1;
    hipLaunchKernelGGL(page_report_kernel, dim3((unsigned)(blocks < 256 ? blocks : 256)), dim3(1024), 0, stream, a, (int *)nullptr, 0);
    if (const hipError_t e = hipGetLastError()) return e;
    rest.max_rows = 0;
  }
  hipLaunchKernelGGL(page_report_kernel, dim3(1), dim3(1024), 0, stream, rest, host, words);
  return hipGetLastError();
}

hipError_t launch_page_reset(int *lens, int n_seqs, int *free_pages, int *n_free, int n_pages, hipStream_t stream) {
  const int items = n_seqs > n_pages ? n_seqs : n_pages;
  hipLaunchKernelGGL(page_reset_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, lens, n_seqs, free_pages,
                     n_free, n_pages);
  return hipGetLastError();
}

}  // namespace shainet
