// Keys and values in pages: which page holds which rows (paged_map.hip), new rows into their slots (paged_append.hip),
// attention of one new row per sequence over its pages (paged_attn.hip).  paged_cache.hip keeps the arrays and the C ABI.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "paged_tile.hpp"

namespace shainet {

constexpr int kMaxPagedSeqs = 4096;  // entries of a map, rows of an attention launch: their prefix sums lie in LDS

// One layer's pages, [n_pages][KV][1 << shift][hd] for K and for V, and the table of all sequences.
struct PagePool {
  void *k, *v;
  int dtype, KV, hd;
  int n_pages, shift;     // rows per page: 1 << shift
  const int *table;       // [n_seqs][seq_pages]
  int n_seqs, seq_pages;
};

// A change of lengths: entry i is sequence ids[i], whose length changes by delta[i].
struct MapArgs {
  int n;
  const int *ids, *delta;      // device; null: see `inlined`, else sequence i and one row
  int inlined;                 // the lists below instead, n <= kMaxSeqs; a sequence whose length is not `was` is a bad entry
  int id[kMaxSeqs], was[kMaxSeqs], change[kMaxSeqs];
  int *table, *lens, *free_pages;
  int *n_free;                 // and, behind it, the count of launches that changed something; on 8 bytes
  int n_seqs, seq_pages, n_pages, shift;
  int reach;                   // entries that grow become no longer than this
  int *slots, *positions, *row_seqs;  // of the new rows in the entries' order; -1 from the last one to max_rows
  int max_rows;
  int *rows_epoch;             // nullable: set to the count that the lists are of
  int *scratch;                // a word, zero, which a launch leaves so
  int *error;                  // device-writable: set to kMapNoRoom or kMapBadEntry where nothing was changed
};
constexpr int kMapNoRoom = 3, kMapBadEntry = 4, kRowsGone = 5, kRowsFar = 6, kKeysOutside = 7, kRowsOutside = 8;
hipError_t launch_page_map(const MapArgs &a, hipStream_t stream);
// every length 0, every page free, page 0 to be taken first
hipError_t launch_page_reset(int *lens, int n_seqs, int *free_pages, int *n_free, int n_pages, hipStream_t stream);
// The lengths and, behind them, the first `words` words at a.n_free to `host`, which the device can write to.  Before that counts a change
// where a.max_rows rows of a map (a.slots, positions, row_seqs; may be none) are not the last ones of their sequences any more, in the slots
// that the table says.
hipError_t launch_page_report(const MapArgs &a, int *host, int words, hipStream_t stream);

// Lists that a map for an earlier layer wrote: where lengths, tables or pages were changed since, the rows are nobody's or
// another's.  Then none is placed, their row_seqs become -1 (so that attention leaves them alone) and *error kRowsGone; one at a position
// that this layer's cos/sin table does not have goes the same way, with kRowsFar, and one whose page is none of the pool with kRowsOutside.
struct MappedRows {
  const int *epoch, *rows_epoch;  // (the same word: never)
  int *row_seqs, *error;          // row_seqs null: lists of the caller's
};

// bias -> QK-norm -> RoPE of `rows` rows, whose K and V parts go to slots[row] (page << shift | row in the page);
// a.kc, a.vc are not used.  A row whose slot or position is out of range is left alone.
hipError_t launch_paged_append(const PrepArgs &a, const PagePool &p, int H, const int *slots, const int *positions,
                               int rope_positions, int rows, const MappedRows &mapped, hipStream_t stream);

// Attention of row r of q ([rows][H * hd], rows q_stride floats apart) over the first positions[r] + 1 rows of sequence
// row_seqs[r].  A row with row_seqs < 0 is left alone; one with positions < 0 gets zeros.
struct PagedAttendArgs {
  const float *q;
  float *out;
  long long q_stride, out_stride;
  const int *row_seqs, *positions;
  int rows, H, g;              // g: query heads per kv head
  float scale;
  void *workspace;             // paged_attend_workspace() bytes, zero when allocated; a launch leaves its counts zero
};
size_t paged_attend_workspace(int hd);
hipError_t launch_paged_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream);

// Rows pos0 .. pos0 + n - 1 of a sequence, as floats, into [KV][cap][hd] arrays.  A row in no page of the pool is zeros, and *error (if any)
// kKeysOutside.
hipError_t launch_page_gather(const PagePool &p, int seq, int pos0, int n, int cap, float *k, float *v, int *error, hipStream_t stream);

}  // namespace shainet
