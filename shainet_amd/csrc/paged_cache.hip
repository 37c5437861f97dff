// shainet_paged_cache: keys and values in pages, the tables that say which sequence holds which page, and the calls of an
// AttnContext over them (declared in include/shainet_hip_attn.h).
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <new>
#include <vector>

#include "../../include/shainet_hip_attn.h"
#include "attn_context.hpp"
#include "attn_kernels.hpp"
#include "llama_internal.hpp"
#include "paged.hpp"
#include "rope_table.hpp"

using namespace shainet;

void shainet_hip_set_error(int code, const char *msg);

struct shainet_paged_cache {
  shainet_attn_ctx *ctx;
  int device;
  int layers, KV, hd, dtype, n_pages, shift, n_seqs, seq_pages;
  size_t layer_bytes;  // of K, and of V
  char *k = nullptr, *v = nullptr;
  int *table = nullptr, *lens = nullptr, *free_pages = nullptr;
  // kWords on the device: the number of free pages; the count of maps that changed something; the counts that the lists of
  // step and forward calls are of
  int *n_free = nullptr;
  int *pin = nullptr;      // [n_seqs + kWords] pinned, which launch_page_report writes
  int *scratch = nullptr;  // a word for maps
  void *workspace = nullptr;
  // steps: allocated with the cache, so that a step allocates nothing
  int *step_slots = nullptr, *step_positions = nullptr, *step_seqs = nullptr;  // [n_seqs]
  DevBuf step_q;           // [n_seqs, H hd] of the owner's context; other contexts have at most as many heads
  int step_rows = 0;       // of the last step that mapped rows; 0: none yet
  // forward calls: grow on demand
  DevBuf rows;             // three lists of ints
  DevBuf gathered;
  std::vector<int> len;    // per sequence, while the host knows them
  int free_count;
  int reach;               // rows that a sequence may come to have, as far as the host knows: the context's cos/sin tables go as far
  bool lengths_on_device = false;
  std::vector<int> last_ids, last_new;  // of the last forward call for layer 0
};

namespace {

enum { kFree, kEpoch, kStepEpoch, kForwardEpoch, kWords };

int fail(int code, const char *fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  shainet_hip_set_error(code, text);
  return code;
}

int hip_fail(hipError_t e, const char *what) {
  (void)hipGetLastError();
  return fail(e == hipErrorOutOfMemory ? SHAINET_HIP_ERR_ALLOC : SHAINET_HIP_ERR_RUNTIME, "%s: %s", what, hipGetErrorString(e));
}

#define HIP_TRY(expr)                                 \
  do {                                                \
    hipError_t e_ = (expr);                           \
    if (e_ != hipSuccess) return hip_fail(e_, #expr); \
  } while (0)

int pages_of(const shainet_paged_cache *pc, long long rows) { return (int)((rows + (1 << pc->shift) - 1) >> pc->shift); }
long long reach_of(const shainet_paged_cache *pc) { return (long long)pc->seq_pages << pc->shift; }

PagePool pool_of(const shainet_paged_cache *pc, int layer) {
  PagePool p;
  p.k = pc->k + (size_t)layer * pc->layer_bytes;
  p.v = pc->v + (size_t)layer * pc->layer_bytes;
  p.dtype = pc->dtype;
  p.KV = pc->KV;
  p.hd = pc->hd;
  p.n_pages = pc->n_pages;
  p.shift = pc->shift;
  p.table = pc->table;
  p.n_seqs = pc->n_seqs;
  p.seq_pages = pc->seq_pages;
  return p;
}

// What every call that launches something asks first.
int check_device(const shainet_paged_cache *pc) {
  int device = -1;
  HIP_TRY(hipGetDevice(&device));
  if (device != pc->device)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "the cache is on device %d, the current device is %d", pc->device, device);
  return SHAINET_HIP_OK;
}

int check_pair(const shainet_attn_ctx *c, const shainet_paged_cache *pc, int layer) {
  if (!c || !pc || c->KV != pc->KV || c->hd != pc->hd || c->v_hd != pc->hd || c->window || c->rope_fp64)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "context and cache do not belong together");
  if (c->H > pc->ctx->H) return fail(SHAINET_HIP_ERR_ARGUMENT, "the context has more query heads than the one the cache was made with");
  if (c->stream != pc->ctx->stream)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "contexts that share a cache work on one stream: shainet_attn_set_stream");
  if (layer < 0 || layer >= pc->layers) return fail(SHAINET_HIP_ERR_ARGUMENT, "layer must be in 0..%d", pc->layers - 1);
  return check_device(pc);
}

// Calls whose work depends on what the host knows now, or that wait: good for one execution only.
int refuse_recording(const shainet_attn_ctx *c, const char *what) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (c->stream) HIP_TRY(hipStreamIsCapturing(c->stream, &status));
  if (status == hipStreamCaptureStatusNone) return SHAINET_HIP_OK;
  return fail(SHAINET_HIP_ERR_ARGUMENT, "%s cannot be recorded", what);
}

int refuse_unknown_lengths(const shainet_paged_cache *pc, const char *what) {
  if (!pc->lengths_on_device) return SHAINET_HIP_OK;
  return fail(SHAINET_HIP_ERR_ARGUMENT, "%s: the lengths were changed on the device; call shainet_paged_cache_lengths_from_device first", what);
}

// The rows that layer 0 mapped last are no longer those that other layers may place: their pages can be others' by now.
void forget_rows(shainet_paged_cache *pc) {
  pc->last_ids.clear();
  pc->step_rows = 0;
}

MapArgs map_of(const shainet_paged_cache *pc) {
  MapArgs a;
  memset(&a, 0, sizeof a);
  a.table = pc->table;
  a.lens = pc->lens;
  a.free_pages = pc->free_pages;
  a.n_free = pc->n_free;
  a.n_seqs = pc->n_seqs;
  a.seq_pages = pc->seq_pages;
  a.n_pages = pc->n_pages;
  a.shift = pc->shift;
  a.reach = (int)reach_of(pc);
  a.scratch = pc->scratch;
  a.error = pc->ctx->error;
  return a;
}

// Rows that c places have an angle each: maps of rows for its calls refuse those behind its table.
int reach_with(const shainet_attn_ctx *c, const shainet_paged_cache *pc) {
  return (int)(c->rope_positions < reach_of(pc) ? c->rope_positions : reach_of(pc));
}

// The lengths of up to kMaxSeqs sequences, `was` as far as the host knows, change by `change`; rows (nullable): three lists of max_rows.
int map_listed(shainet_paged_cache *pc, const int *ids, const int *was, const int *change, int n, int reach, int *rows, int max_rows) {
  MapArgs a = map_of(pc);
  a.reach = reach;
  a.n = n;
  a.inlined = 1;
  for (int i = 0; i < n; ++i) {
    a.id[i] = ids[i];
    a.was[i] = was[i];
    a.change[i] = change[i];
  }
  a.max_rows = max_rows;
  if (rows) {
    a.slots = rows;
    a.positions = rows + max_rows;
    a.row_seqs = rows + 2 * (size_t)max_rows;
    a.rows_epoch = pc->n_free + kForwardEpoch;
  }
  const hipError_t e = launch_page_map(a, pc->ctx->stream);
  return e == hipSuccess ? SHAINET_HIP_OK : hip_fail(e, "map launch");
}

// Sequences that hold pages of the pool only, each its own, are no longer than the pool; of those that a caller made longer (entries of
// no page, pages shared) the host knows once it is told their lengths.
void extend_reach(shainet_paged_cache *pc, long long rows) {
  if (rows <= pc->reach) return;
  const long long most = most_table_positions(pc->hd * 4), more = 2 * rows < most ? 2 * rows : rows < most ? most : rows;
  pc->reach = (int)(more < reach_of(pc) ? more : reach_of(pc));
}

// The cos/sin table goes as far as rows can: at which positions they are is known to the device only.
int reach_table(shainet_attn_ctx *c, long long reach) {
  if (c->rope_positions >= reach) return SHAINET_HIP_OK;
  if (refuse_recording(c, ""))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "the context's cos/sin table must be extended to %lld positions, which cannot be recorded: create the context "
                "with that many, or place rows once before recording", reach);
  if (reach > most_table_positions(c->hd * 4))
    return fail(SHAINET_HIP_ERR_ALLOC, "a cos/sin table of %lld positions would take more than 8 GiB: the cache's table is that wide", reach);
  return ensure_rope_table(c, (int)reach);
}

PrepArgs prep_of(const shainet_attn_ctx *c, const float *q, long long q_stride, const float *k, long long k_stride, const float *v,
                 long long v_stride, float *q_rot) {
  PrepArgs pa;
  memset(&pa, 0, sizeof pa);
  pa.q = q;
  pa.k = k;
  pa.v = v;
  pa.q_stride = q_stride;
  pa.k_stride = k_stride;
  pa.v_stride = v_stride;
  pa.b_q = c->d_bq;
  pa.b_k = c->d_bk;
  pa.b_v = c->d_bv;
  pa.q_norm = c->d_q_norm;
  pa.k_norm = c->d_k_norm;
  pa.eps = c->eps;
  pa.rope_tab = c->d_rope;
  pa.q_rot = q_rot;
  return pa;
}

// row_seqs: of rows that a map for layer 0 made, whose count is the word `of_map`; null: the caller's own lists
int append(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const PrepArgs &pa, const int *slots, const int *positions,
           int rows, int *row_seqs, int of_map) {
  const int *epoch = pc->n_free + kEpoch;
  const MappedRows mapped = {epoch, row_seqs && layer ? pc->n_free + of_map : epoch, row_seqs, pc->ctx->error};
  const hipError_t e = launch_paged_append(pa, pool_of(pc, layer), c->H, slots, positions, c->rope_positions, rows, mapped, c->stream);
  return e == hipSuccess ? SHAINET_HIP_OK : hip_fail(e, "append launch");
}

// Tiles of 16 keys are counted in 32 bits, and so are those of a workgroup's span of all pairs.
int refuse_many_keys(const shainet_attn_ctx *c, const shainet_paged_cache *pc, int rows) {
  if (rows * reach_of(pc) >= 1LL << 34 || rows * reach_of(pc) * c->KV * ((c->g + 15) / 16) >= 1LL << 42)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "%d rows of up to %lld keys in one call: their product must stay below 2^34, and times the kv heads below 2^42",
                rows, reach_of(pc));
  return SHAINET_HIP_OK;
}

int attend(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const int *row_seqs, const int *positions, int rows,
           const float *q, long long q_stride, float *out, long long out_stride) {
  if (int rc = refuse_many_keys(c, pc, rows)) return rc;
  PagedAttendArgs a;
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.row_seqs = row_seqs;
  a.positions = positions;
  a.rows = rows;
  a.H = c->H;
  a.g = c->g;
  a.scale = c->scale;
  a.workspace = pc->workspace;
  const hipError_t e = launch_paged_attend(a, pool_of(pc, layer), c->stream);
  return e == hipSuccess ? SHAINET_HIP_OK : hip_fail(e, "attention launch");
}

// Whether writing a row of b can change a row of a that somebody still reads: rows of `width` floats at a distance each.  Where the rows are the
// same ones, each is written by those that read it, behind that.
bool in_the_way(const float *a, long long a_stride, long long a_width, const float *b, long long b_stride, long long b_width, int rows) {
  const long long word = sizeof(float), step_a = a_stride * word, step_b = b_stride * word, bytes_a = a_width * word, bytes_b = b_width * word;
  const long long d = (long long)((uintptr_t)b - (uintptr_t)a);
  if ((rows - 1) * step_a + bytes_a <= d || (rows - 1) * step_b + bytes_b <= -d) return false;
  if (rows == 1 || (d == 0 && step_a == step_b)) return d != 0 || bytes_a != bytes_b;
  if (step_a == step_b) {
    const long long behind = ((d % step_a) + step_a) % step_a;
    return behind < bytes_a || step_a - behind < bytes_b;
  }
  for (long long i = 0, j = 0; i < rows; ++i) {  // (the first row of b that ends behind where row i of a begins, and those that begin before its end)
    while (j < rows && d + j * step_b + bytes_b <= i * step_a) ++j;
    for (long long k = j; k < rows && d + k * step_b < i * step_a + bytes_a; ++k)
      if (k != i || d + k * step_b != i * step_a || bytes_a != bytes_b) return true;
  }
  return false;
}

// New rows of a sequence up to this many read the pages themselves, one by one; for more the pages are gathered first, once for
// all of them.  32 heads of 128 on 8 kv heads, us from pages | gathered: 8 rows on 500 keys of float32 14.5 | 21, of bfloat16 10.6 | 20; on
// 16000 160 | 166 and 85 | 117; 12 rows on 16000 233 | 199 and 115 | 169.
constexpr int kRowsFromPages = 8;

}  // namespace

extern "C" {

int shainet_paged_cache_create(shainet_paged_cache **out, shainet_attn_ctx *ctx, int layers, int n_pages, int page_rows, int n_seqs,
                               int seq_pages, int dtype) {
  if (!out) return fail(SHAINET_HIP_ERR_ARGUMENT, "out is null");
  *out = nullptr;
  if (!ctx) return fail(SHAINET_HIP_ERR_ARGUMENT, "ctx is null");
  if (ctx->v_hd != ctx->hd || ctx->window || ctx->rope_fp64 || (ctx->hd & 7))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "a cache in pages needs grouped-query attention with rotation and a head_dim that is a multiple of 8 up to 256");
  if (page_rows < 8 || page_rows > 1024 || (page_rows & (page_rows - 1)))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "page_rows must be a power of two in 8..1024");
  if (dtype != SHAINET_HIP_PAGE_F32 && dtype != SHAINET_HIP_PAGE_BF16 && dtype != SHAINET_HIP_PAGE_F16)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "dtype must be one of SHAINET_HIP_PAGE_F32, _BF16 and _F16");
  if (n_seqs < 1 || n_seqs > SHAINET_HIP_MAX_PAGED_SEQS)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "n_seqs must be in 1..%d", SHAINET_HIP_MAX_PAGED_SEQS);
  if (layers < 1 || n_pages < 1 || seq_pages < 1 || (long long)n_pages * page_rows > 0x7fffffffLL ||
      (long long)seq_pages * page_rows > 0x3fffffffLL || (long long)n_seqs * seq_pages > 0x7fffffffLL)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "invalid cache geometry: slots and table entries are 32-bit numbers, positions 30-bit ones");
  if (int rc = refuse_recording(ctx, "shainet_paged_cache_create")) return rc;
  shainet_paged_cache *pc = new (std::nothrow) shainet_paged_cache();
  if (!pc) return fail(SHAINET_HIP_ERR_ALLOC, "out of host memory");
  pc->ctx = ctx;
  pc->layers = layers;
  pc->KV = ctx->KV;
  pc->hd = ctx->hd;
  pc->dtype = dtype;
  pc->n_pages = n_pages;
  pc->shift = __builtin_ctz((unsigned)page_rows);
  pc->n_seqs = n_seqs;
  pc->seq_pages = seq_pages;
  pc->free_count = n_pages;
  pc->reach = (seq_pages < n_pages ? seq_pages : n_pages) * page_rows;
  pc->layer_bytes = (size_t)n_pages * ctx->KV * page_rows * ctx->hd * page_element_bytes(dtype);
  int rc = SHAINET_HIP_OK;
  try {
    pc->len.assign(n_seqs, 0);
  } catch (const std::bad_alloc &) {
    rc = fail(SHAINET_HIP_ERR_ALLOC, "out of host memory");
  }
  const size_t pool = pc->layer_bytes * layers, table = (size_t)n_seqs * seq_pages, ws = paged_attend_workspace(ctx->hd);
  hipError_t e = rc ? hipErrorOutOfMemory : hipGetDevice(&pc->device);
  if (e == hipSuccess) e = hipMalloc((void **)&pc->k, pool);
  if (e == hipSuccess) e = hipMalloc((void **)&pc->v, pool);
  if (e == hipSuccess) e = hipMalloc((void **)&pc->table, table * sizeof(int));
  if (e == hipSuccess) e = hipMalloc((void **)&pc->lens, n_seqs * sizeof(int));
  if (e == hipSuccess) e = hipMalloc((void **)&pc->free_pages, (size_t)n_pages * sizeof(int));
  if (e == hipSuccess) e = hipMalloc((void **)&pc->n_free, kWords * sizeof(int));
  if (e == hipSuccess) e = hipHostMalloc((void **)&pc->pin, (n_seqs + kWords) * sizeof(int), hipHostMallocDefault);
  if (e == hipSuccess) e = hipMalloc((void **)&pc->scratch, sizeof(int));
  if (e == hipSuccess) e = hipMalloc(&pc->workspace, ws);
  if (e == hipSuccess) e = hipMalloc((void **)&pc->step_slots, n_seqs * sizeof(int));
  if (e == hipSuccess) e = hipMalloc((void **)&pc->step_positions, n_seqs * sizeof(int));
  if (e == hipSuccess) e = hipMalloc((void **)&pc->step_seqs, n_seqs * sizeof(int));
  // (rows never written hold zeros; on the stream that uses them, and waited for)
  if (e == hipSuccess) e = hipMemsetAsync(pc->k, 0, pool, ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(pc->v, 0, pool, ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(pc->table, 0xff, table * sizeof(int), ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(pc->workspace, 0, ws, ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(pc->scratch, 0, sizeof(int), ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(pc->n_free, 0, kWords * sizeof(int), ctx->stream);
  if (e == hipSuccess) e = launch_page_reset(pc->lens, n_seqs, pc->free_pages, pc->n_free, n_pages, ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess && !rc) rc = hip_fail(e, "allocation of a cache in pages");
  if (!rc) rc = pc->step_q.reserve((size_t)n_seqs * ctx->H * ctx->hd);
  if (rc) {
    shainet_paged_cache_destroy(pc);
    return rc;
  }
  *out = pc;
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_destroy(shainet_paged_cache *pc) {
  if (!pc) return SHAINET_HIP_OK;
  (void)hipStreamSynchronize(pc->ctx->stream);
  for (void *p : {(void *)pc->k, (void *)pc->v, (void *)pc->table, (void *)pc->lens, (void *)pc->free_pages, (void *)pc->n_free,
                  (void *)pc->scratch, pc->workspace, (void *)pc->step_slots, (void *)pc->step_positions, (void *)pc->step_seqs})
    if (p) (void)hipFree(p);
  if (pc->pin) (void)hipHostFree(pc->pin);
  for (DevBuf *b : {&pc->step_q, &pc->rows, &pc->gathered}) b->release();
  delete pc;
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_arrays(shainet_paged_cache *pc, int layer, void **k, void **v, int **table, int **lens, int **free_pages,
                               int **n_free) {
  if (!pc || layer < 0 || layer >= pc->layers) return fail(SHAINET_HIP_ERR_ARGUMENT, "invalid cache or layer");
  const PagePool p = pool_of(pc, layer);
  if (k) *k = p.k;
  if (v) *v = p.v;
  if (table) *table = pc->table;
  if (lens) *lens = pc->lens;
  if (free_pages) *free_pages = pc->free_pages;
  if (n_free) *n_free = pc->n_free;
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_map_rows(shainet_paged_cache *pc, const int *seq_ids, const int *delta, int n, int *slots, int *positions,
                                 int *row_seqs, int max_rows) {
  if (!pc || !delta) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (n < 1 || n > pc->n_seqs) return fail(SHAINET_HIP_ERR_ARGUMENT, "n must be in 1..%d", pc->n_seqs);
  if (max_rows < 0) return fail(SHAINET_HIP_ERR_ARGUMENT, "max_rows must not be negative");
  if (max_rows && (!slots || !positions || !row_seqs)) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (int rc = check_device(pc)) return rc;
  MapArgs a = map_of(pc);
  a.n = n;
  a.ids = seq_ids;
  a.delta = delta;
  a.slots = slots;
  a.positions = positions;
  a.row_seqs = row_seqs;
  a.max_rows = max_rows;
  const hipError_t e = launch_page_map(a, pc->ctx->stream);
  if (e != hipSuccess) return hip_fail(e, "map launch");
  pc->lengths_on_device = true;
  forget_rows(pc);
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_lengths_from_device(shainet_paged_cache *pc) {
  if (!pc) return fail(SHAINET_HIP_ERR_ARGUMENT, "cache is null");
  if (int rc = check_device(pc)) return rc;
  if (int rc = refuse_recording(pc->ctx, "shainet_paged_cache_lengths_from_device")) return rc;
  // Rows that other layers may still place: whether they are where they were, whoever wrote to lengths or table.  (Those of a step stay
  // the device's matter: a replay can have made new ones by the time of the next layer.)
  MapArgs a = map_of(pc);
  if (pc->layers > 1 && pc->step_rows) {
    a.max_rows = pc->step_rows;
    a.slots = pc->step_slots;
    a.positions = pc->step_positions;
    a.row_seqs = pc->step_seqs;
  } else if (pc->layers > 1 && !pc->last_ids.empty()) {
    for (int n : pc->last_new) a.max_rows += n;
    a.slots = (int *)pc->rows.p;
    a.positions = a.slots + a.max_rows;
    a.row_seqs = a.slots + 2 * (size_t)a.max_rows;
  }
  const int *words = pc->pin + pc->n_seqs;
  const hipError_t e = launch_page_report(a, pc->pin, kWords, pc->ctx->stream);
  if (e != hipSuccess) return hip_fail(e, "report launch");
  HIP_TRY(hipStreamSynchronize(pc->ctx->stream));
  if (words[kEpoch] != words[kForwardEpoch]) pc->last_ids.clear();
  int longest = 0;
  for (int s = 0; s < pc->n_seqs; ++s) {
    if (pc->pin[s] < 0 || pc->pin[s] > reach_of(pc))
      return fail(SHAINET_HIP_ERR_RUNTIME, "the device holds length %d for sequence %d", pc->pin[s], s);
    if (pc->pin[s] > longest) longest = pc->pin[s];
  }
  if (words[kFree] < 0 || words[kFree] > pc->n_pages)
    return fail(SHAINET_HIP_ERR_RUNTIME, "the device holds %d free pages of %d", words[kFree], pc->n_pages);
  memcpy(pc->len.data(), pc->pin, pc->n_seqs * sizeof(int));
  pc->free_count = words[kFree];
  if (longest > pc->reach || (longest == pc->reach && pc->free_count)) extend_reach(pc, (long long)longest + 1);
  pc->lengths_on_device = false;
  return check_error_word(pc->ctx->error);
}

int shainet_paged_cache_len(const shainet_paged_cache *pc, int seq) {
  if (!pc || seq < 0 || seq >= pc->n_seqs || refuse_unknown_lengths(pc, "shainet_paged_cache_len")) return -1;
  return pc->len[seq];
}

int shainet_paged_cache_free_pages(const shainet_paged_cache *pc) {
  if (!pc || refuse_unknown_lengths(pc, "shainet_paged_cache_free_pages")) return -1;
  return pc->free_count;
}

int shainet_paged_cache_truncate(shainet_paged_cache *pc, int seq, int len) {
  if (!pc || seq < 0 || seq >= pc->n_seqs) return fail(SHAINET_HIP_ERR_ARGUMENT, "invalid sequence");
  if (int rc = refuse_unknown_lengths(pc, "shainet_paged_cache_truncate")) return rc;
  if (len < 0 || len > pc->len[seq]) return fail(SHAINET_HIP_ERR_ARGUMENT, "truncate to %d outside 0..%d", len, pc->len[seq]);
  if (int rc = check_device(pc)) return rc;
  if (int rc = refuse_recording(pc->ctx, "shainet_paged_cache_truncate")) return rc;
  const int was = pc->len[seq], change = len - was;
  if (change == 0) return SHAINET_HIP_OK;
  if (int rc = map_listed(pc, &seq, &was, &change, 1, 0, nullptr, 0)) return rc;
  pc->free_count += pages_of(pc, pc->len[seq]) - pages_of(pc, len);
  pc->len[seq] = len;
  forget_rows(pc);
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_clear(shainet_paged_cache *pc, int seq) {
  if (!pc || seq >= pc->n_seqs) return fail(SHAINET_HIP_ERR_ARGUMENT, "invalid sequence");
  if (seq >= 0) return shainet_paged_cache_truncate(pc, seq, 0);
  if (int rc = check_device(pc)) return rc;
  if (int rc = refuse_recording(pc->ctx, "shainet_paged_cache_clear")) return rc;
  const hipError_t e = launch_page_reset(pc->lens, pc->n_seqs, pc->free_pages, pc->n_free, pc->n_pages, pc->ctx->stream);
  if (e != hipSuccess) return hip_fail(e, "reset launch");
  pc->len.assign(pc->n_seqs, 0);
  pc->free_count = pc->n_pages;
  pc->lengths_on_device = false;
  forget_rows(pc);
  return SHAINET_HIP_OK;
}

int shainet_paged_cache_read(shainet_paged_cache *pc, int layer, int seq, int kv_head, int pos0, int n, float *k_out, float *v_out) {
  if (!pc || layer < 0 || layer >= pc->layers || seq < 0 || seq >= pc->n_seqs || kv_head < 0 || kv_head >= pc->KV || pos0 < 0 || n < 0)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "invalid read arguments");
  if (int rc = refuse_unknown_lengths(pc, "shainet_paged_cache_read")) return rc;
  if ((long long)pos0 + n > pc->len[seq]) return fail(SHAINET_HIP_ERR_ARGUMENT, "rows %d..%lld of a sequence of %d", pos0, (long long)pos0 + n - 1, pc->len[seq]);
  if (n == 0) return SHAINET_HIP_OK;
  if (int rc = check_device(pc)) return rc;
  if (int rc = refuse_recording(pc->ctx, "shainet_paged_cache_read")) return rc;
  const size_t each = (size_t)pc->KV * n * pc->hd;
  if (int rc = pc->gathered.reserve(2 * each)) return rc;
  float *k = pc->gathered.p, *v = k + each;
  const hipError_t e = launch_page_gather(pool_of(pc, layer), seq, pos0, n, n, k, v, nullptr, pc->ctx->stream);
  if (e != hipSuccess) return hip_fail(e, "gather launch");
  HIP_TRY(hipStreamSynchronize(pc->ctx->stream));
  const size_t first = (size_t)kv_head * n * pc->hd, bytes = (size_t)n * pc->hd * sizeof(float);
  if (k_out) HIP_TRY(hipMemcpy(k_out, k + first, bytes, hipMemcpyDeviceToHost));
  if (v_out) HIP_TRY(hipMemcpy(v_out, v + first, bytes, hipMemcpyDeviceToHost));
  return SHAINET_HIP_OK;
}

int shainet_attn_append_paged(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const int *slots, const int *positions, int rows,
                              const float *q, long long q_stride, const float *k, long long k_stride, const float *v,
                              long long v_stride, float *q_rot) {
  if (int rc = check_pair(c, pc, layer)) return rc;
  if (!slots || !positions || !q || !k || !v || !q_rot) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (rows < 1 || rows > 0x3fffffff / (c->H + 2 * c->KV)) return fail(SHAINET_HIP_ERR_ARGUMENT, "rows must be in 1..%d", 0x3fffffff / (c->H + 2 * c->KV));
  if (q_stride < (long long)c->H * c->hd || k_stride < (long long)c->KV * c->hd || v_stride < (long long)c->KV * c->hd)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "row strides must be at least the row widths %d and %d", c->H * c->hd, c->KV * c->hd);
  const long long q_dim = (long long)c->H * c->hd, kv_dim = (long long)c->KV * c->hd;
  if (in_the_way(q, q_stride, q_dim, q_rot, q_dim, q_dim, rows) || in_the_way(k, k_stride, kv_dim, q_rot, q_dim, q_dim, rows) ||
      in_the_way(v, v_stride, kv_dim, q_rot, q_dim, q_dim, rows))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "q_rot must lie apart from q, k and v, or be q with rows as far apart");
  if (int rc = reach_table(c, reach_of(pc))) return rc;
  return append(c, pc, layer, prep_of(c, q, q_stride, k, k_stride, v, v_stride, q_rot), slots, positions, rows, nullptr, 0);
}

int shainet_attn_attend_paged(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const int *row_seqs, const int *positions,
                              int rows, const float *q_rot, long long q_stride, float *out, long long out_stride) {
  if (int rc = check_pair(c, pc, layer)) return rc;
  if (!row_seqs || !positions || !q_rot || !out) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (rows < 1 || rows > SHAINET_HIP_MAX_PAGED_SEQS)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "rows must be in 1..%d", SHAINET_HIP_MAX_PAGED_SEQS);
  if (q_stride < (long long)c->H * c->hd || out_stride < (long long)c->H * c->hd)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "row strides must be at least the row width %d", c->H * c->hd);
  const long long q_dim = (long long)c->H * c->hd;
  if (in_the_way(q_rot, q_stride, q_dim, out, out_stride, q_dim, rows))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "out must lie apart from q_rot, or be q_rot with rows as far apart");
  return attend(c, pc, layer, row_seqs, positions, rows, q_rot, q_stride, out, out_stride);
}

int shainet_attn_step_paged(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const int *seq_ids, int n, const float *q,
                            const float *k, const float *v, float *out) {
  if (int rc = check_pair(c, pc, layer)) return rc;
  if (!q || !k || !v || !out) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (n < 1 || n > pc->n_seqs) return fail(SHAINET_HIP_ERR_ARGUMENT, "n must be in 1..%d", pc->n_seqs);
  if (layer > 0 && n != pc->step_rows)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "layer %d of a step of %d rows: layer 0 mapped %d", layer, n, pc->step_rows);
  if (int rc = refuse_many_keys(c, pc, n)) return rc;  // (before a row is mapped)
  if (int rc = reach_table(c, pc->reach)) return rc;
  if (layer == 0) {
    MapArgs a = map_of(pc);
    a.n = n;
    a.reach = reach_with(c, pc);
    a.ids = seq_ids;
    a.slots = pc->step_slots;
    a.positions = pc->step_positions;
    a.row_seqs = pc->step_seqs;
    a.max_rows = n;
    a.rows_epoch = pc->n_free + kStepEpoch;
    const hipError_t e = launch_page_map(a, c->stream);
    if (e != hipSuccess) return hip_fail(e, "map launch");
    pc->lengths_on_device = true;
    pc->step_rows = n;
    pc->last_ids.clear();
  }
  const long long q_dim = (long long)c->H * c->hd, kv_dim = (long long)c->KV * c->hd;
  float *q_rot = pc->step_q.p;
  if (int rc = append(c, pc, layer, prep_of(c, q, q_dim, k, kv_dim, v, kv_dim, q_rot), pc->step_slots, pc->step_positions, n,
                      pc->step_seqs, kStepEpoch))
    return rc;
  return attend(c, pc, layer, pc->step_seqs, pc->step_positions, n, q_rot, q_dim, out, q_dim);
}

int shainet_attn_forward_paged(shainet_attn_ctx *c, shainet_paged_cache *pc, int layer, const int *seq_ids, const int *new_tokens,
                               int n_seqs, const float *q, const float *k, const float *v, float *out, int mem) {
  if (int rc = check_pair(c, pc, layer)) return rc;
  if (!new_tokens || !q || !k || !v || !out) return fail(SHAINET_HIP_ERR_ARGUMENT, "null argument");
  if (mem != SHAINET_HIP_MEM_HOST && mem != SHAINET_HIP_MEM_DEVICE)
    return fail(SHAINET_HIP_ERR_ARGUMENT, "mem must be SHAINET_HIP_MEM_HOST or SHAINET_HIP_MEM_DEVICE");
  if (n_seqs < 1 || n_seqs > SHAINET_HIP_MAX_BATCH) return fail(SHAINET_HIP_ERR_ARGUMENT, "n_seqs must be in 1..%d", SHAINET_HIP_MAX_BATCH);
  if (int rc = refuse_recording(c, "shainet_attn_forward_paged")) return rc;
  if (int rc = refuse_unknown_lengths(pc, "shainet_attn_forward_paged")) return rc;
  int ids[kMaxSeqs], start[kMaxSeqs], change[kMaxSeqs], longest = 0, furthest = 0;
  long long total = 0, pages = 0;
  for (int s = 0; s < n_seqs; ++s) {
    const int id = ids[s] = seq_ids ? seq_ids[s] : s, more = change[s] = new_tokens[s];
    if (id < 0 || id >= pc->n_seqs) return fail(SHAINET_HIP_ERR_ARGUMENT, "sequence id %d out of range", id);
    for (int t = 0; t < s; ++t)
      if (ids[t] == id) return fail(SHAINET_HIP_ERR_ARGUMENT, "sequence id %d appears twice", id);
    if (more < 1) return fail(SHAINET_HIP_ERR_ARGUMENT, "new_tokens must be positive");
    // (layers behind the first: the rows are counted already)
    start[s] = layer == 0 ? pc->len[id] : pc->len[id] - more;
    if (start[s] < 0) return fail(SHAINET_HIP_ERR_ARGUMENT, "layer %d: other rows than layer 0 had last: sequence %d has %d, not %d new ones", layer, id, pc->len[id], more);
    if ((long long)start[s] + more > reach_of(pc))
      return fail(SHAINET_HIP_ERR_CAPACITY, "sequence %d: %d cached + %d new rows exceed the %lld of its table", id, start[s], more, reach_of(pc));
    pages += pages_of(pc, (long long)start[s] + more) - pages_of(pc, start[s]);
    total += more;
    if (total > 0x3fffffff / (c->H + 2 * c->KV)) return fail(SHAINET_HIP_ERR_ARGUMENT, "too many rows in one call");
    if (more > kRowsFromPages && start[s] + more > longest) longest = start[s] + more;
    if (start[s] + more > furthest) furthest = start[s] + more;
  }
  if (layer == 0 && pages > pc->free_count)
    return fail(SHAINET_HIP_ERR_CAPACITY, "%lld pages wanted, %d free", pages, pc->free_count);
  if (layer > 0 && ((int)pc->last_ids.size() != n_seqs || memcmp(pc->last_ids.data(), ids, n_seqs * sizeof(int)) ||
                    memcmp(pc->last_new.data(), change, n_seqs * sizeof(int))))
    return fail(SHAINET_HIP_ERR_ARGUMENT, "layer %d: other rows than layer 0 of this cache had last", layer);
  const int rows = (int)total;
  const size_t q_floats = (size_t)rows * c->H * c->hd, kv_floats = (size_t)rows * c->KV * c->hd, gathered = (size_t)c->KV * longest * c->hd;
  const int reach = pc->reach;
  extend_reach(pc, furthest);
  int rc = reach_table(c, pc->reach);
  if (rc) pc->reach = reach;
  if (!rc) rc = c->q_rot.reserve(q_floats);
  if (!rc && longest) rc = pc->gathered.reserve(2 * gathered);
  const float *dq = q, *dk = k, *dv = v;
  float *dout = out;
  if (!rc && mem == SHAINET_HIP_MEM_HOST)
    (void)((rc = c->in_q.reserve(q_floats)) || (rc = c->in_k.reserve(kv_floats)) || (rc = c->in_v.reserve(kv_floats)) ||
           (rc = c->out.reserve(q_floats)) || (rc = c->pin_in.reserve(q_floats + 2 * kv_floats)) || (rc = c->pin_out.reserve(q_floats)));
  // (the last call's lists go when nothing else can be lacking any more: until then its other layers use them)
  if (!rc && layer == 0) rc = pc->rows.reserve(3 * (size_t)rows);
  if (rc) return rc;
  if (layer == 0) forget_rows(pc);
  if (mem == SHAINET_HIP_MEM_HOST) {
    float *pq = c->pin_in.p, *pk = pq + q_floats, *pv = pk + kv_floats;
    memcpy(pq, q, q_floats * sizeof(float));
    memcpy(pk, k, kv_floats * sizeof(float));
    memcpy(pv, v, kv_floats * sizeof(float));
    hipError_t ce = hipMemcpyAsync(c->in_q.p, pq, q_floats * sizeof(float), hipMemcpyHostToDevice, c->stream);
    if (ce == hipSuccess) ce = hipMemcpyAsync(c->in_k.p, pk, kv_floats * sizeof(float), hipMemcpyHostToDevice, c->stream);
    if (ce == hipSuccess) ce = hipMemcpyAsync(c->in_v.p, pv, kv_floats * sizeof(float), hipMemcpyHostToDevice, c->stream);
    if (ce != hipSuccess) {
      (void)hipStreamSynchronize(c->stream);  // a copy already queued may still read the staging buffer
      return hip_fail(ce, "hipMemcpyAsync(q, k, v)");
    }
    dq = c->in_q.p;
    dk = c->in_k.p;
    dv = c->in_v.p;
    dout = c->out.p;
  }
  int *lists = (int *)pc->rows.p;
  const int *slots = lists, *positions = lists + rows;
  int *row_seqs = lists + 2 * (size_t)rows;
  if (layer == 0) {
    try {
      pc->last_new.assign(change, change + n_seqs);
      pc->last_ids.assign(ids, ids + n_seqs);
    } catch (const std::bad_alloc &) {
      rc = fail(SHAINET_HIP_ERR_ALLOC, "out of host memory");
    }
    if (!rc) rc = map_listed(pc, ids, start, change, n_seqs, reach_with(c, pc), lists, rows);
    if (rc) {
      forget_rows(pc);
      if (mem == SHAINET_HIP_MEM_HOST) (void)hipStreamSynchronize(c->stream);
      return rc;
    }
  }
  const long long q_dim = (long long)c->H * c->hd, kv_dim = (long long)c->KV * c->hd;
  rc = append(c, pc, layer, prep_of(c, dq, q_dim, dk, kv_dim, dv, kv_dim, c->q_rot.p), slots, positions, rows,
              row_seqs, kForwardEpoch);
  // entries of a few rows each go together, from row `done` on; one of many by itself
  int at = 0, done = 0;
  for (int s = 0; s <= n_seqs && !rc; ++s) {
    const bool many = s < n_seqs && change[s] > kRowsFromPages;
    while ((many || s == n_seqs) && done < at && !rc) {
      const int some = at - done < kMaxPagedSeqs ? at - done : kMaxPagedSeqs;
      rc = attend(c, pc, layer, row_seqs + done, positions + done, some, c->q_rot.p + done * q_dim, q_dim, dout + done * q_dim, q_dim);
      done += some;
    }
    if (s == n_seqs || rc) break;
    if (many) {
      const int cap = start[s] + change[s];
      float *gk = pc->gathered.p, *gv = gk + gathered;
      const hipError_t e = launch_page_gather(pool_of(pc, layer), ids[s], 0, cap, cap, gk, gv, pc->ctx->error, c->stream);
      rc = e == hipSuccess ? shainet_attn_run_rows(c, c->q_rot.p + at * q_dim, gk, gv, cap, start[s], change[s], dout + at * q_dim)
                           : hip_fail(e, "gather launch");
      done = at + change[s];
    }
    at += change[s];
  }
  if (rc) {
    if (layer == 0) {  // the rows leave again: the call did not happen
      for (int s = 0; s < n_seqs; ++s) {
        start[s] += change[s];
        change[s] = -change[s];
      }
      (void)map_listed(pc, ids, start, change, n_seqs, 0, nullptr, 0);
      forget_rows(pc);
    }
    if (mem == SHAINET_HIP_MEM_HOST) (void)hipStreamSynchronize(c->stream);
    return rc;
  }
  if (layer == 0) {
    for (int s = 0; s < n_seqs; ++s) pc->len[ids[s]] += change[s];
    pc->free_count -= (int)pages;
  }
  c->last_rows = rows;
  if (mem == SHAINET_HIP_MEM_HOST) {
    const hipError_t ce = hipMemcpyAsync(c->pin_out.p, dout, q_floats * sizeof(float), hipMemcpyDeviceToHost, c->stream);
    const hipError_t se = hipStreamSynchronize(c->stream);  // also when the copy could not be queued
    if (ce != hipSuccess) return hip_fail(ce, "hipMemcpyAsync(out)");
    if (se != hipSuccess) return hip_fail(se, "hipStreamSynchronize");
    memcpy(out, c->pin_out.p, q_floats * sizeof(float));
    if (int of_map = check_error_word(pc->ctx->error)) return of_map;
    return check_error_word(c->error);
  }
  return SHAINET_HIP_OK;
}

}  // extern "C"
