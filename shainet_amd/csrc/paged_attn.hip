// Attention of one new row per sequence over its pages, and pages back into one piece of memory.
//
// out_h = sum_t p_t v_t / sum_t p_t,  p_t = exp(q_h . k_t / sqrt(hd) - max),  over the first positions + 1 rows of a sequence.
// A launch reads every key and value once for all query heads of its group and computes 4 g flops per number read, so the
// pages' bytes bound it; a short one is bound by what a launch, the plan and a trip to memory take.
//
// Work split.  The key tiles (16 rows of float32, 32 of 16-bit numbers: 8 KiB of K and 8 of V at head_dim 128) of all
// (row, kv head) pairs lie end to end, each pair behind a few empty places for what it costs to begin one, and are cut into
// equal spans, one per workgroup, whatever the lengths; every workgroup makes the sums that tell it where its span lies from the
// lengths themselves, so that nothing of a launch depends on them but what it does, and a recorded one is good for any
// lengths.  The wavefronts of a workgroup take its tiles in turn, each with a softmax of its own (running maximum, sum and
// output), and merge through LDS.  A pair that several workgroups share leaves a part with each; the workgroup that adds its
// part last (a count per pair) adds them all up, in the order of the keys, so results do not depend on who that is, and nobody
// waits for anybody.  Short pairs are cut into chunks, one per workgroup, instead, and many short ones go to a wavefront each.
//
// Measured (shared rows of all: K and V of 8 kv heads of 128, 32 query heads, pages of 16): 64 sequences of 8192 to 32768 keys of bfloat16
// 763 us, 6.8 TB/s (8 KiB pieces in any order, 64 KB on their way per compute unit, come at 6.5, 128 KB at 6.8); 16 of 2048 to 8192 of
// float32 105 us, 6.2 TB/s; one sequence of 1024 (heads of 64) 9 us, of which an empty launch takes 4.
//
// A wavefront has one tile in registers: it asks for the next tile's K once the scores are made, and for its V once the outputs are,
// straight from memory in the layout of the MFMA operands: for K 16 rows x 64 bytes per load, for V whole rows.  (Read
// that way 4 GiB came at 7.0 to 7.2 TB/s, with both halves as whole rows at 7.0 to 7.3, K's way alone at 6.1.)
//
// MFMA 16 x 16 layout (lane l, m = n = l % 16, quarter j = l / 16): A[m][k], B[k][n] with k = j (fp32) or 8 j .. 8 j + 7 (16 bits);
// D[m = 4 j + i][n] in register i.  Rows may be numbered as one likes: row m of the s-th 16 keys of a tile is key
// (m / 4) 4 S + 4 s + m % 4 of it (S = 1 or 2 of them per tile), so that quarter j's scores S^T = K Q^T are those of its 4 S neighbouring keys
// 4 S j .., in the order in which O^T += V^T P^T wants them as B: nothing crosses lanes.  And its V operand is the same
// keys' rows, a few neighbouring columns of each, transposed within the lane's registers.
#include "paged.hpp"
#include "lane_quarters.hpp"
#include "lane_sums.hpp"
#include "split_mfma.hpp"

namespace shainet {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DTYPE>
__device__ __forceinline__ float page_value(const void *pool, long long i) {
  if constexpr (DTYPE == kPageF32)
    return ((const float *)pool)[i];
  else if constexpr (DTYPE == kPageBf16)
    return (float)((const __bf16 *)pool)[i];
  else
    return (float)((const _Float16 *)pool)[i];
}

// Parts cross workgroups on XCDs whose L2 caches do not see each other's ordinary stores: relaxed atomic accesses at agent
// scope write through.  A part is in memory before its count goes up (the wait for its stores).
__device__ __forceinline__ void coherent_store(float *p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void coherent_store4(float *p, f32x4 v) {  // the same, 16 bytes at a time
  asm volatile("global_store_dwordx4 %0, %1, off sc1" : : "v"(p), "v"(v) : "memory");
}

__device__ __forceinline__ float coherent_load(const float *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 coherent_load4(const float *p) {
  typedef unsigned long long u64;
  const u64 a = __hip_atomic_load((const u64 *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const u64 b = __hip_atomic_load((const u64 *)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return f32x4{__builtin_bit_cast(float, (unsigned)a), __builtin_bit_cast(float, (unsigned)(a >> 32)),
               __builtin_bit_cast(float, (unsigned)b), __builtin_bit_cast(float, (unsigned)(b >> 32))};
}

constexpr int kCols = 16;  // query heads of a pair, at most: a larger group is several pairs
constexpr int kMaxWorkgroups = 512;
constexpr int kTickets = 4 * kMaxWorkgroups;  // two places a workgroup, two levels
// Parts that are added up at once: a sequence of 1024 keys, whose 16 parts then take one round, 8.9 us | 11.3 by 8; 32 is as good.
constexpr int kTeam = 16;
// Pairs of which each workgroup would have less than this many tiles are cut into chunks, if there are no more of them than workgroups: 24
// sequences of 20 to 700 keys (bfloat16) 10.5 us | as spans 15.6; 16 of 500 (float32), 16 tiles each, as spans 19 | as chunks 23.
constexpr int kShortSpan = 16;
// Pairs of up to this many, if there are more of them than workgroups, go to a wavefront each: 160 sequences of 50 to 480 keys, 8 kv heads
// (bfloat16), 41 us | as spans 55; of 100 to 960, 30 tiles, 80 | 82, and 100 of those 53 | 60 but 75 | 72 where all are long.
constexpr int kWavefrontTiles = 16;
// Tiles that the beginning of a pair costs a workgroup: 39 sequences of up to 5000 keys (bfloat16) 64 us | 86 with none; with 8, 65.  Where all
// are as long it costs a little: 16 of 500 (float32) 19 us | 17.8.
constexpr int kBegin = 4;
// Tiles of a pair, on average, that are many (launch_attend).
constexpr int kLongPair = 40;

// ... and what the kernel makes of it.
template <int DTYPE, int HD>
struct Tile : PageTile<DTYPE, HD> {
  static constexpr int PARTS = DTYPE == kPageF32 ? 1 : 3;  // of a float operand
  static constexpr int WAVES = 4;                          // of a workgroup
  static constexpr int LONG = HD == 64 ? 160 : 40;         // tiles of a span that one workgroup on a compute unit reads faster than two
  // Tiles of a pair that is not worth being cut: one sequence of 100 keys (7 tiles of float32) 6.7 us | cut 8.4.
  static constexpr int WHOLE = 12;
};

template <int WORDS>
struct Words;
template <>
struct Words<2> {
  typedef u32x2 T;
};
template <>
struct Words<3> {
  typedef unsigned T __attribute__((ext_vector_type(3), aligned(4)));  // (pieces of 12 bytes)
};
template <>
struct Words<4> {
  typedef u32x4 T;
};

template <int DTYPE, int HD, bool PAD>
struct Wave {
  using T = Tile<DTYPE, HD>;
  typedef typename Words<T::WORDS>::T VWords;
  static constexpr int KEYS_EACH = T::KEYS_EACH;

  // A tile in registers, or on its way there.
  struct Held {
    u32x4 k[T::S][T::CHUNKS];
    VWords v[KEYS_EACH][T::PIECES];
    bool in;  // whether this lane's V rows, which are the keys of its scores, lie in the pool
  };
  // This wavefront's share of a row of queries: chunks `first`, first + step, ...
  static constexpr int SHARE = (T::CHUNKS + T::WAVES - 1) / T::WAVES;
  struct Raw {
    f32x4 x[SHARE][T::PER / 4];
  };

  const PagePool &p;
  const u32x4 *q;  // the queries' parts in LDS, [PARTS][CHUNKS][64]
  const int lane, m, j;
  const int hd;
  Held held;
  f32x4 acc[T::PIECES][T::VEC];
  float top, sum;  // running maximum of the scores in log2 units, and this lane's share of the sum
  float c;         // scores to log2 units
  int down;        // float16: the queries were multiplied by 2^down
  struct Pages {
    int k, v;  // of this lane's K row and V rows in a tile
  };
  Pages now, next;  // of a walk's first tile, and of the tile to be asked for next
  const int *table;
  int last_page, len;
  const char *k_base, *v_base;

  __device__ __forceinline__ Wave(const PagePool &pool, float scale)
      : p(pool), lane(threadIdx.x & 63), m(lane & 15), j(lane >> 4), hd(PAD ? pool.hd : HD), c(scale * 1.44269504088896340736f), down(0) {}

  // (behind the last tile: its last page again)
  __device__ __forceinline__ void look_up(Pages &at_page, int tile) const {
    const int k0 = tile * T::KEYS;
    at_page.k = table[min((k0 + (m >> 2) * KEYS_EACH) >> p.shift, last_page)];
    at_page.v = table[min((k0 + j * KEYS_EACH) >> p.shift, last_page)];
  }
  __device__ __forceinline__ const char *row_at(const char *base, int page, int key) const {
    const long long row = ((long long)((unsigned)page < (unsigned)p.n_pages ? page : 0) * p.KV << p.shift) + (key & ((1 << p.shift) - 1));
    return base + row * (hd * T::E);
  }
  // (anew each time, so that there is no register for each load's offset over the loop)
  __device__ __forceinline__ int row_bytes() const {
    int n = hd * T::E;
    if (PAD) asm volatile("" : "+v"(n));
    return n;
  }
  __device__ __forceinline__ void ask_k(const Pages &at_page, int tile) {
    const int bytes = row_bytes();
#pragma unroll
    for (int s = 0; s < T::S; ++s) {
      const char *row = row_at(k_base, at_page.k, tile * T::KEYS + (m >> 2) * KEYS_EACH + 4 * s + (m & 3));
#pragma unroll
      for (int u = 0; u < T::CHUNKS; ++u) {
        const int at = PAD ? T::key_byte(u, j, bytes) : (u * 4 + j) * 16;
        held.k[s][u] = __builtin_nontemporal_load((const u32x4 *)(row + at));
      }
    }
  }
  // Row `row` of the values' operand, and so of the outputs: the first column of its piece u (or one behind the row's end, which nobody reads)
  __device__ __forceinline__ int column(int u, int row) const { return PAD && T::RUNS_OVER ? T::value_column(u, row, hd) : T::VEC * (row + 16 * u); }
  __device__ __forceinline__ void ask_v(const Pages &at_page, int tile) {
    const int numbers = row_bytes() / T::E;
    const char *row = row_at(v_base, at_page.v, tile * T::KEYS + j * KEYS_EACH);
    held.in = (unsigned)at_page.v < (unsigned)p.n_pages;
#pragma unroll
    for (int r = 0; r < KEYS_EACH; ++r)
#pragma unroll
      for (int u = 0; u < T::PIECES; ++u)
        held.v[r][u] = __builtin_nontemporal_load((const VWords *)(row + r * (hd * T::E) + (PAD ? T::value_column(u, m, numbers) : T::VEC * (m + 16 * u)) * T::E));
  }

  // The queries as B operands: chunk u of quarter j is d = (4 u + j) PER .. + PER - 1, as K's.
  __device__ __forceinline__ f32x4 query(const float *rows, int cols, int u, int w) const {
    const int d = (4 * u + j) * T::PER + 4 * w;
    f32x4 x = {0, 0, 0, 0};
    if (m < cols && (!PAD || d < hd) && u < T::CHUNKS)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = rows[m * hd + d + e];
    return x;
  }
  __device__ __forceinline__ void ask_queries(Raw &raw, const float *rows, int cols, int first, int step) const {
#pragma unroll
    for (int i = 0; i < SHARE; ++i)
#pragma unroll
      for (int w = 0; w < T::PER / 4; ++w) raw.x[i][w] = query(rows, cols, first + i * step, w);
  }
  // Three float16 parts of 11 bits hold all 24 of a float, but none below 2^-24: the largest of a row is brought to 2^14 .. 2^15, so that
  // numbers down to 2^-15 of it are exact and smaller ones, whose products vanish beside its, good to 2^-40 of it.
  __device__ __forceinline__ static float larger(float most, f32x4 x) {
    return fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
  }
  __device__ __forceinline__ float largest(const Raw &raw) const {  // of this wavefront's share
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < SHARE; ++i)
#pragma unroll
      for (int w = 0; w < T::PER / 4; ++w) most = larger(most, raw.x[i][w]);
    return max_across_quarters(most);
  }
  __device__ __forceinline__ void set_down(float most) { down = most > 0.0f && most < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(most) : 0; }
  __device__ __forceinline__ void put_query(u32x4 *to, const f32x4 (&x)[T::PER / 4], int u) const {
    u32x4 part[T::PARTS];
    if constexpr (DTYPE == kPageF32) {
      part[0] = __builtin_bit_cast(u32x4, x[0]);
    } else if constexpr (DTYPE == kPageBf16) {
      split_octet(x[0], x[1], part[0], part[1], part[2]);
    } else {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = ldexpf(x[e >> 2][e & 3], down);
      split_f16(y, part);
    }
#pragma unroll
    for (int i = 0; i < T::PARTS; ++i) to[(i * T::CHUNKS + u) * 64 + lane] = part[i];
  }
  __device__ __forceinline__ void put_queries(u32x4 *to, const Raw &raw, int first, int step) const {
#pragma unroll
    for (int i = 0; i < SHARE; ++i)
      if (first + i * step < T::CHUNKS) put_query(to, raw.x[i], first + i * step);
  }
  // ... all of them by this wavefront, for itself
  __device__ __forceinline__ void own_queries(u32x4 *to, const float *rows, int cols) {
    if constexpr (DTYPE == kPageF16) {
      float most = 0.0f;
#pragma unroll
      for (int u = 0; u < T::CHUNKS; ++u)
#pragma unroll
        for (int w = 0; w < T::PER / 4; ++w) most = larger(most, query(rows, cols, u, w));
      set_down(max_across_quarters(most));
    }
#pragma unroll
    for (int u = 0; u < T::CHUNKS; ++u) {
      f32x4 x[T::PER / 4];
#pragma unroll
      for (int w = 0; w < T::PER / 4; ++w) x[w] = query(rows, cols, u, w);
      put_query(to, x, u);
    }
  }
  __device__ __forceinline__ static void split_f16(const float (&y)[8], u32x4 (&part)[T::PARTS]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = y[2 * e], b = y[2 * e + 1];
#pragma unroll
      for (int i = 0; i < T::PARTS; ++i) {
        const f16x2 h = f16x2{(_Float16)a, (_Float16)b};
        part[i][e] = __builtin_bit_cast(unsigned, h);
        a -= (float)h.x;
        b -= (float)h.y;
      }
    }
  }
  __device__ __forceinline__ static f32x4 mfma16(u32x4 a, u32x4 b, f32x4 x) {
    if constexpr (DTYPE == kPageBf16)
      return mfma_bf16_16(a, b, x);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), x, 0, 0, 0);
  }

  // Looks up the first two of a sequence's tiles first, first + step, ...; `ask` asks for the first, if it is below last.
  __device__ __forceinline__ void start(int seq, int keys, int kv, int first, int step) {
    len = keys;
    table = p.table + (long long)seq * p.seq_pages;
    last_page = (len - 1) >> p.shift;
    const long long head = ((long long)kv << p.shift) * (hd * T::E);
    k_base = (const char *)p.k + head;
    v_base = (const char *)p.v + head;
    look_up(now, first);
    look_up(next, first + step);
  }
  __device__ __forceinline__ void ask(int first, int last) {
    // (the entries are waited for here, where nothing is behind them yet)
    asm volatile("" : "+v"(now.k), "+v"(now.v), "+v"(next.k), "+v"(next.v));
    if (first >= last) return;
    ask_k(now, first);
    ask_v(now, first);
  }

  // What is held becomes part of sums and outputs.  MORE: and its place is asked to hold tile `then`, whose pages were looked
  // up, those of `after` before it.  (Loads come back in order and are waited for by their number: how many are on their way has to be the same
  // however the code is reached, and an address that came by a load behind others would wait for all of them.)
  template <bool MORE>
  __device__ __forceinline__ void take(int tile, int then, int after) {
    f32x4 x[T::S];
#pragma unroll
    for (int s = 0; s < T::S; ++s) x[s] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int part = T::PARTS - 1; part >= 0; --part)
#pragma unroll
      for (int u = 0; u < T::CHUNKS; ++u) {
        const u32x4 mine = q[(part * T::CHUNKS + u) * 64 + lane];
#pragma unroll
        for (int s = 0; s < T::S; ++s) {
          if constexpr (DTYPE == kPageF32) {
            const f32x4 k = __builtin_bit_cast(f32x4, held.k[s][u]), y = __builtin_bit_cast(f32x4, mine);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[s] = mfma_f32_16(k[e], y[e], x[s]);
          } else {
            x[s] = mfma16(held.k[s][u], mine, x[s]);
          }
        }
      }
    const Pages its = next;
    if constexpr (MORE) {
      look_up(next, after);
      ask_k(its, then);
    }
    // keys behind the sequence's end or in no page: no score, and a value that is no number would not vanish at weight 0
    float most = -INFINITY;
    if (__any(!held.in || (tile + 1) * T::KEYS > len)) {
      const int key = tile * T::KEYS + j * KEYS_EACH;
#pragma unroll
      for (int r = 0; r < KEYS_EACH; ++r)
        if (!held.in || key + r >= len) {
          x[r >> 2][r & 3] = -INFINITY;
#pragma unroll
          for (int u = 0; u < T::PIECES; ++u) held.v[r][u] = VWords{};
        }
    }
#pragma unroll
    for (int r = 0; r < KEYS_EACH; ++r) {
      if constexpr (DTYPE == kPageF16) x[r >> 2][r & 3] = ldexpf(x[r >> 2][r & 3], -down);
      most = fmaxf(most, x[r >> 2][r & 3]);
    }
    most = max_across_quarters(most) * c;
    if (__any(most > top)) {
      const float now = fmaxf(top, most);
      const float fade = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= fade;
#pragma unroll
      for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) acc[u][e] *= fade;
    }
    // (float16 parts of a weight: lifted by 2^15, as the queries are; the sum is lifted with them.  A weight of 2^-16 of the largest and less is
    // good to 2^-40 of that one, which beside it no float32 sum keeps.)
    const float from = top == -INFINITY ? 0.0f : DTYPE == kPageF16 ? top - 15.0f : top;
    float w[KEYS_EACH];
#pragma unroll
    for (int r = 0; r < KEYS_EACH; ++r) {
      w[r] = __builtin_amdgcn_exp2f(fmaf(x[r >> 2][r & 3], c, -from));
      sum += w[r];
    }
    if constexpr (DTYPE == kPageF32) {
#pragma unroll
      for (int r = 0; r < KEYS_EACH; ++r)
#pragma unroll
        for (int u = 0; u < T::PIECES; ++u) {
          typedef float Columns __attribute__((ext_vector_type(T::WORDS)));
          const Columns columns = __builtin_bit_cast(Columns, held.v[r][u]);
#pragma unroll
          for (int e = 0; e < T::VEC; ++e) acc[u][e] = mfma_f32_16(columns[e], w[r], acc[u][e]);
        }
    } else {
      u32x4 weights[T::PARTS];
      if constexpr (DTYPE == kPageBf16)
        split_octet(f32x4{w[0], w[1], w[2], w[3]}, f32x4{w[4], w[5], w[6], w[7]}, weights[0], weights[1], weights[2]);
      else
        split_f16(w, weights);
#pragma unroll
      for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) {
          u32x4 column;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            column[r] = __builtin_amdgcn_perm(held.v[2 * r + 1][u][e >> 1], held.v[2 * r][u][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int part = T::PARTS - 1; part >= 0; --part) acc[u][e] = mfma16(column, weights[part], acc[u][e]);
        }
    }
    if constexpr (MORE) ask_v(its, then);
  }

  // Sums and outputs of those tiles.
  __device__ __forceinline__ void walk(int first, int last, int step) {
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
      for (int e = 0; e < T::VEC; ++e) acc[u][e] = f32x4{0, 0, 0, 0};
    if (first >= last) return;
    int tile = first;
#pragma unroll 1
    for (; tile + step < last; tile += step) take<true>(tile, tile + step, tile + 2 * step);
    take<false>(tile, 0, 0);
  }
};

// a / b of whole numbers, a below 2^53: the rounded quotient is off by at most 2^-53 a / b, less than the 1 / b that parts a
// quotient from the next whole number above.  (A division of 64-bit integers is over a hundred instructions.)
__device__ __forceinline__ int quotient(long long a, long long b) { return (int)((double)a / (double)b); }

// How a launch shares out its work; the same for all workgroups, each of which makes it for itself.
enum { kSpans, kChunks, kWavefronts };

// PER_CU: workgroups of a compute unit, 1 or 2.
template <int DTYPE, int HD, bool PAD, int PER_CU>
__global__ __launch_bounds__((64 * Tile<DTYPE, HD>::WAVES), (Tile<DTYPE, HD>::WAVES / 4 * PER_CU)) void paged_attend_kernel(PagedAttendArgs a, PagePool p) {
  using T = Tile<DTYPE, HD>;
  constexpr int WAVES = T::WAVES, THREADS = 64 * WAVES, STRIDE = HD + 4;
  constexpr int NEAR = 512;                                 // rows whose lengths stay at hand
  __shared__ int starts[kMaxPagedSeqs + 1];                 // units of one kv head in the rows before: tiles or chunks
  __shared__ int seqs[NEAR], lens[NEAR];
  // the queries, and the wavefronts' outputs behind them; of wavefronts that go their own ways, the queries of each
  constexpr int QUERIES = T::PARTS * T::CHUNKS * 64 * 4, OUTS = WAVES * kCols * STRIDE;
  __shared__ __align__(16) float shared[QUERIES + (OUTS > (WAVES - 1) * QUERIES ? OUTS : (WAVES - 1) * QUERIES)];
  auto outs = [&](int v, int n, int d) { return shared + QUERIES + (v * kCols + n) * STRIDE + d; };
  __shared__ float tops[WAVES][kCols], sums[WAVES][kCols], larges[WAVES][kCols];
  __shared__ int scan[WAVES], held[WAVES], longest[WAVES], last_one;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // (values from LDS that are the same in all lanes are said to be: they live in scalar registers then)
  auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int hd = PAD ? p.hd : HD;
  const int g = a.g, per_kv = (g + kCols - 1) / kCols, pairs = p.KV * per_kv;
  const int most_keys = (int)min((long long)p.seq_pages << p.shift, 0x3fffffffLL);
  constexpr int all_wgs = 256 * PER_CU;  // of every launch

  // rows of a length that has a sequence; -1: a row to be left alone
  auto length_of = [&](int r, int &seq) {
    seq = a.row_seqs[r];
    return (unsigned)seq < (unsigned)p.n_seqs ? max(0, min(a.positions[r], most_keys - 1) + 1) : -1;
  };
  auto known_length = [&](int r) {
    int seq;
    return r < NEAR ? lens[r] : length_of(r, seq);
  };
  auto tiles_of = [](int len) { return (max(len, 0) + T::KEYS - 1) / T::KEYS; };
  // the rows' tiles in all, how many rows have any, and the most of one.  Up to a wavefront's lanes of rows: every wavefront
  // makes them for itself (they all write the same to LDS, and each reads what it wrote), and nobody waits at a barrier.
  const bool few = a.rows <= 64;
  const int each = few ? 1 : (a.rows + THREADS - 1) / THREADS, first_row = few ? lane : t * each;
  int row_tiles = 0, some = 0, most = 0;
  for (int i = 0; i < each; ++i) {
    const int r = first_row + i;
    if (r >= a.rows) break;
    int seq;
    const int len = length_of(r, seq), tiles = tiles_of(len);
    if (r < NEAR) {
      seqs[r] = seq;
      lens[r] = len;
    }
    row_tiles += tiles;
    some += tiles > 0 ? 1 : 0;
    most = max(most, tiles);
  }
  row_tiles = __builtin_amdgcn_readlane(sum_lanes(row_tiles), 63);
  some = few ? (int)__builtin_popcountll(__ballot(some)) : __builtin_amdgcn_readlane(sum_lanes(some), 63);
  most = __builtin_amdgcn_readlane(max_lanes(most), 63);
  if (!few) {
    if (lane == 0) {
      scan[wave] = row_tiles;
      held[wave] = some;
      longest[wave] = most;
    }
    __syncthreads();
    row_tiles = some = most = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      row_tiles += scan[w];
      some += held[w];
      most = max(most, longest[w]);
    }
  }
  row_tiles = same(row_tiles);
  some = same(some);
  most = same(most);
  // outputs of rows without keys
  for (int r = blockIdx.x; r < a.rows; r += all_wgs)
    if (known_length(r) == 0)
      for (int i = t; i < a.H * hd; i += THREADS) a.out[r * a.out_stride + i] = 0.0f;
  const long long total = (long long)row_tiles * pairs, n_pairs = (long long)some * pairs;
  // Of long spans of long pairs one workgroup on a compute unit is enough, and the others leave (see launch_attend)
  const int wgs = PER_CU == 2 && total >= (long long)all_wgs * T::LONG && total >= n_pairs * kLongPair ? all_wgs / 2 : all_wgs;
  if ((int)blockIdx.x >= wgs) return;
  int mode = kSpans;
  int unit = 1;  // tiles and beginnings of a span, or tiles of a chunk at most (32 bits: half a microsecond of a short launch)
  if (n_pairs > wgs && most <= kWavefrontTiles) {
    mode = kWavefronts;
  } else if (total <= (long long)wgs * (kShortSpan - 1) && n_pairs <= wgs) {
    // chunks of pairs, one a workgroup: sum of ceil(tiles / unit) <= total / unit + pairs
    mode = kChunks;
    unit = n_pairs < wgs && most > T::WHOLE ? max(quotient(total + (wgs - n_pairs) - 1, wgs - n_pairs), WAVES) : max(most, 1);
  } else {
    unit = max(1, (int)((total + kBegin * n_pairs + wgs - 1) / wgs));
  }
  if (mode != kWavefronts) {  // units of one kv head before each row
    auto units_of = [&](int r) {
      const int tiles = tiles_of(known_length(r));
      return mode == kSpans ? (tiles > 0 ? tiles + kBegin : 0) : quotient((long long)tiles + unit - 1, unit);
    };
    if (few) {
      const int mine = lane < a.rows ? units_of(lane) : 0, upto = sum_lanes(mine);
      if (lane < a.rows) starts[lane + 1] = upto;
      if (lane == 0) starts[0] = 0;
    } else {
      int mine = 0;
      for (int i = 0; i < each && first_row + i < a.rows; ++i) mine += units_of(first_row + i);
      const int upto = sum_lanes(mine);
      __syncthreads();  // (`scan` has been read)
      if (lane == 63) scan[wave] = upto;
      __syncthreads();
      int before = upto - mine;
      for (int w = 0; w < wave; ++w) before += scan[w];
      for (int i = 0; i < each && first_row + i < a.rows; ++i) {
        starts[first_row + i] = before;
        before += units_of(first_row + i);
        if (first_row + i == a.rows - 1) starts[a.rows] = before;
      }
      __syncthreads();
    }
  }

  const long long all_units = mode == kWavefronts ? (long long)a.rows * pairs : (long long)same(starts[a.rows]) * pairs;
  long long at = mode == kSpans ? (long long)blockIdx.x * unit : mode == kChunks ? blockIdx.x : blockIdx.x + (long long)wgs * wave;
  const long long end = mode == kSpans ? min(all_units, at + unit) : mode == kChunks ? min(all_units, at + 1) : all_units;
  unsigned *tickets = (unsigned *)a.workspace;
  float *parts = (float *)(tickets + kTickets);
  constexpr int PART = kCols * HD + 4 * kCols;  // a workgroup has two: of the pair that it begins with, and of the one that goes on behind it
  int row = 0;
  if (mode != kWavefronts && at < end) {
    int lo = 0, hi = a.rows - 1;
    while (lo < hi) {  // the last row that begins at or before it
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)same(starts[mid]) * pairs <= at)
        lo = mid;
      else
        hi = mid - 1;
    }
    row = lo;
  }
  // A pair, and which of its tiles are this workgroup's (wavefront's); first_wg .. last_wg: whose the pair is
  struct Segment {
    int row, seq, len, pair, first, last;
    int first_wg, last_wg;
    bool late, first_late;  // the pair begins in this workgroup's span (in first_wg's) but not with it: its part is the second there
  };
  auto next_segment = [&](Segment &s) {
    while (at < end) {
      if (mode == kWavefronts) {
        row = quotient(at, pairs);
        s.pair = (int)(at - (long long)row * pairs);
        at += (long long)wgs * WAVES;
      } else {
        while ((long long)same(starts[row + 1]) * pairs <= at) ++row;
      }
      row = same(row);
      s.row = row;
      if (row < NEAR) {
        s.seq = same(seqs[row]);
        s.len = same(lens[row]);
      } else {
        s.len = length_of(row, s.seq);
      }
      const int tiles = tiles_of(s.len);
      s.first = 0;
      s.last = tiles;
      if (mode == kWavefronts) {
        if (tiles == 0) continue;
        s.pair = same(s.pair);
        return true;
      }
      const int units = same(starts[row + 1] - starts[row]);
      const long long of_row = (long long)same(starts[row]) * pairs;
      s.pair = same(quotient(at - of_row, units));
      const long long begins = of_row + (long long)s.pair * units;
      const int from = (int)(at - begins);
      if (mode == kSpans) {
        const long long first_tile = begins + kBegin;
        s.first = max(from - kBegin, 0);
        s.last = (int)(min(end, begins + units) - first_tile);
        at = min(end, begins + units);
        if (s.last <= s.first) continue;
        s.first_wg = quotient(first_tile, unit);
        s.last_wg = quotient(begins + units - 1, unit);
        s.late = first_tile > (long long)blockIdx.x * unit;
        s.first_late = first_tile > (long long)s.first_wg * unit;
      } else {  // equal shares
        s.first = quotient((long long)tiles * from, units);
        s.last = quotient((long long)tiles * (from + 1), units);
        at += 1;
        s.first_wg = (int)begins;
        s.last_wg = (int)begins + units - 1;
        s.late = s.first_late = false;
      }
      return true;
    }
    return false;
  };

  // Of two workgroups on a compute unit the first one's requests go before the other's: with equal spans the first ones ended at
  // 77 to 100 us and the others at 108 to 118 (16 sequences of 2048 to 8192 keys, float32, two on each).  The others' instructions
  // go first, therefore: half to one per cent of most launches.  (Spans of unequal lengths, or short ones for whoever is
  // ready, cost more in parts of pairs than they gave: 110 -> 113 and 121 us.)
  if (PER_CU == 2 && (int)blockIdx.x >= all_wgs / 2) __builtin_amdgcn_s_setprio(3);
  Wave<DTYPE, HD, PAD> w(p, a.scale);
  const bool alone = mode == kWavefronts;
  const int step = alone ? 1 : WAVES, mine = alone ? 0 : wave;
  u32x4 *const queries = (u32x4 *)shared + (alone ? wave * (QUERIES / 4) : 0);
  w.q = queries;
  auto kv_of = [&](const Segment &s) { return per_kv == 1 ? s.pair : s.pair / per_kv; };
  auto head_of = [&](const Segment &s) { return kv_of(s) * g + (s.pair - kv_of(s) * per_kv) * kCols; };
  auto cols_of = [&](const Segment &s) { return min(kCols, g - (s.pair - kv_of(s) * per_kv) * kCols); };
  auto rows_of = [&](const Segment &s) { return a.q + s.row * a.q_stride + (long long)head_of(s) * hd; };
  typename Wave<DTYPE, HD, PAD>::Raw raw;
  // a segment's table entries and queries are asked for first, then its first tile
  auto start = [&](const Segment &s) {
    w.start(s.seq, s.len, kv_of(s), s.first + mine, step);
    if (!alone) w.ask_queries(raw, rows_of(s), cols_of(s), wave, WAVES);
    w.ask(s.first + mine, s.last);
  };
  auto put_largest = [&] {  // (before a barrier, and put_queries behind it)
    if constexpr (DTYPE == kPageF16) {
      const float most = w.largest(raw);
      if (lane < kCols) larges[wave][lane] = most;
    }
  };
  auto put_queries = [&](const Segment &s) {
    if (alone) {
      w.own_queries(queries, rows_of(s), cols_of(s));
      return;
    }
    if constexpr (DTYPE == kPageF16) {
      float most = larges[0][w.m];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) most = fmaxf(most, larges[v][w.m]);
      w.set_down(most);
    }
    w.put_queries(queries, raw, wave, WAVES);
  };
  Segment s;
  bool more = next_segment(s);
  if (more) {
    start(s);
    if (DTYPE == kPageF16 && !alone) {  // (then all wavefronts have the same segment)
      put_largest();
      __syncthreads();
    }
    put_queries(s);
  }
  __syncthreads();
  while (more) {
    const int cols = cols_of(s);
    float *out = a.out + s.row * a.out_stride + (long long)head_of(s) * hd;
    w.walk(s.first + mine, s.last, step);
    // the next segment's first tile is on its way while this one's outputs are put together
    const Segment now = s;
    more = next_segment(s);
    if (more) start(s);
    const float its_sum = sum_across_quarters(w.sum);
    if (alone) {
      const float over = its_sum == 0.0f ? 0.0f : 1.0f / its_sum;
      if (w.m < cols)  // (columns that two pieces have are the same number twice)
#pragma unroll
        for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < T::VEC; ++e)
              if (!PAD || T::VEC * (4 * w.j + i + 16 * u) < hd) out[w.m * hd + w.column(u, 4 * w.j + i) + e] = w.acc[u][e][i] * over;
      if (more) put_queries(s);
      continue;
    }

    // the wavefronts' parts, on one maximum
    if (lane < kCols) {
      tops[wave][lane] = w.top;
      sums[wave][lane] = its_sum;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, tops[i][w.m]);
    const float fade = w.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w.top - top);
    if (w.m < cols)
#pragma unroll
      for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < T::VEC; ++e)
            *outs(wave, w.m, w.column(u, 4 * w.j + i) + e) = w.acc[u][e][i] * fade;
    if (more) put_largest();
    __syncthreads();
    if (more) put_queries(s);  // (nobody reads the old ones any more)
    const bool whole = now.first_wg == now.last_wg;
    const int fours = cols * hd / 4;
    // Parts of a pair: k = 0 .. n_parts - 1, each in its workgroup's first or second place.
    const int n_parts = now.last_wg - now.first_wg + 1;
    auto place_of = [&](int k) { return (now.first_wg + k) * 2 + (k == 0 && now.first_late ? 1 : 0); };
    float *part = parts + (blockIdx.x * 2 + (now.late ? 1 : 0)) * PART;
    for (int i = t; i < fours; i += THREADS) {
      const int n = 4 * i / hd, d = 4 * i - n * hd;
      f32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) x += *(const f32x4 *)outs(v, n, d);
      if (whole || d == 0) {
        float best = -INFINITY, l = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) best = fmaxf(best, tops[v][n]);
#pragma unroll
        for (int v = 0; v < WAVES; ++v) l += sums[v][n] * (tops[v][n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(tops[v][n] - best));
        if (whole) {
          const float over = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int e = 0; e < 4; ++e) out[4 * i + e] = x[e] * over;
        } else {
          coherent_store(part + kCols * HD + n, best);
          coherent_store(part + kCols * HD + kCols + n, l);
        }
      }
      if (!whole) coherent_store4(part + 4 * i, x);
    }
    // Up to kTeam parts are added up by the last one's workgroup; of more, each so many first, by the last of theirs, into the
    // place of their first, and then what that leaves.
    int first_part = 0, gap = 1, count = n_parts;
    if (n_parts > kTeam) {
      first_part = (blockIdx.x - now.first_wg) / kTeam * kTeam;
      count = min(kTeam, n_parts - first_part);
    }
#pragma unroll 1
    for (bool going = !whole; going;) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t == 0) {
        unsigned *ticket = tickets + (gap == 1 ? 0 : 2 * kMaxWorkgroups) + place_of(first_part);
        const unsigned before = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_one = before == (unsigned)count - 1;
        if (last_one) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (!last_one) break;
      const bool final = gap > 1 || n_parts <= kTeam;
      // A thread adds up four neighbouring outputs over the parts, with a running maximum as a wavefront does over tiles; where
      // there are fewer outputs than threads, teams of threads take every so-manieth part each.
      const int teams = max(1, THREADS / fours), team = teams > 1 ? t / fours : 0;
      float *work = shared + QUERIES;  // [teams][fours][6]
      float *to = parts + place_of(first_part) * PART;
      auto finish = [&](int i, f32x4 x, float best, float l) {
        if (final) {
          const float over = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int e = 0; e < 4; ++e) out[4 * i + e] = x[e] * over;
        } else {
          const int n = 4 * i / hd;
          coherent_store4(to + 4 * i, x);
          if (4 * i == n * hd) {
            coherent_store(to + kCols * HD + 2 * kCols + n, best);  // (others still read its own)
            coherent_store(to + kCols * HD + 3 * kCols + n, l);
          }
        }
      };
      const int peaks = kCols * HD + (gap > 1 ? 2 * kCols : 0);  // maxima and sums of parts, or of what they were added up to
#pragma unroll 1
      for (int i = teams > 1 ? t - team * fours : t; i < fours && team < teams; i += teams > 1 ? fours : THREADS) {
        const int n = 4 * i / hd;
        float best = -INFINITY, l = 0.0f;
        f32x4 x = {0, 0, 0, 0};
        constexpr int SOME = 8;
#pragma unroll 1
        for (int k = team; k < count; k += SOME * teams) {
          float its[SOME], its_l[SOME];
          f32x4 its_x[SOME];
#pragma unroll
          for (int z = 0; z < SOME; ++z) {
            const float *from = parts + place_of(first_part + min(k + z * teams, count - 1) * gap) * PART;
            its[z] = coherent_load(from + peaks + n);
            its_l[z] = coherent_load(from + peaks + kCols + n);
            its_x[z] = coherent_load4(from + 4 * i);
          }
          float higher = best;
#pragma unroll
          for (int z = 0; z < SOME; ++z) higher = fmaxf(higher, its[z]);
          const float less = best == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(best - higher);
          best = higher;
          l *= less;
          x *= less;
#pragma unroll
          for (int z = 0; z < SOME; ++z) {  // (no branch: loads behind one would wait for the one before)
            const float f = its[z] == -INFINITY || k + z * teams >= count ? 0.0f : __builtin_amdgcn_exp2f(its[z] - higher);
            l = fmaf(its_l[z], f, l);
            x += its_x[z] * f;
          }
        }
        if (teams == 1) {
          finish(i, x, best, l);
        } else {
          float *mine_at = work + (team * fours + i) * 6;
          mine_at[0] = best;
          mine_at[1] = l;
#pragma unroll
          for (int e = 0; e < 4; ++e) mine_at[2 + e] = x[e];
        }
      }
      if (teams > 1) {
        __syncthreads();
        for (int i = t; i < fours; i += THREADS) {
          float best = -INFINITY, l = 0.0f;
          for (int k = 0; k < teams; ++k) best = fmaxf(best, work[(k * fours + i) * 6]);
          f32x4 x = {0, 0, 0, 0};
          for (int k = 0; k < teams; ++k) {
            const float *from = work + (k * fours + i) * 6;
            const float f = from[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(from[0] - best);
            l = fmaf(from[1], f, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(from[2 + e], f, x[e]);
          }
          finish(i, x, best, l);
        }
      }
      going = !final;
      first_part = 0;
      gap = kTeam;
      count = (n_parts + kTeam - 1) / kTeam;
    }
    __syncthreads();  // the next segment writes to LDS
  }
}

// Where the row of key t of a sequence lies in the pools; -1 where the table names no page.
__device__ __forceinline__ long long page_row(const PagePool &p, const int *table, int t, int head) {
  const int page = table[t >> p.shift];
  if ((unsigned)page >= (unsigned)p.n_pages) return -1;
  return (((long long)page * p.KV + head) << p.shift) + (t & ((1 << p.shift) - 1));
}

template <int DTYPE>
__global__ __launch_bounds__(256) void page_gather_kernel(PagePool p, int seq, int pos0, int n, int cap, float *k, float *v, int *error) {
  const int per = p.hd >> 2;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)n * p.KV * per) return;
  const int piece = (int)(i % per), t = (int)(i / per % n), c = (int)(i / per / n);
  const long long row = page_row(p, p.table + (long long)seq * p.seq_pages, pos0 + t, c);
  const long long to = ((long long)c * cap + t) * p.hd + 4 * piece;
  if (row < 0 && error && c == 0 && piece == 0 && *(volatile int *)error == 0) *(volatile int *)error = kKeysOutside;  // (a map that failed before says why)
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (k) k[to + e] = row < 0 ? 0.0f : page_value<DTYPE>(p.k, row * p.hd + 4 * piece + e);
    if (v) v[to + e] = row < 0 ? 0.0f : page_value<DTYPE>(p.v, row * p.hd + 4 * piece + e);
  }
}

}  // namespace

size_t paged_attend_workspace(int hd) {
  const int tile = hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256;
  return kTickets * sizeof(unsigned) + (size_t)kMaxWorkgroups * 2 * kCols * (tile + 4) * sizeof(float);
}

namespace {
template <int DTYPE, int HD, bool PAD, int PER_CU>
hipError_t launch_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  constexpr int wgs = 256 * PER_CU;  // (the kernel counts on that many)
  static_assert(wgs <= kMaxWorkgroups, "counts and parts");
  hipLaunchKernelGGL((paged_attend_kernel<DTYPE, HD, PAD, PER_CU>), dim3((unsigned)wgs), dim3(64 * Tile<DTYPE, HD>::WAVES), 0, stream, a, p);
  return hipGetLastError();
}
// One workgroup on a compute unit reads long stretches of few pairs faster than two, of which the first gets ahead: 16 sequences of 2048 to
// 8192 keys (128 pairs, float32) 105.5 us | two 106.7, one of 131072 (4 pairs, bfloat16) 50 | 53, 24 of 20 to 700 (192 pairs) 10.9 | 12.1.
// Where there are more pairs than compute units two hide each other's beginnings and ends: 64 sequences of 100 to 300 keys
// (512 pairs, float32) two 25 us | one 33, 39 of up to 5000 (312 pairs of heads of 64, tiles of half the bytes) 38 | 46.  How long their
// spans are is known on the device only, where half of the workgroups leave if they are long: 64 sequences of 8192 to 32768 keys
// (bfloat16) 763 us | two 780, 77 of up to 5000 (heads of 96, float16) 63 | 65.5, 100 of 1000 to 3000 (bfloat16) 132 | 137.  Where
// pairs are short two are better whatever the spans: 128 of 1000 (32 tiles of bfloat16) 86 us | one 89, 700 of 100 to 700 228 | 257.
template <int DTYPE, int HD>
hipError_t launch_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  if constexpr (HD == 256) {  // (registers for one)
    return p.hd == HD ? launch_attend<DTYPE, HD, false, 1>(a, p, stream) : launch_attend<DTYPE, HD, true, 1>(a, p, stream);
  } else {
    if (p.hd != HD) return launch_attend<DTYPE, HD, true, 2>(a, p, stream);
    const long long pairs = (long long)a.rows * p.KV * ((a.g + kCols - 1) / kCols);
    return pairs <= 256 ? launch_attend<DTYPE, HD, false, 1>(a, p, stream) : launch_attend<DTYPE, HD, false, 2>(a, p, stream);
  }
}
template <int DTYPE>
hipError_t launch_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  return p.hd <= 64 ? launch_attend<DTYPE, 64>(a, p, stream) : p.hd <= 96 ? launch_attend<DTYPE, 96>(a, p, stream) : p.hd <= 128 ? launch_attend<DTYPE, 128>(a, p, stream) : launch_attend<DTYPE, 256>(a, p, stream);
}
}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  if (a.rows < 1 || a.rows > kMaxPagedSeqs || a.H < 1 || a.H % p.KV || (p.hd & 7) || p.hd < 8 || p.hd > 256 || p.shift < 3)
    return hipErrorInvalidValue;
  return p.dtype == kPageF32 ? launch_attend<kPageF32>(a, p, stream) : p.dtype == kPageBf16 ? launch_attend<kPageBf16>(a, p, stream) : launch_attend<kPageF16>(a, p, stream);
}

hipError_t launch_page_gather(const PagePool &p, int seq, int pos0, int n, int cap, float *k, float *v, int *error, hipStream_t stream) {
  if (n < 1) return hipSuccess;
  if (seq < 0 || seq >= p.n_seqs || pos0 < 0 || (long long)pos0 + n > (long long)p.seq_pages << p.shift || n > cap)
    return hipErrorInvalidValue;
  const long long blocks = ((long long)n * p.KV * (p.hd >> 2) + 255) / 256;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  const auto kernel = p.dtype == kPageF32    ? page_gather_kernel<kPageF32>
                      : p.dtype == kPageBf16 ? page_gather_kernel<kPageBf16>
                                             : page_gather_kernel<kPageF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, seq, pos0, n, cap, k, v, error);
  return hipGetLastError();
}

}  // namespace shainet
