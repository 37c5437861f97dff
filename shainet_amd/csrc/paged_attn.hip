// Attention of one new row per sequence over its pages, and pages back into one piece of memory.
//
// out_h = sum_t p_t v_t / sum_t p_t,  p_t = exp(q_h . k_t / sqrt(hd) - max),  over the first positions + 1 rows of a sequence.
// A launch reads every key and value once for all query heads of its group and computes 4 g flops per number read, so the
// pages' bytes bound it; a short one is bound by what a launch, the plan and a trip to memory take.
//
// Work split.  The key tiles (16 rows of float32, 32 of 16-bit numbers: 8 KiB of K and 8 of V at head_dim 128) of all
// (row, kv head) pairs lie end to end and are cut into equal spans, one per workgroup, whatever the lengths; every workgroup
// makes the sums that tell it where its span lies from the lengths themselves, so that nothing of a launch depends on them
// but what it does, and a recorded one is good for any lengths.  The wavefronts of a workgroup take its tiles in turn, each with a
// softmax of its own (running maximum, sum and output), and merge through LDS.  A pair that several workgroups share leaves
// a part with each; the workgroup that adds its part last (a count per pair) adds them all up, in the order of the keys, so
// results do not depend on who that is, and nobody waits for anybody.
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
// scope write through and read past them.  A part is in memory before its count goes up (the wait for its stores).
__device__ __forceinline__ void coherent_store(float *p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float coherent_load(const float *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kCols = 16;  // query heads of a pair, at most: a larger group is several pairs
constexpr int kMaxWorkgroups = 1024;
// tiles of a span at least: a wavefront's first tile costs it a trip to memory, whose share this keeps down
constexpr int kLeastSpan = 2 * kWaves;

// What is laid out how for pages of a type and heads of up to HD.
template <int DTYPE, int HD>
struct Tile {
  static constexpr int E = DTYPE == kPageF32 ? 4 : 2;      // bytes of a number
  static constexpr int S = DTYPE == kPageF32 ? 1 : 2;      // sixteens of keys
  static constexpr int KEYS = 16 * S;
  static constexpr int CHUNKS = HD * E / 64;               // 16-byte pieces of a K row per lane
  static constexpr int PER = 16 / E;                       // numbers in one
  static constexpr int VEC = HD / 16 < PER ? HD / 16 : PER;  // neighbouring columns of a V row per lane
  static constexpr int PIECES = HD / (16 * VEC);           // ... how often
  static constexpr int WORDS = VEC * E / 4;                // of 4 bytes, in one
  static constexpr int PARTS = DTYPE == kPageF32 ? 1 : DTYPE == kPageBf16 ? 3 : 2;  // of a float operand
  static constexpr int PER_CU = HD == 64 ? 3 : HD == 128 ? 2 : 1;  // workgroups of a compute unit
};

template <int WORDS>
struct Words;
template <>
struct Words<2> {
  typedef u32x2 T;
};
template <>
struct Words<4> {
  typedef u32x4 T;
};

// Where the spans lie.
struct Plan {
  int total, span;
};

struct Segment {
  int row, seq, len, first, last;  // tiles [first, last) of the row's
  int head, cols;                  // query heads head .. head + cols - 1
  int kv;
  int begins, ends;                // of the pair's tiles in the stream
};

template <int DTYPE, int HD, bool PAD>
struct Wave {
  using T = Tile<DTYPE, HD>;
  typedef typename Words<T::WORDS>::T VWords;
  static constexpr int KEYS_EACH = 4 * T::S;  // of a quarter

  const PagePool &p;
  const int lane, m, j;
  const int hd;
  u32x4 k[T::S][T::CHUNKS];
  VWords v[KEYS_EACH][T::PIECES];
  u32x4 q[T::PARTS][DTYPE == kPageF32 ? T::CHUNKS : T::CHUNKS];
  f32x4 acc[T::PIECES][T::VEC];
  float top, sum;  // running maximum of the scores in log2 units, and this lane's share of the sum
  float c;         // scores to log2 units
  int down;        // float16: the queries were multiplied by 2^down
  // pages of this lane's K row and V rows in the tile to be asked for next, and whether those V rows, which are the keys of this lane's
  // scores, lie in the pool; of the tile in registers, too
  int k_page, v_page;
  bool v_in, v_in_next;
  const int *table;
  int last_page, len;
  const char *k_base, *v_base;

  __device__ __forceinline__ Wave(const PagePool &pool) : p(pool), lane(threadIdx.x & 63), m(lane & 15), j(lane >> 4), hd(PAD ? pool.hd : HD) {}

  __device__ __forceinline__ void look_up(int tile) {
    const int k0 = tile * T::KEYS;
    const int kp = table[min((k0 + (m >> 2) * KEYS_EACH) >> p.shift, last_page)];
    const int vp = table[min((k0 + j * KEYS_EACH) >> p.shift, last_page)];
    k_page = (unsigned)kp < (unsigned)p.n_pages ? kp : 0;
    v_in_next = (unsigned)vp < (unsigned)p.n_pages;
    v_page = v_in_next ? vp : 0;
  }

  __device__ __forceinline__ const char *row_at(const char *base, int page, int key) const {
    const long long row = ((long long)page * p.KV << p.shift) + (key & ((1 << p.shift) - 1));
    return base + row * (hd * T::E);
  }
  __device__ __forceinline__ void ask_k(int tile) {
#pragma unroll
    for (int s = 0; s < T::S; ++s) {
      const char *row = row_at(k_base, k_page, tile * T::KEYS + (m >> 2) * KEYS_EACH + 4 * s + (m & 3));
#pragma unroll
      for (int u = 0; u < T::CHUNKS; ++u) {
        int at = (u * 4 + j) * 16;
        if (PAD) at = at < hd * T::E ? at : 0;
        k[s][u] = __builtin_nontemporal_load((const u32x4 *)(row + at));
      }
    }
  }
  __device__ __forceinline__ void ask_v(int tile) {
    const char *row = row_at(v_base, v_page, tile * T::KEYS + j * KEYS_EACH);
#pragma unroll
    for (int r = 0; r < KEYS_EACH; ++r)
#pragma unroll
      for (int u = 0; u < T::PIECES; ++u) {
        int at = (T::VEC * m + 16 * T::VEC * u) * T::E;
        if (PAD) at = at < hd * T::E ? at : 0;
        v[r][u] = __builtin_nontemporal_load((const VWords *)(row + r * (hd * T::E) + at));
      }
    v_in = v_in_next;
  }

  // The queries as B operands: chunk u of quarter j is d = (4 u + j) PER .. + PER - 1, as K's.
  __device__ __forceinline__ void load_queries(const float *rows, int cols, float scale) {
    f32x4 x[T::CHUNKS][T::PER / 4];
    float most = 0.0f;
#pragma unroll
    for (int u = 0; u < T::CHUNKS; ++u)
#pragma unroll
      for (int w = 0; w < T::PER / 4; ++w) {
        const int d = (4 * u + j) * T::PER + 4 * w;
        x[u][w] = f32x4{0, 0, 0, 0};
        if (m < cols && (!PAD || d < hd))
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][w][e] = rows[m * hd + d + e];
        most = fmaxf(fmaxf(most, fmaxf(fabsf(x[u][w].x), fabsf(x[u][w].y))), fmaxf(fabsf(x[u][w].z), fabsf(x[u][w].w)));
      }
    c = scale * 1.44269504088896340736f;
    down = 0;
    if constexpr (DTYPE == kPageF16) {
      // two float16 parts hold 22 bits of a number, down to 2^-24: the largest of the row is brought to 2^14 .. 2^15
      most = max_across_quarters(most);
      down = most > 0.0f && most < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
    }
#pragma unroll
    for (int u = 0; u < T::CHUNKS; ++u) {
      if constexpr (DTYPE == kPageF32) {
        q[0][u] = __builtin_bit_cast(u32x4, x[u][0]);
      } else if constexpr (DTYPE == kPageBf16) {
        split_octet(x[u][0], x[u][1], q[0][u], q[1][u], q[2][u]);
      } else {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = ldexpf(x[u][e >> 2][e & 3], down);
        split_f16(y, q[0][u], q[1][u]);
      }
    }
  }
  __device__ __forceinline__ static void split_f16(const float (&y)[8], u32x4 &high, u32x4 &low) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x2 h = f16x2{(_Float16)y[2 * e], (_Float16)y[2 * e + 1]};
      high[e] = __builtin_bit_cast(unsigned, h);
      low[e] = __builtin_bit_cast(unsigned, f16x2{(_Float16)(y[2 * e] - (float)h.x), (_Float16)(y[2 * e + 1] - (float)h.y)});
    }
  }
  __device__ __forceinline__ static f32x4 mfma16(u32x4 a, u32x4 b, f32x4 x) {
    if constexpr (DTYPE == kPageBf16)
      return mfma_bf16_16(a, b, x);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), x, 0, 0, 0);
  }

  __device__ __forceinline__ void begin(const Segment &s) {
    len = s.len;
    table = p.table + (long long)s.seq * p.seq_pages;
    last_page = (len - 1) >> p.shift;
    const long long head = ((long long)s.kv << p.shift) * (hd * T::E);
    k_base = (const char *)p.k + head;
    v_base = (const char *)p.v + head;
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
      for (int e = 0; e < T::VEC; ++e) acc[u][e] = f32x4{0, 0, 0, 0};
  }

  // Tiles first, first + step, ... below last.
  __device__ __forceinline__ void walk(int first, int last, int step) {
    if (first >= last) return;
    look_up(first);
    ask_k(first);
    ask_v(first);
    if (first + step < last) look_up(first + step);
    for (int tile = first; tile < last; tile += step) {
      const int next = tile + step;
      f32x4 x[T::S];
#pragma unroll
      for (int s = 0; s < T::S; ++s) {
        x[s] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int part = T::PARTS - 1; part >= 0; --part)
#pragma unroll
          for (int u = 0; u < T::CHUNKS; ++u) {
            if constexpr (DTYPE == kPageF32) {
              const f32x4 a = __builtin_bit_cast(f32x4, k[s][u]), b = __builtin_bit_cast(f32x4, q[0][u]);
#pragma unroll
              for (int e = 0; e < 4; ++e) x[s] = mfma_f32_16(a[e], b[e], x[s]);
            } else {
              x[s] = mfma16(k[s][u], q[part][u], x[s]);
            }
          }
      }
      if (next < last) ask_k(next);
      if constexpr (DTYPE == kPageF16)
#pragma unroll
        for (int s = 0; s < T::S; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][i] = ldexpf(x[s][i], -down);
      // keys behind the sequence's end or in no page: no score, and a value that is no number would not vanish at weight 0
      const int key = tile * T::KEYS + j * KEYS_EACH;
      if (__any(!v_in || key + KEYS_EACH > len)) {
#pragma unroll
        for (int r = 0; r < KEYS_EACH; ++r)
          if (!v_in || key + r >= len) {
            x[r >> 2][r & 3] = -INFINITY;
#pragma unroll
            for (int u = 0; u < T::PIECES; ++u) v[r][u] = VWords{};
          }
      }
      float most = fmaxf(fmaxf(x[0].x, x[0].y), fmaxf(x[0].z, x[0].w));
      if constexpr (T::S == 2) most = fmaxf(most, fmaxf(fmaxf(x[1].x, x[1].y), fmaxf(x[1].z, x[1].w)));
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
      // (float16 parts of a weight: lifted by 2^15, as the queries are; the sum is lifted with them)
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
            const f32x4 columns = __builtin_bit_cast(f32x4, v[r][u]);
#pragma unroll
            for (int e = 0; e < T::VEC; ++e) acc[u][e] = mfma_f32_16(columns[e], w[r], acc[u][e]);
          }
      } else {
        u32x4 weights[T::PARTS];
        if constexpr (DTYPE == kPageBf16)
          split_octet(f32x4{w[0], w[1], w[2], w[3]}, f32x4{w[4], w[5], w[6], w[7]}, weights[0], weights[1], weights[2]);
        else
          split_f16(w, weights[0], weights[1]);
#pragma unroll
        for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
          for (int e = 0; e < T::VEC; ++e) {
            u32x4 column;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              column[r] = __builtin_amdgcn_perm(v[2 * r + 1][u][e >> 1], v[2 * r][u][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int part = T::PARTS - 1; part >= 0; --part) acc[u][e] = mfma16(column, weights[part], acc[u][e]);
          }
      }
      if (next < last) {
        ask_v(next);
        if (next + step < last) look_up(next + step);
      }
    }
  }
};

template <int DTYPE, int HD, bool PAD>
__global__ __launch_bounds__(kThreads, (Tile<DTYPE, HD>::PER_CU)) void paged_attend_kernel(PagedAttendArgs a, PagePool p) {
  using T = Tile<DTYPE, HD>;
  constexpr int STRIDE = HD + 4;
  __shared__ int starts[kMaxPagedSeqs + 1];                 // tiles of one kv head in the rows before
  __shared__ float outs[kWaves][kCols][STRIDE];
  __shared__ float tops[kWaves][kCols], sums[kWaves][kCols];
  __shared__ int scan[kWaves], last_one;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int hd = PAD ? p.hd : HD;
  const int g = a.H / p.KV, per_kv = (g + kCols - 1) / kCols, pairs = p.KV * per_kv;
  const int most_keys = (int)min((long long)p.seq_pages << p.shift, 0x3fffffffLL);

  // sums of the rows' tiles; outputs of rows without keys
  {
    const int each = (a.rows + kThreads - 1) / kThreads;
    int mine = 0;
    for (int i = 0; i < each; ++i) {
      const int r = t * each + i;
      int tiles = 0;
      if (r < a.rows && (unsigned)a.row_seqs[r] < (unsigned)p.n_seqs)
        tiles = (max(0, min(a.positions[r], most_keys - 1) + 1) + T::KEYS - 1) / T::KEYS;
      if (r < a.rows) starts[r] = mine;
      mine += tiles;
    }
    int inclusive = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(inclusive, d);
      if (lane >= d) inclusive += x;
    }
    if (lane == 63) scan[wave] = inclusive;
    __syncthreads();
    int before = inclusive - mine, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? scan[w] : 0;
      all += scan[w];
    }
    for (int i = 0; i < each; ++i) {
      const int r = t * each + i;
      if (r < a.rows) starts[r] += before;
    }
    if (t == 0) starts[a.rows] = all;
    __syncthreads();
  }
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x)
    if (starts[r + 1] == starts[r] && (unsigned)a.row_seqs[r] < (unsigned)p.n_seqs)
      for (int i = t; i < a.H * hd; i += kThreads) a.out[r * a.out_stride + i] = 0.0f;

  const long long total = (long long)starts[a.rows] * pairs;
  const long long span = max((long long)kLeastSpan, (total + gridDim.x - 1) / gridDim.x);
  long long at = blockIdx.x * span;
  const long long end = min(total, at + span);
  if (at >= end) return;
  int row;
  {
    int lo = 0, hi = a.rows - 1;
    while (lo < hi) {  // the last row that begins at or before it and has tiles
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)starts[mid] * pairs <= at)
        lo = mid;
      else
        hi = mid - 1;
    }
    row = lo;
  }
  unsigned *tickets = (unsigned *)a.workspace;
  float *parts = (float *)(tickets + kMaxWorkgroups);
  constexpr int PART = kCols * (HD + 2);  // a workgroup has two: of the pair that it begins with, and of the one that goes on behind it
  Wave<DTYPE, HD, PAD> w(p);
  while (at < end) {
    while (starts[row + 1] == starts[row] || (long long)starts[row + 1] * pairs <= at) ++row;
    row = __builtin_amdgcn_readfirstlane(row);
    Segment s;
    const int tiles = __builtin_amdgcn_readfirstlane(starts[row + 1] - starts[row]);
    const long long of_row = (long long)__builtin_amdgcn_readfirstlane(starts[row]) * pairs;
    const int pair = (int)((at - of_row) / tiles);
    const long long begins = of_row + (long long)pair * tiles, ends = begins + tiles;
    s.row = row;
    s.seq = a.row_seqs[row];
    s.len = min(a.positions[row], most_keys - 1) + 1;
    s.first = (int)(at - begins);
    s.last = (int)(min(end, ends) - begins);
    s.kv = pair / per_kv;
    s.head = s.kv * g + (pair - s.kv * per_kv) * kCols;
    s.cols = min(kCols, g - (pair - s.kv * per_kv) * kCols);
    w.begin(s);
    w.load_queries(a.q + s.row * a.q_stride + (long long)s.head * hd, s.cols, a.scale);
    w.walk(s.first + wave, s.last, kWaves);

    // the wavefronts' parts, on one maximum
    const float mine = sum_across_quarters(w.sum);
    if (lane < kCols) {
      tops[wave][lane] = w.top;
      sums[wave][lane] = mine;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, tops[i][w.m]);
    const float fade = w.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w.top - top);
#pragma unroll
    for (int u = 0; u < T::PIECES; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < T::VEC; ++e)
          outs[wave][w.m][T::VEC * (4 * w.j + i) + 16 * T::VEC * u + e] = w.acc[u][e][i] * fade;
    __syncthreads();
    const bool whole = begins == at && ends <= end;
    const long long first_wg = begins / span, last_wg = (ends - 1) / span;
    // (a pair that begins in a workgroup's span but not with it, and does not end there, is the span's last: its second part)
    auto part_of = [&](long long wg) { return parts + (wg * 2 + (wg == first_wg && begins != wg * span ? 1 : 0)) * PART; };
    float *part = part_of(blockIdx.x);
    for (int i = t; i < s.cols * hd; i += kThreads) {
      const int n = i / hd, d = i - n * hd;
      float x = 0.0f, l = 0.0f, best = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        x += outs[v][n][d];
        best = fmaxf(best, tops[v][n]);
      }
#pragma unroll
      for (int v = 0; v < kWaves; ++v) l += sums[v][n] * (tops[v][n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(tops[v][n] - best));
      if (whole) {
        a.out[s.row * a.out_stride + (long long)(s.head + n) * hd + d] = l == 0.0f ? 0.0f : x / l;
      } else {
        coherent_store(part + n * (HD + 2) + d, x);
        if (d == 0) {
          coherent_store(part + n * (HD + 2) + HD, best);
          coherent_store(part + n * (HD + 2) + HD + 1, l);
        }
      }
    }
    if (!whole) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t == 0) {
        const unsigned others = (unsigned)(last_wg - first_wg);
        const unsigned before = __hip_atomic_fetch_add(tickets + first_wg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_one = before == others;
        if (before == others) __hip_atomic_store(tickets + first_wg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (last_one) {
        for (int i = t; i < s.cols * hd; i += kThreads) {
          const int n = i / hd, d = i - n * hd;
          float best = -INFINITY;
          for (long long wg = first_wg; wg <= last_wg; ++wg) best = fmaxf(best, coherent_load(part_of(wg) + n * (HD + 2) + HD));
          float x = 0.0f, l = 0.0f;
          for (long long wg = first_wg; wg <= last_wg; ++wg) {
            const float *from = part_of(wg) + n * (HD + 2);
            const float its = coherent_load(from + HD), fades = its == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(its - best);
            x = fmaf(coherent_load(from + d), fades, x);
            l = fmaf(coherent_load(from + HD + 1), fades, l);
          }
          a.out[s.row * a.out_stride + (long long)(s.head + n) * hd + d] = l == 0.0f ? 0.0f : x / l;
        }
      }
    }
    __syncthreads();  // the next segment writes to LDS
    at += s.last - s.first;
  }
}

// Where the row of key t of a sequence lies in the pools; -1 where the table names no page.
__device__ __forceinline__ long long page_row(const PagePool &p, const int *table, int t, int head) {
  const int page = table[t >> p.shift];
  if ((unsigned)page >= (unsigned)p.n_pages) return -1;
  return (((long long)page * p.KV + head) << p.shift) + (t & ((1 << p.shift) - 1));
}

template <int DTYPE>
__global__ __launch_bounds__(256) void page_gather_kernel(PagePool p, int seq, int pos0, int n, int cap, float *k, float *v) {
  const int per = p.hd >> 2;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)n * p.KV * per) return;
  const int piece = (int)(i % per), t = (int)(i / per % n), c = (int)(i / per / n);
  const long long row = page_row(p, p.table + (long long)seq * p.seq_pages, pos0 + t, c);
  const long long to = ((long long)c * cap + t) * p.hd + 4 * piece;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (k) k[to + e] = row < 0 ? 0.0f : page_value<DTYPE>(p.k, row * p.hd + 4 * piece + e);
    if (v) v[to + e] = row < 0 ? 0.0f : page_value<DTYPE>(p.v, row * p.hd + 4 * piece + e);
  }
}

}  // namespace

size_t paged_attend_workspace(int hd) {
  const int tile = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
  return kMaxWorkgroups * sizeof(unsigned) + (size_t)kMaxWorkgroups * 2 * kCols * (tile + 2) * sizeof(float);
}

namespace {
template <int DTYPE, int HD>
hipError_t launch_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  constexpr int wgs = 256 * Tile<DTYPE, HD>::PER_CU;
  static_assert(wgs <= kMaxWorkgroups, "counts and parts");
  const auto kernel = p.hd == HD ? paged_attend_kernel<DTYPE, HD, false> : paged_attend_kernel<DTYPE, HD, true>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a, p);
  return hipGetLastError();
}
template <int DTYPE>
hipError_t launch_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  return p.hd <= 64 ? launch_attend<DTYPE, 64>(a, p, stream) : p.hd <= 128 ? launch_attend<DTYPE, 128>(a, p, stream) : launch_attend<DTYPE, 256>(a, p, stream);
}
}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  if (a.rows < 1 || a.rows > kMaxPagedSeqs || a.H < 1 || a.H % p.KV || (p.hd & 7) || p.hd < 8 || p.hd > 256 || p.shift < 3)
    return hipErrorInvalidValue;
  return p.dtype == kPageF32 ? launch_attend<kPageF32>(a, p, stream) : p.dtype == kPageBf16 ? launch_attend<kPageBf16>(a, p, stream) : launch_attend<kPageF16>(a, p, stream);
}

hipError_t launch_page_gather(const PagePool &p, int seq, int pos0, int n, int cap, float *k, float *v, hipStream_t stream) {
  if (n < 1) return hipSuccess;
  if (seq < 0 || seq >= p.n_seqs || pos0 < 0 || (long long)pos0 + n > (long long)p.seq_pages << p.shift || n > cap)
    return hipErrorInvalidValue;
  const long long blocks = ((long long)n * p.KV * (p.hd >> 2) + 255) / 256;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  const auto kernel = p.dtype == kPageF32    ? page_gather_kernel<kPageF32>
                      : p.dtype == kPageBf16 ? page_gather_kernel<kPageBf16>
                                             : page_gather_kernel<kPageF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, seq, pos0, n, cap, k, v);
  return hipGetLastError();
}

}  // namespace shainet
