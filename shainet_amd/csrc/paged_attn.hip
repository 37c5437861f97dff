// Attention of one new row per sequence over its pages, and pages back into one piece of memory.
#include "paged.hpp"

namespace shainet {

namespace {

constexpr int kTickets = 1024;

template <int DTYPE>
__device__ __forceinline__ float page_value(const void *pool, long long i) {
  if constexpr (DTYPE == kPageF32)
    return ((const float *)pool)[i];
  else if constexpr (DTYPE == kPageBf16)
    return (float)((const __bf16 *)pool)[i];
  else
    return (float)((const _Float16 *)pool)[i];
}

// Where the row of key t of a sequence lies in the pools; -1 where the table names no page.
__device__ __forceinline__ long long page_row(const PagePool &p, const int *table, int t, int head) {
  const int page = table[t >> p.shift];
  if ((unsigned)page >= (unsigned)p.n_pages) return -1;
  return (((long long)page * p.KV + head) << p.shift) + (t & ((1 << p.shift) - 1));
}

// A workgroup per query head and row, a key per thread, then a dimension per thread.
template <int DTYPE>
__global__ __launch_bounds__(256) void paged_attend_kernel(PagedAttendArgs a, PagePool p) {
  __shared__ float q[256], weight[256], most[4], sum[4];
  __shared__ long long at[256];
  const int t = threadIdx.x, h = blockIdx.x, r = blockIdx.y, c = h / (a.H / p.KV);
  const int seq = a.row_seqs[r];
  if ((unsigned)seq >= (unsigned)p.n_seqs) return;
  const long long reach = (long long)p.seq_pages << p.shift;
  const int len = (int)min((long long)a.positions[r] + 1, reach);
  const int *table = p.table + (long long)seq * p.seq_pages;
  if (t < p.hd) q[t] = a.q[r * a.q_stride + h * p.hd + t] * a.scale;
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int k0 = 0; k0 < len; k0 += 256) {
    __syncthreads();
    float s = -INFINITY;
    long long row = -1;
    if (k0 + t < len) {
      row = page_row(p, table, k0 + t, c);
      if (row >= 0) {
        s = 0.0f;
        for (int d = 0; d < p.hd; ++d) s = fmaf(q[d], page_value<DTYPE>(p.k, row * p.hd + d), s);
      }
    }
    at[t] = row;
    float best = s;
    for (int d = 32; d; d >>= 1) best = fmaxf(best, __shfl_xor(best, d));
    if ((t & 63) == 0) most[t >> 6] = best;
    __syncthreads();
    best = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    const float now = fmaxf(m, best), from = now == -INFINITY ? 0.0f : now;
    const float e = expf(s - from);
    weight[t] = e;
    float total = e;
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    if ((t & 63) == 0) sum[t >> 6] = total;
    __syncthreads();
    const float fade = expf(m - from);
    l = l * fade + (sum[0] + sum[1] + sum[2] + sum[3]);
    o *= fade;
    m = now;
    if (t < p.hd)
      for (int i = 0; i < min(256, len - k0); ++i)
        if (at[i] >= 0) o = fmaf(weight[i], page_value<DTYPE>(p.v, at[i] * p.hd + t), o);
  }
  if (t < p.hd) a.out[r * a.out_stride + h * p.hd + t] = l > 0.0f ? o / l : 0.0f;
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

size_t paged_attend_workspace(int hd) { return kTickets * sizeof(unsigned); }

hipError_t launch_paged_attend(const PagedAttendArgs &a, const PagePool &p, hipStream_t stream) {
  if (a.rows < 1 || a.rows > kMaxPagedSeqs || a.H < 1 || a.H % p.KV || (p.hd & 7) || p.hd < 8 || p.hd > 256) return hipErrorInvalidValue;
  const auto kernel = p.dtype == kPageF32    ? paged_attend_kernel<kPageF32>
                      : p.dtype == kPageBf16 ? paged_attend_kernel<kPageBf16>
                                             : paged_attend_kernel<kPageF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.H, (unsigned)a.rows), dim3(256), 0, stream, a, p);
  return hipGetLastError();
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
