// bias -> per-head QK-RMSNorm -> half-split RoPE of new rows, as prep_kernel.hip does them (the same arithmetic in the same
// order, so rows in float32 pages are bit-identical to those of a shainet_kv_cache), with the K and V rows put where a map of
// slots says and rounded to the pages' type there, once, to the nearest (ties to even).
//
// Bound by the rows' bytes where there are many (2048 rows of 32 heads of 128 on 8 kv heads into bfloat16 pages: 46 MB in 9.3 us,
// as fast as a copy), by a launch and two trips to memory, slot and row, where there are few (333 rows 4.0 us, 16 rows with QK-norm 5.3),
// and with QK-norm by the squares of a row, which are added one after the other as the contiguous cache's are, of many rows by 16 lanes of a
// workgroup: 1400 rows 28 us | 12.8 without.
// This file is compiled with -ffp-contract=off: no product may fuse into an add.
#include "paged.hpp"
#include "prep_math.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#pragma clang fp contract(off)

namespace shainet {

namespace {

struct PagedRow {
  const float *src, *bias, *w;
  void *dst;
  int pos, dtype;
  bool rotate, valid;
};

// Head row r of a token: the H query heads, then the KV key heads, then the KV value heads.
__device__ __forceinline__ PagedRow locate(const PrepArgs &a, const PagePool &p, int H, const int *slots, const int *positions,
                                           int rope_positions, const MappedRows &mapped, int token, int r) {
  PagedRow rr;
  const int slot = slots[token], hd = p.hd;
  const bool gone = *mapped.epoch != *mapped.rows_epoch;  // (asked for with the slot: no trip of its own)
  rr.pos = positions[token];
  const bool outside = (unsigned)slot >= (unsigned)p.n_pages << p.shift;
  rr.valid = !gone && r < H + 2 * p.KV && !outside && (unsigned)rr.pos < (unsigned)rope_positions;
  // (rows of a map that could not be made have positions -1, too)
  if (mapped.row_seqs && r == 0 && rr.pos >= 0 && (gone || outside || rr.pos >= rope_positions)) {
    mapped.row_seqs[token] = -1;
    *(volatile int *)mapped.error = gone ? kRowsGone : outside ? kRowsOutside : kRowsFar;
  }
  rr.rotate = true;
  rr.dtype = kPageF32;
  rr.src = rr.bias = rr.w = nullptr;
  rr.dst = nullptr;
  if (!rr.valid) return rr;
  if (r < H) {
    rr.src = a.q + (long long)token * a.q_stride + r * hd;
    rr.bias = a.b_q ? a.b_q + r * hd : nullptr;
    rr.w = a.q_norm;
    rr.dst = a.q_rot + (long long)token * H * hd + r * hd;
    return rr;
  }
  const bool is_v = r - H >= p.KV;
  const int c = is_v ? r - H - p.KV : r - H;
  const long long row = (((long long)(slot >> p.shift) * p.KV + c) << p.shift) + (slot & ((1 << p.shift) - 1));
  rr.src = is_v ? a.v + (long long)token * a.v_stride + c * hd : a.k + (long long)token * a.k_stride + c * hd;
  const float *bias = is_v ? a.b_v : a.b_k;
  rr.bias = bias ? bias + c * hd : nullptr;
  rr.w = is_v ? nullptr : a.k_norm;
  rr.rotate = !is_v;
  rr.dtype = p.dtype;
  rr.dst = (char *)(is_v ? p.v : p.k) + row * hd * (p.dtype == kPageF32 ? 4 : 2);
  return rr;
}

__device__ __forceinline__ void store_element(void *dst, int dtype, int i, float x) {
  if (dtype == kPageF32)
    ((float *)dst)[i] = x;
  else if (dtype == kPageBf16)
    ((__bf16 *)dst)[i] = (__bf16)x;
  else
    ((_Float16 *)dst)[i] = (_Float16)x;
}
__device__ __forceinline__ void store_quad(void *dst, int dtype, int i, float4 x) {
  if (dtype == kPageF32) {
    *(float4 *)((float *)dst + i) = x;
  } else if (dtype == kPageBf16) {
    typedef __bf16 quad __attribute__((ext_vector_type(4)));
    *(quad *)((__bf16 *)dst + i) = quad{(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w};
  } else {
    typedef _Float16 quad __attribute__((ext_vector_type(4)));
    *(quad *)((_Float16 *)dst + i) = quad{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
  }
}

// head_dim up to 128: a wavefront per head row, lane i < hd / 2 owns the pair (i, i + hd / 2).
__global__ __launch_bounds__(256) void paged_rows_kernel(PrepArgs a, PagePool p, int H, const int *__restrict__ slots,
                                                         const int *__restrict__ positions, int rope_positions, MappedRows mapped) {
  const int lane = threadIdx.x & 63, hd = p.hd, half = hd >> 1;
  const PagedRow rr = locate(a, p, H, slots, positions, rope_positions, mapped, blockIdx.y, blockIdx.x * 4 + (threadIdx.x >> 6));
  if (!rr.valid) return;  // uniform over the wavefront
  const bool active = lane < half;
  const int i = active ? lane : 0;
  float x0 = rr.src[i], x1 = rr.src[i + half];
  if (rr.bias) {
    x0 = x0 + rr.bias[i];
    x1 = x1 + rr.bias[i + half];
  }
  if (rr.rotate) {
    const float w0 = rr.w ? rr.w[i] : 1.0f, w1 = rr.w ? rr.w[i + half] : 1.0f;
    const float2 cs = a.rope_tab[(long long)rr.pos * half + i];
    float y0, y1;
    norm_rotate_pair(x0, x1, rr.w != nullptr, w0, w1, a.eps, hd, half, cs, y0, y1);
    x0 = y0;
    x1 = y1;
  }
  if (active) {
    store_element(rr.dst, rr.dtype, i, x0);
    store_element(rr.dst, rr.dtype, i + half, x1);
  }
}

// Many head rows without QK-norm: a lane takes four neighbouring pairs of a head row with 16-byte accesses.
__global__ __launch_bounds__(256) void paged_rows_vec_kernel(PrepArgs a, PagePool p, int H, const int *__restrict__ slots,
                                                             const int *__restrict__ positions, int rope_positions,
                                                             MappedRows mapped, long long n_items) {
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  if (idx >= n_items) return;
  const int half = p.hd >> 1, tpr = half >> 2, rows = H + 2 * p.KV;
  const int j = (int)(idx % tpr);
  const long long row_g = idx / tpr;
  const int token = (int)(row_g / rows);
  const PagedRow rr = locate(a, p, H, slots, positions, rope_positions, mapped, token, (int)(row_g - (long long)token * rows));
  if (!rr.valid) return;
  const int i0 = 4 * j;
  float4 x0 = *(const float4 *)(rr.src + i0), x1 = *(const float4 *)(rr.src + half + i0);
  if (rr.bias) {
    const float4 b0 = *(const float4 *)(rr.bias + i0), b1 = *(const float4 *)(rr.bias + half + i0);
    x0 = float4{x0.x + b0.x, x0.y + b0.y, x0.z + b0.z, x0.w + b0.w};
    x1 = float4{x1.x + b1.x, x1.y + b1.y, x1.z + b1.z, x1.w + b1.w};
  }
  if (rr.rotate) {
    const float4 *cs = (const float4 *)(a.rope_tab + (long long)rr.pos * half + i0);
    const float4 cs01 = cs[0], cs23 = cs[1];  // (cos, sin) of pairs i0, i0 + 1 and i0 + 2, i0 + 3
    auto turn = [](float &u, float &v, float c, float s) {
      const float p0 = u * c, p1 = v * s, p2 = v * c, p3 = u * s;
      u = p0 - p1;
      v = p2 + p3;
    };
    turn(x0.x, x1.x, cs01.x, cs01.y);
    turn(x0.y, x1.y, cs01.z, cs01.w);
    turn(x0.z, x1.z, cs23.x, cs23.y);
    turn(x0.w, x1.w, cs23.z, cs23.w);
  }
  store_quad(rr.dst, rr.dtype, i0, x0);
  store_quad(rr.dst, rr.dtype, half + i0, x1);
}

// Any head_dim and alignment, and many rows with QK-norm: ROWS head rows of a workgroup go through LDS; one lane per row adds
// up its squares in the reference's order (row stride hd + 1 floats: no bank conflicts).
template <int ROWS>
__global__ __launch_bounds__(256) void paged_rows_lds_kernel(PrepArgs a, PagePool p, int H, const int *__restrict__ slots,
                                                             const int *__restrict__ positions, int rope_positions,
                                                             MappedRows mapped, long long n_rows) {
  extern __shared__ float xs[];  // [ROWS][hd + 1]
  __shared__ PagedRow row_s[ROWS];
  __shared__ float inv_s[ROWS];
  const int hd = p.hd, half = hd >> 1, stride = hd + 1, per_token = H + 2 * p.KV, t = threadIdx.x;
  if (t < ROWS) {
    const long long row_g = (long long)blockIdx.x * ROWS + t;
    PagedRow rr;
    rr.valid = false;
    if (row_g < n_rows) {
      const int token = (int)(row_g / per_token);
      rr = locate(a, p, H, slots, positions, rope_positions, mapped, token, (int)(row_g - (long long)token * per_token));
    }
    row_s[t] = rr;
  }
  __syncthreads();
  for (int idx = t; idx < ROWS * hd; idx += 256) {
    const int r = idx / hd, d = idx - r * hd;
    float x = 0.0f;
    if (row_s[r].valid) {
      x = row_s[r].src[d];
      const float *bias = row_s[r].bias;
      if (bias) x = x + bias[d];
    }
    xs[r * stride + d] = x;
  }
  __syncthreads();
  if (t < ROWS && row_s[t].valid && row_s[t].w) {  // llama_block.cr:626-633
    const float *row = xs + t * stride;
    float ss = 0.0f;
#pragma unroll 8
    for (int d = 0; d < hd; ++d) {
      const float v = row[d];
      const float sq = v * v;
      ss = ss + sq;
    }
    const float mean = ss / (float)hd;
    inv_s[t] = (float)(1.0 / sqrt((double)mean + a.eps));
  }
  __syncthreads();
  for (int idx = t; idx < ROWS * half; idx += 256) {
    const int r = idx / half, i = idx - r * half;
    if (!row_s[r].valid) continue;
    float x0 = xs[r * stride + i], x1 = xs[r * stride + i + half];
    if (row_s[r].rotate) {
      const float *w = row_s[r].w;
      if (w) {  // 636
        const float inv = inv_s[r];
        x0 = x0 * inv;
        x0 = x0 * w[i];
        x1 = x1 * inv;
        x1 = x1 * w[i + half];
      }
      const float2 cs = a.rope_tab[(long long)row_s[r].pos * half + i];
      const float p0 = x0 * cs.x, p1 = x1 * cs.y, p2 = x1 * cs.x, p3 = x0 * cs.y;
      x0 = p0 - p1;
      x1 = p2 + p3;
    }
    store_element(row_s[r].dst, row_s[r].dtype, i, x0);
    store_element(row_s[r].dst, row_s[r].dtype, i + half, x1);
  }
}

}  // namespace

hipError_t launch_paged_append(const PrepArgs &a, const PagePool &p, int H, const int *slots, const int *positions,
                               int rope_positions, int rows, const MappedRows &mapped, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  if ((p.hd & 7) || p.hd < 8 || p.hd > 256) return hipErrorInvalidValue;
  const int per_token = H + 2 * p.KV;
  const long long n_rows = (long long)rows * per_token;
  const auto aligned16 = [](const void *x) { return ((uintptr_t)x & 15) == 0; };
  const bool vec = !a.q_norm && !a.k_norm && ((a.q_stride | a.k_stride | a.v_stride) & 3) == 0 && aligned16(a.q) && aligned16(a.k) &&
                   aligned16(a.v) && aligned16(a.q_rot) && aligned16(p.k) && aligned16(p.v) && aligned16(a.b_q) && aligned16(a.b_k) &&
                   aligned16(a.b_v) && aligned16(a.rope_tab);
  // Few head rows take a wavefront each.  Of many, four pairs a lane move the bytes in fewer requests, and 16 rows in LDS add up their
  // squares side by side.  us a call, 48 head rows of 128 a token: without QK-norm 700 tokens 9.3 | 6.7 by four pairs, 170 as good; with
  // it 85 tokens 7.0 | 8.1 by LDS, 170 10.7 | 8.8, 1400 60 | 28.
  constexpr int kFewRows = 6144;
  // Heads over 128, of which a wavefront has no pair a lane: without QK-norm four pairs a lane, 1 to 180 rows of 24 heads of 256 2.5 to 3.5 us |
  // by LDS 9.5 to 11.1; with it by LDS, whatever the rows.
  if (vec && (n_rows >= kFewRows || p.hd > 128)) {
    const long long n_items = n_rows * (p.hd >> 3), blocks = (n_items + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL(paged_rows_vec_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a, p, H, slots, positions,
                       rope_positions, mapped, n_items);
    return hipGetLastError();
  }
  if (p.hd <= 128 && n_rows < kFewRows && rows <= 65535) {
    hipLaunchKernelGGL(paged_rows_kernel, dim3((unsigned)((per_token + 3) / 4), (unsigned)rows), dim3(256), 0, stream, a, p, H, slots,
                       positions, rope_positions, mapped);
    return hipGetLastError();
  }
  constexpr int kRows = 16;
  const long long blocks = (n_rows + kRows - 1) / kRows;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(paged_rows_lds_kernel<kRows>, dim3((unsigned)blocks), dim3(256), (size_t)kRows * (p.hd + 1) * sizeof(float),
                     stream, a, p, H, slots, positions, rope_positions, mapped, n_rows);
  return hipGetLastError();
}

}  // namespace shainet
