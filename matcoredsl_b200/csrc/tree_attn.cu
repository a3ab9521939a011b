// Attention of a tree of drafted tokens over a paged key/value cache, on CUDA
// cores: any element type, head size up to 256, strides and alignment.
//
// Request b's new tokens i = 0 .. n-1 sit at the end of its kv_len keys, token
// i at position P + i with P = kv_len - n. Row i sees every key before P, and
// of the new ones those whose bit is set in its mask row (without a mask:
// j <= i). o = sum_j p_j v_j / l, p_j = exp(scale q.k_j - m), l = sum_j p_j,
// lse = m + log l; a row that sees nothing gives o = 0, lse = -inf.
//
// One CTA (4 warps) per token, key head, group of kRows query heads and slice
// of the keys. A warp takes 32 keys at a time: each lane computes kRows dot
// products with its own key, the softmax runs across the lanes with one running
// maximum and sum a row, then the lanes turn to the value rows, one element
// slice each. Keys that the token does not see are skipped, never multiplied by
// zero, so infinities and NaN in their values do not reach it.
//
// Bound: instructions (a value or key element costs a conversion and kRows products a
// lane), then L2, since every group of rows reads the keys again. f32, 8 requests of
// up to 8192 keys, 8 key heads of 128, 4 rows each: 132 us, 302 MB at 2.3 TB/s. Several
// tokens in a CTA's rows, each with its own visibility, halved 150 causal tokens of one
// request (72 to 41 us) but cost single tokens 70% (227 us) and drafts 20 to 70%. Two
// warps a CTA: 146 us (but 121 against 193 for 126 requests of up to 54 keys).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_SPLITS = 64;  // two a lane when they are joined
constexpr int MIN_KEYS = 128;  // keys a slice is worth a CTA for (64: shorter contexts lose)

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}

// CTAs an SM whose registers the compiler keeps to, 0: its own choice. f32, four heads of up to 128: 5 (without,
// decoding of 8 requests 141 us instead of 132, of 64 696 instead of 627). The same bound in
// 16 bits: 16 requests of head size 80 123 us instead of 95.
template <typename T, int kRows, int kCols>
constexpr int min_ctas() {
  return sizeof(T) == 4 && kRows == 4 && kCols == 4 ? 5 : 0;
}

// kRows query heads of one token; kCols = elements of a head per lane.
template <typename T, int kRows, int kCols>
__global__ void __launch_bounds__(THREADS, min_ctas<T, kRows, kCols>())
    tree_attn_simt_kernel(const TreeAttn p, float *partial, int splits, int vec) {
  extern __shared__ __align__(16) float smem[];
  float *qs = smem;                                     // [kRows][dim]
  float *red = smem + kRows * p.dim;                    // [WARPS][kRows][dim + 2]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = p.heads / p.kv_heads;
  const int groups = (group + kRows - 1) / kRows;
  const int64_t t = blockIdx.x;
  const int hk = blockIdx.y / groups, g0 = (blockIdx.y - hk * groups) * kRows;
  const int rows = min(kRows, group - g0);
  const int h0 = hk * group + g0;  // first query head
  const T *q = static_cast<const T *>(p.q) + t * p.q_s[0] + h0 * p.q_s[1];
  // The request that token t belongs to, looked for by all threads while the query is read.
  // Where cu_new descends, no token belongs to a request; that is why all of it is read and
  // not searched (for 2000 requests of up to 30 keys, f32, two heads of 64, 24 us
  // instead of 20.5; nothing to see at 100 requests or 100 keys).
  __shared__ int32_t owner;
  int32_t mine = -1;
  bool descends = false;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < p.requests; r += THREADS) {
    const int32_t c0 = p.cu[r], c1 = p.cu[r + 1];
    descends |= c1 < c0;
    if (c0 <= t && t < c1) mine = static_cast<int32_t>(r);
  }
  if (threadIdx.x == 0) owner = -1;
  for (int i = threadIdx.x; i < kRows * p.dim; i += THREADS) {
    const int r = i / p.dim, d = i - r * p.dim;
    qs[i] = r < rows ? to_f32(q[r * p.q_s[1] + d]) * p.scale : 0.0f;
  }
  __syncthreads();
  if (mine >= 0) owner = mine;
  descends = __syncthreads_or(descends) != 0;
  float m[kRows], l[kRows], acc[kRows][kCols];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[r][c] = 0.0f;
  }
  const int32_t b = __shfl_sync(0xffffffffu, descends ? -1 : owner, 0);
  if (b >= 0) {
    const int64_t i = t - p.cu[b], n = p.cu[b + 1] - p.cu[b];
    const int64_t kv = max(0, p.kv_lens[b]), prefix = kv - n;
    const int64_t keys = min(kv, p.columns * p.block);
    const int64_t per = ((keys + splits - 1) / splits + 31) / 32 * 32;
    const int64_t first = per * blockIdx.z, last = min(keys, first + per);
    for (int64_t k0 = first + warp * 32; k0 < last; k0 += WARPS * 32) {
      const int64_t pos = k0 + lane;
      bool visible = pos < last;
      int64_t ko = 0, vo = 0;
      if (visible) {
        const int64_t col = pos / p.block, off = pos - col * p.block;
        const int32_t blk = p.table[b * p.table_stride + col];
        visible = blk >= 0 && blk < p.blocks;
        const int64_t j = pos - prefix;
        if (visible && j >= 0)
          visible = p.mask ? (j >> 5) < p.mask_words &&
                                 ((p.mask[t * p.mask_stride + (j >> 5)] >> (j & 31)) & 1u)
                           : j <= i;
        ko = blk * p.k_s[0] + off * p.k_s[1] + hk * p.k_s[2];
        vo = blk * p.v_s[0] + off * p.v_s[1] + hk * p.v_s[2];
      }
      const uint32_t seen = __ballot_sync(0xffffffffu, visible);
      if (seen == 0) continue;
      float s[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) s[r] = 0.0f;
      if (visible) {
        const T *k = static_cast<const T *>(p.k) + ko;
        if (vec) {  // rows that can be read 16 bytes at a time
          constexpr int VE = 16 / sizeof(T);
#pragma unroll 8
          for (int d = 0; d < p.dim; d += VE) {
            const uint4 w = *reinterpret_cast<const uint4 *>(k + d);
            const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int e = 0; e < VE; e += 4) {
              const float x0 = to_f32(x[e]), x1 = to_f32(x[e + 1]);
              const float x2 = to_f32(x[e + 2]), x3 = to_f32(x[e + 3]);
#pragma unroll
              for (int r = 0; r < kRows; ++r) {
                const float4 q4 = *reinterpret_cast<const float4 *>(qs + r * p.dim + d + e);
                s[r] = fmaf(q4.w, x3, fmaf(q4.z, x2, fmaf(q4.y, x1, fmaf(q4.x, x0, s[r]))));
              }
            }
          }
        } else {
          for (int d = 0; d < p.dim; ++d) {
            const float x = to_f32(k[d]);
#pragma unroll
            for (int r = 0; r < kRows; ++r) s[r] = fmaf(qs[r * p.dim + d], x, s[r]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (!visible) s[r] = -INFINITY;
        float mx = s[r];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        mx = fmaxf(mx, m[r]);
        // A row whose scores are all -inf (or NaN) so far: keep exponents defined.
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float f = expf(m[r] - ref);
        s[r] = visible ? expf(s[r] - ref) : 0.0f;
        float sum = s[r];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l[r] = l[r] * f + sum;
        m[r] = mx;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[r][c] *= f;
      }
      // The values of kMany keys on their way at a time; a key that is not seen
      // is not read and counts 0 x 0.
      constexpr int kMany = kCols >= 8 ? 4 : 8;
#pragma unroll 1
      for (int j0 = 0; j0 < 32; j0 += kMany) {
        if (((seen >> j0) & ((1u << kMany) - 1)) == 0) continue;
        float x[kMany][kCols];
#pragma unroll
        for (int u = 0; u < kMany; ++u) {
          const T *v = static_cast<const T *>(p.v) + __shfl_sync(0xffffffffu, vo, j0 + u);
          const bool bit = (seen >> (j0 + u)) & 1u;
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            x[u][c] = bit && c * 32 + lane < p.dim ? to_f32(v[c * 32 + lane]) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kMany; ++u)
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float w = __shfl_sync(0xffffffffu, s[r], j0 + u);
#pragma unroll
            for (int c = 0; c < kCols; ++c) acc[r][c] = fmaf(w, x[u][c], acc[r][c]);
          }
      }
    }
  }
  // Join the warps, in their order.
  const int stride = p.dim + 2;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float *out = red + (warp * kRows + r) * stride;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (c * 32 + lane < p.dim) out[c * 32 + lane] = acc[r][c];
    if (lane == 0) {
      out[p.dim] = m[r];
      out[p.dim + 1] = l[r];
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += WARPS) {
    float mx = -INFINITY;
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, red[(w * kRows + r) * stride + p.dim]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float f[WARPS], sum = 0.0f;
    for (int w = 0; w < WARPS; ++w) {
      const float *in = red + (w * kRows + r) * stride;
      f[w] = expf(in[p.dim] - ref);
      sum += in[p.dim + 1] * f[w];
    }
    const int64_t row = t * p.heads + h0 + r;
    float *part = partial ? partial + (row * splits + blockIdx.z) * stride : nullptr;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T *o = static_cast<T *>(p.o) + t * p.o_s[0] + (h0 + r) * p.o_s[1];
    for (int d = lane; d < p.dim; d += 32) {
      float x = 0.0f;
      for (int w = 0; w < WARPS; ++w) {
        const float *in = red + (w * kRows + r) * stride;
        if (in[p.dim + 1] != 0.0f) x = fmaf(in[d], f[w], x);
      }
      if (part)
        part[d] = x;
      else
        o[d] = static_cast<T>(x * inv);
    }
    if (lane == 0) {
      if (part) {
        part[p.dim] = mx;
        part[p.dim + 1] = sum;
      } else if (p.lse) {
        p.lse[t * p.lse_s + h0 + r] = sum == 0.0f ? -INFINITY : ref + logf(sum);
      }
    }
  }
}

// Joins the key slices of a row, in their order: one warp a row.
template <typename T>
__global__ void __launch_bounds__(256) tree_attn_join_kernel(const TreeAttn p, const float *partial,
                                                             int splits) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= p.tokens * p.heads) return;
  const int64_t t = row / p.heads, h = row - t * p.heads;
  const int stride = p.dim + 2;
  const float *in = partial + row * splits * stride;
  // Slices z = lane and lane + 32: their maxima and sums, and what they weigh.
  float m[2], l[2], w[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int z = lane + 32 * u;
    m[u] = z < splits ? in[z * stride + p.dim] : -INFINITY;
    l[u] = z < splits ? in[z * stride + p.dim + 1] : 0.0f;
  }
  float mx = fmaxf(m[0], m[1]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
  for (int u = 0; u < 2; ++u) w[u] = expf(m[u] - ref);
  float sum = l[0] * w[0] + l[1] * w[1];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T *o = static_cast<T *>(p.o) + t * p.o_s[0] + h * p.o_s[1];
  for (int d0 = 0; d0 < p.dim; d0 += 32) {
    const int d = d0 + lane;
    float x = 0.0f;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) {
      const float f = __shfl_sync(0xffffffffu, z < 32 ? w[0] : w[1], z & 31);
      x = fmaf(d < p.dim ? in[z * stride + d] : 0.0f, f, x);
    }
    if (d < p.dim) o[d] = static_cast<T>(x * inv);
  }
  if (lane == 0 && p.lse)
    p.lse[t * p.lse_s + h] = sum == 0.0f ? -INFINITY : ref + logf(sum);
}

int rows_of(const TreeAttn &p) {
  const int group = p.heads / p.kv_heads;
  return group == 1 ? 1 : group <= 4 ? 4 : 8;
}

int splits_of(const TreeAttn &p, int sms) {
  const int group = p.heads / p.kv_heads, r = rows_of(p);
  const int64_t units = p.tokens * p.kv_heads * ((group + r - 1) / r);
  int64_t s = units > 0 ? 8 * sms / units : 1;
  const int64_t most = p.columns * p.block / MIN_KEYS;
  s = s < most ? s : most;
  s = s < MAX_SPLITS ? s : MAX_SPLITS;
  return s < 1 ? 1 : static_cast<int>(s);
}

template <typename T, int kRows, int kCols>
cudaError_t run(const TreeAttn &p, float *scratch, int splits, cudaStream_t stream) {
  const int group = p.heads / p.kv_heads;
  const dim3 grid(static_cast<unsigned>(p.tokens),
                  static_cast<unsigned>(p.kv_heads * ((group + kRows - 1) / kRows)),
                  static_cast<unsigned>(splits));
  const size_t smem = sizeof(float) * (kRows * p.dim + WARPS * kRows * (p.dim + 2));
  static_assert(sizeof(float) * (8 * 256 + WARPS * 8 * 258) <= 48 * 1024, "no opt-in needed");
  constexpr int VE = 16 / sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(p.k) % 16 == 0 &&
                   (p.dim | p.k_s[0] | p.k_s[1] | p.k_s[2]) % VE == 0;
  tree_attn_simt_kernel<T, kRows, kCols><<<grid, THREADS, smem, stream>>>(
      p, splits > 1 ? scratch : nullptr, splits, vec ? 1 : 0);
  if (splits > 1)
    tree_attn_join_kernel<T><<<static_cast<unsigned>((p.tokens * p.heads + 7) / 8), 256, 0,
                               stream>>>(p, scratch, splits);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_type(const TreeAttn &p, float *scratch, int splits, cudaStream_t stream) {
  const int r = rows_of(p);
  auto cols = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    return p.dim <= 64    ? run<T, R, 2>(p, scratch, splits, stream)
           : p.dim <= 128 ? run<T, R, 4>(p, scratch, splits, stream)
                          : run<T, R, 8>(p, scratch, splits, stream);
  };
  if (r == 1) return cols(std::integral_constant<int, 1>{});
  if (r == 4) return cols(std::integral_constant<int, 4>{});
  return cols(std::integral_constant<int, 8>{});
}

}  // namespace

uint64_t tree_attn_simt_scratch(const TreeAttn &p, int sms) {
  const int splits = splits_of(p, sms);
  if (splits == 1) return 0;
  return static_cast<uint64_t>(p.tokens) * p.heads * splits * (p.dim + 2) * sizeof(float);
}

cudaError_t launch_tree_attn_simt(const TreeAttn &p, int dtype, float *scratch, int sms,
                                  cudaStream_t stream, LaunchInfo *info) {
  const int group = p.heads / p.kv_heads, r = rows_of(p);
  const int64_t gy = static_cast<int64_t>(p.kv_heads) * ((group + r - 1) / r);
  if (p.dim > 256 || p.tokens > 0x7fffffff || gy > 65535 ||
      (p.tokens * p.heads + 7) / 8 > 0x7fffffff)
    return cudaErrorNotSupported;
  const int splits = splits_of(p, sms);
  cudaError_t e;
  if (dtype == MCB_DTYPE_F32)
    e = run_type<float>(p, scratch, splits, stream);
  else if (dtype == MCB_DTYPE_F16)
    e = run_type<__half>(p, scratch, splits, stream);
  else
    e = run_type<__nv_bfloat16>(p, scratch, splits, stream);
  info->launches = splits > 1 ? 2 : 1;
  info->tile_m = r;
  info->tile_n = 32;
  info->ctas = static_cast<int>(p.tokens * gy * splits);
  info->set_route("simt_tree_attention");
  return e;
}

}  // namespace mcb
