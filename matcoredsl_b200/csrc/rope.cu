// Rotary positions with several axes, and the append of K and V rows to a
// paged cache.
//
// Pair i of a head's first 2R elements, (a, b) = (x[i], x[R + i]) or, for the
// paired layout, (x[2i], x[2i + 1]), turns by the angle of its axis' position:
//   a' = a cos - b sin,  b' = b cos + a sin,
//   cos, sin = table[position[axis(i), t], i], table[position[axis(i), t], R + i]
// in f32, rounded once to the tensor's type. Elements past 2R are copied. The
// inverse (sin -> -sin) is the rotation's gradient. In the append form the
// turned K rows and the V rows go to the cache's slot of their token.
//
// Bound: HBM (q, k, v read once, q and the cache rows written once, the table's
// rows of the tokens' positions read once).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

// The cache row of `slot`, or nullptr when it lies outside the cache.
template <typename T>
__device__ __forceinline__ T *cache_row(T *base, const RopeParams &p, const int64_t *s,
                                        int32_t slot) {
  if (slot < 0 || slot >= p.cache_slots) return nullptr;
  const int32_t blk = slot / p.block;
  return base + blk * s[0] + (slot - blk * p.block) * s[1];
}

// cos and sin of pair i for token t; NaN where the position is outside the table.
__device__ __forceinline__ void angle(const RopeParams &p, int64_t t, int i, float &c, float &s) {
  const int32_t pos = p.positions[p.axis[i] * p.pos_stride + t];
  if (pos < 0 || pos >= p.table_rows) {
    c = s = __int_as_float(0x7fffffff);
    return;
  }
  const float *row = p.cos_sin + pos * p.table_stride;
  c = row[i];
  s = p.inverse ? -row[p.pairs + i] : row[p.pairs + i];
}

// One element pair (or one copied element) per thread: any strides, any
// alignment, any sizes.
template <typename T>
__global__ void __launch_bounds__(256) rope_plain_kernel(const RopeParams p) {
  const int64_t per_head = p.dim - p.pairs;  // pairs, then the elements past them
  const int64_t heads = p.heads + p.kv_heads;
  const int64_t rot = heads * per_head, all = rot + (p.v ? p.kv_heads * p.dim : 0);
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
       w < p.tokens * all; w += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = w / all, r = w - t * all;
    if (r >= rot) {
      const int64_t h = (r - rot) / p.dim, d = (r - rot) - h * p.dim;
      T *row = cache_row(static_cast<T *>(p.v_out), p, p.vo_s, p.slots[t]);
      if (row)
        row[h * p.vo_s[2] + d] = static_cast<const T *>(p.v)[t * p.v_s[0] + h * p.v_s[1] + d];
      continue;
    }
    int64_t h = r / per_head;
    const int i = static_cast<int>(r - h * per_head);
    const T *x;
    T *y;
    if (h < p.heads) {
      x = static_cast<const T *>(p.q) + t * p.q_s[0] + h * p.q_s[1];
      y = static_cast<T *>(p.q_out) + t * p.qo_s[0] + h * p.qo_s[1];
    } else {
      h -= p.heads;
      x = static_cast<const T *>(p.k) + t * p.k_s[0] + h * p.k_s[1];
      if (p.slots) {
        y = cache_row(static_cast<T *>(p.k_out), p, p.ko_s, p.slots[t]);
        if (!y) continue;
        y += h * p.ko_s[2];
      } else {
        y = static_cast<T *>(p.k_out) + t * p.ko_s[0] + h * p.ko_s[1];
      }
    }
    if (i >= p.pairs) {
      y[p.pairs + i] = x[p.pairs + i];
      continue;
    }
    float c, s;
    angle(p, t, i, c, s);
    const int ia = p.paired ? 2 * i : i, ib = p.paired ? 2 * i + 1 : p.pairs + i;
    const float a = to_f32(x[ia]), b = to_f32(x[ib]);
    y[ia] = from_f32<T>(a * c - b * s);
    y[ib] = from_f32<T>(b * c + a * s);
  }
}

template <typename T>
void run_plain(const RopeParams &p, int64_t ctas, cudaStream_t stream) {
  rope_plain_kernel<T><<<static_cast<unsigned>(ctas), 256, 0, stream>>>(p);
}

}  // namespace

cudaError_t launch_rope(const RopeParams &p, int dtype, int sms, cudaStream_t stream,
                        LaunchInfo *info) {
  const int64_t work = p.tokens * ((p.heads + p.kv_heads) * (p.dim - p.pairs) +
                                   (p.v ? p.kv_heads * p.dim : 0));
  if (work == 0) return cudaSuccess;
  int64_t ctas = (work + 255) / 256;
  if (ctas > sms * 32) ctas = sms * 32;
  if (dtype == MCB_DTYPE_F32)
    run_plain<float>(p, ctas, stream);
  else if (dtype == MCB_DTYPE_F16)
    run_plain<__half>(p, ctas, stream);
  else
    run_plain<__nv_bfloat16>(p, ctas, stream);
  info->launches = 1;
  info->ctas = static_cast<int>(ctas);
  info->set_route(p.slots ? "rope_append_plain" : "rope_plain");
  return cudaGetLastError();
}

}  // namespace mcb
