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

// 16 bytes as VE f32 values and back.
template <typename T>
struct Vec {
  static constexpr int VE = 16 / sizeof(T);
  static __device__ __forceinline__ void get(const uint4 &w, float (&f)[VE]) {
    const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = to_f32(x[i]);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[VE]) {
    uint4 w;
    T *x = reinterpret_cast<T *>(&w);
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = from_f32<T>(f[i]);
    return w;
  }
};

// How a CTA of the vector kernel is cut: `tokens` tokens, `slots` head slots
// of a token, `chunks` threads of a head (VE pairs each).
struct RopeCut {
  int tokens, slots, chunks;
  int table_vec;  // table rows can be read 16 bytes at a time
};

// 16-byte accesses. A thread owns VE pairs: their cosines and sines stay in
// registers while it walks over the heads of its token, kAhead heads' loads in
// flight at a time; value rows and elements past the pairs are copied by the
// same threads.
template <typename T, bool kPaired, int kAhead>
__global__ void __launch_bounds__(128) rope_vec_kernel(const RopeParams p, const RopeCut cut) {
  constexpr int VE = Vec<T>::VE;
  const int per = cut.slots * cut.chunks;
  const int tok = threadIdx.x / per, r = threadIdx.x - tok * per;
  const int slot = r / cut.chunks, c = r - slot * cut.chunks;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * cut.tokens + tok;
  if (tok >= cut.tokens || t >= p.tokens) return;
  const T *qk[2] = {static_cast<const T *>(p.q) + t * p.q_s[0],
                    static_cast<const T *>(p.k) + t * p.k_s[0]};
  T *out[2] = {static_cast<T *>(p.q_out) + t * p.qo_s[0], nullptr};
  int64_t out_s = p.ko_s[1];
  T *v_row = nullptr;
  if (p.slots) {
    const int32_t at = p.slots[t];
    out[1] = cache_row(static_cast<T *>(p.k_out), p, p.ko_s, at);
    out_s = p.ko_s[2];
    v_row = cache_row(static_cast<T *>(p.v_out), p, p.vo_s, at);
  } else {
    out[1] = static_cast<T *>(p.k_out) + t * p.ko_s[0];
  }
  const int heads = p.heads + (out[1] ? p.kv_heads : 0);
  // Offsets of the two 16-byte pieces that hold this thread's pairs.
  const int oa = kPaired ? 2 * c * VE : c * VE, ob = kPaired ? oa + VE : p.pairs + c * VE;
  float cs[VE], sn[VE];
  // Usually one axis turns all of them: one table row, read 16 bytes at a time.
  bool one = cut.table_vec;
#pragma unroll
  for (int i = 1; i < VE; ++i) one = one && p.axis[c * VE + i] == p.axis[c * VE];
  const int32_t pos = p.positions[p.axis[c * VE] * p.pos_stride + t];
  if (one && pos >= 0 && pos < p.table_rows) {
    const float4 *row = reinterpret_cast<const float4 *>(p.cos_sin + pos * p.table_stride + c * VE);
    const float4 *sins = reinterpret_cast<const float4 *>(p.cos_sin + pos * p.table_stride +
                                                          p.pairs + c * VE);
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      const float4 x = row[i], y = sins[i];
      cs[4 * i] = x.x, cs[4 * i + 1] = x.y, cs[4 * i + 2] = x.z, cs[4 * i + 3] = x.w;
      sn[4 * i] = y.x, sn[4 * i + 1] = y.y, sn[4 * i + 2] = y.z, sn[4 * i + 3] = y.w;
    }
    if (p.inverse) {
#pragma unroll
      for (int i = 0; i < VE; ++i) sn[i] = -sn[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) angle(p, t, c * VE + i, cs[i], sn[i]);
  }
  for (int h0 = slot; h0 < heads; h0 += kAhead * cut.slots) {
    uint4 a[kAhead], b[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * cut.slots;
      if (h < heads) {
        const T *x = h < p.heads ? qk[0] + h * p.q_s[1] : qk[1] + (h - p.heads) * p.k_s[1];
        a[u] = *reinterpret_cast<const uint4 *>(x + oa);
        b[u] = *reinterpret_cast<const uint4 *>(x + ob);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * cut.slots;
      if (h < heads) {
        float fa[VE], fb[VE], ga[VE], gb[VE];
        Vec<T>::get(a[u], fa);
        Vec<T>::get(b[u], fb);
        if (kPaired) {
          // (fa, fb) is 2 VE elements in a row: pair i = elements 2i, 2i + 1.
#pragma unroll
          for (int i = 0; i < VE / 2; ++i) {
            ga[2 * i] = fa[2 * i] * cs[i] - fa[2 * i + 1] * sn[i];
            ga[2 * i + 1] = fa[2 * i + 1] * cs[i] + fa[2 * i] * sn[i];
            gb[2 * i] = fb[2 * i] * cs[VE / 2 + i] - fb[2 * i + 1] * sn[VE / 2 + i];
            gb[2 * i + 1] = fb[2 * i + 1] * cs[VE / 2 + i] + fb[2 * i] * sn[VE / 2 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            ga[i] = fa[i] * cs[i] - fb[i] * sn[i];
            gb[i] = fb[i] * cs[i] + fa[i] * sn[i];
          }
        }
        T *y = h < p.heads ? out[0] + h * p.qo_s[1] : out[1] + (h - p.heads) * out_s;
        *reinterpret_cast<uint4 *>(y + oa) = Vec<T>::put(ga);
        *reinterpret_cast<uint4 *>(y + ob) = Vec<T>::put(gb);
      }
    }
  }
  // Elements past the pairs, then the value rows: plain copies.
  const int tail = (p.dim - 2 * p.pairs) / VE;
  for (int i = r; i < heads * tail; i += per) {
    const int h = i / tail, d = 2 * p.pairs + (i - h * tail) * VE;
    const T *x = h < p.heads ? qk[0] + h * p.q_s[1] : qk[1] + (h - p.heads) * p.k_s[1];
    T *y = h < p.heads ? out[0] + h * p.qo_s[1] : out[1] + (h - p.heads) * out_s;
    *reinterpret_cast<uint4 *>(y + d) = *reinterpret_cast<const uint4 *>(x + d);
  }
  if (v_row) {
    const T *v = static_cast<const T *>(p.v) + t * p.v_s[0];
    const int pieces = p.dim / VE;
    for (int i = r; i < p.kv_heads * pieces; i += per) {
      const int h = i / pieces, d = (i - h * pieces) * VE;
      *reinterpret_cast<uint4 *>(v_row + h * p.vo_s[2] + d) =
          *reinterpret_cast<const uint4 *>(v + h * p.v_s[1] + d);
    }
  }
}

// The vector kernel's conditions: every piece starts on a 16-byte boundary.
bool vector_ok(const RopeParams &p, int ve) {
  uintptr_t bases = 0;
  for (const void *x : {p.q, p.k, p.v, static_cast<const void *>(p.q_out),
                        static_cast<const void *>(p.k_out), static_cast<const void *>(p.v_out)})
    bases |= reinterpret_cast<uintptr_t>(x);
  int64_t steps = p.dim | p.pairs;
  for (int i = 0; i < 2; ++i) steps |= p.q_s[i] | p.k_s[i] | p.qo_s[i] | (p.v ? p.v_s[i] : 0);
  for (int i = 0; i < (p.slots ? 3 : 2); ++i) steps |= p.ko_s[i] | (p.slots ? p.vo_s[i] : 0);
  return p.pairs > 0 && bases % 16 == 0 && steps % ve == 0;
}

template <typename T>
bool run_vec(const RopeParams &p, cudaStream_t stream, LaunchInfo *info) {
  constexpr int VE = Vec<T>::VE;
  if (!vector_ok(p, VE)) return false;
  const int heads = p.heads + p.kv_heads;
  if (heads == 0) return false;
  RopeCut cut;
  cut.chunks = p.pairs / VE;
  cut.slots = 128 / cut.chunks < heads ? 128 / cut.chunks : heads;
  cut.tokens = 128 / (cut.chunks * cut.slots);
  cut.table_vec = reinterpret_cast<uintptr_t>(p.cos_sin) % 16 == 0 && p.table_stride % 4 == 0;
  const int64_t ctas = (p.tokens + cut.tokens - 1) / cut.tokens;
  if (ctas > 0x7fffffff) return false;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (p.paired)
    rope_vec_kernel<T, true, 2><<<grid, 128, 0, stream>>>(p, cut);
  else
    rope_vec_kernel<T, false, 2><<<grid, 128, 0, stream>>>(p, cut);
  info->launches = 1;
  info->tile_m = cut.tokens;
  info->ctas = static_cast<int>(ctas);
  info->set_route(p.slots ? "rope_append" : "rope");
  return true;
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
  const bool done = dtype == MCB_DTYPE_F32   ? run_vec<float>(p, stream, info)
                    : dtype == MCB_DTYPE_F16 ? run_vec<__half>(p, stream, info)
                                             : run_vec<__nv_bfloat16>(p, stream, info);
  if (done) return cudaGetLastError();
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
