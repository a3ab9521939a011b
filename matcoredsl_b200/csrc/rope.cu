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
// rows of the tokens' positions read once). 8192 tokens of 32 + 8 + 8 heads of 128,
// f16, with the append: 41 us, 204 MB at 5.0 TB/s; 20001 tokens of 16 + 16 heads of 80,
// f32, paired: 80 us, 415 MB at 5.2 TB/s. The plain copy's rate is 6.55 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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
  const int32_t blk = static_cast<int32_t>(fast_div(slot, p.block_div));
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

// 16 bytes as VE f32 values, in pairs for the two-element f32 instructions, and back.
template <typename T>
struct Vec {
  static constexpr int VE = 16 / sizeof(T);
  static __device__ __forceinline__ void get(const uint4 &v, uint64_t (&f)[VE / 2]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = f2_pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else if constexpr (std::is_same_v<T, __half>) {
        const float2 x = __half22float2(reinterpret_cast<const __half2 &>(w[i]));
        f[i] = f2_pack(x.x, x.y);
      } else {
        f[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      }
    }
  }
  static __device__ __forceinline__ uint4 put(const uint64_t (&f)[VE / 2]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      float lo, hi;
      f2_unpack(f[i], lo, hi);
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(lo);
        w[2 * i + 1] = __float_as_uint(hi);
      } else if constexpr (std::is_same_v<T, __half>) {
        w[i] = pack_f16x2(lo, hi);
      } else {
        w[i] = pack_bf16x2(lo, hi);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

constexpr int ROPE_THREADS = 128;

// 16-byte accesses. A CTA has threads (chunk of VE pairs, head slot, token): a
// thread keeps its pairs' cosines and sines in registers while it walks over the
// heads of its token, kAhead heads' loads in flight at a time; value rows and
// elements past the pairs are copied by the same threads. The cosines and sines of
// the CTA's tokens are gathered once into shared memory, after the first loads of
// q, k and v have been issued. Offsets within a token's rows are 32-bit, there is
// no division outside the gather of several tokens, and two elements are turned at
// a time. For 8192 tokens of 32 + 8 + 8 heads of 128 (f16, three axes in turn; HBM
// floor 31 us): 68 us with every thread gathering its own angles, 55 with a flat
// thread index that was divided, 51 with 16 slots of 2.5 heads each (what a thread
// does once per token was more than half of its instructions), 41 as it is.
template <typename T, bool kPaired, int kAhead>
__global__ void __launch_bounds__(ROPE_THREADS) rope_vec_kernel(const RopeParams p) {
  constexpr int VE = Vec<T>::VE;
  // Tokens of a CTA x pairs <= ROPE_THREADS x VE.
  __shared__ __align__(16) float cosines[ROPE_THREADS * VE], sines[ROPE_THREADS * VE];
  const int c = threadIdx.x, slot = threadIdx.y, tok = threadIdx.z;
  const int chunks = blockDim.x, slots = blockDim.y, tokens = blockDim.z;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens, t = t0 + tok;
  const bool live = t < p.tokens;
  const int64_t tl = live ? t : t0;  // dead threads only help with the gather
  const T *q = static_cast<const T *>(p.q) + tl * p.q_s[0];
  const T *k = static_cast<const T *>(p.k) + tl * p.k_s[0];
  const T *v = static_cast<const T *>(p.v) + (p.v ? tl * p.v_s[0] : 0);
  const int q_s = static_cast<int>(p.q_s[1]), k_s = static_cast<int>(p.k_s[1]);
  const int v_s = static_cast<int>(p.v_s[1]);
  const int32_t at = p.slots ? p.slots[tl] : 0;
  // Offsets of the two 16-byte pieces that hold this thread's pairs.
  const int oa = kPaired ? 2 * c * VE : c * VE, ob = kPaired ? oa + VE : p.pairs + c * VE;
  const int all_heads = live ? p.heads + p.kv_heads : 0;
  uint4 a[kAhead], b[kAhead];
  auto load_heads = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * slots;
      if (h < all_heads) {
        const T *x = h < p.heads ? q + h * q_s : k + (h - p.heads) * k_s;
        a[u] = *reinterpret_cast<const uint4 *>(x + oa);
        b[u] = *reinterpret_cast<const uint4 *>(x + ob);
      }
    }
  };
  load_heads(slot);
  // Value rows: this thread's first two pieces of its first head ahead.
  const int v_heads = p.v && live ? p.kv_heads : 0;
  uint4 v0[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (slot < v_heads && (c + u * chunks) * VE < p.dim)
      v0[u] = *reinterpret_cast<const uint4 *>(v + slot * v_s + (c + u * chunks) * VE);
  {
    const int tid = (tok * slots + slot) * chunks + c, threads = chunks * slots * tokens;
    const int here = static_cast<int>(min(static_cast<int64_t>(tokens), p.tokens - t0));
    for (int i = tid; i < here * p.pairs; i += threads) {
      const int gt = tokens == 1 ? 0 : i / p.pairs;
      angle(p, t0 + gt, i - gt * p.pairs, cosines[i], sines[i]);
    }
  }
  __syncthreads();
  if (!live) return;
  T *q_out = static_cast<T *>(p.q_out) + t * p.qo_s[0], *k_out, *v_out = nullptr;
  const int qo_s = static_cast<int>(p.qo_s[1]);
  const int ko_s = static_cast<int>(p.slots ? p.ko_s[2] : p.ko_s[1]);
  if (p.slots) {
    k_out = cache_row(static_cast<T *>(p.k_out), p, p.ko_s, at);
    v_out = cache_row(static_cast<T *>(p.v_out), p, p.vo_s, at);
  } else {
    k_out = static_cast<T *>(p.k_out) + t * p.ko_s[0];
  }
  const int heads = p.heads + (k_out ? p.kv_heads : 0);
  // Pairs 2i and 2i + 1 of this thread: their cosines, sines and negated sines.
  uint64_t cs[VE / 2], sn[VE / 2], ns[VE / 2];
#pragma unroll
  for (int i = 0; i < VE / 2; ++i) {
    const float2 x = *reinterpret_cast<const float2 *>(cosines + tok * p.pairs + c * VE + 2 * i);
    const float2 y = *reinterpret_cast<const float2 *>(sines + tok * p.pairs + c * VE + 2 * i);
    cs[i] = f2_pack(x.x, x.y);
    sn[i] = f2_pack(y.x, y.y);
    ns[i] = f2_pack(-y.x, -y.y);
  }
  for (int h0 = slot; h0 < heads; h0 += kAhead * slots) {
    if (h0 != slot) load_heads(h0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * slots;
      if (h < heads) {
        uint64_t fa[VE / 2], fb[VE / 2], ga[VE / 2], gb[VE / 2];
        Vec<T>::get(a[u], fa);
        Vec<T>::get(b[u], fb);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          if (kPaired) {
            // (fa, fb) is 2 VE elements in a row, a pair's two side by side: part them,
            // turn, and put them back.
            const uint64_t m = i < VE / 4 ? fa[2 * i] : fb[2 * i - VE / 2];
            const uint64_t n = i < VE / 4 ? fa[2 * i + 1] : fb[2 * i + 1 - VE / 2];
            float x0, y0, x1, y1;
            f2_unpack(m, x0, y0);
            f2_unpack(n, x1, y1);
            const uint64_t x = f2_pack(x0, x1), y = f2_pack(y0, y1);
            const uint64_t gx = f2_fma(x, cs[i], f2_mul(y, ns[i]));
            const uint64_t gy = f2_fma(y, cs[i], f2_mul(x, sn[i]));
            f2_unpack(gx, x0, x1);
            f2_unpack(gy, y0, y1);
            (i < VE / 4 ? ga[2 * i] : gb[2 * i - VE / 2]) = f2_pack(x0, y0);
            (i < VE / 4 ? ga[2 * i + 1] : gb[2 * i + 1 - VE / 2]) = f2_pack(x1, y1);
          } else {
            ga[i] = f2_fma(fa[i], cs[i], f2_mul(fb[i], ns[i]));
            gb[i] = f2_fma(fb[i], cs[i], f2_mul(fa[i], sn[i]));
          }
        }
        T *y = h < p.heads ? q_out + h * qo_s : k_out + (h - p.heads) * ko_s;
        *reinterpret_cast<uint4 *>(y + oa) = Vec<T>::put(ga);
        *reinterpret_cast<uint4 *>(y + ob) = Vec<T>::put(gb);
      }
    }
  }
  // Elements past the pairs, then the value rows: plain copies.
  if (2 * p.pairs < p.dim)
    for (int h = slot; h < heads; h += slots)
      for (int d = 2 * p.pairs + c * VE; d < p.dim; d += chunks * VE) {
        const T *x = h < p.heads ? q + h * q_s : k + (h - p.heads) * k_s;
        T *y = h < p.heads ? q_out + h * qo_s : k_out + (h - p.heads) * ko_s;
        *reinterpret_cast<uint4 *>(y + d) = *reinterpret_cast<const uint4 *>(x + d);
      }
  if (v_out) {
    const int vo_s = static_cast<int>(p.vo_s[2]);
    for (int h = slot; h < v_heads; h += slots)
#pragma unroll 2
      for (int u = 0; (c + u * chunks) * VE < p.dim; ++u) {
        const int d = (c + u * chunks) * VE;
        *reinterpret_cast<uint4 *>(v_out + h * vo_s + d) =
            h == slot && u < 2 ? v0[u & 1] : *reinterpret_cast<const uint4 *>(v + h * v_s + d);
      }
  }
}

// The vector kernel's conditions: every piece starts on a 16-byte boundary. (The
// scalar kernel in its place: 211 us instead of 41 and 219 instead of 80 for the calls
// above; at 64 tokens no difference.)
bool vector_ok(const RopeParams &p, int ve) {
  uintptr_t bases = 0;
  for (const void *x : {p.q, p.k, p.v, static_cast<const void *>(p.q_out),
                        static_cast<const void *>(p.k_out), static_cast<const void *>(p.v_out)})
    bases |= reinterpret_cast<uintptr_t>(x);
  int64_t steps = p.dim | p.pairs;
  for (int i = 0; i < 2; ++i) steps |= p.q_s[i] | p.k_s[i] | p.qo_s[i] | (p.v ? p.v_s[i] : 0);
  for (int i = 0; i < (p.slots ? 3 : 2); ++i) steps |= p.ko_s[i] | (p.slots ? p.vo_s[i] : 0);
  // 32-bit offsets within a token's rows.
  int64_t far = 0;
  for (int64_t x : {(p.heads - 1) * p.q_s[1], (p.heads - 1) * p.qo_s[1],
                    (p.kv_heads - 1) * p.k_s[1], (p.kv_heads - 1) * p.ko_s[p.slots ? 2 : 1],
                    p.v ? (p.kv_heads - 1) * p.v_s[1] : 0, p.v ? (p.kv_heads - 1) * p.vo_s[2] : 0})
    far = x > far ? x : far;
  return p.pairs > 0 && bases % 16 == 0 && steps % ve == 0 && far + p.dim <= 0x7fffffff;
}

template <typename T>
bool run_vec(const RopeParams &p, cudaStream_t stream, LaunchInfo *info) {
  constexpr int VE = Vec<T>::VE;
  if (!vector_ok(p, VE)) return false;
  const int heads = p.heads + p.kv_heads;
  if (heads == 0) return false;
  const int chunks = p.pairs / VE;
  // About five heads a thread: what a thread does once per token (addresses, the
  // cache's row) is as much as three heads' work.
  int slots = (heads + 4) / 5;
  if (slots > ROPE_THREADS / chunks) slots = ROPE_THREADS / chunks;
  const int tokens = ROPE_THREADS / (chunks * slots) < 64 ? ROPE_THREADS / (chunks * slots) : 64;
  const int64_t ctas = (p.tokens + tokens - 1) / tokens;
  if (ctas > 0x7fffffff) return false;
  const dim3 block(chunks, slots, tokens);
  if (p.paired)
    rope_vec_kernel<T, true, 2><<<static_cast<unsigned>(ctas), block, 0, stream>>>(p);
  else
    rope_vec_kernel<T, false, 2><<<static_cast<unsigned>(ctas), block, 0, stream>>>(p);
  info->launches = 1;
  info->tile_m = tokens;
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
