// Penalties for repeated tokens, biases and grammar masks on logits.
//
//   x = logits[r, v]
//   x = x > 0 ? x / repetition : x * repetition      if v is in the row's tokens
//   x = x - frequency * n - presence * (n > 0)       n = times v was generated
//   x = x + bias                                     v's last entry in the row's list
//   x = -inf                                         where the grammar forbids v
// in f32 and in this order, rounded once to the output's type.
//
// Bound: HBM (logits and mask bits read once, the result written once). A row
// is cut into slices of the vocabulary; a CTA counts the row's tokens that fall
// into its slice in shared memory (one word a vocabulary entry: bit 31 "in the
// prompt", bit 30 "biased", the rest the generated count; integer atomics, so the
// result does not depend on their order), then finishes the slice. Which of
// several biases of an entry is the last one is settled there, too, by an atomic
// maximum. A thread's logits and mask words are loaded before the counting, which
// then hides their latency. Each slice reads the row's whole history again, from L2.
//
// 256 rows of 131072 bf16 logits to f32, histories of up to 8192 tokens, 300 biases
// and a mask: 64 us, 210 MB at 3.3 TB/s; without histories 49 us, without biases 47.
// The reading of the history costs 15 us, the rest is a CTA's load, mark and store
// following one another with three CTAs to a processor. Measured against it:
// clusters of 8 slices that share the reading, each CTA counting a part of the
// tokens in the others' shared memory, 96 us (of 72 then); the tokens sorted by
// slice in a launch before, 70 us, and 29 against 21 at 64 rows; slices of 4096 with
// 256 threads 72 us (42 without histories and biases, but twice the reading); 1024
// threads 86 us, four CTAs of 32 registers 74 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace {

constexpr int SLICE = 8192;  // vocabulary entries per CTA
constexpr int THREADS = 512;
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kTimes = 0x3fffffffu;

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

// N consecutive entries (a multiple of 8) from a 16-byte boundary on, as loaded.
template <typename T, int N>
struct Raw {
  uint32_t w[N * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T *x) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(x)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void store(T *y) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4 *>(y)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[j]);
    else {
      const uint16_t h = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
      return static_cast<float>(reinterpret_cast<const T &>(h));
    }
  }
  __device__ __forceinline__ void put(const float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 4 / sizeof(T)) {
      if constexpr (sizeof(T) == 4)
        w[j] = __float_as_uint(f[j]);
      else if constexpr (std::is_same_v<T, __half>)
        w[j / 2] = pack_f16x2(f[j], f[j + 1]);
      else
        w[j / 2] = pack_bf16x2(f[j], f[j + 1]);
    }
  }
};

__device__ __forceinline__ void prefetch_l1(const void *x) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(x));
}

constexpr int EARLY = 2;  // groups of four tokens that a thread loads before the counting

// Group q of four tokens: -1 for those before the first or after the last one.
// Only whole groups of the list are read 16 bytes at a time.
__device__ __forceinline__ int4 four(const int4 *ids, int q, int lead, int count) {
  const int a = 4 * q - lead;  // place of the group's first token in the list
  if (a >= 0 && a + 4 <= count) return ids[q];
  const int *one = reinterpret_cast<const int *>(ids + q);
  int4 v;
  v.x = a >= 0 && a < count ? one[0] : -1;
  v.y = a + 1 >= 0 && a + 1 < count ? one[1] : -1;
  v.z = a + 2 >= 0 && a + 2 < count ? one[2] : -1;
  v.w = a + 3 >= 0 && a + 3 < count ? one[3] : -1;
  return v;
}

// kN: consecutive entries of a thread, 8 where rows start on 16-byte
// boundaries (the last ones of a row one by one), else 1.
template <typename TI, typename TO, bool kBias, int kN>
__global__ void __launch_bounds__(THREADS, 3) logits_kernel(const LogitsParams p) {
  constexpr int PER = SLICE / THREADS / kN;  // groups of a thread
  extern __shared__ uint32_t smem[];
  uint32_t *seen = smem;
  int32_t *entry = reinterpret_cast<int32_t *>(smem + SLICE);  // last bias of the entries that have one
  const int64_t row = blockIdx.x;
  const int64_t v0 = static_cast<int64_t>(blockIdx.y) * SLICE;
  const int n = static_cast<int>(min(static_cast<int64_t>(SLICE), p.vocab - v0));
  const int b0 = kBias ? max(0, p.bias_cu[row]) : 0;
  const int b1 = kBias ? static_cast<int>(min(static_cast<int64_t>(p.bias_cu[row + 1]), p.biases)) : 0;
  const int first = max(0, p.cu[row]);
  const int last = static_cast<int>(min(static_cast<int64_t>(p.cu[row + 1]), p.tokens));
  const int generated = static_cast<int>(
      min(static_cast<int64_t>(first) + p.prompt_lens[row], static_cast<int64_t>(0x7ffffff0)));
  const TI *x = static_cast<const TI *>(p.logits) + row * p.ld_in + v0;
  TO *y = static_cast<TO *>(p.out) + row * p.ld_out + v0;
  const uint32_t *mask = p.allowed ? p.allowed + row * p.ld_mask + v0 / 32 : nullptr;
  Raw<TI, kN == 1 ? 8 : kN> raw[kN == 1 ? 1 : PER];  // kN > 1, whole groups
  float loose[kN == 1 ? PER : 1];                    // kN = 1
#pragma unroll
  for (int g = 0; g < PER; ++g) {
    const int i = (g * THREADS + threadIdx.x) * kN;
    if constexpr (kN > 1) {
      if (i + kN <= n) raw[g].load(x + i);
    } else {
      loose[g] = i < n ? static_cast<float>(x[i]) : 0.0f;
    }
  }
  // All that the last pass needs is loaded before the counting, too.
  const float rep = p.repetition ? p.repetition[row] : 1.0f;
  const float pre = p.presence ? p.presence[row] : 0.0f;
  const float fre = p.frequency ? p.frequency[row] : 0.0f;
  uint32_t bits[PER];
#pragma unroll
  for (int g = 0; g < PER; ++g) {
    const int i = (g * THREADS + threadIdx.x) * kN;
    bits[g] = mask && i < n ? mask[i >> 5] >> (i & 31) : 0xffffffffu;
  }
  // Tokens four at a time, from the 16-byte boundary at or before the first one on;
  // `lead` tokens before it and what comes after the last one do not count.
  const int lead = static_cast<int>(
      (reinterpret_cast<uintptr_t>(p.token_ids + first) & 15u) / sizeof(int32_t));
  const int4 *ids = reinterpret_cast<const int4 *>(p.token_ids + first - lead);
  const int groups = last > first ? (last - first + lead + 3) / 4 : 0;
  int4 early[EARLY];
#pragma unroll
  for (int u = 0; u < EARLY; ++u) {
    const int q = u * THREADS + threadIdx.x;
    if (q < groups) early[u] = four(ids, q, lead, last - first);
  }
  for (int i = threadIdx.x * 4; i < SLICE; i += THREADS * 4)
    *reinterpret_cast<uint4 *>(seen + i) = make_uint4(0, 0, 0, 0);
  // One bias per thread and round; `b` its place in the slice, -1: elsewhere.
  auto bias_at = [&](int64_t i) -> int {
    if (i >= b1) return -1;
    const int64_t v = p.bias_ids[i] - v0;
    return v >= 0 && v < n ? static_cast<int>(v) : -1;
  };
  const int64_t bi = static_cast<int64_t>(b0) + threadIdx.x;
  const int mine = kBias ? bias_at(bi) : -1;
  if (mine >= 0) prefetch_l1(p.bias_values + bi);
  if (kBias) {
    if (mine >= 0) entry[mine] = -1;
    for (int64_t i = bi + THREADS; i < b1; i += THREADS) {
      const int v = bias_at(i);
      if (v >= 0) entry[v] = -1;
    }
  }
  __syncthreads();
  const uint32_t low = static_cast<uint32_t>(v0), size = static_cast<uint32_t>(n);
  const int from = generated - first + lead;  // place of the first generated token
  auto count = [&](int at, int id) {
    const uint32_t v = static_cast<uint32_t>(id) - low;
    if (v >= size) return;  // ids below 0, too
    if (at >= from)
      atomicAdd(&seen[v], 1u);
    else if (!(*static_cast<volatile uint32_t *>(&seen[v]) & kSeen))
      atomicOr(&seen[v], kSeen);
  };
  auto count4 = [&](int q, const int4 &id) {
    count(4 * q, id.x);
    count(4 * q + 1, id.y);
    count(4 * q + 2, id.z);
    count(4 * q + 3, id.w);
  };
#pragma unroll
  for (int u = 0; u < EARLY; ++u)
    if (u * THREADS + static_cast<int>(threadIdx.x) < groups)
      count4(u * THREADS + threadIdx.x, early[u]);
#pragma unroll 2
  for (int q = EARLY * THREADS + threadIdx.x; q < groups; q += THREADS)
    count4(q, four(ids, q, lead, last - first));
  if (kBias) {
    if (mine >= 0) {
      atomicMax(&entry[mine], static_cast<int32_t>(bi));
      atomicOr(&seen[mine], kBiased);
    }
    for (int64_t i = bi + THREADS; i < b1; i += THREADS) {
      const int v = bias_at(i);
      if (v >= 0) {
        atomicMax(&entry[v], static_cast<int32_t>(i));
        atomicOr(&seen[v], kBiased);
      }
    }
  }
  const float inv = 1.0f / rep;
  __syncthreads();
  auto penalty = [&](float z, uint32_t s) -> float {
    const uint32_t times = s & kTimes;
    if (p.repetition && (s & ~kBiased)) z *= z > 0.0f ? inv : rep;
    if (times) z = __fsub_rn(__fsub_rn(z, __fmul_rn(fre, static_cast<float>(times))), pre);
    return z;
  };
  auto finish = [&](int i, float z, uint32_t s) -> float {  // an entry with marks
    z = penalty(z, s);
    if (kBias && (s & kBiased)) z += p.bias_values[entry[i]];
    return z;
  };
#pragma unroll
  for (int g = 0; g < PER; ++g) {
    const int i = (g * THREADS + threadIdx.x) * kN;
    if (i >= n) continue;
    if constexpr (kN > 1) {
      if (i + kN > n) {  // the last entries of a row that is no whole group
        for (int j = 0; i + j < n; ++j) {
          const float z = finish(i + j, static_cast<float>(x[i + j]), seen[i + j]);
          y[i + j] = from_f32<TO>((bits[g] >> j) & 1u ? z : -INFINITY);
        }
        continue;
      }
      // Marks 16 bytes at a time (words 8 apart would meet in the same banks); most
      // groups have none.
      Raw<uint32_t, kN> marks;
      float z[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] = raw[g].get(j);
      marks.load(seen + i);
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < kN; ++j) any |= marks.w[j];
      if (any) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (marks.w[j]) z[j] = finish(i + j, z[j], marks.w[j]);
      }
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] = (bits[g] >> j) & 1u ? z[j] : -INFINITY;
      Raw<TO, kN> out;
      out.put(z);
      out.store(y + i);
    } else {
      const float z = finish(i, loose[g], seen[i]);
      y[i] = from_f32<TO>(bits[g] & 1u ? z : -INFINITY);
    }
  }
}

template <typename TI, typename TO>
cudaError_t run(const LogitsParams &p, dim3 grid, cudaStream_t stream) {
  const size_t bytes = SLICE * sizeof(uint32_t) * (p.bias_ids ? 2 : 1);
  auto go = [&](auto kernel) {
    const cudaError_t e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return e;
    kernel<<<grid, THREADS, bytes, stream>>>(p);
    return cudaGetLastError();
  };
  const bool aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(p.out) % 16 == 0 &&
                       (p.rows == 1 || (p.ld_in * sizeof(TI) % 16 == 0 &&
                                        p.ld_out * sizeof(TO) % 16 == 0));
  if (aligned)
    return p.bias_ids ? go(logits_kernel<TI, TO, true, 8>) : go(logits_kernel<TI, TO, false, 8>);
  return p.bias_ids ? go(logits_kernel<TI, TO, true, 1>) : go(logits_kernel<TI, TO, false, 1>);
}

}  // namespace

cudaError_t launch_logits(const LogitsParams &p, int in_dtype, int out_dtype, cudaStream_t stream,
                          LaunchInfo *info) {
  const int64_t slices = (p.vocab + SLICE - 1) / SLICE;
  if (p.rows > 0x7fffffff || slices > 65535) return cudaErrorNotSupported;
  const dim3 grid(static_cast<unsigned>(p.rows), static_cast<unsigned>(slices));
  cudaError_t e;
  if (in_dtype == MCB_DTYPE_F32)
    e = run<float, float>(p, grid, stream);
  else if (in_dtype == MCB_DTYPE_F16)
    e = out_dtype == MCB_DTYPE_F32 ? run<__half, float>(p, grid, stream)
                                   : run<__half, __half>(p, grid, stream);
  else
    e = out_dtype == MCB_DTYPE_F32 ? run<__nv_bfloat16, float>(p, grid, stream)
                                   : run<__nv_bfloat16, __nv_bfloat16>(p, grid, stream);
  info->launches = 1;
  info->tile_n = SLICE;
  info->ctas = static_cast<int>(p.rows * slices);
  info->set_route("logits");
  return e;
}

}  // namespace mcb
