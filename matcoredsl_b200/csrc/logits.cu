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
// into its slice in shared memory (one word a vocabulary entry: bit 31 "seen",
// the rest the generated count; integer atomics, so the result does not
// depend on their order), then passes over the slice once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace {

constexpr int SLICE = 8192;  // vocabulary entries per CTA
constexpr int THREADS = 512;
constexpr uint32_t kSeen = 0x80000000u;

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

template <typename TI, typename TO, bool kBias>
__global__ void __launch_bounds__(THREADS) logits_kernel(const LogitsParams p) {
  extern __shared__ uint32_t smem[];
  uint32_t *seen = smem;
  int32_t *entry = reinterpret_cast<int32_t *>(smem + SLICE);  // last bias entry, -1 none
  const int64_t row = blockIdx.x;
  const int64_t v0 = static_cast<int64_t>(blockIdx.y) * SLICE;
  const int n = static_cast<int>(min(static_cast<int64_t>(SLICE), p.vocab - v0));
  for (int i = threadIdx.x; i < n; i += THREADS) {
    seen[i] = 0;
    if (kBias) entry[i] = -1;
  }
  __syncthreads();
  {
    const int64_t first = max(0, p.cu[row]);
    const int64_t last = min(static_cast<int64_t>(p.cu[row + 1]), p.tokens);
    const int64_t generated = first + p.prompt_lens[row];
    for (int64_t i = first + threadIdx.x; i < last; i += THREADS) {
      const int64_t v = p.token_ids[i] - v0;
      if (v >= 0 && v < n) {
        if (i >= generated) atomicAdd(&seen[v], 1u);
        atomicOr(&seen[v], kSeen);
      }
    }
    if (kBias) {
      const int64_t b0 = max(0, p.bias_cu[row]);
      const int64_t b1 = min(static_cast<int64_t>(p.bias_cu[row + 1]), p.biases);
      for (int64_t i = b0 + threadIdx.x; i < b1; i += THREADS) {
        const int64_t v = p.bias_ids[i] - v0;
        if (v >= 0 && v < n) atomicMax(&entry[v], static_cast<int32_t>(i));
      }
    }
  }
  __syncthreads();
  const float rep = p.repetition ? p.repetition[row] : 1.0f;
  const float pre = p.presence ? p.presence[row] : 0.0f;
  const float fre = p.frequency ? p.frequency[row] : 0.0f;
  const TI *x = static_cast<const TI *>(p.logits) + row * p.ld_in + v0;
  TO *y = static_cast<TO *>(p.out) + row * p.ld_out + v0;
  const uint32_t *mask = p.allowed ? p.allowed + row * p.ld_mask : nullptr;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    float f = static_cast<float>(x[i]);
    const uint32_t s = seen[i];
    if (s) {
      if (p.repetition) f = f > 0.0f ? f / rep : f * rep;
      const uint32_t times = s & ~kSeen;
      if (times) f = __fsub_rn(__fsub_rn(f, __fmul_rn(fre, static_cast<float>(times))), pre);
    }
    if (kBias) {
      const int32_t e = entry[i];
      if (e >= 0) f += p.bias_values[e];
    }
    if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u)) f = -INFINITY;
    y[i] = from_f32<TO>(f);
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
  return p.bias_ids ? go(logits_kernel<TI, TO, true>) : go(logits_kernel<TI, TO, false>);
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
