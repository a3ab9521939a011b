// Block tables and slot maps of a paged key/value cache, from request lengths.
//
// The cache holds blocks of `block` tokens; request b's token at position p
// lives in block table[b, p / block], row p % block. Free blocks are a stack
// free[0 .. count). Growing request b from len to len + new needs
//   want_b = ceil((len + new) / block) - ceil(len / block)
// blocks, taken from the top of the stack in request order: its j-th new block
// is free[count - 1 - (start_b + j)], start_b the exclusive sum of want.
//
// Bound: latency. A step of 64 requests moves 2 KB, the largest calls about
// 1 MB, so the time is the launch plus one chain of dependent loads (lengths,
// scan, table or stack). One launch does everything: every CTA scans the
// requests up to its own tokens again (8 bytes a request from L2) instead of
// waiting for a first kernel's scan. Calls queued back to back: 64 requests by one
// token 6.2 us, 512 prompts of 131072 tokens together 8.2 us, releasing what 1000
// requests hold past new lengths 6.2 us.
#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace {

constexpr int GROW_THREADS = 1024;  // tokens per CTA, one each
constexpr int GROW_ITEMS = 4;       // requests per thread and scan round

// Inclusive scan of (x, y) over the CTA; `total` gets the CTA's sums.
__device__ __forceinline__ void block_scan2(int64_t &x, int64_t &y, int64_t (*sums)[2],
                                            int64_t &total_x, int64_t &total_y) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t px = __shfl_up_sync(0xffffffffu, x, off);
    const int64_t py = __shfl_up_sync(0xffffffffu, y, off);
    if (lane >= off) {
      x += px;
      y += py;
    }
  }
  if (lane == 31) {
    sums[warp][0] = x;
    sums[warp][1] = y;
  }
  __syncthreads();
  if (warp == 0) {
    int64_t sx = sums[lane][0], sy = sums[lane][1];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t px = __shfl_up_sync(0xffffffffu, sx, off);
      const int64_t py = __shfl_up_sync(0xffffffffu, sy, off);
      if (lane >= off) {
        sx += px;
        sy += py;
      }
    }
    sums[lane][0] = sx;
    sums[lane][1] = sy;
  }
  __syncthreads();
  if (warp > 0) {
    x += sums[warp - 1][0];
    y += sums[warp - 1][1];
  }
  total_x = sums[31][0];
  total_y = sums[31][1];
  __syncthreads();  // `sums` may be written again
}

__device__ __forceinline__ int32_t saturate(int64_t v) {
  return v > 0x7fffffff ? 0x7fffffff : static_cast<int32_t>(v);
}

// What the tokens of one request need, kept at its first token of this CTA.
struct Head {
  int32_t request, len, add, had;  // `had` blocks were in use before the call
  int32_t ok;
  int64_t first, start;  // first token of the request; blocks taken before it
};

__global__ void __launch_bounds__(GROW_THREADS) paged_grow_kernel(const PagedGrow p) {
  __shared__ int64_t sums[32][2];
  __shared__ Head heads[GROW_THREADS];
  __shared__ int32_t warp_last[32];
  __shared__ int32_t used;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first_cta = blockIdx.x == 0;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * GROW_THREADS, t1 = t0 + GROW_THREADS;
  const int32_t count = max(0, min(*p.free_count, saturate(p.free_capacity)));
  int32_t owner = -1;  // this thread's place in `heads` when a request starts there
  heads[tid].request = -1;
  if (tid == 0) used = 0;
  __syncthreads();
  int64_t tokens = 0, blocks = 0;  // sums over the requests of earlier rounds
  for (int64_t base = 0; base < p.requests; base += GROW_THREADS * GROW_ITEMS) {
    // The first CTA writes every request's outputs; others stop once the
    // requests of their own tokens are behind them.
    if (!first_cta && tokens >= t1) break;
    int32_t len[GROW_ITEMS], add[GROW_ITEMS], want[GROW_ITEMS];
    bool fits[GROW_ITEMS];
    int64_t x = 0, y = 0;
    const int64_t b0 = base + static_cast<int64_t>(tid) * GROW_ITEMS;
#pragma unroll
    for (int i = 0; i < GROW_ITEMS; ++i) {
      const bool live = b0 + i < p.requests;
      len[i] = live ? max(0, p.lens[b0 + i]) : 0;
      add[i] = live ? max(0, p.new_lens[b0 + i]) : 0;
    }
#pragma unroll
    for (int i = 0; i < GROW_ITEMS; ++i) {
      const int64_t need = (static_cast<int64_t>(len[i]) + add[i] + p.block - 1) / p.block;
      const int64_t had = (static_cast<int64_t>(len[i]) + p.block - 1) / p.block;
      fits[i] = need <= p.columns;
      want[i] = fits[i] ? static_cast<int32_t>(need - had) : 0;
      x += add[i];
      y += want[i];
    }
    const int64_t mine_x = x, mine_y = y;
    int64_t total_x, total_y;
    block_scan2(x, y, sums, total_x, total_y);
    int64_t cu = tokens + x - mine_x, start = blocks + y - mine_y;
#pragma unroll
    for (int i = 0; i < GROW_ITEMS; ++i) {
      if (b0 + i >= p.requests) break;
      const int64_t end = cu + add[i], top = start + want[i];
      const bool ok = fits[i] && (want[i] == 0 || top <= count) && (add[i] == 0 || end <= p.tokens);
      if (first_cta) {
        p.cu[b0 + i + 1] = saturate(end);
        p.after[b0 + i] = saturate(static_cast<int64_t>(len[i]) + (ok ? add[i] : 0));
        if (ok && want[i] > 0) atomicMax(&used, static_cast<int32_t>(top));
      }
      if (add[i] > 0 && cu < t1 && end > t0) {
        Head &h = heads[cu > t0 ? cu - t0 : 0];
        h.len = len[i];
        h.add = add[i];
        h.had = static_cast<int32_t>((static_cast<int64_t>(len[i]) + p.block - 1) / p.block);
        h.ok = ok;
        h.first = cu;
        h.start = start;
        h.request = static_cast<int32_t>(b0 + i);
      }
      cu = end;
      start = top;
    }
    tokens += total_x;
    blocks += total_y;
  }
  __syncthreads();
  if (first_cta && tid == 0) {
    p.cu[0] = 0;
    *p.free_left = count - used;
  }
  // The request of token t0 + tid starts at the last place at or before tid
  // that a request was written to.
  if (heads[tid].request >= 0) owner = tid;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int32_t o = __shfl_up_sync(0xffffffffu, owner, off);
    if (lane >= off) owner = max(owner, o);
  }
  if (lane == 31) warp_last[warp] = owner;
  __syncthreads();
  if (owner < 0)
    for (int w = warp - 1; w >= 0 && owner < 0; --w) owner = warp_last[w];
  const int64_t t = t0 + tid;
  if (t >= p.tokens) return;
  int32_t slot = -1, pos = 0;
  if (owner >= 0) {
    const Head &h = heads[owner];
    // Only tokens of this request: past the last one there are none.
    const int64_t at = static_cast<int64_t>(h.len) + (t - h.first);
    pos = saturate(at);
    if (t - h.first < h.add) {
      const int64_t j = at / p.block, off = at - j * p.block;
      if (h.ok) {
        int32_t *entry = p.table + h.request * p.table_stride + j;
        int32_t blk;
        if (j < h.had) {
          blk = *entry;
        } else {
          blk = p.free[count - 1 - (h.start + j - h.had)];
          if (off == 0) *entry = blk;  // the one token that opens the block
        }
        const int64_t s = static_cast<int64_t>(blk) * p.block + off;
        if (blk >= 0 && s <= 0x7fffffff) slot = static_cast<int32_t>(s);
      }
    } else {
      pos = 0;
    }
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

// ---- release ---------------------------------------------------------------------
// Request b keeps its first ceil(keep / block) blocks; the others, up to
// ceil(len / block), go back onto the stack in request order. One warp copies
// the entries of one request (of a slice of them, where rows are long).
constexpr int REL_WARPS = 32;

__device__ __forceinline__ void released(const PagedRelease &p, int64_t b, int64_t &first,
                                         int64_t &gone) {
  const int64_t len = max(0, p.lens[b]), keep = max(0, p.keep_lens[b]);
  first = (keep + p.block - 1) / p.block;
  const int64_t last = min((len + p.block - 1) / p.block, p.columns);
  gone = max(static_cast<int64_t>(0), last - first);
}

__global__ void __launch_bounds__(REL_WARPS * 32) paged_release_kernel(const PagedRelease p) {
  __shared__ int64_t sums[32][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t count = max(0, min(*p.free_count, saturate(p.free_capacity)));
  const int64_t b0 = static_cast<int64_t>(blockIdx.x) * REL_WARPS;
  // Blocks released by the requests before this CTA's.
  int64_t before = 0, unused = 0;
  for (int64_t b = tid; b < b0; b += REL_WARPS * 32) {
    int64_t first, gone;
    released(p, b, first, gone);
    before += gone;
  }
  int64_t total, total2;
  block_scan2(before, unused, sums, total, total2);
  int64_t first = 0, gone = 0;
  const int64_t b = b0 + warp;
  // Every warp needs the sums of the warps before it: lane w reads request b0 + w.
  int64_t f = 0, n = 0;
  if (b0 + lane < p.requests) released(p, b0 + lane, f, n);
  int64_t incl = n;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  first = __shfl_sync(0xffffffffu, f, warp);
  gone = __shfl_sync(0xffffffffu, n, warp);
  const int64_t to = count + total + __shfl_sync(0xffffffffu, incl, warp) - gone;
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && tid == 31)
    *p.free_left = saturate(min(count + total + incl, p.free_capacity));
  if (b >= p.requests) return;
  const int32_t *row = p.table + b * p.table_stride + first;
  for (int64_t j = blockIdx.y * 32 + lane; j < gone; j += 32 * gridDim.y)
    if (to + j < p.free_capacity) p.free[to + j] = row[j];
}

}  // namespace

cudaError_t launch_paged_grow(const PagedGrow &p, cudaStream_t stream, LaunchInfo *info) {
  const int64_t ctas = p.tokens > 0 ? (p.tokens + GROW_THREADS - 1) / GROW_THREADS : 1;
  if (ctas > 0x7fffffff) return cudaErrorNotSupported;
  paged_grow_kernel<<<static_cast<unsigned>(ctas), GROW_THREADS, 0, stream>>>(p);
  info->launches = 1;
  info->tile_m = GROW_THREADS;
  info->ctas = static_cast<int>(ctas);
  info->set_route("paged_grow");
  return cudaGetLastError();
}

cudaError_t launch_paged_release(const PagedRelease &p, cudaStream_t stream, LaunchInfo *info) {
  const int64_t ctas = p.requests > 0 ? (p.requests + REL_WARPS - 1) / REL_WARPS : 1;
  if (ctas > 0x7fffffff) return cudaErrorNotSupported;
  // Slices of a row: about four entries a lane, no more CTAs than fill the GPU.
  int64_t slices = (p.columns + 127) / 128;
  slices = slices < 1 ? 1 : (slices > 64 ? 64 : slices);
  while (slices > 1 && slices * ctas > 296) slices /= 2;
  paged_release_kernel<<<dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(slices)),
                         REL_WARPS * 32, 0, stream>>>(p);
  info->launches = 1;
  info->tile_m = REL_WARPS;
  info->ctas = static_cast<int>(ctas * slices);
  info->set_route("paged_release");
  return cudaGetLastError();
}

}  // namespace mcb
