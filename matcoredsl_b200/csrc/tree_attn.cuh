// Shared by the tensor-core kernels of the attention over a paged cache
// (tree_attn_tc.cu, tree_attn_few.cu): how units of rows and their key tiles are
// shared out over the CTAs, which keys a row sees, and the launch that joins the
// parts of a unit.
//
// A unit is one request, one key head and up to ROWS of the request's rows
// (row = new token x query heads of the group); its keys are cut into tiles of
// 128. Every CTA takes an equal share of all units' tiles, in order, so a long
// context is split over many CTAs and many short ones are packed into one. The
// share is found on the device from the lengths: nothing is read by the host. A
// unit that lies in one CTA is finished there; the parts of a unit that spans
// CTAs go to scratch (at most two per CTA) and a second launch joins them in
// their order.
//
// The arithmetic of the shares is 32-bit; tree_attn_tc_ok() bounds it for requests that
// share no token. Where cu_new descends somewhere they may, so then nothing is
// shared out: no token belongs to a request.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace mcb {
namespace tree {

constexpr int BK = 128;  // keys per tile
constexpr uint32_t kNoRow = 0xffffffffu;

// A CTA's part of a unit.
struct Segment {
  int32_t kind;          // kWhole, kHead, kTail, or kEnd
  int32_t b, head;       // request, key head
  int32_t row0, nrows;   // rows of the request
  int32_t tok0;          // first new token
  int32_t prefix, keys;  // position of the first new token; keys there are
  int32_t tile0, ntiles;
};
enum : int32_t { kEnd = -1, kWhole = 0, kHead = 1, kTail = 2 };

struct TreeParams {
  TreeAttn a;
  float c;             // |scale| * log2(e)
  FastDiv block, group;
  int32_t heads_per_kv, most_keys;  // most_keys: what a block table row can hold
  uint32_t step[2][2];  // block and row strides of K and V in 16 bytes
  int32_t row_bits;     // bits of a row within a block
  float *partial;      // [2 * CTAs][ROWS][HD] outputs, then [2 * CTAs][ROWS][2] (max, sum)
  TreeAttnPart *part;  // [CTAs]
  uint32_t *status;
};


__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return kF16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
// 16 bytes to shared memory, zeros when `bytes` is 0.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}
// One arrival on `bar` once this thread's copies so far have landed. The
// copies are generic-proxy writes: whoever waits on the barrier fences before a
// tensor-core instruction reads them.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// One request's lengths, clipped to the tensors. tok0 and rows are those of the tokens
// inside [0, T). prefix is the position of the first new token (which the bits of a
// mask count from) or, without a mask, of the first one inside: a row's own key
// counts from there, and all rows see the keys before.
struct Request {
  int32_t tok0, rows, prefix, keys;
  bool descends;                     // cu_new does, at this request
};
__host__ __device__ __forceinline__ Request load_request(const TreeParams &p, int64_t b) {
  const TreeAttn &a = p.a;
  Request r;
  const int64_t c0 = a.cu[b], c1 = a.cu[b + 1], kv = max(0, a.kv_lens[b]);
  const int64_t first = max(c0, static_cast<int64_t>(0));
  const int64_t in = max(static_cast<int64_t>(0), min(c1, a.tokens) - first);
  r.tok0 = static_cast<int32_t>(first);
  r.rows = static_cast<int32_t>(in) * p.heads_per_kv;
  // (A mask has fewer than 2^31 bits a row: a token count past that is as good as that.)
  r.prefix = static_cast<int32_t>(
      kv - (a.mask ? min(c1 - c0, static_cast<int64_t>(0x7fffffff)) : c1 - first));
  r.keys = static_cast<int32_t>(min(kv, static_cast<int64_t>(p.most_keys)));
  r.descends = c1 < c0;
  return r;
}
// Key tiles of row tile `rt`: without a mask the rows see no key past the
// last one's own.
template <int ROWS>
__host__ __device__ __forceinline__ int32_t unit_tiles(const TreeParams &p, const Request &r,
                                                       int32_t rt) {
  int32_t end = r.keys;
  if (!p.a.mask) {
    const int32_t last = min(r.rows, (rt + 1) * ROWS) - 1;
    const int64_t own = static_cast<int64_t>(r.prefix) + fast_div(last, p.group) + 1;
    end = static_cast<int32_t>(min(static_cast<int64_t>(end), max(own, static_cast<int64_t>(0))));
  }
  return end <= BK ? 1 : (end + BK - 1) / BK;
}
// What a unit costs beside its tiles, in tiles: queries, first scores, output. 16 or
// 32 rows: 1 (2 and 3 made decoding of 64 requests with up to 1000 keys 3 and 10%
// slower); 128 or 256 rows: 3 (1 made 24 wide trees 15% slower).
template <int ROWS>
__host__ __device__ constexpr int32_t unit_cost() {
  return ROWS <= 32 ? 1 : 3;
}
template <int ROWS>
__host__ __device__ __forceinline__ int32_t head_cost(const TreeParams &p, const Request &r) {
  const int32_t rts = (r.rows + ROWS - 1) / ROWS;
  if (p.a.mask) return rts ? rts * (unit_tiles<ROWS>(p, r, 0) + unit_cost<ROWS>()) : 0;
  int32_t sum = 0;
  for (int32_t rt = 0; rt < rts; ++rt) sum += unit_tiles<ROWS>(p, r, rt) + unit_cost<ROWS>();
  return sum;
}

// Bits of the 32 keys from position pos on that new token i (mask row `row`)
// may see; bit k is key pos + k.
__device__ __forceinline__ uint32_t visible_word(const TreeAttn &a, const uint32_t *row,
                                                 int32_t pos, int32_t prefix, int32_t i) {
  const int64_t j = static_cast<int64_t>(pos) - prefix;  // new token of bit 0
  if (j <= -32) return 0xffffffffu;
  if (!row) {
    const int64_t n = static_cast<int64_t>(i) - j + 1;  // keys up to the token itself
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
  }
  auto word = [&](int64_t w) -> uint32_t { return w >= 0 && w < a.mask_words ? row[w] : 0u; };
  if (j < 0) return (word(0) << -j) | ((1u << -j) - 1);
  const int32_t s = static_cast<int32_t>(j & 31);
  const uint32_t lo = word(j >> 5);
  return s ? (lo >> s) | (word((j >> 5) + 1) << (32 - s)) : lo;
}

// CTA `cta`'s share [w0, w1) of all units' costs. The first `extra` CTAs take
// share + 1, the others share.
struct Share {
  int32_t w0, w1, share, extra, cta;
  bool descends;  // cu_new does: nothing is shared out
};
__host__ __device__ __forceinline__ Share share_of(int32_t cta, int32_t grid, int32_t total,
                                                   bool usable, bool descends) {
  const int32_t ctas = descends ? 0 : min(grid, total);
  const bool works = cta < ctas && usable;
  Share s;
  s.share = works ? total / ctas : 0;
  s.extra = works ? total - s.share * ctas : 0;
  s.w0 = cta * s.share + min(cta, s.extra);
  s.w1 = works ? s.w0 + s.share + (cta < s.extra) : s.w0;
  s.cta = cta;
  s.descends = descends;
  return s;
}
// Costs of the requests b0 .. b1 - 1, up to one at which cu_new descends.
template <int ROWS>
__host__ __device__ __forceinline__ uint32_t requests_cost(const TreeParams &p, int64_t b0,
                                                           int64_t b1, bool &descends) {
  uint32_t sum = 0;
  for (int64_t b = b0; b < b1 && !descends; ++b) {
    const Request r = load_request(p, b);
    descends = r.descends;
    sum += static_cast<uint32_t>(head_cost<ROWS>(p, r)) * static_cast<uint32_t>(p.a.kv_heads);
  }
  return sum;
}

// This CTA's share, found by all THREADS threads of it (`scan`: THREADS / 32 words of
// shared memory), and where the requests that hold w0 begin.
template <int ROWS, int THREADS>
__device__ __forceinline__ Share find_share(const TreeParams &p, uint32_t *scan, bool usable,
                                            int64_t *start_b, int32_t *start_w) {
  const TreeAttn &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t per_thread = (a.requests + THREADS - 1) / THREADS;
  const int64_t b_first = threadIdx.x * per_thread;
  bool descends = false;
  const uint32_t mine =
      requests_cost<ROWS>(p, b_first, min(a.requests, b_first + per_thread), descends);
  uint32_t incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) scan[warp] = incl;
  descends = __syncthreads_or(descends) != 0;
  uint32_t total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const Share s = share_of(blockIdx.x, gridDim.x, static_cast<int32_t>(total), usable, descends);
  // The thread whose requests hold w0 leaves where they begin.
  const uint32_t w0 = static_cast<uint32_t>(s.w0);
  if (s.w0 < s.w1 && before <= w0 && w0 < before + mine) {
    *start_b = b_first;
    *start_w = static_cast<int32_t>(before);
  }
  __syncthreads();
  return s;
}

// One thread's walk over the segments of a share. A unit's cost lies as its tiles,
// then unit_cost() places that hold none.
template <int ROWS>
struct Walk {
  const TreeParams &p;
  const Share &sh;
  TreeAttnPart &part;  // the unit that starts in this CTA and ends in a later one
  Request r;
  int64_t b;
  int32_t w, head = 0, rt = 0, n = 0, at = 0;  // at: place within the unit of n tiles

  __host__ __device__ __forceinline__ Walk(const TreeParams &args, const Share &share, TreeAttnPart &first,
                                  int64_t start_b, int32_t start_w)
      : p(args), sh(share), part(first), b(start_b), w(share.w0) {
    if (sh.descends) part.parts = -1;
    if (w >= sh.w1) return;
    int32_t from = start_w;  // first place of request b
    r = load_request(p, b);
    int32_t per = head_cost<ROWS>(p, r);
    while (from + per * p.a.kv_heads <= w) {
      from += per * p.a.kv_heads;
      r = load_request(p, ++b);
      per = head_cost<ROWS>(p, r);
    }
    head = (w - from) / per;
    at = w - from - head * per;
    n = unit_tiles<ROWS>(p, r, 0);
    while (at >= n + unit_cost<ROWS>()) {
      at -= n + unit_cost<ROWS>();
      n = unit_tiles<ROWS>(p, r, ++rt);
    }
  }
  // False past the last segment.
  __host__ __device__ __forceinline__ bool next(Segment &sg) {
    while (w < sh.w1) {
      if (at >= n + unit_cost<ROWS>()) {  // a new unit
        if ((rt + 1) * ROWS < r.rows) {
          ++rt;
        } else {
          rt = 0;
          if (++head == p.a.kv_heads) {
            head = 0;
            do r = load_request(p, ++b);
            while (r.rows == 0);
          }
        }
        n = unit_tiles<ROWS>(p, r, rt);
        at = 0;
      }
      const int32_t take = min(n + unit_cost<ROWS>() - at, sh.w1 - w), tile0 = at;
      const int32_t unit0 = w - at;  // first place of the unit
      w += take;
      at += take;
      const int32_t tiles = min(take, n - tile0);
      if (tiles <= 0) continue;
      sg.kind = tile0 > 0 ? kHead : tiles == n ? kWhole : kTail;
      sg.b = static_cast<int32_t>(b);
      sg.head = head;
      sg.row0 = rt * ROWS;
      sg.nrows = min(r.rows - sg.row0, ROWS);
      sg.tok0 = r.tok0;
      sg.prefix = r.prefix;
      sg.keys = r.keys;
      sg.tile0 = tile0;
      sg.ntiles = tiles;
      if (sg.kind == kTail) {
        const int32_t last = unit0 + n - 1, big = sh.extra * (sh.share + 1);  // its last tile
        part.parts = (last < big ? last / (sh.share + 1) : sh.extra + (last - big) / sh.share) -
                     sh.cta + 1;
        part.tok0 = r.tok0;
        part.head = head;
        part.row0 = sg.row0;
        part.nrows = sg.nrows;
      }
      return true;
    }
    return false;
  }
};

// Joins the parts of the units that span CTAs, in their order; the last column
// of CTAs clears the tokens of no request.
template <int HD, int ROWS, bool kF16>
__global__ void __launch_bounds__(256) tree_attn_join_parts_kernel(const TreeParams p, int ctas) {
  grid_dependency_wait();  // launched while the parts are being made
  const TreeAttn &a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = p.heads_per_kv;
  if (blockIdx.x == ctas) {
    int64_t c0 = min(max(static_cast<int64_t>(a.cu[0]), static_cast<int64_t>(0)), a.tokens);
    int64_t c1 = max(c0, min(static_cast<int64_t>(a.cu[a.requests]), a.tokens));
    if (p.part[0].parts < 0) c0 = c1 = 0;  // no request has any
    const int64_t none = c0 + a.tokens - c1;  // tokens before the first and after the last request
    for (int64_t w = blockIdx.y * 8 + warp; w < none * a.heads; w += 8 * gridDim.y) {
      const int64_t at = w / a.heads, h = w - at * a.heads, t = at < c0 ? at : at - c0 + c1;
      uint32_t *o = reinterpret_cast<uint32_t *>(static_cast<char *>(a.o) +
                                                 (t * a.o_s[0] + h * a.o_s[1]) * 2);
      for (int d = lane; d < HD / 2; d += 32) o[d] = 0;
      if (lane == 0 && a.lse) a.lse[t * a.lse_s + h] = -INFINITY;
    }
    return;
  }
  const TreeAttnPart part = p.part[blockIdx.x];
  if (part.parts <= 0) return;
  const float2 *ml = reinterpret_cast<const float2 *>(p.partial +
                                                      static_cast<int64_t>(ctas) * 2 * ROWS * HD);
  // Part k: the tail slot of this CTA, then the head slots of the next ones.
  auto slot = [&](int k) -> int64_t {
    return (static_cast<int64_t>(blockIdx.x) + k) * 2 + (k == 0);
  };
  // A part lies by columns of four: column q of row r at q * ROWS + r. A thread
  // joins one column of one row, neighbours take neighbouring rows.
  const int rows = (part.nrows + 31) / 32 * 32;
  for (int w = blockIdx.y * 256 + threadIdx.x; w < rows * (HD / 4); w += 256 * gridDim.y) {
    const int q = w / rows, r = w - q * rows;
    if (r >= part.nrows) continue;
    // One pass with a running maximum, so that all loads are independent.
    float top = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int k = 0; k < part.parts; ++k) {
      const float2 z = ml[slot(k) * ROWS + r];
      const float4 y =
          reinterpret_cast<const float4 *>(p.partial + slot(k) * ROWS * HD)[q * ROWS + r];
      const float m = fmaxf(top, z.x), ref = m == -INFINITY ? 0.0f : m;
      const float f = ex2(z.x - ref), g = ex2(top - ref);
      top = m;
      l = fmaf(z.y, f, l * g);
      x.x = fmaf(y.x, f, x.x * g);
      x.y = fmaf(y.y, f, x.y * g);
      x.z = fmaf(y.z, f, x.z * g);
      x.w = fmaf(y.w, f, x.w * g);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int row = part.row0 + r, i = fast_div(row, p.group);
    const int64_t tok = static_cast<int64_t>(part.tok0) + i;
    const int head = part.head * group + row - i * group;
    *reinterpret_cast<uint2 *>(static_cast<char *>(a.o) +
                               (tok * a.o_s[0] + head * a.o_s[1] + 4 * q) * 2) =
        make_uint2(pack2<kF16>(x.x * inv, x.y * inv), pack2<kF16>(x.z * inv, x.w * inv));
    if (q == 0 && a.lse)
      a.lse[tok * a.lse_s + head] =
          l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.69314718055994531f;
  }
}

// The arguments that both kernels take.
inline TreeParams tree_params(const TreeAttn &a, void *scratch, int rows, int ctas,
                              uint32_t *status) {
  TreeParams p;
  p.a = a;
  p.c = fabsf(a.scale) * 1.4426950408889634f;
  p.block = make_div(a.block);
  p.heads_per_kv = a.heads / a.kv_heads;
  p.group = make_div(p.heads_per_kv);
  p.most_keys = static_cast<int32_t>(a.columns * a.block);
  for (int i = 0; i < 2; ++i) {
    p.step[0][i] = static_cast<uint32_t>(a.k_s[i] / 8);
    p.step[1][i] = static_cast<uint32_t>(a.v_s[i] / 8);
  }
  p.row_bits = p.block.shift - 31;  // blocks * block < 2^31, so block << bits | row < 2^32 - 1
  p.partial = static_cast<float *>(scratch);
  p.part = reinterpret_cast<TreeAttnPart *>(p.partial +
                                            static_cast<uint64_t>(ctas) * 2 * rows * (a.dim + 2));
  p.status = status;
  return p;
}
// The joining launch, scheduled as the first one's CTAs retire.
template <int HD, int ROWS, bool kF16>
cudaError_t launch_join(const TreeParams &p, int ctas, cudaStream_t stream) {
  const cudaError_t e = cudaGetLastError();  // the first launch's
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  // A thread per four columns of a row, in up to 16 CTAs a unit.
  constexpr int slices = (ROWS * HD / 4 + 255) / 256;
  cfg.gridDim = dim3(ctas + 1, slices < 16 ? slices : 16);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_attn_join_parts_kernel<HD, ROWS, kF16>, p, ctas);
}
inline uint64_t tree_scratch(const TreeAttn &a, int rows, int ctas) {
  return static_cast<uint64_t>(ctas) *
         (2ull * rows * (a.dim + 2) * sizeof(float) + sizeof(TreeAttnPart));
}

}  // namespace tree
}  // namespace mcb
