// Attention of drafted tokens over a paged cache for requests of few rows (a
// row = new token x query heads of the group), up to 16, with short contexts 32: bf16 or f16,
// head size 64 or 128, 16-byte aligned rows. (The mathematics and the masks:
// tree_attn.cu; how the work is shared out: tree_attn.cuh.)
//
// Bound: reading the cache. With R rows a key and value row of 4 * HD bytes
// take 4 * HD * R operations, far below what a CTA can do in the time of the
// read, so the kernel is built around the copies: six half tiles (128 keys or
// values, 32 KiB at HD = 128) of an SM are in shared memory or on their way. The products
// use warp-level matrix instructions on 16-row tiles: the 128-row tile of a
// tcgen05 instruction would be empty but for a few rows, and its softmax would
// run on one warp.
//
// 8 warps share a tile of 128 keys. Warp w takes keys 16w .. 16w + 15 for the
// scores S = Q K^T, makes the weights of those keys and leaves them in shared
// memory as 16-bit numbers; then it takes the HD / 8 columns w of O = P V for all
// 128 keys. So K and V are read from shared memory once, O needs no joining across
// warps, and the only things that the warps share are the weights and a reference
// maximum per row. The maximum moves when a score passes it by 8 (in powers of
// two): whether any does is one barrier with an OR, and the exchange of the
// maxima happens only then.
//
// A ninth warp walks over the segments (a CTA's part of a unit), prepares where
// each key of a tile lies and copies the queries and, where a cache block is a
// whole box of a tensor map (8 rows or more, and a divisor or multiple of 128),
// keys and values by TMA. Blocks of other sizes are copied row by row with
// cp.async by eight more warps: 64 requests of up to 8192 keys take 205 us with blocks of
// 24, 177 with blocks of 16 (1.09 GB at 6.2 TB/s). (The compute warps issuing those copies themselves,
// between their products, took 2.4 us a tile: 1.6 thousand cycles of the copies'
// own.)
#include "tree_attn.cuh"

namespace mcb {
namespace {
using namespace tree;

constexpr int WARPS = 8;
constexpr int COMPUTE = WARPS * 32;
constexpr int COPIERS = 256;  // threads of the row-by-row copies (128: 270 us where these took 211)
template <bool kTma>
constexpr int threads() {
  return COMPUTE + 32 + (kTma ? 0 : COPIERS);
}
// Half tiles (keys or values) in shared memory. With 3 of head size 128 two CTAs fit
// into an SM, with one CTA they are 1% slower than 6.
template <int HD, int MT, bool kTma>
constexpr int halves() {
  return HD == 128 && MT == 1 && kTma ? 3 : 6;
}
constexpr int TILES = 4;   // ring of prepared tiles
constexpr int QBUFS = 2;

struct Tile {
  uint32_t where[BK];  // block << bits | row of each key, kNoRow: nowhere
  uint32_t valid[4];   // bit per key
  Segment seg;
  int32_t tile;        // of the segment
};

template <int HD, int MT, bool kTma>
struct Smem {
  static constexpr int HALVES = halves<HD, MT, kTma>();
  uint8_t kv[HALVES][BK * HD * 2];
  uint8_t q[QBUFS][16 * MT * HD * 2];
  uint8_t p[16 * MT * BK * 2];  // weights; maxima and sums of the warps in between
  Tile tile[TILES];
  uint64_t full[TILES], empty[TILES];
  uint64_t kv_full[HALVES], kv_empty[HALVES], q_full[QBUFS], q_empty[QBUFS];
  int64_t start_b;
  int32_t start_w;
  int abort_flag, dirty;
};
static_assert(sizeof(Smem<128, 2, true>) <= 232448, "exceeds the shared memory per block");

struct Params : TreeParams {
  float sign;         // of the scale
  int32_t page_rows;  // rows of a box (128 without TMA), a power of two
  int32_t give_up;    // self-test: at a segment's first (0) or last (1) tile
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// D += A B, 16x8x16: A 16 rows x 16, B 16 x 8 columns, f32 sums.
template <bool kF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  if (kF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// One box: 64 columns of `page_rows` rows, then the next 64 columns of them.
__device__ __forceinline__ void tma_load_box(void *dst, const void *tmap, uint64_t *bar,
                                             int32_t row, int32_t head, int32_t block) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %3, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(head),
      "r"(block)
      : "memory");
}
// Byte offset of 16-byte piece c of a row of a matrix cut into boxes of `page`
// rows (a power of two): within a box 64 columns of all rows after the other,
// within a row's 128 bytes the pieces permuted by the row (TMA's 128-byte swizzle),
// so that eight rows of one piece, or one row of eight, touch all banks.
template <int COLS>
__device__ __forceinline__ uint32_t piece_at(int row, int c, int page) {
  const uint32_t swz = ((c & 7) ^ (row & 7)) << 4;
  if (COLS == 64) return row * 128 + swz;
  return (row + (row & -page) + (c >> 3) * page) * 128 + swz;
}

// kTest: one compute warp behaves as if its wait for a tile's values had run out
// (launch_tree_attn_stall_selftest).
template <int HD, int MT, bool kF16, bool kTma, bool kTest>
__global__ void __launch_bounds__(threads<kTma>())
    tree_attn_few_kernel(const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const Params p) {
  constexpr int ROWS = 16 * MT;
  constexpr int PIECES = HD / 8;  // 16-byte pieces of a key, value or query row
  constexpr int NT = HD / 64;     // 8-column tiles of O per warp
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int HALVES = halves<HD, MT, kTma>();
  Smem<HD, MT, kTma> &sm = *reinterpret_cast<Smem<HD, MT, kTma> *>(smem_raw);
  const TreeAttn &a = p.a;
  volatile int *abort_flag = &sm.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads_per_kv;

  if (threadIdx.x == 0) {
    for (int s = 0; s < TILES; ++s) {
      mbar_init(&sm.full[s], 32);
      mbar_init(&sm.empty[s], COMPUTE + (kTma ? 0 : COPIERS));
    }
    for (int s = 0; s < HALVES; ++s) {
      mbar_init(&sm.kv_full[s], kTma ? 1 : COPIERS);
      mbar_init(&sm.kv_empty[s], COMPUTE);
    }
    for (int s = 0; s < QBUFS; ++s) {
      mbar_init(&sm.q_full[s], 32);
      mbar_init(&sm.q_empty[s], COMPUTE);
    }
    // The swizzle needs a 1024-byte aligned base.
    sm.abort_flag = (smem_u32(smem_raw) & 1023u) != 0;
    if (sm.abort_flag && p.status) atomicOr(p.status, kErrBadLaunch);
    sm.dirty = 0;
    fence_mbar_init();
  }
  if (kTma && warp == WARPS && lane == 0) {
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  grid_launch_dependents();
  const Share share = find_share<ROWS, threads<kTma>()>(
      p, reinterpret_cast<uint32_t *>(sm.p), true, &sm.start_b, &sm.start_w);

  if (warp == WARPS) {
    // ---------------- tiles, queries and (TMA) keys and values ----------------
    TreeAttnPart part{};
    Walk<ROWS> walk(p, share, part, sm.start_b, sm.start_w);
    Segment sg;
    uint32_t count = 0, segs = 0, armed = 0;  // armed: half tiles that TMA was set to fill
    bool ok = !*abort_flag;
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
      ok = __all_sync(0xffffffffu,
                      mbar_wait(bar, parity, abort_flag, p.status, kErrTimeoutEmpty)) != 0;
      return ok;
    };
    auto slot_free = [&]() -> bool {
      return wait(&sm.empty[count % TILES], ((count / TILES) & 1) ^ 1);
    };
    while (ok && walk.next(sg)) {
      if (!wait(&sm.q_empty[segs % QBUFS], ((segs / QBUFS) & 1) ^ 1)) break;
      {
        // Rows past the last one are zero.
        const int piece = lane % PIECES;
        const char *q = static_cast<const char *>(a.q) +
                        (sg.tok0 * a.q_s[0] + sg.head * group * a.q_s[1] + piece * 8) * 2;
        const uint32_t to = smem_u32(sm.q[segs % QBUFS]);
#pragma unroll 4
        for (int r = lane / PIECES; r < ROWS; r += 32 / PIECES) {
          const bool live = r < sg.nrows;
          const int row = sg.row0 + (live ? r : 0), tok = fast_div(row, p.group);
          cp_async16(to + piece_at<HD>(r, piece, ROWS),
                     q + (tok * a.q_s[0] + (row - tok * group) * a.q_s[1]) * 2, live ? 16 : 0);
        }
        cp_async_arrive(&sm.q_full[segs % QBUFS]);
        ++segs;
      }
      const int32_t *table = a.table + sg.b * a.table_stride;
      int32_t blk[4];
      uint32_t col[4];
      auto look_up = [&](int j) {  // blocks of this lane's keys of tile j
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = (sg.tile0 + j) * BK + 32 * u + lane;
          col[u] = fast_div(key, p.block);
          blk[u] = key < sg.keys && j < sg.ntiles ? table[col[u]] : -1;
        }
      };
      look_up(0);
      for (int j = 0; j < sg.ntiles; ++j) {
        if (!slot_free()) break;
        Tile *t = &sm.tile[count % TILES];
        const int key0 = (sg.tile0 + j) * BK;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = key0 + 32 * u + lane;
          const bool good = blk[u] >= 0 && blk[u] < a.blocks;
          t->where[32 * u + lane] =
              good ? (static_cast<uint32_t>(blk[u]) << p.row_bits) | (key - col[u] * a.block) : kNoRow;
          const uint32_t bits = __ballot_sync(0xffffffffu, good);
          if (lane == 0) t->valid[u] = bits;
        }
        if (lane == 0) {
          t->seg = sg;
          t->tile = j;
        }
        mbar_arrive(&sm.full[count % TILES]);
        look_up(j + 1);
        if (kTma) {
          __syncwarp();
          const int pages = BK / p.page_rows;
          // Box of this lane: outside the cache (zeros) where there is no block.
          const uint32_t w = lane < pages ? t->where[lane * p.page_rows] : kNoRow;
          const int32_t block = w == kNoRow ? static_cast<int32_t>(a.blocks)
                                            : static_cast<int32_t>(w >> p.row_bits);
          const int32_t row = w == kNoRow ? 0 : static_cast<int32_t>(w & ((1u << p.row_bits) - 1));
#pragma unroll
          for (int value = 0; value < 2; ++value) {
            const uint32_t half = 2 * count + value, s = half % HALVES;
            if (!wait(&sm.kv_empty[s], ((half / HALVES) & 1) ^ 1)) break;
            if (lane == 0) mbar_arrive_expect_tx(&sm.kv_full[s], BK * HD * 2);
            armed = half + 1;
            __syncwarp();
            if (lane < pages)
              tma_load_box(sm.kv[s] + lane * p.page_rows * (HD * 2), value ? &tv : &tk,
                           &sm.kv_full[s], row, sg.head, block);
          }
          if (!ok) break;
        }
        ++count;
      }
    }
    if (ok && slot_free()) {
      if (lane == 0) sm.tile[count % TILES].seg.kind = kEnd;
      mbar_arrive(&sm.full[count % TILES]);
    }
    if (!ok) {
      // Given up: the products did not wait for the copies that are still on their way
      // into this CTA's shared memory. Each stage's last phase ends them.
      for (uint32_t s = 0; s < HALVES && s < armed; ++s)
        mbar_wait(&sm.kv_full[s], ((armed - 1 - s) / HALVES) & 1, nullptr, p.status,
                  kErrTimeoutDrain);
    }
    cp_async_wait_all();
    if (lane == 0) p.part[blockIdx.x] = part;
    return;
  }
  if (!kTma && warp > WARPS) {
    // ---------------- row-by-row copies of keys and values ----------------
    const int tid = threadIdx.x - COMPUTE - 32, piece = tid % PIECES;
    constexpr int STEP = COPIERS / PIECES;
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
      return mbar_wait(bar, parity, abort_flag, p.status, kErrTimeoutEmpty);
    };
    for (uint32_t t = 0;; ++t) {
      if (!wait(&sm.full[t % TILES], (t / TILES) & 1)) break;
      const Tile &d = sm.tile[t % TILES];
      if (d.seg.kind == kEnd) break;
      bool ok = true;
      for (int value = 0; value < 2 && ok; ++value) {
        const uint32_t half = 2 * t + value, s = half % HALVES;
        if (!(ok = wait(&sm.kv_empty[s], ((half / HALVES) & 1) ^ 1))) break;
        const char *base = static_cast<const char *>(value ? a.v : a.k) +
                           (d.seg.head * (value ? a.v_s[2] : a.k_s[2]) + piece * 8) * 2;
        const uint32_t blk_step = p.step[value][0], row_step = p.step[value][1];
        const uint32_t dst = smem_u32(sm.kv[s]);
#pragma unroll 8
        for (int r = tid / PIECES; r < BK; r += STEP) {
          const uint32_t w = d.where[r];
          const bool none = w == kNoRow;
          const uint32_t at =
              (w >> p.row_bits) * blk_step + (w & ((1u << p.row_bits) - 1)) * row_step;
          cp_async16(dst + piece_at<HD>(r, piece, BK), base + static_cast<uint64_t>(none ? 0u : at) * 16,
                     none ? 0 : 16);
        }
        cp_async_arrive(&sm.kv_full[s]);
      }
      if (!ok) break;
      mbar_arrive(&sm.empty[t % TILES]);
    }
    cp_async_wait_all();
    return;
  }

  // ---------------- products ----------------
  const int tid = threadIdx.x;
  const int quad = lane >> 2, ql = lane & 3, page = kTma ? p.page_rows : BK;
  float o[MT][NT][4], ref[MT][2], l[MT][2];
  uint32_t seg_no = 0;
  // A warp whose wait runs out says so at the tile's next barrier with an OR, and the
  // warps that found the end come to one, too: all warps leave in the same turn, or a
  // warp would wait at a barrier for others that have left.
  bool ok = true;
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    ok = mbar_wait_warp(bar, parity, abort_flag, p.status, kErrTimeoutFull) && ok;
  };
  // This thread is done with a half tile. TMA will write its place through the async
  // proxy, which only a proxy fence orders behind this thread's reads (and writes) of it:
  // without it, one call in 4000 (of 300 requests whose keys and values lie in L2) had
  // rows of later keys among the values. (Decoding of 64 requests with two CTAs an SM:
  // 177 us with it, 180 without; with one CTA 198 and 187.)
  auto release = [&](uint64_t *bar) {
    if (kTma) fence_async_smem();
    mbar_arrive(bar);
  };
  for (uint32_t t = 0;; ++t) {
    const uint32_t kh = 2 * t, vh = kh + 1;  // half tiles
    wait(&sm.full[t % TILES], (t / TILES) & 1);
    const Tile &d = sm.tile[t % TILES];
    if (ok && d.seg.kind == kEnd) {
      if (named_bar_or(2, COMPUTE, false)) named_bar_or(1, COMPUTE, false);
      break;
    }
    if (ok && d.tile == 0) wait(&sm.q_full[seg_no % QBUFS], (seg_no / QBUFS) & 1);
    if (ok) wait(&sm.kv_full[kh % HALVES], (kh / HALVES) & 1);
    if (!ok) {
      named_bar_or(2, COMPUTE, true);
      named_bar_or(1, COMPUTE, true);
      return;
    }
    if (d.tile == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        ref[m][0] = ref[m][1] = -INFINITY;
        l[m][0] = l[m][1] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.0f;
      }
    }
    const Segment &sg = d.seg;
    const int pos0 = (sg.tile0 + d.tile) * BK;
    // ---- scores of this warp's 16 keys ----
    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.0f;
    {
      const uint32_t kb = smem_u32(sm.kv[kh % HALVES]);
      const uint32_t qb = smem_u32(sm.q[seg_no % QBUFS]);
      // K: matrices (keys 0-7, piece 2k), (0-7, 2k + 1), (8-15, 2k), (8-15, 2k + 1);
      // Q: (rows 0-7, 2k), (8-15, 2k), (0-7, 2k + 1), (8-15, 2k + 1).
      const int krow = 16 * warp + (lane & 7) + ((lane >> 4) << 3), kpc = (lane >> 3) & 1;
      const int qrow = lane & 15, qpc = lane >> 4;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t kf[4];
        ldmatrix4(kf, kb + piece_at<HD>(krow, 2 * k + kpc, page));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t qf[4];
          ldmatrix4(qf, qb + piece_at<HD>(16 * m + qrow, 2 * k + qpc, ROWS));
          mma<kF16>(s[m][0], qf, kf[0], kf[1]);
          mma<kF16>(s[m][1], qf, kf[2], kf[3]);
        }
      }
    }
    release(&sm.kv_empty[kh % HALVES]);
    // ---- masks ----
    const uint32_t good = d.valid[warp >> 1] >> (16 * (warp & 1));
    const bool drafts = pos0 + BK > sg.prefix;  // the tile holds new tokens' keys
    if (drafts || (good & 0xffffu) != 0xffffu) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = min(sg.row0 + 16 * m + quad + 8 * h, sg.row0 + sg.nrows - 1);
          const int i = fast_div(row, p.group);
          const uint32_t *mask_row =
              a.mask ? a.mask + (static_cast<int64_t>(sg.tok0) + i) * a.mask_stride : nullptr;
          const uint32_t see = good & visible_word(a, mask_row, pos0 + 16 * warp, sg.prefix, i);
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((see >> (8 * n + 2 * ql + e)) & 1u)) s[m][n][2 * h + e] = -p.sign * INFINITY;
        }
    }
    // ---- reference maxima: moved when a score passes them by 8 powers of two ----
    bool need = false;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[m][n][2 * h + e] *= p.sign;
            mx = fmaxf(mx, s[m][n][2 * h + e]);
          }
        need |= mx > -INFINITY && !((mx - ref[m][h]) * p.c <= 8.0f);
      }
    if (named_bar_or(2, COMPUTE, need)) {
      if (named_bar_or(1, COMPUTE, false)) return;
      float *most = reinterpret_cast<float *>(sm.p);  // [WARPS][ROWS]
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(fmaxf(s[m][0][2 * h], s[m][0][2 * h + 1]),
                           fmaxf(s[m][1][2 * h], s[m][1][2 * h + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (ql == 0) most[warp * ROWS + 16 * m + quad + 8 * h] = mx;
        }
      named_bar_sync(3, COMPUTE);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = ref[m][h];
#pragma unroll
          for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, most[w * ROWS + 16 * m + quad + 8 * h]);
          // While the old maximum is -inf, O and l are zero.
          const float f = ref[m][h] == -INFINITY ? 1.0f : ex2((ref[m][h] - mx) * p.c);
          ref[m][h] = mx;
          l[m][h] *= f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[m][n][2 * h] *= f;
            o[m][n][2 * h + 1] *= f;
          }
        }
      named_bar_sync(3, COMPUTE);  // the maxima are read: weights may take their place
    }
    // ---- weights ----
    const uint32_t pb = smem_u32(sm.p);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mc = ref[m][h] == -INFINITY ? 0.0f : ref[m][h] * p.c;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float e0 = ex2(fmaf(s[m][n][2 * h], p.c, -mc));
          const float e1 = ex2(fmaf(s[m][n][2 * h + 1], p.c, -mc));
          l[m][h] += e0 + e1;
          const uint32_t at = pb + piece_at<BK>(16 * m + quad + 8 * h, 2 * warp + n, ROWS) + 4 * ql;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(pack2<kF16>(e0, e1)) : "memory");
        }
      }
    wait(&sm.kv_full[vh % HALVES], (vh / HALVES) & 1);
    if (kTest && warp == 0 && d.tile == (p.give_up ? sg.ntiles - 1 : 0)) {
      if (lane == 0) atomicOr(p.status, kErrTimeoutFull);
      *abort_flag = 1;
      ok = false;
    }
    if (named_bar_or(3, COMPUTE, !ok)) return;  // else the weights are there
    uint8_t *values = sm.kv[vh % HALVES];
    if (drafts) {
      // New tokens' values that are not finite become 0: 0 x inf must not reach
      // the rows that do not see them. The others add them at the end. Rows past
      // the last key hold anything and become 0.
      constexpr uint32_t E = kF16 ? 0x7c00u : 0x7f80u;
      for (int i = tid; i < BK * PIECES; i += COMPUTE) {
        const int r = i / PIECES, pos = pos0 + r;
        if (pos < sg.prefix) continue;
        uint4 *at = reinterpret_cast<uint4 *>(values + piece_at<HD>(r, i % PIECES, page));
        if (pos >= sg.keys) {
          *at = make_uint4(0, 0, 0, 0);
          continue;
        }
        uint4 w = *at;
        uint32_t *x = reinterpret_cast<uint32_t *>(&w);
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((x[k] & E) == E) {
            x[k] &= 0xffff0000u;
            bad = true;
          }
          if ((x[k] & (E << 16)) == (E << 16)) {
            x[k] &= 0xffffu;
            bad = true;
          }
        }
        if (bad) {
          *at = w;
          *static_cast<volatile int *>(&sm.dirty) = 1;
        }
      }
      named_bar_sync(3, COMPUTE);
    }
    // ---- O += P V, this warp's HD / 8 columns ----
    {
      const uint32_t vb = smem_u32(values);
      const int prow = lane & 15, ppc = lane >> 4;
      uint32_t held[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < BK / 16; ++k) {
        uint32_t vf[4];
        if (NT == 2)  // keys 0-7 and 8-15 of the step, pieces 2w and 2w + 1
          ldmatrix4_trans(vf,
                          vb + piece_at<HD>(16 * k + (lane & 15), 2 * warp + (lane >> 4), page));
        else if (k % 2 == 0)  // one piece, two steps
          ldmatrix4_trans(vf, vb + piece_at<HD>(16 * k + lane, warp, page));
        if (NT == 1 && k % 2 == 1) {
          vf[0] = held[0];
          vf[1] = held[1];
        } else if (NT == 1) {
          held[0] = vf[2];
          held[1] = vf[3];
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t pf[4];
          ldmatrix4(pf, pb + piece_at<BK>(16 * m + prow, 2 * k + ppc, ROWS));
          mma<kF16>(o[m][0], pf, vf[0], vf[1]);
          if (NT == 2) mma<kF16>(o[m][NT - 1], pf, vf[2], vf[3]);
        }
      }
    }
    release(&sm.kv_empty[vh % HALVES]);
    if (d.tile + 1 == sg.ntiles) {
      // ---- the segment's output ----
      mbar_arrive(&sm.q_empty[seg_no % QBUFS]);
      ++seg_no;
      named_bar_sync(3, COMPUTE);  // the weights are read: sums may take their place
      float *sums = reinterpret_cast<float *>(sm.p);  // [WARPS][ROWS]
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = l[m][h];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (ql == 0) sums[warp * ROWS + 16 * m + quad + 8 * h] = x;
        }
      named_bar_sync(3, COMPUTE);
      const bool whole = sg.kind == kWhole;
      const int64_t part_slot = static_cast<int64_t>(blockIdx.x) * 2 + (sg.kind == kTail);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * m + quad + 8 * h;
          if (r >= sg.nrows) continue;
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) sum += sums[w * ROWS + r];
          const int row = sg.row0 + r, i = fast_div(row, p.group);
          const int64_t tok = static_cast<int64_t>(sg.tok0) + i;
          const int head = sg.head * group + row - i * group;
          float x[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            x[n][0] = o[m][n][2 * h];
            x[n][1] = o[m][n][2 * h + 1];
          }
          const int d0 = 8 * NT * warp + 2 * ql;  // columns d0, d0 + 1 and, 8 further, two more
          if (*static_cast<volatile int *>(&sm.dirty)) {
            const uint32_t *mask_row = a.mask ? a.mask + tok * a.mask_stride : nullptr;
            const int k1 = min((sg.tile0 + sg.ntiles) * BK, sg.keys);
            for (int pos = max(max(sg.tile0 * BK, sg.prefix), 0); pos < k1; ++pos) {
              if (!(visible_word(a, mask_row, pos, sg.prefix, i) & 1u)) continue;
              const int col = pos / a.block;
              const int32_t blk = a.table[sg.b * a.table_stride + col];
              if (blk < 0 || blk >= a.blocks) continue;
              const int64_t at = blk * a.v_s[0] + (pos - col * a.block) * a.v_s[1] +
                                 sg.head * a.v_s[2] + d0;
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float v =
                      kF16 ? __half2float(static_cast<const __half *>(a.v)[at + 8 * n + e])
                           : __bfloat162float(
                                 static_cast<const __nv_bfloat16 *>(a.v)[at + 8 * n + e]);
                  if (!(fabsf(v) < INFINITY)) x[n][e] += v;
                }
            }
          }
          const float mc = ref[m][h] == -INFINITY ? -INFINITY : ref[m][h] * p.c;
          if (whole) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint32_t *out = reinterpret_cast<uint32_t *>(
                static_cast<char *>(a.o) + (tok * a.o_s[0] + head * a.o_s[1] + d0) * 2);
#pragma unroll
            for (int n = 0; n < NT; ++n) out[4 * n] = pack2<kF16>(x[n][0] * inv, x[n][1] * inv);
            if (a.lse && warp == 0 && ql == 0)
              a.lse[tok * a.lse_s + head] =
                  sum == 0.0f ? -INFINITY
                              : ((mc == -INFINITY ? 0.0f : mc) + log2f(sum)) * 0.69314718055994531f;
          } else {
            // Columns of four, a row after the other: this pair is half of one.
            float *out = p.partial + part_slot * ROWS * HD + r * 4 + (ql & 1) * 2;
#pragma unroll
            for (int n = 0; n < NT; ++n)
              *reinterpret_cast<float2 *>(out + (d0 / 4 + 2 * n) * (ROWS * 4)) =
                  make_float2(x[n][0], x[n][1]);
            if (warp == 0 && ql == 0)
              reinterpret_cast<float2 *>(p.partial +
                                         static_cast<int64_t>(gridDim.x) * 2 * ROWS *
                                             HD)[part_slot * ROWS + r] = make_float2(mc, sum);
          }
        }
    }
    mbar_arrive(&sm.empty[t % TILES]);
  }
}

// Row tiles of 16 that a CTA takes, 0 where tcgen05 is the faster. By the rows that a
// request has on average; of drafted tokens some requests have more than that, and
// one whose rows do not fit reads its context twice, so a tile counts as 12 rows then.
//   one tile: 64 requests of 4 rows, up to 8192 keys 177 us (216 on tcgen05, 247 with two
//     tiles); 32 of 16 rows 99 (107); of 12 to 20 rows 217 (215), hence 12.
//   two tiles: 256 requests of 16 to 32 rows, up to 1000 keys 189 us (226 on tcgen05, whose
//     units cost three tiles more than their keys), 2000 keys 301 (322), 4000 keys 514
//     (482); 64 requests with 4000 keys 150 (132), 8192 keys 259 (225); of 20 to 40 rows
//     with 1000 keys 72 (70). So they are taken where no context can pass 2048 keys.
int row_tiles(const TreeAttn &a) {
  const int64_t rows = a.tokens * (a.heads / a.kv_heads);
  const int64_t tile = a.tokens == a.requests ? 16 : 12;
  if (rows <= tile * a.requests) return 1;
  return rows <= 2 * tile * a.requests && a.columns * a.block <= 2048 ? 2 : 0;
}
// CTAs per SM: two where they fit (228 KB of shared memory, 1 KB kept per CTA) and there
// are enough units, else contexts are cut into more parts than the second CTA is worth.
// Head size 128, 8 key heads, up to 8192 keys: 1 request 24.6 us with one, 33 with two; 8
// requests 41 both; 20 requests 73.7 and 68.5, 32 requests 107 and 99, 64 requests 198
// and 177; up to 1000 keys 16 requests 21.5 both, 24 requests 24.6 and 22.6, 64
// requests 45 and 37. Head size 64: 1 request 28.6 and 35, 4 requests 26.6 both, 8
// requests 32.8 and 30.4.
template <int HD, int MT, bool kTma>
int per_sm(const TreeAttn &a, int sms) {
  if (2 * (sizeof(Smem<HD, MT, kTma>) + 1024) > 233472) return 1;
  return a.requests * a.kv_heads >= (HD == 128 ? sms : sms / 4) ? 2 : 1;
}

// Rows of a TMA box, 0 where blocks are no whole boxes.
int page_rows(const TreeAttn &a) {
  if (a.block % BK == 0) return BK;
  return a.block >= 8 && BK % a.block == 0 ? a.block : 0;
}
bool cache_map(CUtensorMap *map, const TreeAttn &a, const void *base, const int64_t *st, bool f16,
               int rows) {
  const uint64_t chunks = a.dim / 64;
  const uint64_t dims[5] = {64, static_cast<uint64_t>(a.block), chunks,
                            static_cast<uint64_t>(a.kv_heads), static_cast<uint64_t>(a.blocks)};
  const uint64_t strides[4] = {static_cast<uint64_t>(st[1]) * 2, 128,
                               static_cast<uint64_t>(st[2]) * 2, static_cast<uint64_t>(st[0]) * 2};
  const uint32_t box[5] = {64, static_cast<uint32_t>(rows), static_cast<uint32_t>(chunks), 1, 1};
  return encode_tmap_5d(map,
                        f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int HD, int MT, bool kF16, bool kTma, bool kTest = false>
cudaError_t run(const TreeAttn &a, const CUtensorMap &tk, const CUtensorMap &tv, void *scratch,
                uint32_t *status, int sms, cudaStream_t stream, LaunchInfo *info,
                int give_up = 0) {
  const int ctas = sms * per_sm<HD, MT, kTma>(a, sms);
  Params p;
  static_cast<TreeParams &>(p) = tree_params(a, scratch, 16 * MT, ctas, status);
  p.sign = a.scale < 0.0f ? -1.0f : 1.0f;
  p.page_rows = kTma ? page_rows(a) : BK;
  p.give_up = give_up;
  auto kernel = tree_attn_few_kernel<HD, MT, kF16, kTma, kTest>;
  constexpr int smem = static_cast<int>(sizeof(Smem<HD, MT, kTma>));
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<ctas, threads<kTma>(), smem, stream>>>(tk, tv, p);
  info->launches = 2;
  info->tile_m = 16 * MT;
  info->tile_n = BK;
  info->tile_k = HD;
  info->stages = halves<HD, MT, kTma>();
  info->ctas = ctas;
  info->set_route("tree_attention_few_rows");
  return launch_join<HD, 16 * MT, kF16>(p, ctas, stream);
}

template <int HD, bool kF16>
cudaError_t run_rows(const TreeAttn &a, void *scratch, uint32_t *status, int sms,
                     cudaStream_t stream, LaunchInfo *info) {
  CUtensorMap tk{}, tv{};
  const int rows = page_rows(a);
  const bool tma =
      rows && cache_map(&tk, a, a.k, a.k_s, kF16, rows) && cache_map(&tv, a, a.v, a.v_s, kF16, rows);
  if (row_tiles(a) == 1)
    return tma ? run<HD, 1, kF16, true>(a, tk, tv, scratch, status, sms, stream, info)
               : run<HD, 1, kF16, false>(a, tk, tv, scratch, status, sms, stream, info);
  return tma ? run<HD, 2, kF16, true>(a, tk, tv, scratch, status, sms, stream, info)
             : run<HD, 2, kF16, false>(a, tk, tv, scratch, status, sms, stream, info);
}

}  // namespace

bool tree_attn_few_ok(const TreeAttn &a, int dtype) {
  return tree_attn_tc_ok(a, dtype) && row_tiles(a) > 0;
}

uint64_t tree_attn_few_scratch(const TreeAttn &a, int sms) {
  const bool one = row_tiles(a) == 1;
  const int n = a.dim == 128 ? (one ? per_sm<128, 1, true>(a, sms) : per_sm<128, 2, true>(a, sms))
                             : (one ? per_sm<64, 1, true>(a, sms) : per_sm<64, 2, true>(a, sms));
  return tree_scratch(a, one ? 16 : 32, n * sms);
}

cudaError_t launch_tree_attn_few(const TreeAttn &a, int dtype, void *scratch, uint32_t *status,
                                 int sms, cudaStream_t stream, LaunchInfo *info) {
  const bool f16 = dtype == MCB_DTYPE_F16;
  if (a.dim == 128)
    return f16 ? run_rows<128, true>(a, scratch, status, sms, stream, info)
               : run_rows<128, false>(a, scratch, status, sms, stream, info);
  return f16 ? run_rows<64, true>(a, scratch, status, sms, stream, info)
             : run_rows<64, false>(a, scratch, status, sms, stream, info);
}

// Self-test of the way out of a wait that ran out: a call on one row tile of head size 64 in which
// one warp of each CTA gives up at its segment's first (last = false) or last tile. bf16,
// blocks of 128; `a` must pass tree_attn_few_ok and its scratch be that of `sms` SMs.
cudaError_t launch_tree_attn_stall_selftest(const TreeAttn &a, bool last, void *scratch,
                                            uint32_t *status, int sms, cudaStream_t stream) {
  CUtensorMap tk{}, tv{};
  if (a.dim != 64 || row_tiles(a) != 1 || page_rows(a) != BK || !status ||
      !cache_map(&tk, a, a.k, a.k_s, false, BK) || !cache_map(&tv, a, a.v, a.v_s, false, BK))
    return cudaErrorInvalidValue;
  LaunchInfo info;
  return run<64, 1, false, true, true>(a, tk, tv, scratch, status, sms, stream, &info, last ? 1 : 0);
}

}  // namespace mcb
