// Attention of a tree of drafted tokens over a paged key/value cache, on
// tcgen05 tensor cores: bf16 or f16, head size 64 or 128, 16-byte aligned rows.
// (The mathematics and the masks: tree_attn.cu.)
//
// Bound: HBM up to about 255 rows a key head, the tensor cores above. Two contexts of
// 131072 and 0 keys, 56 rows by 8 key heads, f16: 104 us, 537 MB at 5.2 TB/s. 24 trees of
// 32 to 64 tokens by 8 heads over up to 6000 keys: 109 us, 61 GFLOP at 560 TFLOP/s, the
// softmax (about 1850 cycles per 64 keys) behind it.
//
// A unit is one request, one key head and up to ROWS of the request's rows
// (row = new token x query heads of the group); its keys are cut into tiles of
// 128. Every CTA (one per SM) takes an equal share of all units' tiles, in
// order, so a long context is split over many CTAs and many short ones are
// packed into one. The share is found on the device from the lengths: nothing
// is read by the host. A unit that lies in one CTA is finished there; the parts
// of a unit that spans CTAs go to scratch (at most two per CTA) and a second
// launch joins them in their order.
//
// Two forms of a CTA, both with two softmax warpgroups g = 0, 1 (one thread a
// row), each with its own scores and output O_g in TMEM:
//   kPair = false  128 rows; a round is two key tiles, one for each warpgroup, so
//                  that the softmax of one overlaps the products of the other.
//   kPair = true   256 rows, 128 for each warpgroup; a round is one key tile for
//                  both. For wide trees and long runs of new tokens.
// A warpgroup works on half tiles of 64 keys with two score accumulators: the
// weights take the scores' place and are the first operand of the product with the
// values, and the scores of the half after the next one follow it there. So one
// half's scores are always waiting: with whole tiles the softmax waited for
// product and scores, 5000 cycles for two 128 x 128 tiles of which the tensor core
// worked 2048. Each warpgroup has its own issuer, because one thread takes about 100
// cycles for a product instruction (24 wide trees: 152 us with one issuer for both,
// 118 with two). From shared memory the weights would cost 64 KiB of writes and
// 64 KiB of reads a tile on a port that the other operands already fill. Five stages
// of keys and values, and outputs stored row by row: a fifth stage given up for
// storing them through shared memory made long contexts 7% slower and short ones no
// faster.
// Warps 0-3 load (cp.async: pages may have any size and end inside a tile),
// 4-7 and 8-11 are the warpgroups, warps 12 and 14 issue their products, warp 13 finds
// the segments (a CTA's part of a unit) and hands them over a small ring.
//
// Keys that a row does not see get the score -inf. Their values must not reach
// it either, and 0 x inf would: the loaders replace what is not finite in the
// new tokens' values by 0, and the rows that do see such a value add it at
// the end. Cache rows past the request's length are not read at all.
#include "tree_attn.cuh"

namespace mcb {
namespace {
using namespace tree;

constexpr int THREADS = 512;
constexpr int CHUNK_BYTES = 128 * 128;  // 128 rows x 64 16-bit columns, one swizzle span
constexpr int HALF = BK / 2;  // keys of a score accumulator
constexpr int LOADERS = 128;
constexpr int SEGS = 4;         // ring of segments
constexpr int VALID_RING = 16;  // key tiles whose validity words are kept
constexpr int INFO_RING = 4;    // key tiles whose row numbers are kept
constexpr int TMEM_COLS = 512;
constexpr uint32_t S_COL = 0, O_COL = 256;

template <int HD>
constexpr int tile_bytes() {
  return 128 * HD * 2;
}
template <int HD, bool kPair>
constexpr int stages() {
  return HD == 128 ? 5 : 8;
}

struct Params : TreeParams {
  uint32_t s_neg;  // negate A in the score product when scale < 0
};

template <int HD, bool kPair>
struct Smem {
  static constexpr int ST = stages<HD, kPair>();
  uint8_t q[kPair ? 2 : 1][tile_bytes<HD>()];
  uint8_t kv[ST][tile_bytes<HD>()];
  // Where a tile's keys lie, block << bits | row, kNoRow: nowhere; ordered so that
  // a loader's keys lie together.
  uint32_t info[INFO_RING][BK];
  uint32_t valid[VALID_RING][4];
  Segment seg[SEGS];
  uint64_t seg_full[SEGS], seg_empty[SEGS];
  uint64_t q_full, q_empty;
  uint64_t kv_full[ST], kv_empty[ST];
  uint64_t s_full[2][2], p_full[2][2];  // per warpgroup and half tile
  uint64_t pv_done[2], o_full[2], o_empty[2];
  uint64_t info_ready, join_full, join_read;
  uint64_t drain[2];
  float2 joined[kPair ? 1 : 128];  // warpgroup 1's maxima and sums
  int64_t start_b;
  int32_t start_w;
  uint32_t tmem_slot;
  int abort_flag, dirty;
};
constexpr size_t kMaxSmem = 232448;
static_assert(sizeof(Smem<128, true>) <= kMaxSmem && sizeof(Smem<128, false>) <= kMaxSmem &&
                  sizeof(Smem<64, true>) <= kMaxSmem && sizeof(Smem<64, false>) <= kMaxSmem,
              "tree attention exceeds the shared memory per block");

__device__ __forceinline__ uint64_t kmajor_desc(uint32_t base, int kk) {
  return make_sdesc_sw128(base + (kk >> 2) * CHUNK_BYTES + (kk & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t base, int kk) {
  return make_sdesc_sw128(base + kk * 2048, CHUNK_BYTES, 1024);
}
template <int HD, bool kPair, bool kF16>
__global__ void __launch_bounds__(THREADS, 1) tree_attn_tc_kernel(const Params p) {
  constexpr int ST = stages<HD, kPair>();
  constexpr int ROWS = kPair ? 256 : 128;
  constexpr int TILES = kPair ? 1 : 2;  // key tiles of a round
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<HD, kPair> &sm = *reinterpret_cast<Smem<HD, kPair> *>(smem_raw);
  uint32_t *scan = &sm.info[0][0];  // before the roles start
  const TreeAttn &a = p.a;
  volatile int *abort_flag = &sm.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads_per_kv;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SEGS; ++s) {
      mbar_init(&sm.seg_full[s], 1);
      mbar_init(&sm.seg_empty[s], LOADERS + 2 + 256);
    }
    mbar_init(&sm.q_full, LOADERS);
    mbar_init(&sm.q_empty, 2);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&sm.kv_full[s], LOADERS);
      mbar_init(&sm.kv_empty[s], kPair ? 2 : 1);
    }
    for (int g = 0; g < 2; ++g) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&sm.s_full[g][h], 1);
        mbar_init(&sm.p_full[g][h], 128);
      }
      mbar_init(&sm.pv_done[g], 1);
      mbar_init(&sm.o_full[g], 1);
      mbar_init(&sm.o_empty[g], 128);
    }
    mbar_init(&sm.info_ready, LOADERS);
    mbar_init(&sm.join_full, 128);
    mbar_init(&sm.join_read, 128);
    mbar_init(&sm.drain[0], 1);
    mbar_init(&sm.drain[1], 1);
    // The tiles' swizzle needs a 1024-byte aligned base.
    sm.abort_flag = (smem_u32(smem_raw) & 1023u) != 0;
    if (sm.abort_flag && p.status) atomicOr(p.status, kErrBadLaunch);
    sm.dirty = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sm.tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }

  grid_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_slot;
  const Share share =
      find_share<ROWS, THREADS>(p, scan, !sm.abort_flag, &sm.start_b, &sm.start_w);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---------------- loaders ----------------
    constexpr int PIECES = HD / 8;              // 16-byte pieces of a row
    constexpr int STEP = LOADERS / PIECES;      // rows per pass
    constexpr int PASSES = 128 / STEP;
    const int l = threadIdx.x, piece = l % PIECES, r0 = l / PIECES;
    // Offset of this thread's piece of row r0 in a tile; rows STEP apart have the
    // same swizzle.
    const uint32_t dst0 = (piece >> 3) * CHUNK_BYTES + r0 * 128 +
                          (((piece & 7) ^ (r0 & 7)) << 4);
    uint32_t kvc = 0, tiles = 0, sc = 0, described = 0;
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status,
                                               kErrTimeoutEmpty)) != 0;
    };
    // This thread's pieces of a value tile whose rows from `first` on are new
    // tokens': what is not finite becomes 0.
    auto clean = [&](uint8_t *tile, int first) {
      for (int it = 0; it < PASSES; ++it) {
        if (r0 + it * STEP < first) continue;
        uint4 *at = reinterpret_cast<uint4 *>(tile + dst0 + it * STEP * 128);
        uint4 w = *at;
        uint32_t *x = reinterpret_cast<uint32_t *>(&w);
        bool bad = false;
        constexpr uint32_t E = kF16 ? 0x7c00u : 0x7f80u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((x[i] & E) == E) {
            x[i] &= 0xffff0000u;
            bad = true;
          }
          if ((x[i] & (E << 16)) == (E << 16)) {
            x[i] &= 0xffffu;
            bad = true;
          }
        }
        if (bad) {
          *at = w;
          *static_cast<volatile int *>(&sm.dirty) = 1;
        }
      }
    };
    for (; ok; ++sc) {
      const int ss = sc % SEGS;
      if (!(ok = wait(&sm.seg_full[ss], (sc / SEGS) & 1))) break;
      const Segment sg = sm.seg[ss];
      mbar_arrive(&sm.seg_empty[ss]);
      if (sg.kind == kEnd) break;
      // ---- queries ----
      if (!(ok = wait(&sm.q_empty, (sc & 1) ^ 1))) break;
      {
        // Rows past the last one keep what they held: a row of a product depends
        // on no other row.
        const char *q = static_cast<const char *>(a.q) +
                        (sg.tok0 * a.q_s[0] + sg.head * group * a.q_s[1] + piece * 8) * 2;
#pragma unroll 4
        for (int r = r0; r < sg.nrows; r += STEP) {
          const int row = sg.row0 + r, tok = fast_div(row, p.group);
          cp_async16(smem_u32(sm.q[0]) + (r >> 7) * tile_bytes<HD>() + dst0 +
                         ((r & 127) - r0) * 128,
                     q + (tok * a.q_s[0] + (row - tok * group) * a.q_s[1]) * 2, 16);
        }
        cp_async_arrive(&sm.q_full);
      }
      // ---- keys and values ----
      const int32_t *table = a.table + sg.b * a.table_stride;
      const int key0 = sg.tile0 * BK;
      auto entry = [&](int j) -> int32_t {  // block of this thread's key of tile j
        const int key = key0 + j * BK + l;
        if (j >= sg.ntiles || key >= sg.keys) return -1;
        return table[fast_div(key, p.block)];
      };
      int32_t next = entry(0);
      // Places count over the segments (`tiles` before this one): a loader reads tile x's
      // numbers for the last time, for its values, before it arrives for the description of
      // tile x + 2, and the place is written again for tile x + 4, which the
      // barrier of x + 3 precedes. Counted from 0 in each segment, a loader that ran ahead
      // would write the next segment's first tile over numbers that another still reads.
      auto describe = [&](int j) -> bool {
        const int key = key0 + j * BK + l;
        const int32_t blk = next;
        next = entry(j + 1);
        const bool good = key < sg.keys && blk >= 0 && blk < a.blocks;
        const uint32_t col = fast_div(key, p.block);
        const uint32_t off = key - col * a.block;
        sm.info[(tiles + j) % INFO_RING][(l % STEP) * PASSES + l / STEP] =
            good ? (static_cast<uint32_t>(blk) << p.row_bits) | off : kNoRow;
        const uint32_t bits = __ballot_sync(0xffffffffu, good);
        if (lane == 0) sm.valid[(tiles + j) % VALID_RING][warp] = bits;
        mbar_arrive(&sm.info_ready);
        return wait(&sm.info_ready, described++ & 1);
      };
      auto load = [&](int j, bool value) -> bool {
        const int s = kvc % ST;
        if (!wait(&sm.kv_empty[s], ((kvc / ST) & 1) ^ 1)) return false;
        ++kvc;
        const char *base = static_cast<const char *>(value ? a.v : a.k) +
                           (sg.head * (value ? a.v_s[2] : a.k_s[2]) + piece * 8) * 2;
        const uint32_t dst = smem_u32(sm.kv[s]) + dst0;
        const uint32_t blk_step = p.step[value][0], row_step = p.step[value][1];
        const uint4 *info =
            reinterpret_cast<const uint4 *>(sm.info[(tiles + j) % INFO_RING]) + r0 * (PASSES / 4);
#pragma unroll
        for (int it = 0; it < PASSES; it += 4) {
          const uint4 w = info[it / 4];
          const uint32_t row[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const bool none = row[u] == kNoRow;
            const uint32_t at = (row[u] >> p.row_bits) * blk_step +
                                (row[u] & ((1u << p.row_bits) - 1)) * row_step;
            cp_async16(dst + (it + u) * STEP * 128,
                       base + static_cast<uint64_t>(none ? 0u : at) * 16, none ? 0 : 16);
          }
        }
        const int first = min(max(sg.prefix - (key0 + j * BK), 0), BK);
        if (value && first < BK) {
          cp_async_wait_all();
          clean(sm.kv[s], first);
          mbar_arrive(&sm.kv_full[s]);
        } else {
          cp_async_arrive(&sm.kv_full[s]);
        }
        return true;
      };
      // The order of the products: a round's values, then the next round's keys.
      for (int j = 0; j < TILES && j < sg.ntiles && ok; ++j) ok = describe(j) && load(j, false);
      for (int j0 = 0; j0 < sg.ntiles && ok; j0 += TILES) {
        for (int j = j0; j < j0 + TILES && j < sg.ntiles && ok; ++j) ok = load(j, true);
        for (int j = j0 + TILES; j < j0 + 2 * TILES && j < sg.ntiles && ok; ++j)
          ok = describe(j) && load(j, false);
      }
      tiles += sg.ntiles;
      if (!ok) break;
    }
    cp_async_wait_all();
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if ((warp & 1) == 0 && lane == 0) {
      // ---------------- MMA issuers: warp 12 for warpgroup 0, warp 14 for 1 ----------------
      const int g = (warp - 12) >> 1;
      constexpr uint32_t F = kF16 ? 0 : 1;
      const uint32_t idesc_s = make_idesc(F, F, 0, 0, 128, HALF) | p.s_neg;
      const uint32_t idesc_o = make_idesc(F, F, 0, 1, 128, HD);
      const uint32_t s_tmem = tmem + S_COL + g * BK, o_tmem = tmem + O_COL + g * HD;
      const uint32_t q_addr = smem_u32(sm.q[kPair ? g : 0]);
      uint32_t kvc = 0, sc = 0, tiles = 0, outs = 0;  // tiles, outs: of this warpgroup
      bool ok = true;
      // The next key or value tile (kvc counts all tiles, used here or not).
      auto stage = [&](uint32_t &addr) -> int {
        const int s = kvc % ST;
        ok = mbar_wait(&sm.kv_full[s], (kvc / ST) & 1, abort_flag, p.status, kErrTimeoutFull);
        fence_async_smem();
        tc_fence_after();
        ++kvc;
        addr = smem_u32(sm.kv[s]);
        return s;
      };
      auto scores = [&](int h, uint32_t k_addr) {  // of half a key tile
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_f16_ss(s_tmem + h * HALF, kmajor_desc(q_addr, kk),
                     kmajor_desc(k_addr + h * (HALF * 128), kk), idesc_s, kk ? 1u : 0u);
        mma_commit(&sm.s_full[g][h]);
      };
      for (; ok; ++sc) {
        const int ss = sc % SEGS;
        if (!mbar_wait(&sm.seg_full[ss], (sc / SEGS) & 1, abort_flag, p.status, kErrTimeoutFull))
          break;
        const Segment sg = sm.seg[ss];
        mbar_arrive(&sm.seg_empty[ss]);
        if (sg.kind == kEnd) break;
        const int n = sg.ntiles;
        if (!mbar_wait(&sm.q_full, sc & 1, abort_flag, p.status, kErrTimeoutFull)) break;
        if (kPair ? g * 128 >= sg.nrows : g >= n) {
          // Nothing to do for this warpgroup: hand everything on.
          mbar_arrive(&sm.q_empty);
          if (kPair) {
            for (int k = 0; k < 2 * n && ok; ++k) {
              uint32_t addr;
              const int s = stage(addr);
              if (ok) mbar_arrive(&sm.kv_empty[s]);
            }
          } else {
            kvc += 2 * n;
          }
          continue;
        }
        // The first scores. From then on a half's next scores follow the product of
        // its weights, which lie in their place, with the values: one half's scores
        // are always ahead. kPair = false: of a round's two tiles the other
        // warpgroup's is skipped.
        const int j0 = kPair ? 0 : g;
        const uint32_t kvc0 = kvc;
        {
          uint32_t k_addr = 0;
          kvc += j0;
          const int s = stage(k_addr);
          if (!ok) break;
          kvc += min(TILES, n) - 1 - j0;
          scores(0, k_addr);
          scores(1, k_addr);
          mma_commit(&sm.kv_empty[s]);
        }
        if (j0 + TILES >= n) mma_commit(&sm.q_empty);
        for (int j = j0; j < n; j += TILES) {
          const int next = j + TILES, round = j - j0;
          uint32_t v_addr = 0, k_addr = 0;
          int ks = 0;
          kvc += j0;
          const int vs = stage(v_addr);
          if (!ok) break;
          kvc += min(TILES, n - round) - 1 - j0;
          if (j == j0) {
            if (!(ok = mbar_wait(&sm.o_empty[g], (outs & 1) ^ 1, abort_flag, p.status,
                                 kErrTimeoutAccum)))
              break;
            ++outs;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (ok)
              ok = mbar_wait(&sm.p_full[g][h], tiles & 1, abort_flag, p.status, kErrTimeoutAccum);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < HALF / 16; ++kk)
              mma_f16_ts(o_tmem, s_tmem + h * HALF + kk * 8,
                         mnmajor_desc(v_addr, h * (HALF / 16) + kk), idesc_o,
                         (round || h || kk) ? 1u : 0u);
            mma_commit(&sm.pv_done[g]);
            if (h == 1) {
              if (next >= n) mma_commit(&sm.o_full[g]);
              mma_commit(&sm.kv_empty[vs]);
            }
            if (next < n) {
              if (h == 0) {
                kvc += j0;
                ks = stage(k_addr);
                if (!ok) break;
                kvc += min(TILES, n - round - TILES) - 1 - j0;
              }
              scores(h, k_addr);
              if (h == 1) {
                mma_commit(&sm.kv_empty[ks]);
                if (next + TILES >= n) mma_commit(&sm.q_empty);
              }
            }
          }
          ++tiles;
        }
        kvc = kvc0 + 2 * n;
      }
      mma_commit(&sm.drain[g]);
      if (!mbar_wait(&sm.drain[g], 0, nullptr, p.status, kErrTimeoutDrain)) *abort_flag = 1;
    } else if (warp == 13 && lane == 0) {
      // ---------------- scheduler ----------------
      uint32_t sc = 0;
      bool ok = true;
      TreeAttnPart part{};
      auto put = [&](const Segment &sg) -> bool {
        const int ss = sc % SEGS;
        if (!mbar_wait(&sm.seg_empty[ss], ((sc / SEGS) & 1) ^ 1, abort_flag, p.status,
                       kErrTimeoutEmpty))
          return false;
        sm.seg[ss] = sg;
        mbar_arrive(&sm.seg_full[ss]);
        ++sc;
        return true;
      };
      Walk<ROWS> walk(p, share, part, sm.start_b, sm.start_w);
      Segment sg;
      while (ok && walk.next(sg)) ok = put(sg);
      p.part[blockIdx.x] = part;
      Segment end{};
      end.kind = kEnd;
      if (ok) put(end);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ---------------- softmax and output ----------------
    const int g = (warp - 4) >> 2, sub = warp & 3;
    const int row = sub * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(sub * 32) << 16);
    const uint32_t s_col = S_COL + g * BK, o_col = O_COL + g * HD;
    uint32_t sc = 0, steps = 0, o_cnt = 0, tiles = 0, joins = 0;
    bool ok = true;
    for (; ok; ++sc) {
      const int ss = sc % SEGS;
      if (!(ok = mbar_wait_warp(&sm.seg_full[ss], (sc / SEGS) & 1, abort_flag, p.status,
                                kErrTimeoutAccum)))
        break;
      const Segment sg = sm.seg[ss];
      mbar_arrive(&sm.seg_empty[ss]);
      if (sg.kind == kEnd) break;
      const int n = sg.ntiles;
      const int base = kPair ? g * 128 : 0;       // first unit row of this warpgroup
      const int step = kPair ? 1 : 2, j0 = kPair ? 0 : g;
      const bool joined = !kPair && n > 1;        // both warpgroups hold a part of each row
      const bool busy = kPair ? base < sg.nrows : g < n;
      const bool live = base + sub * 32 < sg.nrows;  // this warp has rows
      const int urow = min(sg.row0 + base + row, sg.row0 + sg.nrows - 1);
      const int i = fast_div(urow, p.group);         // new token of this row
      const uint32_t *mask_row =
          a.mask ? a.mask + (static_cast<int64_t>(sg.tok0) + i) * a.mask_stride : nullptr;
      float m_ref = -INFINITY, l = 0.0f;
      for (int j2 = 2 * j0; j2 < 2 * n && busy; j2 += (j2 & 1) ? 2 * step - 1 : 1) {
        const int j = j2 >> 1, h = j2 & 1;  // tile, half
        if (!(ok = mbar_wait_warp(&sm.s_full[g][h], (steps >> 1) & 1, abort_flag, p.status,
                                  kErrTimeoutAccum)))
          break;
        ++steps;
        tc_fence_after();
        if (!live) {  // no rows: hand the half on
          mbar_arrive(&sm.p_full[g][h]);
          continue;
        }
        const uint32_t at = lane_base + s_col + h * HALF;
        uint32_t s[HALF];
        {
          uint32_t (&s0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[0]);
          uint32_t (&s1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[32]);
          tmem_ld_32x32b_x32(at, s0);
          tmem_ld_32x32b_x32(at + 32, s1);
          tmem_ld_wait();
          reg_fence(s0);
          reg_fence(s1);
        }
        const int pos0 = (sg.tile0 + j) * BK + h * HALF;
        const uint2 good =
            *reinterpret_cast<const uint2 *>(sm.valid[(tiles + j) % VALID_RING] + 2 * h);
        if (pos0 + HALF > sg.prefix || (good.x & good.y) != 0xffffffffu) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t see = (w ? good.y : good.x) &
                                 visible_word(a, mask_row, pos0 + 32 * w, sg.prefix, i);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[32 * w + k] = 0xff800000u;
          }
        }
        float m4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          m4[q] = fmaxf(__uint_as_float(s[q]), __uint_as_float(s[q + 4]));
#pragma unroll
          for (int k = 8; k < HALF; k += 8)
            m4[q] = fmax3(m4[q], __uint_as_float(s[k + q]), __uint_as_float(s[k + q + 4]));
        }
        const float mx = fmax3(m4[0], m4[1], fmaxf(m4[2], m4[3]));
        // The reference maximum moves only when a weight would pass 2^8. While
        // it is -inf, O and l are zero.
        bool need = false;
        if (m_ref == -INFINITY)
          m_ref = mx > -INFINITY ? mx : -INFINITY;
        else
          need = (mx - m_ref) * p.c > 8.0f;
        if (__any_sync(0xffffffffu, need)) {
          // O is at rest once the previous half's product is done: this half's
          // waits for these weights.
          if (!(ok = mbar_wait_warp(&sm.pv_done[g], (steps - 2) & 1, abort_flag, p.status,
                                    kErrTimeoutAccum)))
            break;
          tc_fence_after();
          const float f = need ? ex2((m_ref - mx) * p.c) : 1.0f;
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 16) {
            uint32_t o[16];
            tmem_ld16_sync(lane_base + o_col + c0, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st_32x32b_x16(lane_base + o_col + c0, o);
          }
          if (need) {
            l *= f;
            m_ref = mx;
          }
        }
        const float mc = m_ref == -INFINITY ? 0.0f : m_ref * p.c;
        const uint64_t c2 = f2_pack(p.c, p.c), nmc2 = f2_pack(-mc, -mc);
        // The weights take the place of the row's scores in TMEM, two a column.
        uint64_t ps[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int e = 32 * c + 2 * k;
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, nmc2),
                      x0, x1);
            const float e0 = ex2(x0), e1 = ex2(x1);
            ps[k & 3] = f2_add(ps[k & 3], f2_pack(e0, e1));
            pk[k] = pack2<kF16>(e0, e1);
          }
          tmem_st_32x32b_x16(at + 16 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_full[g][h]);
        {
          float a0, a1;
          f2_unpack(f2_add(f2_add(ps[0], ps[1]), f2_add(ps[2], ps[3])), a0, a1);
          l += a0 + a1;
        }
      }
      if (!ok) break;
      tiles += n;
      // ---- output ----
      if (!busy) continue;
      float mc = m_ref == -INFINITY ? -INFINITY : m_ref * p.c;
      float w_own = 1.0f, w_other = 0.0f;
      if (!(ok = mbar_wait_warp(&sm.o_full[g], o_cnt++ & 1, abort_flag, p.status,
                                kErrTimeoutAccum)))
        break;
      if (joined && g == 0 &&
          !(ok = mbar_wait_warp(&sm.o_full[1], joins & 1, abort_flag, p.status, kErrTimeoutAccum)))
        break;
      tc_fence_after();
      if (joined) {
        // Warpgroup 1 leaves its maxima and sums and is done; warpgroup 0 reads
        // both outputs, whose rows lie in the same TMEM lanes.
        float2 *shared = sm.joined;
        if (g == 1) {
          shared[row] = make_float2(mc, l);
          mbar_arrive(&sm.join_full);
          // The buffer may be written again once it has been read.
          if (!(ok = mbar_wait_warp(&sm.join_read, joins++ & 1, abort_flag, p.status,
                                    kErrTimeoutAccum)))
            break;
          continue;
        }
        if (!(ok = mbar_wait_warp(&sm.join_full, joins++ & 1, abort_flag, p.status,
                                  kErrTimeoutAccum)))
          break;
        const float2 other = shared[row];
        mbar_arrive(&sm.join_read);
        const float top = fmaxf(mc, other.x), ref = top == -INFINITY ? 0.0f : top;
        w_own = ex2(mc - ref);
        w_other = ex2(other.x - ref);
        l = l * w_own + other.y * w_other;
        mc = top;
      }
      if (live) {
        const bool mine_live = base + row < sg.nrows;
        const bool dirty = *static_cast<volatile int *>(&sm.dirty) != 0;
        const int64_t tok = static_cast<int64_t>(sg.tok0) + i;
        const int head = sg.head * group + urow - i * group;
        const bool whole = sg.kind == kWhole;
        const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (sg.kind == kTail);
        char *orow = static_cast<char *>(a.o) + (tok * a.o_s[0] + head * a.o_s[1]) * 2;
        // Parts lie by columns of four, so that a warp's rows are stored together.
        float4 *pcol = reinterpret_cast<float4 *>(p.partial + slot * ROWS * HD) + base + row;
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 32) {
          uint32_t o[32];
          tmem_ld32_sync(lane_base + o_col + c0, o);
          float x[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = __uint_as_float(o[k]);
          if (joined) {
            tmem_ld32_sync(lane_base + O_COL + HD + c0, o);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              x[k] = x[k] * w_own + __uint_as_float(o[k]) * w_other;
          }
          if (dirty) {
            // Values of new tokens that are not finite, where the row sees them.
            const int k0 = max(sg.tile0 * BK, sg.prefix);
            const int k1 = min((sg.tile0 + n) * BK, sg.keys);
            for (int pos = max(k0, 0); pos < k1; ++pos) {
              if (!(visible_word(a, mask_row, pos, sg.prefix, i) & 1u)) continue;
              const int col = pos / a.block;
              const int32_t blk = a.table[sg.b * a.table_stride + col];
              if (blk < 0 || blk >= a.blocks) continue;
              const int64_t at = blk * a.v_s[0] +
                                 static_cast<int64_t>(pos - col * a.block) * a.v_s[1] +
                                 sg.head * a.v_s[2] + c0;
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const float v =
                    kF16 ? __half2float(static_cast<const __half *>(a.v)[at + k])
                         : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.v)[at + k]);
                if (!(fabsf(v) < INFINITY)) x[k] += v;
              }
            }
          }
          if (mine_live) {
            if (whole) {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4 *>(orow + (c0 + 8 * q) * 2) = make_uint4(
                    pack2<kF16>(x[8 * q] * inv, x[8 * q + 1] * inv),
                    pack2<kF16>(x[8 * q + 2] * inv, x[8 * q + 3] * inv),
                    pack2<kF16>(x[8 * q + 4] * inv, x[8 * q + 5] * inv),
                    pack2<kF16>(x[8 * q + 6] * inv, x[8 * q + 7] * inv));
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                pcol[(c0 / 4 + q) * ROWS] =
                    make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
            }
          }
        }
        if (mine_live) {
          if (whole) {
            if (a.lse)
              a.lse[tok * a.lse_s + head] =
                  l == 0.0f ? -INFINITY
                            : ((mc == -INFINITY ? 0.0f : mc) + log2f(l)) * 0.69314718055994531f;
          } else {
            float2 *ml = reinterpret_cast<float2 *>(
                p.partial + static_cast<int64_t>(gridDim.x) * 2 * ROWS * HD);
            ml[slot * ROWS + base + row] = make_float2(mc, l);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&sm.o_empty[g]);
      if (joined) mbar_arrive(&sm.o_empty[1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

bool pair_of(const TreeAttn &a) {
  // Two row halves per CTA when a request has more than 128 rows on average: 24 trees of
  // 32 to 64 tokens by 8 heads 109 us, 147 us with 128 rows a CTA, which read each
  // context twice; below that the second half would be empty.
  return a.tokens * (a.heads / a.kv_heads) > 128 * a.requests;
}

template <int HD, bool kPair, bool kF16>
cudaError_t run(const Params &p, int ctas, cudaStream_t stream) {
  constexpr int ROWS = kPair ? 256 : 128;
  auto kernel = tree_attn_tc_kernel<HD, kPair, kF16>;
  constexpr int smem = static_cast<int>(sizeof(Smem<HD, kPair>));
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<ctas, THREADS, smem, stream>>>(p);
  return launch_join<HD, ROWS, kF16>(p, ctas, stream);
}

}  // namespace

bool tree_attn_tc_ok(const TreeAttn &a, int dtype) {
  if (dtype != MCB_DTYPE_BF16 && dtype != MCB_DTYPE_F16) return false;
  if (a.dim != 64 && a.dim != 128) return false;
  if (a.scale == 0.0f) return false;  // a masked score times 0 would be NaN
  if (a.blocks == 0) return false;    // no cache row to point copies of nothing at
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                          reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.o);
  int64_t steps = a.q_s[0] | a.q_s[1] | a.o_s[0] | a.o_s[1];
  for (int i = 0; i < 3; ++i) steps |= a.k_s[i] | a.v_s[i];
  if (bases % 16 != 0 || steps % 8 != 0) return false;
  // 32-bit numbers: rows, keys of a request, what all units cost (a tile begun and
  // three more beside a unit's keys), and the offsets of cache rows in 16 bytes (a cache of
  // up to 64 GB).
  const int64_t group = a.heads / a.kv_heads, rows = a.tokens * group;
  if (a.tokens * a.heads > 0x7fffffff || a.columns * a.block > 0x7fffff00) return false;
  const double tiles = (static_cast<double>(rows) / 16 + a.requests) * a.kv_heads *
                       (static_cast<double>(a.columns) * a.block / BK + 4);
  if (tiles > 0x7fffffff) return false;
  for (const int64_t *st : {a.k_s, a.v_s})
    if (st[0] / 8 > 0xffffffffLL || st[1] / 8 > 0xffffffffLL ||
        static_cast<double>(a.blocks) * (st[0] / 8) + static_cast<double>(a.block) * (st[1] / 8) >=
            4294967295.0)
      return false;
  return true;
}

uint64_t tree_attn_tc_scratch(const TreeAttn &a, int sms) {
  return tree_scratch(a, pair_of(a) ? 256 : 128, sms);
}

cudaError_t launch_tree_attn_tc(const TreeAttn &a, int dtype, void *scratch, uint32_t *status,
                                int sms, cudaStream_t stream, LaunchInfo *info) {
  const bool pair = pair_of(a), f16 = dtype == MCB_DTYPE_F16;
  Params p;
  static_cast<TreeParams &>(p) = tree_params(a, scratch, pair ? 256 : 128, sms, status);
  p.s_neg = a.scale < 0.0f ? kIdescNegateA : 0u;
  cudaError_t e;
  auto pick = [&](auto run_bf16, auto run_f16) {
    return f16 ? run_f16(p, sms, stream) : run_bf16(p, sms, stream);
  };
  if (a.dim == 128)
    e = pair ? pick(run<128, true, false>, run<128, true, true>)
             : pick(run<128, false, false>, run<128, false, true>);
  else
    e = pair ? pick(run<64, true, false>, run<64, true, true>)
             : pick(run<64, false, false>, run<64, false, true>);
  info->launches = 2;
  info->tile_m = pair ? 256 : 128;
  info->tile_n = BK;
  info->tile_k = a.dim;
  info->stages = a.dim == 128 ? (pair ? stages<128, true>() : stages<128, false>())
                              : (pair ? stages<64, true>() : stages<64, false>());
  info->ctas = sms;
  info->set_route("tcgen05_tree_attention");
  return e;
}

}  // namespace mcb
