// Attention of drafted tokens over a paged cache for requests of few rows (a
// row = new token x query heads of the group), up to about 64: bf16 or f16,
// head size 64 or 128, 16-byte aligned rows. (The mathematics and the masks:
// tree_attn.cu; how the work is shared out: tree_attn.cuh.)
//
// Bound: reading the cache. With R rows a key and value row of 4 * HD bytes
// take 4 * HD * R operations, far below what a CTA can do in the time of the
// read, so the kernel is built around the copies: at any time three to four
// half tiles (128 keys or values, 32 KiB at HD = 128) are on their way to
// shared memory. The products use warp-level matrix instructions on 16-row tiles:
// the 128-row tile of a tcgen05 instruction would be empty but for a few rows,
// and its softmax would run on one warp.
//
// 8 warps share a tile of 128 keys. Warp w takes keys 16w .. 16w + 15 for the
// scores S = Q K^T (Q from shared memory), makes the weights of those
// keys and leaves them in shared memory as 16-bit numbers; then it takes the
// HD / 8 columns w of O = P V for all 128 keys. So K and V are read from shared memory
// once, O needs no joining across warps, and the only things that the warps
// share are the weights and a reference maximum per row. The maximum moves when a
// score passes it by 8 (in powers of two): whether any does is one barrier with
// an OR, and the exchange of the maxima happens only then.
//
// A ninth warp walks over the segments (a CTA's part of a unit) and prepares, one
// tile ahead of the copies, where each key of a tile lies in the cache.
#include "tree_attn.cuh"

namespace mcb {
namespace {
using namespace tree;

constexpr int WARPS = 8;
constexpr int COMPUTE = WARPS * 32;
constexpr int THREADS = COMPUTE + 32;
constexpr int HALVES = 5;  // half tiles (keys or values) in shared memory
constexpr int TILES = 4;   // ring of prepared tiles
constexpr int QBUFS = 3;   // query tiles: of the tiles at work, copied and prepared

struct Tile {
  uint32_t where[BK];  // block << bits | row of each key, kNoRow: nowhere
  uint32_t valid[4];   // bit per key
  Segment seg;
  int32_t tile;        // of the segment
};

template <int HD, int MT>
struct Smem {
  uint8_t kv[HALVES][BK * HD * 2];
  uint8_t q[QBUFS][16 * MT * HD * 2];
  uint8_t p[16 * MT * BK * 2];  // weights; maxima and sums of the warps in between
  Tile tile[TILES];
  uint64_t full[TILES], empty[TILES];
  int64_t start_b;
  int32_t start_w;
  int abort_flag, dirty;
};
static_assert(sizeof(Smem<128, 4>) <= 232448, "exceeds the shared memory per block");

struct Params : TreeParams {
  float sign;  // of the scale
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
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// Byte offset of 16-byte piece c of a row of BYTES bytes: pieces are permuted
// within groups of eight by the row, so that eight rows of one piece, or one row
// of eight, touch all banks.
template <int BYTES>
__device__ __forceinline__ uint32_t piece_at(int row, int c) {
  return row * BYTES + ((c ^ (row & 7)) << 4);
}

template <int HD, int MT, bool kF16>
__global__ void __launch_bounds__(THREADS) tree_attn_few_kernel(const Params p) {
  constexpr int ROWS = 16 * MT;
  constexpr int ROW = HD * 2;          // bytes of a key, value or query row
  constexpr int PIECES = HD / 8;       // 16-byte pieces of a row
  constexpr int STEP = COMPUTE / PIECES;
  constexpr int NT = HD / 64;          // 8-column tiles of O per warp
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<HD, MT> &sm = *reinterpret_cast<Smem<HD, MT> *>(smem_raw);
  const TreeAttn &a = p.a;
  volatile int *abort_flag = &sm.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.kv_heads;

  if (threadIdx.x == 0) {
    for (int s = 0; s < TILES; ++s) {
      mbar_init(&sm.full[s], 32);
      mbar_init(&sm.empty[s], COMPUTE);
    }
    sm.abort_flag = sm.dirty = 0;
    fence_mbar_init();
  }
  const Share share = find_share<ROWS, THREADS>(a, reinterpret_cast<int32_t *>(sm.p), true,
                                                &sm.start_b, &sm.start_w);

  if (warp == WARPS) {
    // ---------------- tiles, one ahead of the copies ----------------
    TreeAttnPart part{};
    Walk<ROWS> walk(a, share, part, sm.start_b, sm.start_w);
    Segment sg;
    uint32_t count = 0;
    bool ok = true;
    auto slot = [&]() -> Tile * {
      const int s = count % TILES;
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[s], ((count / TILES) & 1) ^ 1, abort_flag,
                                             p.status, kErrTimeoutEmpty)) != 0;
      return ok ? &sm.tile[s] : nullptr;
    };
    while (ok && walk.next(sg)) {
      const int32_t *table = a.table + sg.b * a.table_stride;
      for (int j = 0; j < sg.ntiles; ++j) {
        const int key0 = (sg.tile0 + j) * BK;
        int32_t blk[4];
        uint32_t col[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = key0 + 32 * u + lane;
          col[u] = fast_div(key, p.block);
          blk[u] = key < sg.keys ? table[col[u]] : -1;
        }
        Tile *t = slot();
        if (!t) break;
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
        ++count;
      }
    }
    // Three ends: the copies look two tiles ahead.
    for (int k = 0; k < 3 && ok; ++k) {
      Tile *t = slot();
      if (!t) break;
      if (lane == 0) t->seg.kind = kEnd;
      mbar_arrive(&sm.full[count % TILES]);
      ++count;
    }
    if (lane == 0) p.part[blockIdx.x] = part;
    return;
  }

  // ---------------- copies and products ----------------
  const int tid = threadIdx.x;
  const int piece = tid % PIECES, r0 = tid / PIECES;
  const int quad = lane >> 2, ql = lane & 3;
  auto wait_tile = [&](uint32_t t) -> bool {
    return mbar_wait(&sm.full[t % TILES], (t / TILES) & 1, abort_flag, p.status, kErrTimeoutFull);
  };
  uint32_t qseg = 0;  // segments whose queries were copied
  // Copies of tile t's keys (value = 0) or values into half 2t + value.
  auto copy = [&](uint32_t t, int value) {
    const Tile &d = sm.tile[t % TILES];
    if (d.seg.kind != kEnd) {
      const char *base = static_cast<const char *>(value ? a.v : a.k) +
                         (d.seg.head * (value ? a.v_s[2] : a.k_s[2]) + piece * 8) * 2;
      const uint32_t blk_step = p.step[value][0], row_step = p.step[value][1];
      const uint32_t dst = smem_u32(sm.kv[(2 * t + value) % HALVES]);
#pragma unroll
      for (int it = 0; it < BK / STEP; ++it) {
        const int r = r0 + it * STEP;
        const uint32_t w = d.where[r];
        const bool none = w == kNoRow;
        const uint32_t at = (w >> p.row_bits) * blk_step + (w & ((1u << p.row_bits) - 1)) * row_step;
        cp_async16(dst + piece_at<ROW>(r, piece), base + static_cast<uint64_t>(none ? 0u : at) * 16,
                   none ? 0 : 16);
      }
      if (!value && d.tile == 0) {
        // The segment's queries; rows past the last one are zero.
        const Segment &sg = d.seg;
        const char *q = static_cast<const char *>(a.q) +
                        (sg.tok0 * a.q_s[0] + sg.head * group * a.q_s[1] + piece * 8) * 2;
        const uint32_t to = smem_u32(sm.q[qseg % QBUFS]);
        for (int r = r0; r < ROWS; r += STEP) {
          const bool live = r < sg.nrows;
          const int row = sg.row0 + (live ? r : 0), tok = fast_div(row, p.group);
          cp_async16(to + piece_at<ROW>(r, piece),
                     q + (tok * a.q_s[0] + (row - tok * group) * a.q_s[1]) * 2, live ? 16 : 0);
        }
        ++qseg;
      }
    }
    cp_async_commit();
  };
  bool ok = true;
  for (uint32_t t = 0; t < 2; ++t) {
    ok = ok && wait_tile(t);
    if (named_bar_or(1, COMPUTE, !ok)) return;
    copy(t, 0);
    copy(t, 1);
  }

  float o[MT][NT][4], ref[MT][2], l[MT][2];
  uint32_t seg_no = 0;
  for (uint32_t t = 0;; ++t) {
    // The keys of tile t have landed everywhere, and everyone is done with tile t - 1.
    cp_async_wait<3>();
    ok = wait_tile(t + 2);
    if (named_bar_or(1, COMPUTE, !ok)) return;
    const Tile &d = sm.tile[t % TILES];
    if (d.seg.kind == kEnd) break;
    copy(t + 2, 0);
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
      const uint32_t kb = smem_u32(sm.kv[(2 * t) % HALVES]);
      const uint32_t qb = smem_u32(sm.q[seg_no % QBUFS]);
      // K: matrices (keys 0-7, piece 2k), (0-7, 2k + 1), (8-15, 2k), (8-15, 2k + 1);
      // Q: (rows 0-7, 2k), (8-15, 2k), (0-7, 2k + 1), (8-15, 2k + 1).
      const int krow = 16 * warp + (lane & 7) + ((lane >> 4) << 3), kpc = (lane >> 3) & 1;
      const int qrow = lane & 15, qpc = lane >> 4;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t kf[4];
        ldmatrix4(kf, kb + piece_at<ROW>(krow, 2 * k + kpc));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t qf[4];
          ldmatrix4(qf, qb + piece_at<ROW>(16 * m + qrow, 2 * k + qpc));
          mma<kF16>(s[m][0], qf, kf[0], kf[1]);
          mma<kF16>(s[m][1], qf, kf[2], kf[3]);
        }
      }
    }
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
          const uint32_t at =
              pb + piece_at<BK * 2>(16 * m + quad + 8 * h, 2 * warp + n) + 4 * ql;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(pack2<kF16>(e0, e1)) : "memory");
        }
      }
    // The weights are there and the values have landed; everyone is done with the keys.
    cp_async_wait<3>();
    named_bar_sync(3, COMPUTE);
    copy(t + 2, 1);
    uint8_t *values = sm.kv[(2 * t + 1) % HALVES];
    if (drafts) {
      // New tokens' values that are not finite become 0: 0 x inf must not reach
      // the rows that do not see them. The others add them at the end.
      constexpr uint32_t E = kF16 ? 0x7c00u : 0x7f80u;
      for (int it = 0; it < BK / STEP; ++it) {
        const int r = r0 + it * STEP;
        if (pos0 + r < sg.prefix) continue;
        uint4 *at = reinterpret_cast<uint4 *>(values + piece_at<ROW>(r, piece));
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
          ldmatrix4_trans(vf, vb + piece_at<ROW>(16 * k + (lane & 15), 2 * warp + (lane >> 4)));
        else if (k % 2 == 0)  // one piece, two steps
          ldmatrix4_trans(vf, vb + piece_at<ROW>(16 * k + lane, warp));
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
          ldmatrix4(pf, pb + piece_at<BK * 2>(16 * m + prow, 2 * k + ppc));
          mma<kF16>(o[m][0], pf, vf[0], vf[1]);
          if (NT == 2) mma<kF16>(o[m][NT - 1], pf, vf[2], vf[3]);
        }
      }
    }
    if (d.tile + 1 == sg.ntiles) {
      // ---- the segment's output ----
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
            float2 *out =
                reinterpret_cast<float2 *>(p.partial + (part_slot * ROWS + r) * HD + d0);
#pragma unroll
            for (int n = 0; n < NT; ++n) out[4 * n] = make_float2(x[n][0], x[n][1]);
            if (warp == 0 && ql == 0)
              reinterpret_cast<float2 *>(p.partial +
                                         static_cast<int64_t>(gridDim.x) * 2 * ROWS *
                                             HD)[part_slot * ROWS + r] = make_float2(mc, sum);
          }
        }
    }
    mbar_arrive(&sm.empty[t % TILES]);
  }
  cp_async_wait<0>();
}

// Row tiles of 16 that a CTA takes: by the rows that a request has on average.
int row_tiles(const TreeAttn &a) {
  const int64_t rows = a.tokens * (a.heads / a.kv_heads);
  return rows <= 16 * a.requests ? 1 : rows <= 32 * a.requests ? 2 : 4;
}
template <int HD, int MT>
constexpr int per_sm() {  // CTAs that fit into an SM's shared memory (228 KB, 1 KB kept per CTA)
  return 2 * (sizeof(Smem<HD, MT>) + 1024) <= 233472 ? 2 : 1;
}

template <int HD, int MT, bool kF16>
cudaError_t run(const TreeAttn &a, void *scratch, uint32_t *status, int sms, cudaStream_t stream,
                LaunchInfo *info) {
  const int ctas = sms * per_sm<HD, MT>();
  Params p;
  static_cast<TreeParams &>(p) = tree_params(a, scratch, 16 * MT, ctas, status);
  p.sign = a.scale < 0.0f ? -1.0f : 1.0f;
  auto kernel = tree_attn_few_kernel<HD, MT, kF16>;
  constexpr int smem = static_cast<int>(sizeof(Smem<HD, MT>));
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<ctas, THREADS, smem, stream>>>(p);
  tree_attn_join_parts_kernel<HD, 16 * MT, kF16>
      <<<dim3(ctas + 1, 2 * MT), 256, 0, stream>>>(p, ctas);
  info->launches = 2;
  info->tile_m = 16 * MT;
  info->tile_n = BK;
  info->tile_k = HD;
  info->stages = HALVES;
  info->ctas = ctas;
  info->set_route("tree_attention_few_rows");
  return cudaGetLastError();
}

template <int HD, bool kF16>
cudaError_t run_rows(const TreeAttn &a, void *scratch, uint32_t *status, int sms,
                     cudaStream_t stream, LaunchInfo *info) {
  switch (row_tiles(a)) {
    case 1: return run<HD, 1, kF16>(a, scratch, status, sms, stream, info);
    case 2: return run<HD, 2, kF16>(a, scratch, status, sms, stream, info);
    default: return run<HD, 4, kF16>(a, scratch, status, sms, stream, info);
  }
}

}  // namespace

bool tree_attn_few_ok(const TreeAttn &a, int dtype) {
  return tree_attn_tc_ok(a, dtype) &&
         a.tokens * (a.heads / a.kv_heads) <= kTreeFewRows * a.requests;
}

uint64_t tree_attn_few_scratch(const TreeAttn &a, int sms) {
  const int mt = row_tiles(a);
  const int n = a.dim == 128 ? (mt == 1 ? per_sm<128, 1>() : mt == 2 ? per_sm<128, 2>() : per_sm<128, 4>())
                             : (mt == 1 ? per_sm<64, 1>() : mt == 2 ? per_sm<64, 2>() : per_sm<64, 4>());
  return tree_scratch(a, 16 * mt, n * sms);
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

}  // namespace mcb
