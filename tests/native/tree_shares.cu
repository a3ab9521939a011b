// Runs on the host: how the attention over a paged cache shares out its units, with the lengths at
// the end of a page that no access may pass. Reads from the input
//   rows threads grid tokens heads_per_kv kv_heads block columns masked requests
//   cu_new[requests + 1]  kv_lens[requests]
// and prints a line for each segment: cta kind b head row0 nrows tok0 prefix keys tile0 ntiles,
// then for each CTA: part cta parts tok0 head row0 nrows.
#include <cstdio>

#include "fence.h"
#include "tree_attn.cuh"

using namespace mcb;
using namespace mcb::tree;

template <int ROWS>
static void run(const TreeParams &p, int threads, int grid) {
  const int64_t per = (p.a.requests + threads - 1) / threads;
  bool descends = false;
  std::vector<uint32_t> sums(threads);
  uint32_t total = 0;
  for (int t = 0; t < threads; ++t) {
    bool here = false;
    const int64_t last = min(p.a.requests, (t + 1) * per);
    sums[t] = requests_cost<ROWS>(p, t * per, last, here);
    descends |= here;
    total += sums[t];
  }
  for (int cta = 0; cta < grid; ++cta) {
    const Share s = share_of(cta, grid, static_cast<int32_t>(total), true, descends);
    int64_t start_b = 0;
    uint32_t before = 0;
    int32_t start_w = 0;
    for (int t = 0; t < threads; before += sums[t++])
      if (s.w0 < s.w1 && before <= static_cast<uint32_t>(s.w0) &&
          static_cast<uint32_t>(s.w0) < before + sums[t]) {
        start_b = t * per;
        start_w = static_cast<int32_t>(before);
      }
    TreeAttnPart part{};
    Walk<ROWS> walk(p, s, part, start_b, start_w);
    Segment g;
    while (walk.next(g))
      std::printf("%d %d %d %d %d %d %d %d %d %d %d\n", cta, g.kind, g.b, g.head, g.row0, g.nrows,
                  g.tok0, g.prefix, g.keys, g.tile0, g.ntiles);
    std::printf("part %d %d %d %d %d %d\n", cta, part.parts, part.tok0, part.head, part.row0,
                part.nrows);
  }
}

int main() {
  int rows, threads, grid, masked;
  long long tokens, columns, requests;
  TreeParams p{};
  if (std::scanf("%d %d %d %lld %d %d %d %lld %d %lld", &rows, &threads, &grid, &tokens,
                 &p.heads_per_kv, &p.a.kv_heads, &p.a.block, &columns, &masked, &requests) != 10)
    return 2;
  std::vector<int32_t> cu(requests + 1), kv(requests);
  for (auto &x : cu)
    if (std::scanf("%d", &x) != 1) return 2;
  for (auto &x : kv)
    if (std::scanf("%d", &x) != 1) return 2;
  const uint32_t word = 0;
  p.a.tokens = tokens;
  p.a.requests = requests;
  p.a.columns = columns;
  p.a.cu = fenced(cu);
  p.a.kv_lens = fenced(kv);
  p.a.mask = masked ? &word : nullptr;
  if (!p.a.cu || !p.a.kv_lens) return 2;
  p.group = make_div(p.heads_per_kv);
  p.most_keys = static_cast<int32_t>(columns * p.a.block);
  if (rows == 16)
    run<16>(p, threads, grid);
  else if (rows == 32)
    run<32>(p, threads, grid);
  else if (rows == 128)
    run<128>(p, threads, grid);
  else
    run<256>(p, threads, grid);
  return 0;
}
