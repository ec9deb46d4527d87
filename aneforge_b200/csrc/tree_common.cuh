// Geometry of tree attention shared by its kernels: a sequence's extent, and the cut of all key tiles
// into equal runs for the blocks.
#pragma once
#include "af_common.cuh"
#include "af_kernels.h"

namespace af {

// prefix rows and live nodes of sequence b, cut to what the table can hold
AF_DEV void tree_extent(const AttnTreeArgs& a, int b, int& len, int& nodes) {
  len = min(max(__ldcg(a.lens + b), 0), a.W * a.page);
  nodes = a.nodes ? min(max(__ldcg(a.nodes + b), 0), a.T) : a.T;
  nodes = min(nodes, a.W * a.page - len);
}

// block c of `blocks` (no more than there are units) takes the units from tree_unit(c) to tree_unit(c + 1) of `total`
AF_DEV long long tree_unit(long long c, long long total, int blocks) { return c * total / blocks; }
// the block that takes unit u
AF_DEV int tree_block_of(long long u, long long total, int blocks) {
  int c = (int)(u * blocks / total);
  while (c + 1 < blocks && tree_unit(c + 1, total, blocks) <= u) ++c;
  while (c > 0 && tree_unit(c, total, blocks) > u) --c;
  return c;
}

// The walk of one block through its units. Units are the 128-key tiles of sequence 0's key head 0 (row
// group 0, 1, ...), key head 1, ..., then of sequence 1; a segment is the part of one such pair that the
// block has. A sequence has at least one tile.
struct TreeSched {
  long long u, u1, item0;                      // next unit, end, the current pair's first unit
  int b, h, rg, nt;                            // the pair; its tiles
  int len, nodes;
  int len1, nodes1;                            // the next sequence's, read ahead
  int t0;                                      // the segment's first tile

  AF_DEV void load(const AttnTreeArgs& a) {
    tree_extent(a, b, len, nodes);
    ahead(a);
    nt = max(1, (len + nodes + 127) / 128);
  }
  AF_DEV void ahead(const AttnTreeArgs& a) {
    if (b + 1 < a.B) tree_extent(a, b + 1, len1, nodes1);
  }
  // a whole warp: `first` unit of sequence `want`, `total` units; with want < 0 the sequence that holds
  // unit c * total / blocks
  AF_DEV void scan(const AttnTreeArgs& a, int want, int c, int blocks, int lane, long long& first, long long& total) {
    const int per = a.KV * a.row_groups;
    auto tiles = [&](int s) {
      if (s >= a.B) return 0;
      int l, n;
      tree_extent(a, s, l, n);
      return max(1, (l + n + 127) / 128);
    };
    total = 0;
    int mine = 0;
    for (int s = 0; s < a.B; s += 32) {
      mine = tiles(s + lane);
      total += __reduce_add_sync(0xffffffffu, mine);
    }
    total *= per;
    const int act = (int)min((long long)blocks, total);
    const long long at = want < 0 ? tree_unit(c < act ? c : 0, total, act) : 0;
    long long before = 0;
    b = 0;
    first = 0;
    for (int s = 0; s < a.B; s += 32) {
      const int v = a.B <= 32 ? mine : tiles(s + lane);
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const long long lo = (before + x - v) * per, hi = (before + x) * per;
      const unsigned hit = __ballot_sync(0xffffffffu, want < 0 ? lo <= at && at < hi : s + lane == want);
      if (hit) {
        const int k = __ffs(hit) - 1;
        b = s + k;
        first = __shfl_sync(0xffffffffu, lo, k);
        return;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  // false: nothing for this block
  AF_DEV bool init(const AttnTreeArgs& a, int c, int blocks, int lane) {
    long long first, total;
    scan(a, -1, c, blocks, lane, first, total);
    blocks = (int)min((long long)blocks, total);
    if (c >= blocks) return false;
    u = tree_unit(c, total, blocks);
    u1 = tree_unit(c + 1, total, blocks);
    load(a);
    const int pair = (int)((u - first) / nt);
    h = pair / a.row_groups;
    rg = pair - h * a.row_groups;
    item0 = first + (long long)pair * nt;
    t0 = (int)(u - item0);
    return true;
  }
  AF_DEV void find(const AttnTreeArgs& a, int want, int lane, long long& first, long long& total) {
    scan(a, want, 0, 1, lane, first, total);
    load(a);
  }
  AF_DEV int tiles() const { return (int)min((long long)(nt - t0), u1 - u); }
  AF_DEV bool ends() const { return t0 + tiles() == nt; }
  AF_DEV bool whole() const { return t0 == 0 && ends(); }
  AF_DEV int slot() const { return t0 > 0 ? 0 : 1; }
  AF_DEV void next(const AttnTreeArgs& a) {
    const int k = tiles();
    u += k;
    if (u >= u1) return;
    item0 += nt;                               // u == item0 now
    t0 = 0;
    if (++rg == a.row_groups) {
      rg = 0;
      if (++h == a.KV) {
        h = 0;
        ++b;
        len = len1;
        nodes = nodes1;
        nt = max(1, (len + nodes + 127) / 128);
        ahead(a);
      }
    }
  }
};

}  // namespace af
