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

constexpr int TREE_BK = 64;                    // keys per tile
// what a pair costs beside its tiles, in tiles: the start of its products, the join and the write of its rows
constexpr int TREE_PAIR = 4;

// block c of `blocks` (no more than there are units) takes the units from tree_unit(c) to tree_unit(c + 1) of `total`
AF_DEV long long tree_unit(long long c, long long total, int blocks) { return c * total / blocks; }
// the block that takes unit u
AF_DEV int tree_block_of(long long u, long long total, int blocks) {
  int c = (int)(u * blocks / total);
  while (c + 1 < blocks && tree_unit(c + 1, total, blocks) <= u) ++c;
  while (c > 0 && tree_unit(c, total, blocks) > u) --c;
  return c;
}

// The walk of one block through its units. Every pair of a sequence and a key head (and row group) has
// TREE_PAIR units without work, then one for each tile of 64 keys; the order is sequence 0's key head 0
// (row group 0, 1, ...), key head 1, ..., then sequence 1. A segment is the part of a pair's tiles that
// the block has. A sequence has at least one tile.
struct TreeSched {
  long long u1, pair0;                         // the block's end; the current pair's first tile's unit
  int b, h, rg, nt;                            // the pair; its tiles
  int len, nodes;
  int len1, nodes1;                            // the next sequence's, read ahead
  int t0, t1;                                  // the segment

  AF_DEV static int tiles_of(int len, int nodes) { return max(1, (len + nodes + TREE_BK - 1) / TREE_BK); }
  AF_DEV void ahead(const AttnTreeArgs& a) {
    if (b + 1 < a.B) tree_extent(a, b + 1, len1, nodes1);
  }
  // a whole warp: the first unit of sequence `want` and the total; with want < 0 the sequence that holds the
  // first unit of block c
  AF_DEV void scan(const AttnTreeArgs& a, int want, int c, int blocks, int lane, long long& first, long long& total) {
    const int per = a.KV * a.row_groups;
    auto units = [&](int s) {
      if (s >= a.B) return 0;
      int l, n;
      tree_extent(a, s, l, n);
      return tiles_of(l, n) + TREE_PAIR;
    };
    total = 0;
    int mine = 0;
    for (int s = 0; s < a.B; s += 32) {
      mine = units(s + lane);
      total += __reduce_add_sync(0xffffffffu, mine);
    }
    total *= per;
    const int act = (int)min((long long)blocks, total);
    const long long at = want < 0 ? tree_unit(c < act ? c : 0, total, act) : 0;
    long long before = 0;
    b = 0;
    first = 0;
    for (int s = 0; s < a.B; s += 32) {
      const int v = a.B <= 32 ? mine : units(s + lane);
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
  // the block's first segment; false: it has no tile
  AF_DEV bool init(const AttnTreeArgs& a, int c, int blocks, int lane) {
    long long first, total;
    scan(a, -1, c, blocks, lane, first, total);
    blocks = (int)min((long long)blocks, total);
    if (c >= blocks) return false;
    const long long u = tree_unit(c, total, blocks);
    u1 = tree_unit(c + 1, total, blocks);
    tree_extent(a, b, len, nodes);
    ahead(a);
    nt = tiles_of(len, nodes);
    const int pair = (int)((u - first) / (nt + TREE_PAIR));
    h = pair / a.row_groups;
    rg = pair - h * a.row_groups;
    pair0 = first + (long long)pair * (nt + TREE_PAIR) + TREE_PAIR;
    t0 = (int)max(0ll, u - pair0);
    t1 = (int)min((long long)nt, u1 - pair0);
    return t1 > t0;                            // a block that ends before the pair's tiles has nothing more
  }
  AF_DEV void find(const AttnTreeArgs& a, int want, int lane, long long& first, long long& total) {
    scan(a, want, 0, 1, lane, first, total);
    tree_extent(a, b, len, nodes);
    nt = tiles_of(len, nodes);
  }
  AF_DEV int tiles() const { return t1 - t0; }
  AF_DEV bool ends() const { return t1 == nt; }
  AF_DEV bool whole() const { return t0 == 0 && t1 == nt; }
  AF_DEV int slot() const { return t0 > 0 ? 0 : 1; }
  // the next segment; false: none
  AF_DEV bool next(const AttnTreeArgs& a) {
    if (t1 < nt) return false;
    pair0 += nt + TREE_PAIR;
    if (++rg == a.row_groups) {
      rg = 0;
      if (++h == a.KV) {
        h = 0;
        if (++b >= a.B) return false;
        len = len1;
        nodes = nodes1;
        nt = tiles_of(len, nodes);
        ahead(a);
      }
    }
    t0 = 0;
    t1 = (int)max(0ll, min((long long)nt, u1 - pair0));
    return t1 > 0;
  }
};

}  // namespace af
