// xn_paged_attn.cuh - what the paged attention's kernels share: arguments, the
// work list that the schedule kernel builds on the device, and the walk over it.
//
// Work. A query tile is up to `tile_tokens` consecutive new tokens of one
// request with the group of query heads that share a kv head: rows (token,
// head of the group), token-major. A unit is one key tile against one (query
// tile, kv head). The units of all (tile, head) pairs, in that order, form one
// line, which is cut into parts of equal cost, one per CTA, wherever the cuts
// fall: lengths are known on the device only, and equal parts keep every SM
// busy for ragged batches and for one long request alike. A pair costs its
// units and `pair_cost` more for its query rows and output. A CTA walks its
// part as segments, one per pair it touches. A segment that covers all units
// of its pair writes the output; the others write partial sums (unnormalised
// O, row maximum, row sum), which the combine kernel adds in key order: no
// atomics, and a result that depends on the inputs alone.
#pragma once

#include "xn_common.cuh"
#include "xn_internal.h"

namespace xn {
namespace paged {

struct Tile {
  int32_t req, tok0, ntok;  // request, its first row of q, tokens in the tile
  int32_t units;            // key tiles that its rows see (at least 1)
  int64_t pos0;             // position of the first token; negative: it sees no key
  int64_t cstart;           // cost of the tiles before it (for one kv head)
};

struct Start {
  int32_t tile, head, k;  // where a CTA's part begins: k-th unit of (tile, head)
  int32_t pad;
};

struct Header {
  int32_t ctas;  // parts in use
};

struct Args {
  void *out;
  const void *q, *k, *v;
  const int32_t *table;
  const int64_t *q_start, *kv_len;
  int64_t n_tokens, n_pages, max_blocks, q_stride, page_stride, head_stride, slot_stride, window;
  int32_t requests, h, h_kv, group, group_mul, page_shift;
  int32_t tile_tokens, bn, parts, pair_cost, min_cost;
  float scale_log2;  // scale * log2(e): scores enter exp2
  int *err_flag;
  Header *header;
  Tile *tiles;
  Start *starts;  // of the parts in use, and the end of the last
  float *partial;  // 2 * parts records
};

// First key that a query tile's rows see, and its key tile.
__device__ __forceinline__ int64_t key_lo(const Tile &t, int64_t window) {
  const int64_t lo = t.pos0 - window + 1;
  return window > 0 && lo > 0 ? lo : 0;
}
__device__ __forceinline__ int64_t first_unit(const Tile &t, int64_t window, int bn) { return key_lo(t, window) / bn; }

// Record of part c's partial sums: [rows][D] of O, then rows maxima, rows sums.
// Part c has two: 0 for the segment it begins with, 1 for its last one.
__device__ __forceinline__ float *partial_of(const Args &a, int part, int which, int rows, int d) {
  return a.partial + (static_cast<int64_t>(part) * 2 + which) * (static_cast<int64_t>(rows) * (d + 2));
}

// Token of a query tile's row: row / group for row < 256, group <= 64.
__device__ __forceinline__ int token_of(const Args &a, int row) { return row * a.group_mul >> 16; }

// The segments of one CTA's part, in order.
struct Walk {
  int32_t tile, head, k, take;  // the segment: key tiles k .. k + take - 1 of (tile, head)
  Start end;
  bool first;

  __device__ __forceinline__ Walk(const Args &a, int part) {
    tile = head = k = take = 0;
    end = Start{0, 0, 0, 0};
    first = true;
    if (part >= a.header->ctas) return;
    const Start s = a.starts[part];
    tile = s.tile;
    head = s.head;
    k = s.k;
    end = a.starts[part + 1];
  }
  // Loads the tile of the current segment; false when the part is done.
  __device__ __forceinline__ bool get(const Args &a, Tile &t) {
    const bool same = tile == end.tile && head == end.head;
    if (tile > end.tile || (tile == end.tile && head > end.head) || (same && k >= end.k)) return false;
    t = a.tiles[tile];
    take = (same ? end.k : t.units) - k;
    return true;
  }
  __device__ __forceinline__ bool whole(const Tile &t) const { return k == 0 && take == t.units; }
  __device__ __forceinline__ void next(const Args &a) {
    k = 0;
    first = false;
    if (++head == a.h_kv) {
      head = 0;
      ++tile;
    }
  }
};

}  // namespace paged
}  // namespace xn
