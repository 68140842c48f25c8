// xn_paged_attn.cuh - what the paged attention's kernels share: arguments, the
// work list that the schedule kernel builds on the device, and the walk over it.
//
// Work. A query tile is up to `tile_tokens` consecutive new tokens of one
// request with the group of query heads that share a kv head: rows (token,
// head of the group), token-major. A unit is one key tile of kBN keys against
// one (query tile, kv head). The units of all (tile, head) pairs, in that
// order, form one line, which is cut into equal parts, one per CTA, wherever
// the cuts fall: lengths are known on the device only, and equal parts keep
// every SM busy for ragged batches and for one long request alike. A CTA
// walks its part as segments, one per (tile, head) it touches. A segment that
// covers all units of its pair writes the output; the others write partial
// sums (unnormalised O, row maximum, row sum), which the combine kernel adds
// in key order: no atomics, and a result that depends on the inputs alone.
#pragma once

#include "xn_common.cuh"
#include "xn_internal.h"

namespace xn {
namespace paged {

struct Tile {
  int32_t req, tok0, ntok;  // request, its first row of q, tokens in the tile
  int32_t units;            // key tiles that its rows see (at least 1)
  int64_t pos0;             // position of the first token; negative: it sees no key
  int64_t ustart;           // units of the tiles before it (for one kv head)
};

struct Start {
  int32_t tile, head, k;  // where a CTA's part begins: k-th unit of (tile, head)
  int32_t pad;
};

struct Header {
  int64_t n_tiles, units;  // units: of all heads
  int32_t ctas, pad;       // parts in use
};

struct Args {
  void *out;
  const void *q, *k, *v;
  const int32_t *table;
  const int64_t *q_start, *kv_len;
  int64_t n_tokens, n_pages, max_blocks, q_stride, page_stride, head_stride, slot_stride, window;
  int32_t requests, h, h_kv, group, page_shift;
  int32_t tile_tokens, bn, parts, min_units;
  float scale_log2;  // scale * log2(e): scores enter exp2
  int *err_flag;
  Header *header;
  Tile *tiles;
  Start *starts;  // parts + 1
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

// The segments of one CTA's part, in order.
struct Walk {
  int64_t left;  // units left in the part
  int32_t tile, head, k, take;
  bool first;

  __device__ __forceinline__ Walk(const Args &a, int part) {
    const int64_t w = a.header->units;
    const int ctas = a.header->ctas;
    left = 0;
    first = true;
    take = 0;
    if (part >= ctas) return;
    left = (part + 1) * w / ctas - part * w / ctas;
    const Start s = a.starts[part];
    tile = s.tile;
    head = s.head;
    k = s.k;
  }
  // Loads the tile of the current segment; false when the part is done.
  __device__ __forceinline__ bool get(const Args &a, Tile &t) {
    if (left <= 0) return false;
    t = a.tiles[tile];
    const int64_t rest = t.units - k;
    take = static_cast<int32_t>(rest < left ? rest : left);
    return true;
  }
  __device__ __forceinline__ bool whole(const Tile &t) const { return k == 0 && take == t.units; }
  __device__ __forceinline__ void next(const Args &a) {
    left -= take;
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
