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
// O, row maximum, row sum). Whichever CTA finishes a cut pair last adds them
// (for chunks: a kernel behind), in key order: who that is changes nothing in
// the result.
#pragma once

#include <math.h>

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
  int32_t first;          // k > 0: the first part that begins inside this pair
};

struct Header {
  int32_t ctas;  // parts in use
};

// Of the pair that part c is the first to begin inside: the last such part, and
// how many pieces are done.
struct Cut {
  int32_t last, done;
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
  long long wait_clocks;  // a wait on a barrier gives up after these; 0: the warps of the softmax do before their first one
  int *err_flag;
  Header *header;
  Tile *tiles;
  Start *starts;  // of the parts in use, and the end of the last
  Cut *cuts;      // by first part
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

// Adds rows row0 .. row1 - 1 of a cut pair's partial sums and writes them out:
// `count` threads (a multiple of 32), this one number i. D / 4 lanes take a row
// and 4 columns each; one lane a piece reads its maximum and sum, so that a row
// costs two trips to memory however it was cut, and four rows go together.
template <typename T, int D>
__device__ __forceinline__ void combine_rows(const Args &a, const Tile &t, int head, int first, int last, int bm, int row0,
                                             int row1, int i, int count) {
  constexpr int C = D / 4, R = 4;
  const Start b = a.starts[first - 1];
  const bool own = b.tile == a.starts[first].tile && b.head == head;  // the first piece begins its part
  const int lane = i % C, col = lane * 4, step = count / C, pieces = last - first + 2;
  auto record = [&](int p) { return partial_of(a, first - 1 + p, p == 0 && !own ? 1 : 0, bm, D); };
  for (int base = row0; base < row1; base += R * step) {
    int row[R];
    float mx[R], l[R];
    float4 o[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int at = base + r * step + i / C;
      row[r] = at < row1 ? at : row1 - 1;
      mx[r] = -INFINITY;
      l[r] = 0.f;
      o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int p = lane; p < pieces; p += C) {
      const float *rec = record(p) + bm * D;
#pragma unroll
      for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], __ldcg(rec + row[r]));
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = C / 2; x > 0; x >>= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], x));
    for (int p0 = 0; p0 < pieces; p0 += C) {
      float f[R];  // of piece p0 + lane
#pragma unroll
      for (int r = 0; r < R; ++r) f[r] = 0.f;
      if (p0 + lane < pieces) {
        const float *rec = record(p0 + lane) + bm * D;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m = __ldcg(rec + row[r]), sum = __ldcg(rec + bm + row[r]);
          f[r] = m == -INFINITY ? 0.f : ex2_approx((m - mx[r]) * a.scale_log2);
          l[r] = __fmaf_rn(sum, f[r], l[r]);
        }
      }
      const int n = pieces - p0 < C ? pieces - p0 : C;
#pragma unroll 2
      for (int p = 0; p < n; ++p) {
        const float *rec = record(p0 + p);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 x = __ldcg(reinterpret_cast<const float4 *>(rec + row[r] * D + col));
          const float w = __shfl_sync(0xffffffffu, f[r], p, C);
          o[r].x = __fmaf_rn(x.x, w, o[r].x);
          o[r].y = __fmaf_rn(x.y, w, o[r].y);
          o[r].z = __fmaf_rn(x.z, w, o[r].z);
          o[r].w = __fmaf_rn(x.w, w, o[r].w);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int x = C / 2; x > 0; x >>= 1) l[r] = __fadd_rn(l[r], __shfl_xor_sync(0xffffffffu, l[r], x));
      if (base + r * step + i / C >= row1) continue;
      const int tk = token_of(a, row[r]);
      const float inv = __fdiv_rn(1.f, l[r]);
      const bool none = t.pos0 + tk < 0;
      T *dst = static_cast<T *>(a.out) + (static_cast<int64_t>(t.tok0 + tk) * a.h + head * a.group + row[r] - tk * a.group) * D + col;
      const float y[4] = {o[r].x * inv, o[r].y * inv, o[r].z * inv, o[r].w * inv};
      T v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = Elem<T>::from_f32(none ? 0.f : y[j]);
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(v);
      else
        *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(v);
    }
    __syncwarp();
  }
}

// Ends a segment that is a piece of a cut pair: counts it, and where it is the
// last one to be done combines the pair's rows. For the `count` threads that
// wrote the piece, this one number i; `sync` is their barrier, `flag` a word of shared memory of theirs.
template <typename T, int D, typename Sync>
__device__ __forceinline__ void end_piece(const Args &a, const Walk &w, const Tile &t, int part, int bm, int i, int count,
                                          volatile int *flag, Sync sync) {
  __threadfence();
  sync();
  const int first = w.k > 0 ? a.starts[part].first : a.starts[part + 1].first;
  const int last = a.cuts[first].last;
  if (i == 0) *flag = atomicAdd(&a.cuts[first].done, 1) == last - first + 1;
  sync();
  if (*flag) {
    __threadfence();
    combine_rows<T, D>(a, t, w.head, first, last, bm, 0, t.ntok * a.group, i, count);
  }
}

}  // namespace paged
}  // namespace xn
