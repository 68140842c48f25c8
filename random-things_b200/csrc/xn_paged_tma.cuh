// xn_paged_tma.cuh - the paged attention's kernels that load K and V tiles by
// TMA: barriers with time limits, tile layout, loads of a tile page by page.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "xn_paged_attn_tc.h"

namespace xn {
namespace paged {
namespace {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Waits with a converged warp for the phase of `parity`; false when it did not
// come within `limit` clocks or another role gave up (then nothing that the
// phase stands for may be used). All lanes poll: with one lane polling in a branch of
// its own, what follows no longer counts as equal in all lanes, and operands
// leave the uniform registers (measured: prefill of 8192 tokens 0.69 -> 0.89 ms).
// The limit matters only behind the first look (tested before it: 589 -> 639 us).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *gave_up, long long limit) {
  bool got = mbar_try(bar, parity);
  if (!got) {
    const long long t0 = clock64();
    do {
#pragma unroll 1
      for (int i = 0; i < 64 && !got; ++i) got = mbar_try(bar, parity);
    } while (!got && !*gave_up && clock64() - t0 < limit);
    if (!got) *gave_up = 1;
  }
  return __all_sync(0xffffffffu, got);
}
// The end of a role that copies or products in flight would outlive: waits for
// the phase whoever gave up, and up to the full limit.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try(bar, parity) && clock64() - t0 < kWaitClocks) {
  }
}
// One arrival for a warp, behind what all its lanes did.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A tile of R rows of D 16-bit elements in shared memory as TMA writes it with
// a 128-byte swizzle (64-byte for D = 32): rows of up to 64 elements, wider
// ones as sub-tiles one behind the other; 16-byte chunks of 8 rows permuted so
// that neither row nor column reads meet bank conflicts.
template <int D, int R>
struct Swizzled {
  static constexpr int kRowBytes = D >= 64 ? 128 : 64;  // bytes of a swizzled row
  static constexpr int kHalves = D >= 64 ? D / 64 : 1;  // sub-tiles
  static constexpr int kSub = R * kRowBytes;            // bytes of one sub-tile
  static constexpr int kTile = kHalves * kSub;

  // Byte offset of 16-byte chunk j of row r.
  __device__ __forceinline__ static uint32_t chunk_at(int r, int j) {
    if constexpr (D >= 64)
      return (j >> 3) * kSub + r * 128 + (((j & 7) ^ (r & 7)) << 4);
    else
      return r * 64 + ((j ^ ((r >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int row, int head,
                                         int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(bar), "r"(x), "r"(row), "r"(head), "r"(page)
      : "memory");
}

// The loads of one warp for a key tile of R keys, one box a lane: a page's rows
// (or R rows of a larger page) in one sub-tile.
template <int D, int R>
struct TileLoad {
  using Tiles = Swizzled<D, R>;
  int box_rows, boxes, row0, half;

  __device__ __forceinline__ explicit TileLoad(const Args &a) {
    box_rows = (1 << a.page_shift) < R ? 1 << a.page_shift : R;
    boxes = R / box_rows * Tiles::kHalves;  // at most 32: pages have 8 rows or more
    const int lane = threadIdx.x & 31;
    row0 = lane / Tiles::kHalves * box_rows;
    half = lane % Tiles::kHalves;
  }
  __device__ __forceinline__ bool mine() const { return (threadIdx.x & 31) < boxes; }
  // This lane's page for the tile at key0; keys outside [lo, hi), which no row
  // of the query tile sees, are not looked up. A page outside the pool, like
  // those, reads as zeros: TMA fills what lies outside the tensor.
  __device__ __forceinline__ int page(const Args &a, const Tile &t, int64_t key0, int64_t lo, int64_t hi) const {
    const int64_t key = key0 + row0;
    if (!mine() || key >= hi || key + box_rows <= lo) return static_cast<int>(a.n_pages);
    const int32_t id = a.table[t.req * a.max_blocks + (key >> a.page_shift)];
    if (id >= 0 && id < a.n_pages) return id;
    if (a.err_flag != nullptr) atomicOr(a.err_flag, XN_DEVERR_RANGE);
    return static_cast<int>(a.n_pages);
  }
  __device__ __forceinline__ void load(const Args &a, const CUtensorMap *map, uint32_t tile, uint32_t bar, int64_t key0,
                                       int head, int page) const {
    const int row = static_cast<int>((key0 + row0) & ((int64_t{1} << a.page_shift) - 1));
    if (mine()) tma_load(tile + half * Tiles::kSub + row0 * Tiles::kRowBytes, map, bar, half * 64, row, head, page);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>)
    return f2_to_h2(a, b);
  else
    return f2_to_bf2(a, b);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>)
    return h2_to_f2(w);
  else
    return bf2_to_f2(w);
}
// Whether a pair of 16-bit values holds an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool non_finite2(uint32_t w) {
  constexpr uint32_t e = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A pool as a 4-D tensor (d, slot, head, page); a box is `rows` slots of one page and head, or
// a whole page where that is less.
inline bool make_map(CUtensorMap *map, const void *pool, const Args &a, int d, int rows, bool bf16) {
  const int page_size = 1 << a.page_shift;
  EncodeFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(page_size), static_cast<cuuint64_t>(a.h_kv),
                              static_cast<cuuint64_t>(a.n_pages)};
  // A dimension of one element may come with any stride: give it a valid one.
  const int64_t ss = page_size > 1 ? a.slot_stride : d, hs = a.h_kv > 1 ? a.head_stride : ss * page_size;
  const int64_t ps = a.n_pages > 1 ? a.page_stride : ss * page_size;
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss) * 2, static_cast<cuuint64_t>(hs) * 2, static_cast<cuuint64_t>(ps) * 2};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(d < 64 ? d : 64), static_cast<cuuint32_t>(page_size < rows ? page_size : rows), 1, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(pool), dims,
            strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, d < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace paged
}  // namespace xn
