// xn_paged.cu - the paged KV cache's bookkeeping and its append, for sm_100a:
// block tables, positions and slots of a step built from request lengths, and
// RoPE on the packed projection written straight into the pages.
#include "xn_common.cuh"
#include "xn_internal.h"

namespace xn {
namespace {

// ---------------------------------------------------------------------------
// Plan. Three prefix sums over the requests (new tokens, pages taken, pages
// returned) place everything; the rest is independent lookups. The sums of a
// few thousand lengths cost about as much as one more launch, so every block
// forms them by itself in shared memory and then takes its share of the
// tokens and pages: one launch, no communication between blocks. For that no
// block may read what another writes: tokens of pages taken in this step look
// them up in the ring rather than in the table, pages returned go to ring
// entries that were empty before the step, and lengths and ring state come
// out in other arrays than they came in.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr size_t kPlanStaticSmem = 512;  // at least what the kernel declares besides its prefix sums

struct PlanParams {
  int64_t *q_start, *kv_len, *positions, *slots, *ring_out;
  int32_t *table, *ring;
  const int64_t *lens, *new_len, *ring_state;
  int64_t requests, max_blocks, n_pages, token_cap;
  int page_shift;
  int *err_flag;
};

__device__ __forceinline__ int64_t warp_scan_incl(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Last i in [0, n) with pre[i] <= x (pre ascending, pre[0] = 0 <= x).
__device__ __forceinline__ int find_le(const int32_t *pre, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
  griddep_wait();
  griddep_release();
  extern __shared__ int32_t plan_smem[];
  __shared__ int64_t warp_tot[3][kPlanThreads / 32];
  __shared__ int bad_any;
  static_assert(sizeof(warp_tot) + sizeof(bad_any) + 16 <= kPlanStaticSmem);
  const int n = static_cast<int>(p.requests);
  int32_t *tok_pre = plan_smem, *need_pre = tok_pre + n + 1, *back_pre = need_pre + n + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t page_mask = (int64_t{1} << p.page_shift) - 1;
  const int64_t len_max = p.max_blocks << p.page_shift;
  if (tid == 0) bad_any = 0;
  __syncthreads();

  // Prefix sums: a thread takes a run of requests (their loads go together: with
  // a scan for every 512 requests instead, 4096 took 17 us), then the threads'
  // sums are scanned. Sums are 64-bit; their 32-bit copies are used only when
  // the totals passed the checks below.
  const int run = (n + kPlanThreads - 1) / kPlanThreads, begin = tid * run < n ? tid * run : n;
  const int end = begin + run < n ? begin + run : n;
  int64_t total[3] = {0, 0, 0};
  int bad = 0;
#pragma unroll 4
  for (int i = begin; i < end; ++i) {
    const int64_t len = p.lens[i], add = p.new_len[i];
    int64_t v[3] = {0, 0, 0};
    if (len < 0 || len > len_max) {
      bad |= XN_DEVERR_RANGE;
    } else {
      const int64_t held = (len + page_mask) >> p.page_shift;
      if (add < 0) {
        v[2] = held;
      } else if (add > p.token_cap || len + add > len_max) {
        bad |= XN_DEVERR_FULL;
      } else {
        v[0] = add;
        v[1] = ((len + add + page_mask) >> p.page_shift) - held;
      }
    }
    tok_pre[i] = static_cast<int32_t>(total[0]);
    need_pre[i] = static_cast<int32_t>(total[1]);
    back_pre[i] = static_cast<int32_t>(total[2]);
#pragma unroll
    for (int k = 0; k < 3; ++k) total[k] += v[k];
  }
  int64_t carry[3], before[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    before[k] = warp_scan_incl(total[k]);
    if (lane == 31) warp_tot[k][warp] = before[k];
    before[k] -= total[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int64_t s = warp_scan_incl(lane < kPlanThreads / 32 ? warp_tot[k][lane] : 0);  // every warp for itself
    carry[k] = __shfl_sync(0xffffffffu, s, 31);
    const int64_t u = __shfl_sync(0xffffffffu, s, warp > 0 ? warp - 1 : 0);
    before[k] += warp > 0 ? u : 0;
  }
#pragma unroll 4
  for (int i = begin; i < end; ++i) {
    tok_pre[i] += static_cast<int32_t>(before[0]);
    need_pre[i] += static_cast<int32_t>(before[1]);
    back_pre[i] += static_cast<int32_t>(before[2]);
  }
  const int64_t head = p.ring_state[0], count = p.ring_state[1];
  if (head < 0 || head >= p.n_pages || count < 0 || count > p.n_pages - carry[2]) bad |= XN_DEVERR_RANGE;
  if (carry[0] > p.token_cap || carry[1] > count) bad |= XN_DEVERR_FULL;
  if (bad) atomicOr(&bad_any, bad);
  __syncthreads();
  bad = bad_any;

  const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
  if (bad) {
    if (first == 0) {
      if (p.err_flag != nullptr) atomicOr(p.err_flag, bad);
      p.ring_out[0] = head;
      p.ring_out[1] = count;
      p.q_start[n] = 0;
    }
    for (int64_t i = first; i < n; i += step) {
      p.q_start[i] = 0;
      p.kv_len[i] = p.lens[i];
    }
    for (int64_t k = first; k < p.token_cap; k += step) p.positions[k] = p.slots[k] = -1;
    return;
  }
  const int32_t tokens = static_cast<int32_t>(carry[0]), need = static_cast<int32_t>(carry[1]);
  const int32_t back = static_cast<int32_t>(carry[2]);
  auto ring_at = [&](int64_t k) {  // entry k behind the head; k < 2 n_pages
    int64_t at = head + k;
    if (at >= p.n_pages) at -= p.n_pages;
    return at;
  };
  if (first == 0) {
    p.ring_out[0] = ring_at(need);
    p.ring_out[1] = count - need + back;
    p.q_start[n] = tokens;
  }
  for (int64_t i = first; i < n; i += step) {
    const int64_t add = p.new_len[i];
    p.q_start[i] = tok_pre[i];
    p.kv_len[i] = add < 0 ? 0 : p.lens[i] + add;
  }
  for (int64_t k = first; k < p.token_cap; k += step) {
    int64_t pos = -1, slot = -1;
    if (k < tokens) {
      const int i = find_le(tok_pre, n, static_cast<int32_t>(k));
      const int64_t len = p.lens[i];
      pos = len + (k - tok_pre[i]);
      const int64_t held = (len + page_mask) >> p.page_shift, blk = pos >> p.page_shift;
      const int32_t page = blk < held ? p.table[i * p.max_blocks + blk] : p.ring[ring_at(need_pre[i] + (blk - held))];
      if (page >= 0 && page < p.n_pages)
        slot = (static_cast<int64_t>(page) << p.page_shift) + (pos & page_mask);
      else if (p.err_flag != nullptr)
        atomicOr(p.err_flag, XN_DEVERR_RANGE);
    }
    p.positions[k] = pos;
    p.slots[k] = slot;
  }
  for (int64_t k = first; k < need; k += step) {
    const int i = find_le(need_pre, n, static_cast<int32_t>(k));
    const int64_t held = (p.lens[i] + page_mask) >> p.page_shift;
    p.table[i * p.max_blocks + held + (k - need_pre[i])] = p.ring[ring_at(k)];
  }
  for (int64_t k = first; k < back; k += step) {
    const int i = find_le(back_pre, n, static_cast<int32_t>(k));
    p.ring[ring_at(count + k)] = p.table[i * p.max_blocks + (k - back_pre[i])];
  }
}

// ---------------------------------------------------------------------------
// Append. Bytes bound: every element of the projection is read once and
// written once. A work item is two 16-byte vectors: one of each half of a head
// row (half-split) or two neighbouring ones (interleaved). A thread reads its
// item before it knows the token's slot and position, which the tables wait
// for (timed against each other: this order 129, slot first 154, two items a
// thread 135 us). 32768 tokens of 48 heads of 128 now take 143 to 147 us, 0.85
// of the measured copy rate.
// ---------------------------------------------------------------------------
struct PagedAppendParams {
  void *q_out, *k_pages, *v_pages;
  const void *qkv, *cos, *sin;
  const int64_t *positions, *slots;
  int64_t n_tokens, max_pos, n_slots, page_stride, head_stride, slot_stride;
  int h, h_kv, page_shift;
  int *err_flag;
};

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendParams p) {
  griddep_wait();
  griddep_release();
  constexpr int V = Elem<T>::kVec, C = D / (2 * V);  // work items of a head row
  const int heads = p.h + 2 * p.h_kv, c = threadIdx.x % C;
  const int e1 = kInterleaved ? c * 2 * V : c * V, e2 = kInterleaved ? e1 + V : e1 + D / 2;
  const int64_t src_row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / C;  // head row of the projection
  if (src_row >= p.n_tokens * heads) return;
  const int64_t tok = src_row / heads;
  const int head = static_cast<int>(src_row - tok * heads);
  const T *src = static_cast<const T *>(p.qkv) + src_row * D;
  const uint4 x1 = ld_stream(src + e1), x2 = ld_stream(src + e2);
  const int64_t slot = p.slots[tok], pos = p.positions[tok];
  if (slot == -1) return;
  if (slot < 0 || slot >= p.n_slots || pos < 0 || pos >= p.max_pos) {
    if (head == 0 && c == 0 && p.err_flag != nullptr) atomicOr(p.err_flag, XN_DEVERR_RANGE);
    return;
  }
  T *dst;
  if (head < p.h) {
    dst = static_cast<T *>(p.q_out) + (tok * p.h + head) * D;
  } else {
    const bool is_k = head < p.h + p.h_kv;
    const int kv = head - p.h - (is_k ? 0 : p.h_kv);
    const int64_t page = slot >> p.page_shift, row = slot & ((int64_t{1} << p.page_shift) - 1);
    dst = static_cast<T *>(is_k ? p.k_pages : p.v_pages) + page * p.page_stride + kv * p.head_stride + row * p.slot_stride;
  }
  if (head >= p.h + p.h_kv) {
    st_vec(dst + e1, x1);
    st_vec(dst + e2, x2);
    return;
  }
  // Pair j of the item sits at table entry c * V + j in both forms.
  const T *cs = static_cast<const T *>(p.cos) + pos * (D / 2) + c * V;
  const T *sn = static_cast<const T *>(p.sin) + pos * (D / 2) + c * V;
  float a[V], b[V], cv[V], sv[V], y1[V], y2[V];
  unpack<T>(x1, a);
  unpack<T>(x2, b);
  unpack<T>(ld_cached(cs), cv);
  unpack<T>(ld_cached(sn), sv);
  if constexpr (kInterleaved) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      y1[2 * j] = __fmaf_rn(a[2 * j], cv[j], -__fmul_rn(a[2 * j + 1], sv[j]));
      y1[2 * j + 1] = __fmaf_rn(a[2 * j], sv[j], __fmul_rn(a[2 * j + 1], cv[j]));
      y2[2 * j] = __fmaf_rn(b[2 * j], cv[V / 2 + j], -__fmul_rn(b[2 * j + 1], sv[V / 2 + j]));
      y2[2 * j + 1] = __fmaf_rn(b[2 * j], sv[V / 2 + j], __fmul_rn(b[2 * j + 1], cv[V / 2 + j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      y1[j] = __fmaf_rn(a[j], cv[j], -__fmul_rn(b[j], sv[j]));
      y2[j] = __fmaf_rn(a[j], sv[j], __fmul_rn(b[j], cv[j]));
    }
  }
  st_vec(dst + e1, pack<T>(y1));
  st_vec(dst + e2, pack<T>(y2));
}

template <typename T, int D>
int launch_paged_append(const PagedAppendParams &p, int interleaved, cudaStream_t st, const char *op) {
  const int64_t items = p.n_tokens * (p.h + 2 * p.h_kv) * (D / (2 * Elem<T>::kVec));
  const int64_t grid = ceil_div(items, int64_t{256});
  if (grid > 0x7fffffffLL) return fail(XN_E_INVALID, "%s: too many elements", op);
  launch_k(interleaved ? paged_append_kernel<T, D, true> : paged_append_kernel<T, D, false>, dim3(grid), dim3(256), 0, st, p);
  return check_launch(op);
}

}  // namespace

int check_pages(const char *op, int64_t n_pages, int64_t page_size, int64_t h_kv, int64_t d, int64_t page_stride,
                int64_t head_stride, int64_t slot_stride, int dtype) {
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return fail(XN_E_INVALID, "%s: page size %lld is not a power of two in [8, 256]", op, (long long)page_size);
  if (n_pages <= 0 || n_pages > 0x7fffffffLL) return fail(XN_E_INVALID, "%s: n_pages=%lld out of range", op, (long long)n_pages);
  if (d != 32 && d != 64 && d != 128) return fail(XN_E_INVALID, "%s: head dim %lld not in {32, 64, 128}", op, (long long)d);
  const int64_t per16 = 16 / dtype_bytes(dtype);
  const int64_t strides[3] = {page_stride, head_stride, slot_stride};
  const int64_t counts[3] = {n_pages, h_kv, page_size};
  for (int k = 0; k < 3; ++k) {
    if (strides[k] % per16 != 0)
      return fail(XN_E_INVALID, "%s: cache strides must be multiples of 16 bytes (got %lld elements)", op, (long long)strides[k]);
    if (strides[k] < 0 || (counts[k] > 1 && strides[k] < d) || strides[k] > (int64_t{1} << 39) / dtype_bytes(dtype))
      return fail(XN_E_INVALID, "%s: cache stride %lld out of range", op, (long long)strides[k]);
  }
  return XN_OK;
}

}  // namespace xn

extern "C" {

int xn_paged_plan(int64_t *q_start, int64_t *kv_len, int64_t *positions, int64_t *slots, int64_t *ring_state_out,
                  int32_t *block_table, int32_t *free_ring, const int64_t *lens, const int64_t *new_len,
                  const int64_t *ring_state, int64_t requests, int64_t max_blocks, int64_t n_pages,
                  int64_t page_size, int64_t token_cap, int *err_flag, void *stream) {
  using namespace xn;
  const char *op = "xn_paged_plan";
  if (requests < 0 || max_blocks < 0 || token_cap < 0) return fail(XN_E_INVALID, "%s: negative size", op);
  if (requests > XN_PAGED_MAX_REQUESTS)
    return fail(XN_E_INVALID, "%s: %lld requests exceed %d", op, (long long)requests, XN_PAGED_MAX_REQUESTS);
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return fail(XN_E_INVALID, "%s: page size %lld is not a power of two in [8, 256]", op, (long long)page_size);
  if (n_pages <= 0 || n_pages > 0x7fffffffLL || max_blocks > 0x7fffffffLL || token_cap > 0x7fffffffLL)
    return fail(XN_E_INVALID, "%s: n_pages=%lld max_blocks=%lld token_cap=%lld out of range", op, (long long)n_pages,
                (long long)max_blocks, (long long)token_cap);
  if (q_start == nullptr || ring_state_out == nullptr || ring_state == nullptr || free_ring == nullptr ||
      (requests > 0 && (kv_len == nullptr || lens == nullptr || new_len == nullptr)) ||
      (requests > 0 && max_blocks > 0 && block_table == nullptr) ||
      (token_cap > 0 && (positions == nullptr || slots == nullptr)))
    return fail(XN_E_INVALID, "%s: null pointer", op);
  // Every block reads all lengths and the ring state while others write.
  struct Range {
    const int64_t *at;
    int64_t n;
  };
  const Range in[] = {{lens, requests}, {new_len, requests}, {ring_state, 2}};
  const Range out[] = {{q_start, requests + 1}, {kv_len, requests}, {positions, token_cap}, {slots, token_cap}, {ring_state_out, 2}};
  auto from = [](const Range &r) { return reinterpret_cast<uintptr_t>(r.at); };
  auto to = [](const Range &r) { return reinterpret_cast<uintptr_t>(r.at) + static_cast<uintptr_t>(r.n) * sizeof(int64_t); };
  for (const Range &i : in)
    for (const Range &o : out)
      if (i.n > 0 && o.n > 0 && from(i) < to(o) && from(o) < to(i))
        return fail(XN_E_INVALID, "%s: an output must not overlap an input array", op);
  int shift = 0;
  while ((int64_t{1} << shift) < page_size) ++shift;
  PlanParams p{q_start, kv_len, positions, slots, ring_state_out, block_table, free_ring, lens, new_len, ring_state,
               requests, max_blocks, n_pages, token_cap, shift, err_flag};
  const size_t smem = 3 * static_cast<size_t>(requests + 1) * sizeof(int32_t);
  // The 48 KB that a block has without asking cover both kinds of shared memory.
  if (smem + kPlanStaticSmem > 48 * 1024 &&
      cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(3 * (XN_PAGED_MAX_REQUESTS + 1) * sizeof(int32_t))) != cudaSuccess)
    return check_launch(op);
  const int64_t work = token_cap > requests ? token_cap : requests;
  int64_t grid = ceil_div(work > 0 ? work : 1, int64_t{kPlanThreads});
  if (grid > sm_count()) grid = sm_count();
  launch_k(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, as_stream(stream), p);
  return check_launch(op);
}

int xn_paged_append_rope(void *q_out, void *k_pages, void *v_pages, const void *qkv, const void *cos,
                         const void *sin, const int64_t *positions, const int64_t *slots, int64_t n_tokens,
                         int64_t h, int64_t h_kv, int64_t d, int64_t max_pos, int64_t n_pages, int64_t page_size,
                         int64_t page_stride, int64_t head_stride, int64_t slot_stride, int interleaved, int dtype,
                         int *err_flag, void *stream) {
  using namespace xn;
  const char *op = "xn_paged_append_rope";
  if (!is_float_dtype(dtype)) return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (n_tokens < 0 || h <= 0 || h_kv <= 0 || max_pos < 0) return fail(XN_E_INVALID, "%s: negative or empty size", op);
  if (h > 65536 || h_kv > 65536) return fail(XN_E_INVALID, "%s: too many heads", op);
  if (const int rc = check_pages(op, n_pages, page_size, h_kv, d, page_stride, head_stride, slot_stride, dtype)) return rc;
  if (n_tokens == 0) return ok();
  if (q_out == nullptr || k_pages == nullptr || v_pages == nullptr || qkv == nullptr || cos == nullptr ||
      sin == nullptr || positions == nullptr || slots == nullptr)
    return fail(XN_E_INVALID, "%s: null pointer", op);
  const void *ptrs[] = {q_out, k_pages, v_pages, qkv, cos, sin};
  for (const void *ptr : ptrs)
    if (!is_aligned16(ptr)) return fail(XN_E_INVALID, "%s: tensors must be 16-byte aligned", op);
  int shift = 0;
  while ((int64_t{1} << shift) < page_size) ++shift;
  PagedAppendParams p{q_out, k_pages, v_pages, qkv, cos, sin, positions, slots, n_tokens, max_pos, n_pages * page_size,
                      page_stride, head_stride, slot_stride, static_cast<int>(h), static_cast<int>(h_kv), shift, err_flag};
  XN_DISPATCH_FLOAT(dtype, {
    if (d == 32) return launch_paged_append<T, 32>(p, interleaved, as_stream(stream), op);
    if (d == 64) return launch_paged_append<T, 64>(p, interleaved, as_stream(stream), op);
    return launch_paged_append<T, 128>(p, interleaved, as_stream(stream), op);
  });
  return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
}

}  // extern "C"
