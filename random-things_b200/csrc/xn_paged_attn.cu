// xn_paged_attn.cu - causal attention of a step's new tokens over a paged KV
// cache, for sm_100a: the schedule, the f32 kernel and the call.
//
//   o = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  s_k = scale (q . k),  m = max_k s_k
//
// in one pass over the keys: a tile of scores moves the running maximum m,
// the sums so far shrink by exp(m_old - m_new), and the tile's terms are added.
#include <math.h>

#include <cstdlib>

#include "xn_paged_attn_tc.h"

namespace xn {
namespace paged {
namespace {

constexpr int kSchedThreads = 512;

// Sum of v over the threads before this one; `all` over all threads.
__device__ __forceinline__ int64_t block_scan_excl(int64_t v, int64_t *tot, int64_t &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](int64_t x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    return x;
  };
  const int64_t s = scan(v);
  if (lane == 31) tot[warp] = s;
  __syncthreads();
  const int64_t t = scan(lane < kSchedThreads / 32 ? tot[lane] : 0);  // every warp for itself
  all = __shfl_sync(0xffffffffu, t, 31);
  const int64_t before = __shfl_sync(0xffffffffu, t, warp > 0 ? warp - 1 : 0);
  __syncthreads();
  return (warp > 0 ? before : 0) + s - v;
}

// x / y and the remainder, in 32 bits where both fit (a 64-bit division takes several times as long).
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y)) : x / y;
}

// Builds the work list: one block, since it is a few thousand additions.
__global__ void __launch_bounds__(kSchedThreads) paged_schedule_kernel(const Args a) {
  griddep_wait();
  griddep_release();
  extern __shared__ int32_t tile_pre[];  // tiles of the requests before request i
  constexpr int kNear = 1024;
  __shared__ int64_t near[kNear];  // cstart of the first tiles
  __shared__ int64_t tot[kSchedThreads / 32];
  const int n = a.requests, tid = threadIdx.x;
  int64_t carry = 0, all;
  int bad = 0;
  for (int base = 0; base < n; base += kSchedThreads) {
    const int i = base + tid;
    int64_t v = 0;
    if (i < n) {
      const int64_t q0 = a.q_start[i], q1 = a.q_start[i + 1], kv = a.kv_len[i];
      if (q0 < 0 || q1 < q0 || q1 > a.n_tokens || kv < 0 || kv > (a.max_blocks << a.page_shift))
        bad = XN_DEVERR_RANGE;
      else
        v = (q1 - q0 + a.tile_tokens - 1) / a.tile_tokens;
    }
    const int64_t before = carry + block_scan_excl(v, tot, all);
    if (i < n) tile_pre[i] = static_cast<int32_t>(before);
    carry += all;
  }
  if (bad && a.err_flag != nullptr) atomicOr(a.err_flag, bad);
  // Requests with overlapping tokens (q_start not ascending) could list more
  // tiles than the workspace has room for.
  int64_t n_tiles = carry;
  const int64_t room = a.n_tokens / a.tile_tokens + n;
  if (n_tiles > room) {
    if (tid == 0 && a.err_flag != nullptr) atomicOr(a.err_flag, XN_DEVERR_RANGE);
    n_tiles = 0;
  }
  __syncthreads();
  carry = 0;
  for (int64_t base = 0; base < n_tiles; base += kSchedThreads) {
    const int64_t e = base + tid;
    Tile t{};
    if (e < n_tiles) {
      int lo = 0, hi = n;  // last request with tile_pre <= e
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_pre[mid] <= e)
          lo = mid;
        else
          hi = mid;
      }
      const int64_t j0 = (e - tile_pre[lo]) * a.tile_tokens, q0 = a.q_start[lo], nt = a.q_start[lo + 1] - q0;
      t.req = lo;
      t.tok0 = static_cast<int32_t>(q0 + j0);
      t.ntok = static_cast<int32_t>(nt - j0 < a.tile_tokens ? nt - j0 : a.tile_tokens);
      t.pos0 = a.kv_len[lo] - nt + j0;
      const int64_t end = t.pos0 + t.ntok;  // keys the last row sees end here
      const int64_t u = end <= 0 ? 1 : (end + a.bn - 1) / a.bn - first_unit(t, a.window, a.bn);
      t.units = static_cast<int32_t>(u);
    }
    t.cstart = carry + block_scan_excl(e < n_tiles ? t.units + a.pair_cost : 0, tot, all);
    carry += all;
    if (e < n_tiles) {
      a.tiles[e] = t;
      if (e < kNear) near[e] = t.cstart;
    }
  }
  const int64_t w = carry * a.h_kv;
  int64_t ctas = (w + a.min_cost - 1) / a.min_cost;
  if (ctas > a.parts) ctas = a.parts;
  if (tid == 0) {
    a.header->ctas = static_cast<int32_t>(ctas);
    a.starts[ctas] = Start{static_cast<int32_t>(n_tiles), 0, 0, 0};
  }
  __syncthreads();
  // A thread a part: the pair and the unit it begins with. A cut in what a pair
  // costs beyond its units moves to the pair's begin.
  for (int64_t c = tid; c < ctas; c += kSchedThreads) {
    const int64_t at = quotient(c * w, ctas);
    const int64_t one = quotient(at, a.h_kv);  // the tile with cstart <= at / h_kv
    int64_t lo = 0, hi = n_tiles;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if ((mid < kNear ? near[mid] : a.tiles[mid].cstart) <= one)
        lo = mid;
      else
        hi = mid;
    }
    const Tile t = a.tiles[lo];
    const int64_t pair = t.units + a.pair_cost, r = at - t.cstart * a.h_kv, head = quotient(r, pair);
    const int64_t begin = at - r + head * pair, k = r - head * pair - a.pair_cost;
    int64_t first = 0;
    if (k > 0) {
      // Part i begins at floor(i w / ctas): the first one behind the pair's extra cost, the last one before its end.
      first = quotient((begin + a.pair_cost + 1) * ctas + w - 1, w);
      if (first == c) a.cuts[c] = Cut{static_cast<int32_t>(quotient((begin + pair) * ctas + w - 1, w) - 1), 0};
    }
    a.starts[c] = Start{static_cast<int32_t>(lo), static_cast<int32_t>(head), static_cast<int32_t>(k > 0 ? k : 0),
                        static_cast<int32_t>(first)};
  }
}

// ---------------------------------------------------------------------------
// f32 on the CUDA cores: its tensor-core forms round the operands. 16 x 16
// threads, each with kRows rows and every 16th key (scores) or a run of columns
// (output). K and V tiles arrive by cp.async, the next one while this one is
// worked on; key tiles are as long as two tiles of both leave room for two
// CTAs an SM.
// ---------------------------------------------------------------------------
template <int D, int BM>
struct SimtCfg {
  static constexpr int kBN = D == 128 ? 32 : 64, kRows = BM / 16, kKeys = kBN / 16;
  static constexpr int kK = kBN * (D + 4), kV = kBN * D, kQ = BM * D, kP = BM * (kBN + 4);
  static constexpr size_t kSmem = sizeof(float) * (2 * (kK + kV) + kQ + kP);
};

template <int D, int BM>
__global__ void __launch_bounds__(256, 2) paged_attn_simt_kernel(const Args a) {
  griddep_wait();
  griddep_release();
  using Cfg = SimtCfg<D, BM>;
  constexpr int BN = Cfg::kBN, R = Cfg::kRows, KN = Cfg::kKeys, CP = D / 16, PS = BN + 4;
  extern __shared__ __align__(16) float simt_smem[];
  __shared__ int last_piece;
  float *Qs = simt_smem + 2 * (Cfg::kK + Cfg::kV), *Ps = Qs + Cfg::kQ;
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int part = blockIdx.x;
  const int page_mask = (1 << a.page_shift) - 1;
  Tile t;
  for (Walk w(a, part); w.get(a, t); w.next(a)) {
    const int rows = t.ntok * a.group;
    const int64_t key_hi = t.pos0 + t.ntok;  // keys from here on are seen by no row
    const int64_t lo = key_lo(t, a.window);
    const int64_t u0 = first_unit(t, a.window, BN) + w.k;
    // Starts the copies of key tile u0 + j; what no row sees, and pages outside the pool, become zeros.
    auto load = [&](int j) {
      float *ks = simt_smem + (j & 1) * (Cfg::kK + Cfg::kV), *vs = ks + Cfg::kK;
#pragma unroll
      for (int i = 0; i < BN * (D / 4) / 256; ++i) {
        const int row = (i * 256 + tid) / (D / 4), c = tid % (D / 4) * 4;
        const int64_t key = (u0 + j) * BN + row;
        int64_t at = 0;
        int bytes = 0;
        if (key < key_hi && key >= lo) {
          const int32_t page = a.table[t.req * a.max_blocks + (key >> a.page_shift)];
          if (page >= 0 && page < a.n_pages) {
            at = page * a.page_stride + w.head * a.head_stride + (static_cast<int>(key) & page_mask) * a.slot_stride + c;
            bytes = 16;
          } else if (a.err_flag != nullptr) {
            atomicOr(a.err_flag, XN_DEVERR_RANGE);
          }
        }
        const uint32_t kd = static_cast<uint32_t>(__cvta_generic_to_shared(ks + row * (D + 4) + c));
        const uint32_t vd = static_cast<uint32_t>(__cvta_generic_to_shared(vs + row * D + c));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(kd), "l"(static_cast<const float *>(a.k) + at), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(vd), "l"(static_cast<const float *>(a.v) + at), "r"(bytes) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();  // the last segment's reads are done
    load(0);
    for (int i = tid; i < BM * (D / 4); i += 256) {
      const int row = i / (D / 4), c = i % (D / 4) * 4, tk = token_of(a, row);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows)
        x = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + (t.tok0 + tk) * a.q_stride +
                                              (w.head * a.group + row - tk * a.group) * D + c);
      *reinterpret_cast<float4 *>(&Qs[row * D + c]) = x;
    }
    float o[R][CP], m[R], l[R];
    int64_t pos[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
      pos[r] = t.pos0 + token_of(a, ty * R + r);
#pragma unroll
      for (int c = 0; c < CP; ++c) o[r][c] = 0.f;
    }
    for (int j = 0; j < w.take; ++j) {
      if (j + 1 < w.take) {
        load(j + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      __syncthreads();
      const float *Ks = simt_smem + (j & 1) * (Cfg::kK + Cfg::kV), *Vs = Ks + Cfg::kK;
      const int64_t key0 = (u0 + j) * BN;
      float s[R][KN] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 kf[KN];
#pragma unroll
        for (int k = 0; k < KN; ++k) kf[k] = *reinterpret_cast<const float4 *>(&Ks[(tx + 16 * k) * (D + 4) + d]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 qf = *reinterpret_cast<const float4 *>(&Qs[(ty * R + r) * D + d]);
#pragma unroll
          for (int k = 0; k < KN; ++k) {
            s[r][k] = __fmaf_rn(qf.x, kf[k].x, s[r][k]);
            s[r][k] = __fmaf_rn(qf.y, kf[k].y, s[r][k]);
            s[r][k] = __fmaf_rn(qf.z, kf[k].z, s[r][k]);
            s[r][k] = __fmaf_rn(qf.w, kf[k].w, s[r][k]);
          }
        }
      }
      // Some row does not see some key: the keys' part in each row is then decided one by one.
      const bool masked = key0 + BN - 1 > t.pos0 || (a.window > 0 && key0 <= key_hi - 1 - a.window);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        bool seen[KN];
        float mx = m[r];
#pragma unroll
        for (int k = 0; k < KN; ++k) {
          const int64_t key = key0 + tx + 16 * k;
          seen[k] = !masked || (key <= pos[r] && (a.window == 0 || key > pos[r] - a.window));
          if (seen[k]) mx = fmaxf(mx, s[r][k]);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float base = mx == -INFINITY ? 0.f : mx;
        const float shrink = ex2_approx((m[r] - base) * a.scale_log2);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < KN; ++k) {
          const float p = seen[k] ? ex2_approx((s[r][k] - base) * a.scale_log2) : 0.f;
          sum += p;
          Ps[(ty * R + r) * PS + tx + 16 * k] = seen[k] ? p : -1.f;  // -1: no part in the row
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        m[r] = mx;
        l[r] = __fmaf_rn(l[r], shrink, sum);
#pragma unroll
        for (int c = 0; c < CP; ++c) o[r][c] *= shrink;
      }
      __syncwarp();  // a row's weights are written and read by one half warp
      auto weigh = [&](auto with_mask) {
#pragma unroll 2
        for (int k = 0; k < BN; k += 4) {
          float4 p[R];
#pragma unroll
          for (int r = 0; r < R; ++r) p[r] = *reinterpret_cast<const float4 *>(&Ps[(ty * R + r) * PS + k]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float vf[CP];
#pragma unroll
            for (int c = 0; c < CP; ++c) vf[c] = Vs[(k + i) * D + (CP >= 4 ? (c / 4) * 64 + tx * 4 + c % 4 : tx * CP + c)];
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float pk = i == 0 ? p[r].x : i == 1 ? p[r].y : i == 2 ? p[r].z : p[r].w;
#pragma unroll
              for (int c = 0; c < CP; ++c) {
                const float x = __fmaf_rn(pk, vf[c], o[r][c]);
                o[r][c] = decltype(with_mask)::value && pk < 0.f ? o[r][c] : x;
              }
            }
          }
        }
      };
      if (masked)
        weigh(std::true_type{});
      else
        weigh(std::false_type{});
      __syncthreads();  // before the tile after the next one takes this one's place
    }
    const bool whole = w.whole(t);
    float *part_o = whole ? nullptr : partial_of(a, part, w.first ? 0 : 1, BM, D);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = ty * R + r;
      if (row >= rows) continue;
      const float inv = __fdiv_rn(1.f, l[r]);
      const int tk = token_of(a, row);
      float *dst = static_cast<float *>(a.out) + (static_cast<int64_t>(t.tok0 + tk) * a.h + w.head * a.group + row - tk * a.group) * D;
#pragma unroll
      for (int c = 0; c < CP; ++c) {
        const int col = CP >= 4 ? (c / 4) * 64 + tx * 4 + c % 4 : tx * CP + c;
        if (whole)
          dst[col] = pos[r] < 0 ? 0.f : o[r][c] * inv;
        else
          part_o[row * D + col] = o[r][c];
      }
      if (!whole && tx == 0) {
        part_o[BM * D + row] = m[r];
        part_o[BM * D + BM + row] = l[r];
      }
    }
    if (!whole) end_piece<float, D>(a, w, t, part, BM, tid, 256, &last_piece, [] { __syncthreads(); });
  }
}

// How a call is cut: rows of a query tile, keys of a key tile, parts, what a
// pair costs beyond its units, the least cost of a part. A chunk's pair cost
// measured at heads of 128 (8192-token prompt / ragged chunks): 4 units 657 / 244 us, 6 units
// 547 / 243, 10 units 514 / 229, 13 units 519 / 232.
struct Shape {
  int bm, bn, parts, pair_cost, min_cost;
};

Shape shape_of(int64_t group, int64_t max_new, int64_t d, int dtype) {
  const bool few = max_new * group <= 16 && group <= 16;
  if (dtype == XN_F32) return Shape{few ? 16 : 64, d == 128 ? 32 : 64, 2 * sm_count(), 1, 3};
  return few ? Shape{kDecRows, kDecKeys, 2 * sm_count(), 2, 6} : Shape{kTcRows, kTcKeys, sm_count(), 10, 15};
}

struct Layout {
  int64_t tiles, starts, cuts, partial, bytes;
};

Layout layout_of(const Shape &s, int64_t n_tokens, int64_t requests, int64_t group, int64_t d) {
  auto up = [](int64_t v) { return (v + 255) & ~int64_t{255}; };
  Layout l;
  l.tiles = up(sizeof(Header));
  const int64_t tt = s.bm / group;
  l.starts = l.tiles + up(static_cast<int64_t>(sizeof(Tile)) * (n_tokens / tt + requests));
  l.cuts = l.starts + up(static_cast<int64_t>(sizeof(Start)) * (s.parts + 1));
  l.partial = l.cuts + up(static_cast<int64_t>(sizeof(Cut)) * s.parts);
  l.bytes = l.partial + up(static_cast<int64_t>(sizeof(float)) * 2 * s.parts * s.bm * (d + 2));
  return l;
}

// Clocks after which a wait of the TMA kernels gives up: kWaitClocks, or the
// value of the environment variable XN_PAGED_WAIT_CLOCKS (read once per
// process), a diagnostic that lets a test make the waits give up on valid inputs.
long long wait_clocks() {
  static const long long clocks = [] {
    const char *v = std::getenv("XN_PAGED_WAIT_CLOCKS");
    if (v == nullptr || *v == '\0') return kWaitClocks;
    const long long n = std::strtoll(v, nullptr, 10);
    return n < 0 ? 0 : n < kWaitClocks ? n : kWaitClocks;
  }();
  return clocks;
}

template <int D, int BM>
void launch_simt(const Args &a, cudaStream_t st) {
  constexpr size_t smem = SimtCfg<D, BM>::kSmem;
  cudaFuncSetAttribute(paged_attn_simt_kernel<D, BM>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_k(paged_attn_simt_kernel<D, BM>, dim3(a.parts), dim3(256), smem, st, a);
}

template <typename T, int D>
int launch_attn(const Args &a, const Shape &s, cudaStream_t st, const char *op) {
  const size_t smem = sizeof(int32_t) * (static_cast<size_t>(a.requests) + 1);
  launch_k(paged_schedule_kernel, dim3(1), dim3(kSchedThreads), smem, st, a);
  if constexpr (std::is_same_v<T, float>) {
    if (s.bm == 16)
      launch_simt<D, 16>(a, st);
    else
      launch_simt<D, 64>(a, st);
  } else {
    constexpr int dtype = std::is_same_v<T, __half> ? XN_F16 : XN_BF16;
    if (const int rc = s.bm == kTcRows ? launch_tc(a, D, dtype, st, op) : launch_dec(a, D, dtype, st, op)) return rc;
  }
  return check_launch(op);
}

int check_sizes(const char *op, int64_t n_tokens, int64_t requests, int64_t h, int64_t h_kv, int64_t d,
                int64_t max_new, int dtype) {
  if (!is_float_dtype(dtype)) return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (n_tokens < 0 || requests < 0 || max_new < 0) return fail(XN_E_INVALID, "%s: negative size", op);
  if (h <= 0 || h_kv <= 0 || h % h_kv != 0 || h / h_kv > 64 || h > 65536)
    return fail(XN_E_INVALID, "%s: h=%lld is not 1 to 64 times h_kv=%lld", op, (long long)h, (long long)h_kv);
  if (d != 32 && d != 64 && d != 128) return fail(XN_E_INVALID, "%s: head dim %lld not in {32, 64, 128}", op, (long long)d);
  if (requests > XN_PAGED_MAX_REQUESTS)
    return fail(XN_E_INVALID, "%s: %lld requests exceed %d", op, (long long)requests, XN_PAGED_MAX_REQUESTS);
  if (n_tokens > 0x7fffffffLL) return fail(XN_E_INVALID, "%s: too many tokens (%lld)", op, (long long)n_tokens);
  return XN_OK;
}

}  // namespace
}  // namespace paged
}  // namespace xn

extern "C" {

int xn_paged_attention_workspace(int64_t *bytes, int64_t n_tokens, int64_t requests, int64_t h, int64_t h_kv,
                                 int64_t d, int64_t max_new, int dtype) {
  using namespace xn;
  const char *op = "xn_paged_attention_workspace";
  if (bytes == nullptr) return fail(XN_E_INVALID, "%s: null output pointer", op);
  if (const int rc = paged::check_sizes(op, n_tokens, requests, h, h_kv, d, max_new, dtype)) return rc;
  const paged::Shape s = paged::shape_of(h / h_kv, max_new, d, dtype);
  *bytes = paged::layout_of(s, n_tokens, requests, h / h_kv, d).bytes;
  return ok();
}

int xn_paged_attention(void *out, const void *q, const void *k_pages, const void *v_pages, const int32_t *block_table,
                       const int64_t *q_start, const int64_t *kv_len, int64_t n_tokens, int64_t requests, int64_t h,
                       int64_t h_kv, int64_t d, int64_t n_pages, int64_t page_size, int64_t max_blocks,
                       int64_t q_tok_stride, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                       int64_t max_new, int64_t window, float scale, int dtype, void *workspace,
                       int64_t workspace_bytes, int *err_flag, void *stream) {
  using namespace xn;
  const char *op = "xn_paged_attention";
  if (const int rc = paged::check_sizes(op, n_tokens, requests, h, h_kv, d, max_new, dtype)) return rc;
  if (const int rc = check_pages(op, n_pages, page_size, h_kv, d, page_stride, head_stride, slot_stride, dtype)) return rc;
  if (max_blocks < 0 || max_blocks > ((int64_t{1} << 31) - 1024) / page_size)
    return fail(XN_E_INVALID, "%s: max_blocks=%lld out of range", op, (long long)max_blocks);
  if (window < 0) return fail(XN_E_INVALID, "%s: negative window", op);
  if (!(scale > 0.f) || scale > 0x1p127f)  // scale log2(e) is finite too
    return fail(XN_E_INVALID, "%s: scale must be positive and at most 2^127", op);
  if (q_tok_stride < h * d || q_tok_stride % (16 / dtype_bytes(dtype)) != 0)
    return fail(XN_E_INVALID, "%s: q rows need a stride of at least h * d elements, a multiple of 16 bytes (got %lld)", op,
                (long long)q_tok_stride);
  if (n_tokens == 0 || requests == 0) return ok();
  if (out == nullptr || q == nullptr || k_pages == nullptr || v_pages == nullptr || q_start == nullptr ||
      kv_len == nullptr || workspace == nullptr || (max_blocks > 0 && block_table == nullptr))
    return fail(XN_E_INVALID, "%s: null pointer", op);
  const void *ptrs[] = {out, q, k_pages, v_pages, workspace};
  for (const void *ptr : ptrs)
    if (!is_aligned16(ptr)) return fail(XN_E_INVALID, "%s: tensors must be 16-byte aligned", op);
  const int64_t group = h / h_kv;
  const paged::Shape s = paged::shape_of(group, max_new, d, dtype);
  const paged::Layout l = paged::layout_of(s, n_tokens, requests, group, d);
  if (workspace_bytes < l.bytes)
    return fail(XN_E_INVALID, "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)l.bytes);
  int shift = 0;
  while ((int64_t{1} << shift) < page_size) ++shift;
  char *ws = static_cast<char *>(workspace);
  paged::Args a{};
  a.out = out;
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.table = block_table;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.n_tokens = n_tokens;
  a.n_pages = n_pages;
  a.max_blocks = max_blocks;
  a.q_stride = q_tok_stride;
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.slot_stride = slot_stride;
  // Positions are below 2^31 (max_blocks above): a window as long as that hides nothing, and p - window cannot wrap.
  a.window = window < int64_t{1} << 31 ? window : 0;
  a.requests = static_cast<int32_t>(requests);
  a.h = static_cast<int32_t>(h);
  a.h_kv = static_cast<int32_t>(h_kv);
  a.group = static_cast<int32_t>(group);
  a.group_mul = static_cast<int32_t>((65535 + group) / group);
  a.page_shift = shift;
  a.tile_tokens = static_cast<int32_t>(s.bm / group);
  a.bn = s.bn;
  a.parts = s.parts;
  a.pair_cost = s.pair_cost;
  a.min_cost = s.min_cost;
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  a.wait_clocks = paged::wait_clocks();
  a.err_flag = err_flag;
  a.header = reinterpret_cast<paged::Header *>(ws);
  a.tiles = reinterpret_cast<paged::Tile *>(ws + l.tiles);
  a.starts = reinterpret_cast<paged::Start *>(ws + l.starts);
  a.cuts = reinterpret_cast<paged::Cut *>(ws + l.cuts);
  a.partial = reinterpret_cast<float *>(ws + l.partial);
  cudaStream_t st = as_stream(stream);
  XN_DISPATCH_FLOAT(dtype, {
    if (d == 32) return paged::launch_attn<T, 32>(a, s, st, op);
    if (d == 64) return paged::launch_attn<T, 64>(a, s, st, op);
    return paged::launch_attn<T, 128>(a, s, st, op);
  });
  return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
}

}  // extern "C"
