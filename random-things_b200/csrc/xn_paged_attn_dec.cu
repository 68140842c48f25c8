// xn_paged_attn_dec.cu - the paged attention's kernel for 16-bit single tokens
// and other small query tiles (up to 16 rows), for sm_100a.
//
// Bound by the cache's bytes: each key and value row is read once for all rows
// of its kv head. A producer warp keeps a ring of 64-key tiles in flight by
// TMA; two CTAs an SM hold about 190 KB of loads, several times what the
// memory's latency asks for (64 requests of 500 to 16000 keys, 2.3 GB: 351 us,
// the measured copy rate). Four warps take 16 keys of each tile: scores and
// weighted values as 16 x 8 x 16 products on the tensor cores (mma.sync: with
// 16 rows or fewer the 128-row tcgen05 shape would be mostly padding, and the
// products are a fraction of the load time), the softmax in registers. Each
// warp keeps its own running maximum, sum and output; they are joined at the
// end of a segment, so the warps never wait for one another in between.
//
// Masks as in the kernel for chunks: rows of V that no row sees are zeroed in
// shared memory, and where a row under some tokens' mask holds a non-finite
// value the warp adds its 16 keys on the CUDA cores, each row over its own.
#include "xn_paged_tma.cuh"

namespace xn {
namespace paged {
namespace {

constexpr int kBM = kDecRows, kBN = kDecKeys, kWarps = 4, kThreads = 32 * (kWarps + 1);

template <int D>
struct DecCfg : Swizzled<D, kBN> {
  static constexpr int kStages = D == 128 ? 3 : D == 64 ? 6 : 8;
  static constexpr int kJoin = kWarps * kBM * 36;  // floats of the join buffer: 32 columns, rows padded
  static constexpr size_t kSmem = 1024 + kStages * 2 * Swizzled<D, kBN>::kTile + kJoin * sizeof(float);
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Barrier of the four computing warps. Every one of them comes by: a wait that
// gave up leaves the work out, not the barriers.
__device__ __forceinline__ void join_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

struct Shared {
  uint64_t full[8], empty[8];
  int gave_up, last_piece;
  float max[kWarps][kBM], sum[kWarps][kBM];
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_attn_dec_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  griddep_wait();
  griddep_release();
  using Cfg = DecCfg<D>;
  constexpr int S = Cfg::kStages;
  extern __shared__ unsigned char dec_smem[];
  __shared__ Shared sh;
  const uint32_t base = (smem_u32(dec_smem) + 1023u) & ~1023u;
  unsigned char *base_p = dec_smem + (base - smem_u32(dec_smem));
  float *join = reinterpret_cast<float *>(base_p + S * 2 * Cfg::kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float *weights = join + warp * kBM * 36;  // [16][17] of a poisoned tile: in this warp's own part of the join buffer
  volatile int *gave_up = &sh.gave_up;
  const uint32_t full = smem_u32(sh.full), empty = smem_u32(sh.empty);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kWarps);
    }
    sh.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  __syncthreads();
  Tile t;
  Walk w(a, blockIdx.x);
  uint32_t n = 0;  // tiles so far
  if (warp == kWarps) {
    const TileLoad<D, kBN> ld(a);
    bool ok = true;
    for (; ok && w.get(a, t); w.next(a)) {
      const int64_t hi = t.pos0 + t.ntok, lo = key_lo(t, a.window);
      const int64_t u0 = first_unit(t, a.window, kBN) + w.k;
      int page = ld.page(a, t, u0 * kBN, lo, hi);
      for (int64_t u = u0; u < u0 + w.take; ++u, ++n) {
        const uint32_t st = n % S, round = n / S;
        ok = round == 0 || wait(empty + 8 * st, (round - 1) & 1, gave_up, a.wait_clocks);
        if (!ok) break;
        if (lane == 0) mbar_expect(full + 8 * st, 2 * Cfg::kTile);
        __syncwarp();
        const uint32_t at = base + st * 2 * Cfg::kTile;
        ld.load(a, &kmap, at, full + 8 * st, u * kBN, w.head, page);
        ld.load(a, &vmap, at + Cfg::kTile, full + 8 * st, u * kBN, w.head, page);
        if (u + 1 < u0 + w.take) page = ld.page(a, t, (u + 1) * kBN, lo, hi);
      }
    }
    // Copies in flight end before the block does.
    for (uint32_t i = n > S ? n - S : 0; i < n; ++i) drain(full + 8 * (i % S), (i / S) & 1);
    return;
  }
  const int g = lane >> 2, t4 = lane & 3;
  const float c = a.scale_log2;
  // This lane's row of an 8 x 8 matrix in the loads of K (not transposed) and V (transposed).
  const int k_row = warp * 16 + (lane & 7) + (lane >> 4) * 8, k_chunk = lane >> 3 & 1;
  const int v_row = warp * 16 + (lane & 15), v_chunk = lane >> 4;
  bool ok = a.wait_clocks > 0;
  if (!ok) *gave_up = 1;
  for (; w.get(a, t); w.next(a)) {
    const int rows = t.ntok * a.group;
    uint32_t q[D / 16][4];
    int64_t pos[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + r * 8, tk = token_of(a, row);
      pos[r] = t.pos0 + tk;
      const T *src = static_cast<const T *>(a.q) + (t.tok0 + tk) * a.q_stride + (w.head * a.group + row - tk * a.group) * D + t4 * 2;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][r] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(src + k * 16)) : 0u;
        q[k][r + 2] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(src + k * 16 + 8)) : 0u;
      }
    }
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    const int64_t hi = t.pos0 + t.ntok, lo = key_lo(t, a.window);
    const int64_t u0 = first_unit(t, a.window, kBN) + w.k;
    for (int64_t u = u0; u < u0 + w.take; ++u, ++n) {
      const uint32_t st = n % S;
      ok = ok && wait(full + 8 * st, (n / S) & 1, gave_up, a.wait_clocks);
      if (!ok) continue;
      const uint32_t ks = base + st * 2 * Cfg::kTile, vs = ks + Cfg::kTile;
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];
        ldsm4(ks + Cfg::chunk_at(k_row, 2 * k + k_chunk), b);
        mma16816<T>(s[0], q[k], b[0], b[1]);
        mma16816<T>(s[1], q[k], b[2], b[3]);
      }
      const int64_t key0 = u * kBN + warp * 16;  // this warp's 16 keys
      const bool masked = key0 + 15 > t.pos0 || (a.window > 0 && key0 <= hi - 1 - a.window);
      uint32_t unseen = 0;  // bit i * 4 + j: key of s[i][j] is not seen by its row
      bool poisoned = false;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t key = key0 + (i >> 2) * 8 + t4 * 2 + (i & 1), p = pos[i >> 1 & 1];
          if (key > p || (a.window > 0 && key <= p - a.window)) {
            s[i >> 2][i & 3] = -INFINITY;
            unseen |= 1u << i;
          }
        }
        // V: two lanes a row.
        const int64_t key = key0 + (lane >> 1);
        bool bad = false;
        unsigned char *vp = base_p + (vs - base);
        for (int j = lane & 1; j < D / 8; j += 2) {
          uint4 *x = reinterpret_cast<uint4 *>(vp + Cfg::chunk_at(warp * 16 + (lane >> 1), j));
          if (key >= hi || key < lo)
            *x = make_uint4(0u, 0u, 0u, 0u);
          else
            bad |= non_finite2<T>(x->x) | non_finite2<T>(x->y) | non_finite2<T>(x->z) | non_finite2<T>(x->w);
        }
        proxy_fence();  // before TMA writes the stage again
        __syncwarp();   // other lanes read the zeroed rows (a vote orders no memory)
        poisoned = __any_sync(0xffffffffu, bad);
      }
      float top[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      // Maxima move only when one grew by more than 2^8 (see the kernel for chunks).
      if (__any_sync(0xffffffffu, (top[0] - m[0]) * c > 8.f || (top[1] - m[1]) * c > 8.f)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float to = fmaxf(m[r], top[r]), f = m[r] == to ? 1.f : ex2_approx_ftz((m[r] - to) * c);
          m[r] = to;
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * r] *= f;
            o[i][2 * r + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float low = m[r] == -INFINITY ? 0.f : m[r];  // before the scale, as in the kernel for chunks
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 2 * r; j < 2 * r + 2; ++j) {
            s[i][j] = ex2_approx_ftz((s[i][j] - low) * c);
            l[r] += s[i][j];
          }
      }
      if (!poisoned) {
        const uint32_t p[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                               pack2<T>(s[1][2], s[1][3])};
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t b[4];
          ldsm4_t(vs + Cfg::chunk_at(v_row, 2 * k + v_chunk), b);
          mma16816<T>(o[2 * k], p, b[0], b[1]);
          mma16816<T>(o[2 * k + 1], p, b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)  // -1: no part in the row
          weights[(g + (i >> 1 & 1) * 8) * 17 + (i >> 2) * 8 + t4 * 2 + (i & 1)] = unseen >> i & 1 ? -1.f : s[i >> 2][i & 3];
        __syncwarp();
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const float p0 = weights[g * 17 + k], p1 = weights[(g + 8) * 17 + k];
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t *>(base_p + (vs - base) + Cfg::chunk_at(warp * 16 + k, i) + t4 * 4));
            o[i][0] = p0 < 0.f ? o[i][0] : __fmaf_rn(p0, v.x, o[i][0]);
            o[i][1] = p0 < 0.f ? o[i][1] : __fmaf_rn(p0, v.y, o[i][1]);
            o[i][2] = p1 < 0.f ? o[i][2] : __fmaf_rn(p1, v.x, o[i][2]);
            o[i][3] = p1 < 0.f ? o[i][3] : __fmaf_rn(p1, v.y, o[i][3]);
          }
        }
      }
      warp_arrive(empty + 8 * st);
    }
    // The warps' parts come together, 32 columns at a time.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t4 == 0) {
        sh.max[warp][g + 8 * r] = m[r];
        sh.sum[warp][g + 8 * r] = l[r];
      }
    }
    join_sync();
    auto factor = [&](int wp, int row, float mx) {
      const float mw = sh.max[wp][row];
      return mw == -INFINITY ? 0.f : ex2_approx_ftz((mw - mx) * c);
    };
    auto top_of = [&](int row) { return fmaxf(fmaxf(sh.max[0][row], sh.max[1][row]), fmaxf(sh.max[2][row], sh.max[3][row])); };
    const float f0 = factor(warp, g, top_of(g)), f1 = factor(warp, g + 8, top_of(g + 8));
    const int row = tid >> 3, col = (tid & 7) * 4;  // what this thread adds up
    const float mx = top_of(row);
    float sum = 0.f;
#pragma unroll
    for (int wp = 0; wp < kWarps; ++wp) sum = __fmaf_rn(sh.sum[wp][row], factor(wp, row, mx), sum);
    const bool whole = w.whole(t);
    const int tk = token_of(a, row);
    float *part_o = partial_of(a, blockIdx.x, w.first ? 0 : 1, kBM, D);
    T *dst = static_cast<T *>(a.out) + (static_cast<int64_t>(t.tok0 + tk) * a.h + w.head * a.group + row - tk * a.group) * D;
    const bool none = t.pos0 + tk < 0, dead = *gave_up != 0;
    const float inv = __fdiv_rn(1.f, sum), nan = __int_as_float(0x7fc00000);
    if (dead && tid == 0 && a.err_flag != nullptr) atomicOr(a.err_flag, XN_DEVERR_WAIT);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      float *buf = join;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<float2 *>(buf + (warp * kBM + g) * 36 + j * 8 + t4 * 2) = make_float2(o[i * 4 + j][0] * f0, o[i * 4 + j][1] * f0);
        *reinterpret_cast<float2 *>(buf + (warp * kBM + g + 8) * 36 + j * 8 + t4 * 2) =
            make_float2(o[i * 4 + j][2] * f1, o[i * 4 + j][3] * f1);
      }
      join_sync();
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int wp = 0; wp < kWarps; ++wp) {
        const float4 y = *reinterpret_cast<const float4 *>(buf + (wp * kBM + row) * 36 + col);
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      }
      if (row < rows) {
        if (whole) {
          const float k = dead ? nan : inv;
          *reinterpret_cast<uint2 *>(dst + i * 32 + col) =
              none ? make_uint2(0u, 0u) : make_uint2(pack2<T>(x.x * k, x.y * k), pack2<T>(x.z * k, x.w * k));
        } else {
          *reinterpret_cast<float4 *>(part_o + row * D + i * 32 + col) = x;
        }
      }
      join_sync();  // the buffer, and after the last turn sh.max and sh.sum, are free
    }
    if (!whole) {
      if (row < rows && col == 0) {
        part_o[kBM * D + row] = mx;
        part_o[kBM * D + kBM + row] = dead ? nan : sum;
      }
      end_piece<T, D>(a, w, t, blockIdx.x, kBM, tid, 32 * kWarps, &sh.last_piece, join_sync);
    }
  }
}

template <typename T, int D>
int launch(const Args &a, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t st, const char *op) {
  constexpr int smem = static_cast<int>(DecCfg<D>::kSmem);
  if (cudaFuncSetAttribute(paged_attn_dec_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch(op);
  launch_k(paged_attn_dec_kernel<T, D>, dim3(a.parts), dim3(kThreads), smem, st, a, kmap, vmap);
  return XN_OK;
}

}  // namespace

int launch_dec(const Args &a, int d, int dtype, cudaStream_t st, const char *op) {
  CUtensorMap kmap, vmap;
  const bool bf16 = dtype == XN_BF16;
  if (!make_map(&kmap, a.k, a, d, kBN, bf16) || !make_map(&vmap, a.v, a, d, kBN, bf16))
    return fail(XN_E_CUDA, "%s: the driver refused a tensor map of the pools", op);
  if (bf16) {
    if (d == 32) return launch<__nv_bfloat16, 32>(a, kmap, vmap, st, op);
    if (d == 64) return launch<__nv_bfloat16, 64>(a, kmap, vmap, st, op);
    return launch<__nv_bfloat16, 128>(a, kmap, vmap, st, op);
  }
  if (d == 32) return launch<__half, 32>(a, kmap, vmap, st, op);
  if (d == 64) return launch<__half, 64>(a, kmap, vmap, st, op);
  return launch<__half, 128>(a, kmap, vmap, st, op);
}

}  // namespace paged
}  // namespace xn
