// xn_paged_attn_tc.cu - the paged attention's kernel for chunks of 16-bit
// tokens on the 5th-generation tensor cores (sm_100a).
//
// A CTA takes 256 rows (token, query head of the group) of one kv head: two
// halves of 128, each with its own softmax warpgroup, product warp, scores S
// (two buffers) and output O in tensor memory. Per key tile of 64 keys:
//   S = Q K^T      tcgen05.mma, both operands in shared memory
//   P = exp2((S - m) c), row maxima and sums   one thread a row: no shuffles
//   O = O + P V    tcgen05.mma, P in tensor memory (over S), V in shared memory
// The scores of the next two tiles are issued ahead, so that a half's softmax
// need not wait for its own products. (With one buffer of 128 keys each half
// went softmax, products, softmax, ...: an 8192-token prompt of 32 / 8 heads of
// 128 took 632 us against 547. Now it takes 522 us alone and up to 581 in calls
// back to back, as the power limit lets the clock go: 0.65 to 0.58 of the
// measured bf16 rate. With keys by 64 the score products read shared memory as
// fast as it goes, which bounds the kernel together with the exponentials.) One more warp loads: K and V tiles come by TMA, a box
// per page, swizzled as the MMA reads them, through two rings of stages.
//
// O stays in tensor memory for all key tiles. When a row's maximum grows by
// more than 2^8 (in the exponent's units: 8), its warp rescales O; below that
// the old maximum stays in use, which changes nothing but the common factor
// of numerator and denominator.
//
// Masks. Scores of unseen keys become -inf, weight 0. A weight of 0 does not
// silence an infinite or NaN value in the product, so in a tile with a mask
// the V rows that no row sees (beyond the last token, before the window, stale
// page rows) are zeroed in shared memory, and when a row that some tokens see
// and others do not holds a non-finite value, the half adds the tile's product
// on the CUDA cores, each token over its own keys (poisoned tile).
//
// Every wait has a time limit; see wait(). When one gives up, the rows that are
// left become NaN, and each role still waits for what it has in flight.
#include "xn_paged_tma.cuh"

namespace xn {
namespace paged {
namespace {

constexpr int kBM = kTcRows, kBN = kTcKeys, kThreads = 384;
constexpr int kLoadWarp = 8, kMmaWarp = 9;  // and 10: one for each half
constexpr int kPolyOf8 = 2;  // of 8 pairs of weights, those that the FMA pipe computes

template <int D>
struct TcCfg {
  using Q = Swizzled<D, 128>;  // a half's query rows
  using KV = Swizzled<D, kBN>;  // a K or V tile
  static constexpr int kStages = D == 128 ? 5 : 8;  // of each ring
  static constexpr size_t kSmem = 1024 + 2 * Q::kTile + 2 * kStages * KV::kTile;
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 columns of this warp's 32 lanes (one lane a row) from / to tensor memory.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float *r) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
// Loads are asynchronous: the values pass through empty statements behind the
// wait, so that no use of them is scheduled before it.
template <int N>
__device__ __forceinline__ void tc_wait_ld(uint32_t *u) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i += 4) asm volatile("" : "+r"(u[i]), "+r"(u[i + 1]), "+r"(u[i + 2]), "+r"(u[i + 3]));
}
__device__ __forceinline__ void tc_wait_ld(float *r) { tc_wait_ld<32>(reinterpret_cast<uint32_t *>(r)); }
__device__ __forceinline__ void tc_ld4(uint32_t addr, uint32_t (&u)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
               : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t *u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// D (tensor memory) = A B (+ D): A and B in shared memory, or A in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// Shared-memory operand descriptor. Low word: address and leading byte offset
// in 16-byte units (so a step of n bytes adds n / 16; addresses stay below
// 2^18); high word: stride byte offset, version 1, swizzle of 128 (code 2) or
// 64 bytes (code 4).
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return addr >> 4 | (lbo >> 4) << 16; }
constexpr uint32_t desc_hi(uint32_t sbo, uint32_t swizzle) { return sbo >> 4 | 1u << 14 | swizzle << 29; }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x on the FMA pipe, for a quarter of the weights: the exponential unit's 16
// results a clock an SM take as long as the products. An 8192-token prompt of 32
// / 8 heads without and with it, alone: of 128 553 and 514 us (f16 555 and 521),
// of 64 493 and 469 (f16 496 and 469), of 32 471 and 457 (f16 471 and 451);
// ragged chunks of 12 requests, 24 / 8 heads: of 128 242 and 242 us (f16 244 and
// 242), of 64 203 and 197 (f16 205 and 197), of 32 191 and 186 (f16 191 and 184).
// x = n + f, |f| <= 1/2: adding 1.5 2^23 + 127 leaves n + 127 in the low bits,
// which shifted into place are 2^n; 2^f is a minimax polynomial (fit_exp2.py,
// relative error 2.7e-6, against 2^-9 or 2^-12 for the rounding that follows).
// x <= -127 gives 0, NaN stays NaN; x is at most 8 here.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  const float2 t = __fadd2_rn(x, splat2(12583039.f));
  const float2 f = __ffma2_rn(__fadd2_rn(t, splat2(-12583039.f)), splat2(-1.f), x);
  float2 p = __ffma2_rn(f, splat2(0x1.3997d6p-7f), splat2(0x1.ca1444p-5f));
  p = __ffma2_rn(p, f, splat2(0x1.ec06dap-3f));
  p = __ffma2_rn(p, f, splat2(0x1.62e0dcp-1f));
  p = __ffma2_rn(p, f, splat2(0x1.ffffe8p-1f));
  return __fmul2_rn(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}

// Of a segment's key tiles, the first of them number u0, those from j_diag on
// hold keys behind the first token, those up to j_win keys before the last
// token's window: some row does not see them.
__device__ __forceinline__ void masked_tiles(const Args &a, const Tile &t, int64_t u0, int &j_diag, int &j_win) {
  const int64_t last = t.pos0 + t.ntok - 1;
  j_diag = static_cast<int>((t.pos0 < 0 ? 0 : (t.pos0 + 1) / kBN) - u0);
  j_win = a.window > 0 && last >= a.window ? static_cast<int>((last - a.window) / kBN - u0) : -1;
}

struct Shared {
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], v_seen[2], drain[2];  // [half][S buffer]
  uint32_t tmem;
  int gave_up, skip[2][2];  // skip: a poisoned tile's product is done already
  int poison[2][3];  // non-finite values under a mask, by half; three masked tiles in turn
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_tc_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  griddep_wait();
  griddep_release();
  using Cfg = TcCfg<D>;
  using Q = typename Cfg::Q;
  using KV = typename Cfg::KV;
  constexpr int S = Cfg::kStages;
  extern __shared__ unsigned char tc_smem[];
  __shared__ Shared sh;
  const uint32_t base = (smem_u32(tc_smem) + 1023u) & ~1023u;
  unsigned char *base_p = tc_smem + (base - smem_u32(tc_smem));
  const uint32_t k_base = base + 2 * Q::kTile, v_base = k_base + S * KV::kTile;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int *gave_up = &sh.gave_up;

  const uint32_t k_full = smem_u32(sh.k_full), k_empty = smem_u32(sh.k_empty), v_full = smem_u32(sh.v_full);
  const uint32_t v_empty = smem_u32(sh.v_empty), q_full = smem_u32(sh.q_full), s_full = smem_u32(sh.s_full);
  const uint32_t p_full = smem_u32(sh.p_full), pv_done = smem_u32(sh.pv_done), v_seen = smem_u32(sh.v_seen);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 2);
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 128);
      mbar_init(v_seen + 8 * i, 128);
      mbar_init(smem_u32(&sh.drain[i]), 1);
      sh.skip[i][0] = sh.skip[i][1] = sh.poison[i][0] = sh.poison[i][1] = sh.poison[i][2] = 0;
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 128);
      mbar_init(pv_done + 8 * i, 1);
    }
    sh.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // Tensor memory: two S buffers a half at columns 0 .. 255 (P over them), O behind.
  const uint32_t o_col = 256;

  Tile t;
  Walk w(a, blockIdx.x);
  if (warp == kLoadWarp) {
    const TileLoad<D, kBN> ld(a);
    uint32_t nk = 0, nv = 0;  // tiles loaded
    bool ok = true;
    auto load = [&](const CUtensorMap *map, uint32_t ring, uint32_t full, uint32_t empty, uint32_t &n, int64_t key0, int page) {
      const uint32_t st = n % S, round = n / S;
      ok = ok && (round == 0 || wait(empty + 8 * st, (round - 1) & 1, gave_up, a.wait_clocks));
      if (!ok) return;
      if (lane == 0) mbar_expect(full + 8 * st, KV::kTile);
      __syncwarp();
      ld.load(a, map, ring + st * KV::kTile, full + 8 * st, key0, w.head, page);
      ++n;
    };
    for (; ok && w.get(a, t); w.next(a)) {
      const int64_t hi = t.pos0 + t.ntok, lo = key_lo(t, a.window);
      const int64_t u0 = first_unit(t, a.window, kBN) + w.k;
      // In the order of use: K runs one tile ahead of V.
      int v_page = 0;
      for (int j = 0; ok && j < w.take; ++j) {
        const int64_t key0 = (u0 + j) * kBN;
        const int page = ld.page(a, t, key0, lo, hi);
        load(&kmap, k_base, k_full, k_empty, nk, key0, page);
        if (j > 0) load(&vmap, v_base, v_full, v_empty, nv, key0 - kBN, v_page);
        v_page = page;
      }
      load(&vmap, v_base, v_full, v_empty, nv, (u0 + w.take - 1) * kBN, v_page);
    }
    // Copies in flight end before the block does.
    for (uint32_t i = nk > S ? nk - S : 0; i < nk; ++i) drain(k_full + 8 * (i % S), (i / S) & 1);
    for (uint32_t i = nv > S ? nv - S : 0; i < nv; ++i) drain(v_full + 8 * (i % S), (i / S) & 1);
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // A warp for each half, so that what one waits for does not hold up the other. The whole warp walks along, and
    // what the products need is equal in all lanes by construction (loop counters, broadcast values): their operands
    // then sit in uniform registers. One elected lane issues. (With the walk in one lane's branch, each product took
    // 75 clocks to issue instead of 64 to run.)
    constexpr uint32_t fmt = std::is_same_v<T, __half> ? 0u : 1u;
    constexpr uint32_t idesc = 1u << 4 | fmt << 7 | fmt << 10 | (128u >> 4) << 24;
    constexpr uint32_t idesc_s = idesc | (kBN >> 3) << 17;
    constexpr uint32_t idesc_o = idesc | 1u << 16 | (D >> 3) << 17;  // V: keys are the slow dimension
    constexpr uint32_t group8 = 8 * KV::kRowBytes, hi = desc_hi(group8, D >= 64 ? 2 : 4);
    const int h = __shfl_sync(0xffffffffu, warp - kMmaWarp, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), s_col = tm + h * 2 * kBN, o_at = tm + o_col + h * D;
    const uint32_t q_desc = desc_lo(base + h * Q::kTile, 16);
    struct Ring {
      uint32_t stage = 0, phase = 0;
      __device__ __forceinline__ void advance() {
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
    } rk, rv;
    uint32_t ns = 0, np = 0, nq = 0;  // scores issued, weights used, items
    bool ok = true;
    auto scores = [&] {  // the next S = Q K^T
      if (elect_one()) {
        const uint32_t k = desc_lo(k_base + rk.stage * KV::kTile, 16), to = s_col + (ns & 1) * kBN;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(to, q_desc + ((kk / 4 * Q::kSub + kk % 4 * 32) >> 4), k + ((kk / 4 * KV::kSub + kk % 4 * 32) >> 4), hi, idesc_s,
                 kk > 0);
        tc_commit(s_full + 16 * h + 8 * (ns & 1));
        tc_commit(k_empty + 8 * rk.stage);
      }
      __syncwarp();
      ++ns;
      rk.advance();
    };
    auto output = [&](bool skip, bool add) {  // O (+)= the next P V
      if (elect_one()) {
        const uint32_t v = desc_lo(v_base + rv.stage * KV::kTile, KV::kSub), p = s_col + (np & 1) * kBN;
        if (!skip) {
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)
            mma_ts(o_at, p + kk * 8, v + (kk * 2 * group8 >> 4), hi, idesc_o, add || kk > 0);
        }
        tc_commit(pv_done + 16 * h + 8 * (np & 1));
        tc_commit(v_empty + 8 * rv.stage);
      }
      __syncwarp();
      ++np;
      rv.advance();
    };
    for (; ok && w.get(a, t); w.next(a)) {
      const int take = __shfl_sync(0xffffffffu, w.take, 0);
      if (__shfl_sync(0xffffffffu, t.ntok * a.group <= h * 128 ? 1 : 0, 0)) {
        // Nothing to do for this half, but the stages wait for its word too.
        for (int i = 0; ok && i < take; ++i) {
          ok = wait(k_full + 8 * rk.stage, rk.phase, gave_up, a.wait_clocks);
          if (ok && lane == 0) mbar_arrive(k_empty + 8 * rk.stage);
          ok = ok && wait(v_full + 8 * rv.stage, rv.phase, gave_up, a.wait_clocks);
          if (ok && lane == 0) mbar_arrive(v_empty + 8 * rv.stage);
          rk.advance();
          rv.advance();
        }
        continue;
      }
      // Key tiles with a mask: only there a poisoned tile can be (see the softmax).
      int j_diag, j_win;
      masked_tiles(a, t, first_unit(t, a.window, kBN) + w.k, j_diag, j_win);
      j_diag = __shfl_sync(0xffffffffu, j_diag, 0);
      j_win = __shfl_sync(0xffffffffu, j_win, 0);
      ok = wait(k_full + 8 * rk.stage, rk.phase, gave_up, a.wait_clocks) && wait(q_full + 8 * h, nq++ & 1, gave_up, a.wait_clocks);
      if (!ok) break;
      tc_fence_after();
      scores();
      if (take > 1) {
        ok = wait(k_full + 8 * rk.stage, rk.phase, gave_up, a.wait_clocks);
        if (!ok) break;
        scores();
      }
      for (int j = 0; j < take; ++j) {
        const bool more = j + 2 < take;
        ok = wait(v_full + 8 * rv.stage, rv.phase, gave_up, a.wait_clocks);
        if (ok && more) ok = wait(k_full + 8 * rk.stage, rk.phase, gave_up, a.wait_clocks);
        if (ok) ok = wait(p_full + 16 * h + 8 * (np & 1), np >> 1 & 1, gave_up, a.wait_clocks);
        if (!ok) break;
        tc_fence_after();
        int skip = 0;
        if (j >= j_diag || j <= j_win) skip = __shfl_sync(0xffffffffu, *static_cast<volatile int *>(&sh.skip[h][np & 1]), 0);
        output(skip != 0, j > 0);
        if (more) scores();
      }
    }
    // Products in flight end before tensor memory is freed.
    if (elect_one()) tc_commit(smem_u32(&sh.drain[h]));
    __syncwarp();
    drain(smem_u32(&sh.drain[h]), 0);
  } else if (warp < kLoadWarp) {
    const int h = warp >> 2, wt = tid & 127, row = h * 128 + wt;  // half, thread of the warpgroup = row of the half
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + h * 2 * kBN, o_addr = tmem + lanes + o_col + h * D;
    const float c = a.scale_log2;
    uint32_t ns = 0, nm = 0, tiles = 0;  // S tiles, masked tiles of this half; tiles of the CTA
    bool ok = a.wait_clocks > 0, q_in = false;
    if (!ok) *gave_up = 1;
    // Waits for the products of tile ns - 1. (Two barriers in turn: the scores of tile ns - 1 came behind the products
    // of ns - 3, so that the phase waited for is the only one that can be open.)
    auto pv_wait = [&] { return wait(pv_done + 16 * h + 8 * ((ns - 1) & 1), (ns - 1) >> 1 & 1, gave_up, a.wait_clocks); };
    // This half's query rows of an item into shared memory, asynchronously.
    auto load_q = [&](const Tile &item, int head) {
      const int n_rows = item.ntok * a.group;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const int r = (i * 128 + wt) / (D / 8), j = wt % (D / 8), qr = h * 128 + r, tk = token_of(a, qr);
        const T *src = static_cast<const T *>(a.q) + (item.tok0 + tk) * a.q_stride + (head * a.group + qr - tk * a.group) * D + j * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + h * Q::kTile + Q::chunk_at(r, j)),
                     "l"(qr < n_rows ? src : static_cast<const T *>(a.q)), "r"(qr < n_rows ? 16 : 0)
                     : "memory");
      }
    };
    auto q_loaded = [&] {
      asm volatile("cp.async.wait_all;" ::: "memory");
      proxy_fence();
      mbar_arrive(q_full + 8 * h);
    };
    for (; w.get(a, t); w.next(a)) {
      const int rows = t.ntok * a.group;
      if (rows <= h * 128) {
        tiles += w.take;
        continue;
      }
      float m = -INFINITY, l = 0.f;
      if (ok && !q_in) {
        load_q(t, w.head);
        q_loaded();
      }
      q_in = false;
      // Keys are counted from the segment's first one.
      int j_diag, j_win, see_lo, see_hi, v_lo, v_hi;
      {
        const int64_t u0 = first_unit(t, a.window, kBN) + w.k, key0 = u0 * kBN, pos = t.pos0 + token_of(a, row);
        masked_tiles(a, t, u0, j_diag, j_win);
        const int64_t row_lo = a.window > 0 && pos - a.window + 1 > key0 ? pos - a.window + 1 - key0 : 0;
        see_lo = static_cast<int>(row_lo < (1 << 30) ? row_lo : 1 << 30);
        see_hi = static_cast<int>(pos + 1 - key0);
        const int64_t lo = key_lo(t, a.window) - key0;
        v_lo = static_cast<int>(lo < 0 ? 0 : lo);
        v_hi = static_cast<int>(t.pos0 + t.ntok - key0);
      }
      // One key tile; false when a wait gave up.
      auto tile = [&](int j, auto with_mask) -> bool {
        constexpr bool kMasked = decltype(with_mask)::value;
        const uint32_t buf = ns & 1, s_at = s_addr + buf * kBN;
        if (!wait(s_full + 16 * h + 8 * buf, ns >> 1 & 1, gave_up, a.wait_clocks)) return false;
        tc_fence_after();
        if (j == w.take - 1) {  // the scores are done with Q: the next item's rows may come
          Walk next = w;
          next.next(a);
          Tile item;
          q_in = next.get(a, item) && item.ntok * a.group > h * 128;
          if (q_in) load_q(item, next.head);
        }
        float s[kBN];
        tc_ld32(s_at, s);
        tc_ld32(s_at + 32, s + 32);
        tc_wait_ld<kBN>(reinterpret_cast<uint32_t *>(s));
        if constexpr (kMasked) {
          const int lo = see_lo - j * kBN, hi = see_hi - j * kBN;
#pragma unroll
          for (int i = 0; i < kBN; ++i) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i + 8 <= kBN; i += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
        }
        const float top = max3(max3(mx[0], s[kBN - 4], s[kBN - 3]), max3(mx[1], s[kBN - 2], s[kBN - 1]), fmaxf(mx[2], mx[3]));
        // A larger maximum by more than 2^8: this warp's rows move to it.
        if (__any_sync(0xffffffffu, (top - m) * c > 8.f)) {
          const float to = fmaxf(m, top), f = m == to ? 1.f : ex2_approx_ftz((m - to) * c);
          m = to;
          l *= f;
          if (j > 0) {
            if (!pv_wait()) return false;  // O is at rest
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              float o[32];
              tc_ld32(o_addr + i, o);
              tc_wait_ld(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= f;
              tc_st32(o_addr + i, reinterpret_cast<uint32_t *>(o));
            }
          }
        }
        // The maximum comes off before the scale: a product m c, rounded, would leave the largest key a weight of 2^d, d
        // up to half its unit. (s c - m c in one FMA: no faster, an 8192-token prompt 580 us against 578.)
        const float low = m == -INFINITY ? 0.f : -m;
        float2 sum[2] = {splat2(0.f), splat2(0.f)};
        uint32_t p[kBN / 2];  // in place of the scores
#pragma unroll
        for (int k = 0; k < kBN / 2; ++k) {
          float2 e = __fmul2_rn(__fadd2_rn(make_float2(s[2 * k], s[2 * k + 1]), splat2(low)), splat2(c));
          if (k % 8 >= 8 - kPolyOf8)
            e = exp2_poly(e);
          else
            e = make_float2(ex2_approx_ftz(e.x), ex2_approx_ftz(e.y));
          sum[k & 1] = __fadd2_rn(sum[k & 1], e);
          p[k] = pack2<T>(e.x, e.y);
        }
        tc_st32(s_at, p);
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        if constexpr (kMasked) {
          const uint32_t nv = tiles + j;
          if (!wait(v_full + 8 * (nv % S), (nv / S) & 1, gave_up, a.wait_clocks)) return false;
          unsigned char *vs = base_p + (v_base - base) + (nv % S) * KV::kTile;
          const int vr = wt >> 1, key = j * kBN + vr;  // two threads a V row
          bool bad = false;
#pragma unroll
          for (int q = 0; q < D / 16; ++q) {
            uint4 *x = reinterpret_cast<uint4 *>(vs + KV::chunk_at(vr, 2 * q + (wt & 1)));
            if (key >= v_hi || key < v_lo)
              *x = make_uint4(0u, 0u, 0u, 0u);
            else
              bad |= non_finite2<T>(x->x) | non_finite2<T>(x->y) | non_finite2<T>(x->z) | non_finite2<T>(x->w);
          }
          proxy_fence();
          // The half's 128 threads agree. Slots are used in turn: the next one is
          // cleared when everyone has read its last use (before the wait just passed).
          volatile int *poison = sh.poison[h];
          if (bad) poison[nm % 3] = 1;
          if (wt == 0) poison[(nm + 1) % 3] = 0;
          mbar_arrive(v_seen + 8 * h);
          if (!wait(v_seen + 8 * h, nm & 1, gave_up, a.wait_clocks)) return false;
          const int poisoned = poison[nm++ % 3];
          if (wt == 0) *static_cast<volatile int *>(&sh.skip[h][buf]) = poisoned;
          if (poisoned) {
            const int lo = see_lo - j * kBN, hi = see_hi - j * kBN;
            tc_wait_st();
            if (j > 0 && !pv_wait()) return false;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              float o[32];
              if (j > 0) {
                tc_ld32(o_addr + i, o);
                tc_wait_ld(o);
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = 0.f;
              }
#pragma unroll 1
              for (int kb = 0; kb < kBN; kb += 8) {
                uint32_t pw[4];
                __syncwarp();
                tc_ld4(s_at + kb / 2, pw);
                tc_wait_ld<4>(pw);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  if (kb + k < lo || kb + k >= hi) continue;
                  const float2 p2 = unpack2<T>(pw[k / 2]);
                  const float pk = k & 1 ? p2.y : p2.x;
#pragma unroll
                  for (int q = 0; q < 4; ++q) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(vs + KV::chunk_at(kb + k, i / 8 + q));
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const float2 v2 = unpack2<T>(xw[e]);
                      o[q * 8 + e * 2] = __fmaf_rn(pk, v2.x, o[q * 8 + e * 2]);
                      o[q * 8 + e * 2 + 1] = __fmaf_rn(pk, v2.y, o[q * 8 + e * 2 + 1]);
                    }
                  }
                }
              }
              __syncwarp();
              tc_st32(o_addr + i, reinterpret_cast<uint32_t *>(o));
            }
          }
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(p_full + 16 * h + 8 * buf);
        ++ns;
        return true;
      };
      // Tiles with a mask stand at either end; those between them run in a loop without that code.
      for (int j = 0; ok && j < w.take;) {
        for (; ok && j < w.take && (j <= j_win || j >= j_diag); ++j) ok = tile(j, std::true_type{});
        for (; ok && j < w.take && j > j_win && j < j_diag; ++j) ok = tile(j, std::false_type{});
      }
      tiles += w.take;
      if (ok && q_in) q_loaded();
      ok = ok && pv_wait();
      if (!ok && wt == 0 && a.err_flag != nullptr) atomicOr(a.err_flag, XN_DEVERR_WAIT);
      tc_fence_after();
      const bool whole = w.whole(t), none = t.pos0 + token_of(a, row) < 0;
      // Rows out: a thread writes its row. After a wait that gave up: NaN.
      const float nan = __int_as_float(0x7fc00000);
      float *part_o = partial_of(a, blockIdx.x, w.first ? 0 : 1, kBM, D);
      const int tk = token_of(a, row);
      T *dst = static_cast<T *>(a.out) + (static_cast<int64_t>(t.tok0 + tk) * a.h + w.head * a.group + row - tk * a.group) * D;
      const float inv = __fdiv_rn(1.f, l);
#pragma unroll 1
      for (int i = 0; i < D; i += 32) {
        float o[32];
        __syncwarp();
        if (ok) {
          tc_ld32(o_addr + i, o);
          tc_wait_ld(o);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = nan;
        }
        if (row >= rows) continue;
        if (whole) {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = none ? 0.f : o[k] * inv;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            st_vec(dst + i + k, make_uint4(pack2<T>(o[k], o[k + 1]), pack2<T>(o[k + 2], o[k + 3]), pack2<T>(o[k + 4], o[k + 5]),
                                           pack2<T>(o[k + 6], o[k + 7])));
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4 *>(part_o + row * D + i + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (!whole) {
        if (row < rows) {
          part_o[kBM * D + row] = ok ? m : nan;
          part_o[kBM * D + kBM + row] = ok ? l : nan;
        }
      }
      tc_fence_before();  // O is read before the next item's products write it
    }
    // After a wait that gave up, query rows and stores to tensor memory may be under way.
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    tc_wait_st();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Adds the pieces of the cut pairs: block (c, y) those of the pair that part
// c + 1 is the first to begin inside, 32 rows. (Done at the end of the last
// piece instead, as for single tokens, it saved this launch, 16 us, and cost the
// kernel above 33 to 49 us: its registers are all taken.)
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const Args a) {
  griddep_wait();
  griddep_release();
  const int c = blockIdx.x + 1;
  if (c >= a.header->ctas) return;
  const Start s = a.starts[c];
  if (s.k == 0 || s.first != c) return;
  const Tile t = a.tiles[s.tile];
  const int rows = t.ntok * a.group, row0 = blockIdx.y * 32;
  if (row0 < rows)
    combine_rows<T, D>(a, t, s.head, c, a.cuts[c].last, kBM, row0, rows < row0 + 32 ? rows : row0 + 32, threadIdx.x, 128);
}

template <typename T, int D>
int launch(const Args &a, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t st, const char *op) {
  constexpr int smem = static_cast<int>(TcCfg<D>::kSmem);
  if (cudaFuncSetAttribute(paged_attn_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch(op);
  launch_k(paged_attn_tc_kernel<T, D>, dim3(a.parts), dim3(kThreads), smem, st, a, kmap, vmap);
  if (a.parts > 1) launch_k(paged_combine_kernel<T, D>, dim3(a.parts - 1, kBM / 32), dim3(128), 0, st, a);
  return XN_OK;
}

}  // namespace

int launch_tc(const Args &a, int d, int dtype, cudaStream_t st, const char *op) {
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
