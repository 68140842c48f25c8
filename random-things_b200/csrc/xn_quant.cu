// xn_quant.cu - RMSNorm with the residual's addition and an output in 8 bits
// (OCP e4m3) with one f32 scale per row or per group of columns, for sm_100a.
//
//   h = src or T(src + branch); y = h * (1 / sqrt(sum h^2 / cols + eps)) * alpha
//   scale = max |y| / 448;  dst = e4m3(y * (1 / scale)), the reciprocal rounded
//
// Bytes bound: src, branch and h cross memory once in T, dst in one byte. The
// row stays in registers between the sum of squares, the largest magnitude and
// the conversion. All of it is f32; the roundings are h (the residual stream's
// own type), y's f32 operations, and the one to e4m3. Measured: 32768 x 4096
// bf16 with a residual 143 us (one scale a row) and 163 to 179 us (groups of
// 128), 1.0 and 0.80 to 0.88 of the measured copy rate.
#include <cuda_fp8.h>

#include <type_traits>

#include "xn_common.cuh"
#include "xn_internal.h"

namespace xn {
namespace {

struct Q8Params {
  uint8_t *dst;
  float *scales;
  void *residual_out;
  const void *src, *alpha, *branch;
  int64_t rows, cols;
  int tpr, group;
  float eps;
};

// The larger of magnitudes; NaN if one is NaN, so that a NaN reaches its group's scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// mag / 448, correctly rounded: Markstein's correction of a quotient, one FMA
// step on the product with the rounded reciprocal (an infinite mag has no
// remainder). Half ways between subnormal results may go to either side: there
// the remainder's product with a rounded reciprocal decides. (The division
// itself, for all or for subnormal results alone: 32768 x 4096 by groups 3% slower.)
__device__ __forceinline__ float scale_of(float mag) {
  constexpr float r = 1.f / 448.f;
  const float q = __fmul_rn(mag, r);
  return isinf(mag) ? mag : __fmaf_rn(__fmaf_rn(-448.f, q, mag), r, q);
}

// What y is multiplied with: 1 / scale; 0 for scale 0, whose y are all 0. A
// scale below 2^-100 may have no f32 reciprocal: `up` first lifts y by 2^64.
struct Inverse {
  float inv;
  bool up;
  __device__ __forceinline__ explicit Inverse(float scale) {
    up = scale < 0x1p-100f;
    inv = scale == 0.f ? 0.f : __frcp_rn(up ? scale * 0x1p64f : scale);
  }
};

__device__ __forceinline__ uint32_t e4m3x2(float2 v) { return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3); }

// Largest magnitude over a row group of tpr threads (as group_sum).
__device__ __forceinline__ float row_max(float v, int tpr, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < tpr) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr <= 32) return v;
  const int warp = threadIdx.x >> 5, wpr = tpr >> 5, first = (warp / wpr) * wpr;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float s = red[first];
  for (int w = 1; w < wpr; ++w) s = max_nan(s, red[first + w]);
  return s;
}

__device__ __forceinline__ float rstd_of(float sum, int64_t cols, float eps) {
  return __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(cols)), eps)));
}

// One access of a row: V elements as float2 pairs (V = 1: the second one 0).
template <typename T, int V>
struct Access {
  static constexpr int kAW = V * static_cast<int>(sizeof(T)) / 4;  // 32-bit words
  static constexpr int kP = V > 1 ? V / 2 : 1;
  using Raw = std::conditional_t<V == 1, T, uint4>;  // of a uint4, the kAW low words are in use
  __device__ __forceinline__ static Raw zero() {
    if constexpr (V == 1)
      return Elem<T>::from_f32(0.f);
    else
      return make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ static Raw load(const void *base, int64_t at) {
    const T *p = static_cast<const T *>(base) + at;
    if constexpr (V == 1)
      return *p;
    else
      return ld_stream_w<kAW>(p);
  }
  __device__ __forceinline__ static Raw load_cached(const void *base, int64_t at) {
    const T *p = static_cast<const T *>(base) + at;
    if constexpr (V == 1)
      return *p;
    else
      return ld_cached_w<kAW>(p);
  }
  __device__ __forceinline__ static void store(void *base, int64_t at, Raw v) {
    T *p = static_cast<T *>(base) + at;
    if constexpr (V == 1)
      *p = v;
    else
      st_w<kAW>(p, v);
  }
  __device__ __forceinline__ static Raw add(Raw x, Raw b) {
    if constexpr (V == 1)
      return Elem<T>::from_f32(__fadd_rn(Elem<T>::to_f32(x), Elem<T>::to_f32(b)));
    else
      return residual_vec<T, kAW>(x, b, nullptr);
  }
  __device__ __forceinline__ static void unpack(Raw v, float2 (&h)[kP]) {
    if constexpr (V == 1) {
      h[0] = make_float2(Elem<T>::to_f32(v), 0.f);
    } else {
      float2 all[Pairs<T>::kP];
      Pairs<T>::unpack(v, all);
#pragma unroll
      for (int j = 0; j < kP; ++j) h[j] = all[j];
    }
  }
};

// The row in registers: N accesses of V elements by each of its tpr threads.
template <typename T, int V, int N, int kBlock, bool kGroups>
__global__ void __launch_bounds__(kBlock, kBlock == 256 ? (V * sizeof(T) == 16 ? 4 : 3) : 1) rms_norm_q8_kernel(const Q8Params p) {
  griddep_wait();
  griddep_release();
  using A = Access<T, V>;
  constexpr int P = A::kP;
  __shared__ float red_sum[32], red_max[32];
  const int tpr = p.tpr, g = threadIdx.x / tpr, lr = threadIdx.x - g * tpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + g;
  const int nacc = row < p.rows ? static_cast<int>(p.cols / V) : 0;  // accesses of this row
  const int64_t base = row * p.cols;
  float2 h[N][P];
  {
    // All loads first: each would otherwise wait for the store before it.
    typename A::Raw x[N], br[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = lr + i * tpr;
      x[i] = c < nacc ? A::load(p.src, base + c * V) : A::zero();
      if (p.branch != nullptr) br[i] = c < nacc ? A::load(p.branch, base + c * V) : A::zero();
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = lr + i * tpr;
      if (p.branch != nullptr) x[i] = A::add(x[i], br[i]);
      if (c < nacc && p.residual_out != nullptr) A::store(p.residual_out, base + c * V, x[i]);
      A::unpack(x[i], h[i]);
    }
  }
  // The weights are under way during the first reduction, where registers allow it.
  constexpr bool kEarly = V > 1;
  auto weight = [&](int i) { return lr + i * tpr < nacc ? A::load_cached(p.alpha, (lr + i * tpr) * V) : A::zero(); };
  typename A::Raw w[kEarly ? N : 1];
  if constexpr (kEarly) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = weight(i);
  }
  float2 sq = splat2(0.f);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < P; ++j) sq = __ffma2_rn(h[i][j], h[i][j], sq);
  const float sum = group_sum<false>(__fadd_rn(sq.x, sq.y), tpr, red_sum);
  const float rstd = rstd_of(sum, p.cols, p.eps);
  float mag[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float2 wf[P];
    A::unpack(kEarly ? w[kEarly ? i : 0] : weight(i), wf);
    mag[i] = 0.f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      h[i][j] = __fmul2_rn(__fmul2_rn(h[i][j], splat2(rstd)), wf[j]);
      mag[i] = max_nan(mag[i], fabsf(h[i][j].x), V > 1 ? fabsf(h[i][j].y) : 0.f);
    }
    if (lr + i * tpr >= nacc) mag[i] = 0.f;  // 0 * inf, where rstd is infinite
  }
  float scale[kGroups ? N : 1];
  if constexpr (!kGroups) {
    float all = mag[0];
#pragma unroll
    for (int i = 1; i < N; ++i) all = max_nan(all, mag[i]);
    scale[0] = scale_of(row_max(all, tpr, red_max));
    if (nacc > 0 && lr == 0) p.scales[row] = scale[0];
  } else {
    const int lanes = p.group / V;  // neighbouring lanes of one group; a group is whole or absent
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < lanes) mag[i] = max_nan(mag[i], __shfl_xor_sync(0xffffffffu, mag[i], o));
      scale[i] = scale_of(mag[i]);
      const int c = lr + i * tpr;
      if (c < nacc && lr % lanes == 0) p.scales[row * (nacc / lanes) + c / lanes] = scale[i];
    }
  }
  Inverse s(scale[0]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = lr + i * tpr;
    if (kGroups && i > 0) s = Inverse(scale[kGroups ? i : 0]);
    if (s.up) {
#pragma unroll
      for (int j = 0; j < P; ++j) h[i][j] = __fmul2_rn(h[i][j], splat2(0x1p64f));
    }
    uint32_t two[P];
#pragma unroll
    for (int j = 0; j < P; ++j) two[j] = e4m3x2(__fmul2_rn(h[i][j], splat2(s.inv)));
    if (c >= nacc) continue;
    uint8_t *dst = p.dst + base + c * V;
    if constexpr (V == 8)
      *reinterpret_cast<uint2 *>(dst) = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
    else if constexpr (V == 4)
      *reinterpret_cast<uint32_t *>(dst) = two[0] | two[1] << 16;
    else if constexpr (V == 2)
      *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(two[0]);
    else
      *dst = static_cast<uint8_t>(two[0]);
  }
}

// Rows too wide for registers: one block a row, elements read again for each
// of the three passes. Every element belongs to one thread in all passes, so
// the row that the first pass wrote to residual_out (which may be src or
// branch) can be read back without a barrier.
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_q8_loop_kernel(const Q8Params p) {
  griddep_wait();
  griddep_release();
  __shared__ float red_sum[32], red_max[32];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * p.cols;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = p.group;
  // Column of this thread's k-th element: warps take runs of 128 columns.
  auto column = [&](int64_t k) { return (k / 4 * 32 + warp) * 128 + k % 4 * 32 + lane; };
  const int64_t per_thread = (p.cols + 4095) / 4096 * 4;
  float sum = 0.f;
  for (int64_t k = 0; k < per_thread; ++k) {
    const int64_t c = column(k);
    if (c >= p.cols) continue;
    float x = ld_elem<T>(p.src, base + c);
    if (p.branch != nullptr) x = Elem<T>::round(__fadd_rn(x, ld_elem<T>(p.branch, base + c)));
    if (p.residual_out != nullptr) st_elem<T>(p.residual_out, base + c, x);
    sum = __fmaf_rn(x, x, sum);
  }
  sum = group_sum<false>(sum, 1024, red_sum);
  const float rstd = rstd_of(sum, p.cols, p.eps);
  auto y_at = [&](int64_t c) {
    if (c >= p.cols) return 0.f;
    float x;
    if (p.residual_out != nullptr) {
      x = ld_elem<T>(p.residual_out, base + c);
    } else {
      x = ld_elem<T>(p.src, base + c);
      if (p.branch != nullptr) x = Elem<T>::round(__fadd_rn(x, ld_elem<T>(p.branch, base + c)));
    }
    return __fmul_rn(__fmul_rn(x, rstd), ld_elem<T>(p.alpha, c));
  };
  float all = 0.f;
  if (group == 0) {
    for (int64_t k = 0; k < per_thread; ++k) all = max_nan(all, fabsf(y_at(column(k))));
    all = row_max(all, 1024, red_max);
    if (threadIdx.x == 0) p.scales[blockIdx.x] = scale_of(all);
  }
  const int gi = group == 0 ? 4 : group / 32;  // elements of a thread in one group
  for (int64_t k = 0; k < per_thread; k += gi) {
    float y[4], mag = all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[j] = j < gi ? y_at(column(k + j)) : 0.f;
      if (group != 0) mag = max_nan(mag, fabsf(y[j]));
    }
    if (group != 0) {
      mag = row_max(mag, 32, red_max);
      if (lane == 0 && column(k) < p.cols) p.scales[blockIdx.x * (p.cols / group) + column(k) / group] = scale_of(mag);
    }
    const Inverse s(scale_of(mag));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = column(k + j);
      if (j < gi && c < p.cols)
        p.dst[base + c] = static_cast<uint8_t>(e4m3x2(make_float2(__fmul_rn(s.up ? y[j] * 0x1p64f : y[j], s.inv), 0.f)));
    }
  }
}

template <typename T, int V, int N, bool kGroups>
void launch_q8_n(const Q8Params &p, cudaStream_t st) {
  const int block = p.tpr < 256 ? 256 : p.tpr;
  const dim3 grid(static_cast<unsigned>(ceil_div(p.rows, int64_t{block} / p.tpr)));
  if (block == 256)
    launch_k(rms_norm_q8_kernel<T, V, N, 256, kGroups>, grid, dim3(block), 0, st, p);
  else
    launch_k(rms_norm_q8_kernel<T, V, N, 1024, kGroups>, grid, dim3(block), 0, st, p);
}

// Threads of a row: as few as hold it with n_max accesses each when there are
// rows enough to fill the GPU; with few rows more of them, down to one access
// each, since then the row's own latency is the call's time.
template <typename T, int V, bool kGroups>
bool launch_q8_rows(Q8Params p, cudaStream_t st) {
  constexpr int kMost = V * sizeof(T) == 16 ? 4 : V == 2 ? 8 : 16;
  const int64_t nacc = p.cols / V;
  int64_t tpr = pow2_ceil(ceil_div(nacc, int64_t{kMost}));
  // (Element accesses by 1024 threads leave no registers: 8000 rows of 9001 f16 710 us, against 501 us row by row.)
  if (tpr > (V == 1 ? 512 : 1024)) return false;
  while (tpr < 1024 && tpr < nacc && p.rows * tpr < int64_t{sm_count()} * 512) tpr *= 2;
  if (kGroups && tpr < p.group / V) tpr = p.group / V;
  const int64_t n = ceil_div(nacc, tpr);
  p.tpr = static_cast<int>(tpr);
  if (n <= 1)
    launch_q8_n<T, V, 1, kGroups>(p, st);
  else if (n <= 2)
    launch_q8_n<T, V, 2, kGroups>(p, st);
  else if (n <= 4)
    launch_q8_n<T, V, 4, kGroups>(p, st);
  else if constexpr (kMost >= 8) {
    if (n <= 8)
      launch_q8_n<T, V, 8, kGroups>(p, st);
    else if constexpr (kMost >= 16)
      launch_q8_n<T, V, 16, kGroups>(p, st);
  }
  return true;
}

template <typename T>
int launch_q8(const Q8Params &p, cudaStream_t st, const char *op) {
  // The widest access that every row and pointer is aligned to.
  auto fits = [&](int v) {
    const uintptr_t bytes = v * sizeof(T);
    uintptr_t at = reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.alpha) |
                   reinterpret_cast<uintptr_t>(p.branch) | reinterpret_cast<uintptr_t>(p.residual_out);
    return p.cols % v == 0 && at % bytes == 0 && reinterpret_cast<uintptr_t>(p.dst) % v == 0;
  };
  constexpr int V = Elem<T>::kVec;
  bool done = false;
  if (p.cols == 0)  // scales alone, all 0: the kernel for wide rows has nothing else to do
    ;
  else if (fits(V))
    done = p.group != 0 ? launch_q8_rows<T, V, true>(p, st) : launch_q8_rows<T, V, false>(p, st);
  else if (p.group == 0)
    done = fits(2) ? launch_q8_rows<T, 2, false>(p, st) : launch_q8_rows<T, 1, false>(p, st);
  if (!done) launch_k(rms_norm_q8_loop_kernel<T>, dim3(static_cast<unsigned>(p.rows)), dim3(1024), 0, st, p);
  return check_launch(op);
}

}  // namespace
}  // namespace xn

extern "C" int xn_rms_norm_q8(void *dst, float *scales, void *residual_out, const void *src, const void *alpha,
                              const void *branch, int64_t rows, int64_t cols, int64_t group, float eps, int dtype,
                              void *stream) {
  using namespace xn;
  const char *op = "xn_rms_norm_q8";
  if (!is_float_dtype(dtype)) return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (rows < 0 || cols < 0) return fail(XN_E_INVALID, "%s: negative size", op);
  if (!(eps > 0.f)) return fail(XN_E_INVALID, "%s: eps must be positive", op);
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return fail(XN_E_INVALID, "%s: group %lld not in {0, 32, 64, 128}", op, (long long)group);
  if (group != 0 && cols % group != 0)
    return fail(XN_E_INVALID, "%s: group %lld does not divide cols=%lld", op, (long long)group, (long long)cols);
  if (rows == 0 || (cols == 0 && group != 0)) return ok();
  if (rows > 0x7fffffffLL) return fail(XN_E_INVALID, "%s: too many rows (%lld)", op, (long long)rows);
  if (scales == nullptr || (cols > 0 && (dst == nullptr || src == nullptr || alpha == nullptr)))
    return fail(XN_E_INVALID, "%s: null pointer", op);
  Q8Params p{static_cast<uint8_t *>(dst), scales, residual_out, src, alpha, branch, rows, cols, 0,
             static_cast<int>(group), eps};
  XN_DISPATCH_FLOAT(dtype, return launch_q8<T>(p, as_stream(stream), op));
  return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
}
