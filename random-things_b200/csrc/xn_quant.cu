// xn_quant.cu - RMSNorm with the residual's addition and an output in 8 bits
// (OCP e4m3) with one f32 scale per row or per group of columns, for sm_100a.
//
//   h = src or T(src + branch); y = h * (1 / sqrt(sum h^2 / cols + eps)) * alpha
//   scale = max |y| / 448;  dst = e4m3(y * (1 / scale))
//
// Bytes bound: src, branch and h cross memory once in T, dst in one byte. The
// row stays in registers between the sum of squares, the largest magnitude and
// the conversion. All of it is f32; the roundings are h (the residual stream's
// own type), y's f32 operations, and the one to e4m3.
#include <cuda_fp8.h>

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

// |y| as a whole number: the order of magnitudes, with NaN above infinity, so
// that a NaN is the largest of its group.
__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t umax2(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Multiplies by 1 / scale; a scale too small for its reciprocal divides, a
// scale of 0 has only zeros.
struct Scaler {
  float scale, inv;
  __device__ __forceinline__ explicit Scaler(uint32_t mag) {
    scale = __fdiv_rn(__uint_as_float(mag), 448.f);
    inv = __frcp_rn(scale);
  }
  __device__ __forceinline__ float operator()(float y) const {
    if (scale < 0x1p-100f) return scale == 0.f ? 0.f : __fdiv_rn(y, scale);
    return __fmul_rn(y, inv);
  }
};

__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// Largest value over a row group of tpr threads (as group_sum).
__device__ __forceinline__ uint32_t row_umax(uint32_t v, int tpr, uint32_t *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < tpr) v = umax2(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr <= 32) return v;
  const int warp = threadIdx.x >> 5, wpr = tpr >> 5, first = (warp / wpr) * wpr;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  uint32_t s = red[first];
  for (int w = 1; w < wpr; ++w) s = umax2(s, red[first + w]);
  return s;
}

// The row in registers: N accesses of V elements by each of its tpr threads.
template <typename T, int V, int N>
__global__ void __launch_bounds__(1024) rms_norm_q8_kernel(const Q8Params p) {
  griddep_wait();
  griddep_release();
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int tpr = p.tpr, g = threadIdx.x / tpr, lr = threadIdx.x - g * tpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + g;
  const bool live = row < p.rows;
  const int64_t base = row * p.cols, nvec = p.cols / V;
  float h[N][V];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t c = lr + static_cast<int64_t>(i) * tpr;
    const bool in = live && c < nvec;
    if constexpr (V == 1) {
      float x = in ? ld_elem<T>(p.src, base + c) : 0.f;
      if (in && p.branch != nullptr) x = Elem<T>::round(__fadd_rn(x, ld_elem<T>(p.branch, base + c)));
      if (in && p.residual_out != nullptr) st_elem<T>(p.residual_out, base + c, x);
      h[i][0] = x;
    } else {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (in) {
        x = ld_stream(static_cast<const T *>(p.src) + base + c * V);
        if (p.branch != nullptr) x = residual_vec<T>(x, ld_stream(static_cast<const T *>(p.branch) + base + c * V), nullptr);
        if (p.residual_out != nullptr) st_vec(static_cast<T *>(p.residual_out) + base + c * V, x);
      }
      unpack<T>(x, h[i]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sum = __fmaf_rn(h[i][j], h[i][j], sum);
  }
  sum = group_sum<false>(sum, tpr, red_sum);
  const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.cols)), p.eps)));
  uint32_t mag[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t c = lr + static_cast<int64_t>(i) * tpr;
    float w[V];
    if constexpr (V == 1) {
      w[0] = c < nvec ? ld_elem<T>(p.alpha, c) : 0.f;
    } else {
      unpack<T>(c < nvec ? ld_cached(static_cast<const T *>(p.alpha) + c * V) : make_uint4(0u, 0u, 0u, 0u), w);
    }
    mag[i] = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[i][j] = __fmul_rn(__fmul_rn(h[i][j], rstd), w[j]);
      if (c < nvec) mag[i] = umax2(mag[i], magnitude(h[i][j]));
    }
  }
  if (p.group == 0) {
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) all = umax2(all, mag[i]);
    all = row_umax(all, tpr, red_max);
#pragma unroll
    for (int i = 0; i < N; ++i) mag[i] = all;
    if (live && lr == 0) p.scales[row] = Scaler(all).scale;
  } else if constexpr (V > 1) {
    const int lanes = p.group / V;  // neighbouring lanes of one group; a group is whole or absent
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < lanes) mag[i] = umax2(mag[i], __shfl_xor_sync(0xffffffffu, mag[i], o));
      const int64_t c = lr + static_cast<int64_t>(i) * tpr;
      if (live && c < nvec && lr % lanes == 0) p.scales[row * (nvec / lanes) + c / lanes] = Scaler(mag[i]).scale;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t c = lr + static_cast<int64_t>(i) * tpr;
    if (!live || c >= nvec) continue;
    const Scaler s(mag[i]);
    uint8_t *dst = p.dst + base + c * V;
    if constexpr (V == 1) {
      *dst = static_cast<uint8_t>(e4m3x2(s(h[i][0]), 0.f));
    } else {
      uint32_t word[V / 4];
#pragma unroll
      for (int j = 0; j < V; j += 4) word[j / 4] = e4m3x2(s(h[i][j]), s(h[i][j + 1])) | e4m3x2(s(h[i][j + 2]), s(h[i][j + 3])) << 16;
      if constexpr (V == 8)
        *reinterpret_cast<uint2 *>(dst) = make_uint2(word[0], word[1]);
      else
        *reinterpret_cast<uint32_t *>(dst) = word[0];
    }
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
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
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
  const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.cols)), p.eps)));
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
  uint32_t all = 0;
  if (group == 0) {
    for (int64_t k = 0; k < per_thread; ++k) all = umax2(all, magnitude(y_at(column(k))));
    all = row_umax(all, 1024, red_max);
    if (threadIdx.x == 0) p.scales[blockIdx.x] = Scaler(all).scale;
  }
  const int gi = group == 0 ? 4 : group / 32;  // elements of a thread in one group
  for (int64_t k = 0; k < per_thread; k += gi) {
    float y[4];
    uint32_t mag = all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[j] = j < gi ? y_at(column(k + j)) : 0.f;
      if (group != 0) mag = umax2(mag, magnitude(y[j]));
    }
    if (group != 0) {
      mag = __reduce_max_sync(0xffffffffu, mag);
      if (lane == 0 && column(k) < p.cols) p.scales[blockIdx.x * (p.cols / group) + column(k) / group] = Scaler(mag).scale;
    }
    const Scaler s(mag);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = column(k + j);
      if (j < gi && c < p.cols) p.dst[base + c] = static_cast<uint8_t>(e4m3x2(s(y[j]), 0.f));
    }
  }
}

template <typename T, int V>
bool launch_q8_rows(Q8Params p, cudaStream_t st) {
  const int64_t nvec = p.cols / V;
  int64_t tpr = pow2_ceil(ceil_div(nvec, int64_t{4}));
  if (tpr > 1024) {
    if (V > 1 || nvec > 8 * 1024) return false;
    tpr = 1024;
  }
  if (p.group != 0 && tpr < p.group / V) tpr = p.group / V;
  const int n = static_cast<int>(ceil_div(nvec, tpr));
  const int block = tpr < 256 ? 256 : static_cast<int>(tpr);
  p.tpr = static_cast<int>(tpr);
  const dim3 grid(static_cast<unsigned>(ceil_div(p.rows, int64_t{block} / tpr)));
  if (n <= 1)
    launch_k(rms_norm_q8_kernel<T, V, 1>, grid, dim3(block), 0, st, p);
  else if (n <= 2)
    launch_k(rms_norm_q8_kernel<T, V, 2>, grid, dim3(block), 0, st, p);
  else if (n <= 4)
    launch_k(rms_norm_q8_kernel<T, V, 4>, grid, dim3(block), 0, st, p);
  else if constexpr (V == 1)
    launch_k(rms_norm_q8_kernel<T, V, 8>, grid, dim3(block), 0, st, p);
  return true;
}

template <typename T>
int launch_q8(Q8Params p, cudaStream_t st, const char *op) {
  constexpr int V = Elem<T>::kVec;
  const bool aligned = p.cols % V == 0 && is_aligned16(p.src) && is_aligned16(p.alpha) && is_aligned16(p.dst) &&
                       (p.branch == nullptr || is_aligned16(p.branch)) &&
                       (p.residual_out == nullptr || is_aligned16(p.residual_out));
  bool done = false;
  if (aligned)
    done = launch_q8_rows<T, V>(p, st);
  else if (p.group == 0)
    done = launch_q8_rows<T, 1>(p, st);
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
  if (rows == 0 || cols == 0) return ok();
  if (rows > 0x7fffffffLL) return fail(XN_E_INVALID, "%s: too many rows (%lld)", op, (long long)rows);
  if (dst == nullptr || scales == nullptr || src == nullptr || alpha == nullptr)
    return fail(XN_E_INVALID, "%s: null pointer", op);
  Q8Params p{static_cast<uint8_t *>(dst), scales, residual_out, src, alpha, branch, rows, cols, 0,
             static_cast<int>(group), eps};
  XN_DISPATCH_FLOAT(dtype, return launch_q8<T>(p, as_stream(stream), op));
  return fail(XN_E_DTYPE, "%s: unsupported dtype %d", op, dtype);
}
