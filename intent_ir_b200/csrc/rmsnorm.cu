// Root-mean-square norm with the residual's addition in front and, on request, an 8-bit result with scales:
//   h = x + residual;  y = h / sqrt(mean(h^2) + eps) * w;  per group of columns  s = max|y| / Q,  q = round(y * Q / max|y|)
// with Q = 448 (e4m3) or 127 (int8).  h is stored rounded to the row type; everything else is computed from the unrounded
// f32 sum, so the stored rounding of h does not enter y.
#include "common.cuh"
#include "held8.cuh"

namespace ib200 {
namespace {

struct RmsArgs {
  const void *x, *res, *w;
  void *y, *h;
  float* scale;
  int64_t x_stride, res_stride, h_stride;
  int64_t rows, cols, groups;  // groups: scales per row
  int group;                   // columns per scale, 0: the whole row
  float eps;
};

constexpr float kScaleDown = 0x1p-80f;  // takes every f32 to where its square, and 2^30 of them, stay finite
constexpr int VE = 8;  // elements per thread and vector

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[VE], bool vec, int left) {
  if (vec && left >= VE) {
    float a[4], b[4];
    load4(p, a);
    load4(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[VE], bool vec, int left) {
  if (vec && left >= VE) {
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    store4(p, a);
    store4(p + 4, b);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < left) p[i] = from_f32<T>(v[i]);
  }
}

// One CTA per row, three passes over it (sum of squares, scales, values); any width.
template <typename T, typename TW, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_stream(const RmsArgs a, const bool vec) {
  __shared__ float slots[2][32];
  const int64_t nv = (a.cols + VE - 1) / VE, nv_warp = (nv + 31) / 32 * 32;  // whole warps take part in the group maxima
  const TW* w = static_cast<const TW*>(a.w);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;
    T* h = a.h ? static_cast<T*>(a.h) + row * a.h_stride : nullptr;
    auto sum8 = [&](int64_t v, float(&out)[VE]) {
      const int left = (int)min((int64_t)VE, a.cols - v * VE);
      load8(x + v * VE, out, vec, left);
      if (res) {
        float r[VE];
        load8(res + v * VE, r, vec, left);
#pragma unroll
        for (int i = 0; i < VE; ++i) out[i] += r[i];
      }
      return left;
    };
    auto norm8 = [&](int64_t v, float rstd, float(&out)[VE], int left) {
      float ww[VE];
      if (w) load8(w + v * VE, ww, vec, left);
#pragma unroll
      for (int i = 0; i < VE; ++i) out[i] = out[i] * rstd * (w ? ww[i] : 1.0f);
    };
    auto squares = [&](float pre, float* at) {
      float ss = 0.0f;
      for (int64_t v = threadIdx.x; v < nv; v += THREADS) {
        float e[VE];
        sum8(v, e);
#pragma unroll
        for (int i = 0; i < VE; ++i) ss = fmaf(e[i] * pre, e[i] * pre, ss);
      }
      return block_reduce<SumOp>(ss, at);
    };
    float ss = squares(1.0f, slots[0]), rstd;
    if (isinf(ss)) {  // values beyond 2^60: their squares overflow f32, so the row is summed again scaled down (uniform over the CTA)
      ss = squares(kScaleDown, slots[1]);
      rstd = kScaleDown / sqrtf(ss / (float)a.cols);
      __syncthreads();
    } else {
      rstd = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
    }
    float row_max = 0.0f;
    if (HELD != HELD_NONE && a.group == 0) {
      for (int64_t v = threadIdx.x; v < nv; v += THREADS) {
        float e[VE];
        const int left = sum8(v, e);
        norm8(v, rstd, e, left);
#pragma unroll
        for (int i = 0; i < VE; ++i) row_max = max_nan(row_max, fabsf(e[i]));
      }
      row_max = block_reduce<MaxOp>(row_max, slots[1]);
      if (threadIdx.x == 0) a.scale[row] = row_max / held_top<HELD>();
    }
    for (int64_t v = threadIdx.x; v < nv_warp; v += THREADS) {
      float e[VE];
      int left = 0;
      if (v < nv) {
        left = sum8(v, e);
        if (h) store8(h + v * VE, e, vec, left);
        norm8(v, rstd, e, left);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = 0.0f;
      }
      if constexpr (HELD == HELD_NONE) {
        if (v < nv) store8(static_cast<T*>(a.y) + row * a.cols + v * VE, e, vec, left);
      } else {
        float top = row_max;
        if (a.group) {
          const int lanes = a.group / VE;  // lanes that share a scale: 4, 8, 16 or 32
          top = 0.0f;
#pragma unroll
          for (int i = 0; i < VE; ++i) top = max_nan(top, fabsf(e[i]));
          for (int o = lanes >> 1; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (v < nv && (v % lanes) == 0) a.scale[row * a.groups + v / lanes] = top / held_top<HELD>();
        }
        if (v < nv) hold8<HELD>(static_cast<uint8_t*>(a.y) + row * a.cols + v * VE, e, held_inverse<HELD>(top), vec, left);
      }
    }
    __syncthreads();  // the next row reuses the reduction slots
  }
}

template <typename T, typename TW, int HELD> int run_rms(const RmsArgs& a, bool vec, cudaStream_t s) {
  constexpr int THREADS = 256;
  const int64_t grid = a.rows < (1 << 20) ? a.rows : (1 << 20);
  rmsnorm_stream<T, TW, HELD, THREADS><<<(unsigned)grid, THREADS, 0, s>>>(a, vec);
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "rmsnorm launch");
}
template <typename T, typename TW> int run_rms_held(const RmsArgs& a, int out_dtype, bool vec, cudaStream_t s) {
  if (out_dtype == IB200_E4M3) return run_rms<T, TW, HELD_E4M3>(a, vec, s);
  if (out_dtype == IB200_I8) return run_rms<T, TW, HELD_I8>(a, vec, s);
  return run_rms<T, TW, HELD_NONE>(a, vec, s);
}

}  // namespace

int launch_rmsnorm(const void* x, int64_t x_stride, const void* res, int64_t res_stride, const void* w, void* y, void* h, int64_t h_stride,
                   float* scale, int dtype, int w_dtype, int out_dtype, int64_t rows, int64_t cols, int64_t group, float eps, cudaStream_t s) {
  if (rows < 0 || cols < 0) return fail(IB200_ERR_INVALID, "rmsnorm: negative extent");
  if (beyond_any_device(rows, cols)) return fail(IB200_ERR_INVALID, "rmsnorm: more than 2^40 elements");
  if (dtype != IB200_F32 && dtype != IB200_BF16 && dtype != IB200_F16) return fail(IB200_ERR_UNSUPPORTED, "rmsnorm: rows must be f32, bf16 or f16");
  if (w && w_dtype != dtype && w_dtype != IB200_F32) return fail(IB200_ERR_UNSUPPORTED, "rmsnorm: the weight must be f32 or of the rows' type");
  const bool held = out_dtype == IB200_E4M3 || out_dtype == IB200_I8;
  if (!held && out_dtype != dtype) return fail(IB200_ERR_UNSUPPORTED, "rmsnorm: the result is of the rows' type, e4m3 or int8");
  if (group != 0 && (!held || (group != 32 && group != 64 && group != 128 && group != 256)))
    return fail(IB200_ERR_UNSUPPORTED, "rmsnorm: a scale covers 32, 64, 128 or 256 columns of an 8-bit result, or (0) the whole row");
  if (h && !res) return fail(IB200_ERR_INVALID, "rmsnorm: the sum is written only where there is a residual");
  if (rows == 0 || cols == 0) return IB200_OK;
  if (!x || !y || (held && !scale)) return fail(IB200_ERR_INVALID, "rmsnorm: null operand");
  if (rows > 1 && (x_stride < cols || (res && res_stride < cols) || (h && h_stride < cols)))
    return fail(IB200_ERR_INVALID, "rmsnorm: rows overlap (a row stride below the width)");
  if (beyond_any_device(rows, x_stride > 0 ? x_stride : 1) || (res && beyond_any_device(rows, res_stride > 0 ? res_stride : 1)) ||
      (h && beyond_any_device(rows, h_stride > 0 ? h_stride : 1)))
    return fail(IB200_ERR_INVALID, "rmsnorm: a row stride beyond any device");
  const int e = dtype_size(dtype);
  RmsArgs a{x, res, w, y, h, scale, x_stride, res_stride, h_stride, rows, cols, group ? (cols + group - 1) / group : 1, (int)group, eps};
  // 16-byte loads: every row of every operand has to begin on a 16-byte boundary (8 bytes for the held result)
  auto even = [&](const void* p, int64_t stride, int bytes) { return !p || (aligned16(p) && (rows == 1 || stride * bytes % 16 == 0)); };
  const bool vec = even(x, x_stride, e) && even(res, res_stride, e) && even(h, h_stride, e) && even(w, 0, 4) &&
                   (held ? (reinterpret_cast<uintptr_t>(y) & 7) == 0 && (rows == 1 || cols % 8 == 0) : even(y, cols, e));
  const bool wide_w = w_dtype == IB200_F32 || !w;
  if (dtype == IB200_F32) return run_rms_held<float, float>(a, out_dtype, vec, s);
  if (dtype == IB200_BF16)
    return wide_w ? run_rms_held<__nv_bfloat16, float>(a, out_dtype, vec, s) : run_rms_held<__nv_bfloat16, __nv_bfloat16>(a, out_dtype, vec, s);
  return wide_w ? run_rms_held<__half, float>(a, out_dtype, vec, s) : run_rms_held<__half, __half>(a, out_dtype, vec, s);
}

}  // namespace ib200
