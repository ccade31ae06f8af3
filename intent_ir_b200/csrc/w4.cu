// Products with 4-bit weights:
//   y[m, n] = sum over groups g of  s[n, g] * xs[m, g] * sum over k in g of  x[m, k] * (q[n, k] - z[n, g])   + bias[n]
// q is [N, K/2], the even k of a byte in its low half; z is 8 where there are no zero points; xs (the scales of 8-bit
// activations) is 1, one value per row, or one per row and group.  x * (q - z) is exact in f32 (and in the 16-bit types),
// sums are f32.
#include "common.cuh"
#include "held8.cuh"

namespace ib200 {
namespace {

struct W4Args {
  const void* x;
  const uint8_t* q;
  const void* s;
  const uint8_t* z;
  const void* bias;
  const float* xs;
  void* y;
  int64_t x_stride;
  int m, n, k, group, groups, xs_groups;
};

enum : int { X_BF16 = 0, X_F16 = 1, X_E4M3 = 2, X_I8 = 3 };
template <int XK> __device__ __forceinline__ float x_value(const void* x, int64_t i) {
  if (XK == X_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
  if (XK == X_F16) return __half2float(static_cast<const __half*>(x)[i]);
  return held_value<XK == X_E4M3 ? HELD_E4M3 : HELD_I8>(static_cast<const uint8_t*>(x)[i]);
}

// one warp per output and row of x; a lane takes 8 adjacent k (one word of q), which lie in one group
template <int XK, typename TS, typename TY>
__global__ void __launch_bounds__(256) w4_fma_kernel(const W4Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t total = (int64_t)a.n * a.m;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < total; u += (int64_t)gridDim.x * 8) {
    const int n = (int)(u % a.n), m = (int)(u / a.n);
    float acc = 0.0f;
    for (int k = lane * 8; k < a.k; k += 256) {
      const int g = k / a.group;
      const uint8_t* q = a.q + ((int64_t)n * a.k + k) / 2;
      const float z = a.z ? (float)a.z[(int64_t)n * a.groups + g] : 8.0f;
      float part = 0.0f;
      for (int i = 0; i < 8; ++i) {
        const float v = (float)((q[i >> 1] >> (4 * (i & 1))) & 15) - z;
        part = fmaf(x_value<XK>(a.x, m * a.x_stride + k + i), v, part);
      }
      float s = to_f32(static_cast<const TS*>(a.s)[(int64_t)n * a.groups + g]);
      if (a.xs) s *= a.xs[(int64_t)m * a.xs_groups + (a.xs_groups == 1 ? 0 : g)];
      acc = fmaf(part, s, acc);
    }
    acc = warp_reduce<SumOp>(acc);
    if (lane == 0) {
      if (a.bias) acc += to_f32(static_cast<const TY*>(a.bias)[n]);
      static_cast<TY*>(a.y)[(int64_t)m * a.n + n] = from_f32<TY>(acc);
    }
  }
}

template <int XK, typename TS, typename TY> int run_w4(const W4Args& a, cudaStream_t s) {
  const int64_t blocks = ((int64_t)a.n * a.m + 7) / 8;
  w4_fma_kernel<XK, TS, TY><<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 256, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "w4_matmul launch");
}
template <int XK, typename TS> int run_w4_out(const W4Args& a, int out, cudaStream_t s) {
  if (out == IB200_BF16) return run_w4<XK, TS, __nv_bfloat16>(a, s);
  if (out == IB200_F16) return run_w4<XK, TS, __half>(a, s);
  return run_w4<XK, TS, float>(a, s);
}
template <int XK> int run_w4_scale(const W4Args& a, int st, int out, cudaStream_t s) {
  if (st == IB200_BF16) return run_w4_out<XK, __nv_bfloat16>(a, out, s);
  if (st == IB200_F16) return run_w4_out<XK, __half>(a, out, s);
  return run_w4_out<XK, float>(a, out, s);
}

}  // namespace

size_t w4_scratch_bytes(int, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_w4(const void* x, int64_t x_stride, const float* xs, int64_t xs_groups, const void* q, const void* scales, const void* zeros,
              const void* bias, void* y, int x_dtype, int s_dtype, int out_dtype, int64_t m, int64_t n, int64_t k, int64_t group,
              void*, size_t, int32_t*, cudaStream_t s) {
  if (m < 0 || n < 0 || k < 0) return fail(IB200_ERR_INVALID, "w4_matmul: negative extent");
  if (beyond_any_device(m, k) || beyond_any_device(n, k) || beyond_any_device(m, n)) return fail(IB200_ERR_INVALID, "w4_matmul: more than 2^40 elements");
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX - 1024) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: extents are below 2^31");
  const bool held = x_dtype == IB200_E4M3 || x_dtype == IB200_I8;
  if (!held && x_dtype != IB200_BF16 && x_dtype != IB200_F16) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: x must be bf16, f16, e4m3 or int8");
  auto is_float = [](int t) { return t == IB200_F32 || t == IB200_BF16 || t == IB200_F16; };
  if (!is_float(s_dtype)) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: scales must be f32, bf16 or f16");
  if (!is_float(out_dtype)) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: the result is f32, bf16 or f16");
  if (group != 32 && group != 64 && group != 128) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: groups of 32, 64 or 128");
  if (k % 32) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: K must be a multiple of 32");
  const int64_t groups = (k + group - 1) / group;
  if (held != (xs_groups != 0) || (xs_groups != 0 && xs_groups != 1 && xs_groups != groups))
    return fail(IB200_ERR_INVALID, "w4_matmul: 8-bit x comes with one scale per row or one per row and group, other x with none");
  if (m == 0 || n == 0) return IB200_OK;
  if (!y || (k > 0 && (!x || !q || !scales || (held && !xs)))) return fail(IB200_ERR_INVALID, "w4_matmul: null operand");
  if (!aligned16(q)) return fail(IB200_ERR_INVALID, "w4_matmul: q must be 16-byte aligned");
  if (m > 1 && (x_stride < k || beyond_any_device(m, x_stride > 0 ? x_stride : 1))) return fail(IB200_ERR_INVALID, "w4_matmul: bad row stride of x");
  W4Args a{x, static_cast<const uint8_t*>(q), scales, static_cast<const uint8_t*>(zeros), bias, xs, y, x_stride,
           (int)m, (int)n, (int)k, (int)group, (int)groups, (int)xs_groups};
  if (x_dtype == IB200_BF16) return run_w4_scale<X_BF16>(a, s_dtype, out_dtype, s);
  if (x_dtype == IB200_F16) return run_w4_scale<X_F16>(a, s_dtype, out_dtype, s);
  if (x_dtype == IB200_E4M3) return run_w4_scale<X_E4M3>(a, s_dtype, out_dtype, s);
  return run_w4_scale<X_I8>(a, s_dtype, out_dtype, s);
}

}  // namespace ib200
