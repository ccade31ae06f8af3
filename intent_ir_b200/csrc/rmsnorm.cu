// Root-mean-square norm with the residual's addition in front and, on request, an 8-bit result with scales:
//   h = x + residual;  y = h / sqrt(mean(h^2) + eps) * w;  per group of columns  s = max|y| * (1 / Q),  q = round(y * Q / max|y|)
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
  int out_type, wide_w;        // IB200_E4M3, IB200_I8 or the rows' type; whether w is f32
  float eps, least;            // least: sums of squares below it are taken again
};

// Rows whose squares overflow f32 (values beyond 2^60), and those whose squares vanish beside an eps that small, are summed again scaled by a power of two.
// The sum's threshold leaves what subnormal squares lose (2^-150 each) below 2^-24 of it, and scaled up it stays finite.
constexpr float kScaleDown = 0x1p-80f;  // takes every f32 to where its square, and 2^30 of them, stay finite
constexpr float kScaleUp = 0x1p96f, kVanishing = 0x1p-80f, kVanishingEps = 0x1p-90f, kMost = 3.402823466e38f;
// Such a row's 1 / sqrt(mean + eps) as two factors for its elements, one after the other, so that neither product leaves f32's range
// where the result does not; sum: of the squares of the elements times scale_of(ss).
__device__ __forceinline__ float scale_of(float ss) { return ss > 1.0f ? kScaleDown : kScaleUp; }
__device__ __forceinline__ float2 two_factors(float ss, float sum, float cols, float eps) {
  const float pre = scale_of(ss), r = 1.0f / sqrtf(sum / cols + eps * pre * pre);
  return ss > 1.0f ? make_float2(r * 0x1p-40f, kScaleDown * 0x1p40f) : make_float2(kScaleUp, r);
}
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

template <typename T> __device__ __forceinline__ void load_w8(const RmsArgs& a, int64_t at, float (&v)[VE], bool vec, int left) {
  if (a.wide_w) load8(static_cast<const float*>(a.w) + at, v, vec, left);
  else load8(static_cast<const T*>(a.w) + at, v, vec, left);
}
template <typename T> __device__ __forceinline__ float load_w(const RmsArgs& a, int64_t at) {
  return a.wide_w ? static_cast<const float*>(a.w)[at] : to_f32(static_cast<const T*>(a.w)[at]);
}
__device__ __forceinline__ float top_inverse(int type) { return type == IB200_E4M3 ? held_unit<HELD_E4M3>() : held_unit<HELD_I8>(); }
__device__ __forceinline__ float inverse_of(int type, float top) { return type == IB200_E4M3 ? held_inverse<HELD_E4M3>(top) : held_inverse<HELD_I8>(top); }

// The same to 2 ulp without a division, for the scales of groups, of which there are many: a value within 4 ulp of the middle between two held ones may go to
// the other than a division would send it to.  The error against the unheld value is half a step either way.
__device__ __forceinline__ float inverse_fast(int type, float top) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(top));
  r *= type == IB200_E4M3 ? 448.0f : 127.0f;
  return top == 0.0f || isinf(r) ? 0.0f : r;
}

// ---- rows that fit the registers of a warp or a CTA -------------------------------------------------------
// One read of x and the residual, one write of everything: HBM-bound.  With VECTORS a thread has 8 adjacent columns, 8 * 32
// or 8 * THREADS apart (16-byte accesses).  Rows that do not begin on 16-byte boundaries are read element by
// element, or two by two where 16-bit rows allow it; a warp then has 256 * NV adjacent columns, lane by lane (coalesced).  Either way the columns that share a scale
// lie in one warp.
// bf16 16384 x 8192 + residual -> e4m3 with scales of 128: 155 us (6.1 TB/s, 0.93 of a copy's rate; 70 % of the issue slots); three passes over the row took 254, and
// divisions instead of the approximate reciprocal for the scales of groups 180, bound by instruction issue.  f32 1021 x 5001, where no row is aligned:
// 18.0 us (4.5 TB/s) lane by lane, 46.6 with eight adjacent columns to a thread.  16 x 4096: 3.0 us, one chain of load, two reductions and store.
template <typename T> struct Raw { uint4 v[sizeof(T) / 2]; };  // 8 elements as they lie in memory
template <typename T> __device__ __forceinline__ Raw<T> read8(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T> __device__ __forceinline__ void floats8(const Raw<T>& r, float (&v)[VE]) {
  const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = to_f32(p[i]);
}
template <typename T> __device__ __forceinline__ void write8(T* p, const float (&v)[VE]) {
  Raw<T> r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < VE; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, r.v[i]);
}

enum : int { LANES = 0, PAIRS = 1, VECTORS = 2 };
template <typename T> struct alignas(2 * sizeof(T)) Two { T v[2]; };
template <typename T> __device__ __forceinline__ void read2(const T* p, float& x, float& y) {
  const Two<T> r = *reinterpret_cast<const Two<T>*>(p);
  x = to_f32(r.v[0]), y = to_f32(r.v[1]);
}
template <typename T> __device__ __forceinline__ void write2(T* p, float x, float y) { *reinterpret_cast<Two<T>*>(p) = {from_f32<T>(x), from_f32<T>(y)}; }

template <typename T, bool HELD, int THREADS, int NV, int HOW>
__global__ void __launch_bounds__(THREADS == 32 ? 256 : THREADS) rmsnorm_resident(const RmsArgs a) {
  constexpr bool VEC = HOW == VECTORS, PAIR = HOW == PAIRS;
  __shared__ float slots[2][32];
  const int tid = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31, cols = (int)a.cols;
  const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps, and nothing below waits for other rows' warps
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;
  auto total = [&](float v, float* at) { return THREADS == 32 ? warp_reduce<SumOp>(v) : block_reduce<SumOp>(v, at); };
  // column of element i of vector k
  auto col = [&](int k, int i) { return VEC ? (k * THREADS + tid) * VE + i : PAIR ? (tid >> 5) * (256 * NV) + (k * VE + (i & ~1)) * 32 + lane * 2 + (i & 1) : (tid >> 5) * (256 * NV) + (k * VE + i) * 32 + lane; };

  float e[NV][VE];
  if (VEC) {
    Raw<T> xr[NV], rr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (col(k, 0) < cols) xr[k] = read8(x + col(k, 0));
    if (res) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (col(k, 0) < cols) rr[k] = read8(res + col(k, 0));
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const bool in = col(k, 0) < cols;
#pragma unroll
      for (int i = 0; i < VE; ++i) e[k][i] = 0.0f;
      if (in) {
        floats8(xr[k], e[k]);
        if (res) {
          float r[VE];
          floats8(rr[k], r);
#pragma unroll
          for (int i = 0; i < VE; ++i) e[k][i] += r[i];
        }
      }
    }
  } else if (PAIR) {
    auto read = [&](const T* p, float (&v)[NV][VE]) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; i += 2) {
          v[k][i] = v[k][i + 1] = 0.0f;
          if (col(k, i) < cols) read2(p + col(k, i), v[k][i], v[k][i + 1]);
        }
    };
    read(x, e);
    if (res) {
      float r[NV][VE];
      read(res, r);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) e[k][i] += r[k][i];
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) e[k][i] = col(k, i) < cols ? to_f32(x[col(k, i)]) : 0.0f;
    if (res) {
      float r[NV][VE];
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) r[k][i] = col(k, i) < cols ? to_f32(res[col(k, i)]) : 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) e[k][i] += r[k][i];
    }
  }
  if (a.h) {
    T* h = static_cast<T*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (VEC) {
        if (col(k, 0) < cols) write8(h + col(k, 0), e[k]);
      } else if (PAIR) {
#pragma unroll
        for (int i = 0; i < VE; i += 2)
          if (col(k, i) < cols) write2(h + col(k, i), e[k][i], e[k][i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (col(k, i) < cols) h[col(k, i)] = from_f32<T>(e[k][i]);
      }
    }
  }
  auto squares = [&](float pre) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) s = fmaf(e[k][i] * pre, e[k][i] * pre, s);
    return s;
  };
  const float ss = total(squares(1.0f), slots[0]);
  float rstd = 1.0f / sqrtf(ss / (float)cols + a.eps);
  if (!(ss >= a.least && ss <= kMost)) {  // (uniform over the row's threads; NaN comes here and stays)
    const float2 f = two_factors(ss, total(squares(scale_of(ss)), slots[1]), (float)cols, a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) e[k][i] *= f.x;
    rstd = f.y;
    if (THREADS != 32) __syncthreads();  // the slots are used again
  }
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float w[VE];
    if (a.w) {
      if (VEC) {
        if (col(k, 0) < cols) load_w8<T>(a, col(k, 0), w, true, VE);
      } else if (PAIR) {
#pragma unroll
        for (int i = 0; i < VE; i += 2) {
          w[i] = w[i + 1] = 0.0f;
          if (col(k, i) >= cols) continue;
          if (a.wide_w) read2(static_cast<const float*>(a.w) + col(k, i), w[i], w[i + 1]);
          else read2(static_cast<const T*>(a.w) + col(k, i), w[i], w[i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = col(k, i) < cols ? load_w<T>(a, col(k, i)) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      e[k][i] *= rstd;
      if (a.w && col(k, VEC ? 0 : i) < cols) e[k][i] *= w[i];
      if (HELD && a.group == 0) top = max_nan(top, fabsf(e[k][i]));
    }
  }
  if constexpr (!HELD) {
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (VEC) {
        if (col(k, 0) < cols) write8(y + col(k, 0), e[k]);
      } else if (PAIR) {
#pragma unroll
        for (int i = 0; i < VE; i += 2)
          if (col(k, i) < cols) write2(y + col(k, i), e[k][i], e[k][i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (col(k, i) < cols) y[col(k, i)] = from_f32<T>(e[k][i]);
      }
    }
  } else {
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.cols;
    float inv = 0.0f;
    if (a.group == 0) {
      top = THREADS == 32 ? warp_reduce<MaxOp>(top) : block_reduce<MaxOp>(top, slots[1]);
      if (tid == 0) a.scale[row] = top * top_inverse(a.out_type);
      inv = inverse_of(a.out_type, top);
    }
    const int lanes = a.group / VE, steps = a.group / 32, shift = __ffs(a.group) - 1;  // of a scale: lanes with VEC, elements of a lane without
    float tops[NV];
    if (VEC && a.group) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        tops[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < VE; ++i) tops[k] = max_nan(tops[k], fabsf(e[k][i]));
      }
      for (int o = lanes >> 1; o; o >>= 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) tops[k] = max_nan(tops[k], __shfl_xor_sync(0xffffffffu, tops[k], o));
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (VEC) {
        if (a.group) {
          const int c = col(k, 0);
          if (c < cols && (tid & (lanes - 1)) == 0) a.scale[row * a.groups + (c >> shift)] = tops[k] * top_inverse(a.out_type);
          inv = inverse_fast(a.out_type, tops[k]);
        }
        if (col(k, 0) < cols) {
          if (a.out_type == IB200_E4M3) hold8<HELD_E4M3>(y + col(k, 0), e[k], inv, true, VE);
          else hold8<HELD_I8>(y + col(k, 0), e[k], inv, true, VE);
        }
      } else {
        float m[VE];  // the maximum of element i's group (PAIRS have none)
        if (!PAIR && a.group) {
#pragma unroll
          for (int i = 0; i < VE; ++i) m[i] = warp_reduce<MaxOp>(fabsf(e[k][i]));
#pragma unroll
          for (int o = 1; o < VE; o <<= 1)
            if (o < steps) {
              float n[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) n[i] = max_nan(m[i], m[i ^ o]);
#pragma unroll
              for (int i = 0; i < VE; ++i) m[i] = n[i];
            }
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const int c = col(k, i);
          if (!PAIR && a.group) {
            inv = inverse_fast(a.out_type, m[i]);
            if (c < cols && lane == 0 && i % steps == 0) a.scale[row * a.groups + (c >> shift)] = m[i] * top_inverse(a.out_type);
          }
          if (c < cols) y[c] = (uint8_t)(a.out_type == IB200_E4M3 ? hold1<HELD_E4M3>(e[k][i] * inv) : hold1<HELD_I8>(e[k][i] * inv));
        }
      }
    }
  }
}

// ---- wider rows: one CTA per row, three passes over it (sum of squares, scales, values) -------------------
template <typename T, bool HELD, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_stream(const RmsArgs a, const bool vec) {
  __shared__ float slots[2][32];
  const int64_t nv = (a.cols + VE - 1) / VE, nv_warp = (nv + 31) / 32 * 32;  // whole warps take part in the group maxima
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
    auto norm8 = [&](int64_t v, float first, float rstd, float(&out)[VE], int left) {
      float ww[VE];
      if (a.w) load_w8<T>(a, v * VE, ww, vec, left);
#pragma unroll
      for (int i = 0; i < VE; ++i) out[i] = out[i] * first * rstd * (a.w ? ww[i] : 1.0f);
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
    const float ss = squares(1.0f, slots[0]);
    float rstd = 1.0f / sqrtf(ss / (float)a.cols + a.eps), first = 1.0f;
    if (!(ss >= a.least && ss <= kMost)) {  // (uniform over the CTA; NaN comes here and stays)
      const float2 f = two_factors(ss, squares(scale_of(ss), slots[1]), (float)a.cols, a.eps);
      first = f.x;
      rstd = f.y;
      __syncthreads();
    }
    float row_max = 0.0f;
    if (HELD && a.group == 0) {
      for (int64_t v = threadIdx.x; v < nv; v += THREADS) {
        float e[VE];
        const int left = sum8(v, e);
        norm8(v, first, rstd, e, left);
#pragma unroll
        for (int i = 0; i < VE; ++i) row_max = max_nan(row_max, fabsf(e[i]));
      }
      row_max = block_reduce<MaxOp>(row_max, slots[1]);
      if (threadIdx.x == 0) a.scale[row] = row_max * top_inverse(a.out_type);
    }
    for (int64_t v = threadIdx.x; v < nv_warp; v += THREADS) {
      float e[VE];
      int left = 0;
      if (v < nv) {
        left = sum8(v, e);
        if (h) store8(h + v * VE, e, vec, left);
        norm8(v, first, rstd, e, left);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = 0.0f;
      }
      if constexpr (!HELD) {
        if (v < nv) store8(static_cast<T*>(a.y) + row * a.cols + v * VE, e, vec, left);
      } else {
        float top = row_max;
        if (a.group) {
          const int lanes = a.group / VE;  // lanes that share a scale: 4, 8, 16 or 32
          top = 0.0f;
#pragma unroll
          for (int i = 0; i < VE; ++i) top = max_nan(top, fabsf(e[i]));
          for (int o = lanes >> 1; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (v < nv && (v % lanes) == 0) a.scale[row * a.groups + v / lanes] = top * top_inverse(a.out_type);
        }
        if (v < nv) {
          uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.cols + v * VE;
          if (a.out_type == IB200_E4M3) hold8<HELD_E4M3>(y, e, held_inverse<HELD_E4M3>(top), vec, left);
          else hold8<HELD_I8>(y, e, held_inverse<HELD_I8>(top), vec, left);
        }
      }
    }
    __syncthreads();  // the next row reuses the reduction slots
  }
}

template <typename T, bool HELD, int THREADS, int NV> int run_resident(const RmsArgs& a, int how, cudaStream_t s) {
  const unsigned grid = (unsigned)(THREADS == 32 ? (a.rows + 7) / 8 : a.rows), threads = THREADS == 32 ? 256 : THREADS;
  if (how == VECTORS) rmsnorm_resident<T, HELD, THREADS, NV, VECTORS><<<grid, threads, 0, s>>>(a);
  else if (how == PAIRS && sizeof(T) == 2) rmsnorm_resident<T, HELD, THREADS, NV, sizeof(T) == 2 ? PAIRS : LANES><<<grid, threads, 0, s>>>(a);
  else rmsnorm_resident<T, HELD, THREADS, NV, LANES><<<grid, threads, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "rmsnorm launch");
}
// Threads of a row: many rows want few, with the work of a thread in flight, few rows all that help.  bf16 + residual -> e4m3 with scales of 128, a warp or fewer threads
// against 256: 65 536 x 256 24.7 / 142 us (52 with registers for 1024), 16 384 x 1024 23.0 / 42.4, 16 384 x 1536 32.8 / 46.9, 16 384 x 2560 60.6 / 70.5; 592 x 1024 3.9 / 2.9,
// 16 x 2048 4.0 / 2.7, 600 x 4096 5.7 / 5.1 (and 1500 x 1024 4.8 / 5.4).  4096 x 16 384 in registers 89 us, streamed 140.
template <typename T, bool HELD> int run_rms(const RmsArgs& a, int how, cudaStream_t s) {
  const bool many = a.rows > 4 * kSmCount;
  if (a.rows <= INT32_MAX) {
    if (many && a.cols <= 4096) {
      if (a.cols <= 256) return run_resident<T, HELD, 32, 1>(a, how, s);
      if (a.cols <= 512) return run_resident<T, HELD, 32, 2>(a, how, s);
      if (a.cols <= 1024) return run_resident<T, HELD, 32, 4>(a, how, s);
      return a.cols <= 2048 ? run_resident<T, HELD, 64, 4>(a, how, s) : run_resident<T, HELD, 128, 4>(a, how, s);
    }
    if (a.cols <= 2048) return run_resident<T, HELD, 256, 1>(a, how, s);
    if (a.cols <= 4096) return run_resident<T, HELD, 256, 2>(a, how, s);
    if (a.cols <= 8192) return run_resident<T, HELD, 256, 4>(a, how, s);
    if (a.cols <= 16384) return run_resident<T, HELD, 512, 4>(a, how, s);
  }
  const int64_t grid = a.rows < (1 << 20) ? a.rows : (1 << 20);
  rmsnorm_stream<T, HELD, 512><<<(unsigned)grid, 512, 0, s>>>(a, how == VECTORS);
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "rmsnorm launch");
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
  if (rows > 0 && cols == 0 && held && group == 0) {  // the largest of no values is 0, and so is its scale
    if (!scale) return fail(IB200_ERR_INVALID, "rmsnorm: null operand");
    if (beyond_any_device(rows, 1)) return fail(IB200_ERR_INVALID, "rmsnorm: more than 2^40 rows");
    IB200_CUDA_OK(cudaMemsetAsync(scale, 0, (size_t)rows * sizeof(float), s));
    return IB200_OK;
  }
  if (rows == 0 || cols == 0) return IB200_OK;
  if (!x || !y || (held && !scale)) return fail(IB200_ERR_INVALID, "rmsnorm: null operand");
  if (rows > 1 && (x_stride < cols || (res && res_stride < cols) || (h && h_stride < cols)))
    return fail(IB200_ERR_INVALID, "rmsnorm: rows overlap (a row stride below the width)");
  if (beyond_any_device(rows, x_stride > 0 ? x_stride : 1) || (res && beyond_any_device(rows, res_stride > 0 ? res_stride : 1)) ||
      (h && beyond_any_device(rows, h_stride > 0 ? h_stride : 1)))
    return fail(IB200_ERR_INVALID, "rmsnorm: a row stride beyond any device");
  const int e = dtype_size(dtype);
  RmsArgs a{x, res, w, y, h, scale, x_stride, res_stride, h_stride, rows, cols, group ? (cols + group - 1) / group : 1, (int)group, out_dtype,
            w_dtype == IB200_F32, eps, eps < kVanishingEps ? kVanishing : -1.0f};
  // Every row of every operand has to begin on a boundary of `bytes`: 16 for vectors of eight (8 for the held result), 4 for pairs (2).  Scales of
  // groups are taken over the lanes of whole groups, which pairs do not have.  Pairs halve the accesses of 16-bit rows: f16 10 880 x 3084 63 us (95 element by element),
  // to e4m3 76 (130), 20 000 x 1002 33 (53); f32 rows lose by them (4000 x 5002 63, 54).
  auto at = [&](const void* p, int64_t row_bytes, int bytes) { return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows == 1 || row_bytes % bytes == 0)); };
  auto even = [&](int bytes, int w_bytes, int y_bytes) {
    return at(x, x_stride * e, bytes) && at(res, res_stride * e, bytes) && at(h, h_stride * e, bytes) && at(w, 0, w_bytes) && at(y, held ? cols : cols * e, y_bytes);
  };
  const int how = cols % VE == 0 && even(16, 16, held ? 8 : 16) ? VECTORS : e == 2 && cols % 2 == 0 && group == 0 && even(4, w_dtype == IB200_F32 ? 8 : 4, held ? 2 : 4) ? PAIRS : LANES;
  if (dtype == IB200_F32) return held ? run_rms<float, true>(a, how, s) : run_rms<float, false>(a, how, s);
  if (dtype == IB200_BF16) return held ? run_rms<__nv_bfloat16, true>(a, how, s) : run_rms<__nv_bfloat16, false>(a, how, s);
  return held ? run_rms<__half, true>(a, how, s) : run_rms<__half, false>(a, how, s);
}

}  // namespace ib200
