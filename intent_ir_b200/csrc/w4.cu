// Products with 4-bit weights:
//   y[m, n] = sum over groups g of  s[n, g] * xs[m, g] * sum over k in g of  x[m, k] * (q[n, k] - z[n, g])   + bias[n]
// q is [N, K/2], the even k of a byte in its low half; z is 8 where there are no zero points; xs (the scales of 8-bit
// activations) is 1, one value per row, or one per row and group.  x * (q - z) is exact in f32 (and in the 16-bit types),
// sums are f32.
#include "async.cuh"
#include "common.cuh"
#include "held8.cuh"
#include "tma.h"

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
  int x_type, s_type, y_type, x_vec, split;
  int32_t* status;
};

__device__ __forceinline__ void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_read(const float* local, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map(local, (uint32_t)rank)) : "memory");
  return v;
}
__device__ __forceinline__ float float_of(const void* p, int64_t i, int type) {
  if (type == IB200_F32) return static_cast<const float*>(p)[i];
  if (type == IB200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// ---- few rows of x: weights stream through shared memory into mma.sync ----------------------------------
// A CTA has 128 rows of q, four warps of 32 on each half of a stage's 256 k, and a slice of K; the CTAs of a cluster share the rows and split K, and
// add their sums up through distributed shared memory in a fixed order.  One tensor copy brings a stage of q (128 rows x
// 128 bytes, zeros outside the matrix).  Weights are the 16 rows of m16n8k16, 8 rows of x its
// columns.  A thread's k slots need not be adjacent as long as both operands agree: inside a group of G, thread t of a quad owns
// the G / 4 adjacent k from t * G / 4, one 32-bit word of q (8 k) per two products, which keeps every product inside one
// group; the group's sum is then scaled in f32.  A word gives pairs (0, 4), (1, 5), (2, 6), (3, 7), so x is laid down in that order, in
// the order in which the warps read it.  128 + q in bf16 (1024 + q in f16) is q under the exponent of 128 (1024); minus 128 + z it is exact.
constexpr int kRows = 128, kThreads = 256, kStageK = 256, kStages = 4, kRowBytes = kStageK / 2, kStageBytes = kRows * kRowBytes;

template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 128 + z (1024 + z) in both halves of a word: what brings a nibble under the exponent back to q - z
template <bool BF> __device__ __forceinline__ uint32_t zero_of(uint32_t z) { return ((BF ? 0x4300u : 0x6400u) | z) * 0x10001u; }
// the pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's eight q - z
template <bool BF> __device__ __forceinline__ void weights_of(uint32_t w, uint32_t zero, uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | (BF ? 0x43004300u : 0x64006400u);
    if (BF) {
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&zero));
      v[i] = *reinterpret_cast<const uint32_t*>(&d);
    } else {
      const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&zero));
      v[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}
// 8 adjacent x as they lie in memory.  Loading and converting are apart: a converted value makes its warp wait for the load.
__device__ __forceinline__ uint4 x_raw(const W4Args& a, int row, int k) {
  uint4 r = make_uint4(0, 0, 0, 0);
  if (row >= a.m || k >= a.k) return r;
  const int64_t at = (int64_t)row * a.x_stride + k;
  if (a.x_type == IB200_BF16 || a.x_type == IB200_F16) {
    const uint16_t* p = static_cast<const uint16_t*>(a.x) + at;
    if (a.x_vec) return *reinterpret_cast<const uint4*>(p);
    r.x = p[0] | (uint32_t)p[1] << 16, r.y = p[2] | (uint32_t)p[3] << 16, r.z = p[4] | (uint32_t)p[5] << 16, r.w = p[6] | (uint32_t)p[7] << 16;
  } else {
    const uint8_t* p = static_cast<const uint8_t*>(a.x) + at;
    if (a.x_vec) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      r.x = v.x, r.y = v.y;
    } else {
      r.x = p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16 | (uint32_t)p[3] << 24;
      r.y = p[4] | (uint32_t)p[5] << 8 | (uint32_t)p[6] << 16 | (uint32_t)p[7] << 24;
    }
  }
  return r;
}
// as the pairs above; 8-bit values become f16, which is exact
__device__ __forceinline__ uint4 x_pairs(const uint4& r, int type) {
  if (type == IB200_BF16 || type == IB200_F16)
    return make_uint4(__byte_perm(r.x, r.z, 0x5410), __byte_perm(r.x, r.z, 0x7632), __byte_perm(r.y, r.w, 0x5410), __byte_perm(r.y, r.w, 0x7632));
  uint4 v;
  const uint32_t a01 = __byte_perm(r.x, r.y, 0x5140), a23 = __byte_perm(r.x, r.y, 0x7362);  // bytes 0 4 1 5, 2 6 3 7
  if (type == IB200_E4M3) {
    widen<HELD_E4M3>(a01, v.x, v.y);
    widen<HELD_E4M3>(a23, v.z, v.w);
  } else {
    widen<HELD_I8>(a01, v.x, v.y);
    widen<HELD_I8>(a23, v.z, v.w);
  }
  return v;
}
__device__ __forceinline__ uint32_t raw_of(const void* p, int64_t i, int type) {
  return type == IB200_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float value_of(uint32_t raw, int type) {
  if (type == IB200_F16) return __half2float(__ushort_as_half((unsigned short)raw));
  return __uint_as_float(type == IB200_BF16 ? raw << 16 : raw);
}

// Row of a 16-row tile (below 8) that thread group g reads: with it, and the copy's swizzle (chunk ^ row % 8), eight lanes of a 16-byte
// read and sixteen of an 8-byte one touch all banks once.
template <int G> __device__ __forceinline__ int row_of(int g) { return G == 128 ? (g >> 1) + 4 * (g & 1) : G == 64 ? (g & 3) * 2 + (g >> 2) : g; }

template <bool BF, int NT, int G>
__global__ void __launch_bounds__(kThreads, 2) w4_stream_kernel(const W4Args a, const __grid_constant__ CUtensorMap map) {
  constexpr int GROUPS = kStageK / G, HALF = GROUPS / 2, WORDS = G / 32;  // groups of a stage, of a warp's half; words of a thread in a group
  constexpr int XBYTES = NT * 8 * (kStageK * 2 + GROUPS * 4);
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[kStages];
  uint8_t* xbuf = smem + kStages * kStageBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, wr = warp & 3, wk = warp >> 2, pg = row_of<G>(g);
  const int split = a.split, rank = blockIdx.x % split, n0 = (blockIdx.x / split) * kRows, m0 = blockIdx.y * NT * 8;
  const int stages = (a.k + kStageK - 1) / kStageK, s0 = (int)((int64_t)stages * rank / split), s1 = (int)((int64_t)stages * (rank + 1) / split);

  auto issue = [&](int s) {  // (one thread)
    const int i = (s - s0) % kStages;
    mbarrier_expect_tx(&full[i], kStageBytes);
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_addr(smem + i * kStageBytes)), "l"(&map), "r"(smem_addr(&full[i])), "r"(s * kRowBytes), "r"(n0) : "memory");
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbarrier_init(&full[i], 1);
    mbarrier_init_fence();
    for (int i = 0; i < kStages - 1; ++i)
      if (s0 + i < s1) issue(s0 + i);
  }
  // x: chunk (8 k) of row m, where the warps read it: [group, word][tile of 8 rows][row][thread of the quad]
  auto x_place = [&](int idx) {
    const int row = idx / (kStageK / 8), k = idx % (kStageK / 8) * 8, in = k % G, th = in / (G / 4), word = in % (G / 4) / 8;
    return (((k / G * WORDS + word) * NT + row / 8) * 8 + row % 8) * 4 + th;
  };
  uint4 xr[NT];
  float xsr = 1.0f;  // a scale of x, behind the stage's x: [group][row]
  auto x_load = [&](int s) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int idx = i * kThreads + threadIdx.x;
      xr[i] = x_raw(a, m0 + idx / (kStageK / 8), s * kStageK + idx % (kStageK / 8) * 8);
    }
    if (a.xs_groups > 1 && threadIdx.x < GROUPS * NT * 8) {
      const int m = m0 + threadIdx.x % (NT * 8), grp = s * GROUPS + threadIdx.x / (NT * 8);
      xsr = m < a.m && grp < a.groups ? a.xs[(int64_t)m * a.groups + grp] : 0.0f;
    }
  };
  auto x_store = [&](int s) {
    uint4* to = reinterpret_cast<uint4*>(xbuf + ((s - s0) & 1) * XBYTES);
#pragma unroll
    for (int i = 0; i < NT; ++i) to[x_place(i * kThreads + threadIdx.x)] = x_pairs(xr[i], a.x_type);
    if (a.xs_groups > 1 && threadIdx.x < GROUPS * NT * 8) reinterpret_cast<float*>(to + NT * 8 * kStageK / 8)[threadIdx.x] = xsr;
  };
  // scales and zero points of the thread's four rows (32 * wr + pg, + 8, + 16, + 24) in its half of the stage: lane t of a quad holds group t
  uint32_t sc[4], zp[4];
  int64_t row_at[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = n0 + wr * 32 + pg + 8 * r;
    row_at[r] = row < a.n ? (int64_t)row * a.groups + (t & (HALF - 1)) : -1;
  }
  auto scale_load = [&](int s) {
    const int grp = s * GROUPS + wk * HALF;
    const bool in = grp + (t & (HALF - 1)) < a.groups;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool take = in && row_at[r] >= 0;
      sc[r] = take ? raw_of(a.s, row_at[r] + grp, a.s_type) : 0u;
      zp[r] = take && a.z ? a.z[row_at[r] + grp] : 8u;
    }
  };

  float sum[2][NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[mt][nt][0] = sum[mt][nt][1] = sum[mt][nt][2] = sum[mt][nt][3] = 0.0f;

  if (s0 < s1) {
    x_load(s0);
    scale_load(s0);
    x_store(s0);
    if (s0 + 1 < s1) x_load(s0 + 1);
  }
  for (int s = s0; s < s1; ++s) {
    float scn[4];
    uint32_t zn[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) scn[r] = value_of(sc[r], a.s_type), zn[r] = zero_of<BF>(zp[r] & 15u);
    __syncthreads();  // stage s - 1 is read, x of stage s is there (and, at first, the barriers are)
    if (threadIdx.x == 0 && s + kStages - 1 < s1) issue(s + kStages - 1);
    if (s + 1 < s1) {
      x_store(s + 1);
      if (s + 2 < s1) x_load(s + 2);
      scale_load(s + 1);
    }
    if (!mbarrier_wait_bounded(&full[(s - s0) % kStages], ((s - s0) / kStages) & 1) && a.status) atomicCAS(a.status, 0, 8);
    const uint8_t* wst = smem + ((s - s0) % kStages) * kStageBytes + (wr * 32 + pg) * kRowBytes;
    const uint4* xst = reinterpret_cast<const uint4*>(xbuf + ((s - s0) & 1) * XBYTES) + lane;
#pragma unroll
    for (int gi = 0; gi < HALF; ++gi) {
      const int byte = wk * (kRowBytes / 2) + gi * (G / 2) + t * (G / 8);  // of the row
      const uint8_t* p = wst + ((((byte >> 4) ^ pg) << 4) + (byte & 15));
      uint32_t w[4][WORDS];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (G == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + r * 8 * kRowBytes);
          w[r][0] = v.x, w[r][WORDS > 1 ? 1 : 0] = v.y, w[r][WORDS > 2 ? 2 : 0] = v.z, w[r][WORDS > 3 ? 3 : 0] = v.w;
        } else if (G == 64) {
          const uint2 v = *reinterpret_cast<const uint2*>(p + r * 8 * kRowBytes);
          w[r][0] = v.x, w[r][WORDS > 1 ? 1 : 0] = v.y;
        } else {
          w[r][0] = *reinterpret_cast<const uint32_t*>(p + r * 8 * kRowBytes);
        }
      }
      const int from = (lane & ~3) | gi;
      float sg[4];
      uint32_t zg[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sg[r] = HALF > 1 ? __shfl_sync(0xffffffffu, scn[r], from) : scn[r];
        zg[r] = zn[r];
        if (HALF > 1 && a.z) zg[r] = __shfl_sync(0xffffffffu, zn[r], from);
      }
      float acc[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt][0] = acc[mt][nt][1] = acc[mt][nt][2] = acc[mt][nt][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        uint4 x[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) x[nt] = xst[(((wk * HALF + gi) * WORDS + k) * NT + nt) * 32];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t va[4], vb[4];
          weights_of<BF>(w[2 * mt][k], zg[2 * mt], va);
          weights_of<BF>(w[2 * mt + 1][k], zg[2 * mt + 1], vb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<BF>(acc[mt][nt], va[0], vb[0], va[1], vb[1], x[nt].x, x[nt].y);
            mma<BF>(acc[mt][nt], va[2], vb[2], va[3], vb[3], x[nt].z, x[nt].w);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float2 f = make_float2(1.0f, 1.0f);
        if (a.xs_groups > 1)
          f = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(xst - lane + NT * 8 * kStageK / 8) + (wk * HALF + gi) * NT * 8 + nt * 8 + 2 * t);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[mt][nt][c] = fmaf(acc[mt][nt][c], a.xs_groups > 1 ? sg[2 * mt + (c >> 1)] * (c & 1 ? f.y : f.x) : sg[2 * mt + (c >> 1)], sum[mt][nt][c]);
      }
    }
  }

  // ---- add up the cluster's slices and write --------------------------------------------------------------
  __syncthreads();
  float* box = reinterpret_cast<float*>(smem);  // [half of K][NT * 8][128] sums of this CTA
  constexpr int BOX = NT * 8 * kRows;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) box[wk * BOX + (nt * 8 + 2 * t + (c & 1)) * kRows + wr * 32 + mt * 16 + pg + 8 * (c >> 1)] = sum[mt][nt][c];
  if (split > 1) cluster_arrive_wait(); else __syncthreads();
  const int rows = min(NT * 8, a.m - m0);
  for (int idx = rank * kThreads + threadIdx.x; idx < rows * kRows; idx += split * kThreads) {
    const int m = m0 + idx / kRows, n = n0 + idx % kRows;
    float v = 0.0f;
    for (int r = 0; r < split; ++r)
      v += split > 1 ? cluster_read(box + idx, r) + cluster_read(box + BOX + idx, r) : box[idx] + box[BOX + idx];
    if (n >= a.n) continue;
    if (a.xs_groups == 1) v *= a.xs[m];
    if (a.bias) v += float_of(a.bias, n, a.y_type);
    const int64_t at = (int64_t)m * a.n + n;
    if (a.y_type == IB200_F32) static_cast<float*>(a.y)[at] = v;
    else if (a.y_type == IB200_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(a.y)[at] = __float2half_rn(v);
  }
  if (split > 1) cluster_arrive_wait();  // nobody leaves while its sums are read
}

template <bool BF, int NT, int G> int run_stream(W4Args a, cudaStream_t s) {
  auto* kern = w4_stream_kernel<BF, NT, G>;
  constexpr int SMEM = kStages * kStageBytes + 2 * NT * 8 * (kStageK * 2 + kStageK / G * 4);
  IB200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  // K is split over a cluster so that the CTAs, two per SM at a time, have as few stages one after the other as can be
  const int tiles = (a.n + kRows - 1) / kRows, stages = (a.k + kStageK - 1) / kStageK, mt = (a.m + NT * 8 - 1) / (NT * 8);
  int split = 1;
  int64_t best = INT64_MAX;
  for (int i = 1; i <= 8 && (i == 1 || i <= stages); ++i) {
    const int64_t rounds = ((int64_t)tiles * mt * i + 2 * kSmCount - 1) / (2 * kSmCount), cost = rounds * ((stages + i - 1) / i + 2);  // 2: begin and end
    if (cost < best) best = cost, split = i;
  }
  CUtensorMap map = {};
  if (a.k > 0)
    if (int rc = make_byte_map(&map, a.q, a.n, a.k / 2, kRows)) return rc;
  a.split = split;
  if ((int64_t)tiles * split > INT32_MAX || mt > 65535) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split), (unsigned)mt);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  IB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, map));
  return IB200_OK;
}
template <bool BF, int NT> int run_stream_group(const W4Args& a, cudaStream_t s) {
  if (a.group == 128) return run_stream<BF, NT, 128>(a, s);
  if (a.group == 64) return run_stream<BF, NT, 64>(a, s);
  return run_stream<BF, NT, 32>(a, s);
}
template <bool BF> int run_stream_rows(const W4Args& a, cudaStream_t s) {
  if (a.m <= 8) return run_stream_group<BF, 1>(a, s);
  if (a.m <= 16) return run_stream_group<BF, 2>(a, s);
  return run_stream_group<BF, 4>(a, s);
}

}  // namespace

size_t w4_scratch_bytes(int, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_w4(const void* x, int64_t x_stride, const float* xs, int64_t xs_groups, const void* q, const void* scales, const void* zeros,
              const void* bias, void* y, int x_dtype, int s_dtype, int out_dtype, int64_t m, int64_t n, int64_t k, int64_t group,
              void*, size_t, int32_t* status, cudaStream_t s) {
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
  const int e = held ? 1 : 2;
  const bool x_vec = (reinterpret_cast<uintptr_t>(x) & (held ? 7 : 15)) == 0 && (m == 1 || x_stride * e % (held ? 8 : 16) == 0);
  W4Args a{x, static_cast<const uint8_t*>(q), scales, static_cast<const uint8_t*>(zeros), bias, xs, y, x_stride,
           (int)m, (int)n, (int)k, (int)group, (int)groups, (int)xs_groups, x_dtype, s_dtype, out_dtype, x_vec, 1, status};
  return x_dtype == IB200_BF16 ? run_stream_rows<true>(a, s) : run_stream_rows<false>(a, s);
}

}  // namespace ib200
