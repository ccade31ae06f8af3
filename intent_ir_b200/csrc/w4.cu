// Products with 4-bit weights:
//   y[m, n] = sum over groups g of  s[n, g] * xs[m, g] * sum over k in g of  x[m, k] * (q[n, k] - z[n, g])   + bias[n]
// q is [N, K/2], the even k of a byte in its low half; z is 0 .. 127, and 8 where there are no zero points; xs (the scales of 8-bit
// activations) is 1, one value per row, or one per row and group.  x * (q - z) is exact in f32 (and in the 16-bit types),
// sums are f32.
#include <array>
#include <map>
#include <mutex>

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
  int x_type, s_type, y_type, x_vec, s_vec, z_vec, split;
  int32_t* status;
};

__device__ __forceinline__ float float_of(const void* p, int64_t i, int type) {
  if (type == IB200_F32) return static_cast<const float*>(p)[i];
  if (type == IB200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// ---- few rows of x: weights stream through shared memory into mma.sync -----------------------------------
// A CTA has 128 rows of q, four warps of 32 on each half of a stage's 256 k, and a slice of K; the CTAs of a cluster share the rows and split K, and
// add their sums up through distributed shared memory in a fixed order.  One tensor copy brings a stage of q (128 rows x
// 128 bytes, zeros outside the matrix).  Weights are the 16 rows of m16n8k16, 8 rows of x its
// columns.  A thread's k slots need not be adjacent as long as both operands agree: inside a group of G, thread t of a quad owns
// the G / 4 adjacent k from t * G / 4, one 32-bit word of q (8 k) per two products, which keeps every product inside one
// group; the group's sum is then scaled in f32.  A word gives pairs (0, 4), (1, 5), (2, 6), (3, 7), so x is laid down in that order, in
// the order in which the warps read it.  128 + q in bf16 (1024 + q in f16) is q under the exponent of 128 (1024); minus 128 + z it is exact.
// A ninth warp brings the weights and x as said; it and the others meet at mbarriers only.  The scales are read by the threads that use them.
// 8192 x 8192 of groups of 128 and one row of bf16: 15.2 us (2.3 TB/s); 4096 x 4096: 6.5 us, of which two stages of loads and the cluster's sum are most; 7 x 5003 x 8192 in
// groups of 32 with zero points, f16: 15.5 us.  Waits bound it, not HBM: eight weights cost nine instructions in front of their products, but only 42 % of the issue slots
// (36 % in the last case) are taken.  The warps stand at barriers longest (the scale blocks' and the cluster's), then on fixed latencies and in the pipeline's filling.
// A ring filled by all warps took 24 us for the last case, one warp to an output 161.
constexpr int kRows = 128, kThreads = 288, kStageK = 256, kRowBytes = kStageK / 2;
enum : int { X_BF16 = 0, X_F16 = 1, X_E4M3 = 2, X_I8 = 3 };
constexpr int kRowScales = 144;  // a row's two blocks of eight scales, then of eight zero points' patterns; 16 bytes keep rows in different banks
template <int XK, int NT, int G> struct Stage {  // bytes of a stage's parts
  static constexpr int kStages = NT == 1 ? 4 : 3, GROUPS = kStageK / G;
  static constexpr int X_CHUNK = XK >= X_E4M3 ? 8 : 16;                     // 8 k of a row
  static constexpr int X_AT = kRows * kRowBytes;                              // after q: x in the order of its reads
  static constexpr int XS_AT = X_AT + NT * 8 * (kStageK / 8) * X_CHUNK;       // scales of x: [group][row]
  static constexpr int BYTES = (XS_AT + GROUPS * NT * 8 * 4 + 1023) / 1024 * 1024;
  static constexpr int S_AT = kStages * BYTES, SMEM = S_AT + kRows * kRowScales;  // behind the stages: the rows' scales
};
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {  // the rest of the 4 is zero
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (x & mask) | magic in one instruction; the compiler splits it when both are constants
template <uint32_t MASK> __device__ __forceinline__ uint32_t under(uint32_t x, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "n"(MASK), "r"(magic));
  return y;
}
// What brings a nibble under an exponent back to q - z, in both halves: 128 + z in bf16; 1024 + z, and -(64 + z) for nibbles four bits up, in f16.
// 128 + z fits bf16's eight bits up to z = 127; a zero point above makes the group's products NaN, in every type alike.
struct Zero {
  uint32_t lo, hi;
};
__device__ __forceinline__ uint32_t both_halves(uint32_t x) { return x * 0x10001u; }
template <bool BF> __device__ __forceinline__ uint32_t pattern16_of(uint32_t z) { return z > 127u ? 0x7fffu : (BF ? 0x4300u : 0x6400u) + z; }
template <bool BF> __device__ __forceinline__ uint32_t pattern_of(uint32_t z) { return both_halves(pattern16_of<BF>(z)); }
template <typename H> __device__ __forceinline__ H as_pair(uint32_t x) { return *reinterpret_cast<const H*>(&x); }
template <bool BF> __device__ __forceinline__ Zero zero_of(uint32_t pattern) {
  if (BF) return {pattern, 0u};
  const __half2 hi = __hsub2(__half2half2(__ushort_as_half(0x6380)), as_pair<__half2>(pattern));  // 960 - (1024 + z), exact
  return {pattern, *reinterpret_cast<const uint32_t*>(&hi)};
}
// the pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's eight q - z; `magic`: the exponent, in a register
template <bool BF> __device__ __forceinline__ void weights_of(uint32_t w, const Zero& z, uint32_t magic, uint32_t (&v)[4]) {
  if (BF) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 d = __hsub2(as_pair<__nv_bfloat162>(under<0x000f000fu>(w >> (4 * i), magic)), as_pair<__nv_bfloat162>(z.lo));
      v[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {  // a nibble four bits up is 16 q: one shift for two pairs
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2C00));
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t x = w >> (4 * i);
      const __half2 d = __hsub2(as_pair<__half2>(under<0x000f000fu>(x, magic)), as_pair<__half2>(z.lo));
      const __half2 e = __hfma2(as_pair<__half2>(under<0x00f000f0u>(x, magic)), sixteenth, as_pair<__half2>(z.hi));
      v[i] = *reinterpret_cast<const uint32_t*>(&d);
      v[i + 1] = *reinterpret_cast<const uint32_t*>(&e);
    }
  }
}
// eight adjacent x as the pairs above; 8-bit values become f16, which is exact
template <int XK> __device__ __forceinline__ uint4 x_pairs(const uint8_t* p) {
  if (XK == X_BF16 || XK == X_F16) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    return make_uint4(__byte_perm(r.x, r.z, 0x5410), __byte_perm(r.x, r.z, 0x7632), __byte_perm(r.y, r.w, 0x5410), __byte_perm(r.y, r.w, 0x7632));
  }
  constexpr int HELD = XK == X_E4M3 ? HELD_E4M3 : HELD_I8;
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  uint4 v;
  widen<HELD>(__byte_perm(r.x, r.y, 0x5140), v.x, v.y);  // bytes 0 4 1 5, 2 6 3 7
  widen<HELD>(__byte_perm(r.x, r.y, 0x7362), v.z, v.w);
  return v;
}
__device__ __forceinline__ float value_of(uint32_t raw, int type) {
  if (type == IB200_F16) return __half2float(__ushort_as_half((unsigned short)raw));
  return __uint_as_float(type == IB200_BF16 ? raw << 16 : raw);
}

__device__ __forceinline__ void tensor_copy(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y) : "memory");
}
// Scales and zero points of a row, eight groups at a time.  Of two warps that share 32 rows one reads the scales, a row to a lane, the other the zero
// points, one block ahead of its use, into registers; the block is left in one of two places in shared memory, as f32 and as patterns, when
// the warps come to it.  Groups behind the last one, and rows behind the last, have the scale 0.
struct RowBlock {
  uint32_t v[8];
};
__device__ __forceinline__ RowBlock read_block(const W4Args& a, bool zeros, int row, int block) {
  RowBlock r;
  const int g0 = block * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = 0;
  if (row >= a.n || g0 >= a.groups || (zeros && !a.z)) return r;
  const int64_t at = (int64_t)row * a.groups + g0;
  if (zeros) {
    if (a.z_vec) {
      const uint2 u = *reinterpret_cast<const uint2*>(a.z + at);
      r.v[0] = u.x, r.v[1] = u.y;  // four to a word
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (g0 + i < a.groups) r.v[i] = a.z[at + i];
    }
  } else if (a.s_vec) {
    if (a.s_type == IB200_F32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(a.s) + at);
      const uint4 u = p[0], v = p[1];
      r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w, r.v[4] = v.x, r.v[5] = v.y, r.v[6] = v.z, r.v[7] = v.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.s) + at);
      r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w;  // two to a word
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (g0 + i < a.groups) {
        if (a.s_type == IB200_F32) r.v[i] = static_cast<const uint32_t*>(a.s)[at + i];
        else r.v[i] = static_cast<const uint16_t*>(a.s)[at + i];
      }
  }
  return r;
}
__device__ __forceinline__ float scale_of(const W4Args& a, const RowBlock& r, int i) {
  return value_of(a.s_vec && a.s_type != IB200_F32 ? r.v[i / 2] >> (i & 1) * 16 & 0xffffu : r.v[i], a.s_type);
}
__device__ __forceinline__ uint32_t zero_byte(const W4Args& a, const RowBlock& r, int i) { return a.z_vec ? r.v[i / 4] >> (i & 3) * 8 & 0xffu : r.v[i]; }
template <bool BF> __device__ __forceinline__ void leave_block(const W4Args& a, bool zeros, uint8_t* row, int block, const RowBlock& r) {
  uint4* to = reinterpret_cast<uint4*>(row + (zeros ? 64 : 0) + (block & 1) * 32);
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (zeros) v[e] = pattern_of<BF>(zero_byte(a, r, i + e));
      else v[e] = __float_as_uint(scale_of(a, r, i + e));
    }
    to[i / 4] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

__device__ __forceinline__ void write_y(const W4Args& a, int m, int n, float v) {
  if (n >= a.n) return;
  if (a.xs_groups == 1) v *= a.xs[m];
  if (a.bias) v += float_of(a.bias, n, a.y_type);
  const int64_t at = (int64_t)m * a.n + n;
  if (a.y_type == IB200_F32) static_cast<float*>(a.y)[at] = v;
  else if (a.y_type == IB200_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(a.y)[at] = __float2half_rn(v);
}

// Row of a 16-row tile (below 8) that thread group g reads: with it, and the copy's swizzle (chunk ^ row % 8), eight lanes of a 16-byte
// read and sixteen of an 8-byte one touch all banks once.
template <int G> __device__ __forceinline__ int row_of(int g) { return G == 128 ? (g >> 1) + 4 * (g & 1) : G == 64 ? (g & 3) * 2 + (g >> 2) : g; }

template <int XK, int NT, int G>
__global__ void __launch_bounds__(kThreads, 2) w4_stream_kernel(const W4Args a, const __grid_constant__ CUtensorMap map) {
  using S = Stage<XK, NT, G>;
  constexpr bool BF = XK == X_BF16;
  constexpr int GROUPS = S::GROUPS, HALF = GROUPS / 2, WORDS = G / 32;  // groups of a stage, of a warp's half; words of a thread in a group
  constexpr int kStages = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[kStages], empty[kStages];
  __shared__ volatile int dead, brought;  // dead: a wait ran out, nothing waits any more; brought: stages in all
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, wr = warp & 3, wk = (warp >> 2) & 1, pg = row_of<G>(g);
  const int split = a.split, rank = blockIdx.x % split, n0 = (blockIdx.x / split) * kRows, m0 = blockIdx.y * NT * 8;
  const int stages = (a.k + kStageK - 1) / kStageK, s0 = (int)((int64_t)stages * rank / split), s1 = (int)((int64_t)stages * (rank + 1) / split);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbarrier_try_wait(bar, parity) || dead || mbarrier_wait_bounded(bar, parity)) return;
    dead = 1;
    if (a.status) atomicCAS(a.status, 0, 8);
  };
  if (threadIdx.x == 0) {
    dead = 0;
    brought = s1 - s0;
    for (int i = 0; i < kStages; ++i) mbarrier_init(&full[i], 1 + 32), mbarrier_init(&empty[i], 8);
    mbarrier_init_fence();
  }
  __syncthreads();
  float sum[2][NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[mt][nt][0] = sum[mt][nt][1] = sum[mt][nt][2] = sum[mt][nt][3] = 0.0f;

  if (warp == 8) {
    // ---- the bringing warp ----------------------------------------------------------------------------------
    const uint32_t smem_at = smem_addr(smem);
    for (int s = s0; s < s1; ++s) {
      const int i = (s - s0) % kStages;
      if (s - s0 >= kStages) wait(&empty[i], ((s - s0) / kStages - 1) & 1);
      const uint32_t dst = smem_at + i * S::BYTES;
      if (lane == 0) {
        mbarrier_expect_tx(&full[i], kRows * kRowBytes);
        tensor_copy(dst, &map, &full[i], s * kRowBytes, n0);
      }
      // x: lane l has the chunk (8 k) 8 l of each row, placed where the warps read it: [group, word][tile of 8 rows][row][thread of the quad]
      const int k = lane * 8, in = k % G, th = in / (G / 4), word = in % (G / 4) / 8;
      const uint32_t to0 = dst + S::X_AT + ((k / G * WORDS + word) * NT * 32 + th) * S::X_CHUNK;
      const bool k_in = s * kStageK + k < a.k;
      const uint8_t* x0 = static_cast<const uint8_t*>(a.x) + (k_in ? ((int64_t)m0 * a.x_stride + s * kStageK + k) * (S::X_CHUNK / 8) : 0);
#pragma unroll 8
      for (int row = 0; row < NT * 8; ++row) {
        const uint32_t to = to0 + row * 4 * S::X_CHUNK;
        const bool take = k_in && m0 + row < a.m;
        const uint8_t* src = take ? x0 + (int64_t)row * a.x_stride * (S::X_CHUNK / 8) : static_cast<const uint8_t*>(a.x);
        if (a.x_vec) {
          if (S::X_CHUNK == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(take ? 16 : 0) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(src), "r"(take ? 8 : 0) : "memory");
        } else {
          uint8_t* out = smem + (to - smem_at);
          for (int e = 0; e < 8; ++e) {
            if (S::X_CHUNK == 16) reinterpret_cast<uint16_t*>(out)[e] = take ? reinterpret_cast<const uint16_t*>(src)[e] : (uint16_t)0;
            else out[e] = take ? src[e] : (uint8_t)0;
          }
        }
      }
      if (XK >= X_E4M3 && a.xs_groups > 1) {
        for (int e = lane; e < GROUPS * NT * 8; e += 32) {
          const int m = m0 + e % (NT * 8), grp = s * GROUPS + e / (NT * 8);
          const bool take = m < a.m && grp < a.groups;
          copy4(dst + S::XS_AT + e * 4, a.xs + (take ? (int64_t)m * a.groups + grp : 0), take ? 4 : 0);
        }
      }
      if (a.x_vec) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&full[i])) : "memory");
      } else {  // x was written by stores, which an arrival of this thread's own releases
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&full[i])) : "memory");
      }
    }
  } else {
  // this thread's rows: 32 * wr + pg, + 8, + 16, + 24.  A stage's groups lie in one block.
  const uint8_t* scales = smem + S::S_AT + (wr * 32 + pg) * kRowScales;
  uint8_t* mine = smem + S::S_AT + (wr * 32 + lane) * kRowScales;  // the row whose blocks this lane reads
  const int my_row = n0 + wr * 32 + lane;
  int block = s0 * GROUPS >> 3;
  RowBlock ahead = read_block(a, wk, my_row, block);
  auto next_block = [&] {
    leave_block<BF>(a, wk, mine, block, ahead);
    ahead = read_block(a, wk, my_row, block + 1);
    asm volatile("bar.sync %0, 64;" ::"r"(1 + wr) : "memory");
  };
  next_block();
  uint32_t magic = BF ? 0x43004300u : 0x64006400u;
  asm volatile("" : "+r"(magic));  // (kept in a register)
  const Zero eight = zero_of<BF>(pattern_of<BF>(8));
  const bool xs_many = XK >= X_E4M3 && a.xs_groups > 1;
  for (int s = s0; s < s1; ++s) {
    wait(&full[(s - s0) % kStages], ((s - s0) / kStages) & 1);
    const uint8_t* st = smem + (s - s0) % kStages * S::BYTES;
    const uint8_t *wst = st + (wr * 32 + pg) * kRowBytes, *xst = st + S::X_AT + lane * S::X_CHUNK;
    if (s * GROUPS >> 3 != block) {
      block = s * GROUPS >> 3;
      next_block();
    }
    const uint8_t* from = scales + (block & 1) * 32 + ((s * GROUPS & 7) + wk * HALF) * 4;
    uint32_t sraw[4][HALF], zraw[4][HALF];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* p = from + 8 * r * kRowScales;
      if (HALF == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        sraw[r][0] = v.x, sraw[r][HALF > 1 ? 1 : 0] = v.y, sraw[r][HALF > 2 ? 2 : 0] = v.z, sraw[r][HALF > 3 ? 3 : 0] = v.w;
      } else if (HALF == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        sraw[r][0] = v.x, sraw[r][HALF > 1 ? 1 : 0] = v.y;
      } else {
        sraw[r][0] = *reinterpret_cast<const uint32_t*>(p);
      }
      if (a.z) {
        if (HALF == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + 64);
          zraw[r][0] = v.x, zraw[r][HALF > 1 ? 1 : 0] = v.y, zraw[r][HALF > 2 ? 2 : 0] = v.z, zraw[r][HALF > 3 ? 3 : 0] = v.w;
        } else if (HALF == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(p + 64);
          zraw[r][0] = v.x, zraw[r][HALF > 1 ? 1 : 0] = v.y;
        } else {
          zraw[r][0] = *reinterpret_cast<const uint32_t*>(p + 64);
        }
      }
    }
#pragma unroll
    for (int gi = 0; gi < HALF; ++gi) {
      const int byte = wk * (kRowBytes / 2) + gi * (G / 2) + t * (G / 8);  // of the row
      const uint8_t* p = wst + ((((byte >> 4) ^ pg) << 4) + (byte & 15));
      uint32_t w[4][WORDS];
      Zero zero[4];
      float sg[4];
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
        sg[r] = __uint_as_float(sraw[r][gi]);
        zero[r] = a.z ? zero_of<BF>(zraw[r][gi]) : eight;
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
        for (int nt = 0; nt < NT; ++nt) x[nt] = x_pairs<XK>(xst + (((wk * HALF + gi) * WORDS + k) * NT + nt) * 32 * S::X_CHUNK);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t va[4], vb[4];
          weights_of<BF>(w[2 * mt][k], zero[2 * mt], magic, va);
          weights_of<BF>(w[2 * mt + 1][k], zero[2 * mt + 1], magic, vb);
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
        if (xs_many) f = *reinterpret_cast<const float2*>(st + S::XS_AT + ((wk * HALF + gi) * NT * 8 + nt * 8 + 2 * t) * 4);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[mt][nt][c] = fmaf(acc[mt][nt][c], xs_many ? sg[2 * mt + (c >> 1)] * (c & 1 ? f.y : f.x) : sg[2 * mt + (c >> 1)], sum[mt][nt][c]);
      }
    }
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&empty[(s - s0) % kStages])) : "memory");
  }
  }

  // ---- add up the cluster's slices and write --------------------------------------------------------------
  __syncthreads();
  if (dead) {  // whichever warp gave up: copies that are still on their way land before their memory is used again or the CTA ends
    bool landed = true;
    for (int n = brought, s = max(0, n - kStages); s < n; ++s) landed = landed && mbarrier_wait_bounded(&full[s % kStages], (s / kStages) & 1);
  }
  float* box = reinterpret_cast<float*>(smem);  // [half of K][NT * 8][128] sums of this CTA
  constexpr int BOX = NT * 8 * kRows;
  if (warp < 8)
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) box[wk * BOX + (nt * 8 + 2 * t + (c & 1)) * kRows + wr * 32 + mt * 16 + pg + 8 * (c >> 1)] = sum[mt][nt][c];
  if (split > 1) cluster_sync(); else __syncthreads();
  const int rows = min(NT * 8, a.m - m0);
  for (int idx = rank * kThreads + threadIdx.x; idx < rows * kRows; idx += split * kThreads) {
    const int m = m0 + idx / kRows, n = n0 + idx % kRows;
    float v = 0.0f;
    for (int r = 0; r < split; ++r)
      v += split > 1 ? cluster_read(box + idx, r) + cluster_read(box + BOX + idx, r) : box[idx] + box[BOX + idx];
    write_y(a, m, n, v);
  }
  if (split > 1) cluster_sync();  // nobody leaves while its sums are read
}

// K is split over a cluster so that the CTAs that run at once (clusters stay within a GPC, so larger ones fill the GPU less) have as
// few stages one after the other as can be.
int choose_split(const void* kern, int smem, int threads, int tiles, int mt, int stages, int* split) {
  static std::mutex lock;
  static std::map<std::pair<int, const void*>, std::array<int, 9>> known;
  int dev = 0;
  IB200_CUDA_OK(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> hold(lock);
  auto it = known.find({dev, kern});
  if (it == known.end()) {
    IB200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    std::array<int, 9> at_once{};
    for (int i = 1; i <= 8; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(i * 4 * kSmCount));
      cfg.blockDim = dim3((unsigned)threads);
      cfg.dynamicSmemBytes = (size_t)smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      IB200_CUDA_OK(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
      at_once[i] = clusters * i;
    }
    it = known.emplace(std::make_pair(dev, kern), at_once).first;
  }
  int64_t best = INT64_MAX;
  for (int i = 1; i <= 8 && (i == 1 || i <= stages); ++i) {
    if (it->second[i] <= 0) continue;
    const int64_t rounds = ((int64_t)tiles * mt * i + it->second[i] - 1) / it->second[i], cost = rounds * ((stages + i - 1) / i + 2);  // 2: begin and end
    if (cost < best) best = cost, *split = i;
  }
  return IB200_OK;
}

template <int XK, int NT, int G> int run_stream(W4Args a, cudaStream_t s) {
  auto* kern = w4_stream_kernel<XK, NT, G>;
  constexpr int SMEM = Stage<XK, NT, G>::SMEM;
  static_assert(SMEM <= 112 * 1024, "two CTAs per SM");
  const int tiles = (a.n + kRows - 1) / kRows, stages = (a.k + kStageK - 1) / kStageK, mt = (a.m + NT * 8 - 1) / (NT * 8);
  if (int rc = choose_split(reinterpret_cast<const void*>(kern), SMEM, kThreads, tiles, mt, stages, &a.split)) return rc;
  CUtensorMap map = {};
  if (a.k > 0)
    if (int rc = make_byte_map(&map, a.q, a.n, a.k / 2, kRows)) return rc;
  if ((int64_t)tiles * a.split > INT32_MAX || mt > 65535) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.split), (unsigned)mt);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  IB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, map));
  return IB200_OK;
}
template <int XK, int NT> int run_stream_group(const W4Args& a, cudaStream_t s) {
  if (a.group == 128) return run_stream<XK, NT, 128>(a, s);
  if (a.group == 64) return run_stream<XK, NT, 64>(a, s);
  return run_stream<XK, NT, 32>(a, s);
}
template <int XK> int run_stream_rows(const W4Args& a, cudaStream_t s) {
  return a.m <= 8 ? run_stream_group<XK, 1>(a, s) : run_stream_group<XK, 2>(a, s);
}

// ---- tensor memory ----------------------------------------------------------------------------------------
template <int N> __device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[N]);
template <> __device__ __forceinline__ void tmem_load<8>(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at) : "memory");
}
template <> __device__ __forceinline__ void tmem_load<16>(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at) : "memory");
}
template <> __device__ __forceinline__ void tmem_load<32>(uint32_t at, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(at) : "memory");
}
template <int N> __device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[N]);
template <> __device__ __forceinline__ void tmem_store<8>(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
template <> __device__ __forceinline__ void tmem_store<16>(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// K-major operand in shared memory, 128-byte swizzled rows, eight rows 1024 bytes apart
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t at) {
  return (uint64_t)((at & 0x3FFFF) >> 4) | (uint64_t)(16 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// ---- more rows of x: weights widened into tensor memory, tcgen05.mma ----------------------------------------
// D[128 rows of q, NX rows of x] per group of G, f32 in tensor memory:  A = the 128 x G widened weights (a thread widens its own
// row and stores it to tensor memory, where the MMA reads it), B = x from shared memory (128-byte swizzle, K-major).  The sums of a group are read back
// and scaled into f32 registers, one row to a thread, so nothing but x and q - z, both exact, enters the products.  A CTA has
// two such blocks of 128 rows, so that a stage of x (L2 -> SM traffic) serves 256 rows, and a slice of K; clusters split K as above.
//   warps 0-15  widen chunk i of their 32 rows (two warps to 32 rows, half of k each), then scale the sums of chunk i - 1, whose MMA ran
//               meanwhile (half of the columns each)
//   warp 16     brings the operands; x comes permuted and widened by a small launch in front, on which only x's copies wait
//   warps 17-18 one thread each issues the MMAs of a block
// Chunk i's widened weights arriving says that chunk i - 2 has been read back, so its buffers need no barrier of their own.
// 64 x 16384 x 8192, e4m3, groups of 128: 35.1 us (490 TFLOP/s; the weights' bytes alone 11 us).  The widening is most of it: its instructions take 56 % of the issue slots, the tensor
// cores are busy 27 % of the time, and 128 CTAs leave 20 of 148 SMs without work.  512 rows widen all weights eight times: 233 us (590 TFLOP/s).
// On mma.sync the product of 64 rows took 110 us; with eight widening warps 43, with scales fetched when they were needed 58.
constexpr int kTcRowScales = 100;  // a row's two blocks of eight scales, then of eight zero points' patterns; 25 words, so that rows lie in different banks
constexpr int kTcRows = 256, kTcThreads = 608;
template <int NX, int G> struct TcStage {
  static constexpr int GROUPS = kStageK / G;
  static constexpr int X_AT = kTcRows * kRowBytes;                        // after q: x as four [NX rows][64 k]
  static constexpr int XS_AT = X_AT + NX * kStageK * 2;                   // scales of x: [group][row]
  static constexpr int BYTES = (XS_AT + GROUPS * NX * 4 + 1023) / 1024 * 1024;
  static constexpr int kStages = 3;
  static constexpr int S_AT = kStages * BYTES, SMEM = S_AT + kTcRows * kTcRowScales;  // behind the stages: the rows' scales
};

// x as the MMA reads it: rows of k_pad 16-bit values, each eight in the order (0, 4, 1, 5, 2, 6, 3, 7), zero outside x
template <int XK> __global__ void __launch_bounds__(256) w4_spread_kernel(const W4Args a, uint4* out, int rows, int chunks) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int SIZE = XK >= X_E4M3 ? 1 : 2;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * chunks; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / chunks), k = (int)(i - (int64_t)row * chunks) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < a.m && k < a.k) {
      const uint8_t* p = static_cast<const uint8_t*>(a.x) + ((int64_t)row * a.x_stride + k) * SIZE;
      __align__(16) uint8_t e[16];
      if (a.x_vec) {
        if (SIZE == 2) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
        else *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (SIZE == 2) reinterpret_cast<uint16_t*>(e)[j] = reinterpret_cast<const uint16_t*>(p)[j];
          else e[j] = p[j];
        }
      }
      v = x_pairs<XK>(e);
    }
    out[i] = v;
  }
}

template <bool BF, int NX, int G>
__global__ void __launch_bounds__(kTcThreads, 1) w4_tc_kernel(const W4Args a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_x) {
  using S = TcStage<NX, G>;
  constexpr int GROUPS = S::GROUPS, kStages = S::kStages, NA = 256 / G, ND = 128 / NX;  // groups of a stage; buffers of A (128 columns a block) and D
  constexpr int A_AT = 256;                                                              // tensor memory: D of both blocks, then A of both
  constexpr int COLS = NX / 2, KS = G / 2;  // of a thread: columns of D that it scales, k of a chunk that it widens
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[kStages], empty[kStages], a_full[2][NA], d_full[2][ND];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int dead, brought;  // dead: a wait ran out, nothing waits any more; brought: stages in all
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (known to be the same for a warp)
  const int split = a.split, rank = blockIdx.x % split, n0 = (blockIdx.x / split) * kTcRows, m0 = blockIdx.y * NX;
  const int stages = (a.k + kStageK - 1) / kStageK, s0 = (int)((int64_t)stages * rank / split), s1 = (int)((int64_t)stages * (rank + 1) / split);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbarrier_try_wait(bar, parity) || dead || mbarrier_wait_bounded(bar, parity)) return;
    dead = 1;
    if (a.status) atomicCAS(a.status, 0, 8);
  };
  auto arrive = [](uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory"); };
  if (threadIdx.x == 0) {
    dead = 0;
    brought = s1 - s0;
    for (int i = 0; i < kStages; ++i) mbarrier_init(&full[i], 1 + 32), mbarrier_init(&empty[i], 16 + 2);
    for (int b = 0; b < 2; ++b) {
      for (int i = 0; i < NA; ++i) mbarrier_init(&a_full[b][i], 8);
      for (int i = 0; i < ND; ++i) mbarrier_init(&d_full[b][i], 1);
    }
    mbarrier_init_fence();
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  float sum[COLS];
#pragma unroll
  for (int j = 0; j < COLS; ++j) sum[j] = 0.0f;

  if (warp == 16) {
    // ---- the bringing warp ----------------------------------------------------------------------------------
    const uint32_t smem_at = smem_addr(smem);
    for (int s = s0; s < s1; ++s) {
      const int i = (s - s0) % kStages;
      if (s - s0 >= kStages) wait(&empty[i], ((s - s0) / kStages - 1) & 1);
      const uint32_t dst = smem_at + i * S::BYTES;
      if (lane == 0) {
        mbarrier_expect_tx(&full[i], kTcRows * kRowBytes + NX * kStageK * 2);
        tensor_copy(dst, &map_q, &full[i], s * kRowBytes, n0);
      }
      if (a.xs_groups > 1) {
        for (int e = lane; e < GROUPS * NX; e += 32) {
          const int m = m0 + e % NX, grp = s * GROUPS + e / NX;
          const bool take = m < a.m && grp < a.groups;
          copy4(dst + S::XS_AT + e * 4, a.xs + (take ? (int64_t)m * a.groups + grp : 0), take ? 4 : 0);
        }
      }
      if (lane == 0) {
        if (s == s0) asm volatile("griddepcontrol.wait;\nfence.proxy.async;" ::: "memory");  // the launch that spreads x
#pragma unroll
        for (int j = 0; j < kStageK / 64; ++j) tensor_copy(dst + S::X_AT + j * NX * 128, &map_x, &full[i], s * kStageK * 2 + j * 128, m0);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&full[i])) : "memory");
    }
  } else if (warp >= 17) {
    // ---- the MMA warps, one for each block of rows.  All lanes walk the loop, so that its values stay in uniform registers, and one issues: moved there
    // from one thread's registers they took 100 cycles an MMA, three times its own time.
    // f32 accumulators, both operands K-major, N = NX, M = 128
    constexpr uint32_t idesc = (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((uint32_t)(NX >> 3) << 17) | ((128u >> 4) << 24);
    const int b = warp - 17;
    uint32_t chosen;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(chosen));
    int i = 0;
    for (int s = s0; s < s1; ++s) {
      const int st = (s - s0) % kStages;
      wait(&full[st], ((s - s0) / kStages) & 1);
      const uint64_t x = swizzled_desc(smem_addr(smem) + st * S::BYTES + S::X_AT);
#pragma unroll
      for (int c = 0; c < GROUPS; ++c, ++i) {
        const uint32_t d = tmem + b * 128 + (i % ND) * NX, w = tmem + A_AT + b * 128 + (i % NA) * (G / 2);
        wait(&a_full[b][i % NA], (i / NA) & 1);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (chosen) {
#pragma unroll
          for (int k = 0; k < G / 16; ++k) {
            const int at = c * G + k * 16;  // k of the stage
            const uint64_t xk = x + ((at / 64 * (NX * 128) + at % 64 * 2) >> 4);
            if (k == 0)
              asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(w), "l"(xk), "r"(idesc) : "memory");
            else
              asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                           ::"r"(d), "r"(w + k * 8), "l"(xk), "r"(idesc) : "memory");
          }
          commit(&d_full[b][i % ND]);
        }
      }
      if (chosen) commit(&empty[st]);
      __syncwarp();
    }
  } else {
    // ---- widen and scale ------------------------------------------------------------------------------------
    const int b = warp >> 2 & 1, half = warp >> 3, row = b * 128 + (warp & 3) * 32 + lane;  // the thread's row of q is its lane of tensor memory
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, d_at = tmem + lanes + b * 128 + half * COLS, a_at = tmem + lanes + A_AT + b * 128 + half * (KS / 2);
    uint8_t* scales = smem + S::S_AT + row * kTcRowScales;
    int block = s0 * GROUPS >> 3;
    RowBlock ahead = read_block(a, half, n0 + row, block);
    auto next_block = [&] {
      uint32_t* to = reinterpret_cast<uint32_t*>(scales + (half ? 64 + (block & 1) * 16 : (block & 1) * 32));
      if (half) {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = pattern16_of<BF>(zero_byte(a, ahead, 2 * e)) | pattern16_of<BF>(zero_byte(a, ahead, 2 * e + 1)) << 16;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = __float_as_uint(scale_of(a, ahead, e));
      }
      ahead = read_block(a, half, n0 + row, block + 1);
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 7)) : "memory");
    };
    next_block();
    uint32_t magic = BF ? 0x43004300u : 0x64006400u;
    asm volatile("" : "+r"(magic));  // (kept in a register)
    const Zero eight = zero_of<BF>(pattern_of<BF>(8));
    const bool xs_many = a.xs_groups > 1;
    int i = 0, old_group = 0;
    float old_scale = 0.0f;
    const uint8_t* old_stage = smem;
    auto scale_sums = [&](int j) {  // chunk j's
      wait(&d_full[b][j % ND], (j / ND) & 1);
      __syncwarp();  // (the loads below are the whole warp's)
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint32_t r[COLS];
      tmem_load<COLS>(d_at + (j % ND) * NX, r);
      if (xs_many) {
        const float4* f = reinterpret_cast<const float4*>(old_stage + S::XS_AT + (old_group * NX + half * COLS) * 4);
#pragma unroll
        for (int e = 0; e < COLS; e += 4) {
          const float4 v = f[e / 4];
          sum[e] = fmaf(__uint_as_float(r[e]), old_scale * v.x, sum[e]);
          sum[e + 1] = fmaf(__uint_as_float(r[e + 1]), old_scale * v.y, sum[e + 1]);
          sum[e + 2] = fmaf(__uint_as_float(r[e + 2]), old_scale * v.z, sum[e + 2]);
          sum[e + 3] = fmaf(__uint_as_float(r[e + 3]), old_scale * v.w, sum[e + 3]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < COLS; ++e) sum[e] = fmaf(__uint_as_float(r[e]), old_scale, sum[e]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    };
    for (int s = s0; s < s1; ++s) {
      const uint8_t* st = smem + (s - s0) % kStages * S::BYTES;
      wait(&full[(s - s0) % kStages], ((s - s0) / kStages) & 1);
      __syncwarp();
      if (s * GROUPS >> 3 != block) {
        block = s * GROUPS >> 3;
        next_block();
      }
      // the row's bytes of the stage, chunks swizzled by row % 8: both the chunk and the half only flip address bits
      const uint32_t row_at = (smem_addr(smem) + (uint32_t)((s - s0) % kStages * S::BYTES + row * kRowBytes)) ^ (uint32_t)((row & 7) << 4) ^ (uint32_t)(half * (KS / 2));
      const float* scales_of = reinterpret_cast<const float*>(scales + (block & 1) * 32) + (s * GROUPS & 7);
      const uint16_t* zeros_of = reinterpret_cast<const uint16_t*>(scales + 64 + (block & 1) * 16) + (s * GROUPS & 7);
#pragma unroll
      for (int c = 0; c < GROUPS; ++c, ++i) {
        const Zero zero = a.z ? zero_of<BF>(both_halves(zeros_of[c])) : eight;
        const float scale = scales_of[c];
        constexpr int WORDS = KS >= 32 ? 4 : 2;  // of q a time
#pragma unroll
        for (int q = 0; q < KS / (8 * WORDS); ++q) {
          uint32_t w[4], r[4 * WORDS];
          const uint32_t p = row_at ^ (uint32_t)(c * (G / 2) + q * 16);
          if (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(p) : "memory");
          else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(p) : "memory");
#pragma unroll
          for (int k = 0; k < WORDS; ++k) {
            uint32_t pairs[4];
            weights_of<BF>(w[k], zero, magic, pairs);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[4 * k + e] = pairs[e];
          }
          tmem_store<4 * WORDS>(a_at + (i % NA) * (G / 2) + q * 16, r);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(&a_full[b][i % NA]);
        if (i > 0) scale_sums(i - 1);
        if (c == 0 && s > s0) {
          __syncwarp();
          if (lane == 0) arrive(&empty[(s - 1 - s0) % kStages]);
        }
        old_scale = scale;
        old_stage = st;
        old_group = c;
      }
    }
    if (i > 0) scale_sums(i - 1);
  }

  // ---- add up the cluster's slices and write ----------------------------------------------------------------
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (dead) {  // whichever warp gave up: copies and products that are still on their way end before their memory is used again or freed
    bool ended = true;
    const int n = brought, chunks = n * GROUPS;
    for (int s = max(0, n - kStages); s < n; ++s) ended = ended && mbarrier_wait_bounded(&full[s % kStages], (s / kStages) & 1);
    for (int b = 0; b < 2; ++b)
      for (int i = max(0, chunks - ND); i < chunks; ++i) ended = ended && mbarrier_wait_bounded(&d_full[b][i % ND], (i / ND) & 1);
  }
  if (warp == 17) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  float* box = reinterpret_cast<float*>(smem);  // [NX][256] sums of this CTA
  if (warp < 16) {
#pragma unroll
    for (int j = 0; j < COLS; ++j) box[((warp >> 3) * COLS + j) * kTcRows + threadIdx.x % kTcRows] = sum[j];
  }
  if (split > 1) cluster_sync(); else __syncthreads();
  const int rows = min(NX, a.m - m0);
  for (int idx = rank * kTcThreads + threadIdx.x; idx < rows * kTcRows; idx += split * kTcThreads) {
    const int m = m0 + idx / kTcRows, n = n0 + idx % kTcRows;
    float v = 0.0f;
    for (int r = 0; r < split; ++r) v += split > 1 ? cluster_read(box + idx, r) : box[idx];
    write_y(a, m, n, v);
  }
  if (split > 1) cluster_sync();
}

int64_t padded(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int tc_columns(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

template <int XK, int NX, int G> int run_tc(W4Args a, void* scratch, cudaStream_t s) {
  constexpr bool BF = XK == X_BF16;
  auto* kern = w4_tc_kernel<BF, NX, G>;
  constexpr int SMEM = TcStage<NX, G>::SMEM;
  static_assert(SMEM <= 226 * 1024, "one CTA per SM");
  const int64_t rows = padded(a.m, NX), k_pad = padded(a.k, kStageK);
  CUtensorMap map_q, map_x;
  if (int rc = make_byte_map(&map_q, a.q, a.n, a.k / 2, kTcRows)) return rc;
  if (int rc = make_byte_map(&map_x, scratch, rows, k_pad * 2, NX)) return rc;
  const int tiles = (a.n + kTcRows - 1) / kTcRows, mt = (int)(rows / NX);
  if (mt > 65535) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: too many rows");
  if (int rc = choose_split(reinterpret_cast<const void*>(kern), SMEM, kTcThreads, tiles, mt, (int)(k_pad / kStageK), &a.split)) return rc;
  const int64_t blocks = (rows * (k_pad / 8) + 255) / 256;
  w4_spread_kernel<XK><<<(unsigned)(blocks < kSmCount * 8 ? blocks : kSmCount * 8), 256, 0, s>>>(a, static_cast<uint4*>(scratch), (int)rows, (int)(k_pad / 8));
  if (cudaPeekAtLastError() != cudaSuccess) return cuda_fail(cudaGetLastError(), "w4_matmul launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.split), (unsigned)mt);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  IB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, map_q, map_x));
  return IB200_OK;
}
template <int XK, int NX> int run_tc_group(const W4Args& a, void* scratch, cudaStream_t s) {
  if (a.group == 128) return run_tc<XK, NX, 128>(a, scratch, s);
  if (a.group == 64) return run_tc<XK, NX, 64>(a, scratch, s);
  return run_tc<XK, NX, 32>(a, scratch, s);
}
template <int XK> int run_tc_rows(const W4Args& a, void* scratch, cudaStream_t s) {
  const int nx = tc_columns(a.m);
  if (nx == 16) return run_tc_group<XK, 16>(a, scratch, s);
  return nx == 32 ? run_tc_group<XK, 32>(a, scratch, s) : run_tc_group<XK, 64>(a, scratch, s);
}

}  // namespace

// Which kernel: up to 8 rows of x the weights stream into mma.sync (bf16, groups of 128: one row of 8192 x 8192 14.8 us against 16.6 through tensor memory, 4096 x 4096 6.4 against
// 9.8; eight rows 16.2 / 17.1 and 7.0 / 10.2), above 16 they go through tensor memory.  Between, mma.sync takes two column tiles; 12 and 16 rows of square matrices:
//   groups of 128: 4096 8.8 / 10.4 and 9.1 / 11.1 us, 5760 12.8 / 13.3 and 13.9 / 13.4, 8192 20.5 / 17.6 and 21.0 / 17.5
//   groups of 64:  4096 9.2 / 11.3 and 9.7 / 12.0 us, 5760 14.6 / 15.4 and 15.9 / 15.7, 8192 22.5 / 20.3 and 22.9 / 20.4 (streamed: a rule for them would gain 10 % there)
//   groups of 32, whose sums come back four times as often: 4096 10.3 / 14.1 us, 8192 25.8 / 28.5
// The sides meet between 2^25 and 2^26 weights; 2^26 is the first size measured where tensor memory wins for 12 rows and 16 alike.
static bool through_tensor_memory(int64_t m, int64_t n, int64_t k, int64_t group) {
  return k > 0 && (m > 16 || (m > 8 && group == 128 && n * k >= (int64_t)1 << 26));
}
constexpr int64_t kTcMostK = (int64_t)1 << 30;  // the copies of x count bytes in 32 bits, two to a value

// room for x as the MMA reads it
size_t w4_scratch_bytes(int, int64_t m, int64_t n, int64_t k, int64_t group) {
  if (m <= 0 || n <= 0 || k <= 0 || beyond_any_device(m, k) || beyond_any_device(n, k) || k > kTcMostK || !through_tensor_memory(m, n, k, group)) return 0;
  return (size_t)(padded(m, tc_columns(m)) * padded(k, kStageK) * 2);
}

int launch_w4(const void* x, int64_t x_stride, const float* xs, int64_t xs_groups, const void* q, const void* scales, const void* zeros,
              const void* bias, void* y, int x_dtype, int s_dtype, int out_dtype, int64_t m, int64_t n, int64_t k, int64_t group,
              void* scratch, size_t scratch_bytes, int32_t* status, cudaStream_t s) {
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
  if ((held ? xs_groups == 0 && groups != 0 : xs_groups != 0) || (xs_groups != 0 && xs_groups != 1 && xs_groups != groups))
    return fail(IB200_ERR_INVALID, "w4_matmul: 8-bit x comes with one scale per row or one per row and group, other x with none");
  if (m == 0 || n == 0) return IB200_OK;
  if (!y || (xs_groups && !xs) || (k > 0 && (!x || !q || !scales))) return fail(IB200_ERR_INVALID, "w4_matmul: null operand");
  if (!aligned16(q)) return fail(IB200_ERR_INVALID, "w4_matmul: q must be 16-byte aligned");
  if (m > 1 && (x_stride < k || beyond_any_device(m, x_stride > 0 ? x_stride : 1))) return fail(IB200_ERR_INVALID, "w4_matmul: bad row stride of x");
  const int e = held ? 1 : 2;
  const bool x_vec = (reinterpret_cast<uintptr_t>(x) & (held ? 7 : 15)) == 0 && (m == 1 || x_stride * e % (held ? 8 : 16) == 0);
  W4Args a{x, static_cast<const uint8_t*>(q), scales, static_cast<const uint8_t*>(zeros), bias, xs, y, x_stride,
           (int)m, (int)n, (int)k, (int)group, (int)groups, (int)xs_groups, x_dtype, s_dtype, out_dtype, x_vec, 0, 0, 1, status};
  a.s_vec = groups % 8 == 0 && aligned16(scales);
  a.z_vec = zeros && groups % 8 == 0 && (reinterpret_cast<uintptr_t>(zeros) & 7) == 0;
  if (through_tensor_memory(m, n, k, group)) {
    if (k > kTcMostK) return fail(IB200_ERR_UNSUPPORTED, "w4_matmul: more than 16 rows of x (8 in groups of 128) take K up to 2^30");
    if (!scratch || scratch_bytes < w4_scratch_bytes(x_dtype, m, n, k, group)) return fail(IB200_ERR_BUFFER, "w4_matmul: scratch is smaller than ib200_w4_scratch_bytes");
    if (x_dtype == IB200_BF16) return run_tc_rows<X_BF16>(a, scratch, s);
    if (x_dtype == IB200_F16) return run_tc_rows<X_F16>(a, scratch, s);
    return x_dtype == IB200_E4M3 ? run_tc_rows<X_E4M3>(a, scratch, s) : run_tc_rows<X_I8>(a, scratch, s);
  }
  if (x_dtype == IB200_BF16) return run_stream_rows<X_BF16>(a, s);
  if (x_dtype == IB200_F16) return run_stream_rows<X_F16>(a, s);
  return x_dtype == IB200_E4M3 ? run_stream_rows<X_E4M3>(a, s) : run_stream_rows<X_I8>(a, s);
}

}  // namespace ib200
