// A paged key / value cache held in 8 bits: its layout, and the append (kv8_attention.cu has the attention).
//   cache  [pages, heads, block, D] of e4m3 or int8, scale [pages, heads] f32: a value stands for cache * scale
//   table  [sequences, blocks per sequence]: the page that holds a sequence's tokens i * block .. i * block + block - 1
//   lens   [sequences]: tokens of each sequence, the new ones among them
//   cu     [sequences + 1]: where each sequence's new tokens lie in k, v, q and o (null: the same number for every sequence)
// What a table says is not trusted: a page outside the cache, and a token outside the table, is never read or written.  The
// append leaves such tokens out, attention that would have to read them answers NaN.
#include <type_traits>

#include "kv8.cuh"

namespace ib200 {
namespace {

// ---- append -----------------------------------------------------------------------------------------
// A unit is the new tokens of one block: for a head, one warp for the keys and one for the values (few tokens), or one CTA for both.
//   s' = max(s, max|new| * (1 / Q)), s = 0 for a block that begins here; held values become round(q * s / s') where s' > s, new ones round(x / s')
// Quotients round as IEEE divisions do: the held values depend on nothing but their definition.  The new values are read once
// into registers (up to KEEP vectors of 8 a thread: 16 tokens of 128 in a warp, 64 in a CTA; more are read again) and written 8 bytes at a time.
// Bound by instruction issue (77 % of the slots) and the chain length -> table -> scale in front of each CTA: 30 000 tokens of 8 heads of 128,
// f16 -> int8, blocks of 64, take 46 us (4.1 TB/s) where the bytes alone would take 29; 128 sequences x 1 token 3.3 us.  One CTA for keys and values
// saves a chain (57 -> 52 us; a warp that did both would take 4.2 instead of 3.3); 64 registers a thread let four CTAs share an SM (52 -> 46; five spill: 62).
template <typename T> __device__ __forceinline__ uint4 read_new(const T* p, bool vec) {
  if (vec) return __ldcs(reinterpret_cast<const uint4*>(p));
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  return make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
}
template <typename T> __device__ __forceinline__ void floats_of(const uint4& r, float (&v)[8]) {
  const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(p[i]);
}
// round(v / div) of eight values to the held type.  v * (1 / div) is within 2 ulp of the f32 quotient, so it rounds alike unless it lies that close to
// the middle between two held values (or, in e4m3, in the subnormals, whose middles lie elsewhere).  One test over the eight finds that, one vector in some
// thousand is divided; all are where 1 / div overflows, and those with a NaN.
template <typename T, int HELD> __device__ __noinline__ uint2 hold_divided(uint4 r, float div) {
  float v[8];
  floats_of<T>(r, v);
  return make_uint2(hold4<HELD>(v[0] / div, v[1] / div, v[2] / div, v[3] / div), hold4<HELD>(v[4] / div, v[5] / div, v[6] / div, v[7] / div));
}
template <typename T, int HELD> __device__ __forceinline__ uint2 hold_quotients(const uint4& r, float div, float inv) {
  float v[8];
  floats_of<T>(r, v);
  float q[8], whole[8], least = INFINITY, most = 0.0f;
  int nearest = INT32_MAX;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = v[i] * inv;
    if (HELD == HELD_E4M3) {  // 3 of 23 mantissa bits stay: the other 20, as a signed distance from their middle
      nearest = min(nearest, abs((int)(__float_as_uint(q[i]) * 4096u + 0x80000000u)));
      least = fminf(least, fabsf(q[i]));
    } else {  // |q| < 2^7, so 2 ulp are 2^-16; the sum's low byte is round(q)
      whole[i] = q[i] + 0x1.8p23f;
      most = fmaxf(most, fabsf(q[i] - (whole[i] - 0x1.8p23f)));
    }
  }
  const bool sure = (HELD == HELD_E4M3 ? nearest > 16 * 4096 && least >= 0x1.01p-6f : most < 0.49998f) && inv > 0.0f && inv <= 0x1p127f;
  if (!sure) return hold_divided<T, HELD>(r, div);
  if (HELD == HELD_I8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __byte_perm(__float_as_uint(whole[2 * i]), __float_as_uint(whole[2 * i + 1]), 0x0040);
    return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
  }
  return make_uint2(hold4<HELD>(q[0], q[1], q[2], q[3]), hold4<HELD>(q[4], q[5], q[6], q[7]));
}

template <typename T, int HELD, int D, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 32 ? 1 : 4) append_kernel(const Kv8Append a, const int vec) {
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  constexpr int PER = D / 8, KEEP = THREADS == 32 ? 8 : 4, SIDES = THREADS == 32 ? 1 : 2;  // vectors of a token, of a thread; keys and values
  __shared__ float slots[SIDES][THREADS / 32];
  const int head = blockIdx.y, tid = threadIdx.x, block = (int)a.block;
  // Unit u: with offsets, sequence b has the units from cu[b] / block + 2 b, which leaves room for (its new tokens) / block + 2; without,
  // the same number for each.
  const int u = (int)blockIdx.x;
  int b, first, count, j;
  if (a.cu) {
    int lo = 0, hi = (int)a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] / block + 2 * (int64_t)mid <= u) lo = mid; else hi = mid;
    }
    b = lo;
    first = a.cu[b];
    count = a.cu[b + 1] - first;
    j = (int)(u - (first / block + 2 * (int64_t)b));
    if (first < 0 || count <= 0 || j < 0 || (int64_t)first + count > a.tokens) return;
  } else {
    b = u / a.per;
    j = u - b * a.per;
    first = b * a.each;
    count = a.each;
  }
  const int end = a.lens[b], start = max(end, -1) - count;  // places of the new tokens: start .. end - 1; those below 0 have none
  const int64_t blk = max(0, start) / block + j;
  const int from = (int)max((int64_t)max(0, start), min(blk * block, (int64_t)INT32_MAX)), to = (int)min((int64_t)end, (blk + 1) * block);
  if (from >= to || blk >= a.table_blocks) return;
  const int page = a.table[(int64_t)b * a.table_blocks + blk];  // (looked at when the new values are on their way)
  const int slot = (int)(from - blk * block), vectors = (to - from) * PER;
  // vector k of a thread: THREADS / PER tokens behind the one before
  const T* mine[SIDES];
  int64_t next[SIDES];
  uint4 keep[SIDES][KEEP];
  bool is_v[SIDES];
#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    is_v[s] = SIDES == 2 ? s : blockIdx.z;
    const int64_t token = is_v[s] ? a.v_token : a.k_token;
    mine[s] = static_cast<const T*>(is_v[s] ? a.v : a.k) + (int64_t)(first + (from - start) + tid / PER) * token + (int64_t)head * (is_v[s] ? a.v_head : a.k_head) + tid % PER * 8;
    next[s] = THREADS / PER * token;
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (tid + k * THREADS < vectors) keep[s][k] = read_new(mine[s] + k * next[s], vec);
  }
  if ((unsigned)page >= (unsigned)a.pages) return;
  const int64_t at = (int64_t)page * a.heads + head;
  float *scales[SIDES], before[SIDES], top[SIDES];
#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    scales[s] = (is_v[s] ? a.v_scale : a.k_scale) + at;
    before[s] = slot ? *scales[s] : 0.0f;
  }

#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    Pair largest = {};  // two values at a time, in their own type
    auto enter = [&](const uint4& r) {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t size = w[e] & 0x7fff7fffu;
        largest = __hmax2_nan(largest, *reinterpret_cast<const Pair*>(&size));
      }
    };
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (tid + k * THREADS < vectors) enter(keep[s][k]);
    for (int k = KEEP; tid + k * THREADS < vectors; ++k) enter(read_new(mine[s] + k * next[s], vec));
    top[s] = warp_reduce<MaxOp>(max_nan(to_f32(largest.x), to_f32(largest.y)));
  }
  if (THREADS == 32) {
    __syncwarp();  // every lane has read the old scales
  } else {
    if ((tid & 31) == 0)
      for (int s = 0; s < SIDES; ++s) slots[s][tid >> 5] = top[s];
    __syncthreads();
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      top[s] = slots[s][0];
#pragma unroll
      for (int i = 1; i < THREADS / 32; ++i) top[s] = max_nan(top[s], slots[s][i]);
    }
  }
#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    uint8_t* cache = (is_v[s] ? a.v_cache : a.k_cache) + at * block * D;
    const float after = max_nan(before[s], top[s] * held_unit<HELD>()), div = after == 0.0f ? 1.0f : after, inv = 1.0f / div;
    if (tid == 0) *scales[s] = after;
    if (!(after == before[s])) {
      for (int i = tid; i < slot * PER; i += THREADS) {
        const uint2 old = *reinterpret_cast<const uint2*>(cache + i * 8);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = held_value<HELD>((uint8_t)((e < 4 ? old.x : old.y) >> (8 * (e & 3)))) * before[s] / div;
        *reinterpret_cast<uint2*>(cache + i * 8) = make_uint2(hold4<HELD>(v[0], v[1], v[2], v[3]), hold4<HELD>(v[4], v[5], v[6], v[7]));
      }
    }
    uint8_t* out = cache + slot * D + tid * 8;
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (tid + k * THREADS < vectors) *reinterpret_cast<uint2*>(out + k * THREADS * 8) = hold_quotients<T, HELD>(keep[s][k], div, inv);
    for (int k = KEEP; tid + k * THREADS < vectors; ++k)
      *reinterpret_cast<uint2*>(out + k * THREADS * 8) = hold_quotients<T, HELD>(read_new(mine[s] + k * next[s], vec), div, inv);
  }
}

template <typename T, int HELD, int D> int run_append(const Kv8Append& a, cudaStream_t s) {
  const int64_t units = a.cu ? a.tokens / a.block + 2 * a.batch + 1 : a.batch * a.per;
  if (units > INT32_MAX) return fail(IB200_ERR_UNSUPPORTED, "kv8_append: too many blocks");
  const int vec = aligned16(a.k) && aligned16(a.v) && a.k_token % 8 == 0 && a.k_head % 8 == 0 && a.v_token % 8 == 0 && a.v_head % 8 == 0;
  // a warp holds 16 tokens of 128 in its registers; where a block takes more, a CTA.  128 sequences x 1 token 3.4 / 8.1 us by a warp / a CTA, x 8 6.0 / 9.3,
  // x 16 9.2 / 10.9, x 32 16.6 / 13.1, blocks of 64 filled by long sequences 127 / 46
  const int64_t expect = (a.tokens + a.batch - 1) / a.batch;
  if ((expect < a.block ? expect : a.block) * D <= 16 * 128) append_kernel<T, HELD, D, 32><<<dim3((unsigned)units, (unsigned)a.heads, 2), 32, 0, s>>>(a, vec);
  else append_kernel<T, HELD, D, 256><<<dim3((unsigned)units, (unsigned)a.heads), 256, 0, s>>>(a, vec);
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "kv8_append launch");
}
template <typename T, int HELD> int run_append_dim(const Kv8Append& a, cudaStream_t s) {
  return a.dim == 128 ? run_append<T, HELD, 128>(a, s) : run_append<T, HELD, 64>(a, s);
}

}  // namespace

int check_kv8(const char* what, int64_t pages, int64_t heads, int64_t block, int64_t dim, int64_t batch, int64_t table_blocks, int64_t tokens,
                int held, int dtype, const int* cu) {
  const std::string w(what);
  if (pages < 0 || heads < 0 || batch < 0 || table_blocks < 0 || tokens < 0) return fail(IB200_ERR_INVALID, w + ": negative extent");
  if (held != IB200_E4M3 && held != IB200_I8) return fail(IB200_ERR_UNSUPPORTED, w + ": the cache must be e4m3 or int8");
  if (dtype != IB200_BF16 && dtype != IB200_F16) return fail(IB200_ERR_UNSUPPORTED, w + ": new values must be bf16 or f16");
  if (dim != 64 && dim != 128) return fail(IB200_ERR_UNSUPPORTED, w + ": head widths of 64 and 128");
  if (block < 16 || block > 1024 || block % 16) return fail(IB200_ERR_UNSUPPORTED, w + ": blocks of 16, 32, .. 1024 tokens");
  if (heads > 65535 || pages > INT32_MAX || tokens > INT32_MAX - 65536 || batch > INT32_MAX - 65536) return fail(IB200_ERR_UNSUPPORTED, w + ": extents are below 2^31 (heads: 2^16)");
  if (beyond_any_device(pages, heads, block * dim) || beyond_any_device(batch, table_blocks) || table_blocks * block > INT32_MAX)
    return fail(IB200_ERR_INVALID, w + ": extents beyond any device (or sequences of 2^31 tokens)");
  if (!cu && (batch > 0 ? tokens % batch != 0 : tokens > 0)) return fail(IB200_ERR_INVALID, w + ": without offsets every sequence has the same number of new tokens");
  return IB200_OK;
}

int launch_kv8_append(Kv8Append& a, int dtype, int held, cudaStream_t s) {
  if (int rc = check_kv8("kv8_append", a.pages, a.heads, a.block, a.dim, a.batch, a.table_blocks, a.tokens, held, dtype, a.cu)) return rc;
  if (a.tokens == 0 || a.heads == 0 || a.batch == 0 || a.pages == 0 || a.table_blocks == 0) return IB200_OK;
  if (!a.k || !a.v || !a.k_cache || !a.v_cache || !a.k_scale || !a.v_scale || !a.table || !a.lens) return fail(IB200_ERR_INVALID, "kv8_append: null operand");
  if (!aligned16(a.k_cache) || !aligned16(a.v_cache)) return fail(IB200_ERR_INVALID, "kv8_append: caches must be 16-byte aligned");
  a.each = (int)(a.tokens / a.batch);
  a.per = (int)((a.each + a.block - 2) / a.block + 1);
  if (dtype == IB200_BF16) return held == IB200_E4M3 ? run_append_dim<__nv_bfloat16, HELD_E4M3>(a, s) : run_append_dim<__nv_bfloat16, HELD_I8>(a, s);
  return held == IB200_E4M3 ? run_append_dim<__half, HELD_E4M3>(a, s) : run_append_dim<__half, HELD_I8>(a, s);
}

}  // namespace ib200
