// A paged key / value cache held in 8 bits, and attention over it.
//   cache  [pages, heads, block, D] of e4m3 or int8, scale [pages, heads] f32: a value stands for cache * scale
//   table  [sequences, blocks per sequence]: the page that holds a sequence's tokens i * block .. i * block + block - 1
//   lens   [sequences]: tokens of each sequence, the new ones among them
//   cu     [sequences + 1]: where each sequence's new tokens lie in k, v, q and o (null: the same number for every sequence)
// What a table says is not trusted: a page outside the cache, and a token outside the table, is never read or written.  The
// append leaves such tokens out, attention that would have to read them answers NaN.
#include "common.cuh"
#include "held8.cuh"
#include "kv8.h"

namespace ib200 {
namespace {

// The sequence whose new tokens include token t, its first new token and their number; false for a token behind (or before) all of them.
__device__ __forceinline__ bool find_sequence(const int* cu, int batch, int each, int t, int& b, int& first, int& count) {
  if (!cu) {
    b = t / each;
    first = b * each;
    count = each;
    return b < batch;
  }
  int lo = 0, hi = batch;  // the largest b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  b = lo;
  first = cu[b];
  const int end = cu[b + 1];
  count = end - first;
  return batch > 0 && first >= 0 && first <= t && t < end;
}

// ---- append -----------------------------------------------------------------------------------------
// One CTA per (new token, head, K or V); the CTA of a block's first new token does the whole block, the others leave at once.
//   s' = max(s, max|new| / Q), s = 0 for a block that begins here; held values become round(q * s / s') where s' > s, new ones round(x / s')
// Divisions are IEEE divisions: the held values then depend on nothing but their definition.
template <typename T, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS) append_kernel(const Kv8Append a) {
  __shared__ float slots[32];
  const int t = blockIdx.x, head = blockIdx.y;
  int b, first, count;
  if (!find_sequence(a.cu, a.batch, a.each, t, b, first, count)) return;
  const int64_t start = (int64_t)a.lens[b] - count, pos = start + (t - first);
  if (pos < 0) return;
  const int64_t blk = pos / a.block;
  const int slot = (int)(pos - blk * a.block);
  if (!(t == first || slot == 0 || pos == 0) || blk >= a.table_blocks) return;
  const int page = a.table[(int64_t)b * a.table_blocks + blk];
  if ((unsigned)page >= (unsigned)a.pages) return;
  const int fresh = (int)min(min((int64_t)first + count, a.tokens) - t, (int64_t)(a.block - slot));  // new tokens of this block
  const bool is_v = blockIdx.z;
  const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (int64_t)t * (is_v ? a.v_token : a.k_token) + (int64_t)head * (is_v ? a.v_head : a.k_head);
  const int64_t x_token = is_v ? a.v_token : a.k_token;
  const int64_t at = (int64_t)page * a.heads + head;
  uint8_t* cache = (is_v ? a.v_cache : a.k_cache) + at * a.block * a.dim;
  float* scale = (is_v ? a.v_scale : a.k_scale) + at;
  float top = 0.0f;
  for (int i = threadIdx.x; i < fresh * a.dim; i += THREADS) top = max_nan(top, fabsf(to_f32(x[(i / a.dim) * x_token + i % a.dim])));
  top = block_reduce<MaxOp>(top, slots);
  const float before = slot ? *scale : 0.0f;
  const float after = max_nan(before, top / held_top<HELD>());
  const bool grown = !(after == before);
  const float div = after == 0.0f ? 1.0f : after;
  if (grown)
    for (int i = threadIdx.x; i < slot * a.dim; i += THREADS) cache[i] = (uint8_t)hold1<HELD>(held_value<HELD>(cache[i]) * before / div);
  for (int i = threadIdx.x; i < fresh * a.dim; i += THREADS)
    cache[slot * a.dim + i] = (uint8_t)hold1<HELD>(to_f32(x[(i / a.dim) * x_token + i % a.dim]) / div);
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = after;
}

// ---- attention --------------------------------------------------------------------------------------
// One warp per (new token, query head), 32 keys a step.
template <typename T, int HELD>
__global__ void __launch_bounds__(128) attention_warp_kernel(const Kv8Attention a) {
  __shared__ float qs[4][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * 4 + warp;
  if (u >= (int64_t)a.tokens * a.q_heads) return;
  const int t = (int)(u / a.q_heads), qh = (int)(u % a.q_heads), head = qh / (a.q_heads / a.heads);
  int b, first, count;
  if (!find_sequence(a.cu, a.batch, a.each, t, b, first, count)) return;
  const int64_t pos = (int64_t)a.lens[b] - count + (t - first);
  const int64_t lo = a.window > 0 ? max((int64_t)0, pos - a.window + 1) : 0;
  const T* q = static_cast<const T*>(a.q) + (int64_t)t * a.q_token + (int64_t)qh * a.q_head;
  for (int d = lane; d < a.dim; d += 32) qs[warp][d] = to_f32(q[d]) * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int64_t base = lo; base <= pos; base += 32) {
    const int64_t key = base + lane;
    float s = -INFINITY;
    int64_t row = -1;
    float vs = 0.0f;
    if (key <= pos) {
      const int64_t blk = key / a.block;
      const int page = blk < a.table_blocks ? a.table[(int64_t)b * a.table_blocks + blk] : -1;
      if ((unsigned)page < (unsigned)a.pages) {
        const int64_t at = (int64_t)page * a.heads + head;
        row = (at * a.block + key % a.block) * a.dim;
        s = 0.0f;
        for (int d = 0; d < a.dim; ++d) s = fmaf(qs[warp][d], held_value<HELD>(a.k_cache[row + d]), s);
        s *= a.k_scale[at];
        vs = a.v_scale[at];
      } else {
        s = NAN;
      }
    }
    const float top = max_nan(m, warp_reduce<MaxOp>(s));
    const float p = s == -INFINITY && key > pos ? 0.0f : expf(s - top);
    const float keep = m == -INFINITY ? 0.0f : expf(m - top);
    l = l * keep + warp_reduce<SumOp>(p);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= keep;
    const float pv = p * vs;
    for (int j = 0; j < 32; ++j) {
      const int64_t r = __shfl_sync(0xffffffffu, row, j);
      const float w = __shfl_sync(0xffffffffu, pv, j);
      if (r < 0) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.dim) o[i] = fmaf(w, held_value<HELD>(a.v_cache[r + lane + 32 * i]), o[i]);
    }
  }
  const int64_t out = (int64_t)t * a.q_heads + qh;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < a.dim) static_cast<T*>(a.o)[out * a.dim + lane + 32 * i] = from_f32<T>(pos < 0 ? 0.0f : o[i] / l);
  if (lane == 0 && a.lse) a.lse[out] = pos < 0 ? -INFINITY : m + logf(l);
}

bool held_type(int t) { return t == IB200_E4M3 || t == IB200_I8; }

int check_cache(const char* what, int64_t pages, int64_t heads, int64_t block, int64_t dim, int64_t batch, int64_t table_blocks, int64_t tokens,
                int held, int dtype, const int* cu) {
  const std::string w(what);
  if (pages < 0 || heads < 0 || batch < 0 || table_blocks < 0 || tokens < 0) return fail(IB200_ERR_INVALID, w + ": negative extent");
  if (!held_type(held)) return fail(IB200_ERR_UNSUPPORTED, w + ": the cache must be e4m3 or int8");
  if (dtype != IB200_BF16 && dtype != IB200_F16) return fail(IB200_ERR_UNSUPPORTED, w + ": new values must be bf16 or f16");
  if (dim != 64 && dim != 128) return fail(IB200_ERR_UNSUPPORTED, w + ": head widths of 64 and 128");
  if (block < 16 || block > 1024 || block % 16) return fail(IB200_ERR_UNSUPPORTED, w + ": blocks of 16, 32, .. 1024 tokens");
  if (heads > 65535 || pages > INT32_MAX || tokens > INT32_MAX - 65536 || batch > INT32_MAX - 65536) return fail(IB200_ERR_UNSUPPORTED, w + ": extents are below 2^31 (heads: 2^16)");
  if (beyond_any_device(pages, heads, block * dim) || beyond_any_device(batch, table_blocks) || table_blocks * block > INT32_MAX)
    return fail(IB200_ERR_INVALID, w + ": extents beyond any device (or sequences of 2^31 tokens)");
  if (!cu && batch > 0 && tokens % batch) return fail(IB200_ERR_INVALID, w + ": without offsets every sequence has the same number of new tokens");
  return IB200_OK;
}

}  // namespace

int launch_kv8_append(Kv8Append& a, int dtype, int held, cudaStream_t s) {
  if (int rc = check_cache("kv8_append", a.pages, a.heads, a.block, a.dim, a.batch, a.table_blocks, a.tokens, held, dtype, a.cu)) return rc;
  if (a.tokens == 0 || a.heads == 0 || a.batch == 0 || a.pages == 0 || a.table_blocks == 0) return IB200_OK;
  if (!a.k || !a.v || !a.k_cache || !a.v_cache || !a.k_scale || !a.v_scale || !a.table || !a.lens) return fail(IB200_ERR_INVALID, "kv8_append: null operand");
  if (!aligned16(a.k_cache) || !aligned16(a.v_cache)) return fail(IB200_ERR_INVALID, "kv8_append: caches must be 16-byte aligned");
  a.each = (int)(a.tokens / a.batch);
  const dim3 grid((unsigned)a.tokens, (unsigned)a.heads, 2);
  if (dtype == IB200_BF16) {
    if (held == IB200_E4M3) append_kernel<__nv_bfloat16, HELD_E4M3, 128><<<grid, 128, 0, s>>>(a);
    else append_kernel<__nv_bfloat16, HELD_I8, 128><<<grid, 128, 0, s>>>(a);
  } else {
    if (held == IB200_E4M3) append_kernel<__half, HELD_E4M3, 128><<<grid, 128, 0, s>>>(a);
    else append_kernel<__half, HELD_I8, 128><<<grid, 128, 0, s>>>(a);
  }
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "kv8_append launch");
}

size_t kv8_attention_scratch_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_kv8_attention(Kv8Attention& a, int dtype, int held, void*, size_t, cudaStream_t s) {
  if (int rc = check_cache("attention_kv8", a.pages, a.heads, a.block, a.dim, a.batch, a.table_blocks, a.tokens, held, dtype, a.cu)) return rc;
  if (a.q_heads < 0 || (a.heads > 0 ? a.q_heads % a.heads : a.q_heads)) return fail(IB200_ERR_INVALID, "attention_kv8: query heads must be a multiple of the cache's");
  if (a.q_heads > 65535) return fail(IB200_ERR_UNSUPPORTED, "attention_kv8: fewer than 2^16 query heads");
  if (a.window < 0) return fail(IB200_ERR_INVALID, "attention_kv8: negative window");
  if (a.tokens == 0 || a.q_heads == 0 || a.batch == 0) return IB200_OK;
  if (!a.q || !a.o || !a.lens || (a.table_blocks > 0 && !a.table) || (a.pages > 0 && (!a.k_cache || !a.v_cache || !a.k_scale || !a.v_scale)))
    return fail(IB200_ERR_INVALID, "attention_kv8: null operand");
  if (!aligned16(a.k_cache) || !aligned16(a.v_cache)) return fail(IB200_ERR_INVALID, "attention_kv8: caches must be 16-byte aligned");
  a.each = (int)(a.tokens / a.batch);
  const int64_t units = ((int64_t)a.tokens * a.q_heads + 3) / 4;
  if (units > INT32_MAX) return fail(IB200_ERR_UNSUPPORTED, "attention_kv8: too many rows");
  if (dtype == IB200_BF16) {
    if (held == IB200_E4M3) attention_warp_kernel<__nv_bfloat16, HELD_E4M3><<<(unsigned)units, 128, 0, s>>>(a);
    else attention_warp_kernel<__nv_bfloat16, HELD_I8><<<(unsigned)units, 128, 0, s>>>(a);
  } else {
    if (held == IB200_E4M3) attention_warp_kernel<__half, HELD_E4M3><<<(unsigned)units, 128, 0, s>>>(a);
    else attention_warp_kernel<__half, HELD_I8><<<(unsigned)units, 128, 0, s>>>(a);
  }
  return cudaPeekAtLastError() == cudaSuccess ? IB200_OK : cuda_fail(cudaGetLastError(), "attention_kv8 launch");
}

}  // namespace ib200
