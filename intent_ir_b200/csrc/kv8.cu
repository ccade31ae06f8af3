// A paged key / value cache held in 8 bits: its layout, and the append (kv8_attention.cu has the attention).
//   cache  [pages, heads, block, D] of e4m3 or int8, scale [pages, heads] f32: a value stands for cache * scale
//   table  [sequences, blocks per sequence]: the page that holds a sequence's tokens i * block .. i * block + block - 1
//   lens   [sequences]: tokens of each sequence, the new ones among them
//   cu     [sequences + 1]: where each sequence's new tokens lie in k, v, q and o (null: the same number for every sequence)
// What a table says is not trusted: a page outside the cache, and a token outside the table, is never read or written.  The
// append leaves such tokens out, attention that would have to read them answers NaN.
#include "kv8.cuh"

namespace ib200 {
namespace {

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
  if (!cu && batch > 0 && tokens % batch) return fail(IB200_ERR_INVALID, w + ": without offsets every sequence has the same number of new tokens");
  return IB200_OK;
}

int launch_kv8_append(Kv8Append& a, int dtype, int held, cudaStream_t s) {
  if (int rc = check_kv8("kv8_append", a.pages, a.heads, a.block, a.dim, a.batch, a.table_blocks, a.tokens, held, dtype, a.cu)) return rc;
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

}  // namespace ib200
