// Arguments of the paged 8-bit cache's append and attention (kv8.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ib200 {

struct Kv8Append {
  const void *k, *v;  // [tokens, heads, dim], strides in elements, dim adjacent
  int64_t k_token, k_head, v_token, v_head;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int *table, *lens, *cu;
  int64_t pages, heads, block, dim, batch, table_blocks, tokens;
  int each, per;  // without cu: new tokens per sequence, blocks that they can touch; filled by the launcher
};

struct Kv8Attention {
  const void* q;  // [tokens, q_heads, dim], strides in elements, dim adjacent
  int64_t q_token, q_head;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *table, *lens, *cu;
  void* o;     // [tokens, q_heads, dim] dense
  float* lse;  // [tokens, q_heads] or null
  int64_t pages, heads, block, dim, batch, table_blocks, tokens, q_heads, window;
  float scale;
  int each;
};

// the checks that both entries make of the cache's extents
int check_kv8(const char* what, int64_t pages, int64_t heads, int64_t block, int64_t dim, int64_t batch, int64_t table_blocks, int64_t tokens, int held,
              int dtype, const int* cu);
int launch_kv8_append(Kv8Append& a, int dtype, int held, cudaStream_t s);
int launch_kv8_attention(Kv8Attention& a, int dtype, int held, void* scratch, size_t scratch_bytes, cudaStream_t s);
size_t kv8_attention_scratch_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t heads, int64_t dim, int64_t block, int64_t table_blocks, bool uniform);

}  // namespace ib200
