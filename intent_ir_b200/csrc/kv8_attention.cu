// Attention of new tokens over the paged 8-bit cache (kv8.cu says what the cache is):
//   o[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - m),   k_j = k8 * ks(page, head),   v_j = v8 * vs(page, head)
// in one pass over the keys with a running maximum m and sum, in f32.
//
// Work.  The queries that share a key head (new tokens x heads of a group) are rows, 8 * NT of them to a unit (8, 16 or 24); a unit reads
// its keys in tiles of 128.  All tiles of all units, in order, are cut into one equal range per CTA whatever the lengths are (each
// CTA adds up the lengths itself), so a batch of mixed lengths fills the GPU evenly.  A unit that lies in one range is
// finished there; the pieces of others go to scratch as (sum, maximum, unnormalised o), and a second launch joins them in order.
// Where the units and the table are small enough that a cluster of CTAs can take each unit (CLUSTER), its pieces are joined through
// distributed shared memory instead: one launch, no scratch.
//
// Inside a CTA the four warps take 32 keys each of a tile, with copies of their own two stages deep (cp.async) and no
// barrier between them until the unit ends.  Both products run on mma.sync with the keys as the 16 rows: S' = K Q' and
// O' = V' P', so that 8 queries fill a fragment where queries as rows would need 16.  Bytes are widened to f16, which
// is exact for both types; scales are applied to the scores and to p.  q is scaled by a power of two to below 2 (f16 then holds it to 2^-12 of itself
// down to 2^-14 of the row's largest), and p * vs by what takes the row's own largest to between 2^10 and 2^14: f16 holds each of them to 2^-12 of itself
// or 2^-35 of the largest.  A key that a row does not see or give weight to does not enter that, whatever scale its page has; one whose weight is below
// 2^-112 of the row's largest may count for less than its scale would make of it.
//
// With 8 rows to a unit HBM bounds it: 64 sequences of up to 8193 keys, 32 / 8 heads of 128, e4m3, 94 us (5.7 TB/s, 0.87 of a copy's rate); 2 of 131 073 keys,
// 64 / 8 heads, 69 us (5.4 TB/s).  With more rows no unit is full: 16 x 5 new tokens over 15 000 keys 83 us (3.3 TB/s, 131 TFLOP/s) with 42 % of the issue slots and a third
// of the tensor cycles taken, by eight warps to an SM that wait on fixed latencies, each step a chain of product, maximum, exponential, transpose, product.  6 x 512 new
// tokens over 4608 keys 856 us (256 TFLOP/s).  Short work is a chain of latencies: 702 keys 7.0 us, 33 x up to 5 new tokens in a window of 2048 21.4 us.
// One power for all rows instead, led by every page's scale, took 64 sequences in 92 us, 16 x 5 new tokens in 81; a page in front of a window cost the window's keys their bits.
// A third stage of copies changed nothing at a width of 64 (20.8 / 20.7 us; 64 sequences 58.0 / 55.9).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "async.cuh"
#include "kv8.cuh"

namespace ib200 {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 32, kTile = kWarps * kStep, kStages = 2;
// What beginning a unit costs, in tiles: tables, pages and queries are fetched one after the other and the warps' results joined.
// 64 sequences of up to 8193 tokens: 113 us with 0, 97 with 2, 94 with 4, 95 with 6; 16 x 5 new tokens over 15 000 keys 108, 92, 83, 79; 33 x up to 5 in a window of
// 2048 24.2, 20.3, 21.4, 22.2.
constexpr int kStart = 4;
constexpr float kNone = -3.402823466e38f;  // a row's maxima before its first key: finite, so that differences of two are numbers
constexpr float kUp = 14.0f;               // a row's numerators p * vs are raised to at most 2^kUp
template <int D> struct Cfg {
  static constexpr int kStageBytes = 2 * kStep * D;  // keys, values
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  static constexpr int kCtas = D == 128 ? 3 : 4;  // per SM with one eight of rows; one less with two (registers)
  static constexpr int kPitch = D + 4;            // floats between the rows of the joining buffer
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {  // zeros where nothing is taken
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// the largest of the eight lanes that hold a row's other keys
__device__ __forceinline__ float over_rows(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Byte offset of 16-byte chunk c of token row r in a stage.  Eight lanes that read a quarter-warp's worth of chunks then touch all
// banks once, for keys (two adjacent rows, four chunks) and for values (rows 0, 2, 4, 6, two chunks) alike.
template <int D> __device__ __forceinline__ int at_chunk(int r, int c) {
  if (D == 128) return r * 128 + ((c ^ ((r & 6) ^ ((r & 1) << 2))) << 4);
  const int line = r >> 1;
  return line * 128 + (((((r & 1) << 2) + c) ^ ((line & 3) << 1)) << 4);
}

struct Seq {  // what a sequence asks for
  int first, n, len, keys, tile0, tiles, units_per_head;  // keys: those that the table has room for
  int64_t unit_work, work;  // a unit's, all units' (0 where there are no tiles)
};
__device__ __forceinline__ int first_key(const Kv8Attention& a, int pos) {  // that the token at `pos` sees
  return a.window > 0 && pos >= a.window ? pos - (int)a.window + 1 : 0;
}
struct Divisors {
  FastDiv group, block;
  int split, units_per_head;  // CLUSTER: CTAs to a unit; units of every sequence and head
};
__device__ __forceinline__ Seq seq_of(const Kv8Attention& a, int group, int b, int rows) {
  Seq s;
  s.first = a.cu ? a.cu[b] : b * a.each;
  s.n = a.cu ? a.cu[b + 1] - s.first : a.each;
  s.len = a.lens[b];
  if (s.n <= 0 || s.len <= 0 || s.first < 0 || (int64_t)s.first + s.n > a.tokens) s.n = 0, s.len = 0;  // nothing to do, or offsets that cannot be
  s.keys = (int)min((int64_t)s.len, a.table_blocks * a.block);
  s.tile0 = first_key(a, s.len - s.n) / kTile;
  s.tiles = s.keys > 0 ? max(0, (s.keys - 1) / kTile + 1 - s.tile0) : 0;
  s.units_per_head = (int)(((int64_t)s.n * group + rows - 1) / rows);
  s.unit_work = s.tiles ? s.tiles + kStart : 0;
  s.work = a.heads * s.units_per_head * s.unit_work;
  return s;
}

// scratch: the work in front of every sequence and in all, then two partial results per CTA
struct Scratch {
  int64_t* before;  // [batch + 1]
  float* part;      // [2 * CTAs][rows * (D + 2)]
};
__host__ __device__ inline size_t prefix_bytes(int64_t batch) { return ((size_t)(batch + 1) * 8 + 255) / 256 * 256; }
__host__ __device__ inline Scratch carve(void* p, int64_t batch) {
  return {static_cast<int64_t*>(p), reinterpret_cast<float*>(static_cast<char*>(p) + prefix_bytes(batch))};
}

template <typename V> __device__ __forceinline__ V scan_warp(V v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

template <typename T, int HELD, int D, int NT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, NT == 1 ? Cfg<D>::kCtas : Cfg<D>::kCtas - 1) attention_kernel(const Kv8Attention a, const Scratch sc, const Divisors by, const int q_vec) {
  using C = Cfg<D>;
  constexpr int ROWS = 8 * NT, HALVES = D / 64, MT = D / 16, CH = D / 16;  // CH: 16-byte chunks of a token
  // An f16 result is off by 2^-12 of itself, no more than p rounded to f16 once: there p is multiplied in two parts.  (bf16's 2^-9 hides it; two parts
  // there would take 16 x 5 new tokens over 15 000 keys from 83 to 94 us, as f16 has it.)
  constexpr bool kTwice = std::is_same<T, __half>::value;
  static_assert((kWarps + (CLUSTER ? 1 : 0)) * ROWS * C::kPitch * 4 <= C::kSmem, "the warps' results, and a cluster's piece, where the stages were");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t sums[kWarps], found_before;
  __shared__ int found;
  __shared__ float stat[kWarps][ROWS][2], joined[ROWS][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int batch = (int)a.batch, group = (int)by.group.d;

  // ---- this CTA's range of tiles -------------------------------------------------------------------
  int64_t total = 0, w = 0, w_end = 1, front = 0;
  int b = 0;
  if constexpr (CLUSTER) {
    b = (int)(blockIdx.x / by.split) / ((int)a.heads * by.units_per_head);
  } else {
  w_end = 0;
  if (threadIdx.x == 0) found = -1;
  auto range = [&] {
    const int ctas = (int)min((int64_t)gridDim.x, total);  // with less work than CTAs, one tile to each
    if (blockIdx.x < ctas) {
      w = total * blockIdx.x / ctas;
      w_end = total * (blockIdx.x + 1) / ctas;
    }
  };
  if (batch > kThreads) {
    int64_t mine = 0;
    for (int b = threadIdx.x; b < batch; b += kThreads) mine += seq_of(a, group, b, ROWS).work;
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    total = sums[0] + sums[1] + sums[2] + sums[3];
    range();
  }
  int64_t before = 0;
  for (int base = 0; base < batch; base += kThreads) {
    __syncthreads();
    const int b = base + threadIdx.x;
    const int64_t v = b < batch ? seq_of(a, group, b, ROWS).work : 0;
    const int64_t upto = scan_warp(v, lane);
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t upfront = before;
    for (int i = 0; i < warp; ++i) upfront += sums[i];
    upfront += upto - v;  // the work in front of sequence b
    before += sums[0] + sums[1] + sums[2] + sums[3];
    if (batch <= kThreads) {
      total = before;
      range();
    }
    if (blockIdx.x == 0 && b < batch) sc.before[b] = upfront;
    if (v > 0 && upfront <= w && w < upfront + v) {
      found = b;
      found_before = upfront;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) sc.before[batch] = total;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining launch may line up: it waits for this one's end
  __syncthreads();
  if (w >= w_end) return;
  b = found;
  front = found_before;
  }

  uint8_t* stages = smem + warp * kStages * C::kStageBytes;
  const uint32_t stages_at = (uint32_t)__cvta_generic_to_shared(stages);
  Seq s = seq_of(a, group, b, ROWS);
  const int64_t w_start = w;

  while (w < w_end) {
    // ---- a piece: one unit's tiles [from, to) -------------------------------------------------------
    // a unit's work is kStart for beginning it, then its tiles; a piece without tiles is nothing
    int head, r0, from, to, rows, start;  // start: place of the first new token (negative: fewer tokens than new ones)
    const int64_t piece_start = w;
    if constexpr (CLUSTER) {
      const int unit = (int)(blockIdx.x / by.split) - b * (int)a.heads * by.units_per_head, rank = blockIdx.x % by.split;
      head = unit / by.units_per_head;
      r0 = (unit - head * by.units_per_head) * ROWS;
      from = (int)((int64_t)s.tiles * rank / by.split);
      to = (int)((int64_t)s.tiles * (rank + 1) / by.split);
      rows = min(ROWS, a.each * group - r0);
      start = max(a.lens[b], -1) - a.each;  // (s counts nothing for a sequence without tokens, whose rows are written all the same)
      w = w_end;
    } else {
      const int64_t rel = w - front, unit64 = rel >> 32 ? rel / s.unit_work : (int64_t)((unsigned)rel / (unsigned)s.unit_work), in = rel - unit64 * s.unit_work;
      const int unit = (int)unit64;
      from = (int)max((int64_t)0, in - kStart);
      to = (int)min((int64_t)s.tiles, in + (w_end - w) - kStart);
      w = min(w_end, front + (unit64 + 1) * s.unit_work);
      if (to > from) {
        head = s.units_per_head == 1 ? unit : unit / s.units_per_head;
        r0 = (unit - head * s.units_per_head) * ROWS;
        rows = (int)min((int64_t)ROWS, (int64_t)s.n * group - r0);
        start = s.len - s.n;
      }
    }
    if (CLUSTER || to > from) {
    const int pos_min = start + (int)by.group.div(r0), pos_max = start + (int)by.group.div(r0 + rows - 1);
    const int lo_min = first_key(a, pos_min), lo_max = first_key(a, pos_max);
    // this warp's steps: 32 keys from 128 * tile + 32 * warp, those with a key that any row sees
    const int off = warp * kStep;
    int j0 = s.tile0 + from, j1 = s.tile0 + to;  // tiles
    if (lo_min > off + kStep - 1) j0 = max(j0, (lo_min - off - kStep + 1 + kTile - 1) / kTile);
    j1 = pos_max < off ? j0 : min(j1, (pos_max - off) / kTile + 1);
    const int steps = max(0, j1 - j0);

    // Pages and scales, 16 steps at a time: lane 2i + h looks up the 16 keys of half h of step i.  The next 16 are fetched while these are used.
    struct Meta { int page, slot; float ks, vs; };  // page: page * heads + head, -1: outside the cache
    auto look_up = [&](int step0) {
      Meta x{-1, 0, NAN, NAN};
      const int step = step0 + (lane >> 1);
      const unsigned key = (unsigned)(j0 + step) * kTile + off + (lane & 1) * 16;
      if (step < steps && key < (unsigned)s.keys) {
        unsigned blk, slot;
        by.block.divmod(key, blk, slot);
        x.slot = (int)slot;
        const int page = a.table[(int64_t)b * a.table_blocks + blk];
        if ((unsigned)page < (unsigned)a.pages) x.page = page * (int)a.heads + head;
      }
      return x;
    };
    auto look_scales = [&](Meta& x) {
      if (x.page >= 0) {
        x.ks = a.k_scale[x.page];
        x.vs = a.v_scale[x.page];
      }
    };
    // The 16 keys of a half are one run of bytes in memory.  Chunk i * 32 + lane of it goes to row (i * 32 + lane) / CH; rows 8 apart are
    // swizzled alike, so two places of a lane give all others by adding constants.
    const uint32_t place0 = at_chunk<D>(lane / CH, lane % CH), place1 = at_chunk<D>((32 + lane) / CH, lane % CH) - 512;
    auto issue = [&](int step, const Meta& meta) {
      const uint32_t dst = stages_at + (step % kStages) * C::kStageBytes;
      const int key0 = (j0 + step) * kTile + off;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = __shfl_sync(0xffffffffu, meta.page, 2 * (step & 15) + h), slot = __shfl_sync(0xffffffffu, meta.slot, 2 * (step & 15) + h);
        const int left = page < 0 ? 0 : s.keys - (key0 + h * 16);  // keys of these 16 that exist; what lies behind the last one is never read
        const int64_t base = page < 0 ? 0 : ((int64_t)page * a.block + slot) * D;
        const uint8_t *ksrc = a.k_cache + base + lane * 16, *vsrc = a.v_cache + base + lane * 16;
        const uint32_t even = dst + h * 16 * D + place0, odd = dst + h * 16 * D + place1;
        if (left >= 16) {
#pragma unroll
          for (int i = 0; i < 16 * CH / 32; ++i) {
            copy16((i & 1 ? odd : even) + i * 512, ksrc + i * 512);
            copy16((i & 1 ? odd : even) + i * 512 + kStep * D, vsrc + i * 512);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16 * CH / 32; ++i) {
            const bool take = (i * 32 + lane) / CH < left;
            copy16((i & 1 ? odd : even) + i * 512, take ? ksrc + i * 512 : a.k_cache, take);
            copy16((i & 1 ? odd : even) + i * 512 + kStep * D, take ? vsrc + i * 512 : a.v_cache, take);
          }
        }
      }
    };

    Meta cur = look_up(0);
    look_scales(cur);
    Meta nxt = cur;
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < steps) issue(i, cur);
      copy_commit();
    }
    // queries as the k x 8 operand: chunk bytes 4w .. 4w + 3 of half h are the k slots (2t, 2t + 1, 2t + 8, 2t + 9) of product 4h + w
    uint32_t qf[NT][HALVES * 4][2];
    float mult[NT][2];
    int hi[NT][2], low[NT][2];  // the keys that this thread's two columns (rows of the unit) see: low .. hi
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = r0 + nt * 8 + g;
      const bool real = nt * 8 + g < rows;
      const int i = real ? (int)by.group.div(row) : 0, jq = real ? row - i * group : 0;
      const T* q = static_cast<const T*>(a.q) + (int64_t)(s.first + i) * a.q_token + (int64_t)(head * group + jq) * a.q_head;
      float v[HALVES * 4][4], top = 0.0f;
#pragma unroll
      for (int k = 0; k < HALVES * 4; ++k) {
        const int d = (k >> 2) * 64 + t * 16 + (k & 3) * 4;
        if (!real) {
          v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
        } else if (q_vec) {
          load4(q + d, v[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k][e] = to_f32(q[d + e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[k][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e for top in [2^e, 2^(e+1)); 1 for a row of zeros or with an infinity
      const int e = (int)(__float_as_uint(top) >> 23);
      const float down = top == 0.0f || e == 255 ? 1.0f : __uint_as_float((uint32_t)min(253, max(1, 254 - e)) << 23);
#pragma unroll
      for (int k = 0; k < HALVES * 4; ++k) {
        qf[nt][k][0] = pack16(v[k][0] * down, v[k][1] * down);
        qf[nt][k][1] = pack16(v[k][2] * down, v[k][3] * down);
      }
      const float m = a.scale * 1.4426950408889634f / down;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mult[nt][c] = __shfl_sync(0xffffffffu, m, (2 * t + c) * 4);
        const int rr = nt * 8 + 2 * t + c;
        hi[nt][c] = rr < rows ? start + (int)by.group.div(r0 + rr) : -1;
        low[nt][c] = first_key(a, hi[nt][c]);
      }
    }

    // l is the sum of p = 2^(score - m), o that of p * vs * v8 * 2^(m - high): m is the row's largest score so far, high that of score + log2(vs) - kUp (a bound)
    float o[NT][MT][4], m[NT][2], high[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) m[nt][c] = high[nt][c] = kNone, l[nt][c] = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.0f;
    }

    // one step; masked: some row does not see all of its keys
    auto compute = [&](int step, auto kind) {
      constexpr bool masked = decltype(kind)::value;
      const uint8_t* kst = stages + (step % kStages) * C::kStageBytes;
      const uint8_t* vst = kst + kStep * D;
      const int key0 = (j0 + step) * kTile + off;

      // ---- S' = K Q' --------------------------------------------------------------------------------
      float sv[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sv[mt][nt][0] = sv[mt][nt][1] = sv[mt][nt][2] = sv[mt][nt][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint4 x = *reinterpret_cast<const uint4*>(kst + at_chunk<D>(mt * 16 + g, h * 4 + t));
          const uint4 y = *reinterpret_cast<const uint4*>(kst + at_chunk<D>(mt * 16 + 8 + g, h * 4 + t));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t a0, a1, a2, a3;
            widen<HELD>(xs[k], a0, a2);
            widen<HELD>(ys[k], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(sv[mt][nt], a0, a1, a2, a3, qf[nt][h * 4 + k][0], qf[nt][h * 4 + k][1]);
          }
        }
      }

      // ---- running maximum and sum ------------------------------------------------------------------
      const float ks[2] = {__shfl_sync(0xffffffffu, cur.ks, 2 * (step & 15)), __shfl_sync(0xffffffffu, cur.ks, 2 * (step & 15) + 1)};
      const float vs[2] = {__shfl_sync(0xffffffffu, cur.vs, 2 * (step & 15)), __shfl_sync(0xffffffffu, cur.vs, 2 * (step & 15) + 1)};
      // log2 of the values' larger scale, 2^-100 at least; a NaN counts for nothing (it reaches p below)
      const float vs_top = fmaxf(fmaxf(fabsf(vs[0]), fabsf(vs[1])), 0x1p-100f);
      float vs_most = log2_fast(vs_top) - kUp;
      // every row's largest score of the step (over both halves' keys), and a bound on score + log2(vs)
      float top[NT][2], most[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x = sv[mt][nt][c] * (mult[nt][c & 1] * ks[mt]);
            if constexpr (masked) {
              const int key = key0 + mt * 16 + (c >> 1) * 8 + g;
              if (key > hi[nt][c & 1] || key < low[nt][c & 1]) x = -INFINITY;
            }
            sv[mt][nt][c] = x;
            top[nt][c & 1] = fmaxf(top[nt][c & 1], x);
          }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[nt][c] = over_rows(top[nt][c]);
          most[nt][c] = top[nt][c] + vs_most;
        }
      }
      if (!(vs_top <= fminf(16.0f * fminf(fabsf(vs[0]), fabsf(vs[1])), 3.402823466e38f))) {  // far apart: a half's scale counts with the half's own scores only,
        float by_half[2];                                                                  // an infinite one (whose rows are not finite) not at all
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) by_half[mt] = isinf(vs[mt]) ? -100.0f - kUp : log2_fast(fmaxf(fabsf(vs[mt]), 0x1p-100f)) - kUp;
        vs_most = fmaxf(by_half[0], by_half[1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            most[nt][c] = fmaxf(over_rows(fmaxf(sv[0][nt][c], sv[0][nt][c + 2])) + by_half[0], over_rows(fmaxf(sv[1][nt][c], sv[1][nt][c + 2])) + by_half[1]);
      }
      uint32_t pf[NT][2][2];
      [[maybe_unused]] uint32_t pl[NT][2][2];  // what p's rounding left
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float keep[2], raise[2];  // what o is to be multiplied by, and p for its numerators
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float now = fmaxf(m[nt][c], top[nt][c]), now_most = fmaxf(high[nt][c], most[nt][c]);
          l[nt][c] *= exp2_fast(m[nt][c] - now);
          keep[c] = exp2_fast(high[nt][c] - now_most);
          raise[c] = exp2_fast(fminf(now - now_most, (126.0f - kUp) - vs_most));  // (finite times either scale)
          m[nt][c] = now;
          high[nt][c] = now_most;
        }
        float p[2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float raised[2] = {vs[mt] * raise[0], vs[mt] * raise[1]};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float x = exp2_fast(sv[mt][nt][c] - m[nt][c & 1]);
            l[nt][c & 1] += x;
            p[mt][c] = x * raised[c & 1];
            if constexpr (masked) {  // a NaN scale counts only for the rows that see the key
              const int key = key0 + mt * 16 + (c >> 1) * 8 + g;
              if (key > hi[nt][c & 1] || key < low[nt][c & 1]) p[mt][c] = 0.0f;
            }
          }
          const uint32_t p0 = pack16(p[mt][0], p[mt][1]), p1 = pack16(p[mt][2], p[mt][3]);
          pf[nt][mt][0] = transpose8x8(p0);
          pf[nt][mt][1] = transpose8x8(p1);
          if constexpr (kTwice) {
            const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&p0)), h1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
            pl[nt][mt][0] = transpose8x8(pack16(p[mt][0] - h0.x, p[mt][1] - h0.y));
            pl[nt][mt][1] = transpose8x8(pack16(p[mt][2] - h1.x, p[mt][3] - h1.y));
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[nt][i][0] *= keep[0];
          o[nt][i][1] *= keep[1];
          o[nt][i][2] *= keep[0];
          o[nt][i][3] *= keep[1];
        }
      }

      // ---- O' += V' P' ------------------------------------------------------------------------------
      // thread (g, t) has d = (D / 8) g .. of keys 2t, 2t + 1, 2t + 8, 2t + 9: adjacent keys' bytes are paired, tile i has d = (D / 8) g + 2i in row g, + 1 in row g + 8
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t vb[4][D / 32];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = mt * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
          if (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(vst + at_chunk<D>(r, g));
            vb[e][0] = x.x, vb[e][1] = x.y, vb[e][D / 32 - 2] = x.z, vb[e][D / 32 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(vst + at_chunk<D>(r, g >> 1) + (g & 1) * 8);
            vb[e][0] = x.x, vb[e][1] = x.y;
          }
        }
        bool by_row = false;  // a NaN among values that some rows do not see: the rows' products are taken one by one
        if constexpr (HELD == HELD_E4M3 && masked) {
          uint32_t any = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < D / 32; ++k) any |= __vcmpeq4(vb[e][k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
          by_row = __any_sync(0xffffffffu, any != 0);
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          uint32_t f[2][4];
          widen<HELD>(__byte_perm(vb[0][k], vb[1][k], 0x5140), f[0][0], f[0][1]);
          widen<HELD>(__byte_perm(vb[2][k], vb[3][k], 0x5140), f[0][2], f[0][3]);
          widen<HELD>(__byte_perm(vb[0][k], vb[1][k], 0x7362), f[1][0], f[1][1]);
          widen<HELD>(__byte_perm(vb[2][k], vb[3][k], 0x7362), f[1][2], f[1][3]);
          if (!by_row) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                mma16816(o[nt][2 * k + i], f[i][0], f[i][1], f[i][2], f[i][3], pf[nt][mt][0], pf[nt][mt][1]);
                if constexpr (kTwice) mma16816(o[nt][2 * k + i], f[i][0], f[i][1], f[i][2], f[i][3], pl[nt][mt][0], pl[nt][mt][1]);
              }
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll 1
              for (int col = 0; col < 8; ++col) {
                const int last = __shfl_sync(0xffffffffu, (col & 1) ? hi[nt][1] : hi[nt][0], col >> 1), begin = __shfl_sync(0xffffffffu, (col & 1) ? low[nt][1] : low[nt][0], col >> 1);
                uint32_t keep[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int key = key0 + mt * 16 + 2 * t + e * 8;
                  keep[e] = (key <= last && key >= begin ? 0xffffu : 0u) | (key + 1 <= last && key + 1 >= begin ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  mma16816(o[nt][2 * k + i], f[i][0] & keep[0], f[i][1] & keep[0], f[i][2] & keep[1], f[i][3] & keep[1], g == col ? pf[nt][mt][0] : 0u,
                           g == col ? pf[nt][mt][1] : 0u);
                  if constexpr (kTwice)
                    mma16816(o[nt][2 * k + i], f[i][0] & keep[0], f[i][1] & keep[0], f[i][2] & keep[1], f[i][3] & keep[1], g == col ? pl[nt][mt][0] : 0u,
                             g == col ? pl[nt][mt][1] : 0u);
                }
              }
          }
        }
      }
    };

    for (int step = 0; step < steps; ++step) {
      if ((step & 15) == 0) {
        if (step) cur = nxt;
        nxt = look_up(step + 16);
      } else if ((step & 15) == 8) {
        look_scales(nxt);
      }
      copy_wait<kStages - 2>();
      __syncwarp();
      {
        const int ahead = step + kStages - 1;
        if (ahead < steps) {
          if ((ahead >> 4) == (step >> 4)) issue(ahead, cur); else issue(ahead, nxt);
        }
        copy_commit();
      }
      const int key0 = (j0 + step) * kTile + off;
      if (key0 + kStep - 1 > pos_min || key0 < lo_max) compute(step, std::true_type()); else compute(step, std::false_type());
    }

    // ---- join the warps -------------------------------------------------------------------------------
    copy_wait<0>();
    __syncthreads();  // all stages are read; their memory takes the warps' results
    float* box = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int row = nt * 8 + 2 * t + c;
        if (g == 0) {
          stat[warp][row][0] = m[nt][c];
          stat[warp][row][1] = x;
        }
        float* to_row = box + (warp * ROWS + row) * C::kPitch + g * (D / 8);
        const float down = exp2_fast(high[nt][c] - m[nt][c]);
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(to_row + 2 * i) = make_float2(o[nt][i][c] * down, o[nt][i][2 + c] * down);
      }
    }
    __syncthreads();
    const bool whole = from == 0 && to == s.tiles;
    float* part = CLUSTER ? nullptr : sc.part + ((int64_t)blockIdx.x * 2 + (piece_start == w_start ? 0 : 1)) * (ROWS * (D + 2));
    float* joint = box + kWarps * ROWS * C::kPitch;  // CLUSTER: this CTA's piece
    auto write = [&](int row, int d, float mm, float sum, float (&v)[4]) {
      const int i = (int)by.group.div(r0 + row);
      const int64_t out = (int64_t)(s.first + i) * a.q_heads + head * group + (r0 + row - i * group);
      const bool empty = start + i < 0;
      if (start + i >= s.keys) sum = NAN;  // its own key is outside the table
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = empty ? 0.0f : v[e] / sum;
      store4(static_cast<T*>(a.o) + out * D + d, v);
      if (a.lse && d == 0) a.lse[out] = empty ? -INFINITY : (mm + log2f(sum)) * 0.6931471805599453f;
    };
    for (int idx = threadIdx.x; idx < ROWS * (D / 4); idx += kThreads) {
      const int row = idx / (D / 4), d = idx % (D / 4) * 4;
      if (row >= rows) break;
      const float mm = fmaxf(fmaxf(stat[0][row][0], stat[1][row][0]), fmaxf(stat[2][row][0], stat[3][row][0]));
      float sum = 0.0f, v[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float f = exp2_fast(stat[i][row][0] - mm);
        sum += stat[i][row][1] * f;
        const float4 x = *reinterpret_cast<const float4*>(box + (i * ROWS + row) * C::kPitch + d);
        v[0] += x.x * f, v[1] += x.y * f, v[2] += x.z * f, v[3] += x.w * f;
      }
      if constexpr (CLUSTER) {
        *reinterpret_cast<float4*>(joint + row * C::kPitch + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) joined[row][0] = mm, joined[row][1] = sum;
      } else if (whole) {
        write(row, d, mm, sum, v);
      } else {
        *reinterpret_cast<float4*>(part + row * D + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) {
          part[ROWS * D + row] = mm;
          part[ROWS * D + ROWS + row] = sum;
        }
      }
    }
    if constexpr (CLUSTER) {
      cluster_sync();
      for (int idx = (int)(blockIdx.x % by.split) * kThreads + threadIdx.x; idx < rows * (D / 4); idx += by.split * kThreads) {
        const int row = idx / (D / 4), d = idx % (D / 4) * 4;
        float mm = -INFINITY, sum = 0.0f, v[4] = {0, 0, 0, 0};
        for (int r = 0; r < by.split; ++r) mm = fmaxf(mm, cluster_read(&joined[row][0], r));
        for (int r = 0; r < by.split; ++r) {
          const float f = exp2_fast(cluster_read(&joined[row][0], r) - mm);
          sum += cluster_read(&joined[row][1], r) * f;
          const float4 x = cluster_read4(joint + row * C::kPitch + d, r);
          v[0] += x.x * f, v[1] += x.y * f, v[2] += x.z * f, v[3] += x.w * f;
        }
        write(row, d, mm, sum, v);
      }
      cluster_sync();  // nobody leaves while its piece is read
      return;
    }
    __syncthreads();  // the next piece copies over the box
    }
    if (w < w_end && w == front + s.work) {
      front = w;
      do s = seq_of(a, group, ++b, ROWS); while (s.work == 0);  // w < total: there is one
    }
  }
}

// A row whose unit was cut is joined from its pieces, one without keys is zero.  WARPS warps to a row take every WARPS-th piece.
constexpr int kJoin = 128;
template <typename T, int D, int NT, int WARPS>
__global__ void __launch_bounds__(kJoin) join_kernel(const Kv8Attention a, const Scratch sc, const Divisors by, const int grid) {
  constexpr int ROWS = 8 * NT, PER = D / 32;
  __shared__ float box[kJoin / 32][D];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS;
  const int64_t u = (int64_t)blockIdx.x * (kJoin / 32 / WARPS) + (threadIdx.x >> 5) / WARPS;
  if (u >= a.tokens * a.q_heads) return;  // (warps of one row leave together, here and below)
  const int t = (int)(u / a.q_heads), qh = (int)(u - (int64_t)t * a.q_heads), group = (int)by.group.d;
  int b, first, count;
  if (!find_sequence(a.cu, (int)a.batch, a.each, t, b, first, count)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (this launch ends after the one in front, whatever the offsets say)
    return;
  }
  const Seq s = seq_of(a, group, b, ROWS);
  const int64_t pos = (int64_t)a.lens[b] - count + (t - first);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  T* o = static_cast<T*>(a.o) + u * D;
  if (pos < 0 || pos >= s.keys || s.tiles == 0) {  // no keys; or its own key is outside the table (or offsets that cannot be)
    for (int d = warp * 32 + lane; d < D; d += WARPS * 32) o[d] = from_f32<T>(pos < 0 ? 0.0f : NAN);
    if (a.lse && warp == 0 && lane == 0) a.lse[u] = pos < 0 ? -INFINITY : NAN;
    return;
  }
  const int head = (int)by.group.div(qh), r = (t - first) * group + (qh - head * group), row = r % ROWS;
  // the CTAs whose ranges hold the unit's first and last tile
  const int64_t total = sc.before[a.batch], unit = sc.before[b] + ((int64_t)head * s.units_per_head + r / ROWS) * s.unit_work;
  const int64_t ctas = min((int64_t)grid, total), lo = unit + kStart, hi = unit + s.unit_work - 1;
  const int c0 = (int)(((lo + 1) * ctas - 1) / total), c1 = (int)(((hi + 1) * ctas - 1) / total);
  if (c0 == c1) return;
  const int64_t size = ROWS * (D + 2);
  const float* p0 = sc.part + ((int64_t)c0 * 2 + (total * c0 / ctas >= unit ? 0 : 1)) * size;
  auto piece = [&](int c) { return c == c0 ? p0 : sc.part + (int64_t)c * 2 * size; };
  float m = -INFINITY, sum = 0.0f, v[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) v[e] = 0.0f;
  for (int base = c0; base <= c1; base += 32) {  // every warp has the weights of 32 pieces, a lane each
    const int c = base + lane, n = min(32, c1 - base + 1);
    const float pm = c <= c1 ? piece(c)[ROWS * D + row] : -INFINITY, pl = c <= c1 ? piece(c)[ROWS * D + ROWS + row] : 0.0f;
    const float now = fmaxf(m, warp_reduce<MaxOp>(pm)), keep = exp2_fast(m - now), f = exp2_fast(pm - now);
    sum = sum * keep + warp_reduce<SumOp>(c <= c1 ? pl * f : 0.0f);
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] *= keep;
    m = now;
#pragma unroll 4
    for (int i = warp; i < n; i += WARPS) {
      const float* p = piece(base + i) + row * D + lane * PER;
      const float g = __shfl_sync(0xffffffffu, f, i);
      if (PER == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] += x.x * g, v[1] += x.y * g, v[PER - 2] += x.z * g, v[PER - 1] += x.w * g;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] += x.x * g, v[1] += x.y * g;
      }
    }
  }
  if (WARPS > 1) {  // (one row to the CTA)
#pragma unroll
    for (int e = 0; e < PER; ++e) box[warp][lane * PER + e] = v[e];
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int e = 0; e < PER; ++e)
#pragma unroll
      for (int i = 1; i < WARPS; ++i) v[e] += box[i][lane * PER + e];
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) o[lane * PER + e] = from_f32<T>(v[e] / sum);
  if (a.lse && lane == 0) a.lse[u] = (m + log2f(sum)) * 0.6931471805599453f;
}

int64_t most_ctas(int64_t dim, int nt) { return (int64_t)kSmCount * ((dim == 128 ? Cfg<128>::kCtas : Cfg<64>::kCtas) - (nt > 1)); }

// Rows of a unit, in eights: one where 8 rows suffice, two or three where a sequence has more (several new tokens, many heads to a group) so
// that its keys are read and widened less often.  A unit of three takes 1.36 to 1.6 times a unit of two: 16 x 15 000 keys of 128 for 20 rows (one unit or
// two) 84 / 104 us, 40 rows (two or three) 139 / 154, 6 x 512 tokens over 4608 keys 857 / 933, up to 512 with offsets 616 / 661, but 33 x up to 8 tokens x 4 heads of 64 27.6 / 24.8, and
// 11.5 / 10.1 us where two sequences of 705 keys leave the GPU room for every tile of twice the units.  With offsets only the average number of new tokens is known here.
// (Units of three spill up to 38 words at D = 128, 27 at 64.)
int tiles_of_rows(int64_t tokens, int64_t batch, int64_t heads, int64_t group, int64_t dim, int64_t block, int64_t table_blocks, bool uniform) {
  const int64_t rows = group * ((tokens + batch - 1) / batch), two = (rows + 15) / 16, three = (rows + 23) / 24;
  if (rows <= 8) return 1;
  const int64_t units = batch * heads * two, most = most_ctas(dim, 2);
  if (units <= most && units * ((table_blocks * block + kTile - 1) / kTile) <= most) return 2;
  return (uniform ? 4 * three <= 3 * two : rows > 48) ? 3 : 2;
}
int64_t grid_of(int64_t tokens, int64_t batch, int64_t heads, int64_t group, int64_t dim, int64_t block, int64_t table_blocks, int nt) {
  // no more CTAs than there can be tiles
  const int64_t units = heads * ((tokens * group + 8 * nt - 1) / (8 * nt) + batch), tiles = table_blocks * block / kTile + 2 + kStart;
  const int64_t most = most_ctas(dim, nt);
  return units > most || units * tiles > most ? most : units * tiles;
}

// CTAs of a cluster that takes a unit, 0 where the general form is to be used.  Its CTAs must all run at once and have at most eight tiles each, by the
// room in the table.  Device time against the general form's: 1 sequence of 701 tokens 7.0 / 9.1 us, 1 of 8000 13.4 / 14.9, 16 of up to 3000 18.6 / 21.0, 48 of
// up to 900 17.3 / 21.5, and 4.5 us less to enqueue; with sixteen tiles 2 of 16 000 took 22.4 / 19.2: longer ones gain from the even split of all tiles.
int cluster_of(int64_t tokens, int64_t batch, int64_t heads, int64_t group, int64_t dim, int64_t block, int64_t table_blocks, int nt, bool uniform) {
  if (!uniform) return 0;
  const int64_t units = batch * heads * ((tokens / batch * group + 8 * nt - 1) / (8 * nt)), tiles = (table_blocks * block + kTile - 1) / kTile;
  const int64_t most = most_ctas(dim, nt);
  if (units <= 0 || units > most) return 0;
  const int64_t split = std::min<int64_t>(8, std::max<int64_t>(1, std::min(tiles, most / units)));
  return tiles <= 8 * split ? (int)split : 0;
}

template <typename T, int HELD, int D, int NT, bool CLUSTER> int run_attention(const Kv8Attention& a, int grid, int split, void* scratch, cudaStream_t s) {
  auto* kern = attention_kernel<T, HELD, D, NT, CLUSTER>;
  static std::atomic<uint64_t> ready{0};  // devices that have been told of the shared memory
  int dev = 0;
  IB200_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    IB200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
    if (dev <= 63) ready.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  }
  const Scratch sc = carve(scratch, a.batch);
  const int q_vec = (reinterpret_cast<uintptr_t>(a.q) & 7) == 0 && a.q_token % 4 == 0 && a.q_head % 4 == 0;
  const int per_head = (int)(((int64_t)a.each * (a.q_heads / a.heads) + 8 * NT - 1) / (8 * NT));
  const Divisors by{FastDiv((uint32_t)(a.q_heads / a.heads)), FastDiv((uint32_t)a.block), split, per_head};
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if constexpr (CLUSTER) {
    cfg.gridDim = dim3((unsigned)(a.batch * a.heads * per_head * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<D>::kSmem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    IB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, sc, by, q_vec));
    return IB200_OK;
  }
  kern<<<grid, kThreads, Cfg<D>::kSmem, s>>>(a, sc, by, q_vec);
  if (cudaPeekAtLastError() != cudaSuccess) return cuda_fail(cudaGetLastError(), "attention_kv8 launch");
  // few rows have many pieces each: a CTA for a row (2 sequences of 131 073 keys: 70.5 us in all, 74.7 with a warp); many rows have few: a warp (64 of up to
  // 8193: 94.0, 95.3 with a CTA)
  const int64_t rows = a.tokens * a.q_heads;
  const bool many = rows > 4 * kSmCount;
  cfg.gridDim = dim3((unsigned)(many ? (rows + 3) / 4 : rows));
  cfg.blockDim = dim3(kJoin);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  IB200_CUDA_OK(cudaLaunchKernelEx(&cfg, many ? join_kernel<T, D, NT, 1> : join_kernel<T, D, NT, 4>, a, sc, by, grid));
  return IB200_OK;
}
template <typename T, int HELD, int D> int run_nt(const Kv8Attention& a, int nt, int grid, int split, void* scratch, cudaStream_t s) {
  if (nt == 1) return split ? run_attention<T, HELD, D, 1, true>(a, grid, split, scratch, s) : run_attention<T, HELD, D, 1, false>(a, grid, split, scratch, s);
  if (nt == 2) return split ? run_attention<T, HELD, D, 2, true>(a, grid, split, scratch, s) : run_attention<T, HELD, D, 2, false>(a, grid, split, scratch, s);
  return split ? run_attention<T, HELD, D, 3, true>(a, grid, split, scratch, s) : run_attention<T, HELD, D, 3, false>(a, grid, split, scratch, s);
}
template <typename T, int HELD> int run_dim(const Kv8Attention& a, int nt, int grid, int split, void* scratch, cudaStream_t s) {
  return a.dim == 128 ? run_nt<T, HELD, 128>(a, nt, grid, split, scratch, s) : run_nt<T, HELD, 64>(a, nt, grid, split, scratch, s);
}

}  // namespace

size_t kv8_attention_scratch_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t heads, int64_t dim, int64_t block, int64_t table_blocks, bool uniform) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || q_heads < heads || (dim != 64 && dim != 128) || block <= 0 || table_blocks < 0 || batch > INT32_MAX ||
      tokens > INT32_MAX || q_heads > 65535 || beyond_any_device(table_blocks, block))
    return 0;  // the launch refuses these, or does nothing
  const int nt = tiles_of_rows(tokens, batch, heads, q_heads / heads, dim, block, table_blocks, uniform);
  if (cluster_of(tokens, batch, heads, q_heads / heads, dim, block, table_blocks, nt, uniform)) return 0;
  return prefix_bytes(batch) + (size_t)grid_of(tokens, batch, heads, q_heads / heads, dim, block, table_blocks, nt) * 2 * 8 * nt * (dim + 2) * 4;
}

int launch_kv8_attention(Kv8Attention& a, int dtype, int held, void* scratch, size_t scratch_bytes, cudaStream_t s) {
  if (int rc = check_kv8("attention_kv8", a.pages, a.heads, a.block, a.dim, a.batch, a.table_blocks, a.tokens, held, dtype, a.cu)) return rc;
  if (a.q_heads < 0 || (a.heads > 0 ? a.q_heads % a.heads : a.q_heads)) return fail(IB200_ERR_INVALID, "attention_kv8: query heads must be a multiple of the cache's");
  if (a.q_heads > 65535) return fail(IB200_ERR_UNSUPPORTED, "attention_kv8: fewer than 2^16 query heads");
  if (a.window < 0) return fail(IB200_ERR_INVALID, "attention_kv8: negative window");
  if (a.tokens == 0 || a.q_heads == 0 || a.batch == 0) return IB200_OK;
  if (!a.q || !a.o || !a.lens || (a.table_blocks > 0 && !a.table) || (a.pages > 0 && (!a.k_cache || !a.v_cache || !a.k_scale || !a.v_scale)))
    return fail(IB200_ERR_INVALID, "attention_kv8: null operand");
  if (!aligned16(a.k_cache) || !aligned16(a.v_cache)) return fail(IB200_ERR_INVALID, "attention_kv8: caches must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(a.o) & 7) return fail(IB200_ERR_INVALID, "attention_kv8: o must be 8-byte aligned");
  if (a.tokens * a.q_heads >= INT32_MAX || beyond_any_device(a.tokens, a.q_heads, a.dim)) return fail(IB200_ERR_UNSUPPORTED, "attention_kv8: too many rows");
  const size_t need = kv8_attention_scratch_bytes(a.tokens, a.batch, a.q_heads, a.heads, a.dim, a.block, a.table_blocks, !a.cu);
  if (need && (!scratch || scratch_bytes < need)) return fail(IB200_ERR_BUFFER, "attention_kv8: scratch is smaller than ib200_attention_kv8_scratch_bytes");
  // a cache without pages is never read, but copies that take nothing want an aligned address all the same
  if (a.pages == 0) a.k_cache = a.v_cache = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(a.lens) & ~(uintptr_t)15);
  a.each = (int)(a.tokens / a.batch);
  const int64_t group = a.q_heads / a.heads;
  const int nt = tiles_of_rows(a.tokens, a.batch, a.heads, group, a.dim, a.block, a.table_blocks, !a.cu), split = cluster_of(a.tokens, a.batch, a.heads, group, a.dim, a.block, a.table_blocks, nt, !a.cu);
  const int grid = (int)grid_of(a.tokens, a.batch, a.heads, group, a.dim, a.block, a.table_blocks, nt);
  if (dtype == IB200_BF16)
    return held == IB200_E4M3 ? run_dim<__nv_bfloat16, HELD_E4M3>(a, nt, grid, split, scratch, s) : run_dim<__nv_bfloat16, HELD_I8>(a, nt, grid, split, scratch, s);
  return held == IB200_E4M3 ? run_dim<__half, HELD_E4M3>(a, nt, grid, split, scratch, s) : run_dim<__half, HELD_I8>(a, nt, grid, split, scratch, s);
}

}  // namespace ib200
