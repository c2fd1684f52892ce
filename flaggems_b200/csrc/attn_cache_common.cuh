// Shared definitions of the attention over an 8-bit or windowed cache (fg_flash_attn_cache).
//
//   S_ij = scale * k_scale * q_i . c_j,   O_i = v_scale * sum_j softmax(S)_ij cv_j
//
// over the keys j that query i sees: j < k_len, j <= p_i + wr (causal: wr = 0), and j >= p_i - wl or j < sinks, with
// p_i = i + k_len - q_len.  The scales factor out of both products, so the kernels multiply what the cache holds.
//
// The 8-bit types are subsets of fp16 and the products run in fp16 with fp32 accumulators: exact for K and V, and for
// fp16 queries.  A bf16 query row is multiplied by a power of two that brings its largest value to [2^14, 2^15): its
// 8-bit significands stay exact down to 2^-31 of the row's largest, and the power is taken out of the scores in fp32.
// Probabilities are rounded to fp16 (2^-12 of themselves; four times finer than bf16, 2^-9, which a bf16 cache takes), and their
// sum is taken before that.  fp16 ends at 2^-25: they are multiplied by a power of two that takes the largest to 2^15, which the
// division by the sum takes out, so that many small ones beside a first token that draws all attention are not lost.
//
// `group` query heads share a KV head.  The rows of a tile are (token, head of the group) pairs, head fastest, so that
// every K/V byte is fetched once for all of them.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "attn_common.cuh"
#include "fp8.cuh"

namespace fg {

struct CacheAttnArgs {
  AttnArgs a;
  const float *k_scale, *v_scale;          // null: 1
  int64_t ks_batch, ks_head, vs_batch, vs_head;
  int sinks;
  int table_cols;                          // entries of a block table row
  int tiles_per_split;                     // K/V tiles of one split
  int64_t part_rows;                       // tokens that the partial results of the split forms have room for
  int64_t dense;                           // chunk kernel: rows of each sequence in a 16-bit copy that k and v point at; 0: none
  int whole;                               // tensor-core kernels: runs are cut between items only, and nothing is joined
  __host__ __device__ bool pages() const { return a.paged && dense == 0; }
};
// Lengths that contradict the sizes of the call (rows behind q or K/V, more keys than max_seqlen_k, by which the work was counted on
// the host) are cut, so that they cannot fault.
__device__ __forceinline__ SeqInfo stored_seq_info(const CacheAttnArgs& c, int b) {
  SeqInfo s = seq_info(c.a, b);
  s.q_begin = max(0, min(s.q_begin, (int)c.a.total_q));
  s.q_len = min(s.q_len, (int)c.a.total_q - s.q_begin);
  s.k_len = min(s.k_len, c.a.max_k);
  if (!c.a.paged) {
    s.k_begin = max(0, min(s.k_begin, (int)c.a.total_k));
    s.k_len = min(s.k_len, (int)c.a.total_k - s.k_begin);
  }
  return s;
}
// As the attention kernels see it: k_begin in the 16-bit copy when there is one.
__device__ __forceinline__ SeqInfo cache_seq_info(const CacheAttnArgs& c, int b) {
  SeqInfo s = stored_seq_info(c, b);
  if (c.dense > 0) s.k_begin = (int)(b * c.dense);
  return s;
}

__device__ __forceinline__ float cache_scale(const float* s, int64_t batch_stride, int64_t head_stride, int b, int hk) {
  return s ? s[b * batch_stride + hk * head_stride] : 1.f;
}

// Row of the paged store (elements) of token `tok`; page numbers are clamped into the table and the cache, so that a
// wrong table entry or length cannot fault.
__device__ __forceinline__ int cache_page(const CacheAttnArgs& c, const int32_t* bt_row, int pg) {
  const int page = bt_row[min(pg, c.table_cols - 1)];
  return max(0, min(page, c.a.num_blocks - 1));
}
__device__ __forceinline__ int64_t cache_row(const CacheAttnArgs& c, const int32_t* bt_row, int k_begin, int tok, int64_t rs,
                                             int64_t bs) {
  if (c.a.paged) {
    const int pg = tok / c.a.block_size;
    return (int64_t)cache_page(c, bt_row, pg) * bs + (int64_t)(tok - pg * c.a.block_size) * rs;
  }
  return (int64_t)(k_begin + tok) * rs;
}

// K/V tiles of BN keys that the queries at positions [p_first, p_last] see any key of: `sink` tiles from the start of
// the sequence, then the tiles [win, win + n - sink).
struct TileSpan {
  int sink, win, n;
  __device__ __forceinline__ int tile(int i) const { return i < sink ? i : win + i - sink; }
};
template <int BN>
__device__ __forceinline__ TileSpan tile_span(const CacheAttnArgs& c, int k_len, int p_first, int p_last) {
  const AttnArgs& a = c.a;
  int hi = k_len;                               // keys [0, hi) at most
  if (a.causal || a.wr >= 0) hi = min(hi, p_last + (a.causal ? 0 : a.wr) + 1);
  TileSpan t;
  if (hi <= 0) {
    t.sink = t.win = t.n = 0;
    return t;
  }
  const int lo = a.wl >= 0 ? max(0, min(hi, p_first - a.wl)) : 0;
  t.win = lo / BN;
  t.sink = min((min(c.sinks, hi) + BN - 1) / BN, t.win);
  t.n = t.sink + (hi + BN - 1) / BN - t.win;
  return t;
}

// What one row sees: columns [lo, hi) and [0, sinks).
struct RowMask {
  int lo, hi, sinks;
  __device__ __forceinline__ bool dead(int col) const { return col >= hi || (col < lo && col >= sinks); }
};
__device__ __forceinline__ RowMask row_mask(const CacheAttnArgs& c, int k_len, int p) {
  const AttnArgs& a = c.a;
  RowMask m;
  m.hi = k_len;
  if (a.causal || a.wr >= 0) m.hi = min(m.hi, p + (a.causal ? 0 : a.wr) + 1);
  m.lo = a.wl >= 0 ? max(0, p - a.wl) : 0;
  m.sinks = c.sinks;
  return m;
}

// Place of a token's partial results, which count from the first sequence's first token `q_first` on, so that rows of a padded q
// take no room; -1 for tokens beyond what the sizes of the call allow.
__device__ __forceinline__ int64_t part_row(const CacheAttnArgs& c, int q_first, int64_t qtok) {
  const int64_t row = qtok - q_first;
  return row >= 0 && row < c.part_rows ? row : -1;
}

// What an item of n K/V tiles counts where the tiles of all items are cut into runs.
__device__ __forceinline__ int item_weight(const CacheAttnArgs& c, int n) { return c.whole ? min(n, 1) : n; }

// Power of two (as a float) that takes a row whose largest magnitude is `top` to [2^14, 2^15), and its inverse.
__device__ __forceinline__ void row_power(float top, float& up, float& down) {
  const int e = (int)((__float_as_uint(top) >> 23) & 0xff);   // biased exponent; 0 for zero and subnormals
  if (e == 0xff || top == 0.f) {                               // infinity or NaN: left alone, they stay what they are
    up = down = 1.f;
    return;
  }
  const int k = min(14 - (max(e, 1) - 127), 112);
  up = __int_as_float((127 + k) << 23);
  down = __int_as_float((127 - k) << 23);
}

// log2 of what probabilities of at most 2^most are multiplied by before they are rounded to M.
template <typename M>
__host__ __device__ constexpr float p_shift(float most) {
  return std::is_same<M, __half>::value ? 15.f - most : 0.f;
}

// Kernel families of fg_flash_attn_cache.
int attn_cache_generic(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st);
int attn_cache_decode(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st);
int64_t attn_cache_decode_sm100_bytes(int64_t rows, int64_t head_dim, int sms);
int attn_cache_decode_sm100(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st);
int64_t attn_cache_chunk_bytes(int64_t max_q, int64_t group, int64_t batch, int64_t heads_k, int64_t head_dim, int64_t max_k,
                               int64_t dense, bool whole, int sms);
int attn_cache_chunk(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st);
int attn_cache_combine(const CacheAttnArgs& c, int dtype, cudaStream_t st);

}  // namespace fg
