// fg_flash_attn_cache: argument validation, choice of the kernel family and of the split over the keys.
#include <initializer_list>

#include "attn_cache_common.cuh"

namespace fg {

int* device_status_ptr();

namespace {

enum { kPathGeneric = 0, kPathChunk = 1, kPathDecode = 2, kPathDecodeSm100 = 3 };

struct Plan {
  int path;
  int splits, tiles_per_split;
  int64_t bytes;       // of workspace
  int whole;           // tensor-core kernels: no item is cut
  int64_t dense;       // rows of each sequence in a 16-bit copy of an 8-bit store, or 0
};

// Most tiles of 128 keys of an item for which the tensor-core kernels cut no item: one launch less, and no workspace.  Cut and whole:
// 16 decodes of up to 1000 keys 20.1 and 15.8 us, of up to 2000 21.9 and 22.9 us (2 of them 17.6 and 22.5 us); 16 chunks of up
// to 200 tokens over up to 500 keys 81.7 and 61.9 us, 8 of up to 60 over up to 1000 31.7 and 32.4 us.
constexpr int64_t kWholeDecode = 8, kWholeChunk = 4;

// Fewest tiles of 128 keys, of all sequences and KV heads, for which the decode form on tcgen05 is worth its longer way through a
// tile, which grows with the query rows; below, the mma.sync form splits the keys over more and smaller CTAs.  On mma.sync and on
// tcgen05, 8-bit: 4 rows of 128: 256 tiles 12.3 and 15.6 us, 704 19.7 and 17.2; 8 rows: 704 21.7 and 21.5, 2048 33.8 and 30.5;
// 16 rows: 2048 39.7 and 44.4, 8192 140 and 91; 4 rows of 256: 256 16.4 and 18.2, 704 33.8 and 21.3; 16: 48.7 and 43.6.
int64_t least_decode(int64_t rows, int64_t head_dim) {
  if (head_dim == 256) return 400;
  return rows <= 4 ? 600 : rows <= 8 ? 1800 : 4000;
}

// Most bytes of partial results of the mma.sync decode form, whose splits go by max_seqlen_k: a captured step's bound may be far
// above its contexts, and ranges that no sequence reaches cost an empty CTA and a place in the workspace each.  256 decodes of up to
// 8192 keys (soft-capped, 32 heads over 8) under a bound of 131072 in ranges of 1024 keys, 541 MB, and 16384 keys, 34 MB: 1732 and
// 894 us; under a bound of 10^6 7209 and 898 us.
constexpr int64_t kMostSplitBytes = 64ll << 20;

// Keys that one sequence can have visible to one row tile: everything, or window and first tokens.
int64_t most_keys(const fg_attn_cache_params* p, int64_t tokens) {
  const fg_attn_params& b = p->base;
  if (b.window_left < 0 || b.window_left >= b.max_seqlen_k) return b.max_seqlen_k;
  const int64_t right = b.causal ? 0 : (b.window_right < 0 ? b.max_seqlen_k : b.window_right);
  const int64_t keys = b.window_left + 1 + right + tokens + p->sink_tokens + 3 * 128;   // ends of the tile runs
  return keys < b.max_seqlen_k ? keys : b.max_seqlen_k;
}

// `ctas` row tiles without a split, `tiles` K/V tiles each at most: enough splits to fill `want` CTAs, of at least `least`
// tiles each.
void split_plan(int64_t ctas, int64_t tiles, int64_t want, int64_t least, Plan* plan) {
  int64_t splits = ctas > 0 ? (want + ctas - 1) / ctas : 1;
  if (splits > tiles / least) splits = tiles / least;
  if (splits < 1) splits = 1;
  if (splits > 4096) splits = 4096;
  int64_t per = (tiles + splits - 1) / splits;
  if (per < 1) per = 1;
  plan->tiles_per_split = (int)per;
  plan->splits = (int)((tiles + per - 1) / per);
  if (plan->splits < 1) plan->splits = 1;
}

// Whether TMA can fetch the cache: strides in multiples of 16 bytes, and pages that tile a K/V tile.
bool tma_ready(const fg_attn_cache_params* p) {
  const fg_attn_params& b = p->base;
  const int64_t es = is_fp8(p->cache_dtype) ? 1 : 2;
  for (int64_t st : {b.k_row_stride, b.k_head_stride, b.v_row_stride, b.v_head_stride})
    if (st <= 0 || (st * es) % 16 != 0 || st * es >= (1ll << 40)) return false;
  if (b.block_table == nullptr) return true;
  for (int64_t st : {b.k_block_stride, b.v_block_stride})
    if (st <= 0 || (st * es) % 16 != 0 || st * es >= (1ll << 40)) return false;
  return b.block_size >= 8 && (b.block_size & (b.block_size - 1)) == 0;
}

// Tokens that the split forms' partial results are for: `q` may have many more rows than its sequences.
int64_t part_rows(const fg_attn_params& b) {
  return b.max_seqlen_q <= 0 || b.batch < b.total_q / b.max_seqlen_q ? b.batch * b.max_seqlen_q : b.total_q;
}

// `workspace`: whether the caller has any.
Plan make_plan(const fg_attn_cache_params* p, int sms, bool workspace) {
  const fg_attn_params& b = p->base;
  Plan plan;
  plan.dense = 0;
  plan.whole = 0;
  const int64_t group = b.num_heads / b.num_heads_k;
  const bool tma = tma_ready(p);
  // At head dim 64 an 8-bit store's copy has to pay for itself: 1056 tiles of the general kernel (two chunks of up to 300 tokens)
  // take 21 us there and 29 us with the copy, 15872 (eight of up to 64 tokens over 4000) 152 and 60 us.
  const bool few = b.head_dim == 64 && is_fp8(p->cache_dtype) &&
                   b.batch * b.num_heads_k * ((b.max_seqlen_q * group + 63) / 64) * ((most_keys(p, b.max_seqlen_q) + 63) / 64) < 1536;
  const int64_t key_tiles = (most_keys(p, b.max_seqlen_q) + 127) / 128;
  const bool decode_dim = (b.head_dim == 64 || b.head_dim == 128 || (b.head_dim == 256 && is_fp8(p->cache_dtype))) &&
                          b.batch * b.num_heads_k * key_tiles >= least_decode(b.max_seqlen_q * group, b.head_dim);
  if (b.max_seqlen_q * group <= 16 && tma && decode_dim && b.softcap == 0.0 && (workspace || key_tiles <= kWholeDecode) &&
      b.batch * b.num_heads_k * (b.max_seqlen_k / 128 + 1) <= 2147483647LL) {
    plan.path = kPathDecodeSm100;      // cuts the keys itself, on the device
    plan.splits = plan.tiles_per_split = 1;
    plan.whole = key_tiles <= kWholeDecode;
    plan.bytes = plan.whole ? 0 : attn_cache_decode_sm100_bytes(b.max_seqlen_q * group, b.head_dim, sms);
    return plan;
  }
  const bool chunk_dim = b.head_dim == 64 || b.head_dim == 128 || b.head_dim == 256;
  if (b.max_seqlen_q * group > 16 && tma && !few && chunk_dim && b.softcap == 0.0 && b.softmax_scale > 0.0 && group <= 128 &&
      b.q_head_stride > 0 && b.q_row_stride > 0) {
    plan.path = kPathChunk;            // cuts the keys itself, on the device
    plan.splits = plan.tiles_per_split = 1;
    plan.whole = key_tiles <= kWholeChunk;
    // An 8-bit store is widened once, ahead of the attention, when at least four items (of 256 query rows) read each key and
    // the copy takes at most 1 GiB.  The kernel's own widening is for head dim 128: at the others shorter chunks are too.
    int64_t rows = (b.max_seqlen_k + 63) / 64 * 64;
    if (b.window_left >= 0 && b.window_left < b.max_seqlen_k &&
        (b.causal || (b.window_right >= 0 && b.window_right < b.max_seqlen_k))) {
      const int64_t right = b.causal ? 0 : b.window_right;   // first tokens, then the keys of all new tokens' windows
      const int64_t seen = (p->sink_tokens + 63) / 64 * 64 + (b.window_left + right + b.max_seqlen_q + 2 * 63) / 64 * 64;
      if (seen < rows) rows = seen;
    }
    if (!(p->flags & FG_CACHE_NO_COPY) && is_fp8(p->cache_dtype) &&
        (b.max_seqlen_q * group >= 1024 || b.head_dim != 128) && rows > 0 &&
        b.batch * rows <= (1ll << 30) / (4 * b.head_dim * b.num_heads_k))
      plan.dense = rows;
    plan.bytes = attn_cache_chunk_bytes(b.max_seqlen_q, group, b.batch, b.num_heads_k, b.head_dim, b.max_seqlen_k, plan.dense,
                                        plan.whole, sms);
    if (plan.bytes >= 0 && (workspace || plan.bytes == 0) && (!is_fp8(p->cache_dtype) || b.head_dim == 128 || plan.dense > 0))
      return plan;
    plan.dense = plan.whole = 0;
  }
  if (b.max_seqlen_q * group <= 16 && tma) {
    // Enough CTAs to balance contexts of very different length over all SMs (two resident each), but no range shorter
    // than 256 keys.
    plan.path = kPathDecode;
    const int64_t bn = is_fp8(p->cache_dtype) ? 128 : 64;
    const int64_t keys = most_keys(p, b.max_seqlen_q), ctas = b.num_heads_k * b.batch;
    int64_t chunk = 1024;
    while (chunk > 256 && ctas * ((keys + chunk - 1) / chunk) < (int64_t)sms * 2 * 8) chunk >>= 1;
    const int64_t split_bytes = (part_rows(b) > 0 ? part_rows(b) : 1) * b.num_heads * (b.head_dim + 1) * 4;
    while (chunk < keys && (keys + chunk - 1) / chunk > kMostSplitBytes / split_bytes) chunk <<= 1;
    plan.tiles_per_split = (int)(chunk / bn);
    plan.splits = (int)((keys + chunk - 1) / chunk);
    if (plan.splits < 1) plan.splits = 1;
  } else {
    plan.path = kPathGeneric;
    const int64_t mb = (b.max_seqlen_q * group + 63) / 64;
    const int64_t tiles = (most_keys(p, 64 / group + 1) + 63) / 64;
    split_plan(mb * b.num_heads_k * b.batch, tiles, (int64_t)sms * 2, 4, &plan);
  }
  if (!workspace) plan.splits = 1;
  plan.bytes = plan.splits > 1 ? (int64_t)plan.splits * part_rows(b) * b.num_heads * (b.head_dim + 1) * 4 : 0;
  return plan;
}

bool sizes_ok(const fg_attn_cache_params* p) {
  const fg_attn_params& b = p->base;
  return b.batch >= 0 && b.total_q >= 0 && b.num_heads > 0 && b.num_heads_k > 0 && b.num_heads % b.num_heads_k == 0 &&
         b.head_dim > 0 && b.head_dim <= 256 && b.head_dim % 8 == 0 && b.max_seqlen_q >= 0 && b.max_seqlen_k >= 0 &&
         b.max_seqlen_q <= 2147483647LL / 64 && b.max_seqlen_k <= 2147483647LL / 64 && p->sink_tokens >= 0 &&
         b.batch <= 2147483647LL && b.num_heads <= 2147483647LL && b.total_q <= 2147483647LL * 4 / b.num_heads;
}

}  // namespace
}  // namespace fg

extern "C" int fg_flash_attn_cache_path(const fg_attn_cache_params* p) {
  using namespace fg;
  return p && sizes_ok(p) ? make_plan(p, num_sms(), true).path : 0;
}

extern "C" int64_t fg_flash_attn_cache_workspace_bytes(const fg_attn_cache_params* p) {
  using namespace fg;
  if (p == nullptr || !sizes_ok(p)) return 0;
  return make_plan(p, num_sms(), true).bytes;
}

extern "C" int fg_flash_attn_cache(const fg_attn_cache_params* p, void* stream) {
  using namespace fg;
  FG_REQUIRE_HEALTHY("flash_attn_cache");
  FG_REQUIRE(p != nullptr, "flash_attn_cache: null params");
  const fg_attn_params& b = p->base;
  FG_REQUIRE(b.dtype == FG_F16 || b.dtype == FG_BF16, "FlashAttention only support fp16 and bf16 data type");
  FG_REQUIRE(p->cache_dtype == b.dtype || is_fp8(p->cache_dtype),
             "flash_attn_cache: the cache must hold the type of the queries or an 8-bit type");
  FG_REQUIRE(is_fp8(p->cache_dtype) || (p->k_scale == nullptr && p->v_scale == nullptr),
             "flash_attn_cache: scales belong to an 8-bit cache");
  FG_REQUIRE((p->flags & ~FG_CACHE_NO_COPY) == 0, "flash_attn_cache: unknown flags %d", p->flags);
  FG_REQUIRE(b.batch >= 0 && b.total_q >= 0, "flash_attn_cache: negative size");
  FG_REQUIRE(b.num_heads > 0 && b.num_heads_k > 0, "flash_attn_cache: head counts must be positive");
  FG_REQUIRE(b.num_heads % b.num_heads_k == 0, "Number of heads in key/value must divide number of heads in query");
  FG_REQUIRE(b.head_dim > 0 && b.head_dim <= 256, "FlashAttention forward only supports head dimension at most 256");
  FG_REQUIRE(b.head_dim % 8 == 0, "head_size must be a multiple of 8");
  FG_REQUIRE(p->sink_tokens >= 0, "flash_attn_cache: sink_tokens must not be negative");
  FG_REQUIRE(b.max_seqlen_q >= 0 && b.max_seqlen_k >= 0, "flash_attn_cache: negative max_seqlen");
  FG_REQUIRE(sizes_ok(p) && b.total_q <= 2147483647LL, "flash_attn_cache: sequence too long, or too many rows");
  FG_REQUIRE(b.alibi_slopes == nullptr, "flash_attn_cache: ALiBi is not supported over an 8-bit cache or with sink_tokens");
  FG_REQUIRE((b.q_batch_stride | b.k_batch_stride | b.v_batch_stride | b.o_batch_stride) == 0,
             "flash_attn_cache: batch strides are not supported");
  FG_REQUIRE(b.softcap >= 0.0, "flash_attn_cache: softcap must be >= 0");
  if (b.batch == 0 || b.total_q == 0 || b.max_seqlen_q == 0) return FG_OK;
  FG_REQUIRE(b.batch <= 65535 && b.num_heads_k <= 65535, "flash_attn_cache: batch or heads above 65535");
  FG_REQUIRE(b.q && b.k && b.v && b.out, "flash_attn_cache: null tensor");
  FG_REQUIRE(b.cu_seqlens_q != nullptr, "flash_attn_cache: cu_seqlens_q is required");
  const bool paged = b.block_table != nullptr;
  if (paged) {
    FG_REQUIRE(b.seqused_k != nullptr, "seqused_k must be provided if block_table is provided");
    FG_REQUIRE(b.block_size > 0 && b.num_blocks > 0, "flash_attn_cache: paged KV needs block_size and num_blocks");
    FG_REQUIRE(b.block_size <= 2147483647LL && b.num_blocks <= 2147483647LL, "flash_attn_cache: cache too large");
    FG_REQUIRE(p->block_table_cols > 0 && p->block_table_cols <= 2147483647LL, "flash_attn_cache: block_table has no columns");
  } else {
    FG_REQUIRE(b.cu_seqlens_k != nullptr, "cu_seqlens_k or seqused_k must be provided");
    FG_REQUIRE(b.total_k >= 0 && b.total_k <= 2147483647LL, "flash_attn_cache: bad total_k");
  }
  FG_REQUIRE(aligned16(b.q) && aligned16(b.k) && aligned16(b.v) && aligned16(b.out),
             "flash_attn_cache: tensors must be 16-byte aligned");
  FG_REQUIRE(b.q_row_stride % 8 == 0 && b.q_head_stride % 8 == 0 && b.k_row_stride % 8 == 0 && b.k_head_stride % 8 == 0 &&
                 b.v_row_stride % 8 == 0 && b.v_head_stride % 8 == 0 && b.o_row_stride % 8 == 0 &&
                 b.o_head_stride % 8 == 0 && (!paged || (b.k_block_stride % 8 == 0 && b.v_block_stride % 8 == 0)),
             "flash_attn_cache: strides must be multiples of 8 elements");

  CacheAttnArgs c;
  AttnArgs& a = c.a;
  a.q = b.q; a.k = b.k; a.v = b.v; a.out = b.out; a.lse = b.lse;
  a.cu_q = b.cu_seqlens_q; a.cu_k = b.cu_seqlens_k; a.seqused_k = b.seqused_k;
  a.block_table = b.block_table; a.alibi = nullptr;
  a.q_rs = b.q_row_stride; a.q_hs = b.q_head_stride;
  a.k_rs = b.k_row_stride; a.k_hs = b.k_head_stride; a.k_bs = b.k_block_stride;
  a.v_rs = b.v_row_stride; a.v_hs = b.v_head_stride; a.v_bs = b.v_block_stride;
  a.o_rs = b.o_row_stride; a.o_hs = b.o_head_stride;
  a.bt_stride = b.block_table_stride; a.alibi_bs = 0;
  a.total_q = b.total_q; a.total_k = b.total_k;
  a.q_batch = a.k_batch = a.v_batch = a.o_batch = 0;
  a.batch_strided = 0;
  a.batch = (int)b.batch; a.H = (int)b.num_heads; a.Hk = (int)b.num_heads_k;
  a.group = a.H / a.Hk; a.D = (int)b.head_dim;
  a.max_q = (int)b.max_seqlen_q; a.max_k = (int)b.max_seqlen_k;
  a.block_size = (int)b.block_size; a.num_blocks = (int)b.num_blocks;
  a.paged = paged;
  a.has_alibi = 0;
  a.causal = b.causal != 0;
  int64_t wl = b.window_left, wr = b.window_right;
  if (a.causal) wr = 0;
  // Bounds that hide nothing: the last token is at k_len - 1, the first at k_len - q_len, which is negative where there are more new
  // tokens than keys.
  if (wl >= b.max_seqlen_k) wl = -1;
  if (wr >= b.max_seqlen_q - 1) wr = -1;
  a.wl = (int)(wl < 0 ? -1 : wl);
  a.wr = (int)(wr < 0 ? -1 : wr);
  a.local = a.wl >= 0 || (!a.causal && a.wr >= 0);
  a.has_softcap = b.softcap > 0.0;
  const double LOG2E = 1.4426950408889634074;
  a.scale = (float)(a.has_softcap ? b.softcap : b.softmax_scale);
  a.softcap_pre = a.has_softcap ? (float)(b.softmax_scale / b.softcap) : 0.f;
  a.scale_log2 = (float)((a.has_softcap ? b.softcap : b.softmax_scale) * LOG2E);
  a.status = device_status_ptr();
  c.k_scale = p->k_scale; c.v_scale = p->v_scale;
  c.ks_batch = p->k_scale_batch_stride; c.ks_head = p->k_scale_head_stride;
  c.vs_batch = p->v_scale_batch_stride; c.vs_head = p->v_scale_head_stride;
  c.sinks = a.wl < 0 ? 0 : (int)(p->sink_tokens < b.max_seqlen_k ? p->sink_tokens : b.max_seqlen_k);
  c.table_cols = (int)p->block_table_cols;

  const Plan plan = make_plan(p, num_sms(), b.workspace != nullptr);
  a.ws_o = nullptr;
  a.ws_lse = nullptr;
  if (plan.bytes > 0) {
    FG_REQUIRE(b.workspace_bytes >= plan.bytes, "flash_attn_cache: workspace of %lld bytes, %lld needed",
               (long long)b.workspace_bytes, (long long)plan.bytes);
    FG_REQUIRE(aligned16(b.workspace), "flash_attn_cache: workspace must be 16-byte aligned");
    a.ws_o = reinterpret_cast<float*>(b.workspace);
    a.ws_lse = a.ws_o + (int64_t)plan.splits * part_rows(b) * b.num_heads * b.head_dim;   // split forms only
  }
  a.num_splits = plan.splits;
  c.tiles_per_split = plan.tiles_per_split;
  c.part_rows = part_rows(b);
  c.dense = plan.dense;
  c.whole = plan.whole;
  const int kind = p->cache_dtype == FG_E4M3 ? kCacheE4M3 : p->cache_dtype == FG_E5M2 ? kCacheE5M2 : kCache16;
  cudaStream_t st = (cudaStream_t)stream;
  FG_REQUIRE((b.max_seqlen_q * a.group + 63) / 64 * plan.splits <= 2147483647LL, "flash_attn_cache: too many row tiles");
  const int rc = plan.path == kPathDecodeSm100 ? attn_cache_decode_sm100(c, b.dtype, kind, st)
                 : plan.path == kPathDecode    ? attn_cache_decode(c, b.dtype, kind, st)
                 : plan.path == kPathChunk     ? attn_cache_chunk(c, b.dtype, kind, st)
                                               : attn_cache_generic(c, b.dtype, kind, st);
  if (rc != FG_OK || a.num_splits == 1) return rc;
  return attn_cache_combine(c, b.dtype, st);
}
