// Attention of a chunk of new tokens over an 8-bit or windowed cache, head dim 64, 128 or 256, on the tcgen05 tensor cores.
//
// An item is one or two 128-row Q tiles of one (sequence, KV head).  A row is a (token, head of the group) pair, so a chunk of a
// few tokens fills the tiles as well as a long one, and all query heads of the group share every K/V tile.  A tile holds
// floor(128 / group) tokens (at head dim 256 an item is one tile).  The kernel is persistent, one CTA an SM: the K/V tiles (64
// keys) of all items, laid end to end, are cut into equal runs, one per CTA, so that few long items and many short ones fill the
// SMs alike (in whole items, 336 CTAs on 148 SMs would take three rounds for 2.27).  Short items are not cut (attn_cache_api.cu
// has the rule).  The parts of an item that runs cut are joined by a second kernel, in order.  Nothing synchronises the CTA
// between items: the roles follow the barrier phases with running counters.
//
//   warps 0-7    softmax, one warpgroup per Q tile, one thread per row (TMEM lane = row): scores of 64 keys from TMEM to
//                registers, mask, running maximum (raised only when it grows by more than 8 in log2 units), exponentials,
//                probabilities back to TMEM as 16 bit; at the end they normalise and write the output rows
//   16-bit caches:
//   warps 8, 9   TMA producers of K (and Q) and of V, walking the tile runs (first tokens, then the window).  A page of 16 keys is
//                two boxes, and a warp issues one in about 95 clocks: one warp for both would need 1900 clocks a tile
//   warp 10      scores of both Q tiles: S = Q K^T, 64 keys a step
//   8-bit caches (head dim 128):
//   warp 8       TMA producer of Q; warps 9, 10 the scores of one Q tile each
//   warps 12-15  load K and V rows (one tile ahead, in registers), widen them to fp16 and store them as the 128-byte
//                swizzled tiles that the tensor cores read; rows that no row of the item sees are neither read nor kept.
//                (Landing the 8-bit tiles in shared memory by TMA first costs two more waits and a read for each: two chunks
//                of 2048 tokens took 789 us, 663 us so.)
//   warp 11      O += P V of both tiles
// Widening inside the kernel makes a step half as long again, and every item widens the keys it reads anew.  Where the chunk is
// long (several items read each key) and the store's 16-bit copy is not too large, a kernel before this one widens the visible
// rows once into the workspace, and this one reads them as a 16-bit store (attn_cache_api.cu has the rule; two chunks of 2048
// tokens 513 to 529 us, the copy included).  At head dims 64 and 256 that is the only form.
// What bounds it: with two Q tiles of head dim 128 a step of 64 keys is 2 x 2 products of 128 x 64 x 128, 1024 clocks of the tensor
// cores at 4096 multiply-adds a clock, and 16384 exponentials, 1024 clocks of the special function units at 16 a clock.  Long
// chunks reach half of a large library product's rate, since each of the two waits for the other at times (tensor pipe and
// special-function unit 36 to 38 % busy); short ones over an 8-bit cache by the latency of the widening warps' loads, one tile on
// its way behind its table entries (23 %; DRAM 15 %).
// Two 2048-token prompts at head dim 256 607 us, at 64 202 us (mma.sync: 1654 and 343).
// Over 8-bit caches bf16 queries are brought to fp16, each row by a power of two, by the softmax warps before an item's first
// step.
// P is rounded once: to fp16 (2^-12 of itself, or 2^-32 of its row's largest), and over a bf16 cache to bf16 (2^-9): a second
// piece, which the decode kernel has, would double the products P V, and those bound the step.
// TMEM columns: tile t has its scores at t*128 (64 columns), two probability buffers at t*128+64 and +96, its output at
// 256+t*128.  Every wait is an mbarrier wait with a limit.
#include "attn_cache_common.cuh"
#include "sm100_common.cuh"

namespace fg {
namespace {

constexpr int BM = 128, BN = 64;
constexpr int HALF_BYTES = 128 * 64 * 2;     // one [128 x 64] swizzled 16-bit piece of a Q tile
constexpr int UNIT_HALF = BN * 128;          // one [64 keys x 64 columns] swizzled piece of a 16-bit K or V tile
constexpr int TMA_WARP = 8, MMA_WARP0 = 9, PV_WARP = 11, CONV_WARP0 = 12;
constexpr int TMEM_COLS = 512;
constexpr float kRescaleThreshold = 8.0f;    // log2 units

// Fewest K/V tiles that a run is worth starting a CTA for: 4 chunks of 20 to 60 tokens take 26.8 us with 8, 22.7 with 4, 22.3 with 2;
// 2 of up to 300 tokens 30.1, 25.4 and 27.0 us.
constexpr int kMinRun = 4;
constexpr int kInfo = 32;                    // sequences of a run whose lengths are kept in shared memory

constexpr int threads_of(int kind) { return kind == kCache16 ? 12 * 32 : 16 * 32; }

// By head dim.  At 256 a Q tile takes 64 KB of shared memory and its output half of the tensor memory: one tile, two stages.
template <int HD>
struct Shape {
  static constexpr int PIECES = HD / 64;                   // 64-column pieces of a row
  static constexpr int TILES = HD > 128 ? 1 : 2;           // Q tiles of an item, at most
  static constexpr int TILE_BYTES = PIECES * HALF_BYTES;   // a Q tile
  static constexpr int UNIT = PIECES * UNIT_HALF;          // a 16-bit K or V tile
  static constexpr int STAGES = HD > 128 ? 2 : 4;          // tiles of K, and of V
  static constexpr int SMEM = TILES * TILE_BYTES + 2 * STAGES * UNIT + 1024 + 512 + kInfo * 16;
};

// What a CTA leaves for the joining kernel: the KV head of the item whose start it holds but not its end (or -1), in how many
// parts the item is, its first query row and its tokens.
struct PartRecord {
  int hk, parts, q_row, tokens;
};

struct ChunkArgs {
  CacheAttnArgs c;
  int tiles;            // Q tiles of an item (1 or 2)
  int tokens;           // tokens of a Q tile
  int page_rows;        // keys per TMA box
  int pages_per_tile;
  int num_mb;           // items of the longest chunk, for each KV head
  float* part_o;        // [2 * CTAs][tiles * 128][128]: head part, tail part of each CTA
  float* part_lse;      // [2 * CTAs][tiles * 128]
  PartRecord* record;   // [CTAs]
};

// One item's part of a CTA's run.
struct Segment {
  int b, m, hk, lo, hi, n;      // K/V tiles [lo, hi) of the n of (sequence b, Q tiles m, KV head hk)
  int left;                     // tiles of the run from lo on
  int m0, nt, shift;            // first token; Q tiles that hold one; position of token 0
  int gap;                      // 16-bit copy of an 8-bit store: rows between first tokens and window that it leaves out
  SeqInfo s;
  TileSpan span;
  RowMask first, last;          // what the first and the last token see
};
__device__ __forceinline__ int item_tiles(const ChunkArgs& pa, const SeqInfo& s, int m, TileSpan& span) {
  const int m0 = m * pa.tiles * pa.tokens;
  if (m0 >= s.q_len) return 0;
  const int shift = s.k_len - s.q_len;
  span = tile_span<BN>(pa.c, s.k_len, m0 + shift, min(s.q_len, m0 + pa.tiles * pa.tokens) - 1 + shift);
  return max(span.n, 1);        // nothing visible: one tile, all of it masked, gives the zeros
}
// The 16-bit copy of an 8-bit store holds the tiles that some query of the sequence sees, without a gap between the first tokens
// and the window: tokens from `win` on come `gap` rows earlier.
struct CopySpan {
  int win, gap;
};
__device__ __forceinline__ CopySpan copy_span(const CacheAttnArgs& c, const SeqInfo& s) {
  const TileSpan t = tile_span<BN>(c, s.k_len, s.k_len - s.q_len, s.k_len - 1);
  return CopySpan{t.win * BN, (t.win - t.sink) * BN};
}
// Lengths of the sequences [b0, b0 + n) as the CTA found them at its start; the others come from global memory.
struct InfoTable {
  const SeqInfo* info;
  int b0, n;
};
__device__ __forceinline__ void set_part(const ChunkArgs& pa, Segment& g, int lo) {
  g.lo = lo;
  g.hi = pa.c.whole ? g.n : min(g.n, lo + g.left);
}
__device__ __forceinline__ void fill_segment(const ChunkArgs& pa, const InfoTable& table, Segment& g) {
  g.s = (unsigned)(g.b - table.b0) < (unsigned)table.n ? table.info[g.b - table.b0] : cache_seq_info(pa.c, g.b);
  g.n = item_tiles(pa, g.s, g.m, g.span);
  g.m0 = g.m * pa.tiles * pa.tokens;
  g.nt = g.m0 + pa.tokens < g.s.q_len ? pa.tiles : 1;
  g.shift = g.s.k_len - g.s.q_len;
  g.first = row_mask(pa.c, g.s.k_len, g.m0 + g.shift);
  g.last = row_mask(pa.c, g.s.k_len, min(g.s.q_len, g.m0 + pa.tiles * pa.tokens) - 1 + g.shift);
  g.gap = pa.c.dense > 0 ? copy_span(pa.c, g.s).gap : 0;
}
// The part after `g`, in place; false when the run ends with g.
__device__ __forceinline__ bool next_segment(const ChunkArgs& pa, const InfoTable& table, Segment& g) {
  g.left -= item_weight(pa.c, g.hi - g.lo);
  if (g.left <= 0) return false;
  if (++g.hk == pa.c.a.Hk) {
    g.hk = 0;
    do {
      if (++g.m == pa.num_mb) {
        g.m = 0;
        if (++g.b >= pa.c.a.batch) return false;
      }
      fill_segment(pa, table, g);
    } while (g.n == 0);
  }
  set_part(pa, g, 0);
  return true;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));   // volatile: back to back, in program order
  return y;
}
__device__ __forceinline__ uint64_t pack2f(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void fma2(float& a0, float& a1, uint64_t sc, uint64_t ng) {
  asm("{\n .reg .b64 x, r;\n mov.b64 x, {%0, %1};\n fma.rn.f32x2 r, x, %2, %3;\n mov.b64 {%0, %1}, r;\n}\n"
      : "+f"(a0), "+f"(a1)
      : "l"(sc), "l"(ng));
}
__device__ __forceinline__ void add2(float& s0, float& s1, float p0, float p1) {
  asm("{\n .reg .b64 x, y, r;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n add.rn.f32x2 r, x, y;\n mov.b64 {%0, %1}, r;\n}\n"
      : "+f"(s0), "+f"(s1)
      : "f"(p0), "f"(p1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// T: type of q and out; KIND: what K and V are read as; M: type of the products; HD: head dim
template <typename T, int KIND, typename M, int HD>
__global__ void __launch_bounds__(threads_of(KIND), 1)
attn_cache_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ ChunkArgs pa) {
  using namespace sm100;
  constexpr bool kBf16 = std::is_same<M, __nv_bfloat16>::value;
  constexpr bool kConvQ = !std::is_same<T, M>::value;
  constexpr bool kWiden = KIND != kCache16;
  constexpr int THREADS = threads_of(KIND);
  constexpr float kShift = p_shift<M>(kRescaleThreshold);
  using G = Shape<HD>;
  constexpr int PIECES = G::PIECES, TILE_BYTES = G::TILE_BYTES, UNIT = G::UNIT, STAGES = G::STAGES;
  static_assert(!kWiden || HD == 128, "the widening warps take rows of 128");
  const CacheAttnArgs& c = pa.c;
  const AttnArgs& a = c.a;
  const int NT = pa.tiles;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // [tiles][pieces][128 x 64]
  uint8_t* sK = smem + G::TILES * TILE_BYTES;   // [STAGES]
  uint8_t* sV = sK + STAGES * UNIT;         // [STAGES]
  uint8_t* rest = sV + STAGES * UNIT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(rest);
  uint64_t* q_full = bars;            // Q tiles of an item have landed
  uint64_t* q_empty = bars + 1;       // every score of an item has been computed: Q may be overwritten
  uint64_t* k_full = bars + 2;        // [STAGES]
  uint64_t* k_empty = bars + 6;
  uint64_t* v_full = bars + 10;
  uint64_t* v_empty = bars + 14;
  uint64_t* s_full = bars + 18;       // [2 tiles] scores of a step have landed in the tile's score buffer
  uint64_t* s_free = bars + 20;       // [2 tiles] ... and have been read into registers
  uint64_t* p_ready = bars + 22;      // [2 tiles][2 probability buffers]
  uint64_t* o_done = bars + 26;       // [2 tiles][2]: P V of even / odd steps
  uint64_t* q_ready = bars + 30;      // [2 tiles] the tile's Q holds M
  uint64_t* o_free = bars + 32;       // [2 tiles] the output of the previous item has been read out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SeqInfo* sInfo = reinterpret_cast<SeqInfo*>(rest + 512);   // [kInfo]

  __shared__ int s_drain, s_sum[THREADS / 32], s_top[THREADS / 32], s_off, s_pair;
  // ---- this CTA's run: tiles [begin, begin + run) of all items' tiles; a pair is (sequence, Q tiles), the items of a pair are
  // its KV heads
  const int pairs = a.batch * pa.num_mb;
  TileSpan span;
  int mine = 0, longest = 0;
  if (tid < pairs) {
    longest = item_tiles(pa, cache_seq_info(c, tid / pa.num_mb), tid % pa.num_mb, span);
    mine = item_weight(c, longest) * a.Hk;
  }
  if (tid == 0) {
    s_drain = *reinterpret_cast<volatile int*>(a.status);
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, kWiden ? NT : 1);   // one arrival per score-issuing thread
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_full[i], kWiden ? 4 : 1);
      mbar_init(&k_empty[i], kWiden ? NT : 1);
      mbar_init(&v_full[i], kWiden ? 4 : 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);       // one arrival per softmax warp of the tile
      mbar_init(&q_ready[i], 4);
      mbar_init(&o_free[i], 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_ready[i], 4);
    for (int i = 0; i < 4; ++i) mbar_init(&o_done[i], 1);
    mbar_fence_init();
    prefetch_tmap(&tmap_q);
    if constexpr (!kWiden) {
      prefetch_tmap(&tmap_k);
      prefetch_tmap(&tmap_v);
    }
  }
  int total = mine;
  for (int p = tid + THREADS; p < pairs; p += THREADS) {
    const int n = item_tiles(pa, cache_seq_info(c, p / pa.num_mb), p % pa.num_mb, span);
    longest = max(longest, n);
    total += item_weight(c, n) * a.Hk;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) {
    s_sum[warp] = total;
    s_top[warp] = longest;
  }
  __syncthreads();
  if (s_drain != 0) return;   // a wait gave up on this device: finish the launch quickly
  total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    total += s_sum[i];
    longest = max(longest, s_top[i]);
  }
  // Short items need not share a CTA.  An item of n tiles in n / run parts takes about 1 us a tile and 0.5 us a part to join: run is
  // at least the root of n / 2 (20 tokens over 16000 keys: 55 us in runs of 4 tiles, 38 in runs of 11).
  const int min_run = c.whole ? 1 : max(min(kMinRun, longest), (int)sqrtf(0.5f * longest));
  const int run = max((total + (int)gridDim.x - 1) / (int)gridDim.x, max(min_run, 1));
  const int64_t begin = (int64_t)run * blockIdx.x;
  if (begin >= total) {
    if (tid == 0 && !c.whole) pa.record[blockIdx.x] = PartRecord{-1, 0, 0, 0};
    return;
  }
  int before = 0;
  for (int p0 = 0;; p0 += THREADS) {
    if (p0 > 0) {
      const int p = p0 + tid;
      mine = p < pairs ? item_weight(c, item_tiles(pa, cache_seq_info(c, p / pa.num_mb), p % pa.num_mb, span)) * a.Hk : 0;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int base = before;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) base += s_sum[i];
      before += s_sum[i];
    }
    if (mine > 0 && base + incl - mine <= begin && begin < base + incl) {
      s_pair = p0 + tid;
      s_off = (int)begin - (base + incl - mine);
    }
    if (before > begin) break;
  }
  if (warp == MMA_WARP0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  Segment seg;
  seg.b = s_pair / pa.num_mb;
  seg.m = s_pair - seg.b * pa.num_mb;
  const InfoTable table{sInfo, seg.b, min(kInfo, a.batch - seg.b)};
  if (tid < table.n) sInfo[tid] = cache_seq_info(c, seg.b + tid);
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;");   // the joining kernel may be set up: it waits for this one's end
  seg.left = min(total - (int)begin, run);
  fill_segment(pa, table, seg);
  const int weight = item_weight(c, seg.n);
  seg.hk = s_off / weight;
  set_part(pa, seg, s_off - seg.hk * weight);

  auto wait1 = [&](uint64_t* bar, uint32_t parity) -> bool {
    return mbar_wait(bar, parity, abort_flag, a.status, kStatusAttnTimeout);
  };
  // lane 0 polls for its warp, so that a wait that gave up takes the whole warp the same way
  auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool {
    int r = 1;
    if (lane == 0) r = wait1(bar, parity) ? 1 : 0;
    r = __shfl_sync(0xffffffffu, r, 0);
    __syncwarp();   // what lane 0 has seen arrive is there for the others
    return r != 0;
  };

  if (warp == TMA_WARP || (!kWiden && warp == TMA_WARP + 1)) {
    // ================================ TMA producers of K and Q, and of V ===========
    const bool is_v = warp != TMA_WARP;
    // Lane i holds the place of the i-th page of a tile, or -1 where no row of the item sees any of its keys: such a page is
    // not fetched (its scores are masked and its V rows zeroed).
    auto lookup = [&](int j, int& page, int& row) {
      const int tok = seg.span.tile(j) * BN + lane * pa.page_rows;
      page = -1;
      row = seg.s.k_begin + tok - (j < seg.span.sink ? 0 : seg.gap);
      if (lane >= pa.pages_per_tile || tok >= seg.last.hi || (tok + pa.page_rows <= seg.first.lo && tok >= c.sinks)) return;
      page = 0;
      if (c.pages()) {
        const int pg = tok / a.block_size;
        row = tok - pg * a.block_size;
        page = cache_page(c, a.block_table + (int64_t)seg.b * a.bt_stride, pg);
      }
    };
    const CUtensorMap* tm = is_v ? &tmap_v : &tmap_k;
    uint8_t* ring = is_v ? sV : sK;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    uint32_t item = 0, kv = 0;     // items and K/V tiles so far
    bool ok = true;
    do {
      int page = -1, row = 0;
      if constexpr (!kWiden) lookup(seg.lo, page, row);
      if (!is_v) {
        if (item > 0 && !wwait(q_empty, (item - 1) & 1)) break;
        if (lane == 0) {
          mbar_expect_tx(q_full, seg.nt * PIECES * pa.tokens * a.group * 128);
          for (int t = 0; t < seg.nt; ++t)
            for (int hf = 0; hf < PIECES; ++hf)
              tma_load_3d(sQ + t * TILE_BYTES + hf * HALF_BYTES, &tmap_q, q_full, hf * 64, seg.hk * a.group,
                          seg.s.q_begin + seg.m0 + t * pa.tokens);
        }
        __syncwarp();
        ++item;
      }
      if constexpr (!kWiden) {
        for (int j = seg.lo; j < seg.hi; ++j, ++kv) {
          int npage = -1, nrow = 0;
          if (j + 1 < seg.hi) lookup(j + 1, npage, nrow);   // in flight while this tile is issued
          const int pages = __popc(__ballot_sync(0xffffffffu, page >= 0));
          const uint32_t stg = kv % STAGES;
          if (!wwait(&empty[stg], ((kv / STAGES) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(&full[stg], pages * pa.page_rows * (HD * 2));
          __syncwarp();
          if (page >= 0) {
            uint8_t* dst = ring + stg * UNIT + lane * pa.page_rows * 128;
            for (int hf = 0; hf < PIECES; ++hf) tma_load_4d(dst + hf * UNIT_HALF, tm, &full[stg], hf * 64, seg.hk, row, page);
          }
          page = npage;
          row = nrow;
        }
      }
    } while (ok && next_segment(pa, table, seg));
  } else if (kWiden ? warp >= MMA_WARP0 && warp < MMA_WARP0 + NT : warp == MMA_WARP0 + 1) {
    // ================================ scores =======================================
    if (lane == 0) {
      constexpr int TILES = kWiden ? 1 : 2;              // Q tiles of this thread
      const int t0 = kWiden ? warp - MMA_WARP0 : 0;
      const uint32_t idesc = umma_idesc_f16(kBf16, false, false, BM, BN);
      const uint32_t desc_hi = (uint32_t)(umma_desc_sw128(0, 0, 1024) >> 32);
      const uint32_t k_lo0 = (uint32_t)umma_desc_sw128(smem_u32(sK), 0, 1024);
      uint32_t item = 0, kv = 0, g[TILES] = {};   // items, K/V tiles, and steps of each Q tile so far
      bool ok = true;
      do {
        // (of every Q tile of this thread, whether it holds a token or not)
        ok = wait1(kConvQ ? &q_ready[t0] : q_full, item & 1) &&
             (!kConvQ || t0 + TILES > NT || TILES == 1 || wait1(&q_ready[1], item & 1));
        ++item;
        for (int i = seg.lo; i < seg.hi && ok; ++i, ++kv) {
          const uint32_t stg = kv % STAGES;
          if (!wait1(&k_full[stg], (kv / STAGES) & 1)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int x = 0; x < TILES; ++x) {
            const int t = t0 + x;
            if (t >= seg.nt || !ok) continue;
            // the previous step's scores must have been read out; and the softmax warps will store P over the buffer that the
            // P V two steps back reads (steps 0 and 1: the softmax warps waited for the previous item's last P V)
            if ((g[x] > 0 && !wait1(&s_free[t], (g[x] - 1) & 1)) ||
                (i >= seg.lo + 2 && !wait1(&o_done[t * 2 + (g[x] & 1)], ((g[x] - 2) >> 1) & 1))) {
              ok = false;
              continue;
            }
            tc_fence_after();
            const uint32_t q_lo = (uint32_t)umma_desc_sw128(smem_u32(sQ + t * TILE_BYTES), 0, 1024);
            const uint32_t k_lo = k_lo0 + stg * (UNIT >> 4);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              mma_f16_ss_lohi(tmem_base + t * 128, q_lo + (((k >> 2) * HALF_BYTES + (k & 3) * 32) >> 4),
                              k_lo + (((k >> 2) * UNIT_HALF + (k & 3) * 32) >> 4), desc_hi, idesc, k != 0 ? 1u : 0u);
            tc_commit(&s_full[t]);
            ++g[x];
          }
          if (!ok) break;
          tc_commit(&k_empty[stg]);
          if (i == seg.hi - 1) tc_commit(q_empty);
        }
      } while (ok && next_segment(pa, table, seg));
    }
  } else if (warp == PV_WARP) {
    // ================================ O += P V of both tiles =======================
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_f16(kBf16, false, true, BM, HD);   // V is MN-major
      const uint32_t desc_hi = (uint32_t)(umma_desc_sw128(0, 0, 1024) >> 32);
      const uint32_t v_lo0 = (uint32_t)umma_desc_sw128(smem_u32(sV), UNIT_HALF, 1024);
      uint32_t used[2] = {0, 0}, kv = 0, g[2] = {0, 0};
      bool ok = true;
      do {
        for (int i = seg.lo; i < seg.hi && ok; ++i, ++kv) {
          const uint32_t stg = kv % STAGES;
          if (!wait1(&v_full[stg], (kv / STAGES) & 1)) {
            ok = false;
            break;
          }
          const uint32_t v_lo = v_lo0 + stg * (UNIT >> 4);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= seg.nt || !ok) continue;
            const uint32_t par = g[t] & 1;
            // the first product of an item overwrites O: the previous item's must have been read out
            if (!wait1(&p_ready[t * 2 + par], (g[t] >> 1) & 1) ||
                (i == seg.lo && used[t] > 0 && !wait1(&o_free[t], (used[t] - 1) & 1))) {
              ok = false;
              continue;
            }
            tc_fence_after();
            const uint32_t p_tmem = tmem_base + t * 128 + BN + par * 32;
            const uint32_t o_tmem = tmem_base + 256 + t * 128;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16_ts_lohi(o_tmem, p_tmem + k * 8, v_lo + k * (2048 >> 4), desc_hi, idesc, (i > seg.lo || k > 0) ? 1u : 0u);
            tc_commit(&o_done[t * 2 + par]);
            ++g[t];
          }
          if (ok) tc_commit(&v_empty[stg]);
        }
        ++used[0];
        used[1] += seg.nt > 1;
      } while (ok && next_segment(pa, table, seg));
    }
  } else if (kWiden && warp >= CONV_WARP0) {
    // ================================ widening =====================================
    if constexpr (kWiden) {
      const int w = warp - CONV_WARP0;
      // lane = (row of four, 16-byte piece): eight lanes read one row's 128 bytes and write one row's 128 bytes of
      // either half at a time (pieces 4-7 store their second eight values first), without bank conflicts
      const int ch = lane & 7, sub = lane >> 3;
      const uint8_t* base[2] = {reinterpret_cast<const uint8_t*>(a.k) + ch * 16, reinterpret_cast<const uint8_t*>(a.v) + ch * 16};
      const int page_shift = a.paged ? 31 - __clz(a.block_size) : 0;   // a power of two of at least 8
      uint4 next[2][4];              // K and V rows w * 16 + k * 4 + sub of the next tile
      auto load = [&](int j) {
        const int row0 = seg.span.tile(j) * BN + w * 16;
        int page[2] = {0, 0};        // of the rows' first and second eight
        if (a.paged) {
          const int32_t* bt_row = a.block_table + (int64_t)seg.b * a.bt_stride;
          page[0] = cache_page(c, bt_row, row0 >> page_shift);
          page[1] = cache_page(c, bt_row, (row0 + 8) >> page_shift);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int col = row0 + k * 4 + sub;
          const bool seen = col < seg.last.hi && (col >= seg.first.lo || col < c.sinks);
          const int64_t in = a.paged ? col & (a.block_size - 1) : seg.s.k_begin + col;
#pragma unroll
          for (int which = 0; which < 2; ++which)
            next[which][k] = seen ? ldg16_stream(base[which] + page[k >> 1] * (which ? a.v_bs : a.k_bs) +
                                                 in * (which ? a.v_rs : a.k_rs) + seg.hk * (which ? a.v_hs : a.k_hs))
                                  : make_uint4(0, 0, 0, 0);
        }
      };
      uint32_t kv = 0;     // K/V tiles so far
      bool ok = true;
      load(seg.lo);
      do {
        Segment cur = seg;
        for (int j = cur.lo; j < cur.hi && ok; ++j, ++kv) {
          uint4 raw[2][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            raw[0][k] = next[0][k];
            raw[1][k] = next[1][k];
          }
          if (j + 1 < cur.hi)
            load(j + 1);
          else if (next_segment(pa, table, seg))
            load(seg.lo);
          else
            ok = false;              // the last tile of the run
          const uint32_t stg = kv % STAGES;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            if (!wwait(which ? &v_empty[stg] : &k_empty[stg], ((kv / STAGES) & 1) ^ 1)) {
              ok = false;
              break;
            }
            uint8_t* dst = (which ? sV : sK) + stg * UNIT + (ch >> 2) * UNIT_HALF;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = w * 16 + k * 4 + sub;
              uint4 lo, hi;
              fp8x4_to_f16x4<KIND>(raw[which][k].x, lo.x, lo.y);
              fp8x4_to_f16x4<KIND>(raw[which][k].y, lo.z, lo.w);
              fp8x4_to_f16x4<KIND>(raw[which][k].z, hi.x, hi.y);
              fp8x4_to_f16x4<KIND>(raw[which][k].w, hi.z, hi.w);
              const bool swap = ch & 4;
              const int c0 = (ch & 3) * 2 + (swap ? 1 : 0);
              uint8_t* row = dst + r * 128;
              *reinterpret_cast<uint4*>(row + ((c0 ^ (r & 7)) << 4)) = swap ? hi : lo;
              *reinterpret_cast<uint4*>(row + (((c0 ^ 1) ^ (r & 7)) << 4)) = swap ? lo : hi;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(which ? &v_full[stg] : &k_full[stg]);
          }
        }
      } while (ok);
    }
  } else if (warp < 4 * NT) {
    // ================================ softmax / epilogue ===========================
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;     // row inside the tile == TMEM lane
    const int in_tok = r / a.group, in_head = r - in_tok * a.group;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + t * 128;
    const uint32_t o_addr = tmem_base + lane_addr + 256 + t * 128;
    PartRecord rec{-1, 0, 0, 0};
    uint32_t item = 0, kv = 0, g = 0;         // items, K/V tiles and this tile's steps so far
    bool ok = true;
    do {
      if (t >= seg.nt) {                      // no token in this tile
        if constexpr (kConvQ) {
          // But every item's q_full is waited for, and q_ready holds its Q until then: a barrier may not run two phases ahead
          // of one that waits for it, since a parity cannot tell them apart.
          if (!wwait(q_full, item & 1)) break;
          if (lane == 0) mbar_arrive(&q_ready[t]);
        }
        ++item;
        kv += (uint32_t)(seg.hi - seg.lo);
        continue;
      }
      const int tile_first = seg.m0 + t * pa.tokens;
      const int tok = tile_first + in_tok, h = seg.hk * a.group + in_head;
      const bool valid = in_tok < pa.tokens && tok < seg.s.q_len;
      const int k_len = seg.s.k_len;
      const RowMask mask = row_mask(c, k_len, tok + seg.shift);
      // what the first and the last row of the tile see: steps between need no mask
      const RowMask first = row_mask(c, k_len, tile_first + seg.shift);
      const RowMask last = row_mask(c, k_len, min(tile_first + pa.tokens, seg.s.q_len) - 1 + seg.shift);
      float m_used = -INFINITY, l_run = 0.f;
      float scale = a.scale_log2 * cache_scale(c.k_scale, c.ks_batch, c.ks_head, seg.b, seg.hk);
      const float v_scale = cache_scale(c.v_scale, c.vs_batch, c.vs_head, seg.b, seg.hk);
      if constexpr (kConvQ) {
        // my row of Q, from bf16 to fp16 with its power of two
        if (!wwait(q_full, item & 1)) break;
        uint8_t* q = sQ + t * TILE_BYTES + r * 128;
        float top = 0.f;
#pragma unroll 4
        for (int ch = 0; ch < HD / 8; ++ch) {
          float f[8];
          Vec16<T>::unpack(*reinterpret_cast<const uint4*>(q + (ch >> 3) * HALF_BYTES + (((ch & 7) ^ (r & 7)) << 4)), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
        }
        float up, down;
        row_power(top, up, down);
#pragma unroll 4
        for (int ch = 0; ch < HD / 8; ++ch) {
          uint4* at = reinterpret_cast<uint4*>(q + (ch >> 3) * HALF_BYTES + (((ch & 7) ^ (r & 7)) << 4));
          float f[8];
          Vec16<T>::unpack(*at, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= up;
          *at = Vec16<__half>::pack(f);
        }
        scale *= down;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[t]);
      }
      ++item;
      const bool odd_scale = !(scale > 0.f);  // a K scale that is zero, negative or NaN: scale the scores first

      for (int i = seg.lo; i < seg.hi; ++i, ++g, ++kv) {
        const uint32_t p_addr = s_addr + BN + (g & 1) * 32;
        if (!wwait(&s_full[t], g & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float sv[64];
        tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
        tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);   // the next step's scores may be computed into the same columns
        float sc = scale;
        if (odd_scale) {
#pragma unroll
          for (int e = 0; e < 64; ++e) sv[e] *= scale;
          sc = 1.f;
        }
        const int col0 = seg.span.tile(i) * BN;
        if (col0 + BN > first.hi || (col0 < last.lo && col0 + BN > c.sinks)) {
          // a bit for each key of the tile: below hi, and not below lo or below the first tokens' end
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
          const int hi = mask.hi - col0, lo = mask.lo - col0, sk = c.sinks - col0;
          const uint32_t seen[2] = {below(hi) & (~below(lo) | below(sk)), below(hi - 32) & (~below(lo - 32) | below(sk - 32))};
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (!((seen[e >> 5] >> (e & 31)) & 1u)) sv[e] = -INFINITY;
        }
        float m4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
        for (int e = 4; e < 64; e += 8) {
          m4[0] = max3(m4[0], sv[e], sv[e + 1]);
          m4[1] = max3(m4[1], sv[e + 2], sv[e + 3]);
          if (e + 4 < 64) {
            m4[2] = max3(m4[2], sv[e + 4], sv[e + 5]);
            m4[3] = max3(m4[3], sv[e + 6], sv[e + 7]);
          }
        }
        const float m_tile = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * sc;   // sc > 0; -inf stays -inf
        const bool raise = m_tile > m_used + kRescaleThreshold || (m_used == -INFINITY && m_tile > -INFINITY);
        if (i > seg.lo && __any_sync(0xffffffffu, raise)) {
          // every P V issued so far must have landed before O is touched
          if (!wwait(&o_done[t * 2 + ((g - 1) & 1)], ((g - 1) >> 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float f = raise ? ex2(m_used - m_tile) : 1.0f;
#pragma unroll 1
          for (int q = 0; q < HD / 16; ++q) {
            uint32_t o[16];
            tmem_ld16(o_addr + q * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(o_addr + q * 16, o);
          }
          l_run *= f;
        }
        if (raise) m_used = m_tile;
        const float neg_m = m_used == -INFINITY ? 0.f : kShift - m_used;
        if constexpr (!kWiden) {
          // V rows of this step that no row of the item sees must not reach the products: zeroed in place, by each tile's
          // warps for themselves (the other tile writes the same zeros)
          if (col0 + BN > seg.last.hi || (col0 < seg.first.lo && col0 + BN > c.sinks)) {
            const uint32_t stg = kv % STAGES;
            if (!wwait(&v_full[stg], (kv / STAGES) & 1)) {
              ok = false;
              break;
            }
            uint8_t* vt = sV + stg * UNIT;
            for (int at = r; at < BN * (HD / 8); at += 128) {
              const int row = at / (HD / 8), ch = at % (HD / 8), col = col0 + row;
              if (col >= seg.last.hi || (col < seg.first.lo && col >= c.sinks))
                *reinterpret_cast<uint4*>(vt + (ch >> 3) * UNIT_HALF + row * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
        {
          const uint64_t sc2 = pack2f(sc, sc), ng2 = pack2f(neg_m, neg_m);
#pragma unroll
          for (int e = 0; e < 64; e += 2) fma2(sv[e], sv[e + 1], sc2, ng2);
        }
#pragma unroll
        for (int e = 0; e < 64; ++e) sv[e] = ex2(sv[e]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = sv[q * 32 + 2 * e], p1 = sv[q * 32 + 2 * e + 1];
            add2(sum4[(e & 1) * 2], sum4[(e & 1) * 2 + 1], p0, p1);
            pk[e] = Pair<M>::pack(p0, p1);
          }
          tmem_st16(p_addr + q * 16, pk);
        }
        l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t * 2 + (g & 1)]);
      }
      if (!ok) break;

      // ---- epilogue: normalise my row of O and write it out
      if (!wwait(&o_done[t * 2 + ((g - 1) & 1)], ((g - 1) >> 1) & 1)) break;
      tc_fence_after();
      // a NaN sum stays one: only a row that saw nothing is set to zero
      const float inv = v_scale / l_run;
      const bool whole = seg.lo == 0 && seg.hi == seg.n;
      const int64_t qtok = seg.s.q_begin + tok;
      const int64_t part = ((int64_t)2 * blockIdx.x + (seg.lo == 0 ? 1 : 0)) * NT + t;   // 128 rows
      if (!whole && seg.lo == 0)   // the last of the run: each later CTA takes `run` tiles of the rest
        rec = PartRecord{seg.hk, 1 + (seg.n - seg.hi + run - 1) / run, seg.s.q_begin + seg.m0, seg.s.q_len - seg.m0};
      T* orow = reinterpret_cast<T*>(a.out) + qtok * a.o_rs + (int64_t)h * a.o_hs;
      float4* prow = reinterpret_cast<float4*>(pa.part_o + part * BM * HD) + r;   // 16-byte piece p of row r at p * 128 + r
#pragma unroll 1
      for (int q = 0; q < HD / 16; ++q) {
        uint32_t o[16];
        tmem_ld16(o_addr + q * 16, o);
        tmem_ld_wait();
        if (q == HD / 16 - 1) {   // my row is in registers: the next item's first product may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[t]);
        }
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = l_run == 0.f ? 0.f : __uint_as_float(o[e]) * inv;
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            prow[(q * 4 + e) * BM] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<uint4*>(orow + q * 16 + e * 8) =
                make_uint4(Pair<T>::pack(f[8 * e], f[8 * e + 1]), Pair<T>::pack(f[8 * e + 2], f[8 * e + 3]),
                           Pair<T>::pack(f[8 * e + 4], f[8 * e + 5]), Pair<T>::pack(f[8 * e + 6], f[8 * e + 7]));
        }
        __syncwarp();
      }
      if (!whole || (valid && a.lse)) {
        const float lse2 = l_run == 0.f ? -INFINITY : m_used - kShift + log2f(l_run);
        if (!whole)
          pa.part_lse[part * BM + r] = lse2;
        else
          a.lse[(int64_t)h * a.total_q + qtok] = l_run == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
      }
    } while (next_segment(pa, table, seg));
    if (tid == 0 && !c.whole) pa.record[blockIdx.x] = rec;
  }

  // ================================ teardown ======================================
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {   // a wait gave up: leave the copies and products in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (warp == MMA_WARP0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Joins the parts of the items that runs cut.  Block (i, t, y) does dims [32 y, 32 y + 32) of Q tile t of the item whose start, but
// not end, CTA i holds, a row a thread: its tail part, then the head parts of the CTAs after it, in order.
template <typename T, int HD>
__global__ void __launch_bounds__(BM) attn_cache_join_rows_kernel(ChunkArgs pa, int ctas) {
  const AttnArgs& a = pa.c.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");              // launched early: the parts are complete after this
  const int i = blockIdx.x, t = blockIdx.y, r = threadIdx.x;
  const PartRecord rec = pa.record[i];
  if (*reinterpret_cast<volatile int*>(a.status) != 0) return;   // the parts and the records may be missing
  const int in_tok = r / a.group, tok = t * pa.tokens + in_tok;
  if (rec.hk < 0 || in_tok >= pa.tokens || tok >= rec.tokens) return;
  const int n = min(rec.parts, ctas - i);
  auto slot = [&](int k) { return (int64_t)(k == 0 ? 2 * i + 1 : 2 * (i + k)) * pa.tiles + t; };
  float m = -INFINITY;
#pragma unroll 16
  for (int k = 0; k < n; ++k) m = fmaxf(m, pa.part_lse[slot(k) * BM + r]);
  const float ms = m == -INFINITY ? 0.f : m;
  float acc[32], wsum = 0.f;
#pragma unroll
  for (int e = 0; e < 32; ++e) acc[e] = 0.f;
#pragma unroll 4   // an item may be in many parts: their loads are in flight together
  for (int k = 0; k < n; ++k) {
    const float w = exp2f(pa.part_lse[slot(k) * BM + r] - ms);
    const float4* o = reinterpret_cast<const float4*>(pa.part_o + slot(k) * BM * HD) + blockIdx.z * 8 * BM + r;
    wsum += w;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float4 v = o[e * BM];
      acc[4 * e] += w * v.x;
      acc[4 * e + 1] += w * v.y;
      acc[4 * e + 2] += w * v.z;
      acc[4 * e + 3] += w * v.w;
    }
  }
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  const int64_t qtok = rec.q_row + tok;
  const int h = rec.hk * a.group + r - in_tok * a.group;
  T* out = reinterpret_cast<T*>(a.out) + qtok * a.o_rs + (int64_t)h * a.o_hs + blockIdx.z * 32;
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = acc[e + k] * inv;
    stg16(out + e, Vec16<T>::pack(f));
  }
  if (a.lse && blockIdx.z == 0)
    a.lse[(int64_t)h * a.total_q + qtok] = wsum == 0.f ? INFINITY : (m + log2f(wsum)) * 0.6931471805599453f;
}

// Q tiles of an item, tokens of a tile and items (for each KV head) of the longest chunk.
void chunk_shape(int64_t max_q, int64_t group, int64_t head_dim, int* tiles, int* tokens, int64_t* num_mb) {
  *tokens = (int)(BM / group);
  *tiles = max_q > *tokens && head_dim <= 128 ? 2 : 1;
  *num_mb = (max_q + *tiles * *tokens - 1) / (*tiles * *tokens);
}

template <typename T, int KIND, typename M, int HD>
int launch(ChunkArgs& pa, cudaStream_t st) {
  const AttnArgs& a = pa.c.a;
  const bool pages = pa.c.pages();
  const int64_t stored = pa.c.dense > 0 ? a.batch * pa.c.dense : a.total_k;   // rows of a store without pages
  pa.page_rows = pages && a.block_size < BN ? a.block_size : BN;
  pa.pages_per_tile = BN / pa.page_rows;
  CUtensorMap tq, maps[2] = {};        // of K and V: the widening form loads them without
  {
    const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)a.H, (uint64_t)a.total_q};
    const uint64_t strides[2] = {(uint64_t)a.q_hs * 2, (uint64_t)a.q_rs * 2};
    const uint32_t box[3] = {64, (uint32_t)a.group, (uint32_t)pa.tokens};
    const int rc = encode_tmap_16bit(&tq, a.q, 3, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  if constexpr (KIND == kCache16) {
    for (int i = 0; i < 2; ++i) {
      const uint64_t hs = (uint64_t)(i ? a.v_hs : a.k_hs) * 2, rs = (uint64_t)(i ? a.v_rs : a.k_rs) * 2;
      const uint64_t bs = (uint64_t)(i ? a.v_bs : a.k_bs) * 2;
      const uint64_t rows = pages ? (uint64_t)a.block_size : (uint64_t)(stored > 0 ? stored : 1);
      const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)a.Hk, rows, pages ? (uint64_t)a.num_blocks : 1};
      const uint64_t strides[3] = {hs, rs, pages ? bs : rs * rows};
      const uint32_t box[4] = {64, 1, (uint32_t)pa.page_rows, 1};
      const int rc = encode_tmap_16bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box);
      if (rc != FG_OK) return rc;
    }
  }
  constexpr int smem = Shape<HD>::SMEM;
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_chunk_kernel<T, KIND, M, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_dev = dev;
  }
  const int ctas = num_sms();
  pa.part_o = a.ws_o;
  pa.part_lse = pa.part_o + (int64_t)2 * ctas * pa.tiles * BM * HD;
  pa.record = reinterpret_cast<PartRecord*>(pa.part_lse + (int64_t)2 * ctas * pa.tiles * BM);
  attn_cache_chunk_kernel<T, KIND, M, HD><<<ctas, threads_of(KIND), smem, st>>>(tq, maps[0], maps[1], pa);
  FG_CHECK_LAUNCH("attn_cache_chunk_kernel");
  if (pa.c.whole) return FG_OK;
  // Launched while the kernel above still runs (programmatic dependent launch); it waits for its end on the device.
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)pa.tiles, HD / 32);
  cfg.blockDim = dim3(BM);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  FG_CUDA_OK(cudaLaunchKernelEx(&cfg, attn_cache_join_rows_kernel<T, HD>, pa, ctas));
  FG_CHECK_LAUNCH("attn_cache_join_rows_kernel");
  return FG_OK;
}

// Widens the rows of an 8-bit store that some query sees: the tokens of sequence b, in the order of copy_span, to the rows from
// b * dense on of fp16 [rows, Hk, D] K and V.
// A block does 16 tokens; a thread 16 values at a time, four of them in flight.
constexpr int kWidenRows = 16;
template <int KIND>
__global__ void __launch_bounds__(256) attn_cache_widen_kernel(CacheAttnArgs c, __half* k16, __half* v16, int64_t dense) {
  const AttnArgs& a = c.a;
  __shared__ int64_t s_row[2][kWidenRows];       // of K and V: elements from the store's base, or -1
  const SeqInfo s = stored_seq_info(c, blockIdx.y);
  if (s.q_len < 1) return;
  const CopySpan copy = copy_span(c, s);
  const int b = blockIdx.y, row0 = blockIdx.x * kWidenRows, tok0 = row0 + (row0 + copy.gap < copy.win ? 0 : copy.gap);
  const RowMask first = row_mask(c, s.k_len, s.k_len - s.q_len), last = row_mask(c, s.k_len, s.k_len - 1);
  if (tok0 >= last.hi || (tok0 + kWidenRows <= first.lo && tok0 >= c.sinks)) return;
  if (threadIdx.x < kWidenRows) {
    const int tok = tok0 + threadIdx.x;
    const bool seen = tok < last.hi && (tok >= first.lo || tok < c.sinks);
    const int32_t* bt_row = a.paged ? a.block_table + (int64_t)b * a.bt_stride : nullptr;
    s_row[0][threadIdx.x] = seen ? cache_row(c, bt_row, s.k_begin, tok, a.k_rs, a.k_bs) : -1;
    s_row[1][threadIdx.x] = seen ? cache_row(c, bt_row, s.k_begin, tok, a.v_rs, a.v_bs) : -1;
  }
  __syncthreads();
  const int pieces = a.D >> 4, shift = 31 - __clz(pieces);   // a power of two
  const int per_row = a.Hk * pieces, total = 2 * kWidenRows * per_row;
  for (int base = threadIdx.x; base < total; base += 4 * 256) {
    uint4 raw[4];
    __half* dst[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * 256;
      dst[u] = nullptr;
      if (i >= total) continue;
      const int ch = i & (pieces - 1), hk = (i >> shift) % a.Hk, row = i / per_row;
      const bool is_v = row >= kWidenRows;
      const int r = is_v ? row - kWidenRows : row;
      const int64_t at = s_row[is_v][r];
      if (at < 0) continue;
      const uint8_t* from = reinterpret_cast<const uint8_t*>(is_v ? a.v : a.k);
      raw[u] = ldg16_stream(from + at + (int64_t)hk * (is_v ? a.v_hs : a.k_hs) + ch * 16);
      dst[u] = (is_v ? v16 : k16) + (((int64_t)b * dense + row0 + r) * a.Hk + hk) * a.D + ch * 16;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (dst[u] == nullptr) continue;
      uint4 lo, hi;
      fp8x4_to_f16x4<KIND>(raw[u].x, lo.x, lo.y);
      fp8x4_to_f16x4<KIND>(raw[u].y, lo.z, lo.w);
      fp8x4_to_f16x4<KIND>(raw[u].z, hi.x, hi.y);
      fp8x4_to_f16x4<KIND>(raw[u].w, hi.z, hi.w);
      stg16(dst[u], lo);
      stg16(dst[u] + 8, hi);
    }
  }
}

// Bytes of the parts and records that come first in the workspace.
int64_t part_bytes(int tiles, int64_t head_dim, int sms) {
  return ((int64_t)sms * (2 * tiles * BM * (head_dim + 1) * 4 + (int64_t)sizeof(PartRecord)) + 1023) / 1024 * 1024;
}

template <typename T, typename M>
int launch_16(ChunkArgs& pa, cudaStream_t st) {
  if (pa.c.a.D == 64) return launch<T, kCache16, M, 64>(pa, st);
  if (pa.c.a.D == 256) return launch<T, kCache16, M, 256>(pa, st);
  return launch<T, kCache16, M, 128>(pa, st);
}

template <typename T>
int launch_kind(ChunkArgs& pa, int kind, cudaStream_t st) {
  CacheAttnArgs& c = pa.c;
  if (kind == kCache16) return launch_16<T, T>(pa, st);
  if (c.dense > 0) {   // rows of a sequence in the 16-bit copy
    AttnArgs& a = c.a;
    const int64_t rows = a.batch * c.dense;
    __half* k16 = reinterpret_cast<__half*>(reinterpret_cast<char*>(a.ws_o) + (c.whole ? 0 : part_bytes(pa.tiles, a.D, num_sms())));
    __half* v16 = k16 + rows * a.Hk * a.D;
    const dim3 grid((unsigned)((c.dense + kWidenRows - 1) / kWidenRows), (unsigned)a.batch);
    if (kind == kCacheE4M3)
      attn_cache_widen_kernel<kCacheE4M3><<<grid, 256, 0, st>>>(c, k16, v16, c.dense);
    else
      attn_cache_widen_kernel<kCacheE5M2><<<grid, 256, 0, st>>>(c, k16, v16, c.dense);
    FG_CHECK_LAUNCH("attn_cache_widen_kernel");
    a.k = k16;
    a.v = v16;
    a.k_hs = a.v_hs = a.D;
    a.k_rs = a.v_rs = (int64_t)a.Hk * a.D;
    return launch_16<T, __half>(pa, st);
  }
  if (kind == kCacheE4M3) return launch<T, kCacheE4M3, __half, 128>(pa, st);
  return launch<T, kCacheE5M2, __half, 128>(pa, st);
}

}  // namespace

// Bytes of workspace: a head and a tail part, and a record, for each CTA; with `dense` rows for each sequence also their 16-bit copy.
// -1: more tiles than the kernel counts in 32 bits.
int64_t attn_cache_chunk_bytes(int64_t max_q, int64_t group, int64_t batch, int64_t heads_k, int64_t head_dim, int64_t max_k,
                               int64_t dense, bool whole, int sms) {
  int tiles, tokens;
  int64_t num_mb;
  chunk_shape(max_q, group, head_dim, &tiles, &tokens, &num_mb);
  if (batch * num_mb > 2147483647LL / 2 || batch * num_mb * heads_k > 2147483647LL / (max_k / BN + 1)) return -1;
  return (whole ? 0 : part_bytes(tiles, head_dim, sms)) + 2 * batch * dense * heads_k * head_dim * 2;
}

int attn_cache_chunk(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  ChunkArgs pa;
  pa.c = c;
  if (!c.a.status) return fail(FG_ERR_CUDA, "flash_attn_cache: device status word unavailable");
  int64_t num_mb;
  chunk_shape(c.a.max_q, c.a.group, c.a.D, &pa.tiles, &pa.tokens, &num_mb);
  pa.num_mb = (int)num_mb;
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(pa, kind, st) : launch_kind<__half>(pa, kind, st);
}

}  // namespace fg
