// Attention of a few query rows (at most 16 (token, head of the group) pairs of a sequence) over an 8-bit or windowed
// cache, head dim 64, 128 or (8-bit) 256, on the tcgen05 tensor cores.  Memory bound: every cached byte is read once, and nothing
// else is done with it -- the tensor cores read K and V from shared memory in the type and layout that TMA delivers.
//
// The products are turned round, so that the many keys fill the 128 rows of the instruction and the few query rows its
// columns:
//     S^T [128 keys x N] = K [keys x 128] Q^T          K is the K-major A operand as it lies in the cache
//     O^T [128 dims x N] += V^T [128 x keys] P^T       V is the MN-major A operand as it lies in the cache (256 dims: two
//                                                      products; 64: the 64 dims are read twice, the second half is not used)
// A thread of the four softmax warps owns one key (TMEM lane): it holds that key's scores of all rows, so nothing is spent
// on rows that are not there.
//
// 8-bit caches: Q and P are split into 8-bit pieces, each with columns of its own, and the columns are added up in fp32.
// A piece is the rounding of what the ones before it left, times a power of two that brings it back to the top of the type's
// range: a common scale would cut all pieces at the same subnormal step.
//   Q   a row is multiplied by a power of two that takes its largest value to [2^7, 2^8) and parted into three e4m3 pieces, 2^5
//       apart: exact for bf16 and fp16 values down to 2^-16 of the row's largest one, and within 2^-27 of it below (a
//       subnormal step of the last piece).  Rows whose largest channel meets small keys need that range; two pieces would do
//       for the 8 bits of bf16 near the top, but end at 2^-22.  The third costs nothing at 4 rows (its columns are there
//       anyway) and most at 16 rows of 256 dims, 172 -> 180 us for 64 sequences.
//   P   2^11 p (p <= 2^4, see below), rounded to fp16 (2^-12 of itself, or 2^-36), in four e5m2 pieces of three bits, 2^3
//       apart, which hold every fp16 value exactly; e5m2 for its range: long contexts have many small probabilities
// 16-bit caches: Q as it is; P in one fp16 piece, or two bf16 pieces (2^-17).
//
// The running maximum is shared by the CTA and raised only when a score exceeds it by more than 4 (log2 units); the warps
// agree on that with one barrier reduction a tile.  Only a raise needs the exact maximum and rescales O in TMEM.
//
//   warps 0-3   softmax and output
//   warps 4, 5  TMA producers of K and of V tiles (128 keys), each with a ring of its own.  A page of 16 keys is one box, and a
//               warp issues one in about 95 clocks (lanes in turn; 125 when one lane issues them all): with one warp for both
//               rings the issue bounded the kernel (256 sequences: 521 us by one lane, 412 us by eight)
//   warp 6      issues the products: scores of the next tile before P V of the current one when its keys are there
//
// Measured: 256 sequences of 512 to 8192 tokens, 32 heads over 8, 8-bit: 2.29 GB in 375 to 388 us, 5.9 to 6.1 TB/s (the
// tensor pipe is 4 % busy); windowed, 64 sequences of up to 16384, 16-bit 74 us, 8-bit 104 us.  A tile takes about 1 us (4
// rows) to 1.6 us (16 rows) through the chain of score product, maximum, probabilities and their pieces, which bounds short
// runs; mma.sync in smaller CTAs is faster there (attn_cache_api.cu).
//
// The kernel is persistent.  An item is one (sequence, KV head).  A team of CTAs walks the same sequences, each for a KV head of
// its own, so that the heads' pieces of a cached row, which lie side by side in memory, are fetched at about the same time.
// The K/V tiles of all sequences, laid end to end, are cut into equal runs, one per team, whatever the lengths (each CTA sums
// the tile counts up once at its start).  The ring, the tensor
// memory and the barriers carry on from item to item: the producer runs ahead into the next one, and the softmax warps
// prepare the next item's Q while they work on the current one.  An item inside one run is written out at once; the
// parts of an item that runs cut are joined by a second kernel, in order.  Short items are not cut, and there is no second kernel.
#include "attn_cache_common.cuh"
#include "sm100_common.cuh"

namespace fg {
namespace {

constexpr int BN = 128, NUM_THREADS = 224;
constexpr int TMA_WARP = 4, MMA_WARP = 6;
constexpr float kRaise = 4.0f;               // log2 units
constexpr float kPScale = 2048.0f;           // of P before it is split (8-bit caches)
constexpr float kQStep = 32.f;               // a residual of Q is at most half an e4m3 step of four bits: 2^3 below 2^8
constexpr float kPStep = 8.f;                // of P at most half an e5m2 step of three bits: 2^11 below 2^15

constexpr int kInfo = 32;                    // sequences of a run whose lengths are kept in shared memory

constexpr int up(int n, int to) { return (n + to - 1) / to * to; }

// T: query type; KIND: cache; RP: query rows, rounded up to 4, 8 or 16; HD: head dim
template <typename T, int KIND, int RP, int HD>
struct Cfg {
  static constexpr bool k8 = KIND != kCache16;
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int PQ = k8 ? 3 : 1;                       // pieces of Q
  static constexpr int PP = k8 ? 4 : (kBf16 ? 2 : 1);         // pieces of P
  static constexpr bool kPieces = PP > 1 && KIND != kCacheE4M3;   // V may hold infinities, and meets several pieces (e4m3 has none)
  static constexpr int NS = up(RP * PQ, 16), NP = up(RP * PP, 16);   // columns of the two products
  // Rows of Q and P that shared memory holds: whole 8-row swizzle groups.  Where the product has 8 columns more, it reads
  // whatever follows there; nothing uses those columns.
  static constexpr int QR = up(RP * PQ, 8), PR = up(RP * PP, 8);
  static constexpr int ES = k8 ? 1 : 2;                       // bytes of a cached value, and of a piece of Q or P
  static constexpr int ROW = HD * ES;                         // bytes of a cached row: 64, 128 or 256
  static constexpr int ATOM = ROW < 128 ? ROW : 128;          // ... in one swizzled column block (TMA box)
  static constexpr int BLOCKS = ROW / ATOM;
  static constexpr int BLOCK = BN * ATOM;                     // bytes of a tile's column block
  static constexpr int TILE = BN * ROW;                       // bytes of a K or V tile
  static constexpr int OM = HD > 128 ? 2 : 1;                 // products P V of 128 dims; at 64 the upper half repeats the lower
  // One CTA an SM, or two where 128 registers a thread are enough.
  static constexpr int CTAS = k8 && RP == 4 && HD <= 128 ? 2 : 1;
  static constexpr int QW = ROW > 128 ? 2 : 1;                // 128-byte column blocks of a Q buffer
  static constexpr int QB = QR * QW * 128;                    // bytes of one Q buffer
  static constexpr int PB = PR * BN * (k8 ? 1 : 2);           // bytes of one P buffer
  static constexpr int REST = 2 * QB + 2 * PB + 1024 + 1024 + kInfo * 16;
  // tiles of each ring: what shared memory holds (192 KB of tiles on their way where they divide it), and the barriers' space
  static constexpr int FIT = ((CTAS == 2 ? 115712 : 232448) - REST) / (2 * TILE);
  static constexpr int SLOTS = FIT < 9 ? FIT : 9;
  static constexpr int SCOL = NS <= 32 ? 32 : 64;             // TMEM columns of one score buffer
  static constexpr int OCOL = 2 * SCOL;
  static constexpr int TCOLS = OCOL + OM * NP <= 128 ? 128 : 256;
  static_assert(OCOL + OM * NP <= 256, "tensor memory");
  static constexpr int QV = HD * RP / 128 < 4 ? 4 : HD * RP / 128;   // values of a Q row that a thread splits
  static constexpr int SMEM = 2 * SLOTS * TILE + REST;
};

// What a CTA leaves for the joining kernel: the item whose start it holds but not its end (or -1), in how many parts the item
// is, and its first query token and rows.
struct PartRecord {
  int item, parts, q_begin, rows;
};

struct DecodeArgs {
  CacheAttnArgs c;
  int page_rows, pages_per_tile;
  float* part_o;        // [2 * CTAs][RP][128]: head part, tail part of each CTA
  float* part_lse;      // [2 * CTAs][RP]
  PartRecord* record;   // [CTAs]
  int min_run;          // fewest tiles of a run
  int team, rounds;     // CTAs of a team, a divisor of the KV heads; KV heads of each member
};

// Fewest tiles that a run is worth starting a CTA for.  8 sequences of up to 1328 keys, 8 KV heads (456 tiles), in runs of at least
// 1, 2, 4 and 8 tiles: 18.7, 18.7, 17.6 and 23.9 us in a graph; 2 of up to 6000 keys 24.3, 24.4, 22.8 and 22.1: a part more to join
// costs about what a tile does.
constexpr int kMinRun = 4;

// One item's part of a CTA's run.
struct Segment {
  int b, hk, lo, hi, n;         // K/V tiles [lo, hi) of the item's n; hk goes up in steps of the team
  int left;                     // tiles of the run from lo on
  int rows, shift;
  SeqInfo s;
  TileSpan span;
};
template <int RP>
__device__ __forceinline__ int item_tiles(const CacheAttnArgs& c, const SeqInfo& s, TileSpan& span) {
  const int rows = min(s.q_len * c.a.group, RP);
  if (rows < 1) return 0;
  const int shift = s.k_len - s.q_len;
  span = tile_span<BN>(c, s.k_len, shift, (rows - 1) / c.a.group + shift);
  return max(span.n, 1);        // nothing visible: one tile, all of it masked, gives the zeros
}
// Lengths of the sequences [b0, b0 + n) as the CTA found them at its start; the others come from global memory.
struct InfoTable {
  const SeqInfo* info;
  int b0, n;
};
template <int RP>
__device__ __forceinline__ void fill_segment(const CacheAttnArgs& c, const InfoTable& table, Segment& g, int lo) {
  g.s = (unsigned)(g.b - table.b0) < (unsigned)table.n ? table.info[g.b - table.b0] : cache_seq_info(c, g.b);
  g.n = item_tiles<RP>(c, g.s, g.span);
  g.rows = min(g.s.q_len * c.a.group, RP);
  g.shift = g.s.k_len - g.s.q_len;
  g.lo = lo;
  g.hi = c.whole ? g.n : min(g.n, lo + g.left);
}
// The part after `g`; false when the run ends with g.
template <int RP>
__device__ __forceinline__ bool next_segment(const CacheAttnArgs& c, const InfoTable& table, int team, const Segment& g,
                                             Segment& to) {
  to = g;
  to.left = g.left - item_weight(c, g.hi - g.lo);
  if (to.left <= 0) return false;
  to.hk += team;
  if (to.hk < c.a.Hk) {
    to.lo = 0;
    to.hi = c.whole ? to.n : min(to.n, to.left);
    return true;
  }
  to.hk -= c.a.Hk;
  do {
    if (++to.b >= c.a.batch) return false;
    fill_segment<RP>(c, table, to, 0);
  } while (to.n == 0);
  return true;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// whether any of the 128 softmax threads says yes
__device__ __forceinline__ bool softmax_any(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(yes ? 1u : 0u)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ uint16_t f16x2_to_e5m2x2(uint32_t h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(h));
  return r;
}

// ---- Infinities.  Piece by piece a product with an infinity may be a NaN where the whole is none (a later piece can be zero or
// of the other sign).  A NaN is looked into where it shows up, outside the loops' registers; finite values never come here.

// Which query rows see +inf, -inf or NaN among the V values of dim d at the keys of segment g: bits r, 16 + r, 32 + r.
template <typename T, int KIND>
__device__ __noinline__ uint64_t odd_values(const CacheAttnArgs& c, const Segment& g, int d) {
  using E = typename std::conditional<KIND == kCache16, T, uint8_t>::type;
  const int group = c.a.group;
  const E* v = reinterpret_cast<const E*>(c.a.v) + (int64_t)g.hk * c.a.v_hs + d;
  const int32_t* bt_row = c.a.paged ? c.a.block_table + (int64_t)g.b * c.a.bt_stride : nullptr;
  uint64_t bits = 0;
  for (int t = g.lo; t < g.hi; ++t) {
    const int j0 = g.span.tile(t) * BN, end = min(j0 + BN, g.s.k_len);
    for (int j = j0; j < end; j += 8) {          // rows of one page
      const int64_t row = cache_row(c, bt_row, g.s.k_begin, j, c.a.v_rs, c.a.v_bs);
      E raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = j + i < end ? v[row + i * c.a.v_rs] : E{};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x;
        if constexpr (KIND == kCache16)
          x = Cvt<T>::to_f32(raw[i]);
        else
          x = Pair<__half>::unpack(fp8x2_to_f16x2<KIND>(raw[i])).x;
        if (j + i >= end || fabsf(x) < INFINITY) continue;
        for (int r = 0; r < g.rows; ++r)
          if (!row_mask(c, g.s.k_len, r / group + g.shift).dead(j + i)) bits |= 1ull << (r + (x != x ? 32 : x > 0.f ? 0 : 16));
      }
    }
    const uint64_t nan = bits >> 32 | (bits & bits >> 16);
    if ((nan & 0xffff) == (1ull << g.rows) - 1) break;      // every row has its NaN
  }
  return bits;
}

// Puts the infinities where bits of `odd` (16 m + r) say that dim m * 128 + threadIdx.x of row r came out as a NaN.
template <typename T, int KIND, int RP, int HD>
__device__ __noinline__ void write_infinities(const DecodeArgs& da, const Segment& g, int part, uint32_t odd, float v_scale) {
  const AttnArgs& a = da.c.a;
  for (int m = 0; m < 2; ++m) {
    if ((odd >> (16 * m) & 0xffff) == 0) continue;
    const int d = m * 128 + threadIdx.x;
    const uint64_t seen = odd_values<T, KIND>(da.c, g, d);
    for (int r = 0; r < g.rows; ++r) {
      const bool up = seen >> r & 1, down = seen >> (16 + r) & 1, nan = seen >> (32 + r) & 1;
      if (!(odd >> (16 * m + r) & 1) || nan || up == down) continue;
      const float v = (up ? INFINITY : -INFINITY) * v_scale;
      const int tok = r / a.group;
      if (part < 0)
        reinterpret_cast<T*>(a.out)[(int64_t)(g.s.q_begin + tok) * a.o_rs +
                                    (int64_t)(g.hk * a.group + r - tok * a.group) * a.o_hs + d] = Cvt<T>::from_f32(v);
      else
        da.part_o[((int64_t)part * RP + r) * HD + d] = v;
    }
  }
}

// The score of row r (times log2 e) at key `key`, in fp32.
template <typename T, int KIND, int HD>
__device__ __noinline__ float whole_score(const CacheAttnArgs& c, const Segment& g, int r, int key) {
  const AttnArgs& a = c.a;
  const int tok = r / a.group;
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(g.s.q_begin + tok) * a.q_rs +
               (int64_t)(g.hk * a.group + r - tok * a.group) * a.q_hs;
  const int32_t* bt_row = a.paged ? a.block_table + (int64_t)g.b * a.bt_stride : nullptr;
  const uint8_t* k = reinterpret_cast<const uint8_t*>(a.k) + cache_row(c, bt_row, g.s.k_begin, key, a.k_rs, a.k_bs) +
                     (int64_t)g.hk * a.k_hs;
  float sum = 0.f;
  for (int d = 0; d < HD; ++d) sum = fmaf(Cvt<T>::to_f32(q[d]), Pair<__half>::unpack(fp8x2_to_f16x2<KIND>(k[d])).x, sum);
  return sum * (cache_scale(c.k_scale, c.ks_batch, c.ks_head, g.b, g.hk) * a.scale_log2);
}

template <typename T, int KIND, int RP, int HD>
__global__ void __launch_bounds__(NUM_THREADS, Cfg<T, KIND, RP, HD>::CTAS)
attn_cache_decode_tcgen05_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                 const __grid_constant__ DecodeArgs da) {
  using namespace sm100;
  using C = Cfg<T, KIND, RP, HD>;
  const CacheAttnArgs& c = da.c;
  const AttnArgs& a = c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.group;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;                                             // [KS]
  uint8_t* sV = sK + C::SLOTS * C::TILE;                             // [VS]
  uint8_t* sQ = sV + C::SLOTS * C::TILE;                             // [2 buffers]: items alternate
  uint8_t* sP = sQ + 2 * C::QB;                                   // [2 buffers]: tiles alternate
  uint8_t* rest = sP + 2 * C::PB;                                 // 384 bytes of barriers, 640 of scratch
  uint64_t* k_full = reinterpret_cast<uint64_t*>(rest);           // [KS]
  uint64_t* k_empty = k_full + C::SLOTS;
  uint64_t* v_full = k_empty + C::SLOTS;    // [VS]
  uint64_t* v_empty = v_full + C::SLOTS;
  uint64_t* s_full = v_empty + C::SLOTS;    // [2] scores of a tile have landed
  uint64_t* s_free = s_full + 2;         // [2] ... and have been read into registers
  uint64_t* p_ready = s_free + 2;        // [2]
  uint64_t* o_done = p_ready + 2;        // [2] P V of even / odd tiles
  uint64_t* q_ready = o_done + 2;        // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_ready + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((4 * C::SLOTS + 10) * 8 + 8 <= 384, "the barriers end before the scratch");
  float* sMax = reinterpret_cast<float*>(rest + 384);             // [4 warps][16]
  float* sSum = sMax + 64;                                        // [4 warps][16]
  float* sDown = sSum + 64;                                       // [2 buffers][16]
  SeqInfo* sInfo = reinterpret_cast<SeqInfo*>(rest + 1024);       // [kInfo]

  __shared__ int s_drain;
  __shared__ int s_sum[NUM_THREADS / 32], s_off, s_b;
  // ---- this team's run: tiles [begin, begin + left) of the tiles that each of its members has
  const int rounds = da.rounds, cta = blockIdx.y * gridDim.x + blockIdx.x;   // block (member, team)
  TileSpan span;
  SeqInfo mine_info{0, 0, 0, 0};          // of sequence tid, for batches of at most a thread each
  if (tid < a.batch) mine_info = cache_seq_info(c, tid);
  if (tid == 0) {
    s_drain = *reinterpret_cast<volatile int*>(a.status);
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&q_ready[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  int mine = tid < a.batch ? item_weight(c, item_tiles<RP>(c, mine_info, span)) * rounds : 0;
  int total = mine;
  for (int b = tid + NUM_THREADS; b < a.batch; b += NUM_THREADS)
    total += item_weight(c, item_tiles<RP>(c, cache_seq_info(c, b), span)) * rounds;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  if (s_drain != 0) return;   // a wait gave up on this device: finish the launch quickly
  total = 0;
#pragma unroll
  for (int i = 0; i < NUM_THREADS / 32; ++i) total += s_sum[i];
  const int run = max((total + (int)gridDim.y - 1) / (int)gridDim.y, da.min_run);
  const int64_t begin = (int64_t)run * blockIdx.y;
  if (begin >= total) {
    if (tid == 0 && !c.whole) da.record[cta] = PartRecord{-1, 0, 0, 0};
    return;
  }
  // the sequence that holds tile `begin`
  int before = 0, b0 = 0;
  for (;; b0 += NUM_THREADS) {
    if (b0 > 0) {
      mine = 0;
      if (b0 + tid < a.batch) {
        mine_info = cache_seq_info(c, b0 + tid);
        mine = item_weight(c, item_tiles<RP>(c, mine_info, span)) * rounds;
      }
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
    for (int i = 0; i < NUM_THREADS / 32; ++i) {
      if (i < warp) base += s_sum[i];
      before += s_sum[i];
    }
    if (mine > 0 && base + incl - mine <= begin && begin < base + incl) {
      s_b = b0 + tid;
      s_off = (int)begin - (base + incl - mine);
    }
    if (before > begin) break;
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, C::TCOLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const InfoTable table{sInfo, s_b, min(min(kInfo, a.batch - s_b), b0 + NUM_THREADS - s_b)};
  if ((unsigned)(b0 + tid - table.b0) < (unsigned)table.n) sInfo[b0 + tid - table.b0] = mine_info;
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;");   // the joining kernel may be set up: it waits for this one's end
  Segment seg;
  seg.b = s_b;
  seg.left = min(total - (int)begin, run);
  fill_segment<RP>(c, table, seg, 0);
  const int weight = item_weight(c, seg.n);
  const int round = rounds > 1 ? s_off / weight : 0;
  seg.hk = round * gridDim.x + blockIdx.x;
  seg.lo = s_off - round * weight;
  seg.hi = c.whole ? seg.n : min(seg.n, seg.lo + seg.left);
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

  if (warp == TMA_WARP || warp == TMA_WARP + 1) {
    // ================================ producers of K and of V =====================
    const bool is_v = warp != TMA_WARP;
    const CUtensorMap* tm = is_v ? &tmap_v : &tmap_k;
    uint8_t* ring = is_v ? sV : sK;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    // Lane i holds the place of the i-th page of a tile, or -1 where no query row sees any of its keys: such a page is not
    // fetched (its scores are masked and its V rows zeroed).
    auto lookup = [&](const Segment& g, int t, int& page, int& row) {
      const int tok = g.span.tile(t) * BN + lane * da.page_rows;
      const RowMask first = row_mask(c, g.s.k_len, g.shift), last = row_mask(c, g.s.k_len, (g.rows - 1) / group + g.shift);
      page = -1;
      row = g.s.k_begin + tok;
      if (lane >= da.pages_per_tile || tok >= last.hi || (tok + da.page_rows <= first.lo && tok >= c.sinks)) return;
      page = 0;
      if (a.paged) {
        const int pg = tok / a.block_size;
        row = tok - pg * a.block_size;
        page = cache_page(c, a.block_table + (int64_t)g.b * a.bt_stride, pg);
      }
    };
    int page, row;
    lookup(seg, seg.lo, page, row);
    uint32_t g = 0;    // tiles so far
    bool ok = true;
    while (ok) {
      Segment next;
      const bool more = next_segment<RP>(c, table, gridDim.x, seg, next);
      for (int t = seg.lo; t < seg.hi && ok; ++t, ++g) {
        int npage = -1, nrow = 0;   // the table entry of the next tile is in flight while this one is issued
        if (t + 1 < seg.hi)
          lookup(seg, t + 1, npage, nrow);
        else if (more)
          lookup(next, next.lo, npage, nrow);
        const uint32_t slot = g % C::SLOTS;
        if (!wwait(&empty[slot], ((g / C::SLOTS) & 1) ^ 1)) {
          ok = false;
          break;
        }
        const int pages = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_expect_tx(&full[slot], pages * da.page_rows * (C::TILE / BN));
        __syncwarp();
        if (page >= 0) {
          uint8_t* dst = ring + slot * C::TILE + lane * da.page_rows * C::ATOM;
#pragma unroll
          for (int i = 0; i < C::BLOCKS; ++i)
            tma_load_4d(dst + i * C::BLOCK, tm, &full[slot], i * (C::ATOM / C::ES), seg.hk, row, page);
        }
        page = npage;
        row = nrow;
      }
      if (!more) break;
      seg = next;
    }
  } else if (warp == MMA_WARP) {
    // ================================ products ====================================
    if (lane == 0) {
      const uint32_t id_s = C::k8 ? umma_idesc_f8(KIND == kCacheE5M2, false, false, false, BN, C::NS)
                                  : umma_idesc_f16(C::kBf16, false, false, BN, C::NS);
      const uint32_t id_o = C::k8 ? umma_idesc_f8(KIND == kCacheE5M2, true, true, false, 128, C::NP)
                                  : umma_idesc_f16(C::kBf16, true, false, 128, C::NP);
      // A product takes 32 bytes of K's and Q's rows at a time, four to a 128-byte column block.
      auto kv_desc = [](uint32_t at, uint32_t lbo) {
        return C::ATOM == 64 ? umma_desc_sw64(at, lbo, 512) : umma_desc_sw128(at, lbo, 1024);
      };
      // scores of tile g of the run (tiles count on through all items); `item`: the how-manieth
      auto scores_ready = [&](uint32_t g, bool first, uint32_t item) -> bool {   // without waiting
        return (!first || mbar_test(&q_ready[item & 1], (item >> 1) & 1)) && mbar_test(&k_full[g % C::SLOTS], (g / C::SLOTS) & 1) &&
               (g < 2 || mbar_test(&s_free[g & 1], ((g - 2) >> 1) & 1));
      };
      auto scores = [&](uint32_t g, bool first, uint32_t item) -> bool {
        const uint32_t slot = g % C::SLOTS;
        if (first && !wait1(&q_ready[item & 1], (item >> 1) & 1)) return false;
        if (!wait1(&k_full[slot], (g / C::SLOTS) & 1)) return false;
        if (g >= 2 && !wait1(&s_free[g & 1], ((g - 2) >> 1) & 1)) return false;   // scores two tiles back are read
        tc_fence_after();
        const uint64_t k_desc = kv_desc(smem_u32(sK + slot * C::TILE), 0);
        const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ + (item & 1) * C::QB), 0, 1024);
        const uint32_t d = tmem_base + (g & 1) * C::SCOL;
#pragma unroll
        for (int k = 0; k < C::ROW / 32; ++k) {
          const uint64_t kd = k_desc + (k >> 2) * (C::BLOCK / 16) + (k & 3) * 2;
          const uint64_t qd = q_desc + (k >> 2) * (C::QR * 128 / 16) + (k & 3) * 2;
          if constexpr (C::k8)
            mma_f8_ss(d, kd, qd, id_s, k != 0);
          else
            mma_f16_ss(d, kd, qd, id_s, k != 0);
        }
        tc_commit(&s_full[g & 1]);
        tc_commit(&k_empty[slot]);
        return true;
      };
      Segment ahead = seg;                 // where the scores are, one tile ahead of P V
      int at = seg.lo;
      uint32_t ahead_item = 0, g = 0;
      bool ok = scores(0, true, 0), left = true;
      while (ok && left) {
        for (int t = seg.lo; t < seg.hi && ok; ++t, ++g) {
          bool first = false, more = true;
          if (++at >= ahead.hi) {
            Segment to;
            more = next_segment<RP>(c, table, gridDim.x, ahead, to);
            ahead = to;
            at = to.lo;
            first = true;
            ++ahead_item;
          }
          // the next tile's scores first, so that the softmax warps find them -- unless its keys have yet to arrive
          const bool early = more && scores_ready(g + 1, first, ahead_item);
          if (early && !scores(g + 1, first, ahead_item)) {
            ok = false;
            break;
          }
          const uint32_t slot = g % C::SLOTS;
          if (!wait1(&v_full[slot], (g / C::SLOTS) & 1) || !wait1(&p_ready[g & 1], (g >> 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          // 128 dims are one column block of 8-bit rows or two of 16-bit ones; 64 dims are read twice
          const uint64_t v_desc = kv_desc(smem_u32(sV + slot * C::TILE), HD == 64 ? 0 : C::BLOCK);
          const uint64_t p_desc = umma_desc_sw128(smem_u32(sP + (g & 1) * C::PB), 0, 1024);
          const bool add = t > seg.lo;     // the first tile of an item overwrites
#pragma unroll
          for (int m = 0; m < C::OM; ++m) {
            const uint32_t d = tmem_base + C::OCOL + m * C::NP;
            if constexpr (C::k8) {
#pragma unroll
              for (int k = 0; k < BN / 32; ++k)
                mma_f8_ss(d, v_desc + m * (C::BLOCK >> 4) + k * (32 * C::ATOM >> 4), p_desc + k * 2, id_o, add || k > 0);
            } else {
#pragma unroll
              for (int k = 0; k < BN / 16; ++k)
                mma_f16_ss(d, v_desc + k * (2048 >> 4), p_desc + (k >> 2) * (C::PR * 128 / 16) + (k & 3) * 2, id_o, add || k > 0);
            }
          }
          tc_commit(&o_done[g & 1]);
          tc_commit(&v_empty[slot]);
          if (more && !early && !scores(g + 1, first, ahead_item)) {
            ok = false;
            break;
          }
        }
        Segment to;
        left = next_segment<RP>(c, table, gridDim.x, seg, to);
        seg = to;
      }
    }
  } else {
    // ================================ softmax / output =============================
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    // ---- an item's Q: QV values of a row a thread, loaded ahead and then split into pieces
    constexpr int TPR = HD / C::QV;
    const int q_row = tid / TPR, d0 = (tid % TPR) * C::QV;    // rows from RP on: nothing to do
    uint32_t qw[C::QV / 2];
    float ksc = 1.f, vsc = 1.f;
    auto load_q = [&](const Segment& g) {
      const bool live = q_row < g.rows;
      const int tok = live ? q_row / group : 0;
      const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(g.s.q_begin + tok) * a.q_rs +
                   (int64_t)(g.hk * group + (live ? q_row - tok * group : 0)) * a.q_hs + d0;
#pragma unroll
      for (int i = 0; i < C::QV / 4; ++i) {
        const uint2 u = live ? *reinterpret_cast<const uint2*>(q + i * 4) : make_uint2(0, 0);
        qw[2 * i] = u.x;
        qw[2 * i + 1] = u.y;
      }
      ksc = cache_scale(c.k_scale, c.ks_batch, c.ks_head, g.b, g.hk);
      vsc = cache_scale(c.v_scale, c.vs_batch, c.vs_head, g.b, g.hk);
    };
    auto store_q = [&](uint32_t item) {
      uint8_t* buf = sQ + (item & 1) * C::QB;
      float down = 1.f;
      if constexpr (C::k8) {
        float x[C::QV], top = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < C::QV / 2; ++i) {
          const float2 f = Pair<T>::unpack(qw[i]);
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          bad = bad || !(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY);
        }
#pragma unroll
        for (int o = TPR / 2; o > 0; o >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          bad = __shfl_xor_sync(0xffffffffu, (int)bad, o) || bad;
        }
        float up;
        row_power(top, up, down);
        up *= 0.0078125f;          // [2^14, 2^15) -> [2^7, 2^8)
        down = bad ? NAN : down * 128.f;   // infinities and NaN have no pieces: the whole row is NaN
#pragma unroll
        for (int i = 0; i < C::QV; ++i) x[i] *= up;
#pragma unroll
        for (int p = 0; p < C::PQ; ++p) {
          const int n = p * RP + q_row;
#pragma unroll
          for (int i = 0; i < C::QV / 4; ++i) {
            const int d = d0 + i * 4;
            const uint16_t e0 = f32x2_to_fp8x2<kCacheE4M3>(x[4 * i], x[4 * i + 1]);
            const uint16_t e1 = f32x2_to_fp8x2<kCacheE4M3>(x[4 * i + 2], x[4 * i + 3]);
            const float2 f0 = Pair<__half>::unpack(fp8x2_to_f16x2<kCacheE4M3>(e0));
            const float2 f1 = Pair<__half>::unpack(fp8x2_to_f16x2<kCacheE4M3>(e1));
            x[4 * i] = (x[4 * i] - f0.x) * kQStep;
            x[4 * i + 1] = (x[4 * i + 1] - f0.y) * kQStep;
            x[4 * i + 2] = (x[4 * i + 2] - f1.x) * kQStep;
            x[4 * i + 3] = (x[4 * i + 3] - f1.y) * kQStep;
            if (q_row < RP)
              *reinterpret_cast<uint32_t*>(buf + (d >> 7) * (C::QR * 128) + n * 128 +
                                           ((((d & 127) >> 4) ^ (n & 7)) << 4) + (d & 15)) =
                  e0 | ((uint32_t)e1 << 16);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < C::QV / 4; ++i) {
          const int d = d0 + i * 4;
          if (q_row < RP)
            *reinterpret_cast<uint2*>(buf + (d >> 6) * (C::QR * 128) + q_row * 128 + ((((d & 63) >> 3) ^ (q_row & 7)) << 4) +
                                    (d & 7) * 2) = make_uint2(qw[2 * i], qw[2 * i + 1]);
        }
      }
      if (tid % TPR == 0 && q_row < RP) sDown[(item & 1) * 16 + q_row] = down;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[item & 1]);
    };
    load_q(seg);
    store_q(0);
    softmax_sync();
    PartRecord rec{-1, 0, 0, 0};
    uint32_t g = 0;            // tiles so far
    // A wait that gave up does not end the loops: the barriers below need every warp.
    bool ok = true;
    for (uint32_t item = 0;; ++item) {
      float pre[RP];           // takes a sum of columns to the scores
#pragma unroll
      for (int i = 0; i < RP; ++i) pre[i] = sDown[(item & 1) * 16 + i] * (ksc * a.scale_log2);
      const float v_scale = vsc;
      Segment next;
      const bool more = next_segment<RP>(c, table, gridDim.x, seg, next);
      if (more) load_q(next);   // on its way during this item's first tile
      const int k_len = seg.s.k_len, shift = seg.shift;
      const RowMask first = row_mask(c, k_len, shift), last = row_mask(c, k_len, (seg.rows - 1) / group + shift);
      float m_ref[RP], l_run[RP];
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        m_ref[r] = -INFINITY;
        l_run[r] = 0.f;
      }
      for (int t = seg.lo; t < seg.hi; ++t, ++g) {
        ok = ok && wwait(&s_full[g & 1], (g >> 1) & 1);
        tc_fence_after();
        float x[RP];
        {
          uint32_t col[C::NS];
#pragma unroll
          for (int q = 0; q < C::NS / 16; ++q)
            tmem_ld16(tmem_base + lane_addr + (g & 1) * C::SCOL + q * 16, *reinterpret_cast<uint32_t(*)[16]>(&col[q * 16]));
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[g & 1]);
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            float v = __uint_as_float(col[(C::PQ - 1) * RP + r]);   // the smallest piece first
#pragma unroll
            for (int p = C::PQ - 2; p >= 0; --p) v = fmaf(v, 1.f / kQStep, __uint_as_float(col[p * RP + r]));
            x[r] = v * pre[r];
          }
        }
        const int j0 = seg.span.tile(t) * BN;
        if (j0 + BN > first.hi || (j0 < last.lo && j0 + BN > c.sinks)) {
          const int col = j0 + tid;
          int tok = 0, in = 0;
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            if (row_mask(c, k_len, tok + shift).dead(col)) x[r] = -INFINITY;
            if (++in == group) {
              in = 0;
              ++tok;
            }
          }
          // a V row that no query row sees must not reach the product
          const uint32_t v_slot = g % C::SLOTS;
          ok = ok && wwait(&v_full[v_slot], (g / C::SLOTS) & 1);
          if (ok) {
            // this warp's 32 rows, a group of lanes a row and column block
            constexpr int LPR = C::ATOM / 16;
#pragma unroll
            for (int i = 0; i < LPR; ++i) {
              const int row = warp * 32 + i * (32 / LPR) + lane / LPR, key = j0 + row;
              if (key >= last.hi || (key < first.lo && key >= c.sinks)) {
                uint8_t* v = sV + v_slot * C::TILE + row * C::ATOM + (lane % LPR) * 16;
#pragma unroll
                for (int blk = 0; blk < C::BLOCKS; ++blk) *reinterpret_cast<uint4*>(v + blk * C::BLOCK) = make_uint4(0, 0, 0, 0);
              }
            }
          }
        }
        bool raise = false;
#pragma unroll
        for (int r = 0; r < RP; ++r)   // where keys may be infinite, a NaN too
          raise = raise || (KIND == kCacheE5M2 ? !(x[r] <= m_ref[r] + kRaise) : x[r] > m_ref[r] + kRaise);
        if (softmax_any(raise)) {
          if constexpr (KIND == kCacheE5M2) {
#pragma unroll
            for (int r = 0; r < RP; ++r)   // rows of Q that hold a NaN or an infinity keep theirs
              if (r < seg.rows && x[r] != x[r] && pre[r] == pre[r]) {
                const Segment copy = seg;
                x[r] = whole_score<T, KIND, HD>(c, copy, r, j0 + tid);
              }
          }
          // exact maxima of the tile, shared by the four warps
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            const float m = warp_max(x[r]);
            if (lane == 0) sMax[warp * 16 + r] = m;
          }
          softmax_sync();
          float f[RP];
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            const float m = fmaxf(fmaxf(fmaxf(sMax[r], sMax[16 + r]), fmaxf(sMax[32 + r], sMax[48 + r])), m_ref[r]);
            f[r] = m == -INFINITY ? 1.f : ex2(m_ref[r] - m);
            m_ref[r] = m;
            l_run[r] *= f[r];
          }
          if (t > seg.lo) {
            ok = ok && wwait(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);   // every product so far has landed
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < C::OM * C::NP / 16; ++q) {
              uint32_t o[16];
              tmem_ld16(tmem_base + lane_addr + C::OCOL + q * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if ((q * 16 + e) % C::NP < C::PP * RP) o[e] = __float_as_uint(__uint_as_float(o[e]) * f[(q * 16 + e) % C::NP % RP]);
              tmem_st16(tmem_base + lane_addr + C::OCOL + q * 16, o);
            }
            tmem_st_wait();
            tc_fence_before();
          }
        }
        if (g >= 2) ok = ok && wwait(&o_done[g & 1], ((g - 2) >> 1) & 1);   // the P buffer has been read
        uint8_t* buf = sP + (g & 1) * C::PB;
#pragma unroll
        for (int r = 0; r < RP; r += 2) {
          const float p0 = ex2(x[r] - (m_ref[r] == -INFINITY ? 0.f : m_ref[r]));
          const float p1 = ex2(x[r + 1] - (m_ref[r + 1] == -INFINITY ? 0.f : m_ref[r + 1]));
          l_run[r] += p0;
          l_run[r + 1] += p1;
          if constexpr (C::k8) {
            uint32_t h = Pair<__half>::pack(p0 * kPScale, p1 * kPScale);
            const int at = tid & 15, ch = tid >> 4;
#pragma unroll
            for (int p = 0; p < C::PP; ++p) {
              const uint16_t e = f16x2_to_e5m2x2(h);
              const uint32_t back = fp8x2_to_f16x2<kCacheE5M2>(e);
              const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&back));
              const __half2 rest = __hmul2(d, __float2half2_rn(kPStep));
              h = *reinterpret_cast<const uint32_t*>(&rest);
              const int n = p * RP + r;
              buf[n * 128 + ((ch ^ (n & 7)) << 4) + at] = (uint8_t)(e & 0xff);
              buf[(n + 1) * 128 + ((ch ^ ((n + 1) & 7)) << 4) + at] = (uint8_t)(e >> 8);
            }
          } else {
            const int at = (tid & 7) * 2, ch = (tid & 63) >> 3;
            uint8_t* half = buf + (tid >> 6) * (C::PR * 128);
            float y0 = p0, y1 = p1;
#pragma unroll
            for (int p = 0; p < C::PP; ++p) {
              const uint32_t e = Pair<T>::pack(y0, y1);
              const float2 back = Pair<T>::unpack(e);
              y0 -= back.x;
              y1 -= back.y;
              const int n = p * RP + r;
              *reinterpret_cast<uint16_t*>(half + n * 128 + ((ch ^ (n & 7)) << 4) + at) = (uint16_t)(e & 0xffff);
              *reinterpret_cast<uint16_t*>(half + (n + 1) * 128 + ((ch ^ ((n + 1) & 7)) << 4) + at) = (uint16_t)(e >> 16);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[g & 1]);
        // the next item's Q, into the buffer whose item's scores have all landed
        if (t == seg.lo && more) store_q(item + 1);
      }

      // ---- sums over the keys (threads), then one output dim a thread
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const float l = warp_sum(l_run[r]);
        if (lane == 0) sSum[warp * 16 + r] = l;
      }
      softmax_sync();
      ok = ok && wwait(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
      tc_fence_after();
      uint32_t o[C::OM * C::NP];
#pragma unroll
      for (int q = 0; q < C::OM * C::NP / 16; ++q)
        tmem_ld16(tmem_base + lane_addr + C::OCOL + q * 16, *reinterpret_cast<uint32_t(*)[16]>(&o[q * 16]));
      tmem_ld_wait();
      tc_fence_before();   // the next item's first product overwrites O after its P, which this thread has yet to store
      const bool whole = seg.lo == 0 && seg.hi == seg.n;
      const int part = 2 * cta + (seg.lo == 0 ? 1 : 0);
      if (!whole && seg.lo == 0)   // the last of the run: each later team takes `run` tiles of the rest
        rec = PartRecord{seg.b * a.Hk + seg.hk, 1 + (seg.n - seg.hi + run - 1) / run, seg.s.q_begin, seg.rows};
      if (ok) {
        int tok = 0, in = 0;
        float my_l = 0.f, my_m = 0.f;       // of row tid
        uint32_t odd = 0;                   // bit 16 m + r: dim m * 128 + tid of row r is a NaN, and its scores are not
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          if (r < seg.rows) {
            const float l = (sSum[r] + sSum[16 + r]) + (sSum[32 + r] + sSum[48 + r]);
            const int64_t qtok = seg.s.q_begin + tok;
            const int h = seg.hk * group + in;
#pragma unroll
            for (int m = 0; m < C::OM; ++m) {
              float v = __uint_as_float(o[m * C::NP + (C::PP - 1) * RP + r]);
#pragma unroll
              for (int p = C::PP - 2; p >= 0; --p)
                v = fmaf(v, C::k8 ? 1.f / kPStep : 1.f, __uint_as_float(o[m * C::NP + p * RP + r]));
              // a NaN sum stays one: only a row that saw nothing is set to zero
              v = l == 0.f ? 0.f : v * (C::k8 ? 1.f / kPScale : 1.f) * (v_scale / l);
              const int d = m * 128 + tid;
              if (HD == 64 && tid >= 64) continue;
              if (C::kPieces && v != v && l == l) odd |= 1u << (16 * m + r);
              if (whole)
                reinterpret_cast<T*>(a.out)[qtok * a.o_rs + (int64_t)h * a.o_hs + d] = Cvt<T>::from_f32(v);
              else
                da.part_o[((int64_t)part * RP + r) * HD + d] = v;
            }
            if (tid == r) {
              my_l = l;
              my_m = m_ref[r];
            }
          }
          if (++in == group) {
            in = 0;
            ++tok;
          }
        }
        if (C::kPieces && odd != 0) {
          const Segment copy = seg;         // keeps seg itself in registers
          write_infinities<T, KIND, RP, HD>(da, copy, whole ? -1 : part, odd, v_scale);
        }
        if (tid < seg.rows && (!whole || a.lse)) {
          const float lse2 = my_l == 0.f ? -INFINITY : my_m + log2f(my_l);
          if (!whole)
            da.part_lse[part * RP + tid] = lse2;
          else
            a.lse[(int64_t)(seg.hk * group + tid % group) * a.total_q + seg.s.q_begin + tid / group] =
                my_l == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
        }
      }
      if (!more) break;
      seg = next;
    }
    if (tid == 0 && !c.whole) da.record[cta] = rec;
  }

  // ================================ teardown ======================================
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {   // a wait gave up: leave the copies and products in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TCOLS);
  }
}

// Joins the parts of the items that runs cut.  Block i does the item whose start, but not end, CTA i holds: its tail part, then
// the head parts of the same member of the teams after it.  A group of HD threads takes a row at a time; items in many parts
// (few, long sequences) have their parts dealt out over the groups instead, whose sums are added in a fixed order.
constexpr int kJoinThreads = 512;
template <typename T, int RP, int HD>
__global__ void __launch_bounds__(kJoinThreads) attn_cache_join_kernel(DecodeArgs da, int ctas) {
  const AttnArgs& a = da.c.a;
  constexpr int kJoinGroups = kJoinThreads / HD;
  __shared__ float s_acc[kJoinGroups][HD], s_w[kJoinGroups];
  asm volatile("griddepcontrol.wait;" ::: "memory");              // launched early: the parts are complete after this
  const int i = blockIdx.x;
  const PartRecord rec = da.record[i];
  if (*reinterpret_cast<volatile int*>(a.status) != 0) return;   // the parts and the records may be missing
  if (rec.item < 0) return;
  const int hk = rec.item % a.Hk;
  const int n = min(rec.parts, 1 + (ctas - 1 - i) / da.team);
  const int grp = threadIdx.x / HD, d = threadIdx.x % HD;
  const bool deal = n > 8;
  for (int r = deal ? 0 : grp; r < rec.rows; r += deal ? 1 : kJoinGroups) {
    auto slot = [&](int k) { return (int64_t)(k == 0 ? 2 * i + 1 : 2 * (i + k * da.team)) * RP + r; };
    float m = -INFINITY;
#pragma unroll 8
    for (int k = 0; k < n; ++k) m = fmaxf(m, da.part_lse[slot(k)]);
    const float ms = m == -INFINITY ? 0.f : m;
    float acc = 0.f, wsum = 0.f;
#pragma unroll 4
    for (int k = deal ? grp : 0; k < n; k += deal ? kJoinGroups : 1) {
      const float w = exp2f(da.part_lse[slot(k)] - ms), o = da.part_o[slot(k) * HD + d];
      wsum += w;
      if (w != 0.f) acc += w * o;   // NaN goes on
    }
    if (deal) {
      __syncthreads();
      s_acc[grp][d] = acc;
      if (d == 0) s_w[grp] = wsum;
      __syncthreads();
      acc = wsum = 0.f;
#pragma unroll
      for (int k = 0; k < kJoinGroups; ++k) {
        acc += s_acc[k][d];
        wsum += s_w[k];
      }
      if (grp != 0) continue;
    }
    const int64_t qtok = rec.q_begin + r / a.group;
    const int h = hk * a.group + r % a.group;
    reinterpret_cast<T*>(a.out)[qtok * a.o_rs + (int64_t)h * a.o_hs + d] = Cvt<T>::from_f32(wsum == 0.f ? 0.f : acc / wsum);
    if (a.lse && d == 0)
      a.lse[(int64_t)h * a.total_q + qtok] = wsum == 0.f ? INFINITY : (m + log2f(wsum)) * 0.6931471805599453f;
  }
}

template <typename T, int KIND, int RP, int HD>
int launch(DecodeArgs& da, cudaStream_t st) {
  using C = Cfg<T, KIND, RP, HD>;
  static_assert(C::SMEM <= 232448 && C::CTAS * (C::SMEM + 1024) <= 233472, "CTAs an SM");
  const AttnArgs& a = da.c.a;
  constexpr int ES = C::ES;
  da.page_rows = a.paged && a.block_size < BN ? a.block_size : BN;
  da.pages_per_tile = BN / da.page_rows;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const uint64_t hs = (uint64_t)(i ? a.v_hs : a.k_hs) * ES, rs = (uint64_t)(i ? a.v_rs : a.k_rs) * ES;
    const uint64_t bs = (uint64_t)(i ? a.v_bs : a.k_bs) * ES;
    const uint64_t rows = a.paged ? (uint64_t)a.block_size : (uint64_t)(a.total_k > 0 ? a.total_k : 1);
    const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)a.Hk, rows, a.paged ? (uint64_t)a.num_blocks : 1};
    const uint64_t strides[3] = {hs, rs, a.paged ? bs : rs * rows};
    const uint32_t box[4] = {(uint32_t)(C::ATOM / ES), 1, (uint32_t)da.page_rows, 1};
    const int rc = ES == 2 ? encode_tmap_16bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box)
                           : encode_tmap_8bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_decode_tcgen05_kernel<T, KIND, RP, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::SMEM));
    attr_dev = dev;
  }
  da.team = 1;
  for (int t = 2; t <= 16; ++t)
    if (a.Hk % t == 0) da.team = t;
  da.rounds = a.Hk / da.team;
  da.min_run = max(1, min(kMinRun, da.c.whole ? 1 : (a.max_k + BN - 1) / BN));   // short items need not share a CTA
  const int teams = C::CTAS * num_sms() / da.team, ctas = teams * da.team;
  da.part_o = a.ws_o;
  da.part_lse = a.ws_o + (int64_t)2 * ctas * RP * HD;
  da.record = reinterpret_cast<PartRecord*>(da.part_lse + 2 * ctas * RP);
  attn_cache_decode_tcgen05_kernel<T, KIND, RP, HD><<<dim3(da.team, teams), NUM_THREADS, C::SMEM, st>>>(maps[0], maps[1], da);
  FG_CHECK_LAUNCH("attn_cache_decode_tcgen05_kernel");
  if (da.c.whole) return FG_OK;
  // The joining kernel is launched while this one still runs (programmatic dependent launch) and waits for its end on the
  // device: the launch's latency is out of the way.
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  FG_CUDA_OK(cudaLaunchKernelEx(&cfg, attn_cache_join_kernel<T, RP, HD>, da, ctas));
  FG_CHECK_LAUNCH("attn_cache_join_kernel");
  return FG_OK;
}

template <typename T, int KIND, int HD>
int launch_rows(DecodeArgs& da, cudaStream_t st) {
  const int rows = da.c.a.max_q * da.c.a.group;
  if (rows <= 4) return launch<T, KIND, 4, HD>(da, st);
  if (rows <= 8) return launch<T, KIND, 8, HD>(da, st);
  return launch<T, KIND, 16, HD>(da, st);
}

template <typename T, int KIND>
int launch_dim(DecodeArgs& da, cudaStream_t st) {
  if (da.c.a.D == 64) return launch_rows<T, KIND, 64>(da, st);
  if constexpr (KIND != kCache16)
    if (da.c.a.D == 256) return launch_rows<T, KIND, 256>(da, st);
  return launch_rows<T, KIND, 128>(da, st);
}

template <typename T>
int launch_kind(DecodeArgs& da, int kind, cudaStream_t st) {
  if (kind == kCacheE4M3) return launch_dim<T, kCacheE4M3>(da, st);
  if (kind == kCacheE5M2) return launch_dim<T, kCacheE5M2>(da, st);
  return launch_dim<T, kCache16>(da, st);
}

}  // namespace

// Bytes of workspace for `rows` query rows of a sequence and KV head: a head and a tail part, and a record, for each CTA.
int64_t attn_cache_decode_sm100_bytes(int64_t rows, int64_t head_dim, int sms) {
  const int64_t rp = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  return 2 * (int64_t)sms * (2 * rp * (head_dim + 1) * 4 + (int64_t)sizeof(PartRecord));
}

int attn_cache_decode_sm100(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  DecodeArgs da;
  da.c = c;
  if (!c.a.status) return fail(FG_ERR_CUDA, "flash_attn_cache: device status word unavailable");
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(da, kind, st) : launch_kind<__half>(da, kind, st);
}

}  // namespace fg
