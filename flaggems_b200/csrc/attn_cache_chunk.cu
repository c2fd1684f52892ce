// Attention of a chunk of new tokens over an 8-bit or windowed cache, head dim 128, on the tcgen05 tensor cores.
//
// CTA = one or two 128-row Q tiles of one (sequence, KV head) and a range of its K/V tiles of 128 keys.  A row is a
// (token, head of the group) pair, so a chunk of a few tokens fills the tiles as well as a long one, and all query heads
// of the group share every K/V tile.  A tile holds floor(128 / group) tokens.
//
//   warps 0-7    softmax, one warpgroup per Q tile, one thread per row (TMEM lane = row): scores of 64 keys from TMEM to
//                registers, mask, running maximum (raised only when it grows by more than 8 in log2 units), exponentials,
//                probabilities back to TMEM as 16 bit; at the end they normalise and write the output rows
//   warp 8       TMA producer: Q once, then K and V tiles, walking the tile runs (first tokens, then the window)
//   warps 9, 10  score-issuing thread of each Q tile: S = Q K^T, 64 keys a step
//   warp 11      O += P V of both tiles
//   warps 12-15  8-bit caches: widen each K/V tile from the 16 KB landing slots to the fp16 tiles that the tensor cores
//                read (128-byte swizzled, K-major), zeroing V rows that no row of the CTA sees; for bf16 queries they first
//                bring Q to fp16, each row by a power of two
// TMEM columns: tile t has its scores at t*128 (64 columns), two probability buffers at t*128+64 and +96, its output at
// 256+t*128.  Every wait is an mbarrier wait with a limit.
#include "attn_cache_common.cuh"
#include "sm100_common.cuh"

namespace fg {
namespace {

constexpr int BM = 128, BN = 128, HD = 128, STEP = 64;
constexpr int HALF_BYTES = 128 * 64 * 2;     // one [128 x 64] swizzled 16-bit sub-tile
constexpr int TILE_BYTES = 2 * HALF_BYTES;   // 32 KB
constexpr int RAW_BYTES = BN * HD;           // one 8-bit K or V tile, 16 KB
constexpr int TMA_WARP = 8, MMA_WARP0 = 9, CONV_WARP0 = 12;
constexpr int TMEM_COLS = 512;
constexpr float kRescaleThreshold = 8.0f;    // log2 units

constexpr int threads_of(int kind) { return kind == kCache16 ? 12 * 32 : 16 * 32; }
constexpr int smem_of(int kind) { return 6 * TILE_BYTES + (kind == kCache16 ? 0 : 2 * RAW_BYTES) + 1024 + 256 + 2 * BM * 4; }

struct ChunkArgs {
  CacheAttnArgs c;
  int tiles;            // Q tiles per CTA (1 or 2)
  int tokens;           // tokens of a Q tile
  int page_rows;        // keys per TMA box
  int pages_per_tile;
  int num_mb;           // Q tile pairs of the longest chunk
};

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

template <typename T, int KIND>
__global__ void __launch_bounds__(threads_of(KIND), 1)
attn_cache_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ ChunkArgs pa) {
  using namespace sm100;
  using M = typename std::conditional<KIND == kCache16, T, __half>::type;   // type of the products
  constexpr bool kBf16 = std::is_same<M, __nv_bfloat16>::value;
  constexpr bool kConvQ = !std::is_same<T, M>::value;
  constexpr bool kWiden = KIND != kCache16;
  const CacheAttnArgs& c = pa.c;
  const AttnArgs& a = c.a;
  const int NT = pa.tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // heaviest (latest) query blocks of all sequences and heads first
  int idx = blockIdx.x;
  const int split = idx % a.num_splits;
  idx /= a.num_splits;
  const int hk = idx % a.Hk;
  idx /= a.Hk;
  const int b = idx % a.batch;
  const int m0 = (pa.num_mb - 1 - idx / a.batch) * NT * pa.tokens;   // first token
  const SeqInfo s = seq_info(a, b);
  if (m0 >= s.q_len) return;
  __shared__ int s_drain;
  if (threadIdx.x == 0) s_drain = *reinterpret_cast<volatile int*>(a.status);
  __syncthreads();
  if (s_drain != 0) return;   // a wait gave up on this device: finish the launch quickly

  const int shift = s.k_len - s.q_len;
  const int m_last = min(s.q_len, m0 + NT * pa.tokens) - 1;          // last token
  const TileSpan span = tile_span<BN>(c, s.k_len, m0 + shift, m_last + shift);
  const int i_begin = split * c.tiles_per_split;
  const int n_tiles = max(0, (a.num_splits > 1 ? min(span.n, i_begin + c.tiles_per_split) : span.n) - i_begin);
  const RowMask cta_first = row_mask(c, s.k_len, m0 + shift), cta_last = row_mask(c, s.k_len, m_last + shift);
  // steps of 64 keys; the second half of the last tile is left out when it is not visible
  const int n_steps = n_tiles == 0 ? 0
                                   : 2 * n_tiles - (span.tile(i_begin + n_tiles - 1) * BN + STEP >= cta_last.hi ? 1 : 0);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // [2 tiles][2 halves][128 x 64]
  uint8_t* sK = smem + 2 * TILE_BYTES;      // [2 stages]
  uint8_t* sV = smem + 4 * TILE_BYTES;      // [2 stages]
  uint8_t* sR = smem + 6 * TILE_BYTES;      // [2 slots] 8-bit tiles as they arrive: K, V, K, V, ...
  uint8_t* rest = sR + (kWiden ? 2 * RAW_BYTES : 0);
  uint64_t* bars = reinterpret_cast<uint64_t*>(rest);
  uint64_t* q_full = bars;            // Q tiles have landed
  uint64_t* q_ready = bars + 1;       // ... and hold M
  uint64_t* k_full = bars + 2;        // [2]
  uint64_t* k_empty = bars + 4;       // [2]
  uint64_t* v_full = bars + 6;        // [2]
  uint64_t* v_empty = bars + 8;       // [2]
  uint64_t* s_full = bars + 10;       // [2 tiles] scores of a step have landed in the tile's score buffer
  uint64_t* s_free = bars + 12;       // [2 tiles] ... and have been read into registers
  uint64_t* p_ready = bars + 14;      // [2 tiles][2 probability buffers]
  uint64_t* o_done = bars + 18;       // [2 tiles][2]: P V of even / odd steps
  uint64_t* r_full = bars + 22;       // [2 slots]
  uint64_t* r_empty = bars + 24;      // [2 slots]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 26);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sDown = reinterpret_cast<float*>(rest + 256);   // [2 tiles][128]

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_ready, 4);            // one arrival per widening warp
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], kWiden ? 4 : 1);
      mbar_init(&k_empty[i], NT);
      mbar_init(&v_full[i], kWiden ? 4 : 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);       // one arrival per softmax warp of the tile
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_ready[i], 4);
    for (int i = 0; i < 4; ++i) mbar_init(&o_done[i], 1);
    mbar_fence_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == MMA_WARP0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // lane 0 polls for its warp, so that a wait that gave up takes the whole warp the same way
  auto wait1 = [&](uint64_t* bar, uint32_t parity) -> bool {
    return mbar_wait(bar, parity, abort_flag, a.status, kStatusAttnTimeout);
  };
  auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool {
    int r = 1;
    if (lane == 0) r = wait1(bar, parity) ? 1 : 0;
    r = __shfl_sync(0xffffffffu, r, 0);
    __syncwarp();   // what lane 0 has seen arrive is there for the others
    return r != 0;
  };

  if (n_steps > 0 && warp == TMA_WARP) {
    // ================================ TMA producer ================================
    if (lane == 0) {
      mbar_expect_tx(q_full, NT * 2 * pa.tokens * a.group * 128);
      for (int t = 0; t < NT; ++t)
        for (int hf = 0; hf < 2; ++hf)
          tma_load_3d(sQ + t * TILE_BYTES + hf * HALF_BYTES, &tmap_q, q_full, hf * 64, hk * a.group,
                      s.q_begin + m0 + t * pa.tokens);
    }
    __syncwarp();
    const int32_t* bt_row = a.paged ? a.block_table + (int64_t)b * a.bt_stride : nullptr;
    const int last_page = a.paged ? max(0, (s.k_len - 1) / a.block_size) : 0;
    auto lookup = [&](int j, int& page, int& row) {
      page = 0;
      row = 0;
      if (j >= n_tiles) return;
      const int tok = span.tile(i_begin + j) * BN + lane * pa.page_rows;
      if (!a.paged) {
        row = s.k_begin + tok;
      } else if (lane < pa.pages_per_tile) {
        const int pg = tok / a.block_size;
        row = tok - pg * a.block_size;
        page = cache_page(c, bt_row, min(pg, last_page));  // past the sequence: any valid page (those keys are masked)
      }
    };
    int page, row;
    lookup(0, page, row);
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      int npage, nrow;
      lookup(j + 1, npage, nrow);
      for (int which = 0; which < 2; ++which) {
        const CUtensorMap* tm = which ? &tmap_v : &tmap_k;
        if constexpr (kWiden) {
          const uint32_t n = 2 * j + which;
          const int slot = n & 1;
          if (!wwait(&r_empty[slot], ((n >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(&r_full[slot], RAW_BYTES);
          __syncwarp();
          if (lane < pa.pages_per_tile)
            tma_load_4d(sR + slot * RAW_BYTES + lane * pa.page_rows * 128, tm, &r_full[slot], 0, hk, row, page);
        } else {
          const int stg = j & 1;
          uint64_t* full = which ? &v_full[stg] : &k_full[stg];
          if (!wwait(which ? &v_empty[stg] : &k_empty[stg], ((j >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(full, TILE_BYTES);
          __syncwarp();
          if (lane < pa.pages_per_tile) {
            uint8_t* dst = (which ? sV : sK) + stg * TILE_BYTES + lane * pa.page_rows * 128;
            for (int hf = 0; hf < 2; ++hf) tma_load_4d(dst + hf * HALF_BYTES, tm, full, hf * 64, hk, row, page);
          }
        }
      }
      page = npage;
      row = nrow;
    }
  } else if (n_steps > 0 && warp >= MMA_WARP0 && warp < MMA_WARP0 + NT) {
    // ================================ scores of one tile ==========================
    const int t = warp - MMA_WARP0;
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_f16(kBf16, false, false, BM, STEP);
      const uint32_t desc_hi = (uint32_t)(umma_desc_sw128(0, 0, 1024) >> 32);
      const uint32_t q_lo = (uint32_t)umma_desc_sw128(smem_u32(sQ + t * TILE_BYTES), 0, 1024);
      const uint32_t k_lo0 = (uint32_t)umma_desc_sw128(smem_u32(sK), 0, 1024);
      const uint32_t s_tmem = tmem_base + t * 128;
      bool ok = wait1(kConvQ ? q_ready : q_full, 0);
      for (int i = 0; i < n_steps && ok; ++i) {
        const int j = i >> 1, stg = j & 1;
        if (!(i & 1) && !wait1(&k_full[stg], (j >> 1) & 1)) break;
        // the previous step's scores must have been read out
        if (i > 0 && !wait1(&s_free[t], (i - 1) & 1)) break;
        // the softmax warps will store P(i) over the buffer that the P V of step i - 2 reads
        if (i >= 2 && !wait1(&o_done[t * 2 + (i & 1)], ((i - 2) >> 1) & 1)) break;
        tc_fence_after();
        const uint32_t k_lo = k_lo0 + stg * (TILE_BYTES >> 4) + (i & 1) * (STEP * 128 >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k >> 2) * HALF_BYTES + (k & 3) * 32) >> 4;
          mma_f16_ss_lohi(s_tmem, q_lo + off, k_lo + off, desc_hi, idesc, k != 0 ? 1u : 0u);
        }
        tc_commit(&s_full[t]);
        if ((i & 1) || i == n_steps - 1) tc_commit(&k_empty[stg]);
      }
    }
  } else if (n_steps > 0 && warp == MMA_WARP0 + 2) {
    // ================================ O += P V of both tiles =======================
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_f16(kBf16, false, true, BM, HD);   // V is MN-major
      const uint32_t desc_hi = (uint32_t)(umma_desc_sw128(0, 0, 1024) >> 32);
      const uint32_t v_lo0 = (uint32_t)umma_desc_sw128(smem_u32(sV), HALF_BYTES, 1024);
      bool ok = true;
      for (int i = 0; i < n_steps && ok; ++i) {
        const int j = i >> 1, stg = j & 1;
        if (!(i & 1) && !wait1(&v_full[stg], (j >> 1) & 1)) break;
        const uint32_t v_lo = v_lo0 + stg * (TILE_BYTES >> 4) + (i & 1) * (4 * 2048 >> 4);
        for (int t = 0; t < NT && ok; ++t) {
          if (!wait1(&p_ready[t * 2 + (i & 1)], (i >> 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t p_tmem = tmem_base + t * 128 + STEP + (i & 1) * 32;
          const uint32_t o_tmem = tmem_base + 256 + t * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_ts_lohi(o_tmem, p_tmem + k * 8, v_lo + k * (2048 >> 4), desc_hi, idesc, (i > 0 || k > 0) ? 1u : 0u);
          tc_commit(&o_done[t * 2 + (i & 1)]);
        }
        if (ok && ((i & 1) || i == n_steps - 1)) tc_commit(&v_empty[stg]);
      }
    }
  } else if (kWiden && n_steps > 0 && warp >= CONV_WARP0) {
    // ================================ widening =====================================
    if constexpr (kWiden) {
      const int w = warp - CONV_WARP0;
      bool ok = true;
      if constexpr (kConvQ) {
        ok = wwait(q_full, 0);
        if (ok) {
          const int r = w * 32 + lane;   // a thread per row
          for (int t = 0; t < NT; ++t) {
            uint8_t* q = sQ + t * TILE_BYTES + r * 128;
            float top = 0.f;
#pragma unroll 4
            for (int ch = 0; ch < 16; ++ch) {
              float f[8];
              Vec16<T>::unpack(*reinterpret_cast<const uint4*>(q + (ch >> 3) * HALF_BYTES + (((ch & 7) ^ (r & 7)) << 4)), f);
#pragma unroll
              for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
            }
            float up, down;
            row_power(top, up, down);
#pragma unroll 4
            for (int ch = 0; ch < 16; ++ch) {
              uint4* at = reinterpret_cast<uint4*>(q + (ch >> 3) * HALF_BYTES + (((ch & 7) ^ (r & 7)) << 4));
              float f[8];
              Vec16<T>::unpack(*at, f);
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] *= up;
              *at = Vec16<__half>::pack(f);
            }
            sDown[t * BM + r] = down;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_ready);
        }
      }
      // lane = (row of four, 16-byte piece): eight lanes read one row's 128 bytes and write one row's 128 bytes of
      // either half at a time (pieces 4-7 store their second eight values first), without bank conflicts
      const int ch = lane & 7, sub = lane >> 3;
      for (int n = 0; n < 2 * n_tiles && ok; ++n) {
        const int j = n >> 1, stg = j & 1, slot = n & 1;
        const bool is_v = n & 1;
        if (!wwait(&r_full[slot], j & 1) || !wwait(is_v ? &v_empty[stg] : &k_empty[stg], ((j >> 1) & 1) ^ 1)) break;
        const uint8_t* src = sR + slot * RAW_BYTES;
        uint8_t* dst = (is_v ? sV : sK) + stg * TILE_BYTES + (ch >> 2) * HALF_BYTES;
        const int j0 = span.tile(i_begin + j) * BN;
        const bool zero = is_v && (j0 + BN > cta_last.hi || (j0 < cta_first.lo && j0 + BN > c.sinks));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = w * 32 + k * 4 + sub;
          uint4 raw = *reinterpret_cast<const uint4*>(src + r * 128 + ((ch ^ (r & 7)) << 4));
          if (zero) {   // V rows that no row of the CTA sees must not reach the products
            const int col = j0 + r;
            if (col >= cta_last.hi || (col < cta_first.lo && col >= c.sinks)) raw = make_uint4(0, 0, 0, 0);
          }
          uint4 lo, hi;
          fp8x4_to_f16x4<KIND>(raw.x, lo.x, lo.y);
          fp8x4_to_f16x4<KIND>(raw.y, lo.z, lo.w);
          fp8x4_to_f16x4<KIND>(raw.z, hi.x, hi.y);
          fp8x4_to_f16x4<KIND>(raw.w, hi.z, hi.w);
          const bool swap = ch & 4;
          const int c0 = (ch & 3) * 2 + (swap ? 1 : 0);
          uint8_t* row = dst + r * 128;
          *reinterpret_cast<uint4*>(row + ((c0 ^ (r & 7)) << 4)) = swap ? hi : lo;
          *reinterpret_cast<uint4*>(row + (((c0 ^ 1) ^ (r & 7)) << 4)) = swap ? lo : hi;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(is_v ? &v_full[stg] : &k_full[stg]);
          mbar_arrive(&r_empty[slot]);
        }
      }
    }
  } else if (warp < 4 * NT) {
    // ================================ softmax / epilogue ===========================
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;     // row inside the tile == TMEM lane
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + t * 128;
    const uint32_t o_addr = tmem_base + lane_addr + 256 + t * 128;
    const int tile_first = m0 + t * pa.tokens;
    const int tok = tile_first + r / a.group, h = hk * a.group + r % a.group;
    const bool valid = r < pa.tokens * a.group && tok < s.q_len;
    const int64_t qtok = s.q_begin + tok;
    const RowMask mask = row_mask(c, s.k_len, tok + shift);
    // what the first and the last row of the tile see: steps between need no mask
    const RowMask first = row_mask(c, s.k_len, tile_first + shift);
    const RowMask last = row_mask(c, s.k_len, min(tile_first + pa.tokens, s.q_len) - 1 + shift);
    float m_used = -INFINITY, l_run = 0.f;
    float scale = a.scale_log2 * cache_scale(c.k_scale, c.ks_batch, c.ks_head, b, hk);
    bool ok = true;
    if constexpr (kConvQ) {
      if (n_steps > 0) {
        ok = wwait(q_ready, 0);
        scale *= sDown[t * BM + r];
      }
    }
    const bool odd_scale = !(scale > 0.f);    // a K scale that is zero, negative or NaN: scale the scores first

    for (int i = 0; i < n_steps && ok; ++i) {
      const uint32_t p_addr = s_addr + STEP + (i & 1) * 32;
      if (!wwait(&s_full[t], i & 1)) {
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
      const int col0 = span.tile(i_begin + (i >> 1)) * BN + (i & 1) * STEP;
      if (col0 + STEP > first.hi || (col0 < last.lo && col0 + STEP > c.sinks)) {
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (mask.dead(col0 + e)) sv[e] = -INFINITY;
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
      if (i > 0 && __any_sync(0xffffffffu, raise)) {
        // every P V issued so far must have landed before O is touched
        if (!wwait(&o_done[t * 2 + ((i - 1) & 1)], ((i - 1) >> 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float f = raise ? ex2(m_used - m_tile) : 1.0f;
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
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
      const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
      if constexpr (!kWiden) {
        // V rows of this step that no row of the CTA sees must not reach the products: zeroed in place, by each tile's
        // warps for themselves (the other tile writes the same zeros)
        if (col0 + STEP > cta_last.hi || (col0 < cta_first.lo && col0 + STEP > c.sinks)) {
          const int j = i >> 1, stg = j & 1;
          if (!wwait(&v_full[stg], (j >> 1) & 1)) {
            ok = false;
            break;
          }
          uint8_t* vt = sV + stg * TILE_BYTES + (i & 1) * STEP * 128;
          for (int at = r; at < STEP * 16; at += 128) {
            const int row = at / 16, ch = at % 16, col = col0 + row;
            if (col >= cta_last.hi || (col < cta_first.lo && col >= c.sinks))
              *reinterpret_cast<uint4*>(vt + (ch >> 3) * HALF_BYTES + row * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
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
      if (lane == 0) mbar_arrive(&p_ready[t * 2 + (i & 1)]);
    }

    // ---- epilogue: normalise my row of O and write it out
    if (ok && n_steps > 0) {
      ok = wwait(&o_done[t * 2 + ((n_steps - 1) & 1)], ((n_steps - 1) >> 1) & 1);
      tc_fence_after();
    }
    if (ok) {
      // a NaN sum stays one: only a row that saw nothing is set to zero
      const float inv = l_run == 0.f ? 0.f : cache_scale(c.v_scale, c.vs_batch, c.vs_head, b, hk) / l_run;
      const bool parts = a.num_splits > 1;
      char* orow = parts ? reinterpret_cast<char*>(a.ws_o + (((int64_t)split * a.total_q + qtok) * a.H + h) * HD)
                         : reinterpret_cast<char*>(a.out) + (qtok * a.o_rs + (int64_t)h * a.o_hs) * 2;
      // an empty split's partial output is never read (its weight is zero)
      if (n_steps > 0 || !parts) {
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
          uint32_t o[16];
          if (n_steps > 0) {
            tmem_ld16(o_addr + q * 16, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0u;
          }
          float f[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]) * inv;
          if (valid && parts) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(orow + q * 64 + e * 16) = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<uint4*>(orow + q * 32 + e * 16) =
                  make_uint4(Pair<T>::pack(f[8 * e], f[8 * e + 1]), Pair<T>::pack(f[8 * e + 2], f[8 * e + 3]),
                             Pair<T>::pack(f[8 * e + 4], f[8 * e + 5]), Pair<T>::pack(f[8 * e + 6], f[8 * e + 7]));
          }
          __syncwarp();
        }
      }
      if (valid) {
        const float lse2 = l_run == 0.f ? -INFINITY : m_used + log2f(l_run);
        if (parts)
          a.ws_lse[((int64_t)split * a.H + h) * a.total_q + qtok] = lse2;
        else if (a.lse)
          a.lse[(int64_t)h * a.total_q + qtok] = l_run == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
      }
    }
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

template <typename T, int KIND>
int launch(ChunkArgs& pa, cudaStream_t st) {
  const AttnArgs& a = pa.c.a;
  constexpr int ES = KIND == kCache16 ? 2 : 1;
  pa.page_rows = a.paged && a.block_size < BN ? a.block_size : BN;
  pa.pages_per_tile = BN / pa.page_rows;
  CUtensorMap tq, maps[2];
  {
    const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)a.H, (uint64_t)a.total_q};
    const uint64_t strides[2] = {(uint64_t)a.q_hs * 2, (uint64_t)a.q_rs * 2};
    const uint32_t box[3] = {64, (uint32_t)a.group, (uint32_t)pa.tokens};
    const int rc = encode_tmap_16bit(&tq, a.q, 3, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    const uint64_t hs = (uint64_t)(i ? a.v_hs : a.k_hs) * ES, rs = (uint64_t)(i ? a.v_rs : a.k_rs) * ES;
    const uint64_t bs = (uint64_t)(i ? a.v_bs : a.k_bs) * ES;
    const uint64_t rows = a.paged ? (uint64_t)a.block_size : (uint64_t)(a.total_k > 0 ? a.total_k : 1);
    const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)a.Hk, rows, a.paged ? (uint64_t)a.num_blocks : 1};
    const uint64_t strides[3] = {hs, rs, a.paged ? bs : rs * rows};
    const uint32_t box[4] = {(uint32_t)(128 / ES), 1, (uint32_t)pa.page_rows, 1};
    const int rc = ES == 2 ? encode_tmap_16bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box)
                           : encode_tmap_8bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  constexpr int smem = smem_of(KIND);
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_chunk_kernel<T, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_dev = dev;
  }
  const int64_t ctas = (int64_t)pa.num_mb * a.batch * a.Hk * a.num_splits;
  if (ctas > 2147483647LL) return fail(FG_ERR_TOO_LARGE, "flash_attn_cache: too many query blocks");
  attn_cache_chunk_kernel<T, KIND><<<(unsigned)ctas, threads_of(KIND), smem, st>>>(tq, maps[0], maps[1], pa);
  FG_CHECK_LAUNCH("attn_cache_chunk_kernel");
  return FG_OK;
}

template <typename T>
int launch_kind(ChunkArgs& pa, int kind, cudaStream_t st) {
  if (kind == kCacheE4M3) return launch<T, kCacheE4M3>(pa, st);
  if (kind == kCacheE5M2) return launch<T, kCacheE5M2>(pa, st);
  return launch<T, kCache16>(pa, st);
}

}  // namespace

int attn_cache_chunk(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  ChunkArgs pa;
  pa.c = c;
  if (!c.a.status) return fail(FG_ERR_CUDA, "flash_attn_cache: device status word unavailable");
  pa.tokens = BM / c.a.group;
  pa.tiles = c.a.max_q > pa.tokens ? 2 : 1;
  pa.num_mb = (c.a.max_q + pa.tiles * pa.tokens - 1) / (pa.tiles * pa.tokens);
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(pa, kind, st) : launch_kind<__half>(pa, kind, st);
}

}  // namespace fg
