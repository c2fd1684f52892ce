// Attention of a few query rows (at most 16 (token, head of the group) pairs of a sequence) over an 8-bit or windowed
// cache, head dim 128, on the tcgen05 tensor cores.  Memory bound: every cached byte is read once, and nothing else is
// done with it -- the tensor cores read K and V from shared memory in the type and layout that TMA delivers.
//
// The products are turned round, so that the many keys fill the 128 rows of the instruction and the few query rows its
// columns:
//     S^T [128 keys x N] = K [keys x 128] Q^T          K is the K-major A operand as it lies in the cache
//     O^T [128 dims x N] += V^T [128 x keys] P^T       V is the MN-major A operand as it lies in the cache
// A thread of the four softmax warps owns one key (TMEM lane): it holds that key's scores of all rows, so nothing is spent
// on rows that are not there.
//
// 8-bit caches: Q and P are split into 8-bit pieces, each with columns of its own, and the columns are added up in fp32.
//   Q   a row is multiplied by a power of two that takes its largest value to [2^7, 2^8) and parted into e4m3 pieces, each
//       the rounding of what the previous left: 2 pieces hold the 8 bits of a bf16 significand, 3 the 11 bits of fp16,
//       down to 2^-18 of the row's largest value (an e4m3 subnormal step)
//   P   2^11 p (p <= 2^4, see below), rounded to fp16, in four e5m2 pieces of three bits, which hold all of it down to
//       2^-28; e5m2 for its range: long contexts have many small probabilities
// 16-bit caches: Q as it is; P in one fp16 piece, or two bf16 pieces (2^-17).
//
// The running maximum is shared by the CTA and raised only when a score exceeds it by more than 4 (log2 units); the warps
// agree on that with one barrier reduction a tile.  Only a raise needs the exact maximum and rescales O in TMEM.
//
//   warps 0-3   softmax and output        warp 4   TMA producer (K and V tiles of 128 keys alternate in one ring)
//   warp 5      issues the products: scores of the next tile before P V of the current one
#include "attn_cache_common.cuh"
#include "sm100_common.cuh"

namespace fg {
namespace {

constexpr int BN = 128, HD = 128, NUM_THREADS = 192;
constexpr int TMA_WARP = 4, MMA_WARP = 5;
constexpr float kRaise = 4.0f;               // log2 units
constexpr float kPScale = 2048.0f;           // of P before it is split (8-bit caches)

constexpr int up16(int n) { return (n + 15) / 16 * 16; }

// T: query type; KIND: cache; RP: query rows, rounded up to 4, 8 or 16
template <typename T, int KIND, int RP>
struct Cfg {
  static constexpr bool k8 = KIND != kCache16;
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int PQ = !k8 ? 1 : (kBf16 ? 2 : 3);        // pieces of Q
  static constexpr int PP = k8 ? 4 : (kBf16 ? 2 : 1);         // pieces of P
  static constexpr int NS = up16(RP * PQ), NP = up16(RP * PP);   // columns of the two products
  static constexpr int TILE = BN * HD * (k8 ? 1 : 2);         // bytes of a K or V tile
  static constexpr int SLOTS = k8 ? (RP == 16 ? 5 : 6) : 3;   // 80 to 96 KB: two CTAs an SM (one for RP 16, 16 bit)
  static constexpr int QB = NS * HD * (k8 ? 1 : 2);           // bytes of Q
  static constexpr int PB = NP * BN * (k8 ? 1 : 2);           // bytes of one P buffer
  static constexpr int SCOL = NS <= 32 ? 32 : 64;             // TMEM columns of one score buffer
  static constexpr int OCOL = 2 * SCOL;
  static constexpr int TCOLS = OCOL + NP <= 128 ? 128 : 256;
  static constexpr int SMEM = SLOTS * TILE + QB + 2 * PB + 1024 + 256 + 2 * 4 * 16 * 4;
};

struct DecodeArgs {
  CacheAttnArgs c;
  int page_rows, pages_per_tile;
};

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

template <typename T, int KIND, int RP>
__global__ void __launch_bounds__(NUM_THREADS, 2)
attn_cache_decode_tcgen05_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                 const __grid_constant__ DecodeArgs da) {
  using namespace sm100;
  using C = Cfg<T, KIND, RP>;
  const CacheAttnArgs& c = da.c;
  const AttnArgs& a = c.a;
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const SeqInfo s = seq_info(a, b);
  const int group = a.group;
  const int rows = min(s.q_len * group, RP);
  if (rows < 1) return;
  __shared__ int s_drain;
  if (threadIdx.x == 0) s_drain = *reinterpret_cast<volatile int*>(a.status);
  __syncthreads();
  if (s_drain != 0) return;   // a wait gave up on this device: finish the launch quickly
  const int shift = s.k_len - s.q_len;
  const int t_last = (rows - 1) / group;
  const TileSpan span = tile_span<BN>(c, s.k_len, shift, t_last + shift);
  const int i_begin = split * c.tiles_per_split;
  const int n_tiles = (a.num_splits > 1 ? min(span.n, i_begin + c.tiles_per_split) : span.n) - i_begin;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t q0 = s.q_begin;

  if (n_tiles <= 0) {  // nothing visible in this range: contributes nothing
    if (tid < rows) {
      const int64_t qtok = q0 + tid / group;
      const int h = hk * group + tid % group;
      if (a.num_splits > 1)
        a.ws_lse[((int64_t)split * a.H + h) * a.total_q + qtok] = -INFINITY;
      else if (a.lse)
        a.lse[(int64_t)h * a.total_q + qtok] = INFINITY;
    }
    if (a.num_splits == 1)
      for (int i = tid; i < rows * HD; i += NUM_THREADS) {
        const int r = i / HD;
        reinterpret_cast<T*>(a.out)[(q0 + r / group) * a.o_rs + (int64_t)(hk * group + r % group) * a.o_hs + i - r * HD] =
            Cvt<T>::from_f32(0.f);
      }
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sP = smem + C::SLOTS * C::TILE;                        // [2 buffers]
  uint8_t* sQ = sP + 2 * C::PB;
  uint64_t* full = reinterpret_cast<uint64_t*>(sQ + C::QB);       // [SLOTS]
  uint64_t* empty = full + C::SLOTS;
  uint64_t* s_full = empty + C::SLOTS;   // [2] scores of a tile have landed
  uint64_t* s_free = s_full + 2;         // [2] ... and have been read into registers
  uint64_t* p_ready = s_free + 2;        // [2]
  uint64_t* o_done = p_ready + 2;        // [2] P V of even / odd tiles
  uint64_t* q_ready = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sRed = reinterpret_cast<float*>(sQ + C::QB + 256);       // [4 warps][16] maxima, then as many sums

  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_ready, 4);
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, C::TCOLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
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

  if (warp == TMA_WARP) {
    // ================================ producer ====================================
    const int32_t* bt_row = a.paged ? a.block_table + (int64_t)b * a.bt_stride : nullptr;
    const int last_page = a.paged ? max(0, (s.k_len - 1) / a.block_size) : 0;
    auto lookup = [&](int t, int& page, int& row) {
      page = 0;
      row = 0;
      if (t >= n_tiles) return;
      const int tok = span.tile(i_begin + t) * BN + lane * da.page_rows;
      if (!a.paged) {
        row = s.k_begin + tok;
      } else if (lane < da.pages_per_tile) {
        const int pg = tok / a.block_size;
        row = tok - pg * a.block_size;
        page = cache_page(c, bt_row, min(pg, last_page));  // past the sequence: any valid page (those keys are masked)
      }
    };
    int page, row;
    lookup(0, page, row);
    bool ok = true;
    for (int t = 0; t < n_tiles && ok; ++t) {
      int npage, nrow;
      lookup(t + 1, npage, nrow);  // the table entry of the next tile is in flight while this one is issued
      for (int which = 0; which < 2; ++which) {
        const int n = 2 * t + which, slot = n % C::SLOTS;
        if (!wwait(&empty[slot], ((n / C::SLOTS) & 1) ^ 1)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(&full[slot], C::TILE);
        __syncwarp();
        if (lane < da.pages_per_tile) {
          uint8_t* dst = smem + slot * C::TILE + lane * da.page_rows * 128;
          const CUtensorMap* tm = which ? &tmap_v : &tmap_k;
          tma_load_4d(dst, tm, &full[slot], 0, hk, row, page);
          if constexpr (!C::k8) tma_load_4d(dst + C::TILE / 2, tm, &full[slot], 64, hk, row, page);
        }
      }
      page = npage;
      row = nrow;
    }
  } else if (warp == MMA_WARP) {
    // ================================ products ====================================
    if (lane == 0) {
      const uint32_t id_s = C::k8 ? umma_idesc_f8(KIND == kCacheE5M2, false, false, false, BN, C::NS)
                                  : umma_idesc_f16(C::kBf16, false, false, BN, C::NS);
      const uint32_t id_o = C::k8 ? umma_idesc_f8(KIND == kCacheE5M2, true, true, false, HD, C::NP)
                                  : umma_idesc_f16(C::kBf16, true, false, HD, C::NP);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ), 0, 1024);
      auto scores = [&](int t) -> bool {
        const int n = 2 * t, slot = n % C::SLOTS;
        if (!wait1(&full[slot], (n / C::SLOTS) & 1)) return false;
        if (t >= 2 && !wait1(&s_free[t & 1], ((t - 2) >> 1) & 1)) return false;   // scores two tiles back are read
        tc_fence_after();
        const uint64_t k_desc = umma_desc_sw128(smem_u32(smem + slot * C::TILE), 0, 1024);
        const uint32_t d = tmem_base + (t & 1) * C::SCOL;
        if constexpr (C::k8) {
#pragma unroll
          for (int k = 0; k < HD / 32; ++k) mma_f8_ss(d, k_desc + k * 2, q_desc + k * 2, id_s, k != 0);
        } else {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            mma_f16_ss(d, k_desc + (k >> 2) * (C::TILE / 2 / 16) + (k & 3) * 2, q_desc + (k >> 2) * (C::NS * 128 / 16) + (k & 3) * 2,
                       id_s, k != 0);
        }
        tc_commit(&s_full[t & 1]);
        tc_commit(&empty[slot]);
        return true;
      };
      bool ok = wait1(q_ready, 0) && scores(0);
      for (int t = 0; t < n_tiles && ok; ++t) {
        if (t + 1 < n_tiles && !scores(t + 1)) break;
        const int n = 2 * t + 1, slot = n % C::SLOTS;
        if (!wait1(&full[slot], (n / C::SLOTS) & 1) || !wait1(&p_ready[t & 1], (t >> 1) & 1)) break;
        tc_fence_after();
        const uint64_t v_desc = umma_desc_sw128(smem_u32(smem + slot * C::TILE), C::k8 ? C::TILE : C::TILE / 2, 1024);
        const uint64_t p_desc = umma_desc_sw128(smem_u32(sP + (t & 1) * C::PB), 0, 1024);
        const uint32_t d = tmem_base + C::OCOL;
        if constexpr (C::k8) {
#pragma unroll
          for (int k = 0; k < BN / 32; ++k) mma_f8_ss(d, v_desc + k * (4096 >> 4), p_desc + k * 2, id_o, t > 0 || k > 0);
        } else {
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            mma_f16_ss(d, v_desc + k * (2048 >> 4), p_desc + (k >> 2) * (C::NP * 128 / 16) + (k & 3) * 2, id_o, t > 0 || k > 0);
        }
        tc_commit(&o_done[t & 1]);
        tc_commit(&empty[slot]);
      }
    }
  } else {
    // ================================ softmax / output =============================
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    // ---- Q, split into pieces: 128 / RP threads a row, RP values each
    float pre[RP];           // takes a sum of columns to the scores
    {
      constexpr int TPR = 128 / RP;
      const int r = tid / TPR, d0 = (tid % TPR) * RP;
      const bool live = r < rows;
      const int tok = live ? r / group : 0;
      const T* q = reinterpret_cast<const T*>(a.q) + (q0 + tok) * a.q_rs + (int64_t)(hk * group + (live ? r - tok * group : 0)) * a.q_hs + d0;
      uint32_t w[RP / 2];
#pragma unroll
      for (int i = 0; i < RP / 4; ++i) {
        const uint2 u = live ? *reinterpret_cast<const uint2*>(q + i * 4) : make_uint2(0, 0);
        w[2 * i] = u.x;
        w[2 * i + 1] = u.y;
      }
      float down = 1.f;
      if constexpr (C::k8) {
        float x[RP], top = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < RP / 2; ++i) {
          const float2 f = Pair<T>::unpack(w[i]);
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
        for (int i = 0; i < RP; ++i) x[i] *= up;
#pragma unroll
        for (int p = 0; p < C::PQ; ++p) {
          const int n = p * RP + r;
          uint8_t* dst = sQ + n * 128 + (((d0 >> 4) ^ (n & 7)) << 4) + (d0 & 15);
#pragma unroll
          for (int i = 0; i < RP / 4; ++i) {
            const uint16_t e0 = f32x2_to_fp8x2<kCacheE4M3>(x[4 * i], x[4 * i + 1]);
            const uint16_t e1 = f32x2_to_fp8x2<kCacheE4M3>(x[4 * i + 2], x[4 * i + 3]);
            const float2 f0 = Pair<__half>::unpack(fp8x2_to_f16x2<kCacheE4M3>(e0));
            const float2 f1 = Pair<__half>::unpack(fp8x2_to_f16x2<kCacheE4M3>(e1));
            x[4 * i] -= f0.x;
            x[4 * i + 1] -= f0.y;
            x[4 * i + 2] -= f1.x;
            x[4 * i + 3] -= f1.y;
            *reinterpret_cast<uint32_t*>(dst + i * 4) = e0 | ((uint32_t)e1 << 16);
          }
        }
        // the columns behind the pieces
        for (int i = tid; i < (C::NS - C::PQ * RP) * 8; i += 128)
          *reinterpret_cast<uint4*>(sQ + C::PQ * RP * 128 + i * 16) = make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < RP / 4; ++i) {
          const int d = d0 + i * 4;
          *reinterpret_cast<uint2*>(sQ + (d >> 6) * (C::NS * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 7) * 2) =
              make_uint2(w[2 * i], w[2 * i + 1]);
        }
        // the columns behind the pieces, of Q (both halves of the dims) and of P (both buffers, both halves of the keys)
        for (int i = tid; i < (C::NS - RP) * 8; i += 128)
          for (int hf = 0; hf < 2; ++hf)
            *reinterpret_cast<uint4*>(sQ + hf * (C::NS * 128) + RP * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < (C::NP - C::PP * RP) * 8; i += 128)
          for (int part = 0; part < 4; ++part)
            *reinterpret_cast<uint4*>(sP + part * (C::NP * 128) + C::PP * RP * 128 + i * 16) = make_uint4(0, 0, 0, 0);
      }
      // every thread needs every row's power: through the reduction scratch
      if (tid % TPR == 0) sRed[r] = down;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
      softmax_sync();
      const float ksc = cache_scale(c.k_scale, c.ks_batch, c.ks_head, b, hk) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < RP; ++i) pre[i] = sRed[i] * ksc;
    }
    const RowMask first = row_mask(c, s.k_len, shift), last = row_mask(c, s.k_len, t_last + shift);
    float m_ref[RP], l_run[RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      m_ref[r] = -INFINITY;
      l_run[r] = 0.f;
    }
    // A wait that gave up does not end the loop: the barriers below need every warp.
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      ok = ok && wwait(&s_full[t & 1], (t >> 1) & 1);
      tc_fence_after();
      float x[RP];
      {
        uint32_t col[C::NS];
#pragma unroll
        for (int q = 0; q < C::NS / 16; ++q)
          tmem_ld16(tmem_base + lane_addr + (t & 1) * C::SCOL + q * 16, *reinterpret_cast<uint32_t(*)[16]>(&col[q * 16]));
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t & 1]);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float v = __uint_as_float(col[r]);
#pragma unroll
          for (int p = 1; p < C::PQ; ++p) v += __uint_as_float(col[p * RP + r]);
          x[r] = v * pre[r];
        }
      }
      const int j0 = span.tile(i_begin + t) * BN;
      const int n_v = 2 * t + 1, v_slot = n_v % C::SLOTS;
      if (j0 + BN > first.hi || (j0 < last.lo && j0 + BN > c.sinks)) {
        const int col = j0 + tid;
        int tok = 0, in = 0;
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          if (row_mask(c, s.k_len, tok + shift).dead(col)) x[r] = -INFINITY;
          if (++in == group) {
            in = 0;
            ++tok;
          }
        }
        // a V row that no query row sees must not reach the product
        ok = ok && wwait(&full[v_slot], (n_v / C::SLOTS) & 1);
        if (ok && (col >= last.hi || (col < first.lo && col >= c.sinks))) {
          uint8_t* v = smem + v_slot * C::TILE + tid * 128;
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0, 0, 0, 0);
          if constexpr (!C::k8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + C::TILE / 2 + i * 16) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      bool raise = false;
#pragma unroll
      for (int r = 0; r < RP; ++r) raise = raise || x[r] > m_ref[r] + kRaise;
      if (softmax_any(raise)) {
        // exact maxima of the tile, shared by the four warps
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float m = warp_max(x[r]);
          if (lane == 0) sRed[warp * 16 + r] = m;
        }
        softmax_sync();
        float f[RP];
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float m = fmaxf(fmaxf(fmaxf(sRed[r], sRed[16 + r]), fmaxf(sRed[32 + r], sRed[48 + r])), m_ref[r]);
          f[r] = m == -INFINITY ? 1.f : ex2(m_ref[r] - m);
          m_ref[r] = m;
          l_run[r] *= f[r];
        }
        if (t > 0) {
          ok = ok && wwait(&o_done[(t - 1) & 1], ((t - 1) >> 1) & 1);   // every product so far has landed
          tc_fence_after();
#pragma unroll
          for (int q = 0; q < C::NP / 16; ++q) {
            uint32_t o[16];
            tmem_ld16(tmem_base + lane_addr + C::OCOL + q * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (q * 16 + e < C::PP * RP) o[e] = __float_as_uint(__uint_as_float(o[e]) * f[(q * 16 + e) % RP]);
            tmem_st16(tmem_base + lane_addr + C::OCOL + q * 16, o);
          }
          tmem_st_wait();
          tc_fence_before();
        }
      }
      if (t >= 2) ok = ok && wwait(&o_done[t & 1], ((t - 2) >> 1) & 1);   // the P buffer has been read
      uint8_t* buf = sP + (t & 1) * C::PB;
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
            h = *reinterpret_cast<const uint32_t*>(&d);
            const int n = p * RP + r;
            buf[n * 128 + ((ch ^ (n & 7)) << 4) + at] = (uint8_t)(e & 0xff);
            buf[(n + 1) * 128 + ((ch ^ ((n + 1) & 7)) << 4) + at] = (uint8_t)(e >> 8);
          }
        } else {
          const int at = (tid & 7) * 2, ch = (tid & 63) >> 3;
          uint8_t* half = buf + (tid >> 6) * (C::NP * 128);
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
      if (lane == 0) mbar_arrive(&p_ready[t & 1]);
    }

    // ---- sums over the keys (threads), then one output dim a thread
    softmax_sync();          // the scratch of the maxima has been read
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const float l = warp_sum(l_run[r]);
      if (lane == 0) sRed[warp * 16 + r] = l;
    }
    softmax_sync();
    ok = ok && wwait(&o_done[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1);
    tc_fence_after();
    if (ok) {
      uint32_t o[C::NP];
#pragma unroll
      for (int q = 0; q < C::NP / 16; ++q)
        tmem_ld16(tmem_base + lane_addr + C::OCOL + q * 16, *reinterpret_cast<uint32_t(*)[16]>(&o[q * 16]));
      tmem_ld_wait();
      const float vsc = cache_scale(c.v_scale, c.vs_batch, c.vs_head, b, hk);
      int tok = 0, in = 0;
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        if (r < rows) {
          float v = __uint_as_float(o[r]);
#pragma unroll
          for (int p = 1; p < C::PP; ++p) v += __uint_as_float(o[p * RP + r]);
          const float l = (sRed[r] + sRed[16 + r]) + (sRed[32 + r] + sRed[48 + r]);
          // a NaN sum stays one: only a row that saw nothing is set to zero
          v = l == 0.f ? 0.f : v * (C::k8 ? 1.f / kPScale : 1.f) * (vsc / l);
          const int64_t qtok = q0 + tok;
          const int h = hk * group + in;
          if (a.num_splits > 1)
            a.ws_o[(((int64_t)split * a.total_q + qtok) * a.H + h) * HD + tid] = v;
          else
            reinterpret_cast<T*>(a.out)[qtok * a.o_rs + (int64_t)h * a.o_hs + tid] = Cvt<T>::from_f32(v);
          if (tid == 0) {
            const float lse2 = l == 0.f ? -INFINITY : m_ref[r] + log2f(l);
            if (a.num_splits > 1)
              a.ws_lse[((int64_t)split * a.H + h) * a.total_q + qtok] = lse2;
            else if (a.lse)
              a.lse[(int64_t)h * a.total_q + qtok] = l == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
          }
        }
        if (++in == group) {
          in = 0;
          ++tok;
        }
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
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TCOLS);
  }
}

template <typename T, int KIND, int RP>
int launch(DecodeArgs& da, cudaStream_t st) {
  using C = Cfg<T, KIND, RP>;
  static_assert(!C::k8 && RP == 16 ? C::SMEM <= 232448 : 2 * (C::SMEM + 1024) <= 233472, "CTAs an SM");
  const AttnArgs& a = da.c.a;
  constexpr int ES = C::k8 ? 1 : 2;
  da.page_rows = a.paged && a.block_size < BN ? a.block_size : BN;
  da.pages_per_tile = BN / da.page_rows;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const uint64_t hs = (uint64_t)(i ? a.v_hs : a.k_hs) * ES, rs = (uint64_t)(i ? a.v_rs : a.k_rs) * ES;
    const uint64_t bs = (uint64_t)(i ? a.v_bs : a.k_bs) * ES;
    const uint64_t rows = a.paged ? (uint64_t)a.block_size : (uint64_t)(a.total_k > 0 ? a.total_k : 1);
    const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)a.Hk, rows, a.paged ? (uint64_t)a.num_blocks : 1};
    const uint64_t strides[3] = {hs, rs, a.paged ? bs : rs * rows};
    const uint32_t box[4] = {(uint32_t)(128 / ES), 1, (uint32_t)da.page_rows, 1};
    const int rc = ES == 2 ? encode_tmap_16bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box)
                           : encode_tmap_8bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_decode_tcgen05_kernel<T, KIND, RP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::SMEM));
    attr_dev = dev;
  }
  dim3 grid(a.num_splits, a.Hk, a.batch);
  attn_cache_decode_tcgen05_kernel<T, KIND, RP><<<grid, NUM_THREADS, C::SMEM, st>>>(maps[0], maps[1], da);
  FG_CHECK_LAUNCH("attn_cache_decode_tcgen05_kernel");
  return FG_OK;
}

template <typename T, int KIND>
int launch_rows(DecodeArgs& da, cudaStream_t st) {
  const int rows = da.c.a.max_q * da.c.a.group;
  if (rows <= 4) return launch<T, KIND, 4>(da, st);
  if (rows <= 8) return launch<T, KIND, 8>(da, st);
  return launch<T, KIND, 16>(da, st);
}

template <typename T>
int launch_kind(DecodeArgs& da, int kind, cudaStream_t st) {
  if (kind == kCacheE4M3) return launch_rows<T, kCacheE4M3>(da, st);
  if (kind == kCacheE5M2) return launch_rows<T, kCacheE5M2>(da, st);
  return launch_rows<T, kCache16>(da, st);
}

}  // namespace

int attn_cache_decode_sm100(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  DecodeArgs da;
  da.c = c;
  if (!c.a.status) return fail(FG_ERR_CUDA, "flash_attn_cache: device status word unavailable");
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(da, kind, st) : launch_kind<__half>(da, kind, st);
}

}  // namespace fg
