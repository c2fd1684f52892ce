// Attention of a few query rows (at most 16 (token, head of the group) pairs of a sequence) over an 8-bit or windowed
// cache: single-token decode, and a few tokens at a time.  Every cached byte is read once.  For few keys in all, where many small
// CTAs hide the way through a tile better than the tcgen05 form's runs, and for what that form does not take (soft-capping, 16-bit
// head dim 256, other head dims); attn_cache_api.cu has the rule and both sides' times.  Long contexts it moves at about
// 2.5 TB/s (8-bit head dim 128), bound by the widening.
//
// CTA = (range of K/V tiles, KV head, sequence), 5 warps:
//   warp 0     producer: walks the tile runs (first tokens, then the window), looks the pages of each tile up and
//              issues one TMA box per page and 128-byte column block into a swizzled shared-memory ring
//   warps 1-4  consumers: each owns a quarter of every tile's keys; S = Q K^T and O += P V with mma.sync over the 16
//              rows, a private online softmax per warp, merged through shared memory at the end
// A tile is 32 KB at head dim 128 in both forms: 64 keys of 16 bits, 128 keys of 8 bits.  8-bit K/V are widened to fp16 in
// registers, between ldmatrix and the product: a 16-byte row piece lands as four consecutive values per thread, so
// the product's k positions (2t, 2t+1, 2t+8, 2t+9) are given the head-dim columns 4t .. 4t+3, for Q alike; for V,
// ldmatrix.trans moves pairs of columns, which a byte permutation parts into the two products of even and odd columns.
#include "attn_cache_common.cuh"
#include "mma_helpers.cuh"
#include "sm100_common.cuh"

namespace fg {
namespace {

constexpr int NUM_THREADS = 160;

template <int KIND, int DP>
struct Tile {
  static constexpr int BN = KIND == kCache16 ? 64 : 128;              // keys
  static constexpr int KPW = BN / 4;                                  // keys of a consumer warp
  static constexpr int ROW = DP * (KIND == kCache16 ? 2 : 1);         // bytes of a row
  static constexpr int PITCH = ROW < 128 ? ROW : 128;                 // bytes of a row in one column block
  static constexpr int BLOCKS = ROW / PITCH;                          // column blocks
  static constexpr int HALF = BN * PITCH;                             // bytes of one column block
  static constexpr int KV = BLOCKS * HALF;                            // one K (or V) tile
  static constexpr int STAGES = KV <= 8192 ? 6 : 3;
  static constexpr int MERGE = (4 * 16 * DP + 2 * 4 * 16) * 4;
  static constexpr int RING = STAGES * 2 * KV > MERGE ? STAGES * 2 * KV : MERGE;
  static constexpr int SMEM = RING + 1024 + 128;
  // byte of 16-byte piece `ch` (over the whole row) of row `r`: TMA's 128-byte or 64-byte swizzle
  static __device__ __forceinline__ int at(int r, int ch) {
    if constexpr (PITCH == 128) return (ch >> 3) * HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
    return r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
  }
};

struct DecodeArgs {
  CacheAttnArgs c;
  int page_rows;       // keys per TMA box
  int pages_per_tile;
};

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, int KIND, int DP>
__global__ void __launch_bounds__(NUM_THREADS, DP <= 128 ? 2 : 1)   // two CTAs an SM: at most 200 registers
attn_cache_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                         const __grid_constant__ DecodeArgs da) {
  using namespace sm100;
  using L = Tile<KIND, DP>;
  using M = typename std::conditional<KIND == kCache16, T, __half>::type;   // type of the products
  constexpr int BN = L::BN, KPW = L::KPW, STAGES = L::STAGES;
  constexpr float kShift = p_shift<M>(0.f);
  const CacheAttnArgs& c = da.c;
  const AttnArgs& a = c.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::RING);
  uint64_t* empty = full + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);

  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const SeqInfo s = cache_seq_info(c, b);
  const int q_first = a.num_splits > 1 ? a.cu_q[0] : 0;
  const int group = a.group;
  const int rows = min(s.q_len * group, 16);
  if (rows < 1) return;
  // drain after a timed-out wait on this device (one thread reads: CTA-uniform decision)
  __shared__ int s_drain;
  if (threadIdx.x == 0) s_drain = *reinterpret_cast<volatile int*>(a.status);
  __syncthreads();
  if (s_drain != 0) return;
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
      if (a.num_splits > 1) {
        const int64_t at = part_row(c, q_first, qtok);
        if (at >= 0) a.ws_lse[((int64_t)split * a.H + h) * c.part_rows + at] = -INFINITY;
      } else if (a.lse) {
        a.lse[(int64_t)h * a.total_q + qtok] = INFINITY;
      }
    }
    if (a.num_splits == 1)
      for (int i = tid; i < rows * a.D; i += NUM_THREADS) {
        const int r = i / a.D;
        reinterpret_cast<T*>(a.out)[(q0 + r / group) * a.o_rs + (int64_t)(hk * group + r % group) * a.o_hs + i - r * a.D] =
            Cvt<T>::from_f32(0.f);
      }
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  __syncthreads();

  // lane 0 polls for its warp, so that a wait that gave up takes the whole warp the same way
  auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool {
    int r = 1;
    if (lane == 0) r = mbar_wait(bar, parity, abort_flag, a.status, kStatusAttnTimeout) ? 1 : 0;
    r = __shfl_sync(0xffffffffu, r, 0);
    __syncwarp();   // what lane 0 has seen arrive is there for the others
    return r != 0;
  };

  if (warp == 0) {
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
    for (int t = 0; t < n_tiles; ++t) {
      const int stg = t % STAGES;
      const uint32_t ph = (uint32_t)((t / STAGES) & 1);
      int npage, nrow;
      lookup(t + 1, npage, nrow);  // the table entry of the next tile is in flight while this one is issued
      if (!wwait(&empty[stg], ph ^ 1)) break;
      if (lane == 0) mbar_expect_tx(&full[stg], 2 * L::KV);
      __syncwarp();
      if (lane < da.pages_per_tile) {
        uint8_t* kdst = smem + stg * 2 * L::KV + lane * da.page_rows * L::PITCH;
        constexpr int COLS = L::PITCH / (KIND == kCache16 ? 2 : 1);
#pragma unroll
        for (int blk = 0; blk < L::BLOCKS; ++blk) {
          tma_load_4d(kdst + blk * L::HALF, &tmap_k, &full[stg], blk * COLS, hk, row, page);
          tma_load_4d(kdst + L::KV + blk * L::HALF, &tmap_v, &full[stg], blk * COLS, hk, row, page);
        }
      }
      page = npage;
      row = nrow;
    }
  } else {
    // ================================ consumers ===================================
    const int w = warp - 1;
    const int g = lane >> 2, tq = lane & 3;
    // Q as A fragments, straight from global memory (rows >= `rows` and columns >= D are zero)
    uint32_t qf[DP / 16][4];
    float pre[2];            // takes the accumulator to the scores
    RowMask mask[2];
    {
      const T* Q[2];
      bool live[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + r * 8;
        live[r] = row < rows;
        const int tok = live[r] ? row / group : 0;
        Q[r] = reinterpret_cast<const T*>(a.q) + (q0 + tok) * a.q_rs +
               (int64_t)(hk * group + (live[r] ? row - tok * group : 0)) * a.q_hs;
        mask[r] = row_mask(c, s.k_len, tok + shift);
      }
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = kk * 16 + (KIND == kCache16 ? tq * 2 + (i >> 1) * 8 : tq * 4 + (i >> 1) * 2);
          qf[kk][i] = (live[i & 1] && col < a.D) ? *reinterpret_cast<const uint32_t*>(Q[i & 1] + col) : 0u;
        }
      }
      float down[2] = {1.f, 1.f};
      if constexpr (!std::is_same<T, M>::value) {   // bf16 queries: scaled by a power of two for each row
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Pair<T>::unpack(qf[kk][i]);
            top[i & 1] = fmaxf(top[i & 1], fmaxf(fabsf(f.x), fabsf(f.y)));   // NaN entries stay NaN whatever the power
          }
        float up[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          row_power(top[r], up[r], down[r]);
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Pair<T>::unpack(qf[kk][i]);
            qf[kk][i] = Pair<__half>::pack(f.x * up[i & 1], f.y * up[i & 1]);
          }
      }
      const float ksc = cache_scale(c.k_scale, c.ks_batch, c.ks_head, b, hk);
#pragma unroll
      for (int r = 0; r < 2; ++r) pre[r] = ksc * down[r] * (a.has_softcap ? a.softcap_pre : a.scale_log2);
    }
    const RowMask first = row_mask(c, s.k_len, shift), last = row_mask(c, s.k_len, t_last + shift);
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY};
    float l_run[2] = {0.f, 0.f};
    bool ok = true;

    for (int t = 0; t < n_tiles; ++t) {
      const int stg = t % STAGES;
      const uint32_t ph = (uint32_t)((t / STAGES) & 1);
      if (!wwait(&full[stg], ph)) {
        ok = false;
        break;
      }
      const uint8_t* sK = smem + stg * 2 * L::KV;
      uint8_t* sV = smem + stg * 2 * L::KV + L::KV;
      const int j0 = span.tile(i_begin + t) * BN + w * KPW;   // first key of this warp

      float sacc[KPW / 8][4];
#pragma unroll
      for (int i = 0; i < KPW / 8; ++i) sacc[i][0] = sacc[i][1] = sacc[i][2] = sacc[i][3] = 0.f;
      if constexpr (KIND == kCache16) {
        const int r = w * KPW + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          uint32_t bf[4];
          ldmatrix_x4(bf, sK + L::at(r, kk * 2 + ((lane >> 3) & 1)));
          mma16816<M>(sacc[0], qf[kk], bf[0], bf[1]);
          mma16816<M>(sacc[1], qf[kk], bf[2], bf[3]);
        }
      } else {
#pragma unroll
        for (int cg = 0; cg < DP / 64; ++cg) {
#pragma unroll
          for (int ng = 0; ng < KPW / 8; ++ng) {
            uint32_t raw[4];
            ldmatrix_x4(raw, sK + L::at(w * KPW + ng * 8 + (lane & 7), cg * 4 + (lane >> 3)));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b0, b1;
              fp8x4_to_f16x4<KIND>(raw[i], b0, b1);
              mma16816<M>(sacc[ng], qf[cg * 4 + i], b0, b1);
            }
          }
        }
      }
      // some row does not see all of this warp's keys; V rows that no row sees must not reach the products
      const bool need_mask = j0 + KPW > first.hi || (j0 < last.lo && j0 + KPW > c.sinks);
      float mx[2] = {m_run[0], m_run[1]};
#pragma unroll
      for (int nt = 0; nt < KPW / 8; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sacc[nt][e] * pre[e >> 1];
          if (a.has_softcap) v = tanhf(v) * a.scale_log2;
          if (need_mask && mask[e >> 1].dead(j0 + nt * 8 + tq * 2 + (e & 1))) v = -INFINITY;
          sacc[nt][e] = v;
          mx[e >> 1] = fmaxf(mx[e >> 1], v);
        }
      }
      if (need_mask) {
        for (int idx = lane; idx < KPW * L::BLOCKS * (L::PITCH / 16); idx += 32) {
          const int ch = idx % (L::BLOCKS * (L::PITCH / 16)), r = idx / (L::BLOCKS * (L::PITCH / 16));
          const int col = j0 + r;
          if (col >= last.hi || (col < first.lo && col >= c.sinks))
            *reinterpret_cast<uint4*>(sV + L::at(w * KPW + r, ch)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();   // the next copy into this stage comes after these writes
        __syncwarp();
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      float corr[2], mp[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float msafe = mx[r] == -INFINITY ? 0.f : mx[r];
        corr[r] = ex2(m_run[r] - msafe);
        mp[r] = msafe - kShift;
        m_run[r] = mx[r];
        l_run[r] *= corr[r];
      }
      if (corr[0] != 1.f || corr[1] != 1.f) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= corr[0];
          o[i][1] *= corr[0];
          o[i][2] *= corr[1];
          o[i][3] *= corr[1];
        }
      }
      uint32_t pf[KPW / 16][4];
#pragma unroll
      for (int nt = 0; nt < KPW / 8; ++nt) {
        const float p0 = ex2(sacc[nt][0] - mp[0]), p1 = ex2(sacc[nt][1] - mp[0]);
        const float p2 = ex2(sacc[nt][2] - mp[1]), p3 = ex2(sacc[nt][3] - mp[1]);
        l_run[0] += p0 + p1;
        l_run[1] += p2 + p3;
        pf[nt >> 1][(nt & 1) * 2 + 0] = pack_pair<M>(p0, p1);
        pf[nt >> 1][(nt & 1) * 2 + 1] = pack_pair<M>(p2, p3);
      }
      const int v_row = w * KPW + (lane & 7) + ((lane >> 3) & 1) * 8;
      if constexpr (KIND == kCache16) {
#pragma unroll
        for (int dp = 0; dp < DP / 16; ++dp) {
          uint32_t bf[4];
          ldmatrix_x4_trans(bf, sV + L::at(v_row, dp * 2 + (lane >> 4)));
          mma16816<M>(o[dp * 2], pf[0], bf[0], bf[1]);
          mma16816<M>(o[dp * 2 + 1], pf[0], bf[2], bf[3]);
        }
      } else {
#pragma unroll
        for (int kg = 0; kg < KPW / 16; ++kg) {
#pragma unroll
          for (int dc = 0; dc < DP / 32; ++dc) {
            uint32_t raw[4];   // keys 0-7 and 8-15 of two 16-byte pieces
            ldmatrix_x4_trans(raw, sV + L::at(v_row + kg * 16, dc * 2 + (lane >> 4)));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t e0, o0, e1, o1;   // even and odd columns of the first and second eight keys
              fp8x4_to_f16x4<KIND>(__byte_perm(raw[i * 2], 0, 0x3120), e0, o0);
              fp8x4_to_f16x4<KIND>(__byte_perm(raw[i * 2 + 1], 0, 0x3120), e1, o1);
              mma16816<M>(o[dc * 4 + i * 2], pf[kg], e0, e1);
              mma16816<M>(o[dc * 4 + i * 2 + 1], pf[kg], o0, o1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stg]);  // this warp is done with the stage
    }

    // ---- merge the 4 consumer warps (the ring is idle: every tile has been consumed) ----
    consumer_sync();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
    }
    float* sO = reinterpret_cast<float*>(smem);  // [4 warps][16 rows][DP]
    float* sM = sO + 4 * 16 * DP;                // [4][16]
    float* sL = sM + 4 * 16;                     // [4][16]
    if (ok) {
      if (tq == 0) {
        sM[w * 16 + g] = m_run[0];
        sM[w * 16 + g + 8] = m_run[1];
        sL[w * 16 + g] = l_run[0];
        sL[w * 16 + g + 8] = l_run[1];
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (g + r * 8 >= rows) continue;
        float* dst = sO + (w * 16 + g + r * 8) * DP;
        if constexpr (KIND == kCache16) {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i)
            *reinterpret_cast<float2*>(dst + i * 8 + tq * 2) = make_float2(o[i][r * 2], o[i][r * 2 + 1]);
        } else {
#pragma unroll
          for (int i = 0; i < DP / 16; ++i)
            *reinterpret_cast<float4*>(dst + i * 16 + tq * 4) =
                make_float4(o[2 * i][r * 2], o[2 * i + 1][r * 2], o[2 * i][r * 2 + 1], o[2 * i + 1][r * 2 + 1]);
        }
      }
    }
    consumer_sync();
    if (ok && !*abort_flag) {
      const float vsc = cache_scale(c.v_scale, c.vs_batch, c.vs_head, b, hk);
      for (int idx = tid - 32; idx < rows * (DP / 2); idx += 128) {
        const int r = idx / (DP / 2), d = (idx - r * (DP / 2)) * 2;
        float m = -INFINITY;
#pragma unroll
        for (int ww = 0; ww < 4; ++ww) m = fmaxf(m, sM[ww * 16 + r]);
        const float ms = m == -INFINITY ? 0.f : m;
        float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int ww = 0; ww < 4; ++ww) {
          const float sc = ex2(sM[ww * 16 + r] - ms);
          const float2 v = *reinterpret_cast<const float2*>(sO + (ww * 16 + r) * DP + d);
          l += sL[ww * 16 + r] * sc;
          x += v.x * sc;
          y += v.y * sc;
        }
        const float inv = l == 0.f ? 0.f : vsc / l;   // a NaN sum stays one
        const int64_t qtok = q0 + r / group;
        const int h = hk * group + r % group;
        const int64_t at = a.num_splits > 1 ? part_row(c, q_first, qtok) : 0;
        if (at < 0) continue;
        if (d < a.D) {
          if (a.num_splits > 1)
            *reinterpret_cast<float2*>(a.ws_o + (((int64_t)split * c.part_rows + at) * a.H + h) * a.D + d) =
                make_float2(x * inv, y * inv);
          else
            *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + qtok * a.o_rs + (int64_t)h * a.o_hs + d) =
                pack_pair<T>(x * inv, y * inv);
        }
        if (d == 0) {
          const float lse2 = l == 0.f ? -INFINITY : m - kShift + log2f(l);
          if (a.num_splits > 1)
            a.ws_lse[((int64_t)split * a.H + h) * c.part_rows + at] = lse2;
          else if (a.lse)
            a.lse[(int64_t)h * a.total_q + qtok] = l == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
        }
      }
    }
  }
  if (*abort_flag) {   // a wait gave up: leave the copies in flight time to land before the shared memory is given away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

template <typename T, int KIND, int DP>
int launch(DecodeArgs& da, cudaStream_t st) {
  using L = Tile<KIND, DP>;
  const AttnArgs& a = da.c.a;
  constexpr int ES = KIND == kCache16 ? 2 : 1;
  da.page_rows = a.paged && a.block_size < L::BN ? a.block_size : L::BN;
  da.pages_per_tile = L::BN / da.page_rows;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const uint64_t hs = (uint64_t)(i ? a.v_hs : a.k_hs) * ES, rs = (uint64_t)(i ? a.v_rs : a.k_rs) * ES;
    const uint64_t bs = (uint64_t)(i ? a.v_bs : a.k_bs) * ES;
    const uint64_t rows = a.paged ? (uint64_t)a.block_size : (uint64_t)(a.total_k > 0 ? a.total_k : 1);
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)a.Hk, rows, a.paged ? (uint64_t)a.num_blocks : 1};
    const uint64_t strides[3] = {hs, rs, a.paged ? bs : rs * rows};
    const uint32_t box[4] = {(uint32_t)(L::PITCH / ES), 1, (uint32_t)da.page_rows, 1};
    const int rc = ES == 2 ? encode_tmap_16bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box)
                           : encode_tmap_8bit(&maps[i], i ? a.v : a.k, 4, dims, strides, box);
    if (rc != FG_OK) return rc;
  }
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_decode_kernel<T, KIND, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
    attr_dev = dev;
  }
  dim3 grid(a.num_splits, a.Hk, a.batch);
  attn_cache_decode_kernel<T, KIND, DP><<<grid, NUM_THREADS, L::SMEM, st>>>(maps[0], maps[1], da);
  FG_CHECK_LAUNCH("attn_cache_decode_kernel");
  return FG_OK;
}

template <typename T, int KIND>
int launch_dim(DecodeArgs& da, cudaStream_t st) {
  if (da.c.a.D <= 64) return launch<T, KIND, 64>(da, st);
  if (da.c.a.D <= 128) return launch<T, KIND, 128>(da, st);
  return launch<T, KIND, 256>(da, st);
}

template <typename T>
int launch_kind(DecodeArgs& da, int kind, cudaStream_t st) {
  if (kind == kCacheE4M3) return launch_dim<T, kCacheE4M3>(da, st);
  if (kind == kCacheE5M2) return launch_dim<T, kCacheE5M2>(da, st);
  return launch_dim<T, kCache16>(da, st);
}

}  // namespace

int attn_cache_decode(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  DecodeArgs da;
  da.c = c;
  if (!c.a.status) return fail(FG_ERR_CUDA, "flash_attn_cache: device status word unavailable");
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(da, kind, st) : launch_kind<__half>(da, kind, st);
}

}  // namespace fg
