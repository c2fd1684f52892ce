// Attention over an 8-bit or windowed cache, general form: any head dim <= 256 (multiple of 8), paged with any block
// size or contiguous, causal / window / first-token masks, soft-capping.  Warp-level mma.sync with fp32 accumulation.
//
// One CTA = 64 rows ((token, head of the group) pairs) of one (sequence, KV head) and a range of its K/V tiles of 64
// keys, 4 warps x 16 rows.  The raw K/V rows arrive through a two-stage cp.async ring; 8-bit rows are widened into a
// second, single-buffered pair of tiles.  The tensor-core kernels take what they cover (attn_cache_api.cu); this one
// covers the rest.
#include "attn_cache_common.cuh"
#include "mma_helpers.cuh"

namespace fg {
namespace {

constexpr int BM = 64, BN = 64, NTHREADS = 128;

__device__ __forceinline__ void cp_async8(void* smem_dst, const void* gsrc, bool valid) {
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(smem_dst));
  const int sz = valid ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(gsrc), "r"(sz) : "memory");
}

template <typename T, int KIND, int DP>
struct Layout {
  using M = typename std::conditional<KIND == kCache16, T, __half>::type;   // type of the products
  static constexpr int LD = DP + 8;                      // row pitch of the 16-bit tiles (elements)
  static constexpr int RAW = KIND == kCache16 ? LD * 2 : DP + 16;   // row pitch of the ring (bytes)
  static constexpr int STAGE = 2 * BN * RAW;             // K rows, then V rows
  static constexpr int WIDE = KIND == kCache16 ? 0 : 2 * BN * LD * 2;
  static constexpr int SMEM = BM * LD * 2 + 2 * STAGE + WIDE + BM * 4;
};

template <typename T, int KIND, int DP>
__global__ void __launch_bounds__(NTHREADS) attn_cache_generic_kernel(CacheAttnArgs c) {
  using L = Layout<T, KIND, DP>;
  using M = typename L::M;
  constexpr int LD = L::LD;
  constexpr int ES = KIND == kCache16 ? 2 : 1;           // bytes of a cached element
  const AttnArgs& a = c.a;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  M* sQ = reinterpret_cast<M*>(smem_raw);
  uint8_t* ring = smem_raw + BM * LD * 2;
  M* wide = reinterpret_cast<M*>(ring + 2 * L::STAGE);
  float* sDown = reinterpret_cast<float*>(ring + 2 * L::STAGE + L::WIDE);

  const int num_mb = gridDim.x / a.num_splits;
  const int m_block = num_mb - 1 - blockIdx.x / a.num_splits;  // long (late) causal rows first
  const int split = blockIdx.x % a.num_splits;
  const int hk = blockIdx.y, b = blockIdx.z;
  const SeqInfo s = cache_seq_info(c, b);
  const int q_first = a.num_splits > 1 ? a.cu_q[0] : 0;
  const int rows = s.q_len * a.group;
  const int r0 = m_block * BM;
  if (r0 >= rows) return;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int shift = s.k_len - s.q_len;
  const int t_first = r0 / a.group, t_last = min(s.q_len - 1, (r0 + BM - 1) / a.group);
  const TileSpan span = tile_span<BN>(c, s.k_len, t_first + shift, t_last + shift);
  const int i_begin = split * c.tiles_per_split;
  const int i_end = a.num_splits > 1 ? min(span.n, i_begin + c.tiles_per_split) : span.n;

  const uint8_t* K = reinterpret_cast<const uint8_t*>(a.k) + (int64_t)hk * a.k_hs * ES;
  const uint8_t* V = reinterpret_cast<const uint8_t*>(a.v) + (int64_t)hk * a.v_hs * ES;
  const int32_t* bt_row = a.paged ? a.block_table + (int64_t)b * a.bt_stride : nullptr;
  const int lrow = tid >> 1, lpart = tid & 1;  // loader mapping: 2 threads per tile row

  auto load_kv = [&](int i, int stage) {
    const int tok = span.tile(i) * BN + lrow;
    const bool ok = tok < s.k_len;
    int64_t koff = 0, voff = 0;
    if (ok) {
      koff = cache_row(c, bt_row, s.k_begin, tok, a.k_rs, a.k_bs) * ES;
      voff = cache_row(c, bt_row, s.k_begin, tok, a.v_rs, a.v_bs) * ES;
    }
    uint8_t* kd = ring + stage * L::STAGE + lrow * L::RAW;
    uint8_t* vd = kd + BN * L::RAW;
    const int bytes = a.D * ES;
    if constexpr (KIND == kCache16) {
#pragma unroll
      for (int ch = lpart * (DP / 16); ch < (lpart + 1) * (DP / 16); ++ch) {
        const bool in = ok && ch * 16 < bytes;
        cp_async16(kd + ch * 16, in ? K + koff + ch * 16 : K, in);
        cp_async16(vd + ch * 16, in ? V + voff + ch * 16 : V, in);
      }
    } else {   // rows of a multiple of 8 bytes
#pragma unroll
      for (int ch = lpart * (DP / 16); ch < (lpart + 1) * (DP / 16); ++ch) {
        const bool in = ok && ch * 8 < bytes;
        cp_async8(kd + ch * 8, in ? K + koff + ch * 8 : K, in);
        cp_async8(vd + ch * 8, in ? V + voff + ch * 8 : V, in);
      }
    }
  };
  if (i_begin < i_end) load_kv(i_begin, 0);
  cp_async_commit();

  // ---- Q rows, as M; 8-bit caches with bf16 queries: scaled by a power of two for each row
  {
    const int r = r0 + lrow;
    const bool ok = r < rows;
    const int tok = ok ? r / a.group : 0;
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(s.q_begin + tok) * a.q_rs +
                 (int64_t)(hk * a.group + (ok ? r - tok * a.group : 0)) * a.q_hs;
    float up = 1.f, down = 1.f;
    if constexpr (KIND != kCache16 && std::is_same<T, __nv_bfloat16>::value) {
      float top = 0.f;
      for (int ch = lpart; ch * 8 < a.D; ch += 2) {
        if (!ok) break;
        float f[8];
        Vec16<T>::unpack(ldg16(q + ch * 8), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = fabsf(f[e]);
          top = m > top || m != m ? m : top;   // a NaN is kept
        }
      }
      const float other = __shfl_xor_sync(0xffffffffu, top, 1);
      top = other > top || other != other ? other : top;
      row_power(top, up, down);
    }
    for (int ch = lpart; ch < DP / 8; ch += 2) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (ok && ch * 8 < a.D) {
        w = ldg16(q + ch * 8);
        if constexpr (!std::is_same<T, M>::value) {
          float f[8];
          Vec16<T>::unpack(w, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= up;
          w = Vec16<M>::pack(f);
        }
      }
      *reinterpret_cast<uint4*>(sQ + lrow * LD + ch * 8) = w;
    }
    if (lpart == 0) sDown[lrow] = down;
  }

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY};
  float l_run[2] = {0.f, 0.f};
  const int row_in_tile = warp * 16 + (lane >> 2);  // + 8 for the second row
  const float ksc = cache_scale(c.k_scale, c.ks_batch, c.ks_head, b, hk);
  constexpr float kShift = p_shift<M>(0.f);
  float pre[2];                                      // takes the accumulator to the scores
  RowMask mask[2];
  __syncthreads();                                   // sDown
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row_in_tile + r * 8;
    mask[r] = row_mask(c, s.k_len, (r0 + row) / a.group + shift);
    pre[r] = ksc * sDown[row] * (a.has_softcap ? a.softcap_pre : a.scale_log2);
  }
  const RowMask block_first = row_mask(c, s.k_len, t_first + shift), block_last = row_mask(c, s.k_len, t_last + shift);

  for (int i = i_begin; i < i_end; ++i) {
    const int stage = (i - i_begin) & 1;
    if (i + 1 < i_end) load_kv(i + 1, stage ^ 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const int j0 = span.tile(i) * BN;
    // a tile that some row sees in part only; its V rows that no row sees (behind the sequence, or between the first
    // tokens and the window, where the pages may have been given away) must not reach the products
    const bool need_mask = j0 + BN > block_first.hi || (j0 < block_last.lo && j0 + BN > c.sinks);
    const M *sK, *sV;
    if constexpr (KIND == kCache16) {
      M* k = reinterpret_cast<M*>(ring + stage * L::STAGE);
      M* v = k + BN * LD;
      if (need_mask) {
        const int col = j0 + lrow;
        if (col >= block_last.hi || (col < block_first.lo && col >= c.sinks))
          for (int ch = lpart; ch < DP / 8; ch += 2) *reinterpret_cast<uint4*>(v + lrow * LD + ch * 8) = make_uint4(0, 0, 0, 0);
        __syncthreads();
      }
      sK = k;
      sV = v;
    } else {
      const int col = j0 + lrow;
      const bool zero = col >= block_last.hi || (col < block_first.lo && col >= c.sinks);
      const uint8_t* kr = ring + stage * L::STAGE + lrow * L::RAW;
      const uint8_t* vr = kr + BN * L::RAW;
#pragma unroll
      for (int ch = lpart; ch < DP / 16; ch += 2) {
        const uint4 kw = *reinterpret_cast<const uint4*>(kr + ch * 16);
        uint4 vw = *reinterpret_cast<const uint4*>(vr + ch * 16);
        if (zero) vw = make_uint4(0, 0, 0, 0);
        const uint32_t ki[4] = {kw.x, kw.y, kw.z, kw.w}, vi[4] = {vw.x, vw.y, vw.z, vw.w};
        uint32_t ko[8], vo[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fp8x4_to_f16x4<KIND>(ki[e], ko[2 * e], ko[2 * e + 1]);
          fp8x4_to_f16x4<KIND>(vi[e], vo[2 * e], vo[2 * e + 1]);
        }
        M* kd = wide + lrow * LD + ch * 16;
        M* vd = kd + BN * LD;
        *reinterpret_cast<uint4*>(kd) = make_uint4(ko[0], ko[1], ko[2], ko[3]);
        *reinterpret_cast<uint4*>(kd + 8) = make_uint4(ko[4], ko[5], ko[6], ko[7]);
        *reinterpret_cast<uint4*>(vd) = make_uint4(vo[0], vo[1], vo[2], vo[3]);
        *reinterpret_cast<uint4*>(vd + 8) = make_uint4(vo[4], vo[5], vo[6], vo[7]);
      }
      __syncthreads();
      sK = wide;
      sV = wide + BN * LD;
    }

    // ---- S = Q K^T (16 x 64 per warp)
    float sacc[BN / 8][4];
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) sacc[n][0] = sacc[n][1] = sacc[n][2] = sacc[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      uint32_t af[4];
      ldmatrix_x4(af, sQ + (warp * 16 + (lane & 15)) * LD + kk * 16 + (lane >> 4) * 8);
#pragma unroll
      for (int np = 0; np < BN / 16; ++np) {
        uint32_t bf[4];
        ldmatrix_x4(bf, sK + (np * 16 + (lane & 7) + (lane >> 4) * 8) * LD + kk * 16 + ((lane >> 3) & 1) * 8);
        mma16816<M>(sacc[np * 2], af, bf[0], bf[1]);
        mma16816<M>(sacc[np * 2 + 1], af, bf[2], bf[3]);
      }
    }
    float mx[2] = {m_run[0], m_run[1]};
#pragma unroll
    for (int nt = 0; nt < BN / 8; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = sacc[nt][e] * pre[e >> 1];
        if (a.has_softcap) v = tanhf(v) * a.scale_log2;
        if (need_mask && mask[e >> 1].dead(j0 + nt * 8 + (lane & 3) * 2 + (e & 1))) v = -INFINITY;
        sacc[nt][e] = v;
        mx[e >> 1] = fmaxf(mx[e >> 1], v);
      }
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
      corr[r] = exp2f(m_run[r] - msafe);  // m_run == -inf -> 0
      mp[r] = msafe - kShift;
      m_run[r] = mx[r];
      l_run[r] *= corr[r];
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      o[n][0] *= corr[0];
      o[n][1] *= corr[0];
      o[n][2] *= corr[1];
      o[n][3] *= corr[1];
    }
    uint32_t pf[BN / 16][4];  // P as A fragments (k = kv index)
#pragma unroll
    for (int nt = 0; nt < BN / 8; ++nt) {
      const float p0 = exp2f(sacc[nt][0] - mp[0]), p1 = exp2f(sacc[nt][1] - mp[0]);
      const float p2 = exp2f(sacc[nt][2] - mp[1]), p3 = exp2f(sacc[nt][3] - mp[1]);
      l_run[0] += p0 + p1;
      l_run[1] += p2 + p3;
      pf[nt >> 1][(nt & 1) * 2 + 0] = pack_pair<M>(p0, p1);
      pf[nt >> 1][(nt & 1) * 2 + 1] = pack_pair<M>(p2, p3);
    }
    // ---- O += P V
#pragma unroll
    for (int kk = 0; kk < BN / 16; ++kk) {
#pragma unroll
      for (int dp = 0; dp < DP / 16; ++dp) {
        uint32_t bf[4];
        ldmatrix_x4_trans(bf, sV + (kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * LD + dp * 16 + (lane >> 4) * 8);
        mma16816<M>(o[dp * 2], pf[kk], bf[0], bf[1]);
        mma16816<M>(o[dp * 2 + 1], pf[kk], bf[2], bf[3]);
      }
    }
    __syncthreads();  // everyone is done with this stage (and the wide tiles) before it is refilled
  }
  cp_async_wait<0>();

  // ---- epilogue
  const float vsc = cache_scale(c.v_scale, c.vs_batch, c.vs_head, b, hk);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
    const int row = r0 + row_in_tile + r * 8;
    if (row >= rows) continue;
    // a NaN sum stays one: only a row that saw nothing is set to zero
    const float inv = l_run[r] == 0.f ? 0.f : vsc / l_run[r];
    const int tok = row / a.group, h = hk * a.group + row - tok * a.group;
    const int64_t qtok = s.q_begin + tok;
    const float lse2 = l_run[r] == 0.f ? -INFINITY : m_run[r] - kShift + log2f(l_run[r]);
    if (a.num_splits > 1) {
      const int64_t at = part_row(c, q_first, qtok);
      if (at < 0) continue;
      float* out = a.ws_o + (((int64_t)split * c.part_rows + at) * a.H + h) * a.D;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int col = i * 8 + (lane & 3) * 2;
        if (col < a.D) *reinterpret_cast<float2*>(out + col) = make_float2(o[i][r * 2] * inv, o[i][r * 2 + 1] * inv);
      }
      if ((lane & 3) == 0) a.ws_lse[((int64_t)split * a.H + h) * c.part_rows + at] = lse2;
    } else {
      T* out = reinterpret_cast<T*>(a.out) + qtok * a.o_rs + (int64_t)h * a.o_hs;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int col = i * 8 + (lane & 3) * 2;
        if (col < a.D) *reinterpret_cast<uint32_t*>(out + col) = pack_pair<T>(o[i][r * 2] * inv, o[i][r * 2 + 1] * inv);
      }
      if (a.lse && (lane & 3) == 0)
        a.lse[(int64_t)h * a.total_q + qtok] = l_run[r] == 0.f ? INFINITY : lse2 * 0.6931471805599453f;
    }
  }
}

template <typename T, int KIND, int DP>
int launch(const CacheAttnArgs& c, cudaStream_t st) {
  constexpr int smem = Layout<T, KIND, DP>::SMEM;
  static thread_local int attr_dev = -1;
  int dev = 0;
  FG_CUDA_OK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    FG_CUDA_OK(cudaFuncSetAttribute(attn_cache_generic_kernel<T, KIND, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_dev = dev;
  }
  const AttnArgs& a = c.a;
  const int64_t mb = ((int64_t)a.max_q * a.group + BM - 1) / BM;
  dim3 grid((unsigned)(mb * a.num_splits), a.Hk, a.batch);
  attn_cache_generic_kernel<T, KIND, DP><<<grid, NTHREADS, smem, st>>>(c);
  FG_CHECK_LAUNCH("attn_cache_generic_kernel");
  return FG_OK;
}

template <typename T, int KIND>
int launch_dim(const CacheAttnArgs& c, cudaStream_t st) {
  if (c.a.D <= 64) return launch<T, KIND, 64>(c, st);
  if (c.a.D <= 128) return launch<T, KIND, 128>(c, st);
  return launch<T, KIND, 256>(c, st);
}

template <typename T>
int launch_kind(const CacheAttnArgs& c, int kind, cudaStream_t st) {
  if (kind == kCacheE4M3) return launch_dim<T, kCacheE4M3>(c, st);
  if (kind == kCacheE5M2) return launch_dim<T, kCacheE5M2>(c, st);
  return launch_dim<T, kCache16>(c, st);
}

// Joins the partial results of the splits: out = sum_s w_s O_s / sum_s w_s with w_s = 2^(lse_s - max lse).  One warp
// per (token, head); tokens outside the sequences have no partial results and stay as they were.
constexpr int kCombineWarps = 4;
template <typename T>
__global__ void __launch_bounds__(kCombineWarps * 32) attn_cache_combine_kernel(CacheAttnArgs c) {
  const AttnArgs& a = c.a;
  const int lane = threadIdx.x & 31;
  const int64_t pair = (int64_t)blockIdx.x * kCombineWarps + (threadIdx.x >> 5);  // head fastest
  const int64_t row = pair / a.H, tok = row + a.cu_q[0];
  if (row >= c.part_rows || tok < 0 || tok >= a.cu_q[a.batch] || tok >= a.total_q) return;
  const int h = (int)(pair - row * a.H);
  const float* lse = a.ws_lse + (int64_t)h * c.part_rows + row;
  const int64_t lse_step = (int64_t)a.H * c.part_rows;
  float m = -INFINITY;
  for (int s = lane; s < a.num_splits; s += 32) m = fmaxf(m, lse[s * lse_step]);
  m = warp_max(m);
  const float msafe = m == -INFINITY ? 0.f : m;
  float wsum = 0.f;
  for (int s = lane; s < a.num_splits; s += 32) wsum += exp2f(lse[s * lse_step] - msafe);
  wsum = warp_sum(wsum);
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  const float* part = a.ws_o + (row * a.H + h) * (int64_t)a.D;
  const int64_t part_step = c.part_rows * (int64_t)a.H * a.D;
  T* out = reinterpret_cast<T*>(a.out) + tok * a.o_rs + (int64_t)h * a.o_hs;
  for (int d = lane * 4; d < a.D; d += 128) {   // D is a multiple of 8, the workspace and the rows are 16-byte aligned
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.num_splits; ++s) {
      const float w = exp2f(lse[s * lse_step] - msafe);
      if (w == 0.f) continue;                   // a split without visible keys; NaN goes on
      const float4 v = *reinterpret_cast<const float4*>(part + s * part_step + d);
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
    uint2 w2;
    w2.x = Pair<T>::pack(acc.x * inv, acc.y * inv);
    w2.y = Pair<T>::pack(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out + d) = w2;
  }
  if (a.lse && lane == 0)
    a.lse[(int64_t)h * a.total_q + tok] =
        wsum == 0.f ? INFINITY : (m + log2f(wsum)) * 0.6931471805599453f;
}

}  // namespace

int attn_cache_generic(const CacheAttnArgs& c, int dtype, int kind, cudaStream_t st) {
  return dtype == FG_BF16 ? launch_kind<__nv_bfloat16>(c, kind, st) : launch_kind<__half>(c, kind, st);
}

int attn_cache_combine(const CacheAttnArgs& c, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)((c.part_rows * (int64_t)c.a.H + kCombineWarps - 1) / kCombineWarps);
  if (dtype == FG_BF16)
    attn_cache_combine_kernel<__nv_bfloat16><<<grid, kCombineWarps * 32, 0, st>>>(c);
  else
    attn_cache_combine_kernel<__half><<<grid, kCombineWarps * 32, 0, st>>>(c);
  FG_CHECK_LAUNCH("attn_cache_combine_kernel");
  return FG_OK;
}

}  // namespace fg
