// The 8-bit paged cache: quantise K/V rows as they are written, and read rows back.
//
//   write   c = RN8(RN32(x / s_h)) saturated at the largest finite value, s_h the head's scale
//   gather  y = RN(fp32(c) * s_h)
//
// Both move each byte once and compute next to nothing, so memory bounds them; the quotient is the
// one costly operation (see quotient()).
#include "fp8.cuh"

namespace fg {
namespace {

struct QuantArgs {
  const char *key, *value;
  uint8_t *kc, *vc;
  const int64_t* slots;
  const float *k_scale, *v_scale;   // null: 1
  int64_t ksh, vsh;                 // elements between the scales of two heads (0: one scale)
  int64_t T, H, D, BS, NB;
  int64_t ks, vs;                   // token strides of key / value (elements)
  int64_t cbs, crs, chs;            // cache block / row / head strides (bytes)
};

// x / s rounded to fp32, for a scale in [2^-60, 2^60] with r = RN(1 / s): the approximation x r and
// one correction with the exact remainder (Markstein, 1990), five instructions where the division
// operator takes about three times as many.  The approximation is clamped far above both types' largest value: an
// overflowing or infinite quotient then comes out as an infinity of its sign (saturated by the conversion) instead of
// inf - inf, and NaN passes through the remainder.  Quotients that differ from the division's below 2^-20 are zero in
// both types.  (The remainder is taken as q s - x: as x - q s its zero, which is +0, would turn a quotient of -0 into +0.)
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = fminf(fmaxf(x * r, -1048576.f), 1048576.f);
  return fmaf(fmaf(q, s, -x), -r, q);
}

template <typename T, int KIND>
__device__ __forceinline__ uint4 quantise16(const float (&x)[16], float s) {
  uint16_t o[8];
  if (s >= 8.6736174e-19f && s <= 1.1529215e18f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f32x2_to_fp8x2<KIND>(quotient(x[2 * i], s, r), quotient(x[2 * i + 1], s, r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f32x2_to_fp8x2<KIND>(__fdiv_rn(x[2 * i], s), __fdiv_rn(x[2 * i + 1], s));
  }
  uint4 u;
  u.x = o[0] | ((uint32_t)o[1] << 16);
  u.y = o[2] | ((uint32_t)o[3] << 16);
  u.z = o[4] | ((uint32_t)o[5] << 16);
  u.w = o[6] | ((uint32_t)o[7] << 16);
  return u;
}

// One packet = 16 elements of one head's row: sizeof(T) 16-byte loads, one 16-byte store.  32-bit
// index arithmetic (the host checks that the packets and the slots fit).
template <typename T, int KIND>
__global__ void __launch_bounds__(256) cache_quant_vec_kernel(QuantArgs a, FastDiv per_tok, FastDiv per_head, FastDiv page,
                                                              uint32_t total, uint32_t num_slots) {
  for (uint32_t idx = blockIdx.x * 256u + threadIdx.x; idx < total; idx += gridDim.x * 256u) {
    const uint32_t tk = per_tok.div(idx);  // token * 2 + which
    const uint32_t r = idx - tk * per_tok.d;
    const uint32_t tok = tk >> 1;
    const bool which = tk & 1;
    const uint32_t h = per_head.div(r);
    const uint32_t c = r - h * per_head.d;
    const T* src = reinterpret_cast<const T*>(which ? a.value : a.key) + (int64_t)tok * (which ? a.vs : a.ks) +
                   (int64_t)h * a.D + c * 16;
    // neither the payload nor the scale depends on the slot: all of them in the same round trip
    uint4 raw[sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) raw[i] = ldg16_stream(reinterpret_cast<const char*>(src) + i * 16);
    const float* sp = which ? a.v_scale : a.k_scale;
    const float s = sp ? sp[(int64_t)h * (which ? a.vsh : a.ksh)] : 1.f;
    const int64_t slot64 = a.slots[tok];
    if (slot64 < 0 || slot64 >= (int64_t)num_slots) continue;  // padding, or outside the cache
    float x[16];
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      float f[E];
      Vec16<T>::unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i * E + e] = f[e];
    }
    const uint32_t blk = page.div((uint32_t)slot64), off = (uint32_t)slot64 - blk * page.d;
    uint8_t* dst = (which ? a.vc : a.kc) + (int64_t)blk * a.cbs + (int64_t)off * a.crs + (int64_t)h * a.chs + c * 16;
    stg16(dst, quantise16<T, KIND>(x, s));
  }
}

// Any head size, stride and alignment, an element at a time.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) cache_quant_scalar_kernel(QuantArgs a) {
  const int64_t n = a.H * a.D;
  const int64_t total = a.T * n * 2;
  for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * blockDim.x) {
    const int64_t tk = idx / n;
    const int64_t i = idx - tk * n;
    const int64_t tok = tk >> 1;
    const bool which = tk & 1;
    const int64_t slot = a.slots[tok];
    if (slot < 0 || slot >= a.NB * a.BS) continue;  // padding, or outside the cache
    const int64_t h = i / a.D, d = i - h * a.D;
    const int64_t blk = slot / a.BS, off = slot - blk * a.BS;
    const float* sp = which ? a.v_scale : a.k_scale;
    const float s = sp ? sp[h * (which ? a.vsh : a.ksh)] : 1.f;
    const float x = Cvt<T>::to_f32(reinterpret_cast<const T*>(which ? a.value : a.key)[tok * (which ? a.vs : a.ks) + i]);
    const uint16_t o = f32x2_to_fp8x2<KIND>(__fdiv_rn(x, s), 0.f);
    (which ? a.vc : a.kc)[blk * a.cbs + off * a.crs + h * a.chs + d] = (uint8_t)(o & 0xff);
  }
}

template <typename T, int KIND>
int launch_quant(const QuantArgs& a, bool vec, cudaStream_t st) {
  const int64_t cap = (int64_t)num_sms() * 32;
  const int64_t total = a.T * a.H * a.D * 2;
  int64_t blocks = ((vec ? total / 16 : total) + 255) / 256;
  if (blocks > cap) blocks = cap;
  if (vec) {
    cache_quant_vec_kernel<T, KIND><<<(unsigned)blocks, 256, 0, st>>>(
        a, FastDiv((uint32_t)(a.H * (a.D / 16))), FastDiv((uint32_t)(a.D / 16)), FastDiv((uint32_t)a.BS),
        (uint32_t)(total / 16), (uint32_t)(a.NB * a.BS));
    FG_CHECK_LAUNCH("cache_quant_vec_kernel");
  } else {
    cache_quant_scalar_kernel<T, KIND><<<(unsigned)blocks, 256, 0, st>>>(a);
    FG_CHECK_LAUNCH("cache_quant_scalar_kernel");
  }
  return FG_OK;
}

struct GatherArgs {
  const uint8_t *kc, *vc;
  char *key, *value;                // [rows, H, D] with dense heads
  const int32_t *table, *cu, *starts;
  const float *k_scale, *v_scale;
  int64_t ksh, vsh;
  int64_t rows, H, D, BS, NB, B;
  int64_t table_stride, table_cols;
  int64_t ks, vs;                   // row strides of key / value (elements)
  int64_t cbs, crs, chs;            // cache block / row / head strides (elements of the cache)
};

// Offset (cache elements) of the cached row that packed row `row` holds, or -1 for a row outside the sequences
// [cu[0], cu[B]).  Pages are clamped into the table and the cache, so that a bad table entry cannot fault.
__device__ __forceinline__ int64_t gather_row(const GatherArgs& a, int64_t row) {
  if (row < a.cu[0] || row >= a.cu[a.B]) return -1;
  int64_t lo = 0, hi = a.B;         // cu[lo] <= row < cu[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (a.cu[mid] <= row) lo = mid; else hi = mid;
  }
  int64_t pos = row - a.cu[lo] + (a.starts ? a.starts[lo] : 0);
  if (pos < 0) pos = 0;
  const int64_t pg = pos / a.BS;
  int64_t page = a.table[lo * a.table_stride + (pg < a.table_cols ? pg : a.table_cols - 1)];
  page = page < 0 ? 0 : (page >= a.NB ? a.NB - 1 : page);
  return page * a.cbs + (pos - pg * a.BS) * a.crs;
}

template <typename T>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t f16x2, float s) {
  const float2 f = Pair<__half>::unpack(f16x2);
  return Pair<T>::pack(f.x * s, f.y * s);
}

constexpr int kGatherRows = 16;   // packed rows of a block

// A block looks its rows' pages up once (one thread each) and streams them: 16 elements a thread and step, four steps
// in flight.  KIND kCache16 copies 16-byte packets of a cache that holds T.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) cache_gather_vec_kernel(GatherArgs a, FastDiv per_row, FastDiv per_head) {
  __shared__ int64_t s_off[kGatherRows];
  const int64_t row0 = (int64_t)blockIdx.x * kGatherRows;
  if (threadIdx.x < kGatherRows) {
    const int64_t row = row0 + threadIdx.x;
    s_off[threadIdx.x] = row < a.rows ? gather_row(a, row) : -1;
  }
  __syncthreads();
  constexpr int EB = KIND == kCache16 ? (int)sizeof(T) : 1;   // bytes of a cached element
  constexpr int PE = 16 / EB;                                  // elements of a packet
  const uint32_t half = kGatherRows * per_row.d;               // packets of K, then as many of V
  constexpr int U = 4;
  for (uint32_t base = threadIdx.x; base < 2 * half; base += 256 * U) {
    uint4 raw[U];
    char* dst[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t idx = base + u * 256;
      dst[u] = nullptr;
      sc[u] = 1.f;
      if (idx < 2 * half) {
        const bool which = idx >= half;
        const uint32_t r = which ? idx - half : idx;
        const uint32_t rr = per_row.div(r);
        const uint32_t in = r - rr * per_row.d;
        const uint32_t h = per_head.div(in), c = in - h * per_head.d;
        const int64_t off = s_off[rr];
        if (off >= 0) {
          raw[u] = ldg16_stream((which ? a.vc : a.kc) + (off + (int64_t)h * a.chs + c * PE) * EB);
          dst[u] = (which ? a.value : a.key) +
                   ((row0 + rr) * (which ? a.vs : a.ks) + (int64_t)h * a.D + c * PE) * (int64_t)sizeof(T);
          const float* sp = which ? a.v_scale : a.k_scale;
          if (KIND != kCache16 && sp) sc[u] = sp[(int64_t)h * (which ? a.vsh : a.ksh)];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (dst[u] == nullptr) continue;
      if constexpr (KIND == kCache16) {
        stg16(dst[u], raw[u]);
      } else {
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;
            fp8x4_to_f16x4<KIND>(w[i], lo, hi);
            const float2 f = Pair<__half>::unpack(lo), g = Pair<__half>::unpack(hi);
            *reinterpret_cast<float4*>(dst[u] + i * 16) = make_float4(f.x * sc[u], f.y * sc[u], g.x * sc[u], g.y * sc[u]);
          }
        } else {
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;
            fp8x4_to_f16x4<KIND>(w[i], lo, hi);
            o[2 * i] = scaled_pair<T>(lo, sc[u]);
            o[2 * i + 1] = scaled_pair<T>(hi, sc[u]);
          }
          stg16(dst[u], make_uint4(o[0], o[1], o[2], o[3]));
          stg16(dst[u] + 16, make_uint4(o[4], o[5], o[6], o[7]));
        }
      }
    }
  }
}

// Any head size, stride and alignment, an element at a time; a block per row.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) cache_gather_scalar_kernel(GatherArgs a) {
  __shared__ int64_t s_off;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    __syncthreads();
    if (threadIdx.x == 0) s_off = gather_row(a, row);
    __syncthreads();
    const int64_t off = s_off;
    if (off < 0) continue;
    const int64_t n = a.H * a.D;
    for (int64_t i = threadIdx.x; i < 2 * n; i += 256) {
      const bool which = i >= n;
      const int64_t e = which ? i - n : i;
      const int64_t h = e / a.D, d = e - h * a.D;
      const int64_t at = off + h * a.chs + d;
      T* out = reinterpret_cast<T*>(which ? a.value : a.key) + row * (which ? a.vs : a.ks) + e;
      if constexpr (KIND == kCache16) {
        *out = reinterpret_cast<const T*>(which ? a.vc : a.kc)[at];
      } else {
        const float* sp = which ? a.v_scale : a.k_scale;
        const float s = sp ? sp[h * (which ? a.vsh : a.ksh)] : 1.f;
        const uint32_t f = fp8x2_to_f16x2<KIND>((uint16_t)(which ? a.vc : a.kc)[at]);
        *out = Cvt<T>::from_f32(Pair<__half>::unpack(f).x * s);
      }
    }
  }
}

template <typename T, int KIND>
int launch_gather(const GatherArgs& a, bool vec, cudaStream_t st) {
  if (vec) {
    constexpr int PE = KIND == kCache16 ? 16 / (int)sizeof(T) : 16;
    const int64_t blocks = (a.rows + kGatherRows - 1) / kGatherRows;
    cache_gather_vec_kernel<T, KIND><<<(unsigned)blocks, 256, 0, st>>>(a, FastDiv((uint32_t)(a.H * (a.D / PE))),
                                                                       FastDiv((uint32_t)(a.D / PE)));
    FG_CHECK_LAUNCH("cache_gather_vec_kernel");
  } else {
    const int64_t cap = (int64_t)num_sms() * 32;
    cache_gather_scalar_kernel<T, KIND><<<(unsigned)(a.rows < cap ? a.rows : cap), 256, 0, st>>>(a);
    FG_CHECK_LAUNCH("cache_gather_scalar_kernel");
  }
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int fg_reshape_and_cache_flash_fp8(const fg_cache_write_params* p, void* stream) {
  using namespace fg;
  FG_REQUIRE_HEALTHY("reshape_and_cache_flash");
  FG_REQUIRE(p != nullptr, "reshape_and_cache_flash: null params");
  FG_REQUIRE(p->num_tokens >= 0 && p->num_heads >= 0 && p->head_size >= 0, "reshape_and_cache_flash: negative size");
  FG_REQUIRE(p->block_size > 0 && p->num_blocks >= 0, "reshape_and_cache_flash: block_size must be positive");
  FG_REQUIRE(is_fp8(p->cache_dtype), "reshape_and_cache_flash: cache dtype code %d is no 8-bit type", p->cache_dtype);
  if (p->num_tokens == 0 || p->num_heads * p->head_size == 0) return FG_OK;
  FG_REQUIRE(p->key && p->value && p->key_cache && p->value_cache && p->slot_mapping,
             "reshape_and_cache_flash: null pointer");
  QuantArgs a;
  a.key = (const char*)p->key; a.value = (const char*)p->value;
  a.kc = (uint8_t*)p->key_cache; a.vc = (uint8_t*)p->value_cache;
  a.slots = p->slot_mapping; a.k_scale = p->k_scale; a.v_scale = p->v_scale;
  a.ksh = p->k_scale_stride; a.vsh = p->v_scale_stride;
  a.T = p->num_tokens; a.H = p->num_heads; a.D = p->head_size; a.BS = p->block_size; a.NB = p->num_blocks;
  a.ks = p->key_stride; a.vs = p->value_stride;
  a.cbs = p->cache_block_stride; a.crs = p->cache_row_stride; a.chs = p->cache_head_stride;
  const int es = dtype_size(p->dtype);
  const bool vec = a.D % 16 == 0 && (a.ks * es) % 16 == 0 && (a.vs * es) % 16 == 0 && a.cbs % 16 == 0 && a.crs % 16 == 0 &&
                   a.chs % 16 == 0 && aligned16(a.key) && aligned16(a.value) && aligned16(a.kc) && aligned16(a.vc) &&
                   a.T * a.H * (a.D / 16) * 2 < 4000000000LL && a.NB * a.BS < 4000000000LL;
  cudaStream_t st = (cudaStream_t)stream;
  FG_DISPATCH_FLOAT(p->dtype, T, {
    return p->cache_dtype == FG_E4M3 ? launch_quant<T, kCacheE4M3>(a, vec, st) : launch_quant<T, kCacheE5M2>(a, vec, st);
  });
  return FG_OK;
}

extern "C" int fg_gather_cache_flash(const fg_cache_gather_params* p, void* stream) {
  using namespace fg;
  FG_REQUIRE_HEALTHY("gather_cache_flash");
  FG_REQUIRE(p != nullptr, "gather_cache_flash: null params");
  FG_REQUIRE(p->num_rows >= 0 && p->batch >= 0 && p->num_heads >= 0 && p->head_size >= 0,
             "gather_cache_flash: negative size");
  FG_REQUIRE(is_fp8(p->cache_dtype) || p->cache_dtype == p->dtype,
             "gather_cache_flash: a cache that is not 8-bit must hold the type of the output");
  if (p->num_rows == 0 || p->batch == 0 || p->num_heads * p->head_size == 0) return FG_OK;
  FG_REQUIRE(p->block_size > 0 && p->num_blocks > 0, "gather_cache_flash: empty cache");
  FG_REQUIRE(p->block_table_cols > 0, "gather_cache_flash: block_table has no columns");
  FG_REQUIRE(p->key && p->value && p->key_cache && p->value_cache && p->block_table && p->cu_seqlens,
             "gather_cache_flash: null pointer");
  GatherArgs a;
  a.kc = (const uint8_t*)p->key_cache; a.vc = (const uint8_t*)p->value_cache;
  a.key = (char*)p->key; a.value = (char*)p->value;
  a.table = p->block_table; a.cu = p->cu_seqlens; a.starts = p->seq_starts;
  a.k_scale = p->k_scale; a.v_scale = p->v_scale; a.ksh = p->k_scale_stride; a.vsh = p->v_scale_stride;
  a.rows = p->num_rows; a.H = p->num_heads; a.D = p->head_size; a.BS = p->block_size; a.NB = p->num_blocks; a.B = p->batch;
  a.table_stride = p->block_table_stride; a.table_cols = p->block_table_cols;
  a.ks = p->key_stride; a.vs = p->value_stride;
  a.cbs = p->cache_block_stride; a.crs = p->cache_row_stride; a.chs = p->cache_head_stride;
  const int es = dtype_size(p->dtype), ec = is_fp8(p->cache_dtype) ? 1 : es;
  const bool vec = a.D % (16 / ec) == 0 && (a.ks * es) % 16 == 0 && (a.vs * es) % 16 == 0 && (a.cbs * ec) % 16 == 0 &&
                   (a.crs * ec) % 16 == 0 && (a.chs * ec) % 16 == 0 && aligned16(a.key) && aligned16(a.value) &&
                   aligned16(a.kc) && aligned16(a.vc) && a.H * a.D < 100000000LL && a.rows < 2147483647LL * kGatherRows;
  cudaStream_t st = (cudaStream_t)stream;
  FG_DISPATCH_FLOAT(p->dtype, T, {
    if (p->cache_dtype == FG_E4M3) return launch_gather<T, kCacheE4M3>(a, vec, st);
    if (p->cache_dtype == FG_E5M2) return launch_gather<T, kCacheE5M2>(a, vec, st);
    return launch_gather<T, kCache16>(a, vec, st);
  });
  return FG_OK;
}
