// Paged cache: the quantizing write.  One CTA takes a (list entry, page, kv head): keys by columns (a thread owns 16 tokens of two channels), values
// by rows (a thread owns half of a token's 64 channels), smallest and largest value first, then the codes through the table of nearest levels in shared
// memory.  Tokens that stay are copied to the ring by the same grid, or by a second launch where a new token could take the place of an old
// one that is still to be quantized.
#include "mz_paged.cuh"

namespace {
constexpr int THREADS = 256;

struct AppendArgs {
  mz_paged_cache c;
  const uint16_t *key, *value;
  long long kst, ksh, vst, vsh;
  const int *rows, *offsets;
  int layer, batch, tokens, max_new, slots;
  int quantize, keep;                           // which of the two parts this launch does
};

// 16-bit pair -> two floats
template <bool BF>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

template <int D, bool BF>
__global__ void __launch_bounds__(THREADS) append_kernel(const AppendArgs a, const uint8_t* __restrict__ nearest) {
  constexpr int QUARTERS = THREADS / (D / 2);   // parts of the 64 tokens that a pair of channels is shared out in: 4 (D = 128) or 8
  constexpr int KT = MZP_PAGE / QUARTERS;       // key tokens per thread
  constexpr int VPARTS = THREADS / (MZP_PAGE * D / 64), VN = 64 / VPARTS;     // threads per row of 64 values, and values per thread: 2 x 32 or 4 x 16
  __shared__ __align__(16) uint8_t s_near[MZP_BOOKS * 128];
  __shared__ float2 s_range[QUARTERS][D];
  __shared__ float4 s_row[D];                   // quantizer constants of the keys' rows
  __shared__ __align__(16) uint8_t s_out[D * 32];
  const mz_paged_cache& c = a.c;
  if (*c.status & (MZ_PAGED_NO_PAGES | MZ_PAGED_TOO_LONG)) return;      // the extension failed: there is no room for these tokens
  bool have_table = false;
  const long long units = (long long)a.batch * a.slots * c.kv_heads;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int head = (int)(unit % c.kv_heads), slot = (int)(unit / c.kv_heads % a.slots), i = (int)(unit / c.kv_heads / a.slots);
    const int row = a.rows ? a.rows[i] : i;
    const int first = a.offsets ? a.offsets[i] : i, n = a.offsets ? a.offsets[i + 1] - first : 1;
    if (row < 0 || row >= c.rows || n < 0 || n > a.max_new || first < 0 || first > a.tokens - n) {
      if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
      continue;
    }
    const int after = c.lengths[row], before = after - n;
    if (before < 0) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
    const int packed = mzp_packed(after, c.residual);
    uint16_t* ring_k = (uint16_t*)c.tail + (long long)a.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)head * c.ring * D;
    uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D;
    const uint16_t *new_k = a.key + (long long)head * a.ksh, *new_v = a.value + (long long)head * a.vsh;
    if (a.keep) {
      // 64 of the tokens that stay
      const int start = max(packed, before) + slot * MZP_PAGE, count = min(MZP_PAGE, after - start);
      constexpr int PIECES = D / 8;
      for (int x = threadIdx.x; x < count * PIECES; x += THREADS) {
        const int pos = start + x / PIECES, piece = x % PIECES * 8;
        const long long from = first + (pos - before);
        const int to = pos % c.ring * D + piece;
        *(uint4*)(ring_k + to) = *(const uint4*)(new_k + from * a.kst + piece);
        *(uint4*)(ring_v + to) = *(const uint4*)(new_v + from * a.vst + piece);
      }
    }
    const int page = mzp_packed(before, c.residual) / MZP_PAGE + slot;
    if (!a.quantize || page >= packed / MZP_PAGE || page >= c.width) continue;
    const int id = c.block_table[(long long)row * c.width + page];
    if (id < 0 || id >= c.pages) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
    if (!have_table) {
      for (int x = threadIdx.x; x < MZP_BOOKS * 128 / 16; x += THREADS) ((uint4*)s_near)[x] = ((const uint4*)nearest)[x];
      have_table = true;                        // (the barriers below come before its first use)
    }
    uint8_t* out = (uint8_t*)c.store + (long long)a.layer * c.store_stride_layer + (long long)id * c.store_stride_page + (long long)head * mzp_page_bytes(D);
    const int tok0 = page * MZP_PAGE;
    auto key_of = [&](int t) { const int pos = tok0 + t; return pos < before ? ring_k + pos % c.ring * D : new_k + (long long)(first + pos - before) * a.kst; };
    auto value_of = [&](int t) { const int pos = tok0 + t; return pos < before ? ring_v + pos % c.ring * D : new_v + (long long)(first + pos - before) * a.vst; };
    // ---- keys
    const int pair = threadIdx.x % (D / 2), quarter = threadIdx.x / (D / 2);
    uint32_t x[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) x[t] = *(const uint32_t*)(key_of(quarter * KT + t) + 2 * pair);
    {
      float lo0 = INFINITY, hi0 = -INFINITY, lo1 = INFINITY, hi1 = -INFINITY;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        float2 f = widen<BF>(x[t]);
        f.x = mzp_finite(f.x); f.y = mzp_finite(f.y);
        lo0 = fminf(lo0, f.x); hi0 = fmaxf(hi0, f.x);
        lo1 = fminf(lo1, f.y); hi1 = fmaxf(hi1, f.y);
      }
      s_range[quarter][2 * pair] = make_float2(lo0, hi0);
      s_range[quarter][2 * pair + 1] = make_float2(lo1, hi1);
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float2 r = s_range[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < QUARTERS; ++k) { const float2 s = s_range[k][threadIdx.x]; r.x = fminf(r.x, s.x); r.y = fmaxf(r.y, s.y); }
      const MzpQuant q = mzp_quant(r.x, r.y);
      s_row[threadIdx.x] = make_float4(q.a, q.inv, q.z, 0.f);
      ((uint32_t*)(out + 32 * D))[threadIdx.x] = q.word;
    }
    __syncthreads();
    {
      const float4 r0 = s_row[2 * pair], r1 = s_row[2 * pair + 1];
      const MzpQuant q0 = {r0.x, r0.y, r0.z, 0}, q1 = {r1.x, r1.y, r1.z, 0};
      const uint8_t *n0 = s_near + (int)r0.z * 128, *n1 = s_near + (int)r1.z * 128;
#pragma unroll
      for (int w = 0; w < KT / 8; ++w) {
        uint32_t c0 = 0, c1 = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float2 f = widen<BF>(x[8 * w + t]);
          c0 |= (uint32_t)n0[mzp_level(q0, mzp_finite(f.x))] << (4 * t);
          c1 |= (uint32_t)n1[mzp_level(q1, mzp_finite(f.y))] << (4 * t);
        }
        *(uint32_t*)(s_out + (2 * pair) * 32 + quarter * (KT / 2) + 4 * w) = c0;
        *(uint32_t*)(s_out + (2 * pair + 1) * 32 + quarter * (KT / 2) + 4 * w) = c1;
      }
    }
    // ---- values
    const int vrow = threadIdx.x / VPARTS, part = threadIdx.x % VPARTS;
    uint4 v[VN / 8];
    {
      const uint16_t* src = value_of(vrow / (D / 64)) + vrow % (D / 64) * 64 + part * VN;
#pragma unroll
      for (int k = 0; k < VN / 8; ++k) v[k] = *(const uint4*)(src + 8 * k);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < D * 2; k += THREADS) ((uint4*)out)[k] = ((const uint4*)s_out)[k];
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int k = 0; k < VN / 8; ++k) {
      const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = widen<BF>(w[j]);
        const float f0 = mzp_finite(f.x), f1 = mzp_finite(f.y);
        lo = fminf(lo, fminf(f0, f1));
        hi = fmaxf(hi, fmaxf(f0, f1));
      }
    }
#pragma unroll
    for (int o = 1; o < VPARTS; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const MzpQuant q = mzp_quant(lo, hi);
    const uint8_t* near_row = s_near + (int)q.z * 128;
    uint32_t code[VN / 8];
#pragma unroll
    for (int k = 0; k < VN / 8; ++k) {
      const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
      code[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = widen<BF>(w[j]);
        code[k] |= (uint32_t)near_row[mzp_level(q, mzp_finite(f.x))] << (8 * j) | (uint32_t)near_row[mzp_level(q, mzp_finite(f.y))] << (8 * j + 4);
      }
    }
    uint32_t* vout = (uint32_t*)(out + 36 * D + vrow * 32 + part * (VN / 2));
#pragma unroll
    for (int k = 0; k < VN / 8; ++k) vout[k] = code[k];
    if (part == 0) ((uint32_t*)(out + 68 * D))[vrow] = q.word;
    __syncthreads();                            // s_out, s_range and s_row are written again
  }
}

int launch(const AppendArgs& a, cudaStream_t st) {
  const uint8_t* nearest = nullptr;
  int rc = mz_paged_tables(nullptr, &nearest);
  if (rc != MZ_OK) return rc;
  int dev = 0, sms = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  MZ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const long long units = (long long)a.batch * a.slots * a.c.kv_heads;
  const unsigned ctas = (unsigned)(units < 4ll * sms ? units : 4ll * sms);
  const bool bf = a.c.kv_dtype == MZ_BF16;
  if (a.c.head_dim == 128) {
    if (bf) append_kernel<128, true><<<ctas, THREADS, 0, st>>>(a, nearest);
    else append_kernel<128, false><<<ctas, THREADS, 0, st>>>(a, nearest);
  } else {
    if (bf) append_kernel<64, true><<<ctas, THREADS, 0, st>>>(a, nearest);
    else append_kernel<64, false><<<ctas, THREADS, 0, st>>>(a, nearest);
  }
  MZ_LAUNCH_CHECK("append");
  return MZ_OK;
}
}  // namespace

extern "C" int mz_paged_append(const mz_paged_cache* cache, int layer, const void* key, long long k_stride_token, long long k_stride_head,
                               const void* value, long long v_stride_token, long long v_stride_head, const int* rows, const int* offsets, int batch,
                               int tokens, int max_new, void* stream) {
  MZ_RANGE("mz_paged_append");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(layer >= 0 && layer < cache->layers, "layer %d of %d", layer, cache->layers);
  MZ_REQUIRE(batch >= 0 && tokens >= 0 && max_new >= 0, "batch %d, tokens %d, max_new %d", batch, tokens, max_new);
  MZ_REQUIRE(rows != nullptr || batch <= cache->rows, "batch %d of %d rows", batch, cache->rows);
  MZ_REQUIRE(offsets != nullptr || tokens == batch, "%d tokens for %d rows of one token each", tokens, batch);
  if (batch == 0 || tokens == 0 || max_new == 0) return MZ_OK;
  MZ_REQUIRE(key != nullptr && value != nullptr, "key or value is NULL");
  MZ_REQUIRE(((uintptr_t)key | (uintptr_t)value) % 16 == 0 && (k_stride_token | k_stride_head | v_stride_token | v_stride_head) % 8 == 0,
             "key and value must be 16-byte aligned with strides in multiples of 8 elements");
  AppendArgs a = {*cache, (const uint16_t*)key, (const uint16_t*)value, k_stride_token, k_stride_head, v_stride_token, v_stride_head, rows, offsets,
                  layer, batch, tokens, max_new, 0, 1, 1};
  const int pages = (max_new + MZP_PAGE - 1) / MZP_PAGE, window = cache->residual + MZP_PAGE - 1;       // tokens that may stay
  const int kept = ((max_new < window ? max_new : window) + MZP_PAGE - 1) / MZP_PAGE;
  // from the oldest token that is not in a page to the newest one: no two of so few share a place in the ring
  if ((long long)window + max_new <= cache->ring) {
    a.slots = pages > kept ? pages : kept;
    return launch(a, (cudaStream_t)stream);
  }
  a.slots = pages; a.keep = 0;
  if ((rc = launch(a, (cudaStream_t)stream)) != MZ_OK) return rc;
  a.slots = kept; a.keep = 1; a.quantize = 0;
  return launch(a, (cudaStream_t)stream);
}
