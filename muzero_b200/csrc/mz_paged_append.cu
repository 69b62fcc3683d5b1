// Paged cache: the quantizing write.  One CTA takes a (list entry, page, kv head): keys by columns (a thread owns 16 tokens of two channels), values
// by rows (a thread owns half of a token's 64 channels), smallest and largest value first, then the codes through the table of nearest levels in shared
// memory.  Tokens that stay are copied to the ring by the same grid, or by a second launch where a new token could take the place of an old
// one that is still to be quantized.
//
// What bounds it is the instructions of a value: two to find the range (pairs of 16 bits), eight to its code, of which one is the table's load.  What is
// rare is kept out of them (prompts of 1777 to 4096 tokens x 8 kv heads, head_dim 128, 265 MB read and written: 102.6 us, 2.6 TB/s; issue slots 61 % used,
// shared-memory wavefronts 64 %, most of them the lookups, which meet the same banks; 170 us with the range and the code of every value in the general form): a row with a NaN, an infinity, a value beyond f16 or a scale below f16's normal numbers is done again by the general form.
#include "mz_paged.cuh"

namespace {
constexpr int THREADS = 256, CTAS_PER_SM = 5;      // (four: 105 instead of 102 us for prompts of 1777 to 4096 tokens)

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

constexpr float MAGIC = 12582912.0f;            // 1.5 * 2^23: adding it rounds to an integer, which stands in the low bits

// smallest and largest of 16-bit pairs, as pairs; `odd` becomes NaN where a value is not finite
template <bool BF>
struct Range {
  uint32_t lo, hi, odd;
  __device__ __forceinline__ void start(uint32_t w) {
    lo = hi = w;
    odd = 0;
    note(w);
  }
  __device__ __forceinline__ void note(uint32_t w) {
    if (BF) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(w), "r"(0u));
    else asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(w), "r"(0u));
  }
  __device__ __forceinline__ void add(uint32_t w) {
    if (BF) {
      asm("min.bf16x2 %0, %0, %1;" : "+r"(lo) : "r"(w));
      asm("max.bf16x2 %0, %0, %1;" : "+r"(hi) : "r"(w));
    } else {
      asm("min.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(w));
      asm("max.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(w));
    }
    note(w);
  }
};
// what a thread needs for the codes of a row
struct Coder { float a, inv, z; int near; };    // near: address of the row's entry 0 in the table, less the bits of MAGIC
__device__ __forceinline__ uint32_t code_of(const Coder& q, float x) {
  const float y = __fadd_rn(__fmul_rn(__fsub_rn(x, q.a), q.inv), q.z);
  uint32_t v;
  asm("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(q.near + __float_as_int(__fadd_rn(y, MAGIC))));
  return v;
}
// the general form: any value, any scale
__device__ __forceinline__ uint32_t code_of_any(const Coder& q, float x) {
  const float y = __fadd_rn(__fmul_rn(__fsub_rn(mzp_finite(x), q.a), q.inv), q.z);
  uint32_t v;
  asm("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(q.near + __float_as_int(__fadd_rn(fminf(fmaxf(y, 0.0f), 127.0f), MAGIC))));
  return v;
}
// whether a row is one for the general form: something in it was not finite, or its scale is below f16's normal numbers (then it is coarse)
__device__ __forceinline__ bool needs_care(bool odd, uint32_t word) { return odd || (word & 0x7C00u) == 0u; }

template <int D, bool BF>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) append_kernel(const AppendArgs a, const uint8_t* __restrict__ nearest) {
  constexpr int QUARTERS = THREADS / (D / 2);   // parts of the 64 tokens that a pair of channels is shared out in: 4 (D = 128) or 8
  constexpr int KT = MZP_PAGE / QUARTERS;       // key tokens per thread
  constexpr int VPARTS = THREADS / (MZP_PAGE * D / 64), VN = 64 / VPARTS;     // threads per row of 64 values, and values per thread: 2 x 32 or 4 x 16
  __shared__ __align__(16) uint8_t s_near[MZP_BOOKS * MZP_NEAR_ROW];
  __shared__ float2 s_range[QUARTERS][D];
  __shared__ float4 s_row[D];                   // quantizer constants of the keys' rows; the last is not 0 for the general form
  __shared__ __align__(16) uint8_t s_out[D * 32];
  const mz_paged_cache& c = a.c;
  const bool refused = *c.status & MZ_PAGED_REFUSED;      // nothing has been announced: the lists are looked over, and nothing is written
  const int near0 = (int)__cvta_generic_to_shared(s_near) + 1 - __float_as_int(MAGIC);
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
    if (refused) continue;
    const int after = c.lengths[row], before = after - n;
    if (before < 0) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
    const int packed = mzp_packed(after, c.residual);
    uint16_t* ring_k = (uint16_t*)c.tail + (long long)a.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)head * c.ring * D;
    uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D;
    const uint16_t *new_k = a.key + (long long)first * a.kst + (long long)head * a.ksh, *new_v = a.value + (long long)first * a.vst + (long long)head * a.vsh;
    if (a.keep) {
      // 64 of the tokens that stay
      const int start = max(packed, before) + slot * MZP_PAGE, count = min(MZP_PAGE, after - start);
      constexpr int PIECES = D / 8;
      for (int x = threadIdx.x; x < count * PIECES; x += THREADS) {
        const int pos = start + x / PIECES, piece = x % PIECES * 8;
        const int to = pos % c.ring * D + piece;
        *(uint4*)(ring_k + to) = *(const uint4*)(new_k + (pos - before) * a.kst + piece);
        *(uint4*)(ring_v + to) = *(const uint4*)(new_v + (pos - before) * a.vst + piece);
      }
    }
    const int page = mzp_packed(before, c.residual) / MZP_PAGE + slot;
    if (!a.quantize || page >= packed / MZP_PAGE || page >= c.width) continue;
    const int id = c.block_table[(long long)row * c.width + page];
    if (id < 0 || id >= c.pages) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
    // ---- all loads first
    const int tok0 = page * MZP_PAGE, ring0 = tok0 % c.ring;
    const int pair = threadIdx.x % (D / 2), quarter = threadIdx.x / (D / 2);
    uint32_t x[KT];
    if (tok0 >= before) {                       // the page is all new tokens
      const uint16_t* from = new_k + (tok0 - before + quarter * KT) * a.kst + 2 * pair;
#pragma unroll
      for (int t = 0; t < KT; ++t) x[t] = *(const uint32_t*)(from + t * a.kst);
    } else {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const int tok = quarter * KT + t, pos = tok0 + tok, place = ring0 + tok - (ring0 + tok >= c.ring ? c.ring : 0);
        x[t] = *(const uint32_t*)((pos < before ? ring_k + place * D : new_k + (pos - before) * a.kst) + 2 * pair);
      }
    }
    const int vrow = threadIdx.x / VPARTS, part = threadIdx.x % VPARTS;
    uint4 v[VN / 8];
    {
      const int tok = vrow / (D / 64), pos = tok0 + tok, place = ring0 + tok - (ring0 + tok >= c.ring ? c.ring : 0);
      const uint16_t* src = (pos < before ? ring_v + place * D : new_v + (pos - before) * a.vst) + vrow % (D / 64) * 64 + part * VN;
#pragma unroll
      for (int k = 0; k < VN / 8; ++k) v[k] = *(const uint4*)(src + 8 * k);
    }
    if (!have_table) {
      for (int k = threadIdx.x; k < MZP_BOOKS * MZP_NEAR_ROW / 16; k += THREADS) ((uint4*)s_near)[k] = ((const uint4*)nearest)[k];
      have_table = true;                        // (the barriers below come before its first use)
    }
    uint8_t* out = (uint8_t*)c.store + (long long)a.layer * c.store_stride_layer + (long long)id * c.store_stride_page + (long long)head * mzp_page_bytes(D);
    // ---- keys
    bool odd_pair;
    {
      Range<BF> rg;
      rg.start(x[0]);
#pragma unroll
      for (int t = 1; t < KT; ++t) rg.add(x[t]);
      float2 lo = widen<BF>(rg.lo), hi = widen<BF>(rg.hi);
      const float2 odd = widen<BF>(rg.odd);
      odd_pair = odd.x != 0.f || odd.y != 0.f || fmaxf(fmaxf(hi.x, hi.y), -fminf(lo.x, lo.y)) > 65504.0f;      // (NaN is not 0 either)
      if (odd_pair) {
        lo = make_float2(INFINITY, INFINITY); hi = make_float2(-INFINITY, -INFINITY);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          float2 f = widen<BF>(x[t]);
          f.x = mzp_finite(f.x); f.y = mzp_finite(f.y);
          lo.x = fminf(lo.x, f.x); hi.x = fmaxf(hi.x, f.x);
          lo.y = fminf(lo.y, f.y); hi.y = fmaxf(hi.y, f.y);
        }
      }
      *(float4*)&s_range[quarter][2 * pair] = make_float4(lo.x, hi.x, lo.y, hi.y);
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float2 r = s_range[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < QUARTERS; ++k) { const float2 s = s_range[k][threadIdx.x]; r.x = fminf(r.x, s.x); r.y = fmaxf(r.y, s.y); }
      const MzpQuant q = mzp_quant(r.x, r.y);
      s_row[threadIdx.x] = make_float4(q.a, q.inv, q.z, needs_care(false, q.word) ? 1.f : 0.f);
      ((uint32_t*)(out + 32 * D))[threadIdx.x] = q.word;
    }
    // ---- values' ranges meanwhile
    Range<BF> rg;
    rg.start(v[0].x);
#pragma unroll
    for (int k = 0; k < VN / 8; ++k) {
      if (k > 0) rg.add(v[k].x);
      rg.add(v[k].y); rg.add(v[k].z); rg.add(v[k].w);
    }
    float vlo, vhi;
    bool odd_row;
    {
      const float2 lo = widen<BF>(rg.lo), hi = widen<BF>(rg.hi), odd = widen<BF>(rg.odd);
      vlo = fminf(lo.x, lo.y);
      vhi = fmaxf(hi.x, hi.y);
      odd_row = odd.x != 0.f || odd.y != 0.f || fmaxf(vhi, -vlo) > 65504.0f;
      if (odd_row) {
        vlo = INFINITY; vhi = -INFINITY;
#pragma unroll
        for (int k = 0; k < VN / 8; ++k) {
          const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = widen<BF>(w[j]);
            const float f0 = mzp_finite(f.x), f1 = mzp_finite(f.y);
            vlo = fminf(vlo, fminf(f0, f1));
            vhi = fmaxf(vhi, fmaxf(f0, f1));
          }
        }
      }
#pragma unroll
      for (int o = 1; o < VPARTS; o <<= 1) {
        vlo = fminf(vlo, __shfl_xor_sync(0xffffffffu, vlo, o));
        vhi = fmaxf(vhi, __shfl_xor_sync(0xffffffffu, vhi, o));
      }
    }
    __syncthreads();
    {
      const float4 r0 = s_row[2 * pair], r1 = s_row[2 * pair + 1];
      const Coder q0 = {r0.x, r0.y, r0.z, near0 + (int)r0.z * MZP_NEAR_ROW}, q1 = {r1.x, r1.y, r1.z, near0 + (int)r1.z * MZP_NEAR_ROW};
      const bool care = odd_pair || r0.w != 0.f || r1.w != 0.f;
      uint32_t c0[KT / 8], c1[KT / 8];
#pragma unroll
      for (int w = 0; w < KT / 8; ++w) c0[w] = c1[w] = 0;
      if (!care) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const float2 f = widen<BF>(x[t]);
          c0[t / 8] += code_of(q0, f.x) * (1u << 4 * (t % 8));
          c1[t / 8] += code_of(q1, f.y) * (1u << 4 * (t % 8));
        }
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const float2 f = widen<BF>(x[t]);
          c0[t / 8] += code_of_any(q0, f.x) << 4 * (t % 8);
          c1[t / 8] += code_of_any(q1, f.y) << 4 * (t % 8);
        }
      }
#pragma unroll
      for (int w = 0; w < KT / 8; ++w) {
        *(uint32_t*)(s_out + (2 * pair) * 32 + quarter * (KT / 2) + 4 * w) = c0[w];
        *(uint32_t*)(s_out + (2 * pair + 1) * 32 + quarter * (KT / 2) + 4 * w) = c1[w];
      }
    }
    // ---- values
    {
      const MzpQuant qq = mzp_quant(vlo, vhi);
      const Coder q = {qq.a, qq.inv, qq.z, near0 + (int)qq.z * MZP_NEAR_ROW};
      uint32_t code[VN / 8];
      if (!needs_care(odd_row, qq.word)) {
#pragma unroll
        for (int k = 0; k < VN / 8; ++k) {
          const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          code[k] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = widen<BF>(w[j]);
            code[k] += code_of(q, f.x) * (1u << 8 * j) + code_of(q, f.y) * (1u << (8 * j + 4));
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < VN / 8; ++k) {
          const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          code[k] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = widen<BF>(w[j]);
            code[k] += (code_of_any(q, f.x) << 8 * j) + (code_of_any(q, f.y) << (8 * j + 4));
          }
        }
      }
      uint32_t* vout = (uint32_t*)(out + 36 * D + vrow * 32 + part * (VN / 2));
      if constexpr (VN == 32) *(uint4*)vout = make_uint4(code[0], code[1], code[2], code[3]);
      else *(uint2*)vout = make_uint2(code[0], code[1]);
      if (part == 0) ((uint32_t*)(out + 68 * D))[vrow] = qq.word;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < D * 2; k += THREADS) ((uint4*)out)[k] = ((const uint4*)s_out)[k];
    // (s_out is written again after the next unit's two barriers, s_range and s_row have been read)
  }
}

int launch(const AppendArgs& a, cudaStream_t st) {
  const uint8_t* nearest = nullptr;
  int rc = mz_paged_tables(nullptr, &nearest);
  if (rc != MZ_OK) return rc;
  int sms = 0;
  if ((rc = mz_paged_sms(&sms)) != MZ_OK) return rc;
  const long long units = (long long)a.batch * a.slots * a.c.kv_heads;
  const unsigned ctas = (unsigned)(units < (long long)CTAS_PER_SM * sms ? units : (long long)CTAS_PER_SM * sms);
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
  max_new = max_new < tokens ? max_new : tokens;      // (an entry that brought more would pass the end of the tokens)
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
