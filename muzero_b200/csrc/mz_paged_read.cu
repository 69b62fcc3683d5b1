// Paged cache: tokens back as ordinary keys and values (sm_100a).
//
// A value is A + T (level - z) / 32 (mz_paged.cuh), computed with one fp32 rounding and rounded once to the output's type.  What bounds it is memory: a token's 144
// bytes of codes and words (head_dim 128, 16-bit output) become 512.  A CTA has a piece of an entry, the tokens of one page, for some of the kv heads, one after the other, the
// next one's codes on their way meanwhile.  Keys stand along tokens: a thread of the first half takes 16 tokens of four neighbouring channels, so that a warp's store is a token's
// whole row and nothing is transposed through shared memory.  Values stand along channels: a thread of the second half takes eight of a token's, a warp's store is two tokens' rows
// (head_dim 128).
//
// Measured (B200 at 1965 MHz): 16 rows of 1777 to 4224 tokens, 8 kv heads, head_dim 128, bf16: 62 us for 259 MB, 4.2 TB/s; one head to a CTA of 128 threads 60 us, but 18 instead of 14 us for one row
// of 1000 tokens and 100 instead of 92 for two rows' 101075 later tokens at head_dim 64.
#include <algorithm>

#include "mz_paged_device.cuh"

namespace mzp {
namespace {
constexpr int READ_THREADS = 256, SIDE_THREADS = READ_THREADS / 2, READ_MAX_BATCH = 4096, READ_CTAS = 4, CTAS_PER_SM = 8;

struct ReadArgs {
  mz_paged_cache c;
  mz_paged_read_args a;
  int layer, longest, heads;                     // heads: of a CTA
};

// Four codes -> their levels less z, as f16 pairs (0x6400 + level is 1024 + level)
__device__ __forceinline__ void steps4(uint32_t codes, const uint4& book, __half2 zero, float2& a, float2& b) {
  const uint32_t four = prmt(book.x, book.y, codes) | prmt(book.z, book.w, codes ^ 0x8888u);
  const uint32_t u0 = prmt(four, 0x64646464u, 0x4140u), u1 = prmt(four, 0x64646464u, 0x4342u);
  a = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&u0), zero));
  b = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&u1), zero));
}
template <int DT>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {        // two 16-bit numbers, held to the finite range
  if (DT == MZ_F16) {
    const __half2 h = __floats2half2_rn(fminf(fmaxf(a, -65504.f), 65504.f), fminf(fmaxf(b, -65504.f), 65504.f));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);                // f16's range is well inside
  return *reinterpret_cast<const uint32_t*>(&h);
}
// stores four, or eight, neighbouring values
template <int DT>
__device__ __forceinline__ void put4(void* p, long long at, float a, float b, float c, float d) {
  if (DT == MZ_F32) *(float4*)((float*)p + at) = make_float4(a, b, c, d);
  else *(uint2*)((uint16_t*)p + at) = make_uint2(pair_of<DT>(a, b), pair_of<DT>(c, d));
}
template <int DT>
__device__ __forceinline__ void put8(void* p, long long at, const float (&v)[8]) {
  if (DT == MZ_F32) {
    *(float4*)((float*)p + at) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)((float*)p + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *(uint4*)((uint16_t*)p + at) = make_uint4(pair_of<DT>(v[0], v[1]), pair_of<DT>(v[2], v[3]), pair_of<DT>(v[4], v[5]), pair_of<DT>(v[6], v[7]));
  }
}

// DT: the output's type; BF: the ring's
template <int D, int DT, bool BF>
__global__ void __launch_bounds__(READ_THREADS, READ_CTAS) read_kernel(const ReadArgs p, const uint8_t* __restrict__ book_table) {
  const mz_paged_cache& c = p.c;
  const mz_paged_read_args& a = p.a;
  constexpr int PB = 72 * D;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head0 = blockIdx.y * p.heads, head1 = min(head0 + p.heads, c.kv_heads);
  __shared__ __align__(16) uint8_t s_book[MZP_BOOKS * MZP_LEVELS];
  __shared__ int s_warp[READ_THREADS / 32], s_entry, s_piece;
  if (tid < MZP_BOOKS * MZP_LEVELS / 16) ((uint4*)s_book)[tid] = ((const uint4*)book_table)[tid];
  static_assert(READ_THREADS >= MZP_BOOKS * MZP_LEVELS / 16, "one piece of the books per thread");
  // ---- the entry and its piece: pieces are the pages that an entry's tokens stand in, or would (before the first token too)
  auto page_of = [](long long token) { return token >> 6; };           // rounded down
  static_assert(MZP_PAGE == 64, "page_of");
  auto pieces_of = [&](int i) {
    const long long first = a.first ? a.first[i] : 0, n = (long long)a.offsets[i + 1] - a.offsets[i];
    return n > 0 ? (int)(page_of(first + n - 1) - page_of(first) + 1) : 0;
  };
  if (tid == 0) s_entry = -1;
  long long before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += READ_THREADS) {
    const int i = b0 + tid, n = i < a.batch ? pieces_of(i) : 0;
    int scan = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += y; }
    __syncthreads();
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    long long at = before + scan - n;
#pragma unroll
    for (int w = 0; w < READ_THREADS / 32; ++w) { const int t = s_warp[w]; if (w < warp) at += t; before += t; }
    if (at <= blockIdx.x && blockIdx.x < at + n) { s_entry = i; s_piece = (int)(blockIdx.x - at); }
    if (before > blockIdx.x) break;              // the same for all threads
  }
  __syncthreads();
  const int entry = s_entry;
  if (entry < 0) return;
  const int row = a.rows ? a.rows[entry] : entry;
  if (row < 0 || row >= c.rows) {
    if (tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
    return;
  }
  const long long first = a.first ? a.first[entry] : 0, place0 = a.offsets[entry] - first;       // token t of the row goes to place0 + t
  const long long t0 = (page_of(first) + s_piece) * MZP_PAGE;                                      // the page's first token
  const int len = max(0, min(c.lengths[row], p.longest)), packed = mzp_packed(len, c.residual);
  // the page's tokens lo .. hi - 1 are asked for
  const int lo = (int)max(0ll, max(first - t0, -(place0 + t0)));
  const int hi = (int)max(0ll, min((long long)MZP_PAGE, min(a.offsets[entry + 1], a.tokens) - (place0 + t0)));
  const long long k_at = (place0 + t0) * a.k_stride_token, v_at = (place0 + t0) * a.v_stride_token;
  int id = -1;
  if (t0 >= 0 && t0 < packed) {
    const long long page = t0 / MZP_PAGE;
    id = page < c.width ? c.block_table[(long long)row * c.width + page] : -1;
    if (id < 0 || id >= c.pages) { id = -1; if (tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); }
  }
  if (id < 0) {                                  // the ring's tokens; what is not there is zero
    const uint16_t* ring = (const uint16_t*)c.tail + (long long)p.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row;
    const long long side = (long long)c.kv_heads * c.ring * D;
    for (int i = tid; i < 2 * MZP_PAGE * D / 8 * (head1 - head0); i += READ_THREADS) {
      const int ch = i % (D / 8) * 8, t = i / (D / 8) % MZP_PAGE, value = i / (MZP_PAGE * D / 8) & 1, head = head0 + i / (2 * MZP_PAGE * D / 8);
      if (t < lo || t >= hi) continue;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (t0 >= packed && t0 + t < len) w = *(const uint4*)(ring + (value ? side : 0) + ((long long)head * c.ring + (t0 + t) % c.ring) * D + ch);
      void* out = value ? a.value : a.key;
      const long long at = value ? v_at + head * a.v_stride_head + t * a.v_stride_token + ch : k_at + head * a.k_stride_head + t * a.k_stride_token + ch;
      if (DT == MZ_F32) {
        constexpr int RT = BF ? MZ_BF16 : MZ_F16;
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[2 * k] = mz_u16_to_float((uint16_t)((&w.x)[k] & 0xffffu), RT);
          v[2 * k + 1] = mz_u16_to_float((uint16_t)((&w.x)[k] >> 16), RT);
        }
        put8<DT>(out, at, v);
      } else {
        *(uint4*)((uint16_t*)out + at) = w;
      }
    }
    return;
  }
  const uint8_t* page = (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer + (long long)id * c.store_stride_page + (long long)head0 * PB;
  const uint32_t sbook = smem_u32(s_book);
  const bool whole = lo == 0 && hi == MZP_PAGE;
  const int t = tid % SIDE_THREADS;
  if (tid < SIDE_THREADS) {
    // ---- keys: four channels, 16 tokens (head_dim 64: eight)
    constexpr int TOKENS = MZP_PAGE * (D / 4) / SIDE_THREADS;
    const int ch = t % (D / 4) * 4, t1 = t / (D / 4) * TOKENS;
    uint2 codes[4];
    uint4 words;
    auto load = [&](const uint8_t* at) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (TOKENS == 16) codes[k] = __ldg((const uint2*)(at + 32 * (ch + k) + t1 / 2));
        else codes[k].x = __ldg((const uint32_t*)(at + 32 * (ch + k) + t1 / 2));
      }
      words = __ldg((const uint4*)(at + 32 * D + 4 * ch));
    };
    load(page);
#pragma unroll 1
    for (int head = head0; head < head1; ++head) {
      float scale[4], anchor[4];
      __half2 zero[4];
      uint4 book[4];
      uint2 now[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const MzpRow r = mzp_row((&words.x)[k]);
        scale[k] = r.t * 0.03125f;
        anchor[k] = r.a;
        zero[k] = __float2half2_rn(1024.f + r.z);
        book[k] = book128(sbook + r.z * 16);
        now[k] = codes[k];
      }
      if (head + 1 < head1) load(page + (head + 1 - head0) * PB);
      const long long out = k_at + head * a.k_stride_head + ch;
#pragma unroll
      for (int q = 0; q < TOKENS / 4; ++q) {     // four tokens
        float v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 x, y;
          steps4((q < 2 ? now[k].x : now[k].y) >> (16 * (q & 1)), book[k], zero[k], x, y);
          v[0][k] = fmaf(scale[k], x.x, anchor[k]); v[1][k] = fmaf(scale[k], x.y, anchor[k]);
          v[2][k] = fmaf(scale[k], y.x, anchor[k]); v[3][k] = fmaf(scale[k], y.y, anchor[k]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = t1 + 4 * q + j;
          if (whole || (tok >= lo && tok < hi)) put4<DT>(a.key, out + tok * a.k_stride_token, v[j][0], v[j][1], v[j][2], v[j][3]);
        }
      }
    }
  } else {
    // ---- values: eight channels of every eighth token (head_dim 64: every sixteenth)
    constexpr int TURNS = MZP_PAGE * D / 8 / SIDE_THREADS, STEP_TOKENS = SIDE_THREADS * 8 / D;
    const int tok0 = t / (D / 8), ch = t % (D / 8) * 8;
    uint32_t codes[TURNS], words[TURNS];
    auto load = [&](const uint8_t* at) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        codes[i] = __ldg((const uint32_t*)(at + 36 * D) + t + i * SIDE_THREADS);
        words[i] = __ldg((const uint32_t*)(at + 68 * D) + (t + i * SIDE_THREADS) / 8);
      }
    };
    load(page);
#pragma unroll 1
    for (int head = head0; head < head1; ++head) {
      uint32_t now[TURNS], word[TURNS];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) { now[i] = codes[i]; word[i] = words[i]; }
      if (head + 1 < head1) load(page + (head + 1 - head0) * PB);
      const long long out = v_at + head * a.v_stride_head + ch;
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const MzpRow r = mzp_row(word[i]);
        const uint4 book = book128(sbook + r.z * 16);
        const __half2 zero = __float2half2_rn(1024.f + r.z);
        const float s = r.t * 0.03125f;
        float2 x, y, z, w;
        steps4(now[i], book, zero, x, y);
        steps4(now[i] >> 16, book, zero, z, w);
        const float v[8] = {fmaf(s, x.x, r.a), fmaf(s, x.y, r.a), fmaf(s, y.x, r.a), fmaf(s, y.y, r.a), fmaf(s, z.x, r.a), fmaf(s, z.y, r.a), fmaf(s, w.x, r.a), fmaf(s, w.y, r.a)};
        const int tok = tok0 + i * STEP_TOKENS;
        if (whole || (tok >= lo && tok < hi)) put8<DT>(a.value, out + tok * a.v_stride_token, v);
      }
    }
  }
}

template <int D, int DT, bool BF>
int launch_read(const ReadArgs& p, const uint8_t* book, cudaStream_t st) {
  const long long pieces = p.a.tokens / MZP_PAGE + 2ll * p.a.batch;
  MZ_REQUIRE(pieces < (1ll << 31), "%d tokens of %d entries are too many for one call", p.a.tokens, p.a.batch);
  // heads to a CTA: all that leave 8 CTAs to an SM
  int sms = 0;
  const int rc = mz_paged_sms(&sms);
  if (rc != MZ_OK) return rc;
  ReadArgs q = p;
  q.heads = (int)std::max(1ll, std::min<long long>(p.c.kv_heads, pieces * p.c.kv_heads / (CTAS_PER_SM * sms)));
  read_kernel<D, DT, BF><<<dim3((unsigned)pieces, (p.c.kv_heads + q.heads - 1) / q.heads), READ_THREADS, 0, st>>>(q, book);
  MZ_LAUNCH_CHECK("paged read");
  return MZ_OK;
}
}  // namespace
}  // namespace mzp

extern "C" int mz_paged_read(const mz_paged_cache* cache, int layer, const mz_paged_read_args* args, void* stream) {
  MZ_RANGE("mz_paged_read");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(args != nullptr, "args is NULL");
  MZ_REQUIRE(layer >= 0 && layer < cache->layers, "layer %d of %d", layer, cache->layers);
  MZ_REQUIRE(args->batch >= 0 && args->batch <= mzp::READ_MAX_BATCH, "batch %d (at most %d)", args->batch, mzp::READ_MAX_BATCH);
  MZ_REQUIRE(args->rows != nullptr || args->batch <= cache->rows, "batch %d of %d rows", args->batch, cache->rows);
  MZ_REQUIRE(args->tokens >= 0, "%d tokens", args->tokens);
  MZ_REQUIRE(args->dtype == MZ_F32 || args->dtype == cache->kv_dtype, "dtype must be fp32 or the cache's");
  if (args->batch == 0 || args->tokens == 0) return MZ_OK;
  MZ_REQUIRE(args->key && args->value && args->offsets, "key, value or offsets is NULL");
  const int whole = args->dtype == MZ_F32 ? 4 : 8;
  MZ_REQUIRE(((uintptr_t)args->key | (uintptr_t)args->value) % 16 == 0 &&
                 (args->k_stride_token | args->k_stride_head | args->v_stride_token | args->v_stride_head) % whole == 0,
             "key and value must be 16-byte aligned with strides of whole 16 bytes");
  const uint8_t* book = nullptr;
  if ((rc = mz_paged_tables(&book, nullptr)) != MZ_OK) return rc;
  mzp::ReadArgs p = {*cache, *args, layer, (int)std::min<long long>(0x7fffffff - 2 * MZP_PAGE, cache->residual + (cache->width + 2ll) * MZP_PAGE - 1)};
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = cache->kv_dtype == MZ_BF16, wide = args->dtype == MZ_F32;
#define MZP_GO(D)                                                                                                                  \
  return bf ? (wide ? mzp::launch_read<D, MZ_F32, true>(p, book, st) : mzp::launch_read<D, MZ_BF16, true>(p, book, st))            \
            : (wide ? mzp::launch_read<D, MZ_F32, false>(p, book, st) : mzp::launch_read<D, MZ_F16, false>(p, book, st))
  if (cache->head_dim == 128) MZP_GO(128);
  MZP_GO(64);
#undef MZP_GO
}
