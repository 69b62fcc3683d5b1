// Paged cache: attention of the newest tokens of each row over its pages and its ring.
//
// One CTA takes one query row (list entry, token, head): a page's logits with a thread per token and part of the channels, online softmax, then the values
// with a thread per channel, everything in fp32.
#include "mz_paged.cuh"

namespace {
struct Args {
  mz_paged_cache c;
  mz_paged_attention_args a;
  int layer;
};
constexpr float LOG2E = 1.4426950408889634f;

template <int D, bool BF>
__global__ void __launch_bounds__(128) attention_kernel(const Args p, const uint8_t* __restrict__ book) {
  constexpr int PARTS = 128 / MZP_PAGE;
  constexpr int DT = BF ? MZ_BF16 : MZ_F16;
  __shared__ uint8_t s_book[MZP_BOOKS * MZP_LEVELS];
  __shared__ float s_q[D], s_part[PARTS][MZP_PAGE], s_p[MZP_PAGE];
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x;
  const int h = blockIdx.x % p.a.q_heads, l = blockIdx.x / p.a.q_heads % p.a.q_len, b = blockIdx.x / p.a.q_heads / p.a.q_len;
  const int kvh = h / (p.a.q_heads / c.kv_heads);
  const int row = p.a.rows ? p.a.rows[b] : b;
  for (int i = tid; i < MZP_BOOKS * MZP_LEVELS; i += 128) s_book[i] = book[i];
  if (tid < D) s_q[tid] = MzType<DT>::load(p.a.query, b * p.a.q_stride_b + l * p.a.q_stride_l + h * p.a.q_stride_h + tid);
  const bool known = row >= 0 && row < c.rows;
  if (!known && tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
  const int len = known ? c.lengths[row] : 0;
  const int packed = mzp_packed(len, c.residual), seen = len - p.a.q_len + l + 1;       // tokens this query sees
  float m = -INFINITY, sum = 0.f, acc = 0.f;
  __syncthreads();
  const int tok = tid % MZP_PAGE, part = tid / MZP_PAGE;
  const uint16_t* ring_k = (const uint16_t*)c.tail + (long long)p.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)kvh * c.ring * D;
  const uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D;
  for (int t0 = 0; t0 < seen; t0 += MZP_PAGE) {
    const bool page = t0 < packed;
    const uint8_t* base = nullptr;
    if (page) {
      const int id = t0 / MZP_PAGE < c.width ? c.block_table[(long long)row * c.width + t0 / MZP_PAGE] : -1;
      if (id < 0 || id >= c.pages) { if (tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
      base = (const uint8_t*)c.store + p.layer * c.store_stride_layer + id * c.store_stride_page + (long long)kvh * mzp_page_bytes(D);
    }
    const int n = min(MZP_PAGE, seen - t0);
    float dot = 0.f;
    if (tok < n) {
      for (int d = part * (D / PARTS); d < (part + 1) * (D / PARTS); ++d) {
        float k;
        if (page) {
          const MzpRow r = mzp_row(((const uint32_t*)(base + 32 * D))[d]);
          const int e = base[d * 32 + tok / 2] >> (4 * (tok & 1)) & 15;
          k = r.a + r.t * (float)((int)s_book[r.z * 16 + e] - r.z) * 0.03125f;
        } else {
          k = MzType<DT>::load(ring_k, (long long)((t0 + tok) % c.ring) * D + d);
        }
        dot = fmaf(s_q[d], k, dot);
      }
    }
    s_part[part][tok] = dot;
    __syncthreads();
    float s = -INFINITY;
    if (tok < n) { s = 0.f; for (int i = 0; i < PARTS; ++i) s += s_part[i][tok]; s *= p.a.scaling * LOG2E; }
    __syncthreads();
    s_part[part][tok] = s;
    __syncthreads();
    float top = -INFINITY;
    for (int i = 0; i < n; ++i) top = fmaxf(top, s_part[0][i]);
    const float m_new = fmaxf(m, top), fix = exp2f(m - m_new);
    if (part == 0) s_p[tok] = tok < n ? exp2f(s - m_new) : 0.f;
    __syncthreads();
    acc *= fix; sum *= fix; m = m_new;
    for (int i = 0; i < n; ++i) {
      sum += s_p[i];
      if (tid < D) {
        float v;
        if (page) {
          const MzpRow r = mzp_row(((const uint32_t*)(base + 68 * D))[i * (D / 64) + tid / 64]);
          const int e = base[36 * D + i * (D / 2) + tid / 2] >> (4 * (tid & 1)) & 15;
          v = r.a + r.t * (float)((int)s_book[r.z * 16 + e] - r.z) * 0.03125f;
        } else {
          v = MzType<DT>::load(ring_v, (long long)((t0 + i) % c.ring) * D + tid);
        }
        acc = fmaf(s_p[i], v, acc);
      }
    }
    __syncthreads();
  }
  if (tid < D) {
    const float o = sum == 0.f ? 0.f : acc / sum;
    mz_store_from_float(p.a.out, (((long long)b * p.a.q_len + l) * p.a.q_heads + h) * D + tid, o, p.a.out_dtype);
  }
}
}  // namespace

extern "C" size_t mz_paged_attention_workspace_bytes(const mz_paged_cache* cache, int batch, int q_len, int q_heads) {
  if (mz_paged_check(cache) != MZ_OK || batch < 0 || q_len < 1 || q_heads < 1) return 0;
  return 16;
}

extern "C" int mz_paged_attention(const mz_paged_cache* cache, int layer, const mz_paged_attention_args* args, void* stream) {
  MZ_RANGE("mz_paged_attention");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(args != nullptr, "args is NULL");
  MZ_REQUIRE(layer >= 0 && layer < cache->layers, "layer %d of %d", layer, cache->layers);
  MZ_REQUIRE(args->batch >= 0 && args->batch <= 1024, "batch %d (at most 1024)", args->batch);
  MZ_REQUIRE(args->q_len >= 1 && args->q_heads >= 1 && args->q_heads % cache->kv_heads == 0, "q_len %d, q_heads %d of %d kv heads", args->q_len,
             args->q_heads, cache->kv_heads);
  MZ_REQUIRE(args->rows != nullptr || args->batch <= cache->rows, "batch %d of %d rows", args->batch, cache->rows);
  MZ_REQUIRE(args->out_dtype == MZ_F32 || args->out_dtype == cache->kv_dtype, "out_dtype must be fp32 or the cache's");
  if (args->batch == 0) return MZ_OK;
  MZ_REQUIRE(args->query && args->out, "query or out is NULL");
  if (!args->workspace || args->workspace_bytes < mz_paged_attention_workspace_bytes(cache, args->batch, args->q_len, args->q_heads))
    return mz_fail(MZ_ERR_WORKSPACE, "workspace of %zu bytes", args->workspace_bytes);
  const uint8_t* book = nullptr;
  if ((rc = mz_paged_tables(&book, nullptr)) != MZ_OK) return rc;
  const Args p = {*cache, *args, layer};
  const unsigned ctas = (unsigned)(args->batch * args->q_len * args->q_heads);
  const bool bf = cache->kv_dtype == MZ_BF16;
  cudaStream_t st = (cudaStream_t)stream;
  if (cache->head_dim == 128) {
    if (bf) attention_kernel<128, true><<<ctas, 128, 0, st>>>(p, book);
    else attention_kernel<128, false><<<ctas, 128, 0, st>>>(p, book);
  } else {
    if (bf) attention_kernel<64, true><<<ctas, 128, 0, st>>>(p, book);
    else attention_kernel<64, false><<<ctas, 128, 0, st>>>(p, book);
  }
  MZ_LAUNCH_CHECK("paged attention");
  return MZ_OK;
}
