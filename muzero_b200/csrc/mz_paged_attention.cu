// Paged cache: attention of the newest tokens of each row over its pages and its ring (sm_100a, tcgen05 on the integer tensor cores).
//
// Mathematics.  A code stands for A + T (u - z) / 32 with a level u of 7 bits (mz_paged.cuh), so for a step of two pages
//   logit[t]  = sum_d q_d T_d u_td / 32 + sum_d q_d (A_d - T_d z_d / 32)         (rows of 64 codes: a channel d of a page)
//   out[d]   += sum_t p_t T_t u_td / 32 + sum_t p_t (A_t - T_t z_t / 32)         (rows of 64 codes: 64 channels of a token t)
// The levels go to the tensor cores as the bytes they are: a thread looks the 64 codes of its row up in the 16 levels of book z, held in four
// registers, by byte permutes, four codes at a time, and stores the bytes into an operand that is major along the row.  The other operand is q T
// (p T) as a 31-bit fixed-point number in four signed bytes, scaled by powers of two, so the sums are exact integers; what
// is rounded is q T and p T, to 2^-31 of the step's largest T (queries are scaled into [-1, 1], p is at most 1).
//   M 128 = 2 blocks of 64 positions along the rows (keys: tokens of the two pages; values: the two channel groups at head_dim 128, the two
//   pages at 64), N = 2 blocks x NR query rows x 4 bytes, of which a position reads its block's; K = the rows that are summed over
//
// Work.  A query row is one (token, head) that shares a kv head; NR of them (4, or 8 above 4) go through a step together, more take several
// passes.  The steps of all (list entry, kv head, pass) pairs stand in one line that is cut evenly over the CTAs on the device, from the lengths it
// finds there; a CTA leaves a record (m, l, out) per pair that it met, slot = CTA + pair.  The 16-bit tokens of the rings go to CTAs of their own in
// the same launch (mma.sync), one record per pair.  A second kernel merges a pair's records.
//
// A CTA that has steps: four warps expand keys, one step ahead, four warps have softmax and values.  MMAs are issued by one thread of each team.  Every
// mbarrier wait is bounded; one that runs out makes the CTA's records NaN and ends its MMAs.
#include "mz_paged.cuh"

namespace mzp {
constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 256, MAX_BATCH = 1024;
constexpr int SPIN_LIMIT = 1000000;              // looks of a wait before it gives up; afterwards one look each
constexpr int STEP = 2 * MZP_PAGE;

struct Args {
  mz_paged_cache c;
  const uint16_t* query;
  long long qsb, qsl, qsh;
  const int* rows;
  void* out;
  int out_dtype, layer, batch, q_len, q_heads, group;      // group: query heads per kv head
  int qrows, passes;                             // query rows per kv head, and how many passes of NR they take
  float scaling;                                 // times log2(e)
  // workspace: header {CTAs with steps, pad, steps (64 bits)}, steps before each entry [batch + 1], records
  int* head;
  float2* ml;                                    // [slot][NR] maximum (base 2) and sum
  float* acc;                                    // [slot][NR][D]
  long long pairs;
};

// ---- small wrappers
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(s));
  return d;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) { uint32_t r; asm("redux.sync.max.u32 %0, %1, 0xffffffff;" : "=r"(r) : "r"(v)); return r; }
__device__ __forceinline__ float warp_max(float v) { float r; asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 book128(uint32_t a) {      // constant after the set-up
  uint4 v;
  asm("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 ldg128(const void* p) {    // pages are read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void team_barrier(int team) { asm volatile("bar.sync %0, 128;" ::"r"(team + 1) : "memory"); }
__device__ __forceinline__ void fence_operands() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.shared::cta.b64 t, [%0];\n\t}\n" ::"r"(bar) : "memory");
}
// Waits for the phase of this parity.  Who gives up says so before it goes on.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* s_failed, bool& failed) {
  const int limit = failed ? 1 : SPIN_LIMIT;
  for (int it = 0; it < limit; ++it) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return;
  }
  failed = true;
  *s_failed = 1;
}
// shared-memory operand, not swizzled, major along the kept dimension: cores of 8 rows x 16 bytes, 128 bytes apart along the reduction,
// `chunk` bytes apart along the kept dimension
__device__ __forceinline__ uint64_t descriptor(uint32_t sa, uint32_t chunk) {
  return (uint64_t)((sa >> 4) & 0x3FFF) | (128ull >> 4) << 16 | (uint64_t)(chunk >> 4) << 32 | 1ull << 46;
}
// D[128 x N] (+)= A[128 x 32] * B[32 x N], unsigned times signed bytes into 32 bits
template <int N>
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t accumulate) {
  const uint32_t idesc = (2u << 4) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(N / 8) << 17) | (8u << 24);
  const uint32_t zero = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(zero), "r"(zero), "r"(zero), "r"(zero) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t taddr, int* c) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]), "=r"(c[4]), "=r"(c[5]), "=r"(c[6]), "=r"(c[7]), "=r"(c[8]), "=r"(c[9]),
                 "=r"(c[10]), "=r"(c[11]), "=r"(c[12]), "=r"(c[13]), "=r"(c[14]), "=r"(c[15])
               : "r"(taddr) : "memory");
  // the wait names the registers, so that nothing reads them above it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]), "+r"(c[4]), "+r"(c[5]), "+r"(c[6]), "+r"(c[7]), "+r"(c[8]), "+r"(c[9]),
                 "+r"(c[10]), "+r"(c[11]), "+r"(c[12]), "+r"(c[13]), "+r"(c[14]), "+r"(c[15]) :: "memory");
}
// four bytes' accumulators -> their number
__device__ __forceinline__ float number_of(const int* c) { return fmaf((float)(c[2] + (c[3] << 8)), 65536.0f, (float)(c[0] + (c[1] << 8))); }
// 31-bit fixed point -> four signed bytes
__device__ __forceinline__ uint32_t digits_of(float x) { return ((uint32_t)__float2int_rn(x) + 0x808080u) ^ 0x808080u; }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// Sums of N values over a warp, N values at a time: after it lane l has the sum of value index_of(l).  N a power of two, at most 32
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int lane, int& index) {
  index = 0;
  int off = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, off >>= 1) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if (i < n / 2) {
        const float send = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
      }
    }
    index += up ? n / 2 : 0;
  }
  float x = v[0];
  for (; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// D(16x8, fp32) += A(16x16) * B(16x8)
template <bool BF>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// a page's row of 64 codes -> 64 bytes, stored as four pieces of 16, `chunk` bytes apart.  A selector's top bit asks for the sign of a level, which is
// zero: so the two permutes of a nibble are zero exactly where they are not meant, and their results are or-ed.
__device__ __forceinline__ void expand_row(const uint4& lo, const uint4& hi, const uint4& book, uint32_t dst, uint32_t chunk) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t a = w[2 * q + k], b = a ^ 0x88888888u;
      o[2 * k] = prmt(book.x, book.y, a) | prmt(book.z, book.w, b);
      o[2 * k + 1] = prmt(book.x, book.y, a >> 16) | prmt(book.z, book.w, b >> 16);
    }
    sts128(dst + q * chunk, o[0], o[1], o[2], o[3]);
  }
}

// shared memory of a CTA
template <int D, int NR>
struct Smem {
  static constexpr int ROWS = D;                           // rows of the keys' operand = rows of the values' operand (D == 128: 128 tokens)
  static constexpr int CHUNK = ROWS * 16;
  static constexpr int A_BYTES = 8 * CHUNK;                // 128 positions
  static constexpr int B_BYTES = 2 * NR * 4 / 16 * CHUNK;  // 2 blocks x NR x 4 bytes
  static constexpr int K_A = 0, V_A = A_BYTES, K_B = 2 * A_BYTES, V_B = K_B + B_BYTES;
  static constexpr int OPERANDS = V_B + B_BYTES;
  static constexpr int RINGS = 8 * NR * D * 4;             // a ring CTA's partial outputs lie over the operands
  static constexpr int BOOK = OPERANDS > RINGS ? OPERANDS : RINGS;
  static constexpr int TOTAL = BOOK + MZP_BOOKS * MZP_LEVELS;
  static constexpr int N = 8 * NR, TM_S = 0, TM_O = 2 * N, TM_COLS = NR == 4 ? 128 : 256;
  static constexpr int CTAS = NR == 4 ? 3 : 2;             // per SM
};
// exchange between the warps of a CTA
template <int NR>
struct Exchange {
  float base[4][4][2 * NR];                 // constant terms of the logits, by step and key warp (keys run up to two steps ahead)
  float fin[4][4 * NR];                     // end of a pair: sums of p, constant terms of the output
  float qs[4][NR];                          // logit per unit of the scaled query, by pair
  float qmax[4][4][NR];                     // largest |q|, by pair and warp
  float vmax[2][4][NR];                     // largest logit, by step parity and warp
  uint32_t kt[4][4], vt[2][4];              // largest T (bits) of the keys, by step and warp; of the values
  float ring_m[8][NR], ring_l[8][NR];
  unsigned long long bar[6];                // products of the keys done [2], their sums read [2], products of the values done, end
  int warp_sum[8][2];
  uint32_t tmem;
  int failed;
  int prefix[MAX_BATCH + 1];                // steps of the entries before
};

struct Cursor { int b, kp, step, steps; };

template <int D, bool BF, int NR>
__global__ void __launch_bounds__(THREADS, (Smem<D, NR>::CTAS)) attention_kernel(const Args p, const uint8_t* __restrict__ book_table) {
  using S = Smem<D, NR>;
  constexpr int DT = BF ? MZ_BF16 : MZ_F16;
  constexpr int PB = 72 * D;                     // page bytes per kv head
  constexpr int RPT = D / 64;                    // rows of codes per thread, side and step
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Exchange<NR> x;
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(smem), sbook = sbase + S::BOOK;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t bars = smem_u32(x.bar);
  const uint32_t k_done = bars, k_free = bars + 16, v_done = bars + 32, b_end = bars + 40;
  if (tid == 0) {
    x.failed = 0;
    bar_init(k_done, 2); bar_init(k_done + 8, 2);
    bar_init(k_free, 128); bar_init(k_free + 8, 128);
    bar_init(v_done, 1); bar_init(b_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < MZP_BOOKS * MZP_LEVELS / 16; i += THREADS) ((uint4*)(smem + S::BOOK))[i] = ((const uint4*)book_table)[i];
  asm volatile("griddepcontrol.wait;" ::: "memory");        // what was before is written, and the records are read

  // ---- the line of steps, and how many CTAs take rings
  const int kp_all = c.kv_heads * p.passes;
  auto length_of = [&](int b) {
    const int row = p.rows ? p.rows[b] : b;
    if (row < 0 || row >= c.rows) return 0;
    return max(0, min(c.lengths[row], 0x7fffffff - STEP));
  };
  long long ring_tokens = 0;
  int total_steps;
  {
    constexpr int PER = MAX_BATCH / THREADS;
    int st[PER], sum = 0, rt = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int b = tid * PER + k, len = b < p.batch ? length_of(b) : 0;
      const int packed = mzp_packed(len, c.residual);
      st[k] = (packed + STEP - 1) / STEP;
      sum += st[k];
      rt += len - packed;
    }
    int scan = sum, ring_sum = rt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += y;
      ring_sum += __shfl_xor_sync(0xffffffffu, ring_sum, o);
    }
    if (lane == 31) { x.warp_sum[warp][0] = scan; x.warp_sum[warp][1] = ring_sum; }
    __syncthreads();
    int before = scan - sum;
    total_steps = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += x.warp_sum[w][0];
      total_steps += x.warp_sum[w][0];
      ring_tokens += x.warp_sum[w][1];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int b = tid * PER + k;
      if (b <= p.batch) x.prefix[b] = before;
      before += st[k];
    }
    if (tid == THREADS - 1 && p.batch == MAX_BATCH) x.prefix[MAX_BATCH] = before;
    __syncthreads();
  }
  const long long T = (long long)total_steps * kp_all;
  const int G = gridDim.x;
  // cost of a ring: 16 per token, a step 1024 (measured; see the launch)
  int n_ring = 0;
  if (ring_tokens > 0) {
    const double cr = (double)ring_tokens * kp_all * 16.0, cs = (double)T * 1024.0;
    n_ring = (int)(G * cr / (cr + cs) + 0.5);
    n_ring = max(1, min(n_ring, T > 0 ? G - 1 : G));
  }
  const int W = (int)min((long long)(G - n_ring), T);        // CTAs that share the steps: none is left without one
  if (blockIdx.x == 0) {
    if (tid == 0) { p.head[0] = W; *(long long*)(p.head + 2) = T; }
    for (int b = tid; b <= p.batch; b += THREADS) p.head[4 + b] = x.prefix[b];
  }
  const long long ring_slots = (long long)G + p.pairs;

  if ((int)blockIdx.x < n_ring) {
    // ================= rings: a warp takes 16 tokens at a time; A = keys [token][channel], B = queries; A = values [channel][token], B = p in two parts
    const int g = lane >> 2, t = lane & 3;
    for (long long unit = blockIdx.x; unit < p.pairs; unit += n_ring) {
      const int b = (int)(unit / kp_all), kp = (int)(unit % kp_all), head = kp / p.passes, r0 = kp % p.passes * NR;
      const int row = p.rows ? p.rows[b] : b, len = length_of(b), packed = mzp_packed(len, c.residual);
      if (len == packed) continue;
      const int tokens = len - packed;
      const uint16_t* ring_k = (const uint16_t*)c.tail + (long long)p.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)head * c.ring * D;
      const uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D;
      const int ring0 = packed % c.ring;
      auto place = [&](int i) { int r = ring0 + i; return r >= c.ring ? r - c.ring : r; };      // i < tokens <= ring
      // queries: column g = query row r0 + g; a lane's 8 channels of each block of 32
      uint4 qf[D / 32];
      {
        const int r = r0 + g;
        const bool on = g < NR && r < p.qrows;
        const int l = on ? r / p.group : 0, h = head * p.group + (on ? r % p.group : 0);
        const uint16_t* qp = p.query + (long long)b * p.qsb + l * p.qsl + h * p.qsh + 8 * t;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          qf[k] = make_uint4(0, 0, 0, 0);
          if (on) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (uint32_t)qp[32 * k + 2 * j] | (uint32_t)qp[32 * k + 2 * j + 1] << 16;
            qf[k] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      // columns 2t, 2t + 1 of the logits: the last token that the query sees, counted from the ring's first
      int last[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) last[j] = len - p.q_len + (r0 + 2 * t + j) / p.group - packed;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 16][4];
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
      for (int tile = warp; tile * 16 < tokens; tile += 8) {
        const int i0 = tile * 16;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        {
          const uint16_t* ka = ring_k + (long long)place(min(i0 + g, tokens - 1)) * D + 8 * t;
          const uint16_t* kb = ring_k + (long long)place(min(i0 + g + 8, tokens - 1)) * D + 8 * t;
          uint4 va[D / 32], vb[D / 32];
#pragma unroll
          for (int k = 0; k < D / 32; ++k) { va[k] = *(const uint4*)(ka + 32 * k); vb[k] = *(const uint4*)(kb + 32 * k); }
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            mma16<BF>(s, va[k].x, vb[k].x, va[k].y, vb[k].y, qf[k].x, qf[k].y);
            mma16<BF>(s, va[k].z, vb[k].z, va[k].w, vb[k].w, qf[k].z, qf[k].w);
          }
        }
        // s[0], s[1]: token g, columns 2t, 2t + 1; s[2], s[3]: token g + 8
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + g + 8 * (k >> 1);
          s[k] = i < tokens && i <= last[k & 1] ? s[k] * p.scaling : -INFINITY;
        }
        float pr[4], fix[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(s[j], s[2 + j]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float m_new = fmaxf(m[j], top), ref = m_new == -INFINITY ? 0.f : m_new;
          fix[j] = ex2(m[j] - ref);
          m[j] = m_new;
          pr[j] = ex2(s[j] - ref);
          pr[2 + j] = ex2(s[2 + j] - ref);
          l[j] = l[j] * fix[j] + pr[j] + pr[2 + j];
        }
        if (__any_sync(0xffffffffu, fix[0] != 1.0f || fix[1] != 1.0f)) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) { o[i][0] *= fix[0]; o[i][1] *= fix[1]; o[i][2] *= fix[0]; o[i][3] *= fix[1]; }
        }
        // p in two parts of 16 bits, transposed: column g, tokens 2t, 2t + 1 (part [0]) and 2t + 8, 2t + 9 (part [1])
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t hw, lw;
          if (BF) {
            const __nv_bfloat162 hb = __floats2bfloat162_rn(pr[2 * half], pr[2 * half + 1]);
            const float2 hf = __bfloat1622float2(hb);
            const __nv_bfloat162 lb = __floats2bfloat162_rn(pr[2 * half] - hf.x, pr[2 * half + 1] - hf.y);
            hw = *reinterpret_cast<const uint32_t*>(&hb); lw = *reinterpret_cast<const uint32_t*>(&lb);
          } else {
            const __half2 hb = __floats2half2_rn(pr[2 * half], pr[2 * half + 1]);
            const float2 hf = __half22float2(hb);
            const __half2 lb = __floats2half2_rn(pr[2 * half] - hf.x, pr[2 * half + 1] - hf.y);
            hw = *reinterpret_cast<const uint32_t*>(&hb); lw = *reinterpret_cast<const uint32_t*>(&lb);
          }
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(hi[half]) : "r"(hw));
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(lo[half]) : "r"(lw));
        }
        // A token that is not there, or that only later queries see, must not bring a NaN to a product with p = 0: what is not there is read as zero, and
        // where a tile has tokens that only some of the queries see, each of the queries' tokens takes its turn with what it sees
        const int l_first = r0 / p.group, l_last = min(r0 + NR, p.qrows) - 1;
        const int see0 = len - p.q_len - packed;               // token l sees those up to see0 + l
        const bool apart = i0 + 15 > see0 + l_first && l_last / p.group > l_first;
        const int turns = apart ? l_last / p.group - l_first + 1 : 1;
        for (int turn = 0; turn < turns; ++turn) {
          const int see = apart ? min(see0 + l_first + turn, tokens - 1) : tokens - 1;
          const bool mine = !apart || (r0 + g) / p.group == l_first + turn;
          const uint32_t h0 = mine ? hi[0] : 0u, h1 = mine ? hi[1] : 0u, e0 = mine ? lo[0] : 0u, e1 = mine ? lo[1] : 0u;
#pragma unroll
          for (int grp = 0; grp < D / 64; ++grp) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = i0 + 2 * t + (k & 1) + 8 * (k >> 1);
              v[k] = make_uint4(0, 0, 0, 0);
              if (i <= see) v[k] = *(const uint4*)(ring_v + (long long)place(i) * D + grp * 64 + 8 * g);
            }
            const uint32_t w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
            const uint32_t w2[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, w3[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // rows g / g + 8 = channels 8g + 2k / 8g + 2k + 1
              const uint32_t a0 = prmt(w0[k], w1[k], 0x5410u), a1 = prmt(w0[k], w1[k], 0x7632u);
              const uint32_t a2 = prmt(w2[k], w3[k], 0x5410u), a3 = prmt(w2[k], w3[k], 0x7632u);
              mma16<BF>(o[grp * 4 + k], a0, a1, a2, a3, e0, e1);
              mma16<BF>(o[grp * 4 + k], a0, a1, a2, a3, h0, h1);
            }
          }
        }
      }
      // ---- the eight warps' parts -> one record
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], off);
        if (g == 0 && 2 * t + j < NR) { x.ring_m[warp][2 * t + j] = m[j]; x.ring_l[warp][2 * t + j] = l[j]; }
      }
      __syncthreads();
      float* part = (float*)smem;                // [warp][NR][D]
      if (2 * t < NR) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = x.ring_m[0][2 * t + j];
#pragma unroll
          for (int w = 1; w < 8; ++w) top = fmaxf(top, x.ring_m[w][2 * t + j]);
          const float f = m[j] == -INFINITY ? 0.f : ex2(m[j] - top);
          float* dst = part + (warp * NR + 2 * t + j) * D + 8 * g;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) *(float2*)(dst + (i >> 2) * 64 + 2 * (i & 3)) = make_float2(o[i][j] * f, o[i][2 + j] * f);
        }
      }
      __syncthreads();
      const long long slot = ring_slots + unit;
      for (int i = tid; i < NR * D; i += THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += part[w * NR * D + i];
        p.acc[slot * NR * D + i] = sum;
      }
      if (tid < NR) {
        float top = x.ring_m[0][tid], sum = 0.f;
#pragma unroll
        for (int w = 1; w < 8; ++w) top = fmaxf(top, x.ring_m[w][tid]);
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += x.ring_m[w][tid] == -INFINITY ? 0.f : x.ring_l[w][tid] * ex2(x.ring_m[w][tid] - top);
        p.ml[slot * NR + tid] = make_float2(top, sum);
      }
      __syncthreads();
    }
    return;
  }

  // ================= steps
  const int cta = (int)blockIdx.x - n_ring;
  if (cta >= W) return;
  const long long f0 = T * cta / W, f1 = T * (cta + 1) / W;
  const int n = (int)(f1 - f0);
  if (n <= 0) return;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tm_before();
  }
  __syncthreads();
  tm_after();
  const uint32_t tmem = x.tmem;
  bool failed = false;
  Cursor cur;
  {
    int lo = 0, hi = p.batch;                    // prefix[lo] * kp_all <= f0 < prefix[lo + 1] * kp_all
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if ((long long)x.prefix[mid] * kp_all <= f0) lo = mid; else hi = mid; }
    cur.b = lo;
    cur.steps = x.prefix[lo + 1] - x.prefix[lo];
    const int rem = (int)(f0 - (long long)x.prefix[lo] * kp_all);
    cur.kp = rem / cur.steps;
    cur.step = rem % cur.steps;
  }
  auto advance = [&](Cursor& q) {
    if (++q.step < q.steps) return;
    q.step = 0;
    if (++q.kp < kp_all) return;
    q.kp = 0;
    do { ++q.b; } while (q.b < p.batch && x.prefix[q.b + 1] == x.prefix[q.b]);
    q.steps = q.b < p.batch ? x.prefix[q.b + 1] - x.prefix[q.b] : 1;
  };
  const int r = tid & 127;                       // key channel or token of this thread
  // the page of this thread's rows: both pages (keys, D = 128) or the one that position r lies in
  auto page_at = [&](const Cursor& q, int which) -> const uint8_t* {
    if (q.b >= p.batch) return nullptr;
    const int row = p.rows ? p.rows[q.b] : q.b;
    const int pages = mzp_packed(length_of(q.b), c.residual) / MZP_PAGE, k = 2 * q.step + which;
    if (k >= pages) return nullptr;
    const int id = k < c.width ? __ldg(c.block_table + (long long)row * c.width + k) : -1;
    if (id < 0 || id >= c.pages) { atomicOr(c.status, MZ_PAGED_BAD_INDEX); return nullptr; }
    return (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer + (long long)id * c.store_stride_page + (long long)(q.kp / p.passes) * PB;
  };
  uint4 code[RPT][2];
  uint32_t word[RPT];
  // a row's codes and word; a page that is not there has T = 0
  auto load_row = [&](int j, const uint8_t* codes, const uint8_t* words) {
    code[j][0] = code[j][1] = make_uint4(0, 0, 0, 0);
    word[j] = 0;
    if (codes) {
      code[j][0] = ldg128(codes);
      code[j][1] = ldg128(codes + 16);
      word[j] = __ldg((const uint32_t*)words);
    }
  };

  if (warp < 4) {
    // ================= keys: thread = channel
    const int ch = D == 128 ? r : r & 63;
    auto load_keys = [&](const Cursor& q) {
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const uint8_t* base = page_at(q, D == 128 ? j : r >> 6);
        load_row(j, base ? base + ch * 32 : nullptr, base + 32 * D + 4 * ch);
      }
    };
    float q[NR];
    int pair = -1, seg = -1;
    load_keys(cur);
    for (int it = 0; it < n; ++it) {
      const int this_pair = cur.b * kp_all + cur.kp;
      const bool fresh = this_pair != pair;
      MzpRow row[RPT];
      uint32_t tb = 0;
#pragma unroll
      for (int j = 0; j < RPT; ++j) { row[j] = mzp_row(word[j]); tb = max(tb, word[j] & 0xffffu); }
      tb = warp_max_u32(tb);
      if (lane == 0) x.kt[it & 3][warp] = tb;
      if (fresh) {
        pair = this_pair; ++seg;
        const int head = cur.kp / p.passes, r0 = cur.kp % p.passes * NR;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          q[i] = 0.f;
          if (r0 + i < p.qrows) {
            const int l = (r0 + i) / p.group, h = head * p.group + (r0 + i) % p.group;
            q[i] = MzType<DT>::load(p.query, (long long)cur.b * p.qsb + l * p.qsl + h * p.qsh + ch);
          }
          // as bits, so that a NaN is the largest
          const uint32_t top = warp_max_u32(__float_as_uint(fabsf(q[i])));
          if (lane == 0) x.qmax[seg & 3][warp][i] = __uint_as_float(top);
        }
      }
      team_barrier(0);
      if (fresh) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          uint32_t top = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) top = max(top, __float_as_uint(x.qmax[seg & 3][w][i]));
          const int e = max((int)(top >> 23) - 126, -60), e1 = e >> 1, e2 = e - e1;        // |q| < 2^e, taken off in two factors
          const bool wild = top >= 0x7f800000u;                        // infinity or NaN: the row's logits are NaN
          q[i] = wild ? 0.f : q[i] * pow2(-e1) * pow2(-e2);
          if (tid == 0) x.qs[seg & 3][i] = wild ? __int_as_float(0x7fffffff) : pow2(e1) * p.scaling * pow2(e2);
        }
      }
      const uint32_t top = max(max(x.kt[it & 3][0], x.kt[it & 3][1]), max(x.kt[it & 3][2], x.kt[it & 3][3]));
      const float up = pow2(30 - ((int)(top >> 10) - 14));             // T < 2^(exponent field - 14)
      uint32_t fold[RPT][NR];
      {
        float base[RPT * NR];
#pragma unroll
        for (int j = 0; j < RPT; ++j) {
          const float ts = row[j].t * up, cz = fmaf(row[j].t, (float)row[j].z * -0.03125f, row[j].a);
#pragma unroll
          for (int i = 0; i < NR; ++i) { fold[j][i] = digits_of(q[i] * ts); base[j * NR + i] = q[i] * cz; }
        }
        int index;
        const float sum = warp_sums<RPT * NR>(base, lane, index);
        if ((lane & (32 / (RPT * NR) - 1)) == 0) x.base[it & 3][warp][index] = sum;
      }
      if (it > 0) bar_wait(k_done + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1, &x.failed, failed);      // the operand is free
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const int blk = D == 128 ? j : r >> 6;
#pragma unroll
        for (int i = 0; i < NR; i += 4)
          sts128(sbase + S::K_B + (blk * (NR / 4) + i / 4) * S::CHUNK + ch * 16, fold[j][i], fold[j][i + 1], fold[j][i + 2], fold[j][i + 3]);
        expand_row(code[j][0], code[j][1], book128(sbook + row[j].z * 16), sbase + S::K_A + blk * 4 * S::CHUNK + ch * 16, S::CHUNK);
      }
      Cursor nxt = cur;
      advance(nxt);
      if (it + 1 < n) load_keys(nxt);
      cur = nxt;
      fence_operands();
      team_barrier(0);
      if (tid == 0) {
        if (it >= 2) bar_wait(k_free + 8 * (it & 1), ((it - 2) >> 1) & 1, &x.failed, failed);
        bar_arrive(k_done + 8 * (it & 1));
        if (!x.failed) {
          tm_after();
          const uint64_t a = descriptor(sbase + S::K_A, S::CHUNK), b = descriptor(sbase + S::K_B, S::CHUNK);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma<S::N>(tmem + S::TM_S + (it & 1) * S::N, a + k * (512 >> 4), b + k * (512 >> 4), k > 0);
          umma_commit(k_done + 8 * (it & 1));
        }
      }
    }
  } else {
    // ================= softmax and values: thread = token, and position of the output
    const int tw = warp - 4, blk = r >> 6;
    const uint32_t lanes = tmem + ((uint32_t)(tw * 32) << 16);
    auto load_values = [&](const Cursor& q) {
      const uint8_t* base = page_at(q, r >> 6);
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const int vr = (r & 63) * RPT + j;
        load_row(j, base ? base + 36 * D + vr * 32 : nullptr, base + 68 * D + 4 * vr);
      }
    };
    float m[NR], l[NR], o[NR], base_v[RPT][NR], qs[NR];
    float vunit = 0.f;
    int pair = -1, seg = -1, limit0 = 0, packed = 0;
    bool masked = false;
    int r0 = 0;
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; o[i] = 0.f; qs[i] = 0.f; }
#pragma unroll
    for (int j = 0; j < RPT; ++j)
#pragma unroll
      for (int i = 0; i < NR; ++i) base_v[j][i] = 0.f;
    // the products of the step before, which is number `done`
    auto take_output = [&](int done) {
      bar_wait(v_done, done & 1, &x.failed, failed);
      tm_after();
#pragma unroll
      for (int i = 0; i < NR; i += 4) {
        int a[16];
        tm_ld16(lanes + S::TM_O + blk * (4 * NR) + 4 * i, a);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i + k] = fmaf(number_of(a + 4 * k), vunit, o[i + k]);
      }
    };
    auto write_record = [&]() {
      constexpr int NV = NR * (RPT == 2 ? 4 : 2);            // l, constant terms (and padding)
      float v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        v[i] = l[i];
#pragma unroll
        for (int j = 0; j < RPT; ++j) v[(1 + j) * NR + i] = base_v[j][i];
      }
      int index;
      const float sum = warp_sums<NV>(v, lane, index);
      if ((lane & (32 / NV - 1)) == 0) x.fin[tw][index] = sum;
      float* halves = (float*)(smem + S::V_B);               // D = 64: the second page's part; the products that read this are done
      if (D == 64 && r >= 64) {
#pragma unroll
        for (int i = 0; i < NR; ++i) halves[(r - 64) * NR + i] = o[i];
      }
      team_barrier(1);
      const long long slot = (long long)cta + pair;
      const bool bad = *(volatile int*)&x.failed != 0;
      if (D == 128 || r < 64) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          const int at = (1 + (D == 128 ? blk : 0)) * NR + i;
          float out = o[i] + ((x.fin[0][at] + x.fin[1][at]) + (x.fin[2][at] + x.fin[3][at]));
          if (D == 64) out += halves[r * NR + i];
          p.acc[(slot * NR + i) * D + r] = out;
        }
      }
      if (r < NR) {
        const float sum_l = (x.fin[0][r] + x.fin[1][r]) + (x.fin[2][r] + x.fin[3][r]);
        float top = m[0];
#pragma unroll
        for (int i = 1; i < NR; ++i) top = r == i ? m[i] : top;
        p.ml[slot * NR + r] = bad ? make_float2(INFINITY, __int_as_float(0x7fffffff)) : make_float2(top, sum_l);
      }
      team_barrier(1);                                       // fin and halves are free again
    };
    load_values(cur);
    for (int it = 0; it < n; ++it) {
      const int this_pair = cur.b * kp_all + cur.kp;
      const bool fresh = this_pair != pair;
      if (fresh) {
        if (pair >= 0) {
          take_output(it - 1);
          write_record();
        }
        pair = this_pair; ++seg;
        r0 = cur.kp % p.passes * NR;
        const int len = length_of(cur.b);
        packed = mzp_packed(len, c.residual);
        limit0 = len - p.q_len;
        masked = packed > limit0 + 1;
#pragma unroll
        for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; o[i] = 0.f; }
#pragma unroll
        for (int j = 0; j < RPT; ++j)
#pragma unroll
          for (int i = 0; i < NR; ++i) base_v[j][i] = 0.f;
      }
      MzpRow row[RPT];
      uint32_t tb = 0;
#pragma unroll
      for (int j = 0; j < RPT; ++j) { row[j] = mzp_row(word[j]); tb = max(tb, word[j] & 0xffffu); }
      tb = warp_max_u32(tb);
      // ---- logits
      bar_wait(k_done + 8 * (it & 1), (it >> 1) & 1, &x.failed, failed);
      tm_after();
      if (fresh) {
#pragma unroll
        for (int i = 0; i < NR; ++i) qs[i] = x.qs[seg & 3][i];
      }
      const uint32_t ktop = max(max(x.kt[it & 3][0], x.kt[it & 3][1]), max(x.kt[it & 3][2], x.kt[it & 3][3]));
      const float kunit = pow2((int)(ktop >> 10) - 14 - 35);
      float s[NR];
#pragma unroll
      for (int i = 0; i < NR; i += 4) {
        int a[16];
        tm_ld16(lanes + S::TM_S + (it & 1) * S::N + blk * (4 * NR) + 4 * i, a);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[i + k] = number_of(a + 4 * k) * kunit;
      }
      const int pos = cur.step * STEP + r;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        float base;
        if (D == 128) {
          const int at = blk * NR + i;
          base = (x.base[it & 3][0][at] + x.base[it & 3][1][at]) + (x.base[it & 3][2][at] + x.base[it & 3][3][at]);
        } else {
          base = x.base[it & 3][2 * blk][i] + x.base[it & 3][2 * blk + 1][i];
        }
        s[i] = (s[i] + base) * qs[i];
        if (pos >= packed) s[i] = -INFINITY;
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < NR; ++i) if (pos > limit0 + (r0 + i) / p.group) s[i] = -INFINITY;
      }
      tm_before();
      bar_arrive(k_free + 8 * (it & 1));
      // ---- running maximum
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float top = warp_max(s[i]);
        if (lane == 0) x.vmax[it & 1][tw][i] = top;
      }
      if (lane == 0) x.vt[it & 1][tw] = tb;
      team_barrier(1);
      float fix[NR];
      bool moved = false;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float top = fmaxf(fmaxf(x.vmax[it & 1][0][i], x.vmax[it & 1][1][i]), fmaxf(x.vmax[it & 1][2][i], x.vmax[it & 1][3][i]));
        const float m_new = fmaxf(m[i], top), ref = m_new == -INFINITY ? 0.f : m_new;
        fix[i] = ex2(m[i] - ref);
        moved |= m_new != m[i];
        m[i] = m_new;
        s[i] = ex2(s[i] - ref);
      }
      const uint32_t vtop = max(max(x.vt[it & 1][0], x.vt[it & 1][1]), max(x.vt[it & 1][2], x.vt[it & 1][3]));
      const int ev = (int)(vtop >> 10) - 14;
      const float up = pow2(30 - ev);
      // ---- the output so far; then the operand is free
      if (it > 0 && !fresh) take_output(it - 1);
      if (moved) {                                           // the same for all threads
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          o[i] *= fix[i]; l[i] *= fix[i];
#pragma unroll
          for (int j = 0; j < RPT; ++j) base_v[j][i] *= fix[i];
        }
      }
      vunit = pow2(ev - 35);
#pragma unroll
      for (int i = 0; i < NR; ++i) l[i] += s[i];
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const float ts = row[j].t * up, cz = fmaf(row[j].t, (float)row[j].z * -0.03125f, row[j].a);
        const int b2 = D == 128 ? j : blk, at = D == 128 ? r : r & 63;
#pragma unroll
        for (int i = 0; i < NR; ++i) base_v[j][i] = fmaf(s[i], cz, base_v[j][i]);
#pragma unroll
        for (int i = 0; i < NR; i += 4)
          sts128(sbase + S::V_B + (b2 * (NR / 4) + i / 4) * S::CHUNK + at * 16, digits_of(s[i] * ts), digits_of(s[i + 1] * ts),
                 digits_of(s[i + 2] * ts), digits_of(s[i + 3] * ts));
        expand_row(code[j][0], code[j][1], book128(sbook + row[j].z * 16), sbase + S::V_A + b2 * 4 * S::CHUNK + at * 16, S::CHUNK);
      }
      Cursor nxt = cur;
      advance(nxt);
      if (it + 1 < n) load_values(nxt);
      cur = nxt;
      fence_operands();
      tm_before();
      team_barrier(1);
      if (r == 0 && !*(volatile int*)&x.failed) {
        tm_after();
        const uint64_t a = descriptor(sbase + S::V_A, S::CHUNK), b = descriptor(sbase + S::V_B, S::CHUNK);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) umma<S::N>(tmem + S::TM_O, a + k * (512 >> 4), b + k * (512 >> 4), k > 0);
        umma_commit(v_done);
      }
    }
    take_output(n - 1);
    write_record();
  }
  __syncthreads();
  if (x.failed && tid == 0) {                    // products in flight end before their memory goes back
    umma_commit(b_end);
    bar_wait(b_end, 0, &x.failed, failed = false);
  }
  tm_before();
  __syncthreads();
  if (warp == 0) {
    tm_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TM_COLS));
  }
}

// merges the records of one query row of a pair: a thread per channel, records in their order
template <int D, bool BF, int NR>
__global__ void __launch_bounds__(D) merge_kernel(const Args p, int G) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int i = blockIdx.x % NR, d = threadIdx.x;
  const long long pair = blockIdx.x / NR;
  const int kp_all = p.c.kv_heads * p.passes, b = (int)(pair / kp_all), kp = (int)(pair % kp_all), head = kp / p.passes, qr = kp % p.passes * NR + i;
  if (qr >= p.qrows) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = p.rows ? p.rows[b] : b;
  const bool known = row >= 0 && row < p.c.rows;
  if (!known && d == 0) atomicOr(p.c.status, MZ_PAGED_BAD_INDEX);
  const int len = known ? max(0, min(p.c.lengths[row], 0x7fffffff - STEP)) : 0;
  const bool ring = len > mzp_packed(len, p.c.residual);
  const long long W = p.head[0], T = *(const long long*)(p.head + 2);
  const long long steps = p.head[4 + b + 1] - p.head[4 + b], s0 = (long long)p.head[4 + b] * kp_all + kp * steps;
  float m = -INFINITY, l = 0.f, a = 0.f;
  auto take = [&](float2 ml, float v) {
    const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
    const float f = ex2(m - ref), g = ex2(ml.x - ref);
    l = l * f + ml.y * g;
    a = a * f + v * g;
    m = top;
  };
  if (steps > 0) {
    // CTA c has the steps from T c / W on: the one with step f is ((f + 1) W - 1) / T
    const long long first = ((s0 + 1) * W - 1) / T, last = ((s0 + steps) * W - 1) / T;
    for (long long c0 = first; c0 <= last; c0 += 4) {
      float2 ml[4];
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long slot = (min(c0 + k, last) + pair) * NR + i;
        ml[k] = p.ml[slot];
        v[k] = p.acc[slot * D + d];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) if (c0 + k <= last) take(ml[k], v[k]);
    }
  }
  if (ring) {
    const long long slot = (G + p.pairs + pair) * NR + i;
    take(p.ml[slot], p.acc[slot * D + d]);
  }
  const float out = l == 0.f ? 0.f : a / l;
  const int ql = qr / p.group, h = head * p.group + qr % p.group;
  mz_store_from_float(p.out, (((long long)b * p.q_len + ql) * p.q_heads + h) * D + d, out, p.out_dtype);
}

template <int D, bool BF, int NR>
int launch(const Args& p, const uint8_t* book, int G, cudaStream_t st) {
  auto kern = attention_kernel<D, BF, NR>;
  using S = Smem<D, NR>;
  MZ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)G);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  MZ_CUDA(cudaLaunchKernelEx(&cfg, kern, p, book));
  MZ_LAUNCH_CHECK("paged attention");
  cfg.gridDim = dim3((unsigned)(p.pairs * NR));
  cfg.blockDim = dim3(D);
  cfg.dynamicSmemBytes = 0;
  MZ_CUDA(cudaLaunchKernelEx(&cfg, merge_kernel<D, BF, NR>, p, G));
  MZ_LAUNCH_CHECK("paged attention merge");
  return MZ_OK;
}

struct Shape { int nr, passes, G; long long pairs; size_t head_bytes, slots, bytes; };
int shape_of(const mz_paged_cache* c, int batch, int q_len, int q_heads, Shape* s) {
  MZ_REQUIRE(batch >= 0 && batch <= MAX_BATCH, "batch %d (at most %d)", batch, MAX_BATCH);
  MZ_REQUIRE(q_len >= 1 && q_heads >= 1 && q_heads % c->kv_heads == 0, "q_len %d, q_heads %d of %d kv heads", q_len, q_heads, c->kv_heads);
  const long long qrows = (long long)q_heads / c->kv_heads * q_len;
  MZ_REQUIRE(qrows <= 1 << 20, "%lld query rows per kv head", qrows);
  int dev = 0, sms = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  MZ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  s->nr = qrows <= 4 ? 4 : 8;
  s->passes = (int)((qrows + s->nr - 1) / s->nr);
  s->pairs = (long long)batch * c->kv_heads * s->passes;
  MZ_REQUIRE(s->pairs * s->nr < (1ll << 31), "too many query rows for one call");
  s->G = sms * (s->nr == 4 ? 3 : 2);
  s->head_bytes = ((4 + (size_t)batch + 1) * sizeof(int) + 127) / 128 * 128;
  s->slots = (size_t)s->G + 2 * (size_t)s->pairs;
  s->bytes = s->head_bytes + s->slots * s->nr * (sizeof(float2) + (size_t)c->head_dim * sizeof(float));
  return MZ_OK;
}
}  // namespace mzp

extern "C" size_t mz_paged_attention_workspace_bytes(const mz_paged_cache* cache, int batch, int q_len, int q_heads) {
  mzp::Shape s;
  if (mz_paged_check(cache) != MZ_OK || mzp::shape_of(cache, batch, q_len, q_heads, &s) != MZ_OK) return 0;
  return s.bytes;
}

extern "C" int mz_paged_attention(const mz_paged_cache* cache, int layer, const mz_paged_attention_args* args, void* stream) {
  MZ_RANGE("mz_paged_attention");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(args != nullptr, "args is NULL");
  MZ_REQUIRE(layer >= 0 && layer < cache->layers, "layer %d of %d", layer, cache->layers);
  MZ_REQUIRE(args->rows != nullptr || args->batch <= cache->rows, "batch %d of %d rows", args->batch, cache->rows);
  MZ_REQUIRE(args->out_dtype == MZ_F32 || args->out_dtype == cache->kv_dtype, "out_dtype must be fp32 or the cache's");
  mzp::Shape s;
  if ((rc = mzp::shape_of(cache, args->batch, args->q_len, args->q_heads, &s)) != MZ_OK) return rc;
  if (args->batch == 0) return MZ_OK;
  MZ_REQUIRE(args->query && args->out, "query or out is NULL");
  if (!args->workspace || (uintptr_t)args->workspace % 16 != 0 || args->workspace_bytes < s.bytes)
    return mz_fail(MZ_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed (16-byte aligned)", args->workspace_bytes, s.bytes);
  const uint8_t* book = nullptr;
  if ((rc = mz_paged_tables(&book, nullptr)) != MZ_OK) return rc;
  mzp::Args p = {};
  p.c = *cache;
  p.query = (const uint16_t*)args->query;
  p.qsb = args->q_stride_b; p.qsl = args->q_stride_l; p.qsh = args->q_stride_h;
  p.rows = args->rows;
  p.out = args->out;
  p.out_dtype = args->out_dtype;
  p.layer = layer;
  p.batch = args->batch; p.q_len = args->q_len; p.q_heads = args->q_heads;
  p.group = args->q_heads / cache->kv_heads;
  p.qrows = p.group * args->q_len;
  p.passes = s.passes;
  p.scaling = args->scaling * mzp::LOG2E;
  p.head = (int*)args->workspace;
  p.acc = (float*)((uint8_t*)args->workspace + s.head_bytes);
  p.ml = (float2*)(p.acc + s.slots * s.nr * cache->head_dim);
  p.pairs = s.pairs;
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = cache->kv_dtype == MZ_BF16;
#define MZP_GO(D, NR) return bf ? mzp::launch<D, true, NR>(p, book, s.G, st) : mzp::launch<D, false, NR>(p, book, s.G, st)
  if (cache->head_dim == 128) { if (s.nr == 4) MZP_GO(128, 4); MZP_GO(128, 8); }
  if (s.nr == 4) MZP_GO(64, 4);
  MZP_GO(64, 8);
#undef MZP_GO
}
