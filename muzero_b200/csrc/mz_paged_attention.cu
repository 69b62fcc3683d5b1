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
// finds there; a CTA leaves a record (m, l, out) per pair that it met, slot = CTA + pair.  A CTA is four warps, four CTAs to an SM (three for 8 query
// rows), and every thread does all of a step: keys as channel r, values as token r, output as channel r.  What a step needs from memory was asked for
// a step earlier; the products of the keys run while the values' levels are written, those of the values while the next step's keys are.  Every
// wait for products is bounded; one that runs out makes the CTA's records NaN and ends its MMAs.
//
// A second kernel has a CTA per pair.  It takes the 16-bit tokens of the pair's ring (mma.sync) while the first kernel ends, waits for it, and merges its
// records with that.
//
// Measured (64 rows x 8 kv heads x (4096 packed + 128 ring) tokens, head_dim 128, 4 query heads per kv head, B200 at 1965 MHz): 123 us with both kernels, 2.7 TB/s; two
// rows of 131072 and 100003 tokens 116 us; 16 rows of 700 to 2050 tokens with 4 query tokens (16 query rows per kv head, head_dim 64) 35 us.  Nothing is saturated: about 940
// instructions per warp and step, 340 of them the levels; issue slots 55 % and logic pipe 59 % used while CTAs run, by 3.7 warps per scheduler (registers: 128 x 512
// threads fill the SM) that wait for one another at three barriers a step; the tensor pipe 7 %, DRAM 33 %.  With 8 query rows 1190 instructions, 2.8 warps
// per scheduler, issue slots 52 %.  What the layout was measured against, for the first of these shapes: warps of special duty with two CTAs of 640 threads to an SM 157 us; the rings inside
// the first kernel 167; a fifth CTA by fewer registers 141; a fifth warp that issues 135; parts in two or three turns 137 and 144; values' levels double-buffered 160.
#include <algorithm>
#include <atomic>

#include "mz_paged.cuh"

namespace mzp {
constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 128, MAX_BATCH = 1024;
constexpr int SPIN_LIMIT = 1000000;              // looks of a wait before it gives up
constexpr int STEP = 2 * MZP_PAGE;
struct Args {
  mz_paged_cache c;
  const uint16_t* query;
  long long qsb, qsl, qsh;
  const int* rows;
  void* out;
  int out_dtype, layer, batch, q_len, q_heads, group;      // group: query heads per kv head
  int qrows, passes;                             // query rows per kv head, and how many passes of NR they take
  int sms, per_sm;                               // the grid, if the machine is full
  int longest;                                   // a row is not taken for longer than its table has room for (and a page, which is then reported)
  float scaling;                                 // times log2(e)
  // workspace: header {CTAs, steps before each entry [batch + 1]}, records
  int* head;
  float2* ml;                                    // [slot][NR] maximum (base 2) and sum
  float* acc;                                    // [slot][NR][D]
  long long pairs, slots;
  int fail_waits;                                // checked build: not 0 = waits run out at once
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
// the 64 codes of a row: a whole sector by one thread, read once
__device__ __forceinline__ void ldg256(uint32_t (&v)[8], const void* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p));
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void fence_operands() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Waits for the phase of this parity.  Who gives up says so before it goes on; the others notice.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* s_failed) {
#ifdef MZ_BOUNDS
  if (*s_failed) return;                         // a test makes every wait run out
#endif
  for (int it = 0; it < SPIN_LIMIT; ++it) {
    if (bar_test(bar, parity)) return;
    if ((it & 63) == 63 && *s_failed) return;
  }
  *s_failed = 1;
}
// shared-memory operand, not swizzled, major along the kept dimension: cores of 8 rows x 16 bytes, 128 bytes apart along the reduction,
// `chunk` bytes apart along the kept dimension
__device__ __forceinline__ uint64_t descriptor(uint32_t sa, uint32_t chunk) {
  return (uint64_t)((sa >> 4) & 0x3FFF) | (128ull >> 4) << 16 | (uint64_t)(chunk >> 4) << 32 | 1ull << 46;
}
// D[128 x N] (+)= A[128 x 32] * B[32 x N], unsigned times signed or unsigned bytes into 32 bits
template <int N, bool SIGNED_B>
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t accumulate) {
  const uint32_t idesc = (2u << 4) | ((SIGNED_B ? 1u : 0u) << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(N / 8) << 17) | (8u << 24);
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
// 31-bit fixed point -> four signed bytes.  (A number that is not negative stands for its four unsigned bytes as it is.)
__device__ __forceinline__ uint32_t digits_of(float x) { return ((uint32_t)__float2int_rn(x) + 0x808080u) ^ 0x808080u; }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// pairs of fp32 operations
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2(float& c0, float& c1, float a0, float a1, float f) {      // c += a * f
  asm("{\n\t.reg .b64 a, c, f;\n\tmov.b64 c, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\tfma.rn.f32x2 c, a, f, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(c0), "+f"(c1) : "f"(a0), "f"(a1), "f"(f));
}
// r = (a * f + b) * c
__device__ __forceinline__ void mul_add2(float& r0, float& r1, float a0, float a1, float b0, float b1, float c0, float c1, float f) {
  asm("{\n\t.reg .b64 a, b, c, f;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tmov.b64 f, {%8, %8};\n\t"
      "fma.rn.f32x2 a, a, f, b;\n\tmul.rn.f32x2 a, a, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r0), "=f"(r1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1), "f"(f));
}

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

// Pairs of 16-bit values: `odd` becomes not zero where one is not finite
template <bool BF>
__device__ __forceinline__ void note_odd(uint32_t& odd, uint32_t w) {
  // x * 0 is a zero, of either sign, or NaN; adding +0 leaves +0 or NaN
  if (BF) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(w), "r"(0u));
  else asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(w), "r"(0u));
}
// takes what is not finite out of a pair
template <bool BF>
__device__ __forceinline__ uint32_t take_odd(uint32_t& w) {
  constexpr uint32_t TOP = BF ? 0x7F80u : 0x7C00u;
  const uint32_t mask = ((w & TOP) == TOP ? 0xFFFFu : 0u) | (((w >> 16) & TOP) == TOP ? 0xFFFF0000u : 0u), taken = w & mask;
  w &= ~mask;
  return taken;
}

// A row's 64 codes -> 64 bytes, four pieces of 16, `chunk` bytes apart.  A selector's top bit asks for the sign of a level, which is zero: so the two
// permutes of a nibble are zero exactly where they are not meant, and their results are or-ed.
__device__ __forceinline__ void expand_row(const uint32_t (&w)[8], const uint4& book, uint32_t dst, uint32_t chunk) {
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
  static constexpr int K_A = 0, V_A = A_BYTES, K_B = 2 * A_BYTES, V_B = K_B + B_BYTES, BOOK = V_B + B_BYTES;
  static constexpr int ALIGN = 1024, TOTAL = BOOK + MZP_BOOKS * MZP_LEVELS + ALIGN;      // (a linker of device code may give the window less)
  static constexpr int N = 8 * NR, TM_S = 0, TM_O = N, TM_COLS = 2 * N;
  static constexpr int CTAS = NR == 4 ? 4 : 3;             // per SM
};
// a step of the line: its pages (-1: not there), pair, list entry, kv head, first query row, tokens, last position that the first query token sees
struct Step { int page0, page1, pair, head, b, r0, count, see; };
// exchange between the warps of a CTA
template <int NR>
struct Exchange {
  alignas(16) Step step[32];                // two blocks of 16 of the CTA's steps; one warp fills a block while the other is worked on
  alignas(16) float base[4][2 * NR];        // constant terms of the logits, by warp
  alignas(16) float fin[4][4 * NR];         // end of a pair: sums of p, constant terms of the output
  alignas(16) float vmax[4][NR];            // largest logit, by warp
  alignas(16) uint32_t top[2][2][4];        // largest T (bits) of the rows, by step parity, side (keys, values) and warp
  float qmax[4][NR];                        // largest |q|, by warp
  unsigned long long bar[3];                // products of the keys, of the values done; end
  int warp_sum[4];
  int first, before;                        // list entry of the CTA's first step, steps of the entries before it
  uint32_t tmem;
  int failed;
};
__device__ __forceinline__ uint32_t max4(const uint32_t* s) {
  const uint4 v = *(const uint4*)s;
  return max(max(v.x, v.y), max(v.z, v.w));
}
template <int N>
__device__ __forceinline__ void load_floats(float (&v)[N], const float* s) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 f = *(const float4*)(s + i);
    v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
  }
}

// How the line of T steps is cut over the CTAs.  The warps that have been on an SM for longest come first at its schedulers: with equal parts an SM's four CTAs
// ended after 80, 88, 99 and 111 us (two rows of 131072 and 100003 tokens).  CTAs start in their order, one on each SM before the next ones, so where there
// is enough to share out the k-th on an SM gets 16 + per_sm - 1 - 2 k sixteenths of an equal part.  Otherwise parts are equal, and no CTA is empty.
struct Cut {
  long long T, W;
  int sms, per_sm;                               // per_sm 0: equal parts
  __device__ __forceinline__ Cut(const Args& p, long long steps, int grid) : T(steps), sms(p.sms), per_sm(0) {
    W = min((long long)grid, T);
    if (grid == p.sms * p.per_sm && T >= 2 * W) per_sm = p.per_sm;
  }
  __device__ __forceinline__ long long start(int cta) const {          // the first step of a CTA
    if (per_sm == 0) return T * cta / W;
    const int k = cta / sms;
    return T * ((long long)sms * (k * (16 + per_sm - k)) + (long long)(cta - k * sms) * (15 + per_sm - 2 * k)) / (16ll * per_sm * sms);
  }
  __device__ __forceinline__ int owner(long long step) const {         // the CTA that has a step
    if (per_sm == 0) return (int)(((step + 1) * W - 1) / T);
    const long long v = ((step + 1) * (16ll * per_sm * sms) - 1) / T;
    int k = 0;
    while (k + 1 < per_sm && v >= (long long)sms * ((k + 1) * (16 + per_sm - (k + 1)))) ++k;
    return k * sms + (int)((v - (long long)sms * (k * (16 + per_sm - k))) / (15 + per_sm - 2 * k));
  }
};

// row and length of a list entry; a row that is not there is empty
__device__ __forceinline__ int length_of(const Args& p, int b, int& row) {
  row = p.rows ? p.rows[b] : b;
  return row < 0 || row >= p.c.rows ? 0 : max(0, min(p.c.lengths[row], p.longest));
}

template <int D, bool BF, int NR>
__global__ void __launch_bounds__(THREADS, (Smem<D, NR>::CTAS)) attention_kernel(const Args p, const uint8_t* __restrict__ book_table) {
  using S = Smem<D, NR>;
  constexpr int DT = BF ? MZ_BF16 : MZ_F16;
  constexpr int PB = 72 * D;                     // page bytes per kv head
  constexpr int RPT = D / 64;                    // rows of codes per thread, side and step
  extern __shared__ uint8_t window[];
  uint8_t* smem = window + (S::ALIGN - smem_u32(window) % S::ALIGN) % S::ALIGN;
  __shared__ Exchange<NR> x;
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(smem), sbook = sbase + S::BOOK;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t k_done = smem_u32(x.bar), v_done = k_done + 8, b_end = k_done + 16;
  if (tid == 0) {
    x.failed = p.fail_waits;
    bar_init(k_done, 1); bar_init(v_done, 1); bar_init(b_end, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  ((uint4*)(smem + S::BOOK))[tid] = ((const uint4*)book_table)[tid];
  static_assert(THREADS == MZP_BOOKS * MZP_LEVELS / 16, "one piece of the books per thread");

  // ---- the line of steps
  const int kp_all = c.kv_heads * p.passes, G = gridDim.x, cta = blockIdx.x;
  auto steps_of = [&](int b, int& row, int& len) {
    len = length_of(p, b, row);
    return (mzp_packed(len, c.residual) + STEP - 1) / STEP;
  };
  int total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
    int row, len;
    const int st = b0 + tid < p.batch ? steps_of(b0 + tid, row, len) : 0;
    total += st;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) x.warp_sum[warp] = total;
  __syncthreads();
  total = (x.warp_sum[0] + x.warp_sum[1]) + (x.warp_sum[2] + x.warp_sum[3]);
  const long long T = (long long)total * kp_all;
  const Cut cut(p, T, G);
  const long long f0 = cta < cut.W ? cut.start(cta) : 0;
  const int n = cta < cut.W ? (int)(cut.start(cta + 1) - f0) : 0;
  if (cta == 0 && tid == 0) p.head[0] = G;
  // the list entry of the first step (CTA 0 writes down all of them)
  for (int b0 = 0, before = 0; b0 < p.batch; b0 += THREADS) {
    int row, len;
    const int b = b0 + tid, st = b < p.batch ? steps_of(b, row, len) : 0;
    int scan = st;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += y; }
    __syncthreads();
    if (lane == 31) x.warp_sum[warp] = scan;
    __syncthreads();
    int at = before + scan - st;
#pragma unroll
    for (int w = 0; w < 4; ++w) { const int t = x.warp_sum[w]; if (w < warp) at += t; before += t; }
    if (n > 0 && (long long)at * kp_all <= f0 && f0 < (long long)(at + st) * kp_all) { x.first = b; x.before = at; }
    if (cta == 0 && b < p.batch) p.head[2 + b] = at + st;
    if (before * (long long)kp_all > f0 && cta != 0) break;          // the same for all threads
  }
  if (cta == 0 && tid == 0) p.head[1] = 0;
  if (n == 0) return;

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tm_before();
  }
  __syncthreads();
  tm_after();
  const uint32_t tmem = x.tmem;
  // What the CTA's steps at .. at + 15 are, one per lane: the entries from the CTA's first one on are looked through, 32 at a time
  auto plan = [&](int at) {
    const int it = at + lane;
    const long long f = f0 + it;
    bool open = lane < 16 && it < n;
    Step s = {-1, -1, 0, 0, 0, 0, 0, 0};
    int before = x.before;
    for (int b0 = x.first; b0 < p.batch && __any_sync(0xffffffffu, open); b0 += 32) {
      int row = 0, len = 0;
      const int st = b0 + lane < p.batch ? steps_of(b0 + lane, row, len) : 0;
      int scan = st;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += y; }
      const int start = before + scan - st;      // of entry b0 + lane
      before += __shfl_sync(0xffffffffu, scan, 31);
      int k = 0;                                 // the last entry that starts at or before f
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) if ((long long)__shfl_sync(0xffffffffu, start, k + o) * kp_all <= f) k += o;
      const int steps = __shfl_sync(0xffffffffu, st, k), first = __shfl_sync(0xffffffffu, start, k), its_row = __shfl_sync(0xffffffffu, row, k);
      const int its_len = __shfl_sync(0xffffffffu, len, k);
      if (open && f < (long long)before * kp_all) {
        open = false;
        const int rem = (int)(f - (long long)first * kp_all), kp = rem / steps, step = rem - kp * steps, pages = mzp_packed(its_len, c.residual) / MZP_PAGE;
        s.b = b0 + k;
        s.pair = s.b * kp_all + kp;
        s.head = kp / p.passes;
        s.r0 = (kp - s.head * p.passes) * NR;
        s.count = min(STEP, pages * MZP_PAGE - step * STEP);
        s.see = its_len - p.q_len + s.r0 / p.group - step * STEP;
        int id[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          id[w] = -1;
          if (2 * step + w < pages) {
            id[w] = 2 * step + w < c.width ? c.block_table[(long long)its_row * c.width + 2 * step + w] : -1;
            if (id[w] < 0 || id[w] >= c.pages) { id[w] = -1; atomicOr(c.status, MZ_PAGED_BAD_INDEX); }
          }
        }
        s.page0 = id[0]; s.page1 = id[1];
      }
    }
    if (lane < 16) x.step[it & 31] = s;
  };
  if (warp < 2) plan(16 * warp);
  __syncthreads();

  const int r = tid, blk = r >> 6, in_page = r & 63;         // key channel, token, output channel
  const int ch = D == 128 ? r : in_page;
  const uint8_t* store = (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer;
  const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
  uint32_t kc[RPT][8], vc[RPT][8], kw[RPT], vw[RPT];         // codes and words of the next step to work on
  // a page that is not there has T = 0
  auto load_keys = [&](const Step& s) {
    const uint8_t* base = store + s.head * PB;
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
      const int page = (D == 128 ? j : blk) ? s.page1 : s.page0;
      const uint8_t* at = base + (long long)page * c.store_stride_page;
      kw[j] = page >= 0 ? __ldg((const uint32_t*)(at + 32 * D + 4 * ch)) : 0u;
      if (page >= 0) ldg256(kc[j], at + 32 * ch);
    }
  };
  auto load_values = [&](const Step& s) {
    const int page = blk ? s.page1 : s.page0;
    const uint8_t* at = store + s.head * PB + (long long)page * c.store_stride_page + 36 * D;
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
      vw[j] = page >= 0 ? __ldg((const uint32_t*)(at + 32 * D + 4 * (in_page * RPT + j))) : 0u;
      if (page >= 0) ldg256(vc[j], at + 32 * (in_page * RPT + j));
    }
  };
  // the largest T of a step's rows scales its fixed point
  auto publish = [&](int it) {
    uint32_t kt = 0, vt = 0;
#pragma unroll
    for (int j = 0; j < RPT; ++j) { kt = max(kt, kw[j] & 0xffffu); vt = max(vt, vw[j] & 0xffffu); }
    kt = warp_max_u32(kt);
    vt = warp_max_u32(vt);
    if (lane == 0) { x.top[it & 1][0][warp] = kt; x.top[it & 1][1][warp] = vt; }
  };
#pragma unroll
  for (int j = 0; j < RPT; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) kc[j][k] = vc[j][k] = 0;
  {
    const Step s = x.step[0];
    load_keys(s);
    load_values(s);
  }
  const uint64_t ka = descriptor(sbase + S::K_A, S::CHUNK), kb = descriptor(sbase + S::K_B, S::CHUNK);
  const uint64_t va = descriptor(sbase + S::V_A, S::CHUNK), vb = descriptor(sbase + S::V_B, S::CHUNK);

  float q[NR], qs[NR], m[NR], l[NR], o[NR], base_v[RPT][NR];
  float vunit = 0.f;
  int pair = -1;
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; o[i] = 0.f; }
#pragma unroll
    for (int j = 0; j < RPT; ++j)
#pragma unroll
      for (int i = 0; i < NR; ++i) base_v[j][i] = 0.f;
  };
  // the values' products of step `done`
  auto take_output = [&](int done) {
    bar_wait(v_done, done & 1, &x.failed);
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
    constexpr int NV = NR * (RPT == 2 ? 4 : 2);              // l, constant terms (and padding)
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
    if ((lane & (32 / NV - 1)) == 0) x.fin[warp][index] = sum;
    float* halves = (float*)(smem + S::V_B);                 // D = 64: the second page's part; the products that read this are done
    if (D == 64 && r >= 64) {
#pragma unroll
      for (int i = 0; i < NR; ++i) halves[(r - 64) * NR + i] = o[i];
    }
    __syncthreads();
    const long long slot = (long long)cta + pair;
    const bool bad = *(volatile int*)&x.failed != 0, inside = MZ_IN_BOUNDS(slot, p.slots, 20);
    if (inside && (D == 128 || r < 64)) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int at = (1 + (D == 128 ? blk : 0)) * NR + i;
        float out = o[i] + ((x.fin[0][at] + x.fin[1][at]) + (x.fin[2][at] + x.fin[3][at]));
        if (D == 64) out += halves[r * NR + i];
        p.acc[(slot * NR + i) * D + r] = out;
      }
    }
    if (inside && r < NR) {
      const float sum_l = (x.fin[0][r] + x.fin[1][r]) + (x.fin[2][r] + x.fin[3][r]);
      float top = m[0];
#pragma unroll
      for (int i = 1; i < NR; ++i) top = r == i ? m[i] : top;
      p.ml[slot * NR + r] = bad ? make_float2(INFINITY, __int_as_float(0x7fffffff)) : make_float2(top, sum_l);
    }
    __syncthreads();                                         // fin and halves are free again
  };
  publish(0);
  __syncthreads();
  for (int it = 0; it < n; ++it) {
    const Step s = x.step[it & 31];
    const bool fresh = s.pair != pair;
    if (fresh) {
      if (pair >= 0) {
        take_output(it - 1);
        write_record();
      }
      pair = s.pair;
      reset();
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        q[i] = 0.f;
        if (s.r0 + i < p.qrows) {
          const int ql = (s.r0 + i) / p.group, h = s.head * p.group + (s.r0 + i) % p.group;
          q[i] = MzType<DT>::load(p.query, (long long)s.b * p.qsb + ql * p.qsl + h * p.qsh + ch);
        }
      }
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        // as bits, so that a NaN is the largest
        const uint32_t top = warp_max_u32(__float_as_uint(fabsf(q[i])));
        if (lane == 0) x.qmax[warp][i] = __uint_as_float(top);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max(top, __float_as_uint(x.qmax[w][i]));
        const int e = max((int)(top >> 23) - 126, -60), e1 = e >> 1, e2 = e - e1;        // |q| < 2^e, taken off in two factors
        const bool wild = top >= 0x7f800000u;                          // infinity or NaN: the row's logits are NaN
        q[i] = wild ? 0.f : q[i] * pow2(-e1) * pow2(-e2);
        qs[i] = wild ? __int_as_float(0x7fffffff) : pow2(e1) * p.scaling * pow2(e2);
      }
    }
    // ---- keys: levels and folds (the products of the last step's keys are done)
    const int ek = (int)(max4(x.top[it & 1][0]) >> 10) - 14, ev = (int)(max4(x.top[it & 1][1]) >> 10) - 14;      // T < 2^(exponent field - 14)
    {
      const float up = pow2(30 - ek);
      float base[RPT * NR];
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const MzpRow row = mzp_row(kw[j]);
        const int b2 = D == 128 ? j : blk;
        const float ts = row.t * up, cz = fmaf(row.t, (float)row.z * -0.03125f, row.a);
#pragma unroll
        for (int i = 0; i < NR; i += 4) {
          float f[4] = {0.f, 0.f, 0.f, 0.f};
          fma2(f[0], f[1], q[i], q[i + 1], ts);
          fma2(f[2], f[3], q[i + 2], q[i + 3], ts);
          sts128(sbase + S::K_B + (b2 * (NR / 4) + i / 4) * S::CHUNK + ch * 16, digits_of(f[0]), digits_of(f[1]), digits_of(f[2]), digits_of(f[3]));
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) base[j * NR + i] = q[i] * cz;
        expand_row(kc[j], book128(sbook + row.z * 16), sbase + S::K_A + b2 * 4 * S::CHUNK + ch * 16, S::CHUNK);
      }
      int index;
      const float sum = warp_sums<RPT * NR>(base, lane, index);
      if ((lane & (32 / (RPT * NR) - 1)) == 0) x.base[warp][index] = sum;
    }
    fence_operands();
    tm_before();
    __syncthreads();
    if (tid == 96 && !*(volatile int*)&x.failed) {
      tm_after();
#pragma unroll
      for (int k = 0; k < D / 32; ++k) umma<S::N, true>(tmem + S::TM_S, ka + k * (512 >> 4), kb + k * (512 >> 4), k > 0);
      umma_commit(k_done);
    }
    if (warp == 0 && (it & 15) == 0 && it > 0) plan(it + 16);
    const Step next = x.step[(it + 1) & 31];     // beyond the CTA's last step: pages that are not there, or a step that nobody takes
    if (it + 1 < n) load_keys(next);
    // ---- values: the output so far, then levels while the products of the keys run
    if (it > 0 && !fresh) take_output(it - 1);
    const float up = pow2(30 - ev);
    float ts[RPT], cz[RPT];
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
      const MzpRow row = mzp_row(vw[j]);
      ts[j] = row.t * up;
      cz[j] = fmaf(row.t, (float)row.z * -0.03125f, row.a);
      expand_row(vc[j], book128(sbook + row.z * 16), sbase + S::V_A + (D == 128 ? j : blk) * 4 * S::CHUNK + (D == 128 ? r : in_page) * 16, S::CHUNK);
    }
    if (it + 1 < n) load_values(next);
    // ---- logits
    float base[NR];
    if (D == 128) {
      float b[4][NR];
#pragma unroll
      for (int w = 0; w < 4; ++w) load_floats(b[w], x.base[w] + blk * NR);
#pragma unroll
      for (int i = 0; i < NR; ++i) base[i] = (b[0][i] + b[1][i]) + (b[2][i] + b[3][i]);
    } else {
      float b[2][NR];
#pragma unroll
      for (int w = 0; w < 2; ++w) load_floats(b[w], x.base[2 * blk + w]);
#pragma unroll
      for (int i = 0; i < NR; ++i) base[i] = b[0][i] + b[1][i];
    }
    bar_wait(k_done, it & 1, &x.failed);
    tm_after();
    const float kunit = pow2(ek - 35);
    float w[NR];
#pragma unroll
    for (int i = 0; i < NR; i += 4) {
      int a[16];
      tm_ld16(lanes + S::TM_S + blk * (4 * NR) + 4 * i, a);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[i + k] = number_of(a + 4 * k);
    }
#pragma unroll
    for (int i = 0; i < NR; i += 2) mul_add2(w[i], w[i + 1], w[i], w[i + 1], base[i], base[i + 1], qs[i], qs[i + 1], kunit);
    if (s.count < STEP) {
#pragma unroll
      for (int i = 0; i < NR; ++i) if (r >= s.count) w[i] = -INFINITY;
    }
    if (s.see < s.count - 1) {                               // not every query sees all of the step
#pragma unroll
      for (int i = 0; i < NR; ++i) if (r > s.see + (s.r0 + i) / p.group - s.r0 / p.group) w[i] = -INFINITY;
    }
    // ---- running maximum
    float fix[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) fix[i] = warp_max(w[i]);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NR; i += 4) *(float4*)&x.vmax[warp][i] = make_float4(fix[i], fix[i + 1], fix[i + 2], fix[i + 3]);
    }
    __syncthreads();
    bool moved = false;
    {
      float v[4][NR];
#pragma unroll
      for (int k = 0; k < 4; ++k) load_floats(v[k], x.vmax[k]);
#pragma unroll
      for (int i = 0; i < NR; ++i) fix[i] = fmaxf(fmaxf(v[0][i], v[1][i]), fmaxf(v[2][i], v[3][i]));
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      moved |= fix[i] > m[i];
      fix[i] = fmaxf(m[i], fix[i]);
      w[i] = ex2(w[i] - (fix[i] == -INFINITY ? 0.f : fix[i]));
    }
    if (moved) {                                             // the same for all threads
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float f = ex2(m[i] - (fix[i] == -INFINITY ? 0.f : fix[i]));
        m[i] = fix[i];
        o[i] *= f; l[i] *= f;
#pragma unroll
        for (int j = 0; j < RPT; ++j) base_v[j][i] *= f;
      }
    }
    vunit = pow2(ev - 35);
#pragma unroll
    for (int i = 0; i < NR; i += 2) add2(l[i], l[i + 1], w[i], w[i + 1]);
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
      const int b2 = D == 128 ? j : blk, at = D == 128 ? r : in_page;
#pragma unroll
      for (int i = 0; i < NR; i += 2) fma2(base_v[j][i], base_v[j][i + 1], w[i], w[i + 1], cz[j]);
#pragma unroll
      for (int i = 0; i < NR; i += 4) {
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        fma2(f[0], f[1], w[i], w[i + 1], ts[j]);
        fma2(f[2], f[3], w[i + 2], w[i + 3], ts[j]);
        sts128(sbase + S::V_B + (b2 * (NR / 4) + i / 4) * S::CHUNK + at * 16, __float2int_rn(f[0]), __float2int_rn(f[1]), __float2int_rn(f[2]),
               __float2int_rn(f[3]));
      }
    }
    publish(it + 1);
    fence_operands();
    tm_before();
    __syncthreads();
    if (tid == 32 && !*(volatile int*)&x.failed) {
      tm_after();
#pragma unroll
      for (int k = 0; k < D / 32; ++k) umma<S::N, false>(tmem + S::TM_O, va + k * (512 >> 4), vb + k * (512 >> 4), k > 0);
      umma_commit(v_done);
    }
  }
  take_output(n - 1);
  write_record();
  if (x.failed && (tid & 63) == 32) {             // products in flight end before their memory goes back
    umma_commit(b_end);
    for (int k = 0; k < SPIN_LIMIT && !bar_test(b_end, 0); ++k) {}
  }
  tm_before();
  __syncthreads();
  if (warp == 0) {
    tm_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TM_COLS));
  }
}

// One pair per CTA of eight warps; 23 us alone for 512 pairs of 128 ring tokens (36 MB; it waits for loads), of which about 10 us show behind the first kernel.  Rings: a warp
// takes 16 tokens at a time, and (D = 128) 64 of the channels of the output; A = keys [token][channel], B = queries; A = values [channel][token], B = p in parts of 16 bits, as many as fp32 has bits.  Products go to fresh accumulators that are added in round-to-nearest:
// the tensor cores truncate their running sums.  Then a thread has a channel, and every second query row.
constexpr int END_THREADS = 256;                 // two CTAs to an SM; three have 80 registers, which spill: 64 x 8 x 4224 tokens 129 instead of 123 us
template <int D, bool BF, int NR>
__global__ void __launch_bounds__(END_THREADS, 2) finish_kernel(const Args p) {
  constexpr int HALVES = D / 64, STREAMS = 8 / HALVES, GROUPS = END_THREADS / D, ROWS = NR / GROUPS;      // D = 64: four groups
  __shared__ float s_part[STREAMS][NR][D], s_m[STREAMS][NR], s_l[STREAMS][NR];
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const long long pair = blockIdx.x;
  const int kp_all = c.kv_heads * p.passes, b = (int)(pair / kp_all), kp = (int)(pair - (long long)b * kp_all), head = kp / p.passes;
  const int r0 = (kp - head * p.passes) * NR;
  int row;
  const int len = length_of(p, b, row), packed = mzp_packed(len, c.residual), tokens = len - packed;
  if ((row < 0 || row >= c.rows) && tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
  const int half = warp % HALVES, stream = warp / HALVES;
  if (tokens > 0) {
    const int see0 = tokens - p.q_len;           // query token l sees the ring's tokens up to see0 + l
    const int l_first = r0 / p.group, l_last = (min(r0 + NR, p.qrows) - 1) / p.group;      // the pass's query tokens
    const uint16_t* ring_k = (const uint16_t*)c.tail + (long long)p.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)head * c.ring * D;
    const uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D + half * 64;
    const int ring0 = packed % c.ring;
    auto place = [&](int i) { const int at = ring0 + i; return (at >= c.ring ? at - c.ring : at) * D; };      // i < tokens <= ring
    // query row r0 + g; rows that are not there are zero
    const int qr = r0 + g;
    const bool on = g < NR && qr < p.qrows;
    const uint16_t* query = p.query + (long long)b * p.qsb + (long long)(qr / p.group) * p.qsl + (long long)(head * p.group + qr % p.group) * p.qsh + 8 * t;
    uint4 qf[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      qf[k] = make_uint4(0, 0, 0, 0);
      if (on) qf[k] = *(const uint4*)(query + 32 * k);
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    for (int i0 = stream * 16; i0 < tokens; i0 += STREAMS * 16) {
      uint4 v[4];
      // what is not there is read as zero
      auto load_values = [&](int see) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + 2 * t + (k & 1) + 8 * (k >> 1);
          v[k] = make_uint4(0, 0, 0, 0);
          if (i <= see) v[k] = *(const uint4*)(ring_v + place(i) + 8 * g);
        }
      };
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      {
        const uint16_t* ka = ring_k + place(min(i0 + g, tokens - 1)) + 8 * t;
        const uint16_t* kb = ring_k + place(min(i0 + g + 8, tokens - 1)) + 8 * t;
        uint4 va[D / 32], vb[D / 32];
#pragma unroll
        for (int k = 0; k < D / 32; ++k) { va[k] = *(const uint4*)(ka + 32 * k); vb[k] = *(const uint4*)(kb + 32 * k); }
        load_values(min(see0 + l_last, tokens - 1));
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
          mma16<BF>(c0, va[k].x, vb[k].x, va[k].y, vb[k].y, qf[k].x, qf[k].y);
          mma16<BF>(c1, va[k].z, vb[k].z, va[k].w, vb[k].w, qf[k].z, qf[k].w);
          add2(c0[0], c0[1], c1[0], c1[1]); add2(c0[2], c0[3], c1[2], c1[3]);
          add2(s[0], s[1], c0[0], c0[1]); add2(s[2], s[3], c0[2], c0[3]);
        }
      }
      // s[0], s[1]: token g, columns (query rows) 2t, 2t + 1; s[2], s[3]: token g + 8
      float fix[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int last = min(see0 + (r0 + 2 * t + j) / p.group, tokens - 1);
        s[j] = i0 + g <= last ? s[j] * p.scaling : -INFINITY;
        s[2 + j] = i0 + g + 8 <= last ? s[2 + j] * p.scaling : -INFINITY;
        float top = fmaxf(s[j], s[2 + j]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float m_new = fmaxf(m[j], top), ref = m_new == -INFINITY ? 0.f : m_new;
        fix[j] = ex2(m[j] - ref);
        m[j] = m_new;
        s[j] = ex2(s[j] - ref);
        s[2 + j] = ex2(s[2 + j] - ref);
        l[j] = l[j] * fix[j] + s[j] + s[2 + j];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { o[i][0] *= fix[0]; o[i][1] *= fix[1]; o[i][2] *= fix[0]; o[i][3] *= fix[1]; }
      // p in parts, transposed: column g, tokens 2t, 2t + 1 ([0]) and 2t + 8, 2t + 9 ([1]).  Three of 8 bits or two of 11 leave less than fp32's own
      // rounding; f16 has p times 2^15, so that a second part does not end at its smallest numbers
      constexpr int PARTS = BF ? 3 : 2;
      constexpr uint32_t ONE16 = BF ? 0x3F80u : 0x3C00u;
      constexpr float P_SCALE = BF ? 1.0f : 32768.0f, P_UNIT = 1.0f / P_SCALE;
      uint32_t part[PARTS][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p0 = s[2 * h] * P_SCALE, p1 = s[2 * h + 1] * P_SCALE;
#pragma unroll
        for (int x = 0; x < PARTS; ++x) {
          uint32_t w;
          float2 f;
          if (BF) {
            const __nv_bfloat162 b2 = __floats2bfloat162_rn(p0, p1);
            w = *reinterpret_cast<const uint32_t*>(&b2);
            f = __bfloat1622float2(b2);
          } else {
            const __half2 h2 = __floats2half2_rn(p0, p1);
            w = *reinterpret_cast<const uint32_t*>(&h2);
            f = __half22float2(h2);
          }
          p0 -= f.x;
          p1 -= f.y;
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(part[x][h]) : "r"(w));
        }
      }
      // A token that only later queries see must not bring a NaN to a product with p = 0: what no query of the pass sees is not loaded, and where a tile has
      // tokens that only some of the queries see, each of the queries' tokens takes its turn with what it sees, and only its columns are added
      const bool apart = i0 + 15 > see0 + l_first && l_last > l_first;
      for (int turn = 0; turn <= (apart ? l_last - l_first : 0); ++turn) {
        if (apart) load_values(min(see0 + l_first + turn, tokens - 1));
        const bool mine0 = !apart || (r0 + 2 * t) / p.group == l_first + turn, mine1 = !apart || (r0 + 2 * t + 1) / p.group == l_first + turn;
        uint32_t w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
        uint32_t w2[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, w3[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
        // An infinite value is not a matter of p's parts (a lower one may be zero or negative): values that are not finite are taken out and meet a 1 where
        // p is not zero, in a product of their own
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) { note_odd<BF>(odd, w0[k]); note_odd<BF>(odd, w1[k]); note_odd<BF>(odd, w2[k]); note_odd<BF>(odd, w3[k]); }
        if (__any_sync(0xffffffffu, odd != 0)) {
          uint32_t one[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = (s[2 * h] > 0.f ? ONE16 : 0u) | (s[2 * h + 1] > 0.f ? ONE16 << 16 : 0u);
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(one[h]) : "r"(w));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x0 = take_odd<BF>(w0[k]), x1 = take_odd<BF>(w1[k]), x2 = take_odd<BF>(w2[k]), x3 = take_odd<BF>(w3[k]);
            float c4[4] = {0.f, 0.f, 0.f, 0.f};
            mma16<BF>(c4, prmt(x0, x1, 0x5410u), prmt(x0, x1, 0x7632u), prmt(x2, x3, 0x5410u), prmt(x2, x3, 0x7632u), one[0], one[1]);
            if (mine0) { o[k][0] += c4[0]; o[k][2] += c4[2]; }
            if (mine1) { o[k][1] += c4[1]; o[k][3] += c4[3]; }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // rows g / g + 8 = channels 8g + 2k / 8g + 2k + 1
          const uint32_t a0 = prmt(w0[k], w1[k], 0x5410u), a1 = prmt(w0[k], w1[k], 0x7632u);
          const uint32_t a2 = prmt(w2[k], w3[k], 0x5410u), a3 = prmt(w2[k], w3[k], 0x7632u);
          float c4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = PARTS - 1; x >= 0; --x) mma16<BF>(c4, a0, a1, a2, a3, part[x][0], part[x][1]);
          if (mine0) { o[k][0] = fmaf(c4[0], P_UNIT, o[k][0]); o[k][2] = fmaf(c4[2], P_UNIT, o[k][2]); }
          if (mine1) { o[k][1] = fmaf(c4[1], P_UNIT, o[k][1]); o[k][3] = fmaf(c4[3], P_UNIT, o[k][3]); }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], off);
      if (2 * t + j < NR) {
        float* dst = &s_part[stream][2 * t + j][half * 64 + 8 * g];
#pragma unroll
        for (int k = 0; k < 4; ++k) *(float2*)(dst + 2 * k) = make_float2(o[k][j], o[k][2 + j]);
        if (g == 0 && half == 0) { s_m[stream][2 * t + j] = m[j]; s_l[stream][2 * t + j] = l[j]; }
      }
    }
  }
  __syncthreads();
  // ---- this thread: channel d of query rows i0, i0 + GROUPS, ...
  const int d = tid % D, i0 = tid / D;
  float m[ROWS], l[ROWS], a[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) { m[i] = -INFINITY; l[i] = 0.f; a[i] = 0.f; }
  auto take = [&](int i, float2 ml, float v) {
    const float top = fmaxf(m[i], ml.x), ref = top == -INFINITY ? 0.f : top;
    const float f = ex2(m[i] - ref), h = ex2(ml.x - ref);
    l[i] = l[i] * f + ml.y * h;
    a[i] = a[i] * f + v * h;
    m[i] = top;
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");         // the first kernel's records are written
  const long long before = p.head[1 + b], steps = p.head[2 + b] - before;
  if (steps > 0) {
    const Cut cut(p, (long long)p.head[1 + p.batch] * kp_all, p.head[0]);
    const long long s0 = before * kp_all + kp * steps, first = cut.owner(s0), last = cut.owner(s0 + steps - 1);
    for (long long c0 = first; c0 <= last; c0 += 4) {
      float2 ml[4][ROWS];
      float v[4][ROWS];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const long long slot = (min(c0 + k, last) + pair) * NR + i0 + i * GROUPS;
          ml[k][i] = p.ml[slot];
          v[k][i] = p.acc[slot * D + d];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) if (c0 + k <= last) take(i, ml[k][i], v[k][i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int at = i0 + i * GROUPS, qr = r0 + at;
    if (tokens > 0) {
#pragma unroll
      for (int k = 0; k < STREAMS; ++k) take(i, make_float2(s_m[k][at], s_l[k][at]), s_part[k][at][d]);
    }
    if (qr < p.qrows) {
      const float out = l[i] == 0.f ? 0.f : a[i] / l[i];
      const int ql = qr / p.group, h = head * p.group + qr % p.group;
      mz_store_from_float(p.out, (((long long)b * p.q_len + ql) * p.q_heads + h) * D + d, out, p.out_dtype);
    }
  }
}

template <int D, bool BF, int NR>
int launch(const Args& p, const uint8_t* book, int G, cudaStream_t st) {
  auto kern = attention_kernel<D, BF, NR>;
  using S = Smem<D, NR>;
  static std::atomic<unsigned> ready[8];         // a bit per device: its limits are set
  int dev = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  const bool known = dev < 256 && (ready[dev >> 5].load(std::memory_order_relaxed) >> (dev & 31) & 1u);
  if (!known) {
    MZ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
    MZ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (dev < 256) ready[dev >> 5].fetch_or(1u << (dev & 31), std::memory_order_relaxed);
  }
  kern<<<G, THREADS, S::TOTAL, st>>>(p, book);
  MZ_LAUNCH_CHECK("paged attention");
  // The second kernel starts while the first one ends.  (Not so the first one while the second of the call before ends: an SM does not change its split
  // of L1 and shared memory while a CTA runs on it, and four of these CTAs then do not fit.)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)p.pairs);
  cfg.blockDim = dim3(END_THREADS);
  MZ_CUDA(cudaLaunchKernelEx(&cfg, finish_kernel<D, BF, NR>, p));
  MZ_LAUNCH_CHECK("paged attention end");
  return MZ_OK;
}

struct Shape { int nr, passes, sms, per_sm, G; long long pairs; size_t head_bytes, slots, bytes; };
int shape_of(const mz_paged_cache* c, int batch, int q_len, int q_heads, Shape* s) {
  MZ_REQUIRE(batch >= 0 && batch <= MAX_BATCH, "batch %d (at most %d)", batch, MAX_BATCH);
  MZ_REQUIRE(q_len >= 1 && q_heads >= 1 && q_heads % c->kv_heads == 0, "q_len %d, q_heads %d of %d kv heads", q_len, q_heads, c->kv_heads);
  const long long qrows = (long long)q_heads / c->kv_heads * q_len;
  MZ_REQUIRE(qrows <= 1 << 20, "%lld query rows per kv head", qrows);
  int sms = 0, rc = mz_paged_sms(&sms);
  if (rc != MZ_OK) return rc;
  // 8 query rows to a step where there are more than 4: 64 x 8 x 4224 tokens, head_dim 128, with 5 / 8 of them 163 / 167 us against 235 / 239 in two passes of 4, with 12
  // 300 against 341 in three; with 1 / 4 of them 157 / 161 us against 130 / 134 in a step of 4.  The same order for two long rows (138 / 189, 134 / 112) and at head_dim 64;
  // one row of 500 tokens takes 17 to 21 us either way.
  s->nr = qrows <= 4 ? 4 : 8;
  s->passes = (int)((qrows + s->nr - 1) / s->nr);
  s->pairs = (long long)batch * c->kv_heads * s->passes;
  MZ_REQUIRE(s->pairs < (1ll << 31) - s->nr * 2048, "too many query rows for one call");
  s->sms = sms;
  s->per_sm = s->nr == 4 ? 4 : 3;
  s->G = sms * s->per_sm;
  MZ_REQUIRE((long long)batch * (c->width + 2) <= 1ll << 31, "%d rows of %d pages are too many for one call", batch, c->width);
  // a CTA costs its start (592 of them 6 us): no more than there can be steps
  const long long most = s->pairs * ((c->width + 1) / 2);
  if (s->G > most) s->G = most < 1 ? 1 : (int)most;
  s->head_bytes = ((2 + (size_t)batch) * sizeof(int) + 127) / 128 * 128;
  s->slots = (size_t)s->G + (size_t)s->pairs;
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
  MZ_REQUIRE((uintptr_t)args->query % 16 == 0 && (args->q_stride_b | args->q_stride_l | args->q_stride_h) % 8 == 0,
             "query must be 16-byte aligned with strides in multiples of 8 elements");
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
  p.sms = s.sms; p.per_sm = s.per_sm;
  p.longest = (int)std::min<long long>(0x7fffffff - mzp::STEP, cache->residual + (cache->width + 2ll) * MZP_PAGE - 1);
  p.scaling = args->scaling * mzp::LOG2E;
  p.head = (int*)args->workspace;
  p.acc = (float*)((uint8_t*)args->workspace + s.head_bytes);
  p.ml = (float2*)(p.acc + s.slots * s.nr * cache->head_dim);
  p.pairs = s.pairs;
  p.slots = (long long)s.slots;
  p.fail_waits = mz_waits_fail();
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = cache->kv_dtype == MZ_BF16;
#define MZP_GO(D, NR) return bf ? mzp::launch<D, true, NR>(p, book, s.G, st) : mzp::launch<D, false, NR>(p, book, s.G, st)
  if (cache->head_dim == 128) { if (s.nr == 4) MZP_GO(128, 4); MZP_GO(128, 8); }
  if (s.nr == 4) MZP_GO(64, 4);
  MZP_GO(64, 8);
#undef MZP_GO
}
