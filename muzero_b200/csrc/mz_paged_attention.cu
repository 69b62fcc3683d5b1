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
// finds there; a CTA leaves a record (m, l, out) per pair that it met, slot = CTA + pair.  The 16-bit tokens of the rings are shared out over the CTAs
// as well; their records follow.  A second kernel merges a pair's records.
//
// A CTA is five groups of four warps, two CTAs to an SM; what a group does in a step is short, and the groups are up to two steps apart:
//   key levels     expand the keys' codes                                   (thread = channel)
//   key folds      scale the queries to fixed point, sum the constant terms (thread = channel)
//   value levels   expand the values' codes                                 (thread = token)
//   softmax        logits, probabilities to fixed point, running output     (thread = token, then channel)
//   service        a warp that walks the line, looks pages up and has them copied to shared memory (bulk copies: keys two steps ahead, values three), one
//                  that issues MMAs, two that take the rings' 16-bit tokens from memory on mma.sync, in the gaps of the others
// mbarriers tie them together.  Every wait is bounded; one that runs out makes the CTA's records NaN and ends its MMAs.
#include "mz_paged.cuh"

namespace mzp {
constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 640, MAX_BATCH = 1024, CTAS_PER_SM = 2;
constexpr int SPIN_LIMIT = 1000000;              // looks of a wait before it gives up; afterwards one look each
// registers of the groups: they share what the 640 threads are launched with, 48 each
template <int NR>
struct Regs {
  static constexpr int LEVELS = 32, KEY_FOLDS = NR == 4 ? 48 : 56, SOFTMAX = NR == 4 ? 72 : 88, SERVICE = NR == 4 ? 56 : 32;
  static_assert(2 * LEVELS + KEY_FOLDS + SOFTMAX + SERVICE <= 5 * 48, "register split");
};
constexpr int STEP = 2 * MZP_PAGE;

struct Args {
  mz_paged_cache c;
  const uint16_t* query;
  long long qsb, qsl, qsh;
  const int* rows;
  void* out;
  int out_dtype, layer, batch, q_len, q_heads, group;      // group: query heads per kv head
  int qrows, passes;                             // query rows per kv head, and how many passes of NR they take
  int parts;                                     // that a ring's tiles are cut in
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
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
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
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n\t}\n" ::"r"(bar), "r"(bytes) : "memory");
}
// global -> shared, 16-byte aligned, a multiple of 16 bytes
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Waits for the phase of this parity.  Who gives up says so before it goes on; the others notice.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* s_failed) {
  for (int it = 0; it < SPIN_LIMIT; ++it) {
    if (bar_test(bar, parity)) return;
    if ((it & 63) == 63 && *s_failed) return;
  }
  *s_failed = 1;
}
template <int N>
__device__ __forceinline__ void registers() {    // launched with 48
  if constexpr (N > 48) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  if constexpr (N < 48) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
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

// 32 codes of a row -> 32 bytes, two pieces of 16, `chunk` bytes apart.  A selector's top bit asks for the sign of a level, which is zero: so the two
// permutes of a nibble are zero exactly where they are not meant, and their results are or-ed.
__device__ __forceinline__ void expand_half(const uint4& codes, const uint4& book, uint32_t dst, uint32_t chunk) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
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
// A row's 32 bytes of codes at `src` -> its 64 levels.  Of eight neighbouring threads the upper four (half = 1) take the second half first: then the
// eight read from different banks.  (Callers loop over rows without unrolling: an SM that runs five straight pieces of code waits for instructions.)
__device__ __forceinline__ void expand_row(uint32_t src, const uint4& book, uint32_t dst, uint32_t chunk, uint32_t half) {
#pragma unroll 1
  for (int k = 0; k < 2; ++k, half ^= 1) expand_half(lds128(src + 16 * half), book, dst + 2 * half * chunk, chunk);
}

// shared memory of a CTA
constexpr int K_STAGES = 2, V_STAGES = 3;
template <int D, int NR>
struct Smem {
  static constexpr int ROWS = D;                           // rows of the keys' operand = rows of the values' operand (D == 128: 128 tokens)
  static constexpr int CHUNK = ROWS * 16;
  static constexpr int A_BYTES = 8 * CHUNK;                // 128 positions
  static constexpr int B_BYTES = 2 * NR * 4 / 16 * CHUNK;  // 2 blocks x NR x 4 bytes
  static constexpr int SIDE = 36 * D;                      // keys or values of a page, as they come from memory
  static constexpr int K_A = 0, V_A = A_BYTES, K_B = 2 * A_BYTES, V_B = K_B + B_BYTES, K_IN = V_B + B_BYTES;
  static constexpr int V_IN = K_IN + K_STAGES * 2 * SIDE, BOOK = V_IN + V_STAGES * 2 * SIDE;
  static constexpr int QUERY = BOOK + MZP_BOOKS * MZP_LEVELS;          // the ring warps' queries [8][D], rows 16 bytes apart in the banks
  static constexpr int Q_ROW = 2 * D + 16;
  static constexpr int TOTAL = QUERY + 8 * Q_ROW;
  static constexpr int N = 8 * NR, TM_S = 0, TM_O = 2 * N, TM_COLS = NR == 4 ? 128 : 256;
};
// what a step is, for those who work on it
struct StepInfo {
  int pair, fresh;                          // the pair's number; whether this is the CTA's first step of it
  int count, see;                           // tokens of the step; the last position that the pair's first query token sees
  int b, head, r0, valid;                   // list entry, kv head, first query row; bit p: page p is there
};
// exchange between the warps of a CTA
template <int NR>
struct Exchange {
  alignas(16) float base[4][4][2 * NR];     // constant terms of the logits, by step and key warp (keys run up to two steps ahead)
  alignas(16) float fin[4][4 * NR];         // end of a pair: sums of p, constant terms of the output
  alignas(16) float qs[4][NR];              // logit per unit of the scaled query, by pair
  alignas(16) float vmax[2][4][NR];         // largest logit, by step parity and warp
  alignas(16) StepInfo info[8];             // by step (the line is up to five ahead of the softmax)
  float qmax[2][4][NR];                     // largest |q|, by pair and warp
  float2 row[2][2][2][128];                 // scale and constant term of the rows, by side, step parity, row of a thread, thread
  alignas(16) uint32_t top[2][4][4];        // largest T (bits) of the rows, by side, step and warp
  unsigned long long bar[2 * 11 + 3];
  int warp_sum[THREADS / 32];
  uint32_t tmem;
  int failed;
  int prefix[MAX_BATCH + 1];                // steps of the entries before
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

template <int D, bool BF, int NR>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) attention_kernel(const Args p, const uint8_t* __restrict__ book_table) {
  using S = Smem<D, NR>;
  constexpr int DT = BF ? MZ_BF16 : MZ_F16;
  constexpr int PB = 72 * D;                     // page bytes per kv head
  constexpr int RPT = D / 64;                    // rows of codes per thread, side and step
  constexpr int STREAMS = D == 128 ? 1 : 2;      // records of a ring's part
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Exchange<NR> x;
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(smem), sbook = sbase + S::BOOK;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t bars = smem_u32(x.bar);
  // of a side (keys, values): copied [stage], used [stage], scaled [2], operand written, products done [2]; sums of the keys read [2]; end
  constexpr uint32_t FULL = 0, USED = 24, SCALED = 48, READY = 64, DONE = 72, SIDE_BARS = 88;
  const uint32_t k_scaled = bars + SCALED, k_ready = bars + READY, k_done = bars + DONE, v_scaled = k_scaled + SIDE_BARS, v_ready = k_ready + SIDE_BARS,
                 v_done = k_done + SIDE_BARS, k_free = bars + 2 * SIDE_BARS, b_end = k_free + 16;
  if (tid == 0) {
    x.failed = 0;
    for (int side = 0; side < 2; ++side) {
      const uint32_t b = bars + side * SIDE_BARS;
      for (int i = 0; i < 3; ++i) { bar_init(b + FULL + 8 * i, 1); bar_init(b + USED + 8 * i, 4); }
      for (int i = 0; i < 2; ++i) { bar_init(b + SCALED + 8 * i, 4); bar_init(b + DONE + 8 * i, side ? 1 : 2); }
      bar_init(b + READY, 8);
    }
    for (int i = 0; i < 2; ++i) bar_init(k_free + 8 * i, 4);
    bar_init(b_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < MZP_BOOKS * MZP_LEVELS / 16) ((uint4*)(smem + S::BOOK))[tid] = ((const uint4*)book_table)[tid];

  // ---- the line of steps
  auto length_of = [&](int b, int& row) {
    row = p.rows ? p.rows[b] : b;
    return row < 0 || row >= c.rows ? 0 : max(0, min(c.lengths[row], 0x7fffffff - STEP));
  };
  const int kp_all = c.kv_heads * p.passes;
  int total_steps = 0;
  {
    constexpr int PER = (MAX_BATCH + THREADS) / THREADS;      // one more entry than the batch has: the end
    int st[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int b = tid * PER + k;
      int row;
      st[k] = b < p.batch ? (mzp_packed(length_of(b, row), c.residual) + STEP - 1) / STEP : 0;
      sum += st[k];
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += y; }
    if (lane == 31) x.warp_sum[warp] = scan;
    __syncthreads();
    int before = scan - sum;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) { const int t = x.warp_sum[w]; if (w < warp) before += t; total_steps += t; }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int b = tid * PER + k;
      if (b <= p.batch) x.prefix[b] = before;
      before += st[k];
    }
  }
  const long long T = (long long)total_steps * kp_all;
  const int G = gridDim.x, cta = blockIdx.x;
  const int W = (int)min((long long)G, T);       // CTAs that share the steps: none of them is left without one
  if (cta == 0 && tid == 0) { p.head[0] = W; *(long long*)(p.head + 2) = T; }
  const long long f0 = cta < W ? T * cta / W : 0, f1 = cta < W ? T * (cta + 1) / W : 0;
  const int n = (int)(f1 - f0);
  if (n > 0 && warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tm_before();
  }
  __syncthreads();
  tm_after();
  if (cta == 0) for (int b = tid; b <= p.batch; b += THREADS) p.head[4 + b] = x.prefix[b];
  const uint32_t tmem = n > 0 ? x.tmem : 0u;
  const int team = warp >> 2;
  const int r = tid & 127;                       // key channel or token of this thread

  if (team == 0 || team == 2) {
    // ================= levels, of keys (thread = channel) or values (thread = token): one piece of code, for an SM that runs many short of instructions
    registers<Regs<NR>::LEVELS>();
    const int side = team >> 1, blk = r >> 6, in_page = r & 63;
    const uint32_t half = (lane >> 2) & 1, b = bars + side * SIDE_BARS;
    // a thread's first row; keys of D = 128 have the channel's rows of both pages, values the token's two groups
    const int key_page = D == 128 ? 0 : blk, row0 = side ? in_page * RPT : D == 128 ? r : in_page;
    const uint32_t stages = side ? V_STAGES : K_STAGES, next_row = side ? 32 : S::SIDE, next_word = side ? 4 : S::SIDE;
    uint32_t in = sbase + (side ? S::V_IN + blk * S::SIDE : S::K_IN + key_page * S::SIDE), phase = 0;
    const uint32_t out = sbase + (side ? S::V_A + (D == 128 ? 0 : blk * 4 * S::CHUNK) : S::K_A + key_page * 4 * S::CHUNK) + (D == 128 ? r : in_page) * 16;
    const int valid0 = side ? blk : key_page, valid1 = side ? blk : key_page + 1;
    for (uint32_t it = 0, stage = 0; it < (uint32_t)n; ++it) {
      bar_wait(b + FULL + 8 * stage, phase, &x.failed);
      const int valid = x.info[it & 7].valid;
      uint32_t zeros[RPT], top = 0;
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        uint32_t word = lds32(in + 32 * D + 4 * row0 + j * next_word);
        if (!(valid >> (j ? valid1 : valid0) & 1)) word = 0u;
        top = max(top, word & 0xffffu);
        const MzpRow row = mzp_row(word);
        x.row[side][it & 1][j][r] = make_float2(row.t, fmaf(row.t, (float)row.z * -0.03125f, row.a));
        zeros[j] = sbook + row.z * 16;
      }
      // the step's largest T scales it; what the other lanes wrote goes with it
      top = warp_max_u32(top);
      __syncwarp();
      if (lane == 0) { x.top[side][it & 3][warp & 3] = top; bar_arrive(b + SCALED + 8 * (it & 1)); }
      if (it > 0) bar_wait(b + DONE + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1, &x.failed);    // the operand is free
#pragma unroll 1
      for (int j = 0; j < RPT; ++j) expand_row(in + row0 * 32 + j * next_row, book128(zeros[j ? RPT - 1 : 0]), out + j * 4 * S::CHUNK, S::CHUNK, half);
      fence_operands();
      __syncwarp();
      if (lane == 0) { bar_arrive(b + READY); bar_arrive(b + USED + 8 * stage); }
      in += 2 * S::SIDE;
      if (++stage == stages) { stage = 0; phase ^= 1; in -= stages * 2 * S::SIDE; }
    }
  } else if (team == 1) {
    // ================= key folds: thread = channel
    registers<Regs<NR>::KEY_FOLDS>();
    const int ch = D == 128 ? r : r & 63, tw = warp & 3;
    float q[NR];
    int seg = -1;
    const uint32_t out = sbase + S::K_B + (D == 128 ? 0 : r >> 6) * (NR / 4) * S::CHUNK + ch * 16;
    for (int it = 0; it < n; ++it) {
      bar_wait(k_scaled + 8 * (it & 1), it >> 1 & 1, &x.failed);
      if (x.info[it & 7].fresh) {
        const StepInfo info = x.info[it & 7];
        ++seg;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          q[i] = 0.f;
          if (info.r0 + i < p.qrows) {
            const int l = (info.r0 + i) / p.group, h = info.head * p.group + (info.r0 + i) % p.group;
            q[i] = MzType<DT>::load(p.query, (long long)info.b * p.qsb + l * p.qsl + h * p.qsh + ch);
          }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          // as bits, so that a NaN is the largest
          const uint32_t top = warp_max_u32(__float_as_uint(fabsf(q[i])));
          if (lane == 0) x.qmax[seg & 1][tw][i] = __uint_as_float(top);
        }
        team_barrier(1);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          uint32_t top = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) top = max(top, __float_as_uint(x.qmax[seg & 1][w][i]));
          const int e = max((int)(top >> 23) - 126, -60), e1 = e >> 1, e2 = e - e1;        // |q| < 2^e, taken off in two factors
          const bool wild = top >= 0x7f800000u;                        // infinity or NaN: the row's logits are NaN
          q[i] = wild ? 0.f : q[i] * pow2(-e1) * pow2(-e2);
          if (r == 0) x.qs[seg & 3][i] = wild ? __int_as_float(0x7fffffff) : pow2(e1) * p.scaling * pow2(e2);
        }
      }
      float2 row[RPT];
#pragma unroll
      for (int j = 0; j < RPT; ++j) row[j] = x.row[0][it & 1][j][r];
      {
        float base[RPT * NR];
#pragma unroll
        for (int j = 0; j < RPT; ++j) {
#pragma unroll
          for (int i = 0; i < NR; i += 2) {
            base[j * NR + i] = base[j * NR + i + 1] = 0.f;
            fma2(base[j * NR + i], base[j * NR + i + 1], q[i], q[i + 1], row[j].y);
          }
        }
        int index;
        const float sum = warp_sums<RPT * NR>(base, lane, index);
        if ((lane & (32 / (RPT * NR) - 1)) == 0) x.base[it & 3][tw][index] = sum;
      }
      const float up = pow2(30 - ((int)(max4(x.top[0][it & 3]) >> 10) - 14));      // T < 2^(exponent field - 14)
      if (it > 0) bar_wait(k_done + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1, &x.failed);
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const float ts = row[j].x * up;
#pragma unroll
        for (int i = 0; i < NR; i += 4) {
          float f[4] = {0.f, 0.f, 0.f, 0.f};
          fma2(f[0], f[1], q[i], q[i + 1], ts);
          fma2(f[2], f[3], q[i + 2], q[i + 3], ts);
          sts128(out + (j * (NR / 4) + i / 4) * S::CHUNK, digits_of(f[0]), digits_of(f[1]), digits_of(f[2]), digits_of(f[3]));
        }
      }
      fence_operands();
      __syncwarp();
      if (lane == 0) bar_arrive(k_ready);
    }
  } else if (team == 3) {
    // ================= softmax: thread = token, and position of the output
    registers<Regs<NR>::SOFTMAX>();
    const int tw = warp & 3, blk = r >> 6;
    const uint32_t lanes = tmem + ((uint32_t)(tw * 32) << 16);
    float m[NR], l[NR], o[NR], base_v[RPT][NR], qs[NR];
    float vunit = 0.f;
    int pair = -1, seg = -1;
    auto reset = [&]() {
#pragma unroll
      for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; o[i] = 0.f; }
#pragma unroll
      for (int j = 0; j < RPT; ++j)
#pragma unroll
        for (int i = 0; i < NR; ++i) base_v[j][i] = 0.f;
    };
    // the products of step `done`
    auto take_output = [&](int done) {
      bar_wait(v_done + 8 * (done & 1), done >> 1 & 1, &x.failed);
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
      team_barrier(3);
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
      team_barrier(3);                                       // fin and halves are free again
    };
    reset();
    for (int it = 0; it < n; ++it) {
      bar_wait(k_done + 8 * (it & 1), (it >> 1) & 1, &x.failed);
      tm_after();
      const StepInfo info = x.info[it & 7];
      if (info.fresh) {
        if (pair >= 0) {
          take_output(it - 1);
          write_record();
          reset();
        }
        pair = info.pair; ++seg;
      }
      // ---- logits
      if (info.fresh) load_floats(qs, x.qs[seg & 3]);
      const float kunit = pow2((int)(max4(x.top[0][it & 3]) >> 10) - 14 - 35);
      float s[NR], base[NR];
      if (D == 128) {
        float b[4][NR];
#pragma unroll
        for (int w = 0; w < 4; ++w) load_floats(b[w], x.base[it & 3][w] + blk * NR);
#pragma unroll
        for (int i = 0; i < NR; i += 2) {
          add2(b[0][i], b[0][i + 1], b[1][i], b[1][i + 1]);
          add2(b[2][i], b[2][i + 1], b[3][i], b[3][i + 1]);
          add2(b[0][i], b[0][i + 1], b[2][i], b[2][i + 1]);
          base[i] = b[0][i]; base[i + 1] = b[0][i + 1];
        }
      } else {
        float b[2][NR];
#pragma unroll
        for (int w = 0; w < 2; ++w) load_floats(b[w], x.base[it & 3][2 * blk + w]);
#pragma unroll
        for (int i = 0; i < NR; ++i) base[i] = b[0][i] + b[1][i];
      }
#pragma unroll
      for (int i = 0; i < NR; i += 4) {
        int a[16];
        tm_ld16(lanes + S::TM_S + (it & 1) * S::N + blk * (4 * NR) + 4 * i, a);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[i + k] = number_of(a + 4 * k);
      }
      tm_before();
      __syncwarp();
      if (lane == 0) bar_arrive(k_free + 8 * (it & 1));
#pragma unroll
      for (int i = 0; i < NR; i += 2) mul_add2(s[i], s[i + 1], s[i], s[i + 1], base[i], base[i + 1], qs[i], qs[i + 1], kunit);
      if (info.count < STEP) {
#pragma unroll
        for (int i = 0; i < NR; ++i) if (r >= info.count) s[i] = -INFINITY;
      }
      if (info.see < info.count - 1) {                       // not every query sees all of the step
#pragma unroll
        for (int i = 0; i < NR; ++i) if (r > info.see + (info.r0 + i) / p.group - info.r0 / p.group) s[i] = -INFINITY;
      }
      // ---- running maximum
      float fix[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) fix[i] = warp_max(s[i]);
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < NR; i += 4) *(float4*)&x.vmax[it & 1][tw][i] = make_float4(fix[i], fix[i + 1], fix[i + 2], fix[i + 3]);
      }
      team_barrier(3);
      bool moved = false;
      {
        float v[4][NR];
#pragma unroll
        for (int w = 0; w < 4; ++w) load_floats(v[w], x.vmax[it & 1][w]);
#pragma unroll
        for (int i = 0; i < NR; ++i) fix[i] = fmaxf(fmaxf(v[0][i], v[1][i]), fmaxf(v[2][i], v[3][i]));
      }
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        moved |= fix[i] > m[i];
        fix[i] = fmaxf(m[i], fix[i]);
        s[i] = ex2(s[i] - (fix[i] == -INFINITY ? 0.f : fix[i]));
      }
      bar_wait(v_scaled + 8 * (it & 1), it >> 1 & 1, &x.failed);
      const int ev = (int)(max4(x.top[1][it & 3]) >> 10) - 14;
      const float up = pow2(30 - ev);
      // ---- the output so far; then the operand is free
      if (it > 0 && !info.fresh) take_output(it - 1);
      if (moved) {                                           // the same for all threads
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
      for (int i = 0; i < NR; i += 2) add2(l[i], l[i + 1], s[i], s[i + 1]);
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const float2 row = x.row[1][it & 1][j][r];
        const float ts = row.x * up, cz = row.y;
        const int b2 = D == 128 ? j : blk, at = D == 128 ? r : r & 63;
#pragma unroll
        for (int i = 0; i < NR; i += 2) fma2(base_v[j][i], base_v[j][i + 1], s[i], s[i + 1], cz);
#pragma unroll
        for (int i = 0; i < NR; i += 4) {
          float f[4] = {0.f, 0.f, 0.f, 0.f};
          fma2(f[0], f[1], s[i], s[i + 1], ts);
          fma2(f[2], f[3], s[i + 2], s[i + 3], ts);
          sts128(sbase + S::V_B + (b2 * (NR / 4) + i / 4) * S::CHUNK + at * 16, __float2int_rn(f[0]), __float2int_rn(f[1]), __float2int_rn(f[2]),
                 __float2int_rn(f[3]));
        }
      }
      fence_operands();
      tm_before();
      __syncwarp();
      if (lane == 0) bar_arrive(v_ready);
    }
    if (n > 0) {
      take_output(n - 1);
      write_record();
    }
  } else {
    registers<Regs<NR>::SERVICE>();
    if (warp == 16) {
      // ================= the line: page numbers, copies
      int b = 0, head = 0, pass = 0, step = 0, steps = 1, row = 0, len = 0;
      bool fresh = true;
      if (n > 0) {
        int hi = p.batch;                        // prefix[b] * kp_all <= f0 < prefix[b + 1] * kp_all
        while (hi - b > 1) { const int mid = (b + hi) >> 1; if ((long long)x.prefix[mid] * kp_all <= f0) b = mid; else hi = mid; }
        steps = x.prefix[b + 1] - x.prefix[b];
        const int rem = (int)(f0 - (long long)x.prefix[b] * kp_all), kp = rem / steps;
        head = kp / p.passes;
        pass = kp % p.passes;
        step = rem % steps;
        len = length_of(b, row);
      }
      int ids = -1, ids_at = -64;                // page numbers ids_at .. ids_at + 31 of the row, one per lane
      for (int it = 0; it < n; ++it) {
        const int pages = mzp_packed(len, c.residual) / MZP_PAGE, k0 = 2 * step;
        if (k0 < ids_at || k0 >= ids_at + 32) {
          ids_at = k0;
          ids = -1;
          if (k0 + lane < pages) {
            ids = k0 + lane < c.width ? c.block_table[(long long)row * c.width + k0 + lane] : -1;
            if (ids < 0 || ids >= c.pages) { ids = -1; atomicOr(c.status, MZ_PAGED_BAD_INDEX); }
          }
        }
        const int page0 = __shfl_sync(0xffffffffu, ids, k0 - ids_at), page1 = __shfl_sync(0xffffffffu, ids, k0 + 1 - ids_at);
        const int ks = it % K_STAGES, vs = it % V_STAGES;
        if (it >= K_STAGES) bar_wait(bars + USED + 8 * ks, (it / K_STAGES - 1) & 1, &x.failed);
        const uint32_t bytes = S::SIDE * ((page0 >= 0) + (page1 >= 0));
        const uint8_t* store = (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer + head * PB;
        const uint8_t *src0 = store + (long long)page0 * c.store_stride_page, *src1 = store + (long long)page1 * c.store_stride_page;
        const uint32_t kin = sbase + S::K_IN + 2 * ks * S::SIDE, vin = sbase + S::V_IN + 2 * vs * S::SIDE;
        if (lane == 0) {
          StepInfo info;
          info.pair = (b * c.kv_heads + head) * p.passes + pass;
          info.fresh = fresh;
          info.count = min(STEP, pages * MZP_PAGE - step * STEP);
          info.r0 = pass * NR;
          info.see = len - p.q_len + info.r0 / p.group - step * STEP;
          info.b = b;
          info.head = head;
          info.valid = (page0 >= 0 ? 1 : 0) | (page1 >= 0 ? 2 : 0);
          x.info[it & 7] = info;
          bar_expect(bars + FULL + 8 * ks, bytes);
          if (page0 >= 0) bulk_copy(kin, src0, S::SIDE, bars + FULL + 8 * ks);
          if (page1 >= 0) bulk_copy(kin + S::SIDE, src1, S::SIDE, bars + FULL + 8 * ks);
        }
        if (it >= V_STAGES) bar_wait(bars + SIDE_BARS + USED + 8 * vs, (it / V_STAGES - 1) & 1, &x.failed);
        if (lane == 0) {
          bar_expect(bars + SIDE_BARS + FULL + 8 * vs, bytes);
          if (page0 >= 0) bulk_copy(vin, src0 + S::SIDE, S::SIDE, bars + SIDE_BARS + FULL + 8 * vs);
          if (page1 >= 0) bulk_copy(vin + S::SIDE, src1 + S::SIDE, S::SIDE, bars + SIDE_BARS + FULL + 8 * vs);
        }
        __syncwarp();
        fresh = false;
        if (++step == steps) {
          step = 0; fresh = true; ids_at = -64;
          if (++pass == p.passes) {
            pass = 0;
            if (++head == c.kv_heads) {
              head = 0;
              do { ++b; } while (b < p.batch && x.prefix[b + 1] == x.prefix[b]);
              if (b < p.batch) { steps = x.prefix[b + 1] - x.prefix[b]; len = length_of(b, row); }
            }
          }
        }
      }
      // copies in flight end before the CTA does (the teams have waited for all of them unless a wait ran out)
      for (int it = max(0, n - K_STAGES); it < n; ++it)
        for (int k = 0; k < SPIN_LIMIT && !bar_test(bars + FULL + 8 * (it % K_STAGES), it / K_STAGES & 1); ++k) {}
      for (int it = max(0, n - V_STAGES); it < n; ++it)
        for (int k = 0; k < SPIN_LIMIT && !bar_test(bars + SIDE_BARS + FULL + 8 * (it % V_STAGES), it / V_STAGES & 1); ++k) {}
    } else if (warp == 17) {
      // ================= MMAs, in the order keys 0, keys 1, values 0, keys 2, values 1, ...  (The whole warp waits: a diverged one would poll.)
      const uint64_t ka = descriptor(sbase + S::K_A, S::CHUNK), kb = descriptor(sbase + S::K_B, S::CHUNK);
      const uint64_t va = descriptor(sbase + S::V_A, S::CHUNK), vb = descriptor(sbase + S::V_B, S::CHUNK);
      auto keys = [&](int it) {
        bar_wait(k_ready, it & 1, &x.failed);
        if (it >= 2) bar_wait(k_free + 8 * (it & 1), (it >> 1 & 1) ^ 1, &x.failed);
        if (lane == 0) {
          bar_arrive(k_done + 8 * (it & 1));     // hands on what the keys' threads wrote beside the operand
          if (!*(volatile int*)&x.failed) {
            tm_after();
#pragma unroll
            for (int k = 0; k < D / 32; ++k) umma<S::N, true>(tmem + S::TM_S + (it & 1) * S::N, ka + k * (512 >> 4), kb + k * (512 >> 4), k > 0);
            umma_commit(k_done + 8 * (it & 1));
          }
        }
        __syncwarp();
      };
      if (n > 0) keys(0);
      for (int it = 0; it < n; ++it) {
        if (it + 1 < n) keys(it + 1);
        bar_wait(v_ready, it & 1, &x.failed);
        if (lane == 0 && !*(volatile int*)&x.failed) {
          tm_after();
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma<S::N, false>(tmem + S::TM_O, va + k * (512 >> 4), vb + k * (512 >> 4), k > 0);
          umma_commit(v_done + 8 * (it & 1));
        }
        __syncwarp();
      }
    } else {
      // ================= rings: a warp takes 16 tokens at a time, and (D = 128) 64 of the channels of the output.  A = keys [token][channel], B =
      // queries; A = values [channel][token], B = p in two parts of 16 bits
      const int g = lane >> 2, t = lane & 3, rw = warp - 18;
      const int half = D == 128 ? rw : 0, stream = D == 128 ? 0 : rw;
      const long long units = p.pairs * p.parts, first_slot = (long long)G + p.pairs;
      for (long long unit = G - 1 - cta; unit < units; unit += G) {        // CTAs without steps come first
        const int part = (int)(unit % p.parts);
        const long long pair = unit / p.parts;
        const int b = (int)(pair / kp_all), kp = (int)(pair % kp_all), head = kp / p.passes, r0 = kp % p.passes * NR;
        int row;
        const int len = length_of(b, row), packed = mzp_packed(len, c.residual), tokens = len - packed;
        if (tokens == 0) continue;
        const int tiles = (tokens + 15) / 16, end = tiles * (part + 1) / p.parts;
        const uint16_t* ring_k = (const uint16_t*)c.tail + (long long)p.layer * c.tail_stride_layer + (long long)row * c.tail_stride_row + (long long)head * c.ring * D;
        const uint16_t* ring_v = ring_k + (long long)c.kv_heads * c.ring * D + half * 64;
        const int ring0 = packed % c.ring;
        auto place = [&](int i) { const int at = ring0 + i; return (at >= c.ring ? at - c.ring : at) * D; };      // i < tokens <= ring
        // queries into shared memory; rows that are not there are zero
        asm volatile("bar.sync 6, 64;" ::: "memory");
        for (int i = tid & 63; i < 8 * D; i += 64) {
          const int qi = i / D, d = i % D, qr = r0 + qi;
          uint16_t v = 0;
          if (qi < NR && qr < p.qrows) v = p.query[(long long)b * p.qsb + qr / p.group * p.qsl + (head * p.group + qr % p.group) * p.qsh + d];
          *(uint16_t*)(smem + S::QUERY + qi * S::Q_ROW + 2 * d) = v;
        }
        asm volatile("bar.sync 6, 64;" ::: "memory");
        const int see0 = len - p.q_len - packed;               // query token l sees the ring's tokens up to see0 + l
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[4][4];
  #pragma unroll
        for (int i = 0; i < 4; ++i)
  #pragma unroll
          for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
        for (int tile = tiles * part / p.parts + stream; tile < end; tile += STREAMS) {
          const int i0 = tile * 16;
          float s[4] = {0.f, 0.f, 0.f, 0.f};
          {
            const uint16_t* ka = ring_k + place(min(i0 + g, tokens - 1)) + 8 * t;
            const uint16_t* kb = ring_k + place(min(i0 + g + 8, tokens - 1)) + 8 * t;
  #pragma unroll
            for (int k = 0; k < D / 32; ++k) {
              const uint4 va = *(const uint4*)(ka + 32 * k), vb = *(const uint4*)(kb + 32 * k);
              const uint4 qf = lds128(sbase + S::QUERY + g * S::Q_ROW + (32 * k + 8 * t) * 2);
              mma16<BF>(s, va.x, vb.x, va.y, vb.y, qf.x, qf.y);
              mma16<BF>(s, va.z, vb.z, va.w, vb.w, qf.z, qf.w);
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
          // p in two parts, transposed: column g, tokens 2t, 2t + 1 ([0]) and 2t + 8, 2t + 9 ([1])
          uint32_t hi[2], lo[2];
  #pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t hw, lw;
            if (BF) {
              const __nv_bfloat162 hb = __floats2bfloat162_rn(s[2 * h], s[2 * h + 1]);
              const float2 hf = __bfloat1622float2(hb);
              const __nv_bfloat162 lb = __floats2bfloat162_rn(s[2 * h] - hf.x, s[2 * h + 1] - hf.y);
              hw = *reinterpret_cast<const uint32_t*>(&hb); lw = *reinterpret_cast<const uint32_t*>(&lb);
            } else {
              const __half2 hb = __floats2half2_rn(s[2 * h], s[2 * h + 1]);
              const float2 hf = __half22float2(hb);
              const __half2 lb = __floats2half2_rn(s[2 * h] - hf.x, s[2 * h + 1] - hf.y);
              hw = *reinterpret_cast<const uint32_t*>(&hb); lw = *reinterpret_cast<const uint32_t*>(&lb);
            }
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(hi[h]) : "r"(hw));
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(lo[h]) : "r"(lw));
          }
          // A token that is not there, or that only later queries see, must not bring a NaN to a product with p = 0: what is not there is read as zero, and
          // where a tile has tokens that only some of the queries see, each of the queries' tokens takes its turn with what it sees
          const int l_first = r0 / p.group, l_last = (min(r0 + NR, p.qrows) - 1) / p.group;
          const bool apart = i0 + 15 > see0 + l_first && l_last > l_first;
          for (int turn = 0; turn <= (apart ? l_last - l_first : 0); ++turn) {
            const int see = apart ? min(see0 + l_first + turn, tokens - 1) : tokens - 1;
            const bool mine = !apart || (r0 + g) / p.group == l_first + turn;
            uint4 v[4];
  #pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = i0 + 2 * t + (k & 1) + 8 * (k >> 1);
              v[k] = make_uint4(0, 0, 0, 0);
              if (i <= see) v[k] = *(const uint4*)(ring_v + place(i) + 8 * g);
            }
            const uint32_t w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
            const uint32_t w2[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, w3[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
  #pragma unroll
            for (int k = 0; k < 4; ++k) {
              // rows g / g + 8 = channels 8g + 2k / 8g + 2k + 1
              const uint32_t a0 = prmt(w0[k], w1[k], 0x5410u), a1 = prmt(w0[k], w1[k], 0x7632u);
              const uint32_t a2 = prmt(w2[k], w3[k], 0x5410u), a3 = prmt(w2[k], w3[k], 0x7632u);
              mma16<BF>(o[k], a0, a1, a2, a3, mine ? lo[0] : 0u, mine ? lo[1] : 0u);
              mma16<BF>(o[k], a0, a1, a2, a3, mine ? hi[0] : 0u, mine ? hi[1] : 0u);
            }
          }
        }
  #pragma unroll
        for (int j = 0; j < 2; ++j) {
  #pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], off);
          if (2 * t + j < NR) {
            const long long slot = (first_slot + unit * STREAMS + stream) * NR + 2 * t + j;
            float* dst = p.acc + slot * D + half * 64 + 8 * g;
  #pragma unroll
            for (int k = 0; k < 4; ++k) *(float2*)(dst + 2 * k) = make_float2(o[k][j], o[k][2 + j]);
            if (g == 0 && half == 0) p.ml[slot] = make_float2(m[j], l[j]);
          }
        }
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (n == 0) return;
  if (x.failed && tid == 17 * 32) {      // products in flight end before their memory goes back
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

// merges the records of one query row of a pair: a thread per channel, records in their order
template <int D, bool BF, int NR>
__global__ void __launch_bounds__(D) merge_kernel(const Args p, int G) {
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
  constexpr int STREAMS = D == 128 ? 1 : 2;
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
    const long long first = G + p.pairs + pair * p.parts * STREAMS;
    for (int k0 = 0; k0 < p.parts * STREAMS; k0 += 4) {
      float2 ml[4];
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long slot = (first + min(k0 + k, p.parts * STREAMS - 1)) * NR + i;
        ml[k] = p.ml[slot];
        v[k] = p.acc[slot * D + d];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) if (k0 + k < p.parts * STREAMS) take(ml[k], v[k]);
    }
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
  kern<<<G, THREADS, S::TOTAL, st>>>(p, book);
  MZ_LAUNCH_CHECK("paged attention");
  // The merge kernel's launch overlaps the first kernel's end.  (Not so the first kernel's with the merge before it: an SM does not change its split of
  // L1 and shared memory while a CTA runs on it, and two of these CTAs then do not fit.)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(p.pairs * NR));
  cfg.blockDim = dim3(D);
  MZ_CUDA(cudaLaunchKernelEx(&cfg, merge_kernel<D, BF, NR>, p, G));
  MZ_LAUNCH_CHECK("paged attention merge");
  return MZ_OK;
}

struct Shape { int nr, passes, parts, G; long long pairs; size_t head_bytes, slots, bytes; };
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
  s->G = sms * CTAS_PER_SM;
  // few pairs: their rings are cut until a warp has one tile of 16 tokens or the CTAs are taken
  const int streams = c->head_dim == 128 ? 1 : 2, most = ((c->residual + MZP_PAGE - 1 + 15) / 16 + streams - 1) / streams;
  const long long share = s->pairs > 0 ? s->G / s->pairs : 1;
  s->parts = (int)(share < 1 ? 1 : share > most ? most : share);
  s->head_bytes = ((4 + (size_t)batch + 1) * sizeof(int) + 127) / 128 * 128;
  s->slots = (size_t)s->G + (size_t)s->pairs * (1 + s->parts * streams);
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
  p.parts = s.parts;
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
