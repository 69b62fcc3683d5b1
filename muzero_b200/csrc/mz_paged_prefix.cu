// Paged cache: attention of rows in groups over the pages that a group's rows have in common (sm_100a, tcgen05).
//
// Mathematics.  A code stands for A + T (u - z) / 32 (mz_paged.cuh).  For a tile of query rows and a page of 64 tokens
//   S = q K^T          K as two f16 numbers, value and remainder: 22 bits of every key; q (bf16 or f16) is exact in f16 once its row is scaled by a power of two
//   P = exp2(S f + e - M),  O += P V          V like K, P as two f16 numbers too: three products, all but that of the remainders (2^-22); sums are fp32
// Keys and values of a page are scaled into f16's range by powers of two, ek and ev; f takes ek back.  ev is taken back by the softmax itself: M is the running
// maximum not of the logits t but of t + ev, so P V has one scale whatever the pages' ranges and l sums P 2^-ev in fp32.  P is 2^7 under M itself; M moves when a row's sum of P over a page
// passes 2^15 (the output in tensor memory is scaled then), so P is a f16 number, and what is lost below its smallest one is under 2^-31 of the largest.
// The output's running sums are held in fp32 outside the tensor cores (SUM_JOBS).
// Scales of rows of codes are f16 as well: one below 2^-21 of its page's largest loses bits, 2^-32 of the page's largest value.
// Measured, the output's error against the call without sharing: 1.4e-6 (64 rows behind 4224 tokens) to 1.0e-5 (32 rows behind 131072; against 64 bits 6.6e-6, without sharing 1.1e-5).  With one f16
// number for P and V 2e-4 and 10 to 40 us less, with one for K 1.0e-3 where channels differ by a factor of e^2.5.
//
// Work.  Groups, tiles, units, the line and its cut: mz_paged_prefix.cuh.  A CTA per SM, its warps by duty: a page is copied as it is (one bulk copy), its rows' words are decoded, its codes become
// f16 operands (MN-major, 128-byte swizzle: a thread has a row of 64 codes and stores it as 8 pieces of 16 bytes, nothing is transposed), products, softmax.  Queries and P are operands in tensor
// memory, where 512 columns hold two blocks of queries, two or three of logits with P over them, and two outputs.  Two streams of four softmax warps: with more than 128 rows each has half of
// the rows, otherwise they take the pages in turn and their outputs are merged at the end.
//
// Measured (B200 at 1965 MHz, 8 kv heads, head_dim 128): 32 rows x 4 heads behind 131072 tokens 195 us (its 68.7 GFLOP would take 42 us at the measured cuBLAS rate), 12 prompts of 500 to 16001
// tokens for 4 rows x 8 heads, f16, 147 us.  A page takes 3200 cycles where the tensor cores need 1310 (keys 530, values 780); no unit is saturated (issue 53 %, tensor pipe 46 %, logic pipe 36 %, ex2
// and conversions 22 %): jobs go round from products to softmax and back, and instruction fetch is a part of every turn.
#include <algorithm>
#include <atomic>

#include "mz_paged_prefix.cuh"

namespace mzp {
namespace {
// Warps by duty: 0 .. 7 softmax (a group of four per stream).  Of the others, every fourth one, which are all on one scheduler, has a duty that much waits for: 11 issues the
// products, 15 copies pages as they are, 19 and 23 decode the words of their rows; the rest make the levels, in three teams of four with a page each.
constexpr int SOFTMAX_WARPS = 8, WARPS = 24, ISSUER = 11, FEEDER = 15, DECODER = 19, TEAMS = 3, PREFIX_THREADS = 32 * WARPS;
// of the 80 x 768 registers that a CTA is launched with: 256 x 112 + 512 x 64 are all
constexpr int SOFTMAX_REGS = 112, OTHER_REGS = 64;
template <int N, bool MORE>
__device__ __forceinline__ void registers() {
  if (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr int PLAN_THREADS = 512, PLAN_CTAS = 8;

struct PrefixArgs {
  mz_paged_cache c;
  const uint16_t* query;
  long long qsb, qsl, qsh;
  const int* rows;
  const int* offsets;                            // of the groups
  int layer, batch, q_len, group, qrows, longest;
  float scaling;                                 // times log2(e)
  MzpPrefix out;
  int fail_waits;
};

// ---- which pages a group's rows have in common: a cluster per group
__global__ void __cluster_dims__(PLAN_CTAS, 1, 1) __launch_bounds__(PLAN_THREADS) plan_kernel(const PrefixArgs p) {
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, rank = blockIdx.x % PLAN_CTAS, g = blockIdx.x / PLAN_CTAS, n_groups = p.out.n_groups;
  __shared__ int s_common, s_members, s_row0;
  __shared__ uint8_t s_member[1024];             // (a call has at most 1024 entries)
  bool fine = true;
  for (int i = tid; i < n_groups; i += PLAN_THREADS) {
    const int lo = p.offsets[i], hi = p.offsets[i + 1];
    fine = fine && lo >= 0 && lo <= hi && hi <= p.batch;
  }
  fine = __syncthreads_and(fine);
  const int first = fine ? p.offsets[g] : 0, end = fine ? p.offsets[g + 1] : 0;
  // entries that no group has
  const int zero0 = fine && g == n_groups - 1 ? p.offsets[n_groups] : 0, zero1 = !fine ? (g == 0 ? p.batch : 0) : g == n_groups - 1 ? p.batch : 0;
  for (int i = zero0 + rank * PLAN_THREADS + tid; i < zero1; i += PLAN_CTAS * PLAN_THREADS) p.out.skip[i] = 0;
  if (fine && g == 0) for (int i = rank * PLAN_THREADS + tid; i < first; i += PLAN_CTAS * PLAN_THREADS) p.out.skip[i] = 0;
  if (!fine && g == 0 && rank == 0 && tid == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
  auto row_at = [&](int b) { return p.rows ? p.rows[b] : b; };
  // no further than every query of every row sees, and than every row has pages.  A row that would share no page (it is empty, or not there) stays out and leaves the others theirs
  if (tid == 0) { s_common = c.width; s_members = 0; s_row0 = 0x7fffffff; }
  __syncthreads();
  for (int b = first + tid; b < end; b += PLAN_THREADS) {
    const int row = row_at(b);
    const int len = row < 0 || row >= c.rows ? 0 : max(0, min(c.lengths[row], p.longest));
    const int pages = min(mzp_packed(len, c.residual), max(0, len - p.q_len + 1)) / MZP_PAGE;
    s_member[b - first] = pages > 0;
    if (pages > 0) {
      atomicMin(&s_common, pages);
      atomicAdd(&s_members, 1);
      atomicMin(&s_row0, b);
    }
  }
  __syncthreads();
  int common = s_members < 2 ? 0 : s_common;
  const int row0 = s_members > 0 ? row_at(s_row0) : 0;
  __syncthreads();
  if (tid == 0) s_common = common;
  __syncthreads();
  if (common > 0) {
    // a warp compares 128 columns of its share of the rows with the first row's, four rows' loads on their way at a time
    const int* head = c.block_table + (long long)row0 * c.width;
    const int lane = tid & 31, warps = PLAN_CTAS * (PLAN_THREADS / 32), pieces = (common + 127) / 128, shares = max(1, min(warps / pieces, end - first));
    for (int i = rank * (PLAN_THREADS / 32) + (tid >> 5); i < pieces * shares; i += warps) {
      const int share = i / pieces, at = (i - share * pieces) * 128 + lane;
      int id[4], bad = 0x7fffffff;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        id[k] = at + 32 * k < common ? head[at + 32 * k] : 0;
        if (id[k] < 0 || id[k] >= c.pages) bad = min(bad, at + 32 * k);
      }
      for (int b0 = first + share; b0 < end; b0 += 4 * shares) {
        int other[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int b = min(b0 + r * shares, end - 1);
          const int* theirs = s_member[b - first] ? c.block_table + (long long)row_at(b) * c.width : head;
#pragma unroll
          for (int k = 0; k < 4; ++k) other[r][k] = at + 32 * k < common ? theirs[at + 32 * k] : id[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if ((other[0][k] ^ id[k]) | (other[1][k] ^ id[k]) | (other[2][k] ^ id[k]) | (other[3][k] ^ id[k])) bad = min(bad, at + 32 * k);
      }
      if (bad != 0x7fffffff) atomicMin(&s_common, bad);
    }
  }
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
#pragma unroll
  for (int r = 0; r < PLAN_CTAS; ++r) {
    uint32_t theirs;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(smem_u32(&s_common)), "r"(r));
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(theirs) : "memory");
    common = min(common, v);
  }
  const int entries = end - first, members = s_members;
  const MzpTiles tiles(entries * p.qrows);
  if (mzp_gain(common, c.kv_heads, (long long)members * p.out.passes, p.out.nr, tiles.cost()) == 0) common = 0;
  for (int b = first + rank * PLAN_THREADS + tid; b < end; b += PLAN_CTAS * PLAN_THREADS) { p.out.skip[b] = s_member[b - first] ? common : 0; p.out.group_of[b] = g; }
  if (rank == 0 && tid == 0) p.out.groups[g] = {first, (end - first) * p.qrows, end > first ? common : 0, row0, members};
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // nobody's shared memory goes while it is read
}

// ---- attention over the prefixes
// Pages as they are, stages of keys and of values, blocks of logits where the streams share their rows.  Values stand longer than keys, until P is there: with 5 raw pages and 2 + 2, 3 + 2 (4 raw pages),
// 2 + 3 (4) stages 32 rows behind 131072 tokens take 243, 249, 235 us; a sixth raw page, all products of a job written out, keys and values by code of their own 241, 243, 262.
// The barriers of a stage go round RING places, so that a team, which is behind its own last
// page by TEAMS pages and knows that what was in that one's stage before has been used, cannot take another phase of a barrier for the one that it waits for
constexpr int RAWS = 4, K_STAGES = 2, V_STAGES = 3, BLOCKS = 3, RING = 4;
static_assert(RAWS > TEAMS && RING >= TEAMS && (RING & (RING - 1)) == 0 && RING >= K_STAGES && RING >= V_STAGES, "a wait could take another phase for its own");
template <int D>
struct PrefixSmem {
  static constexpr int PLANE = MZP_PAGE * D * 2;                                 // a page's keys, or values, in 16 bits
  static constexpr int PAGE_BYTES = 72 * D;
  static constexpr int SCALES = 16, ROWS = 2 * D;                                // ROWS: rows of codes of a page
  static constexpr int KEYS = 0, VALUES = K_STAGES * 2 * PLANE, RAW = VALUES + V_STAGES * 2 * PLANE, BOOK = RAW + RAWS * PAGE_BYTES, TERMS = BOOK + MZP_BOOKS * MZP_LEVELS;
  static constexpr int ALIGN = 1024, TOTAL = TERMS + RAWS * ROWS * 16 + ALIGN;
  // columns of tensor memory: queries (A operand, two values to a column), logits of two or three jobs (P stands over their first half, its remainder over the other), outputs of the streams.
  // Where the streams have rows of their own there are two blocks of queries and of logits, where they share theirs one and three
  static constexpr int TM_Q = 0, TM_O = 256, TM_COLS = 512;
  static __host__ __device__ constexpr int tm_s(bool both) { return both ? D : D / 2; }
  static_assert(D + 2 * MZP_PAGE <= TM_O && D / 2 + BLOCKS * MZP_PAGE <= TM_O && TM_O + 2 * D <= TM_COLS, "tensor memory");
};
// Operands stand major along the kept dimension (keys: tokens, values: channels): rows of 64 values (128 bytes) along it, one per index that is summed over, the eight
// 16-byte pieces of a row in the order of their number xor the row's (128-byte swizzle); values of head_dim 128 are two such blocks
constexpr int OPERAND_STEP = 16 * 128 >> 4;      // 16 rows further

struct alignas(16) Segment { int first, row, head, m0, rows, page, count, pad; long long record; };      // a run of steps of one unit
constexpr int ISSUE_UNROLL = 4;
// Jobs of a stream that go into one accumulator.  The tensor cores cut their running sums off, always towards zero: up to 2^-23 of the sum in each of a job's 12 products.  Measured with values of one
// sign: 2.2e-4 of the output after 432 jobs, 1.1e-4 after 216.  So after this many the sum is added in fp32 to what there is: below 2e-5.  32 rows behind 131072 tokens with 8 / 16 / 32 / all jobs to
// an accumulator 259 / 253 / 245 / 245 us (with two stages of values)
constexpr int SUM_JOBS = 32;
constexpr int SEGMENTS = 64;                     // of a CTA at a time
struct PrefixShared {
  Segment seg[SEGMENTS];
  unsigned long long raw_full[RAWS], raw_free[RAWS], scaled[16], full[2][RING], free[2][RING], s_full[4], p_full[4], o_done[4], q_full, end;      // [2]: keys, values
  int2 scale[16];                                // (ek, ev) by page of the CTA's line; pages are scaled ten ahead of their softmax at most
  int there[RAWS];                                // whether a raw page is one
  float2 ml[2][128];                             // of the two streams, where they share rows
  int segments, more;                            // in hand; whether others follow
  uint32_t tmem;
  int failed;
};

// D[128 x N] (+)= A[128 x 16, tensor memory] * B[16 x N], f16 into fp32, B major along N
// (b: the operand's address in 16 bytes; its other fields are constant)
template <int N>
__device__ __forceinline__ void umma16(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t accumulate) {
  constexpr uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(N / 8) << 17) | (8u << 24);
  constexpr uint32_t low = MZP_PAGE * 128 >> 4 << 16, high = 1024u >> 4 | 1u << 14 | 2u << 29;       // blocks 8 KB apart, eight rows 1 KB, 128-byte swizzle
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 d;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 d, {%2, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, p;\n\t}\n"
               ::"r"(d_tmem), "r"(a_tmem), "r"(b | low), "r"(high), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ bool elect() {        // one lane of a whole warp
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
#define MZP_R8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define MZP_I8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
#define MZP_X8(v, i) "+r"((v)[i]), "+r"((v)[i + 1]), "+r"((v)[i + 2]), "+r"((v)[i + 3]), "+r"((v)[i + 4]), "+r"((v)[i + 5]), "+r"((v)[i + 6]), "+r"((v)[i + 7])
#define MZP_REGS32 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"
__device__ __forceinline__ void tm_load32(uint32_t (&v)[32], uint32_t at) {      // not there before tm_loaded
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " MZP_REGS32 ", [%32];" : MZP_R8(v, 0), MZP_R8(v, 8), MZP_R8(v, 16), MZP_R8(v, 24) : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_loaded(uint32_t (&v)[32]) {                   // names the registers, so that nothing reads them above it
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MZP_X8(v, 0), MZP_X8(v, 8), MZP_X8(v, 16), MZP_X8(v, 24) :: "memory");
}
__device__ __forceinline__ void tm_store32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " MZP_REGS32 ";" ::MZP_I8(v, 0), MZP_I8(v, 8), MZP_I8(v, 16), MZP_I8(v, 24), "r"(at) : "memory");
}
__device__ __forceinline__ void tm_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) { uint32_t v; asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a)); return v; }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
// two values times f plus c
__device__ __forceinline__ void mul_add2(float& a, float& b, float f, float c) {
  asm("{\n\t.reg .b64 x, f, c;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 f, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\tfma.rn.f32x2 x, x, f, c;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b) : "f"(f), "f"(c));
}
__device__ __forceinline__ uint32_t half2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ void stg256(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

// Eight codes -> their levels, each plus 1024 as an f16 number (0x6400 + level).  A selector's top bit asks for the sign of a level, which is zero: so the two
// permutes of a nibble are zero exactly where they are not meant, and their results are or-ed.
__device__ __forceinline__ void levels8(uint32_t codes, const uint4& book, uint32_t (&u)[4]) {
  const uint32_t other = codes ^ 0x88888888u;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t four = prmt(book.x, book.y, codes >> (16 * k)) | prmt(book.z, book.w, other >> (16 * k));
    u[2 * k] = prmt(four, 0x64646464u, 0x4140u);
    u[2 * k + 1] = prmt(four, 0x64646464u, 0x4342u);
  }
}

// Lists a CTA's part of the line, SEGMENTS runs of one unit at a time.  For a whole warp.
struct Lister {
  long long steps, records, f0, f1;              // before group g; the part
  int g, unit;                                   // next
  // finds the line's length and the group that the part begins in; CTA 0 writes down where groups begin
  __device__ __forceinline__ bool begin(const PrefixArgs& p, int lane) {
    const int cta = blockIdx.x, n = p.out.n_groups;
    auto size = [&](int i, long long& st, long long& re) {
      st = re = 0;
      if (i < n) {
        const MzpGroup info = p.out.groups[i];
        const MzpTiles tiles(info.rows);
        st = (long long)info.pages * (tiles.weight * tiles.count) * p.c.kv_heads;
        re = info.pages > 0 ? (long long)info.rows * p.c.kv_heads : 0;
      }
    };
    long long st, re, total = 0, gain = 0;
    int heaviest = 1;
    for (int i = lane; i < n; i += 32) {
      size(i, st, re);
      total += st;
      const MzpGroup info = p.out.groups[i];
      const MzpTiles tiles(info.rows);
      if (info.pages > 0) heaviest = max(heaviest, tiles.weight);
      gain += mzp_gain(info.pages, p.c.kv_heads, (long long)info.members * p.out.passes, p.out.nr, tiles.cost());
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      gain += __shfl_xor_sync(0xffffffffu, gain, o);
    }
    heaviest = (int)__reduce_max_sync(0xffffffffu, (unsigned)heaviest);
    if (gain < mzp_gain_needed(p.out.sms, p.c.head_dim)) total = 0;      // then nothing is shared, and the other kernels see that
    const MzpLine line(total, heaviest, gridDim.x);
    const bool some = cta < line.ctas;
    f0 = some ? line.start(cta) : 0;
    f1 = some ? line.start(cta + 1) : 0;
    long long before_s = 0, before_r = 0;
    g = n;
    for (int i0 = 0; i0 < n && total > 0 && (cta == 0 || g == n); i0 += 32) {
      size(i0 + lane, st, re);
      long long ss = st, rr = re;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, ss, o), b = __shfl_up_sync(0xffffffffu, rr, o);
        if (lane >= o) { ss += a; rr += b; }
      }
      const long long my_s = before_s + ss - st, my_r = before_r + rr - re;
      if (cta == 0 && i0 + lane < n) p.out.sums[i0 + lane] = {my_s, my_r, 0, 0};
      const uint32_t mine = __ballot_sync(0xffffffffu, my_s <= f0 && f0 < my_s + st);
      if (some && mine) {
        const int from = __ffs(mine) - 1;
        g = i0 + from;
        steps = __shfl_sync(0xffffffffu, my_s, from);
        records = __shfl_sync(0xffffffffu, my_r, from);
      }
      before_s += __shfl_sync(0xffffffffu, ss, 31);
      before_r += __shfl_sync(0xffffffffu, rr, 31);
    }
    if (cta == 0 && lane == 0) p.out.sums[n] = {total, before_r, heaviest, 0};
    unit = -1;
    return some;
  }
  __device__ __forceinline__ void list(const PrefixArgs& p, PrefixShared& x, int lane) {
    int n = 0;
    while (g < p.out.n_groups && steps < f1 && n < SEGMENTS) {
      const MzpGroup info = p.out.groups[g];
      if (info.pages > 0) {
        const MzpTiles tiles(info.rows);
        const long long len = (long long)info.pages * tiles.weight;
        const int units = p.c.kv_heads * tiles.count;
        if (unit < 0) unit = f0 > steps ? (int)min((f0 - steps) / len, (long long)units) : 0;
        const int end = (int)min((long long)units, (f1 - steps + len - 1) / len);
        while (unit < end && n < SEGMENTS) {
          const int u = unit + lane;
          const long long at = steps + u * len;
          Segment s;
          const MzpRun run(at, info.pages, tiles.weight, f0, f1);
          s.page = run.page;
          s.count = run.count;
          s.head = u / tiles.count;
          s.m0 = (u - s.head * tiles.count) * tiles.rows;
          s.first = info.first; s.row = info.row;
          s.rows = min(tiles.rows, info.rows - s.m0);
          s.record = records + (long long)s.head * info.rows + s.m0 + (long long)MZP_TILE_ROWS * blockIdx.x;
          s.pad = 0;
          const bool mine = u < end && s.count > 0;
          const uint32_t all = __ballot_sync(0xffffffffu, mine);
          const int place = n + __popc(all & ((1u << lane) - 1));
          if (mine && place < SEGMENTS) x.seg[place] = s;
          // the first one that does not fit begins the next list
          const uint32_t late = __ballot_sync(0xffffffffu, mine && place >= SEGMENTS);
          unit += late ? __ffs(late) - 1 : 32;
          n = min(n + __popc(all), SEGMENTS);
        }
        if (unit < end) break;                   // full
        steps += units * len;
        records += (long long)p.c.kv_heads * info.rows;
      }
      ++g;
      unit = 0;
    }
    if (lane == 0) { x.segments = n; x.more = n == SEGMENTS; }
  }
};

template <int D, bool BF>
__global__ void __launch_bounds__(PREFIX_THREADS, 1) prefix_kernel(const PrefixArgs p, const uint8_t* __restrict__ book_table) {
  using S = PrefixSmem<D>;
  constexpr int PB = S::PAGE_BYTES, HALF = MZP_TILE_ROWS / 2;
  extern __shared__ uint8_t window[];
  uint8_t* smem = window + (S::ALIGN - smem_u32(window) % S::ALIGN) % S::ALIGN;
  __shared__ PrefixShared x;
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](unsigned long long& b) { return smem_u32(&b); };
  auto everyone = [&]() { asm volatile("bar.sync 0;" ::: "memory"); };
  if (tid == 0) {
    x.failed = p.fail_waits;
    for (int i = 0; i < RAWS; ++i) { bar_init(bar(x.raw_full[i]), 1); bar_init(bar(x.raw_free[i]), 4); }
    for (int i = 0; i < S::SCALES; ++i) bar_init(bar(x.scaled[i]), 1);
    for (int i = 0; i < 2 * RING; ++i) { bar_init(bar(x.full[i / RING][i % RING]), 4); bar_init(bar(x.free[i / RING][i % RING]), 1); }
    for (int i = 0; i < 4; ++i) { bar_init(bar(x.s_full[i]), 1); bar_init(bar(x.p_full[i]), 4); bar_init(bar(x.o_done[i]), 1); }
    bar_init(bar(x.q_full), SOFTMAX_WARPS);
    bar_init(bar(x.end), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < MZP_BOOKS * MZP_LEVELS / 16) ((uint4*)(smem + S::BOOK))[tid] = ((const uint4*)book_table)[tid];
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tm_before();
  }
  Lister lister;
  if (warp == FEEDER) {
    lister.begin(p, lane);
    lister.list(p, x, lane);
  }
  everyone();
  tm_after();
  constexpr uint32_t tmem = 0;                   // all columns: they begin at 0
  if (tid == 0 && x.tmem != 0) x.failed = 1;
  volatile int* failed = &x.failed;

  if (warp >= SOFTMAX_WARPS) {
    registers<OTHER_REGS, false>();
    if (warp == ISSUER) {
      // ---- products: a job's logits as soon as the P that stands in their place has been used.  One elected lane issues, and all that it issues with is the same for the warp and shown
      // to be (maxima and votes over it), so that it stands in uniform registers.  A look at a barrier takes 200 cycles behind products, as it queues with them: so a job looks at
      // all of its barriers at once, while the products before it run (20 products with one look 776 cycles, with three looks one after the other 1420)
      auto same = [&](int v) { return (int)__reduce_max_sync(0xffffffffu, (unsigned)v); };
      auto wait3 = [&](uint32_t b0, uint32_t parity0, uint32_t b1, uint32_t parity1, uint32_t b2, uint32_t parity2) {
#ifdef MZ_BOUNDS
        if (__any_sync(0xffffffffu, *failed)) return;        // a test makes every wait run out
#endif
        for (int it = 0; it < SPIN_LIMIT; ++it) {
          uint32_t done;
          asm volatile("{\n\t.reg .pred p, q, r;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
                       "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\tand.pred p, p, q;\n\tand.pred p, p, r;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
                       : "=r"(done) : "r"(b0), "r"(parity0), "r"(b1), "r"(parity1), "r"(b2), "r"(parity2) : "memory");
          if (__all_sync(0xffffffffu, done != 0)) return;
          if ((it & 63) == 63 && __any_sync(0xffffffffu, *failed)) return;
        }
        *failed = 1;
      };
      // of the CTA so far: segments, jobs whose logits, whose outputs were issued; pages of both, and the block of logits that is the page's where the streams share rows
      int segment = 0, ahead = 0, behind = 0, k_page = 0, v_page = 0, k_block = 0, v_block = 0;
      const uint32_t keys = same((int)(sbase + S::KEYS) >> 4), values = same((int)(sbase + S::VALUES) >> 4);
      const uint32_t s_full = bar(x.s_full[0]), p_full = bar(x.p_full[0]), o_done = bar(x.o_done[0]), q_full = bar(x.q_full);
      const uint32_t k_full = bar(x.full[0][0]), k_free = bar(x.free[0][0]), v_full = bar(x.full[1][0]), v_free = bar(x.free[1][0]);
      for (int n = same(x.segments); n > 0; n = same(x.segments)) {
        for (int i0 = 0; i0 < n; ++i0, ++segment) {
          const bool both = same(x.seg[i0].rows) > HALF;     // two tiles of rows take each page; otherwise the streams take the pages in turn
          const int jobs = same(x.seg[i0].count) << (both ? 1 : 0), lead = both ? 2 : 3;
          for (int i = 0; i < jobs + lead; ++i) {
            const int j = i - lead;
            // the queries' barrier, which was passed or has to be, stands for what a job does not need
            const uint32_t q_phase = segment & 1, k_bar = i < jobs ? k_full + 8 * (k_page % RING) : q_full, k_want = i < jobs ? k_page / RING & 1 : q_phase;
            if (j >= 0) wait3(v_full + 8 * (v_page % RING), v_page / RING & 1, p_full + 8 * (behind & 3), behind >> 2 & 1, k_bar, k_want);
            else wait3(q_full, q_phase, q_full, q_phase, k_bar, k_want);
            tm_after();
            // short loops: a scheduler's instruction cache is full of the other duties, and what is executed once a page has to be fetched each time
            if (j >= 0) {
              const bool last = !both || (j & 1);
              const uint32_t vd = values + v_page % V_STAGES * (2 * S::PLANE >> 4), t_o = S::TM_O + (j & 1) * D, t_s = S::tm_s(both) + (both ? j & 1 : v_block) * MZP_PAGE;
              if (elect()) {
#pragma unroll 1
                for (int part = 0; part < 3; ++part) {       // P and V as value and remainder: all but the remainders' product
                  const uint32_t p = t_s + (part == 1 ? MZP_PAGE / 2 : 0), v = vd + (part == 2 ? S::PLANE >> 4 : 0);
#pragma unroll
                  for (int k = 0; k < MZP_PAGE / 16; ++k) umma16<D>(t_o, p + k * 8, v + k * OPERAND_STEP, part + k > 0 || (j >> 1) % SUM_JOBS != 0);
                }
                umma_commit(o_done + 8 * (behind & 3));
                if (last) umma_commit(v_free + 8 * (v_page % RING));
              }
              __syncwarp();
              ++behind;
              if (last) {
                ++v_page;
                v_block = v_block == BLOCKS - 1 ? 0 : v_block + 1;
              }
            }
            if (i < jobs) {
              const bool last = !both || (i & 1);
              const uint32_t kd = keys + k_page % K_STAGES * (2 * S::PLANE >> 4), t_q = S::TM_Q + (both ? (i & 1) * (D / 2) : 0), t_s = S::tm_s(both) + (both ? i & 1 : k_block) * MZP_PAGE;
              if (elect()) {
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {       // remainder, then value: what is summed first is small, and so is what the tensor cores cut off of it
                  const uint32_t k0 = kd + (part == 0 ? S::PLANE >> 4 : 0);
#pragma unroll ISSUE_UNROLL
                  for (int k = 0; k < D / 16; ++k) umma16<MZP_PAGE>(t_s, t_q + k * 8, k0 + k * OPERAND_STEP, part + k > 0);
                }
                umma_commit(s_full + 8 * (ahead & 3));
                if (last) umma_commit(k_free + 8 * (k_page % RING));
              }
              __syncwarp();
              ++ahead;
              if (last) {
                ++k_page;
                k_block = k_block == BLOCKS - 1 ? 0 : k_block + 1;
              }
            }
          }
        }
        everyone();
        everyone();
      }
    } else if (warp == FEEDER) {
      // ---- pages as they are, four ahead; then the next list
      const uint8_t* store = (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer;
      int pages = 0, sent = 0;
      while (x.segments > 0) {
        for (int i0 = 0; i0 < x.segments; ++i0) {
          const Segment seg = x.seg[i0];
          const int* table = c.block_table + (long long)seg.row * c.width + seg.page;
          int ids = lane < seg.count ? table[lane] : -1;
          for (int at = 0; at < seg.count; at += 32) {
            const int coming = at + 32 + lane < seg.count ? table[at + 32 + lane] : -1;
            for (int k = 0; k < min(32, seg.count - at); ++k, ++pages) {
              const int slot = pages % RAWS, id = __shfl_sync(0xffffffffu, ids, k);
              const bool there = id >= 0 && id < c.pages;    // a page that is not there any more has T = 0
              bar_wait(bar(x.raw_free[slot]), (pages / RAWS & 1) ^ 1, failed);
              const bool fine = !*failed;
              if (fine) sent = pages + 1;
              if (fine && elect()) {
                x.there[slot] = there;
                if (there) {
                  const uint8_t* src = store + (long long)id * c.store_stride_page + (long long)seg.head * PB;
                  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(x.raw_full[slot])), "n"(PB) : "memory");
                  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                               ::"r"(sbase + S::RAW + slot * PB), "l"(src), "n"(PB), "r"(bar(x.raw_full[slot])) : "memory");
                } else {
                  bar_arrive(bar(x.raw_full[slot]));
                }
              }
              __syncwarp();
            }
            ids = coming;
          }
        }
        everyone();                              // the list has been read
        if (x.more) lister.list(p, x, lane);
        else if (lane == 0) x.segments = 0;
        everyone();
      }
      // copies land before the CTA ends, whatever else went wrong
      for (int j = max(0, sent - RAWS); j < sent; ++j)
        for (int k = 0; k < SPIN_LIMIT && !bar_test(bar(x.raw_full[j % RAWS]), j / RAWS & 1); ++k) {}
    } else if ((warp & 3) == 3) {
      // ---- words: the powers of two above a page's largest key and value (f16 has them below 2^14), and of every row of codes {scale, 1024 + zero level, anchor (as pairs), place of
      // its book}.  Here, and not where the levels are made, as this scheduler has the least to do
      const uint32_t terms = sbase + S::TERMS;
      int page = warp == DECODER ? 0 : 1, pages = 0;
      while (x.segments > 0) {
        for (int i0 = 0; i0 < x.segments; ++i0) pages += x.seg[i0].count;
        for (; page < pages; page += 2) {
          const int slot = page % RAWS;
          const uint32_t raw = sbase + S::RAW + slot * PB + 32 * D;
          static_assert(RAWS % 2 == 0, "the page before in this place was this decoder's: it has waited for its phase");
          bar_wait(bar(x.raw_full[slot]), page / RAWS & 1, failed);
          const bool there = x.there[slot];
          int e[2];
#pragma unroll
          for (int side = 0; side < 2; ++side) {             // two f16 numbers (T, and A or z) at a time
            uint32_t word[D / 32], m = 0;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              word[i] = there ? lds32(raw + side * 36 * D + 128 * i + 4 * lane) : 0u;
              m = __vmaxu2(m, word[i] & 0x7fff7fffu);
            }
            const uint32_t t_max = warp_max_u32(m & 0xffffu), a_max = warp_max_u32(m >> 16);
            const float top = fmaf(4.f, __half2float(__ushort_as_half((unsigned short)t_max)), a_max >= 128u ? __half2float(__ushort_as_half((unsigned short)a_max)) : 0.f);
            e[side] = min(max((int)(__float_as_uint(top) >> 23) - 126, -30), 30) - 14;
            const float scale = pow2(-e[side]);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const MzpRow row = mzp_row(word[i]);
              const float unit = row.t * scale * 0.03125f, anchor = row.a * scale;
              sts128(terms + ((slot * 2 + side) * D + 32 * i + lane) * 16, half2_bits(__floats2half2_rn(unit, unit)), (0x6400u | row.z) * 0x10001u,
                     half2_bits(__floats2half2_rn(anchor, anchor)), row.z * 16);
            }
          }
          if (lane == 0) x.scale[page % S::SCALES] = make_int2(e[0], e[1]);
          __syncwarp();
          if (lane == 0) bar_arrive(bar(x.scaled[page % S::SCALES]));
        }
        everyone();
        everyone();
      }
    } else {
      // ---- levels: a thread has a row of 64 keys, then one of 64 values (head_dim 64: half of either).  Rolled loops: what all duties execute has to stay near the
      // schedulers' instruction caches
      const int member = (warp - SOFTMAX_WARPS) / 4 * 3 + (warp & 3), t = (member & 3) * 32 + lane;
      constexpr int PIECES = D == 128 ? 2 : 1;               // of 32 codes
      const int part = t / 64, token = t % 64, ch = t % D;
      // of keys, of values: the row's number in the page, its place in the operand
      const int k_row = ch, v_row = D == 128 ? 2 * token + part : token, piece0 = D == 128 ? 0 : part;
      const uint32_t k_at = sbase + S::KEYS + 128 * ch, v_at = sbase + S::VALUES + (D == 128 ? part * MZP_PAGE * 128 : 0) + 128 * token;
      const uint32_t k_turn = (ch & 7) << 4, v_turn = (token & 7) << 4, terms = sbase + S::TERMS;
      const uint32_t sbook = sbase + S::BOOK;                // a place in it is masked: where waits ran out, terms are whatever stood there
      int page = member >> 2, pages = 0, slot = page;
      uint32_t raw_phase = 0;
      while (x.segments > 0) {
        for (int i0 = 0; i0 < x.segments; ++i0) pages += x.seg[i0].count;
        for (; page < pages; page += TEAMS) {
          const uint32_t raw = sbase + S::RAW + slot * PB;
          bar_wait(bar(x.scaled[page % S::SCALES]), page / S::SCALES & 1, failed);
          bar_wait(bar(x.raw_full[slot]), raw_phase, failed);
#pragma unroll 1
          for (int side = 0; side < 2; ++side) {
            const int stages = side ? V_STAGES : K_STAGES;
            if (page >= stages) bar_wait(bar(x.free[side][(page - stages) % RING]), (page - stages) / RING & 1, failed);
            const uint32_t at = (side ? v_at : k_at) + page % stages * 2 * S::PLANE, turn = side ? v_turn : k_turn, row = side ? v_row : k_row;
            const uint4 term = lds128(terms + ((slot * 2 + side) * D + row) * 16), book = book128(sbook + (term.w & 0x7f0u));
            const uint32_t from = raw + side * 36 * D + 32 * row;
            const __half2 step = bits_half2(term.x), zero = bits_half2(term.y);
            if (!__any_sync(0xffffffffu, term.z)) {
#pragma unroll 1
              for (int piece = piece0; piece < piece0 + PIECES; ++piece) {
                const uint4 codes = lds128(from + 16 * piece);
#pragma unroll
                for (int q = 0; q < 4; ++q) {    // eight values
                  uint32_t u[4], lo[4];
                  levels8((&codes.x)[q], book, u);
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const __half2 w = __hsub2(bits_half2(u[k]), zero), h = __hmul2(w, step);
                    u[k] = half2_bits(h);
                    lo[k] = half2_bits(__hfma2(w, step, __hneg2(h)));      // exact
                  }
                  const uint32_t dst = at + ((64 * piece + 16 * q) ^ turn);
                  sts128(dst, u[0], u[1], u[2], u[3]);
                  sts128(dst + S::PLANE, lo[0], lo[1], lo[2], lo[3]);
                }
              }
            } else {                             // rows that do not straddle zero: the sum has more than 22 bits' worth of terms, so in fp32
              const float unit = __low2float(step), anchor = __low2float(bits_half2(term.z));
#pragma unroll 1
              for (int piece = piece0; piece < piece0 + PIECES; ++piece) {
                const uint4 codes = lds128(from + 16 * piece);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  uint32_t u[4], lo[4];
                  levels8((&codes.x)[q], book, u);
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const float2 w = __half22float2(__hsub2(bits_half2(u[k]), zero));
                    const float a = fmaf(w.x, unit, anchor), b = fmaf(w.y, unit, anchor);
                    const __half2 h = __floats2half2_rn(a, b);
                    const float2 f = __half22float2(h);
                    u[k] = half2_bits(h);
                    lo[k] = half2_bits(__floats2half2_rn(a - f.x, b - f.y));
                  }
                  const uint32_t dst = at + ((64 * piece + 16 * q) ^ turn);
                  sts128(dst, u[0], u[1], u[2], u[3]);
                  sts128(dst + S::PLANE, lo[0], lo[1], lo[2], lo[3]);
                }
              }
            }
            fence_operands();
            __syncwarp();
            if (lane == 0) {
              bar_arrive(bar(x.full[side][page % RING]));
              if (side) bar_arrive(bar(x.raw_free[slot]));
            }
          }
          slot += TEAMS;
          if (slot >= RAWS) { slot -= RAWS; raw_phase ^= 1; }
        }
        everyone();
        everyone();
      }
    }
  } else {
    // ---- softmax: a thread has a query row
    registers<SOFTMAX_REGS, true>();
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_o = lanes + S::TM_O + s * D;
    int pages = 0, first_job = 0;                            // of the CTA so far
    float4* const part = p.out.part + ((long long)blockIdx.x * 2 + s) * (D / 4) * HALF + r;
    while (x.segments > 0) {
    for (int i0 = 0; i0 < x.segments; ++i0) {
      const Segment seg = x.seg[i0];
      const bool both = seg.rows > HALF;
      const int m = (both ? s * HALF : 0) + r;               // row of the tile
      const bool here = m < seg.rows;
      const bool some = __any_sync(0xffffffffu, here);       // of the warp's rows
      float rowf = 0.f;
      {
        // queries: scaled by a power of two into f16's range, where both 16-bit types are exact
        constexpr int DT = BF ? MZ_BF16 : MZ_F16;
        const int qr = (seg.m0 + m) % p.qrows, b = seg.first + (seg.m0 + m) / p.qrows;
        const uint16_t* q = p.query + (long long)b * p.qsb + (long long)(qr / p.group) * p.qsl + (long long)(seg.head * p.group + qr % p.group) * p.qsh;
        uint32_t top = 0;
        uint4 raw[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          raw[i] = make_uint4(0, 0, 0, 0);
          if (here) raw[i] = ((const uint4*)q)[i];
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = (&raw[i].x)[k];
            top = max(top, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
          }
        }
        const uint32_t size = __float_as_uint(mz_u16_to_float((uint16_t)top, DT));       // NaN is the largest
        const int e = max((int)(size >> 23) - 134, -60), e1 = e >> 1, e2 = e - e1;       // |q| 2^-e < 2^8
        const bool wild = size >= 0x7f800000u;                                           // infinity or NaN: the row's logits are NaN
        const float down1 = pow2(-e1), down2 = pow2(-e2) * (p.scaling < 0.f ? -1.f : 1.f);
        rowf = pow2(e1) * fabsf(p.scaling) * pow2(e2);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t w = (&raw[8 * h + i / 4].x)[i & 3];
            const float a = mz_u16_to_float((uint16_t)(w & 0xffffu), DT) * down1 * down2, b2 = mz_u16_to_float((uint16_t)(w >> 16), DT) * down1 * down2;
            v[i] = wild ? 0x7fff7fffu : half2_bits(__floats2half2_rn(a, b2));
          }
          if (both || s == 0) tm_store32(lanes + S::TM_Q + s * (D / 2) + 32 * h, v);
        }
        tm_stored();
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(x.q_full));
      }
      float M = -INFINITY, l = 0.f, M_part = 0.f;            // M_part: that of the sums so far
      auto keep = [&](bool more) {                           // adds the accumulator to them
        const float f = more ? ex2(M_part - (M == -INFINITY ? 0.f : M)) : 0.f;
        M_part = M;
#pragma unroll 1
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          float4 sum[8];
          tm_load32(o, t_o + 32 * h);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (more) sum[i] = part[(8 * h + i) * HALF];
          }
          tm_loaded(o);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            part[(8 * h + i) * HALF] = make_float4(fmaf(sum[i].x, f, __uint_as_float(o[4 * i])), fmaf(sum[i].y, f, __uint_as_float(o[4 * i + 1])),
                                                   fmaf(sum[i].z, f, __uint_as_float(o[4 * i + 2])), fmaf(sum[i].w, f, __uint_as_float(o[4 * i + 3])));
        }
      };
      const int jobs = both ? 2 * seg.count : seg.count, mine = (jobs + 1 - s) / 2;        // of the segment, of this stream
      for (int j = 0; j < mine; ++j) {
        const int i = 2 * j + s, job = first_job + i, page = pages + (both ? j : i);
        const uint32_t t_s = lanes + S::tm_s(both) + (both ? s : page % BLOCKS) * MZP_PAGE;
        bar_wait(bar(x.scaled[page % S::SCALES]), page / S::SCALES & 1, failed);
        bar_wait(bar(x.s_full[job & 3]), job >> 2 & 1, failed);
        tm_after();
        if (some) {
          const int2 sc = x.scale[page % S::SCALES];
          const float f = rowf * pow2(sc.x), ev = (float)sc.y;
          // P under the maximum so far, of the first pages' logits: its sum stays below 2^15 unless that is passed by 8 or so.  Then the maximum is found and P taken once more
          uint32_t w[32], rest[32];
          float total = 0.f;
          bool known = j > 0;
          for (int turn = 0;; ++turn) {
            if (known) {
              const float add = ev + 7.f - (M == -INFINITY ? 0.f : M);
              float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t v[32];
                tm_load32(v, t_s + 32 * h);
                tm_loaded(v);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  float a = __uint_as_float(v[i]), b = __uint_as_float(v[i + 1]), c2 = __uint_as_float(v[i + 2]), d = __uint_as_float(v[i + 3]);
                  mul_add2(a, b, f, add);
                  mul_add2(c2, d, f, add);
                  a = ex2(a); b = ex2(b); c2 = ex2(c2); d = ex2(d);
                  const __half2 p0 = __floats2half2_rn(a, b), p1 = __floats2half2_rn(c2, d);
                  w[16 * h + i / 2] = half2_bits(p0);
                  w[16 * h + i / 2 + 1] = half2_bits(p1);
                  add2(sum[0], sum[1], a, b);
                  add2(sum[2], sum[3], c2, d);
                  const float2 f0 = __half22float2(p0), f1 = __half22float2(p1);
                  fma2(a, b, f0.x, f0.y, -1.f);              // exact
                  fma2(c2, d, f1.x, f1.y, -1.f);
                  rest[16 * h + i / 2] = half2_bits(__floats2half2_rn(a, b));
                  rest[16 * h + i / 2 + 1] = half2_bits(__floats2half2_rn(c2, d));
                }
              }
              total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
              if (turn > 0 || !__any_sync(0xffffffffu, !(total <= 32768.f))) break;
            }
            float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              uint32_t v[32];
              tm_load32(v, t_s + 32 * h);
              tm_loaded(v);
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                top0 = max3(top0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                top1 = max3(top1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
              }
            }
            const float t = fmaf(fmaxf(top0, top1), f, ev);
            if (!known) {
              M = t;
              known = true;
              continue;
            }
            const bool more = !(total <= 32768.f) && t > M;  // where the sum is NaN it stays
            const float fix = more ? ex2(M - t) : 1.f;
            if (more) M = t;
            l *= fix;
            bar_wait(bar(x.o_done[(job - 2) & 3]), (job - 2) >> 2 & 1, failed);          // the stream's last product is in
            tm_after();
#pragma unroll 1
            for (int h = 0; h < D / 32; ++h) {
              uint32_t o[32];
              tm_load32(o, t_o + 32 * h);
              tm_loaded(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
              tm_store32(t_o + 32 * h, o);
            }
          }
          tm_store32(t_s, w);                    // over logits that have been read
          tm_store32(t_s + 32, rest);
          l = fmaf(total, pow2(-sc.y - 7), l);
          tm_stored();
          if (j > 0 && j % SUM_JOBS == 0) {      // this job's product begins a new sum
            bar_wait(bar(x.o_done[(job - 2) & 3]), (job - 2) >> 2 & 1, failed);
            tm_after();
            keep(j > SUM_JOBS);
          }
        }
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(x.p_full[job & 3]));
      }
      // ---- records
      if (mine > 0) {
        const int job = first_job + 2 * (mine - 1) + s;
        bar_wait(bar(x.o_done[job & 3]), job >> 2 & 1, failed);
      }
      tm_after();
      const bool kept = jobs > 2 * SUM_JOBS;                 // of either stream
      if (kept && some) keep(mine > SUM_JOBS);
      const bool bad = *failed != 0;
      const long long at = seg.record + m;
      const bool inside = here && MZ_IN_BOUNDS(at, p.out.records, 21);
      float f_mine = 0.0078125f, f_other = 0.f;              // P has 2^7
      uint32_t t_other = t_o;
      int d0 = 0, d1 = D;
      if (!both) {
        // both streams have parts of the same rows: each writes half of the channels
        x.ml[s][r] = make_float2(mine > 0 ? M : -INFINITY, l);
        tm_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tm_after();
        const float2 o = x.ml[s ^ 1][r];
        const float top = fmaxf(x.ml[s][r].x, o.x), ref = top == -INFINITY ? 0.f : top;
        const float g0 = mine > 0 ? ex2(M - ref) : 0.f, g1 = seg.count > 1 || s == 1 ? ex2(o.x - ref) : 0.f;
        l = l * g0 + o.y * g1;
        M = top;
        f_mine *= g0;
        f_other = 0.0078125f * g1;
        t_other = lanes + S::TM_O + (s ^ 1) * D;
        d0 = s * (D / 2);
        d1 = d0 + D / 2;
      }
#pragma unroll 1
      for (int d = d0; d < d1; d += 32) {
        float out[32];
        if (kept) {
          const float4* other = part + (s ? -1 : 1) * (D / 4) * HALF;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 a = part[(d / 4 + i) * HALF];
            float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!both) b = other[(d / 4 + i) * HALF];
            out[4 * i] = a.x * f_mine + b.x * f_other; out[4 * i + 1] = a.y * f_mine + b.y * f_other;
            out[4 * i + 2] = a.z * f_mine + b.z * f_other; out[4 * i + 3] = a.w * f_mine + b.w * f_other;
          }
        } else {
          uint32_t v[32], u[32];
          tm_load32(v, t_o + d);
          tm_load32(u, t_other + d);
          tm_loaded(v);
          tm_loaded(u);
          // a stream that had no page left nothing in its accumulator
#pragma unroll
          for (int i = 0; i < 32; ++i) out[i] = (mine > 0 ? __uint_as_float(v[i]) * f_mine : 0.f) + (!both && f_other != 0.f ? __uint_as_float(u[i]) * f_other : 0.f);
        }
        if (inside) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) stg256(p.out.acc + at * D + d + i, out + i);
        }
      }
      if (inside && (both || s == 0)) p.out.ml[at] = bad ? make_float2(INFINITY, __int_as_float(0x7fffffff)) : make_float2(M, l);
      tm_before();
      if (!both) asm volatile("bar.sync 1, 256;" ::: "memory");          // x.ml is free again
      pages += seg.count;
      first_job += jobs;
    }
    everyone();
    everyone();
    }
  }
  if (warp == ISSUER && elect()) {               // the products are done, and so is what they signal
    umma_commit(bar(x.end));
    for (int k = 0; k < SPIN_LIMIT && !bar_test(bar(x.end), 0); ++k) {}
  }
  tm_before();
  everyone();
  if (warp == ISSUER) {
    tm_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TM_COLS));
  }
}

template <int D, bool BF>
int launch_prefix(const PrefixArgs& p, const uint8_t* book, cudaStream_t st) {
  auto kern = prefix_kernel<D, BF>;
  static std::atomic<unsigned> ready[8];         // a bit per device: its limit is set
  int dev = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  const bool known = dev < 256 && (ready[dev >> 5].load(std::memory_order_relaxed) >> (dev & 31) & 1u);
  if (!known) {
    MZ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PrefixSmem<D>::TOTAL));
    if (dev < 256) ready[dev >> 5].fetch_or(1u << (dev & 31), std::memory_order_relaxed);
  }
  plan_kernel<<<p.out.n_groups * PLAN_CTAS, PLAN_THREADS, 0, st>>>(p);
  MZ_LAUNCH_CHECK("paged prefix plan");
  kern<<<p.out.grid, PREFIX_THREADS, PrefixSmem<D>::TOTAL, st>>>(p, book);
  MZ_LAUNCH_CHECK("paged prefix");
  return MZ_OK;
}
}  // namespace
}  // namespace mzp

void mzp_prefix_shape(const mz_paged_cache* c, int batch, int n_groups, int qrows, int sms, MzpPrefixShape* s) {
  auto up = [](size_t n) { return (n + 127) / 128 * 128; };
  s->grid = sms;
  s->records = (long long)batch * qrows * c->kv_heads + (long long)MZP_TILE_ROWS * s->grid;
  s->skip_at = 0;
  s->group_of_at = up(batch * sizeof(int));
  s->groups_at = s->group_of_at + up(batch * sizeof(int));
  s->sums_at = s->groups_at + up(n_groups * sizeof(MzpGroup));
  s->ml_at = s->sums_at + up((n_groups + 1) * sizeof(MzpSums));
  s->acc_at = s->ml_at + up(s->records * sizeof(float2));
  s->part_at = s->acc_at + up(s->records * c->head_dim * sizeof(float));
  s->bytes = s->part_at + (size_t)s->grid * MZP_TILE_ROWS * c->head_dim * sizeof(float);
}

int mzp_prefix_launch(const mz_paged_cache& c, int layer, const mz_paged_attention_args& args, const mz_paged_view& view, const MzpPrefixShape& s, uint8_t* workspace,
                      int longest, int nr, int passes, const uint8_t* book, cudaStream_t stream, MzpPrefix* out) {
  mzp::PrefixArgs p = {};
  p.c = c;
  p.query = (const uint16_t*)args.query;
  p.qsb = args.q_stride_b; p.qsl = args.q_stride_l; p.qsh = args.q_stride_h;
  p.rows = args.rows;
  p.offsets = view.groups;
  p.layer = layer;
  p.batch = args.batch; p.q_len = args.q_len;
  p.group = args.q_heads / c.kv_heads;
  p.qrows = p.group * args.q_len;
  p.longest = longest;
  p.scaling = args.scaling * mzp::LOG2E;
  p.out.skip = (int*)(workspace + s.skip_at);
  p.out.group_of = (int*)(workspace + s.group_of_at);
  p.out.groups = (MzpGroup*)(workspace + s.groups_at);
  p.out.sums = (MzpSums*)(workspace + s.sums_at);
  p.out.ml = (float2*)(workspace + s.ml_at);
  p.out.acc = (float*)(workspace + s.acc_at);
  p.out.part = (float4*)(workspace + s.part_at);
  p.out.n_groups = view.n_groups;
  p.out.grid = p.out.sms = s.grid;               // a CTA per multiprocessor
  p.out.nr = nr;
  p.out.passes = passes;
  p.out.records = s.records;
  p.fail_waits = mz_waits_fail();
  *out = p.out;
  const bool bf = c.kv_dtype == MZ_BF16;
  if (c.head_dim == 128) return bf ? mzp::launch_prefix<128, true>(p, book, stream) : mzp::launch_prefix<128, false>(p, book, stream);
  return bf ? mzp::launch_prefix<64, true>(p, book, stream) : mzp::launch_prefix<64, false>(p, book, stream);
}
