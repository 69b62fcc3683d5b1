// Paged cache: attention of rows in groups over the pages that a group's rows have in common (sm_100a, tcgen05).
//
// Mathematics.  A code stands for A + T (u - z) / 32 (mz_paged.cuh).  For a tile of query rows and a page of 64 tokens
//   S = q K^T          K as two f16 numbers, value and remainder: 22 bits of every key; q (bf16 or f16) is exact in f16 once its row is scaled by a power of two
//   P = exp2(S f + e - M),  O += P V          P and V are rounded to f16 (2^-12 of each value), sums are fp32
// Keys and values of a page are scaled into f16's range by powers of two, ek and ev; f takes ek back.  ev is taken back by the softmax itself: M is the running
// maximum not of the logits t but of t + ev, so P V has one scale whatever the pages' ranges, P stays below 2^15, and l sums P 2^-ev in fp32.  M moves when t + ev
// passes it by more than 8 (the output in tensor memory is scaled then), so P has 7 bits in reserve below 2^15 and what is lost is under 2^-31 of the largest.
#include <algorithm>
#include <atomic>

#include "mz_paged_prefix.cuh"

namespace mzp {
namespace {
// Warps by duty: 0 .. 7 softmax (a group of four per stream), 8 .. 15 levels, 16 issues the products; the three beside it are there for its warpgroup's registers
constexpr int SOFTMAX_WARPS = 8, LEVEL_WARPS = 8, ISSUER = SOFTMAX_WARPS + LEVEL_WARPS, PREFIX_THREADS = 32 * (ISSUER + 4);
// of the 96 x 640 registers that a CTA is launched with: 2 x 128 x 112 + 2 x 128 x 96 + 128 x 56 are 60416 of 61440
constexpr int SOFTMAX_REGS = 112, ISSUER_REGS = 56;
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
  __shared__ int s_common;
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
  // no further than every query of every row sees, and than every row has pages
  int common = 0x7fffffff;
  for (int b = first + tid; b < end; b += PLAN_THREADS) {
    const int row = row_at(b);
    const int len = row < 0 || row >= c.rows ? 0 : max(0, min(c.lengths[row], p.longest));
    common = min(common, min(mzp_packed(len, c.residual), max(0, len - p.q_len + 1)) / MZP_PAGE);
  }
  if (tid == 0) s_common = min(c.width, end - first < 2 ? 0 : 0x7fffffff);
  __syncthreads();
  atomicMin(&s_common, common);
  __syncthreads();
  common = s_common;
  const int row0 = first < end ? row_at(first) : 0;
  if (common > 0) {
    const int* head = c.block_table + (long long)row0 * c.width;
    const int warp = tid >> 5, lane = tid & 31;
    // 32 columns of a row for each warp of the cluster in turn
    const int pieces = (common + 31) / 32;
    const long long all = (long long)pieces * (end - first);
    for (long long i = rank * (PLAN_THREADS / 32) + warp; i < all; i += PLAN_CTAS * (PLAN_THREADS / 32)) {
      const int b = first + (int)(i / pieces), at = (int)(i % pieces) * 32 + lane;
      if (at < common) {
        const int id = head[at];
        const bool same = id >= 0 && id < c.pages && c.block_table[(long long)row_at(b) * c.width + at] == id;
        if (!same) atomicMin(&s_common, at);
      }
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
  for (int b = first + rank * PLAN_THREADS + tid; b < end; b += PLAN_CTAS * PLAN_THREADS) { p.out.skip[b] = common; p.out.group_of[b] = g; }
  if (rank == 0 && tid == 0) p.out.groups[g] = {first, (end - first) * p.qrows, end > first ? common : 0, row0};
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // nobody's shared memory goes while it is read
}

// ---- attention over the prefixes
template <int D>
struct PrefixSmem {
  static constexpr int KEY_CHUNK = D * 16, VALUE_CHUNK = MZP_PAGE * 16;          // 8 tokens of all channels; 8 channels of all tokens
  static constexpr int PLANE = MZP_PAGE * D * 2;                                 // a page's keys, or values, in 16 bits
  static constexpr int STAGES = 4, SCALES = 8;
  static constexpr int KEYS = 0, VALUES = STAGES * 2 * PLANE, BOOK = VALUES + STAGES * PLANE;
  static constexpr int ALIGN = 128, TOTAL = BOOK + MZP_BOOKS * MZP_LEVELS + ALIGN;
  // columns of tensor memory: queries of both streams (A operand, two values to a column), logits (P stands over their first half), outputs
  static constexpr int TM_Q = 0, TM_S = D, TM_O = D + 2 * MZP_PAGE, TM_COLS = 512;
  static_assert(TM_O + 2 * D <= TM_COLS, "tensor memory");
};
struct PrefixShared {
  unsigned long long k_full[4], k_free[4], v_full[4], v_free[4], s_full[2], p_full[2], o_done[2], q_full, end;
  int2 scale[8];                                 // (ek, ev) by page of the CTA's line
  float2 ml[2][128];                             // of the two streams, where they share rows
  long long steps, records;                      // before the group of the CTA's first step
  long long total;
  int group;
  uint32_t tmem;
  int failed;
};
struct Segment { int first, row, head, m0, rows, page, count; long long record; };      // a run of steps of one unit

// D[128 x N] (+)= A[128 x 16, tensor memory] * B[16 x N], f16 into fp32, B major along N
template <int N>
__device__ __forceinline__ void umma16(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t accumulate) {
  constexpr uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(N / 8) << 17) | (8u << 24);
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
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

// Goes through a CTA's part of the line, a run of steps of one unit at a time.  Every role walks by itself.
struct Walk {
  const PrefixArgs& p;
  long long steps, records, f0, f1;
  int g, unit;
  __device__ __forceinline__ Walk(const PrefixArgs& args, const PrefixShared& x, long long from, long long to)
      : p(args), steps(x.steps), records(x.records), f0(from), f1(to), g(x.group), unit(-1) {}
  __device__ __forceinline__ bool next(Segment& s) {
    while (g < p.out.n_groups) {
      const MzpGroup info = p.out.groups[g];
      if (info.pages > 0) {
        const MzpTiles tiles(info.rows);
        const long long len = (long long)info.pages * tiles.weight;
        const int units = p.c.kv_heads * tiles.count;
        if (unit < 0) unit = f0 > steps ? (int)min((f0 - steps) / len, (long long)units) : 0;
        for (; unit < units; ++unit) {
          const long long at = steps + unit * len;
          if (at >= f1) return false;
          const int first = at >= f0 ? 0 : (int)((f0 - at + tiles.weight - 1) / tiles.weight);
          const int end = (int)min((long long)info.pages, (f1 - at + tiles.weight - 1) / tiles.weight);
          if (first >= end) continue;
          const int head = unit / tiles.count, tile = unit - head * tiles.count;
          s.first = info.first; s.row = info.row; s.head = head;
          s.m0 = tile * tiles.rows;
          s.rows = min(tiles.rows, info.rows - s.m0);
          s.page = first;
          s.count = end - first;
          s.record = records + (long long)head * info.rows + s.m0;
          ++unit;
          return true;
        }
        steps += units * len;
        records += (long long)p.c.kv_heads * info.rows;
      }
      ++g;
      unit = 0;
    }
    return false;
  }
};

template <int D, bool BF>
__global__ void __launch_bounds__(PREFIX_THREADS, 1) prefix_kernel(const PrefixArgs p, const uint8_t* __restrict__ book_table) {
  using S = PrefixSmem<D>;
  constexpr int PB = 72 * D, HALF = MZP_TILE_ROWS / 2;
  extern __shared__ uint8_t window[];
  uint8_t* smem = window + (S::ALIGN - smem_u32(window) % S::ALIGN) % S::ALIGN;
  __shared__ PrefixShared x;
  const mz_paged_cache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  const uint32_t sbase = smem_u32(smem), sbook = sbase + S::BOOK;
  auto bar = [&](unsigned long long& b) { return smem_u32(&b); };
  if (tid == 0) {
    x.failed = p.fail_waits;
    for (int i = 0; i < S::STAGES; ++i) { bar_init(bar(x.k_full[i]), 4); bar_init(bar(x.k_free[i]), 1); bar_init(bar(x.v_full[i]), 4); bar_init(bar(x.v_free[i]), 1); }
    for (int i = 0; i < 2; ++i) { bar_init(bar(x.s_full[i]), 2); bar_init(bar(x.p_full[i]), 4); bar_init(bar(x.o_done[i]), 1); }
    bar_init(bar(x.q_full), SOFTMAX_WARPS);
    bar_init(bar(x.end), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < MZP_BOOKS * MZP_LEVELS / 16) ((uint4*)(smem + S::BOOK))[tid] = ((const uint4*)book_table)[tid];
  // ---- the line: its length, and the group that the CTA's part begins in
  if (warp == 0) {
    long long steps = 0;
    for (int i = lane; i < p.out.n_groups; i += 32) {
      const MzpGroup info = p.out.groups[i];
      const MzpTiles tiles(info.rows);
      steps += (long long)info.pages * tiles.weight * tiles.count * c.kv_heads;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) steps += __shfl_xor_sync(0xffffffffu, steps, o);
    const long long total = steps;
    const MzpLine line(total, gridDim.x);
    const long long f0 = cta < line.ctas ? line.start(cta) : 0;
    long long before_s = 0, before_r = 0;
    for (int i0 = 0; i0 < p.out.n_groups; i0 += 32) {
      const int i = i0 + lane;
      long long st = 0, re = 0;
      if (i < p.out.n_groups) {
        const MzpGroup info = p.out.groups[i];
        const MzpTiles tiles(info.rows);
        st = (long long)info.pages * tiles.weight * tiles.count * c.kv_heads;
        re = info.pages > 0 ? (long long)info.rows * c.kv_heads : 0;
      }
      long long ss = st, rr = re;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, ss, o), b = __shfl_up_sync(0xffffffffu, rr, o);
        if (lane >= o) { ss += a; rr += b; }
      }
      const long long my_s = before_s + ss - st, my_r = before_r + rr - re;
      if (i < p.out.n_groups) {
        if (my_s <= f0 && f0 < my_s + st) { x.group = i; x.steps = my_s; x.records = my_r; }
        if (cta == 0) p.out.sums[i] = {my_s, my_r};
      }
      before_s += __shfl_sync(0xffffffffu, ss, 31);
      before_r += __shfl_sync(0xffffffffu, rr, 31);
    }
    if (lane == 0) {
      x.total = total;
      if (cta == 0) p.out.sums[p.out.n_groups] = {total, before_r};
    }
  }
  __syncthreads();
  const MzpLine line(x.total, gridDim.x);
  if (cta >= line.ctas) return;
  const long long f0 = line.start(cta), f1 = line.start(cta + 1);
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&x.tmem)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tm_before();
  }
  __syncthreads();
  tm_after();
  const uint32_t tmem = x.tmem;
  volatile int* failed = &x.failed;
  Walk walk(p, x, f0, f1);
  Segment seg;

  if (warp >= ISSUER) {
    registers<ISSUER_REGS, false>();
    // ---- products: the logits of a job as soon as the stream's last P has been used
    if (warp == ISSUER && lane == 0) {
      int pages = 0, segment = 0, used0 = 0, used1 = 0;      // of the CTA so far: pages, segments, jobs of each stream
      while (walk.next(seg)) {
        const bool both = seg.rows > HALF;                   // two tiles of rows take each page; otherwise the streams take the pages in turn
        const int jobs = both ? 2 * seg.count : seg.count;
        bar_wait(bar(x.q_full), segment & 1, failed);
        tm_after();
        const int fresh0 = used0, fresh1 = used1;
        for (int i = 0; i < jobs + 2; ++i) {
          if (i >= 2) {
            const int j = i - 2, s = j & 1, page = pages + (both ? j >> 1 : j), stage = page % S::STAGES;
            const int used = s ? used1 : used0;
            bar_wait(bar(x.p_full[s]), used & 1, failed);
            if (!both || s == 0) bar_wait(bar(x.v_full[stage]), page / S::STAGES & 1, failed);
            tm_after();
            if (!*failed) {
              const uint64_t vd = descriptor(sbase + S::VALUES + stage * S::PLANE, S::VALUE_CHUNK);
#pragma unroll
              for (int k = 0; k < MZP_PAGE / 16; ++k)
                umma16<D>(tmem + S::TM_O + s * D, tmem + S::TM_S + s * MZP_PAGE + k * 8, vd + k * (256 >> 4), used != (s ? fresh1 : fresh0) || k > 0);
              umma_commit(bar(x.o_done[s]));
              if (!both || s == 1) umma_commit(bar(x.v_free[stage]));
            }
            used0 += s ^ 1;
            used1 += s;
          }
          if (i < jobs) {
            const int s = i & 1, page = pages + (both ? i >> 1 : i), stage = page % S::STAGES;
            if (!both || s == 0) bar_wait(bar(x.k_full[stage]), page / S::STAGES & 1, failed);
            tm_after();
            if (!*failed) {
#pragma unroll
              for (int plane = 0; plane < 2; ++plane) {
                const uint64_t kd = descriptor(sbase + S::KEYS + (2 * stage + plane) * S::PLANE, S::KEY_CHUNK);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                  umma16<MZP_PAGE>(tmem + S::TM_S + s * MZP_PAGE, tmem + S::TM_Q + s * (D / 2) + k * 8, kd + k * (256 >> 4), plane > 0 || k > 0);
              }
              umma_commit(bar(x.s_full[s]));
              if (!both || s == 1) umma_commit(bar(x.k_free[stage]));
            }
            bar_arrive(bar(x.s_full[s]));                    // hands on what the keys' writers left beside them
          }
        }
        pages += seg.count;
        ++segment;
      }
    }
  } else if (warp < SOFTMAX_WARPS) {
    // ---- softmax: a thread has a query row
    registers<SOFTMAX_REGS, true>();
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_s = lanes + S::TM_S + s * MZP_PAGE, t_o = lanes + S::TM_O + s * D;
    int pages = 0, segment = 0, done = 0;
    while (walk.next(seg)) {
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
          tm_store32(lanes + S::TM_Q + s * (D / 2) + 32 * h, v);
        }
        tm_stored();
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(x.q_full));
      }
      float M = -INFINITY, l = 0.f;
      const int mine = both ? seg.count : (seg.count + 1 - s) / 2;         // jobs of this stream
      for (int j = 0; j < mine; ++j) {
        const int page = pages + (both ? j : 2 * j + s);
        bar_wait(bar(x.s_full[s]), done & 1, failed);
        tm_after();
        if (some) {
          const int2 sc = x.scale[page % S::SCALES];
          const float f = rowf * pow2(sc.x), ev = (float)sc.y;
          uint32_t v0[32], v1[32];
          tm_load32(v0, t_s);
          tm_load32(v1, t_s + 32);
          tm_loaded(v0);
          tm_loaded(v1);
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, fmaxf(__uint_as_float(v0[i]), __uint_as_float(v1[i])));
          const float t = fmaf(top, f, ev);
          if (j == 0) {
            M = t;
          } else {
            const bool more = t > M + 8.f;
            if (__any_sync(0xffffffffu, more)) {
              const float to = more ? t : M, fix = more ? ex2(M - to) : 1.f;
              M = to;
              l *= fix;
              bar_wait(bar(x.o_done[s]), (done - 1) & 1, failed);        // the stream's last product is in
              tm_after();
#pragma unroll
              for (int h = 0; h < D / 32; ++h) {
                uint32_t o[32];
                tm_load32(o, t_o + 32 * h);
                tm_loaded(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                tm_store32(t_o + 32 * h, o);
              }
            }
          }
          const float add = ev + 7.f - (M == -INFINITY ? 0.f : M);
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float a = ex2(fmaf(__uint_as_float(v0[i]), f, add)), b = ex2(fmaf(__uint_as_float(v0[i + 1]), f, add));
            const float c2 = ex2(fmaf(__uint_as_float(v1[i]), f, add)), d = ex2(fmaf(__uint_as_float(v1[i + 1]), f, add));
            w[i / 2] = half2_bits(__floats2half2_rn(a, b));
            w[16 + i / 2] = half2_bits(__floats2half2_rn(c2, d));
            add2(sum[0], sum[1], a, b);
            add2(sum[2], sum[3], c2, d);
          }
          tm_store32(t_s, w);
          l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), pow2(-sc.y - 7), l);
          tm_stored();
        }
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(x.p_full[s]));
        ++done;
      }
      // ---- records
      if (mine > 0) bar_wait(bar(x.o_done[s]), (done - 1) & 1, failed);
      tm_after();
      const bool bad = *failed != 0;
      const long long at = seg.record + (long long)MZP_TILE_ROWS * cta + m;
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
        uint32_t v[32], u[32];
        float out[32];
        tm_load32(v, t_o + d);
        tm_load32(u, t_other + d);
        tm_loaded(v);
        tm_loaded(u);
        // a stream that had no page left nothing in its accumulator
#pragma unroll
        for (int i = 0; i < 32; ++i) out[i] = (mine > 0 ? __uint_as_float(v[i]) * f_mine : 0.f) + (!both && f_other != 0.f ? __uint_as_float(u[i]) * f_other : 0.f);
        if (inside) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) stg256(p.out.acc + at * D + d + i, out + i);
        }
      }
      if (inside && (both || s == 0)) p.out.ml[at] = bad ? make_float2(INFINITY, __int_as_float(0x7fffffff)) : make_float2(M, l);
      tm_before();
      if (!both) asm volatile("bar.sync 1, 256;" ::: "memory");          // x.ml is free again
      pages += seg.count;
      ++segment;
    }
  } else {
    // ---- levels: four warps have a page, the other four the next one
    const int team = (warp - SOFTMAX_WARPS) >> 2, t = (warp & 3) * 32 + lane;
    const uint8_t* store = (const uint8_t*)c.store + (long long)p.layer * c.store_stride_layer;
    constexpr int WPL = D / 32;                              // words per lane: all of a side
    struct Raw { uint32_t kc[8], vc[8], kw, vw, all[2 * WPL]; };
    const bool keys = D == 128 || t < 64, values = D == 128 || t >= 64;
    const int ch = t % D, token = t % MZP_PAGE, part = D == 128 ? t / MZP_PAGE : 0;
    int at = team;                                           // page of the segment
    bool more = walk.next(seg);
    auto settle = [&]() {
      while (more && at >= seg.count) { at -= seg.count; more = walk.next(seg); }
    };
    settle();
    auto page_of = [&]() {                                   // of the cursor; -1: none.  What is added: its head's place
      long long place = -1;
      if (more) {
        const int id = c.block_table[(long long)seg.row * c.width + seg.page + at];
        if (id >= 0 && id < c.pages) place = (long long)id * c.store_stride_page + (long long)seg.head * PB;
        else place = -2;                                     // not there any more: T = 0
      }
      at += 2;
      settle();
      return place;
    };
    auto load = [&](Raw& w, long long place) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w.kc[i] = w.vc[i] = 0;
      w.kw = w.vw = 0;
#pragma unroll
      for (int i = 0; i < 2 * WPL; ++i) w.all[i] = 0;
      if (place < 0) return;
      const uint8_t* b = store + place;
      const int row = token * (D / 64) + part;
      if (keys) { ldg256(w.kc, b + 32 * ch); w.kw = __ldg((const uint32_t*)(b + 32 * D + 4 * ch)); }
      if (values) { ldg256(w.vc, b + 36 * D + 32 * row); w.vw = __ldg((const uint32_t*)(b + 68 * D + 4 * row)); }
#pragma unroll
      for (int i = 0; i < WPL; i += 2) {
        const uint2 a = __ldg((const uint2*)(b + 32 * D) + (lane * WPL + i) / 2), v = __ldg((const uint2*)(b + 68 * D) + (lane * WPL + i) / 2);
        w.all[i] = a.x; w.all[i + 1] = a.y;
        w.all[WPL + i] = v.x; w.all[WPL + i + 1] = v.y;
      }
    };
    // the power of two above a side's largest value; f16 has its values below 2^14
    auto exponent = [&](const uint32_t* words) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < WPL; ++i) {
        const MzpRow row = mzp_row(words[i]);
        top = fmaxf(top, fmaf(4.f, fabsf(row.t), fabsf(row.a)));
      }
      return min(max((int)(warp_max_u32(__float_as_uint(top)) >> 23) - 126, -30), 30) - 14;
    };
    long long place = page_of(), ahead = place == -1 ? -1 : page_of();
    Raw now;
    load(now, place);
    for (int page = team; place != -1; page += 2) {
      Raw next;
      load(next, ahead);
      const long long far = ahead == -1 ? -1 : page_of();
      const int stage = page % S::STAGES;
      const uint32_t parity = (page / S::STAGES & 1) ^ 1;
      const int ek = exponent(now.all), ev = exponent(now.all + WPL);
      bar_wait(bar(x.k_free[stage]), parity, failed);
      if (t == 0) x.scale[page % S::SCALES] = make_int2(ek, ev);
      if (keys) {
        const MzpRow row = mzp_row(now.kw);
        const uint4 book = book128(sbook + row.z * 16);
        const float unit = row.t * pow2(-ek) * 0.03125f, anchor = row.a * pow2(-ek);
        const __half2 zero = __floats2half2_rn(1024.f + row.z, 1024.f + row.z), step = __floats2half2_rn(unit, unit);
        const uint32_t hi_at = sbase + S::KEYS + 2 * stage * S::PLANE + ch * 16, lo_at = hi_at + S::PLANE;
#pragma unroll
        for (int q = 0; q < 8; ++q) {            // eight tokens
          uint32_t u[4], hi[4], lo[4];
          levels8(now.kc[q], book, u);
          if (row.a == 0.f) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __half2 w = __hsub2(bits_half2(u[k]), zero), h = __hmul2(w, step);
              hi[k] = half2_bits(h);
              lo[k] = half2_bits(__hfma2(w, step, __hneg2(h)));            // exact
            }
          } else {                               // the sum has more than 22 bits' worth of terms: in fp32
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 w = __half22float2(__hsub2(bits_half2(u[k]), zero));
              const float a = fmaf(w.x, unit, anchor), b = fmaf(w.y, unit, anchor);
              const __half2 h = __floats2half2_rn(a, b);
              const float2 f = __half22float2(h);
              hi[k] = half2_bits(h);
              lo[k] = half2_bits(__floats2half2_rn(a - f.x, b - f.y));
            }
          }
          sts128(hi_at + q * S::KEY_CHUNK, hi[0], hi[1], hi[2], hi[3]);
          sts128(lo_at + q * S::KEY_CHUNK, lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_operands();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(x.k_full[stage]));
      bar_wait(bar(x.v_free[stage]), parity, failed);
      if (values) {
        const MzpRow row = mzp_row(now.vw);
        const uint4 book = book128(sbook + row.z * 16);
        const float unit = row.t * pow2(-ev) * 0.03125f, anchor = row.a * pow2(-ev);
        const __half2 zero = __floats2half2_rn(1024.f + row.z, 1024.f + row.z), step = __floats2half2_rn(unit, unit), base = __floats2half2_rn(anchor, anchor);
        const uint32_t dst = sbase + S::VALUES + stage * S::PLANE + part * 8 * S::VALUE_CHUNK + token * 16;
#pragma unroll
        for (int q = 0; q < 8; ++q) {            // eight channels
          uint32_t u[4];
          levels8(now.vc[q], book, u);
#pragma unroll
          for (int k = 0; k < 4; ++k) u[k] = half2_bits(__hfma2(__hsub2(bits_half2(u[k]), zero), step, base));
          sts128(dst + q * S::VALUE_CHUNK, u[0], u[1], u[2], u[3]);
        }
      }
      fence_operands();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(x.v_full[stage]));
      now = next;
      place = ahead;
      ahead = far;
    }
  }
  if (warp == ISSUER && lane == 0) {          // the products are done, and so is what they signal
    umma_commit(bar(x.end));
    for (int k = 0; k < SPIN_LIMIT && !bar_test(bar(x.end), 0); ++k) {}
  }
  tm_before();
  __syncthreads();
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
  s->bytes = s->acc_at + s->records * c->head_dim * sizeof(float);
}

int mzp_prefix_launch(const mz_paged_cache& c, int layer, const mz_paged_attention_args& args, const mz_paged_view& view, const MzpPrefixShape& s, uint8_t* workspace,
                      int longest, const uint8_t* book, cudaStream_t stream, MzpPrefix* out) {
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
  p.out.n_groups = view.n_groups;
  p.out.grid = s.grid;
  p.out.records = s.records;
  p.fail_waits = mz_waits_fail();
  *out = p.out;
  const bool bf = c.kv_dtype == MZ_BF16;
  if (c.head_dim == 128) return bf ? mzp::launch_prefix<128, true>(p, book, stream) : mzp::launch_prefix<128, false>(p, book, stream);
  return bf ? mzp::launch_prefix<64, true>(p, book, stream) : mzp::launch_prefix<64, false>(p, book, stream);
}
