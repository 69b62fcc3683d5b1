// Paged cache: layout and codec shared by its kernels (include/muzero_b200.h describes both).
//
// The codec is the zero-anchored log compander with its levels rounded to 127ths of the row's range, so that a level is a 7-bit
// integer: one byte per code holds it exactly, and sums of levels times integers are exact on the integer tensor cores.  The zero level z (0..127)
// picks one of 128 books of 16 levels, so a row needs no book of its own.  On normally distributed rows the error is 0.0853 of the standard
// deviation (0.0842 with the unrounded levels of the contiguous store).
#pragma once
#include "mz_common.cuh"

constexpr int MZP_PAGE = 64;                    // tokens per page
constexpr int MZP_BOOKS = 128, MZP_LEVELS = 16;
// Rows of the device's table of nearest levels: entries -1 .. 128 (a value may round to a level beyond the ends), padded so that rows start at different banks
constexpr int MZP_NEAR_ROW = 132;

// device copies of the two tables of mz_paged_books, the second in rows of MZP_NEAR_ROW (static device memory, filled and waited for by mz_paged_prepare, or by the first call on a device)
int mz_paged_tables(const uint8_t** book, const uint8_t** nearest);
// multiprocessors of the current device (asked once)
int mz_paged_sms(int* sms);
// whether mz_debug_fail_waits is on (checked build)
int mz_waits_fail();
// argument checks that every entry point shares
int mz_paged_check(const mz_paged_cache* c);

__host__ __device__ inline int mzp_page_bytes(int head_dim) { return 72 * head_dim; }
__host__ __device__ inline int mzp_packed(int length, int residual) {       // tokens of a row that stand in pages
  const int n = length - residual;
  return n > 0 ? n / MZP_PAGE * MZP_PAGE : 0;
}

// a row's word -> anchor, scale, zero level (0..127 whatever the word: it picks a book in shared memory)
struct MzpRow { float a, t; int z; };
__device__ __forceinline__ MzpRow mzp_row(uint32_t word) {
  MzpRow r;
  const uint32_t field = word >> 16;
  const bool off = (field & 0x7FFFu) >= 128u;
  r.t = __half2float(__ushort_as_half((unsigned short)(word & 0xFFFFu)));
  r.a = off ? __half2float(__ushort_as_half((unsigned short)field)) : 0.0f;
  r.z = off ? ((field & 0x8000u) ? 127 : 0) : (int)(field & 0x7Fu);
  return r;
}

// The other way: smallest and largest value of the row (NaN taken as 0, clamped to f16's range) -> constants of the quantizer and the word.  One IEEE
// operation per step, none contracted: the codes are a definition, not an approximation.
struct MzpQuant { float a, inv, z; uint32_t word; };
__device__ __forceinline__ MzpQuant mzp_quant(float lo, float hi) {
  MzpQuant q;
  const float edge = lo > 0.0f ? lo : hi < 0.0f ? hi : 0.0f;
  const uint32_t bits = __half_as_ushort(__float2half_rn(edge));
  const bool off = (bits & 0x7FFFu) >= 128u;
  q.a = off ? __half2float(__ushort_as_half((unsigned short)bits)) : 0.0f;
  const float dn = q.a > 0.0f ? 0.0f : fmaxf(__fsub_rn(q.a, lo), 0.0f);
  const float up = q.a < 0.0f ? 0.0f : fmaxf(__fsub_rn(hi, q.a), 0.0f);
  const float extent = __fadd_rn(dn, up);
  q.z = extent > 0.0f ? rintf(__fdiv_rn(__fmul_rn(127.0f, dn), extent)) : 0.0f;
  if (q.a < 0.0f) q.z = 127.0f;
  const __half t = __float2half_rn(__fmul_rn(extent, (float)(32.0 / 127.0)));
  const float tf = __half2float(t);
  q.inv = tf > 0.0f ? __fdiv_rn(32.0f, tf) : 0.0f;
  q.word = (uint32_t)__half_as_ushort(t) | (off ? bits : (uint32_t)q.z) << 16;
  return q;
}
__device__ __forceinline__ float mzp_finite(float x) { return x != x ? 0.0f : fminf(fmaxf(x, -65504.0f), 65504.0f); }
