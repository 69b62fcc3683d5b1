// Paged cache: what the kernel for shared prefixes (mz_paged_prefix.cu) leaves for the one that ends an attention call (mz_paged_attention.cu).
//
// A group is a run of list entries; the pages that all its rows' tables begin with are its prefix.  The query rows of a group that share a kv head, entry after entry, are
// cut into tiles of at most 256; a unit is a (group, kv head, tile), a step of it one page.  The steps of all units stand in one line, weighted by 1 where a tile
// has at most 128 rows and 2 above, and the line is cut evenly over the CTAs.  A page goes to the CTA that has its first step, and no part is shorter than the heaviest page: so
// every CTA between those of a unit's first and last page has a page of it.  Each CTA leaves a record (m, l, out) per query row of a unit that it met: with r
// rows in the units before, the record of row i by CTA c has place r + 256 c + i.
#pragma once
#include "mz_paged_device.cuh"

constexpr int MZP_TILE_ROWS = 256;

// first list entry, query rows per kv head, pages of the prefix (0: nothing is shared), a cache row, entries that share
struct alignas(16) MzpGroup { int first, rows, pages, row, members; };
struct MzpSums { long long steps, records; int heaviest, pad; };     // of the groups before; behind the last group the line's length and the weight of its heaviest page

struct MzpPrefix {
  int* skip;                                     // [batch] pages of an entry that its group has taken care of
  int* group_of;                                 // [batch]
  MzpGroup* groups;                              // [n_groups]
  MzpSums* sums;                                 // [n_groups + 1]
  float2* ml;                                    // [record] maximum (base 2) and sum
  float* acc;                                    // [record][D]
  float4* part;                                  // [CTA][stream][D / 4][128] sums of a long run of pages so far
  int n_groups, grid;
  int nr, passes, sms;                           // of the call without sharing: query rows to a step, steps per page
  long long records;
};

// how a group's query rows are cut
struct MzpTiles {
  int count, rows, weight;
  __host__ __device__ __forceinline__ explicit MzpTiles(int m) {
    count = (m + MZP_TILE_ROWS - 1) / MZP_TILE_ROWS;
    rows = ((m + count - 1) / (count > 0 ? count : 1) + 7) / 8 * 8;
    weight = rows > MZP_TILE_ROWS / 2 ? 2 : 1;
  }
  __host__ __device__ __forceinline__ int cost() const { return count * (10 + 24 * weight); }      // of a page, in tenths of a row's visit to it without sharing
};
// Whether sharing pays.  A page of a prefix costs one kv head 2.6 ns of the machine per row and pass without sharing (3.5 with 8 query rows to a step; head_dim 64: 1.9 and 2.5) and with it 9 ns per
// tile of at most 128 query rows, 15 above (6.3 and 11), and a call that shares takes 28 us more in the first place (24).  In tenths of a row's visit to a page; measured on both sides, 32 query
// heads on 8 kv heads, without / with: 8 rows of 4096 tokens 37 / 56 us, of 16384 71 / 69, of 65536 200 / 118, 4 rows of 65536 116 / 120, 32 rows of 1024 38 / 56, of 4096 73 / 67, 64 rows of 1024 60 / 73,
// of 4096 125 / 89; 8 query rows to a step: 4 rows of 65536 149 / 120, 16 of 4096 60 / 65.  cost: of a page's tiles (MzpTiles)
__host__ __device__ __forceinline__ long long mzp_gain(long long pages, int kv_heads, long long rows_passes, int nr, int cost) {
  const long long each = rows_passes * (nr > 4 ? 13 : 10) - cost;
  return each > 0 ? pages * kv_heads * each : 0;
}
__host__ __device__ __forceinline__ long long mzp_gain_needed(int sms, int head_dim) { return (long long)sms * (head_dim == 128 ? 700 : 900); }
// how the line is cut
struct MzpLine {
  long long total, ctas;
  __host__ __device__ __forceinline__ MzpLine(long long steps, int heaviest, int grid) : total(steps), ctas(steps / heaviest < grid ? steps / heaviest : grid) {}
  __host__ __device__ __forceinline__ long long start(int cta) const { return total * cta / ctas; }
  __host__ __device__ __forceinline__ int owner(long long at) const { return (int)(((at + 1) * ctas - 1) / total); }
};
// the pages of a unit, which begins at step `at`, that belong to the part f0 .. f1 - 1
struct MzpRun {
  int page, count;
  __host__ __device__ __forceinline__ MzpRun(long long at, int pages, int weight, long long f0, long long f1) {
    page = at >= f0 ? 0 : (int)((f0 - at + weight - 1) / weight);
    const long long end = (f1 - at + weight - 1) / weight;
    count = (int)(end < pages ? end : pages) - page;
  }
};

// where a list entry's records are
struct MzpUnits {
  MzpGroup g;
  MzpSums before;
  MzpTiles tiles;
  MzpLine line;
  int qrows, kv_heads;
  __host__ __device__ __forceinline__ MzpUnits(const MzpPrefix& p, int b, int query_rows, int heads)
      : g(p.groups[p.group_of[b]]), before(p.sums[p.group_of[b]]), tiles(g.rows), line(p.sums[p.n_groups].steps, p.sums[p.n_groups].heaviest, p.grid), qrows(query_rows),
        kv_heads(heads) {}
  __host__ __device__ __forceinline__ int row_of(int b, int query_row) const { return (b - g.first) * qrows + query_row; }
  // record of a query row of the group without its CTA's share of 256 c, and the CTAs that have one
  __host__ __device__ __forceinline__ long long record(int head, int row, int& first, int& last) const {
    const int tile = row / tiles.rows;
    const long long at = before.steps + (long long)(head * tiles.count + tile) * g.pages * tiles.weight;
    first = line.owner(at);
    last = line.owner(at + (long long)(g.pages - 1) * tiles.weight);
    return before.records + (long long)head * g.rows + row;
  }
};

struct MzpPrefixShape { int grid; long long records; size_t skip_at, group_of_at, groups_at, sums_at, ml_at, acc_at, part_at, bytes; };
void mzp_prefix_shape(const mz_paged_cache* c, int batch, int n_groups, int qrows, int sms, MzpPrefixShape* s);
// Finds the prefixes of the groups and takes the attention of their rows over them; fills `out`.  longest: no row is taken for longer.
int mzp_prefix_launch(const mz_paged_cache& c, int layer, const mz_paged_attention_args& args, const mz_paged_view& view, const MzpPrefixShape& s, uint8_t* workspace,
                      int longest, int nr, int passes, const uint8_t* book, cudaStream_t stream, MzpPrefix* out);
