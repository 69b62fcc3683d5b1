"""Paged cache, shared prefixes: the arithmetic that cuts the line of pages over the CTAs and names the records, as the kernels use it, on the host.

For batches of groups with any number of query rows: every page of every unit is taken by exactly one CTA, every record that the merge reads is one that a CTA wrote, and no two records
have a place in common, none one outside the workspace.
"""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>
#include "mz_paged_prefix.cuh"

struct Batch { int kv_heads, qrows, grid; std::vector<int> entries, pages; };

// 0, or what is wrong
const char* look(const Batch& t) {
  const int n = (int)t.entries.size();
  std::vector<MzpGroup> groups(n);
  std::vector<MzpSums> sums(n + 1);
  std::vector<int> group_of;
  long long steps = 0, records = 0;
  int heaviest = 1;
  for (int g = 0; g < n; ++g) {
    groups[g].first = (int)group_of.size();
    groups[g].rows = t.entries[g] * t.qrows;
    groups[g].pages = t.pages[g];
    for (int i = 0; i < t.entries[g]; ++i) group_of.push_back(g);
    sums[g].steps = steps;
    sums[g].records = records;
    if (t.pages[g] == 0) continue;
    const MzpTiles tiles(groups[g].rows);
    steps += (long long)t.pages[g] * tiles.weight * tiles.count * t.kv_heads;
    records += (long long)groups[g].rows * t.kv_heads;
    heaviest = tiles.weight > heaviest ? tiles.weight : heaviest;
  }
  if (steps == 0) return nullptr;
  sums[n].steps = steps;
  sums[n].records = records;
  sums[n].heaviest = heaviest;
  const long long room = (long long)group_of.size() * t.qrows * t.kv_heads + (long long)MZP_TILE_ROWS * t.grid;
  MzpPrefix p = {};
  p.group_of = group_of.data(); p.groups = groups.data(); p.sums = sums.data();
  p.n_groups = n; p.grid = t.grid;
  const MzpLine line(steps, heaviest, t.grid);
  std::map<long long, long long> places;         // of records: first and behind the last
  for (int g = 0; g < n; ++g) {
    if (t.pages[g] == 0) continue;
    const MzpTiles tiles(groups[g].rows);
    const MzpUnits units(p, groups[g].first, t.qrows, t.kv_heads);
    const long long len = (long long)t.pages[g] * tiles.weight;
    for (int u = 0; u < t.kv_heads * tiles.count; ++u) {
      const long long at = sums[g].steps + u * len;
      const int head = u / tiles.count, row = (u - head * tiles.count) * tiles.rows, rows = std::min(tiles.rows, groups[g].rows - row);
      int first, last, next = 0;
      const long long record = units.record(head, row, first, last);
      for (int r : {row, row + rows - 1}) {      // the same CTAs for all rows of a tile, their places one after the other
        int f, l;
        if (units.record(head, r, f, l) != record + r - row || f != first || l != last) return "rows of a tile";
      }
      if (first < 0 || last >= line.ctas || first > last) return "owners";
      for (int cta = 0; cta < line.ctas; ++cta) {
        const MzpRun run(at, t.pages[g], tiles.weight, line.start(cta), line.start(cta + 1));
        if ((run.count > 0) != (cta >= first && cta <= last)) return "a record that is read and not written, or written and not read";
        if (run.count <= 0) continue;
        if (run.page != next) return "pages";
        next += run.count;
        const long long place = record + (long long)MZP_TILE_ROWS * cta;
        if (place < 0 || place + rows > room) return "outside the workspace";
        const auto after = places.lower_bound(place);
        if (after != places.end() && after->first < place + rows) return "places";
        if (after != places.begin() && std::prev(after)->second > place) return "places";
        places[place] = place + rows;
      }
      if (next != t.pages[g]) return "pages that nobody takes";
    }
  }
  return nullptr;
}

int main() {
  std::vector<Batch> all;
  // one group of many entries with few query rows each, and a short prefix
  const int shapes[][4] = {{256, 1, 6, 8}, {256, 1, 10, 8}, {256, 1, 15, 8}, {128, 2, 12, 8}, {128, 2, 14, 8}, {128, 2, 16, 8}, {85, 3, 17, 8}, {200, 1, 8, 8}, {200, 1, 12, 8}, {160, 1, 4, 32}};
  for (auto& s : shapes) all.push_back({s[3], s[1], 148, {s[0]}, {s[2]}});
  for (int pages = 1; pages < 80; ++pages)
    for (int rows : {1, 127, 128, 129, 256, 257, 300, 513, 1024}) for (int heads : {1, 3, 8}) all.push_back({heads, 1, 148, {rows}, {pages}});
  std::mt19937 rng(5);
  auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
  for (int i = 0; i < 3000; ++i) {
    Batch t = {1 + below(8), 1 + below(12), below(4) ? 148 : 1 + below(160), {}, {}};
    const int groups = 1 + below(below(8) ? 6 : 200), most = 1 << below(9);
    for (int g = 0, left = 1024; g < groups && left > 0; ++g) {
      const int e = std::min(left, below(below(3) ? 20 : 300));
      t.entries.push_back(e);
      t.pages.push_back(e < 2 || !below(5) ? 0 : 1 + below(most));
      left -= e;
    }
    all.push_back(t);
  }
  for (const Batch& t : all) {
    const char* wrong = look(t);
    if (wrong) {
      printf("%s: kv heads %d, query rows %d, grid %d, groups", wrong, t.kv_heads, t.qrows, t.grid);
      for (size_t g = 0; g < t.entries.size(); ++g) printf(" %d x %d", t.entries[g], t.pages[g]);
      printf("\n");
      return 1;
    }
  }
  printf("%zu batches\n", all.size());
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    from muzero_b200.build import CSRC, _nvcc
    at = tmp_path_factory.mktemp("line")
    src, exe = str(at / "line.cu"), str(at / "line")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.check_call([_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-I", CSRC, src, "-o", exe])
    return exe


def test_records_that_are_read_are_written(program):
    res = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "batches" in res.stdout, res.stdout
