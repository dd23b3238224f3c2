// The work of a step's attention, tile by tile and part by part, from the step's lengths (host only). RaggedBatch.row_plan says what it means.
// As array operations in Python it took the host 100 to 250 us a step, here 2 to 10; with the pinned memory and the copy to the GPU 9 to 17 us, where it
// is to be there for every stream 28 to 37.
#include <torch/extension.h>

#include <algorithm>
#include <numeric>

namespace cai {
namespace serving {
namespace {

constexpr int64_t CUS = 256, MOST_PARTS = 64;   // of a tile: to put more together takes longer than they save (one sequence of 32768: 20 us for 17)

struct Tile {
  int64_t seq, t0, t1, begin, steps;
};
struct Part {
  int64_t tile, lo, hi, slot;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The longest part, in steps, that tiles are cut into, `least` at least and MOST_PARTS of a tile at most: where their blocks leave some of the `most`
// that a chip holds at once, the smallest parts that still are all at once; else twice a block's share of all steps, so that tiles are cut that the
// others would wait for (one of 131072 beside 199 of 1024, 32/8 heads of 128: 82 us for 936; 500 tokens over 32000 beside eight over 1000: 472 for 812;
// 200 of 1024, none cut: 43). At once the share 83 and 445 to 488, but 3000 new tokens 124 for 106: parts to join; at four times 120 and 814.
int64_t longest_part(const std::vector<Tile>& tiles, int64_t blocks_each, int64_t most, int64_t least) {
  int64_t hi = 0, total = 0;
  for (const Tile& t : tiles) {
    hi = std::max(hi, t.steps);
    total += t.steps;
  }
  int64_t lo = std::max(least, ceil_div(hi, MOST_PARTS));
  if ((int64_t)tiles.size() * blocks_each >= most) return std::min(hi, std::max(lo, 2 * ceil_div(total * blocks_each, most)));
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    int64_t parts = 0;
    for (const Tile& t : tiles) parts += ceil_div(t.steps, mid);
    if (parts * blocks_each <= most) hi = mid;
    else lo = mid + 1;
  }
  return hi;
}

}  // namespace

std::tuple<at::Tensor, std::vector<int64_t>> row_plan(const std::vector<int64_t>& cu, const std::vector<int64_t>& start, int64_t group, int64_t heads,
                                                      int64_t window, const std::vector<int64_t>& rows, const std::vector<int64_t>& blocks,
                                                      int64_t step, int64_t least, bool pinned) {
  const int64_t B = (int64_t)start.size();
  TORCH_CHECK_VALUE((int64_t)cu.size() == B + 1 && rows.size() == 3 && blocks.size() == 3 && group > 0 && heads > 0 && step > 0 && least > 0,
                    "row_plan: offsets of every sequence, three kinds of tiles");
  std::vector<std::vector<Tile>> tiles(3);
  std::vector<int> kind(B);
  int64_t few = 0, second = 0;
  for (int64_t i = 0; i < B; ++i) {
    const int64_t n = cu[i + 1] - cu[i];
    kind[i] = n == 1 || n * group <= rows[0] ? 0 : 4 * n * group >= 3 * rows[2] ? 2 : 1;
    few += kind[i] == 0;
    second += kind[i] == 1;
  }
  // One launch, where there is room beside the others (10 tokens over 2000 beside 31 single ones over 4000: 39 us, in two launches 43; three of 8 over 300
  // beside ten single ones over 500: 11 and 19). Weights are as precise in every kind of tile.
  if (second > 0 && few * heads < blocks[0] / 2)
    for (int& k : kind) k = k == 0 ? 1 : k;
  for (int64_t i = 0; i < B; ++i) {
    const int64_t per = std::max<int64_t>(1, rows[kind[i]] / group), shift = start[i] - cu[i];
    for (int64_t t0 = cu[i]; t0 < cu[i + 1]; t0 += per) {
      const int64_t t1 = std::min(t0 + per, cu[i + 1]), begin = window > 0 ? std::max<int64_t>(0, t0 + shift - window + 1) / step : 0;
      tiles[kind[i]].push_back({i, t0, t1, begin, (t1 - 1 + shift) / step + 1 - begin});
    }
  }
  std::vector<int> plan;
  std::vector<int64_t> sizes;
  for (int k = 0; k < 3; ++k) {
    const int64_t each_part = heads * ceil_div(group, rows[k]);   // blocks
    const int64_t share = tiles[k].empty() ? 1 : longest_part(tiles[k], each_part, blocks[k], least);
    std::vector<Part> parts;
    std::vector<int> joins;
    int64_t slots = 0;
    for (int64_t t = 0; t < (int64_t)tiles[k].size(); ++t) {
      const Tile& x = tiles[k][t];
      const int64_t each = ceil_div(x.steps, ceil_div(x.steps, share)), count = ceil_div(x.steps, each);   // none is empty
      for (int64_t p = 0; p < count; ++p)
        parts.push_back({t, x.begin + p * each, x.begin + std::min((p + 1) * each, x.steps), count > 1 ? slots + p : -1});
      if (count == 1) continue;
      for (int64_t v : {x.t0, x.t1, slots, count}) joins.push_back((int)v);
      slots += count;
    }
    std::vector<int64_t> order(parts.size());
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return parts[a].hi - parts[a].lo > parts[b].hi - parts[b].lo; });
    const int64_t turn = std::max<int64_t>(1, CUS / each_part), n = (int64_t)parts.size();
    if (n * each_part <= blocks[k])   // all at once: a CU's next part is as short as its first one is long
      for (int64_t i = turn; i < n; i += 2 * turn) std::reverse(order.begin() + i, order.begin() + std::min(i + turn, n));
    for (int64_t i : order) {
      const Part& p = parts[i];
      const Tile& x = tiles[k][p.tile];
      for (int64_t v : {x.seq, x.t0, x.t1, p.lo, p.hi, p.slot}) plan.push_back((int)v);
    }
    plan.insert(plan.end(), joins.begin(), joins.end());
    for (int64_t v : {n, (int64_t)joins.size() / 4, slots}) sizes.push_back(v);
  }
  int64_t longest = 0;
  for (int64_t i = 0; i < B; ++i) longest = std::max(longest, start[i] + cu[i + 1] - cu[i]);
  sizes.push_back(B);
  sizes.push_back(longest);
  const at::Tensor out = at::empty({(int64_t)plan.size()}, at::TensorOptions().dtype(at::kInt).pinned_memory(pinned));
  std::copy(plan.begin(), plan.end(), out.data_ptr<int>());
  return {out, sizes};
}

}  // namespace serving
}  // namespace cai
