// tree_plan.cu -- the work plan of the tree attention, made on the host: which
// CTA attends which tiles of which sequence for which nodes (tree_attend.cuh).
// Host code only.
#include <algorithm>
#include <functional>
#include <queue>
#include <utility>

#include "tree_attend.cuh"

namespace kvl {

// In tiles (bf16 about 1.2 us, Q8 about 2.1): what an item costs beside its tiles
// (query, first tile, epilogue), what the merge launch costs, and a partial's 131
// KB written and read.  Estimates from the traces of bf16 runs, used for Q8 too: a
// plan does not know the pool that it will read.
static constexpr double kItemCost = 3.0, kMergeCost = 3.0, kSlotCost = 0.03;

// A list is kept per CTA, so a grid far beyond any GPU's SMs is cut to this.
static constexpr int kMaxCtas = 1 << 16;

// Whether no drafted row is another sequence's drafted or cached row.  Cached
// rows may be shared (a common prefix), and a sequence's own cached rows end
// where its drafted ones begin.
static bool drafted_rows_apart(const TreeHostPlan &hp) {
  typedef std::pair<long long, long long> Range;  // [first, second)
  std::vector<Range> drafted, cached;
  for (int b = 0; b < hp.batch; ++b) {
    const long long end = hp.row0[b] + hp.len[b];
    if (hp.len[b]) cached.push_back({hp.row0[b], end});
    if (hp.tree[b]) drafted.push_back({end, end + hp.tree[b]});
  }
  std::sort(drafted.begin(), drafted.end());
  std::sort(cached.begin(), cached.end());
  long long drafted_to = 0, cached_to = 0;  // ends of the ranges that begin before this one's end
  size_t c = 0;
  for (const Range &d : drafted) {
    for (; c < cached.size() && cached[c].first < d.second; ++c) cached_to = std::max(cached_to, cached[c].second);
    if (std::max(drafted_to, cached_to) > d.first) return false;
    drafted_to = d.second;
  }
  return true;
}

int set_tree_sequences(TreeHostPlan &hp, int batch, const int *cached_len, const int *nodes, const int64_t *row0) {
  if (batch <= 0) return -1;
  hp = TreeHostPlan();
  hp.batch = batch;
  for (int b = 0; b < batch; ++b) {
    if (cached_len[b] < 0 || nodes[b] < 0 || nodes[b] > kTreeMaxNodes || row0[b] < 0 || row0[b] >= (1LL << 31))
      return -1;
    const long long end = (long long)row0[b] + cached_len[b] + nodes[b];
    if (end >= (1LL << 31)) return -1;
    hp.rows_needed = std::max(hp.rows_needed, end);
    hp.row0.push_back(row0[b]);
    hp.len.push_back(cached_len[b]);
    hp.tree.push_back(nodes[b]);
    hp.first_node.push_back(hp.nodes);
    hp.seq_of_node.insert(hp.seq_of_node.end(), nodes[b], b);
    if (hp.nodes > (1 << 26)) return -1;  // 16 query rows a node stay below 2^31
    hp.nodes += nodes[b];
  }
  if (hp.nodes == 0) return -1;
  hp.own_rows = drafted_rows_apart(hp);
  return 0;
}

void deal_tree_tiles(TreeHostPlan &hp, int ctas) {
  const int batch = hp.batch;
  ctas = std::min(ctas, kMaxCtas);
  struct Seq {
    int tiles, groups;
  };
  std::vector<Seq> seqs(batch);
  long long total = 0;
  int longest = 1, groups = 0;
  bool uniform = true;  // all sequences with drafted rows have as many groups
  for (int b = 0; b < batch; ++b) {
    const long long keys = (long long)hp.len[b] + hp.tree[b];  // up to 2^31 - 1, and kTreeKeys more
    seqs[b] = {hp.tree[b] ? (int)((keys + kTreeKeys - 1) / kTreeKeys) : 0,
               (hp.tree[b] + kTreeGroup - 1) / kTreeGroup};
    total += (long long)seqs[b].tiles * seqs[b].groups;
    longest = std::max(longest, seqs[b].tiles);
    if (seqs[b].groups) {
      uniform &= groups == 0 || groups == seqs[b].groups;
      groups = seqs[b].groups;
    }
  }
  struct Deal {
    std::vector<TreeItem> items;
    std::vector<int> cta;  // of each item
    double cost = 1e30;
  };
  Deal best;
  auto add = [&](Deal &d, int b, int g, int tile0, int tile1, bool part) {
    TreeItem im;
    im.row0 = hp.row0[b];
    im.len = hp.len[b];
    im.tree = hp.tree[b];
    im.node0 = hp.first_node[b] + g * kTreeGroup;
    im.nn = std::min(kTreeGroup, hp.tree[b] - g * kTreeGroup);
    im.tile0 = tile0;
    im.tile1 = tile1;
    im.slot = part ? 0 : -1;
    im.next = -1;
    d.items.push_back(im);
  };
  auto merge_cost = [&](int slots) { return slots ? kMergeCost + kSlotCost * slots : 0.0; };

  // Equal trees: teams of `groups` CTAs, one per group, walk one concatenated
  // list of all sequences' tiles, cut into equal ranges: no CTA has more than
  // its share, and a range boundary splits one sequence at most.  A sequence
  // counts kItemCost tiles more than it has; a cut within them is moved to the
  // sequence's start.
  const int teams = groups ? ctas / groups : 0;
  if (uniform && teams >= 1) {
    Deal d;
    std::vector<double> at(batch + 1, 0.0);  // sequence starts in the list
    for (int b = 0; b < batch; ++b) at[b + 1] = at[b] + (seqs[b].groups ? seqs[b].tiles + kItemCost : 0.0);
    int b = 0, tile = 0, slots = 0;
    double worst = 0;
    for (int m = 0; m < teams; ++m) {
      const double end = at[batch] * (m + 1) / teams;
      double load = 0;
      while (b < batch) {
        if (!seqs[b].groups) {
          ++b;
          continue;
        }
        int upto = m + 1 == teams ? seqs[b].tiles : (int)std::min<double>(seqs[b].tiles, end - at[b] - kItemCost + 0.5);
        if (seqs[b].tiles - upto <= 2 && upto > tile) upto = seqs[b].tiles;  // no crumbs
        if (upto <= tile || (tile == 0 && upto <= 2 && upto < seqs[b].tiles)) break;
        const bool part = tile > 0 || upto < seqs[b].tiles;
        for (int g = 0; g < groups; ++g) {
          add(d, b, g, tile, upto, part);
          d.cta.push_back(m * groups + g);
          slots += part;
        }
        load += upto - tile + kItemCost;
        tile = upto;
        if (tile < seqs[b].tiles) break;
        ++b;
        tile = 0;
      }
      worst = std::max(worst, load);
    }
    d.cost = worst + merge_cost(slots);
    best = std::move(d);
  }
  // Otherwise a sequence's tiles are cut into ceil(tiles / w) equal chunks.  For
  // a few lengths w around the share of a CTA, the items are dealt longest first
  // to the least loaded CTA; the w whose busiest CTA ends first wins.
  const double share = (double)total / ctas;
  for (double f : {1e9, 1.0, 0.5, 0.34, 0.25, 0.17}) {
    const int w = (int)std::min<double>(longest, std::max(1.0, std::ceil(f * share)));
    Deal d;
    int slots = 0;
    for (int b = 0; b < batch; ++b) {
      if (!seqs[b].groups) continue;
      const int n = (seqs[b].tiles + w - 1) / w;
      for (int c = 0; c < n; ++c)
        for (int g = 0; g < seqs[b].groups; ++g) {
          add(d, b, g, (int)((long long)seqs[b].tiles * c / n), (int)((long long)seqs[b].tiles * (c + 1) / n), n > 1);
          slots += n > 1;
        }
    }
    if (d.items.size() > 16384 && best.cost < 1e30) continue;
    std::vector<int> order(d.items.size());
    for (size_t i = 0; i < order.size(); ++i) order[i] = (int)i;
    auto size = [&](int i) { return d.items[i].tile1 - d.items[i].tile0; };
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return size(x) > size(y); });
    typedef std::pair<double, int> Load;
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
    for (int c = 0; c < ctas; ++c) heap.push({0.0, c});
    d.cta.resize(d.items.size());
    double end = 0;
    for (int i : order) {
      Load l = heap.top();
      heap.pop();
      l.first += size(i) + kItemCost;
      end = std::max(end, l.first);
      d.cta[i] = l.second;
      heap.push(l);
    }
    d.cost = end + merge_cost(slots);
    if (d.cost < best.cost) best = std::move(d);
  }
  // items of a CTA in the order of the plan; empty CTAs are left out
  std::vector<std::vector<int>> of(ctas);
  for (size_t i = 0; i < best.items.size(); ++i) of[best.cta[i]].push_back((int)i);
  // partial slots: the chunks of a (sequence, group) lie next to each other
  size_t i0 = 0;
  for (int b = 0; b < batch; ++b) {
    if (!seqs[b].groups) continue;
    size_t i1 = i0;
    while (i1 < best.items.size() && best.items[i1].node0 >= hp.first_node[b] &&
           best.items[i1].node0 < hp.first_node[b] + hp.tree[b])
      ++i1;
    const int n = (int)(i1 - i0) / seqs[b].groups;
    if (n > 1) {
      for (int g = 0; g < seqs[b].groups; ++g) {
        const TreeItem &im = best.items[i0 + g];
        hp.merges.push_back({im.node0, im.nn, hp.slots, n});
        for (int c = 0; c < n; ++c) best.items[i0 + (size_t)c * seqs[b].groups + g].slot = hp.slots + c;
        hp.slots += n;
      }
      hp.max_merge = std::max(hp.max_merge, n);
    }
    i0 = i1;
  }
  // CTA c's items: number c, then along `next`
  for (int c = 0; c < ctas; ++c)
    if (!of[c].empty()) hp.items.push_back(best.items[of[c][0]]);
  hp.grid = (int)hp.items.size();
  for (int c = 0, n = 0; c < ctas; ++c) {
    if (of[c].empty()) continue;
    int last = n++;
    for (size_t k = 1; k < of[c].size(); ++k) {
      hp.items[last].next = (int)hp.items.size();
      last = (int)hp.items.size();
      hp.items.push_back(best.items[of[c][k]]);
    }
    hp.items[last].next = -1;
  }
}

}  // namespace kvl
