// Prints the plans of the tree attention (csrc/tree_plan.cu, host code) for
// batches read from standard input: "batch ctas", then cached length, nodes and
// first row of every sequence.  Per batch: "-1" when it is refused, else
//   grid slots max_merge rows_needed own_rows #items #merges
// and a line per item and per merge entry.
#include <cstdio>
#include <vector>

#include "tree_attend.cuh"

int main() {
  int batch, ctas;
  while (std::scanf("%d %d", &batch, &ctas) == 2) {
    std::vector<int> len(batch), nodes(batch);
    std::vector<int64_t> row0(batch);
    for (int b = 0; b < batch; ++b) {
      long long r;
      if (std::scanf("%d %d %lld", &len[b], &nodes[b], &r) != 3) return 1;
      row0[b] = r;
    }
    kvl::TreeHostPlan p;
    if (kvl::set_tree_sequences(p, batch, len.data(), nodes.data(), row0.data()) != 0) {
      std::puts("-1");
      continue;
    }
    kvl::deal_tree_tiles(p, ctas);
    std::printf("%d %d %d %lld %d %zu %zu\n", p.grid, p.slots, p.max_merge, p.rows_needed, (int)p.own_rows,
                p.items.size(), p.merges.size());
    for (const kvl::TreeItem &i : p.items)
      std::printf("%lld %d %d %d %d %d %d %d %d\n", i.row0, i.len, i.tree, i.node0, i.nn, i.tile0, i.tile1, i.slot,
                  i.next);
    for (const kvl::TreeMerge &m : p.merges) std::printf("%d %d %d %d\n", m.node0, m.nn, m.first, m.count);
  }
  return 0;
}
