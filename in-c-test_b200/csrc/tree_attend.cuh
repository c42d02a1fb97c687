// tree_attend.cuh -- attention of a tree of drafted tokens over the latent
// cache: the work plan (tree_plan.cu) and the launchers (kernels in tree_attend.cu).
//
// Sequence b has L_b cached rows at pool rows [row0_b, row0_b + L_b) and T_b
// drafted rows right behind them.  Node i of its tree (head h) attends the
// cached rows and the drafted rows whose bit is set in the node's mask word:
//     s_j   = (q_lat . latent_j + q_rope . rope_j) * scale
//     out   = sum_j softmax(s)_j * latent_j,   lse = log sum_j exp(s_j)
// over the visible j; a node that sees no row gets out = 0, lse = -inf.
//
// Work decomposition: four nodes (64 query rows: 4 nodes x 16 heads) form a
// group, the M of the score MMA.  The keys of a sequence are cut into tiles of
// 64 rows and the tiles into chunks; an item is (chunk, group).  Items of the
// same chunk lie next to each other in the plan, so the groups of a tree walk
// the same rows at the same time and all but one of them read L2.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <vector>

#include "attend_common.cuh"

namespace kvl {

constexpr int kTreeMaxNodes = 64;                      // one mask word
constexpr int kTreeGroup = 4;                          // nodes of a group
constexpr int kTreeRows = kTreeGroup * kHeads;         // query rows of a group
constexpr int kTreeKeys = 64;                          // key rows of a tile

struct alignas(16) TreeItem {
  long long row0;  // pool row of the sequence's row 0
  int len;         // cached rows of the sequence
  int tree;        // its drafted rows
  int node0;       // first node of the group (index over the batch)
  int nn;          // nodes of the group (1..4)
  int tile0, tile1;  // tiles [tile0, tile1)
  int slot;        // partial slot, or -1 when the chunk is the whole sequence
  int next;        // next item of the CTA, or -1; CTA c starts with item c
};

// The (sequence, group) results that are combined from partials.
struct TreeMerge {
  int node0, nn;
  int first, count;  // partial slots [first, first + count)
};

struct TreeParams {
  CUtensorMap tm_lat;   // bf16 pool: [box of 64 dims][rows][64], 4 x 64 x 64 a load
  CUtensorMap tm_rope;  // bf16 pool or the Q8 pool's rope, 64 rows x 64
  CUtensorMap tm_q;     // the query's latents: [node][pair of boxes][odd][16 heads][64], a load: 4 x 1 x 2 x 16 x 64
  CUtensorMap tm_qr;    // its rope: 64 rows (4 nodes) x 64
  CUtensorMap tm_out;   // out [nodes * 16][512]: 16 rows x 64 dims
  const uint16_t *kv;   // bf16 pool, or
  const int8_t *lat8;   // Q8 pool
  const float *lscale;
  const uint64_t *mask; // [nodes]
  uint16_t *out;        // [nodes][16][512] bf16
  float *lse;           // [nodes][16] or null
  float *part_o;        // [slots][64][512]
  float *part_lse;      // [slots][64]
  const TreeItem *items;
  long long rows;
  float scale_log2;
  int out_32;           // out is 32-byte aligned
  uint32_t *err;
};

// Host copy of a plan.
struct TreeHostPlan {
  int batch = 0, nodes = 0, grid = 0, slots = 0, max_merge = 0;
  std::vector<TreeItem> items;
  std::vector<TreeMerge> merges;
  std::vector<int> len, tree, seq_of_node, first_node;
  std::vector<long long> row0;
  long long rows_needed = 0;  // one past the last pool row that any sequence uses
  bool own_rows = true;       // no drafted row is another sequence's drafted or cached row
};

// The plan in two steps (tree_plan.cu): the batch's sequences, -1 if one is out
// of range, then its items for a grid of at most `ctas` >= 1.
int set_tree_sequences(TreeHostPlan &hp, int batch, const int *cached_len, const int *nodes, const int64_t *row0);
void deal_tree_tiles(TreeHostPlan &hp, int ctas);

struct TreeGenericParams {
  const uint16_t *q;
  const uint16_t *kv;      // bf16 pool, or null for the Q8 arrays
  const int8_t *lat8;
  const float *lscale;
  const uint16_t *rope16;
  const uint64_t *mask;
  uint16_t *out;
  float *lse;
  const int *seq_of_node, *first_node, *len, *tree;
  const long long *row0;
  int nh, R, DR;
  float scale_log2;
};

bool tree_maps(TreeParams &p, const uint16_t *q, const uint16_t *kv, const uint16_t *rope16, uint16_t *out, int nodes,
               int64_t rows);  // kv null: a Q8 pool
cudaError_t launch_tree_attend(const TreeParams &p, bool q8, int grid, cudaStream_t s);
cudaError_t launch_tree_merge(const TreeParams &p, const TreeMerge *entries, int n, int max_count, cudaStream_t s);
cudaError_t launch_tree_generic(const TreeGenericParams &p, int nodes, cudaStream_t s);

}  // namespace kvl
