// tree_capi.cu -- entry points of the tree attention (include/kvl/mla_cuda.h):
// the plan, the attend over a bf16 or Q8 pool, and the host helper that turns
// a tree's parents into mask words.
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <vector>

#include "attend_host.cuh"
#include "kvl/mla_cuda.h"
#include "tree_attend.cuh"
#include "tree_plan.cuh"

#define KVL_EXPORT extern "C" __attribute__((visibility("default")))

namespace kvl {

void set_error_text(const char *msg);

static int fail(const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_error_text(buf);
  return -1;
}

// The plan's arrays in one device allocation, the partials in another.
static int upload(KvlMlaTreePlan &p) {
  const TreeHostPlan &h = p.host;
  std::vector<long long> rows;  // of the nodes in the pool
  rows.reserve(h.nodes);
  for (size_t b = 0; b < h.row0.size(); ++b)
    for (int j = 0; j < h.tree[b]; ++j) rows.push_back(h.row0[b] + h.len[b] + j);
  struct Part {
    const void *src;
    size_t bytes;
    size_t *off;
  } parts[] = {
      {h.items.data(), h.items.size() * sizeof(TreeItem), &p.off_items},
      {h.merges.data(), h.merges.size() * sizeof(TreeMerge), &p.off_merge},
      {h.row0.data(), h.row0.size() * sizeof(long long), &p.off_row0},
      {h.len.data(), h.len.size() * sizeof(int), &p.off_len},
      {h.tree.data(), h.tree.size() * sizeof(int), &p.off_tree},
      {h.first_node.data(), h.first_node.size() * sizeof(int), &p.off_first},
      {h.seq_of_node.data(), h.seq_of_node.size() * sizeof(int), &p.off_seq},
      {rows.data(), rows.size() * sizeof(long long), &p.off_rows},
  };
  size_t at = 256;  // the error word
  for (Part &q : parts) {
    *q.off = at;
    at += (q.bytes + 255) & ~size_t(255);
  }
  std::vector<uint8_t> stage(at, 0);
  for (Part &q : parts)
    if (q.bytes) std::memcpy(stage.data() + *q.off, q.src, q.bytes);
  if (cudaMalloc(&p.d_meta, at) != cudaSuccess) return -1;
  const size_t work = (size_t)h.slots * kTreeRows * (kLatent + 1) * sizeof(float);
  if (work && cudaMalloc(&p.d_work, work) != cudaSuccess) return -1;
  // The copy may return before its last bytes have arrived; the plan can be used
  // on any stream afterwards, also on one that does not wait for this one.
  return cudaMemcpy(p.d_meta, stage.data(), at, cudaMemcpyHostToDevice) == cudaSuccess &&
                 cudaStreamSynchronize(cudaStreamLegacy) == cudaSuccess
             ? 0
             : -1;
}

static void release(KvlMlaTreePlan *p) {
  if (p->d_meta) cudaFree(p->d_meta);
  if (p->d_work) cudaFree(p->d_work);
  delete p;
}

static int attend(const KvlMlaTreePlan *plan, uint16_t *out, float *lse, const uint16_t *q, const uint64_t *mask,
                  const uint16_t *kv, const int8_t *lat8, const float *lscale, const uint16_t *rope16, int64_t rows,
                  int nh, int R, int DR, float softmax_scale, cudaStream_t s) {
  if (!plan || !out || !q || !mask || (!kv && (!lat8 || !lscale || !rope16)))
    return fail("tree attend: null argument");
  if (nh != plan->nh || R != plan->R || DR <= 0 || (DR & 1))
    return fail("tree attend: %d heads x %d, rope %d do not match the plan (%d x %d)", nh, R, DR, plan->nh, plan->R);
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev != plan->device)
    return fail("tree attend: the plan belongs to device %d, the current device is %d", plan->device, dev);
  if (rows < plan->host.rows_needed)
    return fail("tree attend: a sequence ends at pool row %lld, the pool has %lld", plan->host.rows_needed,
                static_cast<long long>(rows));
  const uint8_t *m = static_cast<const uint8_t *>(plan->d_meta);
  const float scale_log2 = softmax_scale * 1.4426950408889634f;
  auto align = [](const void *x) { return reinterpret_cast<uintptr_t>(x); };
  if ((align(mask) & 7) || (align(lse) & 3) || (align(lscale) & 3) ||
      ((align(out) | align(q) | align(kv) | align(rope16)) & 1))
    return fail("tree attend: a pointer is not aligned to its type");
  const bool production = nh == kHeads && R == kLatent && DR == kRope;
  if (production && ((align(out) | align(q) | align(kv) | align(lat8) | align(rope16)) & 15))
    return fail("tree attend: the queries, the output and the pool must be 16-byte aligned");
  if (production) {
    if (rows >= (1LL << 31)) return fail("tree attend: %lld rows", static_cast<long long>(rows));
    TreeParams p;
    std::memset(&p, 0, sizeof p);
    const bool q8 = !kv;
    if (!tree_maps(p, q, kv, rope16, out, plan->host.nodes, rows)) return fail("tree attend: tensor map");
    p.kv = kv;
    p.lat8 = lat8;
    p.lscale = lscale;
    p.mask = mask;
    p.out = out;
    p.lse = lse;
    p.part_o = static_cast<float *>(plan->d_work);
    p.part_lse = p.part_o + (size_t)plan->host.slots * kTreeRows * kLatent;
    p.items = reinterpret_cast<const TreeItem *>(m + plan->off_items);
    p.rows = rows;
    p.scale_log2 = scale_log2;
    p.out_32 = (align(out) & 31) == 0;
    p.err = static_cast<uint32_t *>(plan->d_meta);
    cudaError_t e = launch_tree_attend(p, q8, plan->host.grid, s);
    if (e == cudaSuccess)
      e = launch_tree_merge(p, reinterpret_cast<const TreeMerge *>(m + plan->off_merge),
                            static_cast<int>(plan->host.merges.size()), plan->host.max_merge, s);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail("tree attend launch failed: %s", cudaGetErrorString(e));
    }
    return 0;
  }
  TreeGenericParams g;
  std::memset(&g, 0, sizeof g);
  g.q = q;
  g.kv = kv;
  g.lat8 = lat8;
  g.lscale = lscale;
  g.rope16 = rope16;
  g.mask = mask;
  g.out = out;
  g.lse = lse;
  g.seq_of_node = reinterpret_cast<const int *>(m + plan->off_seq);
  g.first_node = reinterpret_cast<const int *>(m + plan->off_first);
  g.len = reinterpret_cast<const int *>(m + plan->off_len);
  g.tree = reinterpret_cast<const int *>(m + plan->off_tree);
  g.row0 = reinterpret_cast<const long long *>(m + plan->off_row0);
  g.nh = nh;
  g.R = R;
  g.DR = DR;
  g.scale_log2 = scale_log2;
  const cudaError_t e = launch_tree_generic(g, plan->host.nodes, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail("tree attend launch failed: %s", cudaGetErrorString(e));
  }
  return 0;
}

}  // namespace kvl

using namespace kvl;

KVL_EXPORT int kvl_mla_tree_mask(uint64_t *mask, const int *parent, int nodes) {
  if (!mask || !parent || nodes < 1 || nodes > kTreeMaxNodes)
    return fail("tree mask: 1 to %d nodes", kTreeMaxNodes);
  for (int i = 0; i < nodes; ++i)
    if (parent[i] < -1 || parent[i] >= i)
      return fail("tree mask: node %d has parent %d (a parent comes before its children; -1 for a root)", i, parent[i]);
  for (int i = 0; i < nodes; ++i) mask[i] = (parent[i] >= 0 ? mask[parent[i]] : 0) | (uint64_t(1) << i);
  return 0;
}

KVL_EXPORT int kvl_mla_tree_plan_create(KvlMlaTreePlan **plan, int batch, const int *cached_len, const int *nodes,
                                        const int64_t *seq_row0, int num_heads, int kv_lora_rank, int max_ctas) {
  if (!plan) return fail("tree plan: null plan");
  *plan = nullptr;
  if (batch <= 0 || !cached_len || !nodes || !seq_row0 || num_heads <= 0 || num_heads > 65535 || kv_lora_rank <= 0 ||
      max_ctas < 0)
    return fail("tree plan: invalid arguments");
  KvlMlaTreePlan *p = nullptr;
  try {
    p = new KvlMlaTreePlan();
    if (set_tree_sequences(p->host, batch, cached_len, nodes, seq_row0) != 0) {
      release(p);
      return fail("tree plan: cached lengths >= 0, 0 to %d nodes a sequence and one at least, rows >= 0 and below 2^31",
                  kTreeMaxNodes);
    }
    int dev = -1, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      release(p);
      return fail("tree plan: no CUDA device");
    }
    p->device = dev;
    p->nh = num_heads;
    p->R = kv_lora_rank;
    deal_tree_tiles(p->host, max_ctas > 0 ? max_ctas : sms);
    if (upload(*p) != 0) {
      cudaGetLastError();
      release(p);
      return fail("tree plan: device memory");
    }
  } catch (...) {
    if (p) release(p);
    return fail("tree plan: out of host memory");
  }
  *plan = p;
  return 0;
}

KVL_EXPORT void kvl_mla_tree_plan_destroy(KvlMlaTreePlan *plan) {
  if (plan) release(plan);
}

KVL_EXPORT int kvl_mla_tree_plan_info(const KvlMlaTreePlan *plan, int *ctas, int *partials, int *items) {
  if (!plan) return fail("tree plan: null plan");
  if (ctas) *ctas = plan->host.grid;
  if (partials) *partials = plan->host.slots;
  if (items) *items = static_cast<int>(plan->host.items.size());
  return 0;
}

KVL_EXPORT int kvl_mla_tree_attend_bf16(const KvlMlaTreePlan *plan, uint16_t *d_out, float *d_lse,
                                        const uint16_t *d_q, const uint64_t *d_mask, const uint16_t *d_kv,
                                        int64_t rows, int num_heads, int kv_lora_rank, int rope_dim,
                                        float softmax_scale, void *stream) {
  if (!d_kv) return fail("tree attend: null kv pool");
  return attend(plan, d_out, d_lse, d_q, d_mask, d_kv, nullptr, nullptr, nullptr, rows, num_heads, kv_lora_rank,
                rope_dim, softmax_scale, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_tree_attend_q8(const KvlMlaTreePlan *plan, uint16_t *d_out, float *d_lse, const uint16_t *d_q,
                                      const uint64_t *d_mask, const int8_t *d_latent_q8, const float *d_latent_scale,
                                      const uint16_t *d_rope_bf16, int64_t rows, int num_heads, int kv_lora_rank,
                                      int rope_dim, float softmax_scale, void *stream) {
  if (!d_latent_q8 || !d_latent_scale || !d_rope_bf16) return fail("tree attend: null q8 pool");
  return attend(plan, d_out, d_lse, d_q, d_mask, nullptr, d_latent_q8, d_latent_scale, d_rope_bf16, rows, num_heads,
                kv_lora_rank, rope_dim, softmax_scale, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_tree_check(const KvlMlaTreePlan *plan, void *stream) {
  if (!plan) return fail("tree check: null plan");
  uint32_t err = 0;
  if (cudaStreamSynchronize(static_cast<cudaStream_t>(stream)) != cudaSuccess ||
      cudaMemcpy(&err, plan->d_meta, 4, cudaMemcpyDeviceToHost) != cudaSuccess)
    return fail("tree check: %s", cudaGetErrorString(cudaGetLastError()));
  if (err) {
    cudaMemset(plan->d_meta, 0, 4);
    cudaStreamSynchronize(cudaStreamLegacy);
    return fail("tree attend: device-side error 0x%x", err);
  }
  return 0;
}
