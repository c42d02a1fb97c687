// tree_attend.cu -- attention of a tree of drafted tokens over the latent
// cache (tree_attend.cuh has the formula and the work decomposition).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <queue>

#include "merge_core.cuh"
#include "prof.cuh"
#include "sm100.cuh"
#include "tree_attend.cuh"

namespace kvl {

// ------------------------------------------------------------------ plan
// What an item costs beside its tiles (query load, first tile, epilogue), a
// partial one more (fp32 output), and the merge launch, in tiles.
static constexpr double kItemCost = 3.0, kPartCost = 1.0, kMergeCost = 3.0;

int build_tree_plan(TreeHostPlan &hp, int batch, const int *cached_len, const int *nodes, const int64_t *row0,
                    int ctas) {
  if (batch <= 0 || ctas <= 0) return -1;
  hp = TreeHostPlan();
  hp.batch = batch;
  for (int b = 0; b < batch; ++b) {
    if (cached_len[b] < 0 || nodes[b] < 0 || nodes[b] > kTreeMaxNodes || row0[b] < 0) return -1;
    const long long end = (long long)row0[b] + cached_len[b] + nodes[b];
    if (row0[b] >= (1LL << 31) || end >= (1LL << 31)) return -1;
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

  // Chunk length: a sequence's tiles are cut into ceil(tiles / w) equal chunks.
  // For a few lengths w around the share of a CTA, the items are dealt longest
  // first to the least loaded CTA; the w whose busiest CTA ends first wins.
  struct Seq {
    int tiles, groups;
  };
  std::vector<Seq> seqs(batch);
  long long total = 0;
  int longest = 1;
  for (int b = 0; b < batch; ++b) {
    const int keys = hp.len[b] + hp.tree[b];
    seqs[b] = {hp.tree[b] ? (keys + kTreeKeys - 1) / kTreeKeys : 0, (hp.tree[b] + kTreeGroup - 1) / kTreeGroup};
    total += (long long)seqs[b].tiles * seqs[b].groups;
    longest = std::max(longest, seqs[b].tiles);
  }
  struct Deal {
    std::vector<TreeItem> items;
    std::vector<int> cta;  // of each item
    double cost = 1e30;
  };
  Deal best;
  const double share = (double)total / ctas;
  for (double f : {1e9, 1.0, 0.5, 0.34, 0.25, 0.125}) {
    const int w = (int)std::min<double>(longest, std::max(1.0, std::ceil(f * share)));
    Deal d;
    int slots = 0, most = 0;
    for (int b = 0; b < batch; ++b) {
      if (!seqs[b].groups) continue;
      const int n = (seqs[b].tiles + w - 1) / w;
      most = std::max(most, n);
      for (int c = 0; c < n; ++c)
        for (int g = 0; g < seqs[b].groups; ++g) {
          TreeItem im;
          im.row0 = hp.row0[b];
          im.len = hp.len[b];
          im.tree = hp.tree[b];
          im.node0 = hp.first_node[b] + g * kTreeGroup;
          im.nn = std::min(kTreeGroup, hp.tree[b] - g * kTreeGroup);
          im.tile0 = (int)((long long)seqs[b].tiles * c / n);
          im.tile1 = (int)((long long)seqs[b].tiles * (c + 1) / n);
          im.slot = n > 1 ? 0 : -1;
          slots += n > 1;
          d.items.push_back(im);
        }
    }
    if (d.items.size() > 65536 && best.cost < 1e30) continue;
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
      l.first += size(i) + kItemCost + (d.items[i].slot >= 0 ? kPartCost : 0.0);
      end = std::max(end, l.first);
      d.cta[i] = l.second;
      heap.push(l);
    }
    d.cost = end + (most > 1 ? kMergeCost + 0.02 * most + 0.01 * slots : 0.0);
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
  hp.cta_item.push_back(0);
  for (const std::vector<int> &v : of) {
    if (v.empty()) continue;
    for (int i : v) hp.items.push_back(best.items[i]);
    hp.cta_item.push_back((int)hp.items.size());
  }
  hp.grid = (int)hp.cta_item.size() - 1;
  return 0;
}

// ------------------------------------------------------------------ any shape
// One CTA per (head, node); online softmax in fp32 over chunks of 1024 rows.
// Runs for shapes other than 16 heads x 512 x 64.  A row that the node does
// not see is never read, so nothing in it can reach the result.
template <bool Q8>
__global__ void tree_generic_kernel(const TreeGenericParams p) {
  constexpr int kChunk = 1024;
  const int h = blockIdx.y, node = blockIdx.x;
  const int R = p.R, DR = p.DR;
  extern __shared__ float sm[];
  float *qv = sm;              // R + DR
  float *sc = qv + R + DR;     // kChunk
  float *acc = sc + kChunk;    // R
  float *red = acc + R;        // 32
  const int b = p.seq_of_node[node];
  const int L = p.len[b], n = L + p.tree[b];
  const long long r0 = p.row0[b];
  const uint64_t mask = p.mask[node];
  const uint16_t *qs = p.q + ((size_t)node * p.nh + h) * (R + DR);
  for (int i = threadIdx.x; i < R + DR; i += blockDim.x) qv[i] = __bfloat162float(__ushort_as_bfloat16(qs[i]));
  for (int i = threadIdx.x; i < R; i += blockDim.x) acc[i] = 0.f;
  __syncthreads();
  auto lat = [&](long long row, int r) -> float {
    if (Q8) return __fmul_rn((float)p.lat8[row * R + r], p.lscale[row]);
    return __bfloat162float(__ushort_as_bfloat16(p.kv[row * (R + DR) + r]));
  };
  auto rope = [&](long long row, int d) -> float {
    if (Q8) return __bfloat162float(__ushort_as_bfloat16(p.rope16[row * DR + d]));
    return __bfloat162float(__ushort_as_bfloat16(p.kv[row * (R + DR) + R + d]));
  };
  auto seen = [&](int j) { return j < L || ((mask >> (j - L)) & 1) != 0; };
  auto block_reduce = [&](float v, bool is_max) -> float {
    for (int off = 16; off > 0; off >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, off);
      v = is_max ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = is_max ? -INFINITY : 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) r = is_max ? fmaxf(r, red[i]) : r + red[i];
    return r;
  };
  float m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < n; j0 += kChunk) {
    const int c = min(kChunk, n - j0);
    float cmax = -INFINITY;
    for (int j = threadIdx.x; j < c; j += blockDim.x) {
      const long long row = r0 + j0 + j;
      float s = -INFINITY;
      if (seen(j0 + j)) {
        s = 0.f;
        for (int r = 0; r < R; ++r) s = fmaf(qv[r], lat(row, r), s);
        for (int d = 0; d < DR; ++d) s = fmaf(qv[R + d], rope(row, d), s);
        s *= p.scale_log2;
      }
      sc[j] = s;
      cmax = fmaxf(cmax, s);
    }
    cmax = block_reduce(cmax, true);
    const float mn = fmaxf(m, cmax);
    const float base = mn == -INFINITY ? 0.f : mn;  // nothing seen so far: every weight is exp2(-inf) = 0
    const float alpha = (m == -INFINITY) ? 0.f : exp2f(m - mn);
    float psum = 0.f;
    for (int j = threadIdx.x; j < c; j += blockDim.x) {
      sc[j] = exp2f(sc[j] - base);
      psum += sc[j];
    }
    psum = block_reduce(psum, false);
    __syncthreads();
    for (int r = threadIdx.x; r < R; r += blockDim.x) {
      float a = acc[r] * alpha;
      for (int j = 0; j < c; ++j)
        if (seen(j0 + j)) a = fmaf(sc[j], lat(r0 + j0 + j, r), a);
      acc[r] = a;
    }
    l = l * alpha + psum;
    m = mn;
    __syncthreads();
  }
  uint16_t *os = p.out + ((size_t)node * p.nh + h) * R;
  for (int r = threadIdx.x; r < R; r += blockDim.x)
    os[r] = __bfloat16_as_ushort(__float2bfloat16_rn(l == 0.f ? 0.f : acc[r] / l));
  if (p.lse && threadIdx.x == 0)
    p.lse[(size_t)node * p.nh + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

cudaError_t launch_tree_generic(const TreeGenericParams &p, int nodes, cudaStream_t s) {
  const size_t sm = (size_t)(p.R + p.DR + 1024 + p.R + 32) * sizeof(float);
  auto f = p.kv ? tree_generic_kernel<false> : tree_generic_kernel<true>;
  if (sm > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
    if (e != cudaSuccess) return e;
  }
  ProfScope ps("tree_generic", s);
  f<<<dim3(nodes, p.nh), 128, sm, s>>>(p);
  return cudaGetLastError();
}


// ------------------------------------------------------------------ 16 x 512 x 64
namespace treek {

constexpr uint32_t kBox = kTreeKeys * 128;  // 64 rows x 64 dims bf16 = 8 KB, one SW128 box
constexpr int kBoxes = kRow / 64;           // 8 latent boxes and the rope box
constexpr int kStages = 2;                  // key tiles in shared memory
constexpr uint32_t kStage = kBoxes * kBox;
constexpr uint32_t OFF_Q = 0;
constexpr uint32_t OFF_KV = OFF_Q + kBoxes * kBox;
constexpr uint32_t OFF_P = OFF_KV + kStages * kStage;
constexpr uint32_t OFF_BAR = OFF_P + kBox;

// The three pieces of a tile in the order they are loaded: rope, latent dims
// 0-255, latent dims 256-511.  The rope is free once the scores are done, each
// latent half once its half of the P.V is.
enum { CH_ROPE = 0, CH_LO = 1, CH_HI = 2, kChunks = 3 };

struct Bars {
  uint64_t full[kStages][kChunks], empty[kStages][kChunks];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], s_empty[2];
  uint64_t p_full, pv_done, o_empty, drain;
  uint32_t tmem_base;
  int abort;
  uint32_t nonfinite[4];
  float red[3][128];  // row maxima of alternate tiles; row sums at an item's end
  float scale[kStages][kTreeKeys];  // Q8: row scales of the tile
};
constexpr uint32_t kSmemBytes = OFF_BAR + sizeof(Bars);
static_assert(kSmemBytes <= 232448, "shared memory budget");

// Tensor memory: O (64 rows x 512) in 256 columns -- dims [256 i, 256 i + 128)
// in columns [128 i, 128 i + 128) of lanes 0-63, the next 128 dims in lanes
// 64-127 -- and two score buffers of 64 columns (32 latent; Q8: 32 more rope).
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 256;
constexpr uint32_t kSCols = 64;

constexpr int kConvertWarp = 8;  // Q8: warps 8-15 load and convert the latents
constexpr int kConvertThreads = 256;
template <bool Q8>
constexpr int threads() { return Q8 ? 256 + kConvertThreads : 256; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two of the four int8 in `w` (bytes i, i + 1) as bf16.  0x4300 is 128 with a
// unit in the last place: 128 + (b & 127) less 128, or 256 for a negative b
// (128 + 128 = 0x4380), is b exactly.
template <int I>
__device__ __forceinline__ uint32_t s8x2_to_bf16(uint32_t w) {
  const uint32_t v = __byte_perm(w, 0u, I == 0 ? 0x4140 : 0x4342);
  const uint32_t lo = (v & 0x007f007fu) | 0x43004300u, hi = (v & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&lo),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&hi));
  return *reinterpret_cast<const uint32_t *>(&d);
}

}  // namespace treek

using namespace treek;

// One CTA per SM, roles by warp:
//   0      TMA producer (bf16: whole rows; Q8: the rope)
//   1      tcgen05 issuer
//   2      query loader: 64 rows x 576 per item
//   4-7    softmax and epilogue: thread t has query row t % 64 and keys
//          32 (t / 64) .. + 31 of a tile (where .ws puts them)
//   8-15   Q8: latents from global memory, as bf16 into the ring
template <bool Q8>
__global__ void __launch_bounds__(threads<Q8>(), 1) tree_attend_kernel(const __grid_constant__ TreeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars *B = reinterpret_cast<Bars *>(smem + OFF_BAR);
  const uint32_t s_base = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int it0 = p.cta_item[blockIdx.x], it1 = p.cta_item[blockIdx.x + 1];
  volatile int *abort = &B->abort;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i)
      for (int c = 0; c < kChunks; ++c) {
        mbar_init(&B->full[i][c], Q8 && c != CH_ROPE ? kConvertThreads / 32 : 1);
        mbar_init(&B->empty[i][c], 1);
      }
    mbar_init(&B->q_full, 1);
    mbar_init(&B->q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->s_full[i], 1);
      mbar_init(&B->s_empty[i], 4);
    }
    mbar_init(&B->p_full, 4);
    mbar_init(&B->pv_done, 1);
    mbar_init(&B->o_empty, 4);
    mbar_init(&B->drain, 1);
    B->abort = 0;
    if (s_base & 1023) {  // the swizzle atoms
      B->abort = 1;
      atomicOr(p.err, ERR_BAD_PARAM);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&B->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B->tmem_base;
  const bool fit = !*abort;  // the same for all threads
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp == 0 && fit) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tm_kv);
      uint32_t g = 0, issued = 0;  // chunks issued
      bool ok = true;
      for (int it = it0; it < it1 && ok; ++it) {
        const TreeItem im = p.items[it];
        for (int t = im.tile0; t < im.tile1 && ok; ++t, ++g) {
          const uint32_t st = g % kStages, par = ((g / kStages) & 1) ^ 1;
          const int32_t y = static_cast<int32_t>(im.row0 + static_cast<long long>(kTreeKeys) * t);
          uint8_t *dst = smem + OFF_KV + st * kStage;
          for (int c = 0; c < (Q8 ? 1 : kChunks); ++c) {
            ok = mbar_wait(&B->empty[st][c], par, abort, p.err, ERR_TIMEOUT_EMPTY);
            if (!ok) break;
            if (c == CH_ROPE) {
              mbar_arrive_expect_tx(&B->full[st][c], kBox);
              tma_load_2d(dst + 8 * kBox, &p.tm_kv, &B->full[st][c], Q8 ? 0 : kLatent, y);
            } else {
              mbar_arrive_expect_tx(&B->full[st][c], 4 * kBox);
              for (int b = 4 * (c - 1); b < 4 * c; ++b)
                tma_load_2d(dst + b * kBox, &p.tm_kv, &B->full[st][c], 64 * b, y);
            }
            ++issued;
          }
        }
      }
      if (!ok) {  // copies in flight land before the CTA exits
        const uint32_t per = Q8 ? 1 : kChunks;
        for (uint32_t k = issued > kStages * per ? issued - kStages * per : 0; k < issued; ++k)
          drain_wait(&B->full[(k / per) % kStages][k % per], (k / per / kStages) & 1, p.err);
      }
    }
  } else if (warp == 1 && fit) {
    if (elect_one()) {
      constexpr uint32_t id_qk = idesc_f16(1, 1, 0, 0, kTreeRows, kTreeKeys);  // both K-major
      constexpr uint32_t id_pv = idesc_f16(1, 1, 0, 1, kTreeRows, 256);        // V rows as they lie: MN-major
      const uint64_t q_desc = smem_desc(s_base + OFF_Q, 16, 1024, LAYOUT_SW128);
      const uint64_t k_desc = smem_desc(s_base + OFF_KV, 16, 1024, LAYOUT_SW128);
      const uint64_t v_desc = smem_desc(s_base + OFF_KV, kBox, 1024, LAYOUT_SW128);
      const uint64_t p_desc = smem_desc(s_base + OFF_P, 16, 1024, LAYOUT_SW128);
      uint32_t g = 0;
      bool ok = true;
      for (int it = it0, n = 0; it < it1 && ok; ++it, ++n) {
        const int t0 = p.items[it].tile0, t1 = p.items[it].tile1;
        ok = mbar_wait(&B->q_full, n & 1, abort, p.err, ERR_TIMEOUT_FULL);
        for (int t = t0; t < t1 && ok; ++t, ++g) {
          const uint32_t st = g % kStages, par = (g / kStages) & 1, sb = g & 1;
          const uint64_t kd = k_desc + (st * kStage >> 4), vd = v_desc + (st * kStage >> 4);
          const uint32_t s_lat = tmem + kColS + sb * kSCols;
          const uint32_t s_rope = s_lat + (Q8 ? 32 : 0);
          // ---- S = Q . K^T
          ok = mbar_wait(&B->s_empty[sb], ((g >> 1) & 1) ^ 1, abort, p.err, ERR_TIMEOUT_EMPTY) &&
               mbar_wait(&B->full[st][CH_ROPE], par, abort, p.err, ERR_TIMEOUT_FULL);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16_ws_ss(s_rope, q_desc + (8 * kBox + kk * 32) / 16, kd + (8 * kBox + kk * 32) / 16, id_qk, kk > 0);
          for (int c = CH_LO; c <= CH_HI && ok; ++c) {
            ok = mbar_wait(&B->full[st][c], par, abort, p.err, ERR_TIMEOUT_FULL);
            if (!ok) break;
            tc_fence_after();
            const uint32_t o = (c - 1) * (4 * kBox / 16);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              mma_f16_ws_ss(s_lat, q_desc + o + ((k >> 2) * kBox + (k & 3) * 32) / 16,
                            kd + o + ((k >> 2) * kBox + (k & 3) * 32) / 16, id_qk,
                            Q8 ? (c > CH_LO || k > 0) : 1u);
          }
          if (!ok) break;
          mma_commit(&B->s_full[sb]);
          mma_commit(&B->empty[st][CH_ROPE]);
          if (t + 1 == t1) mma_commit(&B->q_empty);
          // ---- O += P . V
          ok = mbar_wait(&B->p_full, g & 1, abort, p.err, ERR_TIMEOUT_FULL);
          if (ok && t == t0 && n > 0) ok = mbar_wait(&B->o_empty, (n - 1) & 1, abort, p.err, ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_ws_ss(tmem + 128 * h, p_desc + kk * 2, vd + (h * 4 * kBox + kk * 2048) / 16, id_pv,
                            t > t0 || kk > 0);
            mma_commit(&B->empty[st][CH_LO + h]);
          }
          mma_commit(&B->pv_done);
        }
      }
      // issued tensor-core work ends before tensor memory is released
      mma_commit(&B->drain);
      drain_wait(&B->drain, 0, p.err);
    }
  } else if (warp == 2 && fit) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tm_q);
      bool ok = true;
      int n = 0;
      for (int it = it0; it < it1; ++it, ++n) {
        const int node0 = p.items[it].node0;
        if (n > 0) ok = mbar_wait(&B->q_empty, (n - 1) & 1, abort, p.err, ERR_TIMEOUT_EMPTY);
        if (!ok) break;
        mbar_arrive_expect_tx(&B->q_full, kBoxes * kBox);
        for (int b = 0; b < kBoxes; ++b)
          tma_load_2d(smem + OFF_Q + b * kBox, &p.tm_q, &B->q_full, 64 * b, node0 * kHeads);
      }
      if (!ok) drain_wait(&B->q_full, (n - 1) & 1, p.err);
    }
  } else if (warp >= 4 && warp < 8 && fit) {
    const int tid = threadIdx.x - 128;
    const int row = tid & 63, half = tid >> 6;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp - 4)) << 16;
    uint32_t g = 0;
    bool bad = false;
    for (int it = it0; it < it1 && !bad; ++it) {
      const TreeItem im = p.items[it];
      const bool real = row < im.nn * kHeads;
      uint64_t mask = real ? p.mask[im.node0 + row / kHeads] : 0;
      if (im.tree < 64) mask &= (uint64_t(1) << im.tree) - 1;
      float m = -INFINITY, l = 0.f;
      for (int t = im.tile0; t < im.tile1; ++t, ++g) {
        const uint32_t st = g % kStages, sb = g & 1;
        bad |= !mbar_wait(&B->s_full[sb], (g >> 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
        if (Q8) bad |= !mbar_wait(&B->full[st][CH_HI], (g / kStages) & 1, abort, p.err, ERR_TIMEOUT_FULL);
        tc_fence_after();
        float s[32], sr[Q8 ? 32 : 1];
        tmem_ld32(tmem + kColS + sb * kSCols + lanes, s);
        if (Q8) tmem_ld32(tmem + kColS + sb * kSCols + 32 + lanes, sr);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->s_empty[sb]);
        const float *ks = B->scale[st] + 32 * half;
        const int k0 = kTreeKeys * t + 32 * half;  // the thread's first key
        uint32_t seen = 0xffffffffu;
        if (Q8)
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = fmaf(s[c], ks[c], sr[c]);
        const bool masked = kTreeKeys * (t + 1) > im.len;
        if (masked) {
          const int d = k0 - im.len;  // drafted row of the first key
          seen = d >= 0 ? (d < 64 ? static_cast<uint32_t>(mask >> d) : 0u)
                        : (d > -32 ? static_cast<uint32_t>(mask << -d) | (0xffffffffu >> (32 + d)) : 0xffffffffu);
          if (!Q8) {
            // A hidden row gets p = 0, but 0 times an infinity or a NaN of the
            // row itself is NaN in the P.V product.  Such a row gives a score
            // that is not finite with every query (a query that is not finite
            // does so with every row, but only its own): clear those rows.
            uint32_t nf = 0;
#pragma unroll
            for (int c = 0; c < 32; ++c) nf |= ((__float_as_uint(s[c]) & 0x7f800000u) == 0x7f800000u) ? 1u << c : 0u;
            if (named_bar_or(2, 128, (nf & ~seen) != 0)) {
              const uint32_t all = __reduce_and_sync(0xffffffffu, nf);
              if (lane == 0) B->nonfinite[warp - 4] = all;
              named_bar_sync(2, 128);
              const uint64_t rows = static_cast<uint64_t>(B->nonfinite[0] & B->nonfinite[1]) |
                                    static_cast<uint64_t>(B->nonfinite[2] & B->nonfinite[3]) << 32;
              uint8_t *v = smem + OFF_KV + st * kStage + (tid >> 3 & 7) * kBox + (tid & 7) * 16;
              for (int k = tid >> 6; k < kTreeKeys; k += 2)
                if (rows >> k & 1) *reinterpret_cast<uint4 *>(v + k * 128) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          s[c] = (seen >> c & 1) ? s[c] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[c]);
        }
        // the other half of the row's keys
        B->red[sb][tid] = mx;
        if (named_bar_or(1, 128, bad)) {
          bad = true;
          break;
        }
        mx = fmaxf(mx, B->red[sb][tid ^ 64]);
        // The reference maximum moves only when a score exceeds it by 2^8; both
        // warps of a row decide alike.
        if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
          const float mn = fmaxf(m, mx);
          const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
          if (t > im.tile0) {
            bad |= !mbar_wait(&B->pv_done, (g - 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 256; c += 32) {
              float o[32];
              tmem_ld32(tmem + c + lanes, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st32(tmem + c + lanes, o);
            }
            tmem_wait_st();
          }
          l *= alpha;
          m = mn;
        }
        const float ref = m == -INFINITY ? 0.f : m;  // a row that has seen nothing: exp2(-inf) = 0
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float p0 = ex2(s[c] - ref), p1 = ex2(s[c + 1] - ref);
          l += p0 + p1;
          if (Q8) {  // O accumulates p * scale * int8 row; a hidden row's scale may be anything
            p0 = (seen >> c & 1) ? p0 * ks[c] : 0.f;
            p1 = (seen >> (c + 1) & 1) ? p1 * ks[c + 1] : 0.f;
          }
          pk[c / 2] = pack_bf16(p0, p1);
        }
        // P of the tile before is read until its P.V ends
        if (g > 0) bad |= !mbar_wait(&B->pv_done, (g - 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
        uint8_t *pd = smem + OFF_P + (row >> 3) * 1024 + (row & 7) * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4 *>(pd + ((4 * half + c) ^ (row & 7)) * 16) =
              make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->p_full);
      }
      if (bad) break;
      // ---- epilogue
      bad |= !mbar_wait(&B->pv_done, (g - 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
      B->red[2][tid] = l;
      if (named_bar_or(1, 128, bad)) {
        bad = true;
        break;
      }
      tc_fence_after();
      l += B->red[2][tid ^ 64];
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // nothing seen: out = 0, lse = -inf
      if (real && half == 0) {
        const float lse = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
        if (im.slot >= 0)
          p.part_lse[static_cast<size_t>(im.slot) * kTreeRows + row] = lse;
        else if (p.lse)
          p.lse[static_cast<size_t>(im.node0) * kHeads + row] = lse;
      }
      const size_t orow = im.slot >= 0 ? static_cast<size_t>(im.slot) * kTreeRows + row
                                       : static_cast<size_t>(im.node0) * kHeads + row;
#pragma unroll
      for (int c = 0; c < 256; c += 32) {
        float o[32];
        tmem_ld32(tmem + c + lanes, o);
        tmem_wait_ld();
        const int d = (c >> 7) * 256 + half * 128 + (c & 127);
        if (real) {
          if (im.slot >= 0) {
            float4 *dst = reinterpret_cast<float4 *>(p.part_o + orow * kLatent + d);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
          } else {
            uint4 *dst = reinterpret_cast<uint4 *>(p.out + orow * kLatent + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              dst[i] = make_uint4(pack_bf16(o[8 * i] * inv, o[8 * i + 1] * inv),
                                  pack_bf16(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                  pack_bf16(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                                  pack_bf16(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->o_empty);
    }
  } else if (Q8 && warp >= kConvertWarp && fit) {
    // Thread t has the 16 latents c = t % 4 of row t / 4 in each of the eight
    // boxes: four threads read 64 consecutive bytes, and the eight lanes of a
    // store phase (two rows) fill the eight 16-byte banks of the swizzle.
    const int tid = threadIdx.x - 32 * kConvertWarp;
    const int r = tid >> 2, c = tid & 3;
    const long long last = p.rows - 1;
    // the CTA's tiles in order
    int it = it0, t = it0 < it1 ? p.items[it0].tile0 : 0, t1 = it0 < it1 ? p.items[it0].tile1 : 0;
    long long row0 = it0 < it1 ? p.items[it0].row0 : 0;
    auto load = [&](uint4(&v)[8], float &sc) -> bool {
      while (it < it1 && t >= t1) {
        if (++it < it1) {
          t = p.items[it].tile0;
          t1 = p.items[it].tile1;
          row0 = p.items[it].row0;
        }
      }
      if (it >= it1) return false;
      const long long first = row0 + static_cast<long long>(kTreeKeys) * t;
      const uint4 *src = reinterpret_cast<const uint4 *>(p.lat8 + min(first + r, last) * kLatent) + c;
#pragma unroll
      for (int b = 0; b < 8; ++b) v[b] = __ldg(src + 4 * b);
      if (tid < kTreeKeys) sc = __ldg(p.lscale + min(first + tid, last));
      ++t;
      return true;
    };
    uint32_t g = 0;
    auto store = [&](const uint4(&v)[8], float sc) -> bool {
      const uint32_t st = g % kStages, par = ((g / kStages) & 1) ^ 1;
      uint8_t *dst = smem + OFF_KV + st * kStage + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!mbar_wait(&B->empty[st][CH_LO + h], par, abort, p.err, ERR_TIMEOUT_EMPTY)) return false;
        if (h == 1 && tid < kTreeKeys) B->scale[st][tid] = sc;
#pragma unroll
        for (int b = 4 * h; b < 4 * h + 4; ++b) {
          *reinterpret_cast<uint4 *>(dst + b * kBox + ((2 * c) ^ (r & 7)) * 16) =
              make_uint4(s8x2_to_bf16<0>(v[b].x), s8x2_to_bf16<1>(v[b].x), s8x2_to_bf16<0>(v[b].y),
                         s8x2_to_bf16<1>(v[b].y));
          *reinterpret_cast<uint4 *>(dst + b * kBox + ((2 * c + 1) ^ (r & 7)) * 16) =
              make_uint4(s8x2_to_bf16<0>(v[b].z), s8x2_to_bf16<1>(v[b].z), s8x2_to_bf16<0>(v[b].w),
                         s8x2_to_bf16<1>(v[b].w));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->full[st][CH_LO + h]);
      }
      ++g;
      return true;
    };
    uint4 v0[8], v1[8];
    float sc0 = 0.f, sc1 = 0.f;
    bool more = load(v0, sc0);
    while (more) {  // the next tile's rows are in flight while this one is stored
      const bool second = load(v1, sc1);
      if (!store(v0, sc0) || !second) break;
      more = load(v0, sc0);
      if (!store(v1, sc1)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

cudaError_t launch_tree_attend(const TreeParams &p, bool q8, int grid, cudaStream_t s) {
  static std::atomic<unsigned long long> opted[2];
  const void *fn = q8 ? reinterpret_cast<const void *>(tree_attend_kernel<true>)
                      : reinterpret_cast<const void *>(tree_attend_kernel<false>);
  cudaError_t e = smem_opt_in(fn, kSmemBytes, opted[q8]);
  if (e != cudaSuccess) return e;
  ProfScope ps(q8 ? "tree_attend_q8" : "tree_attend_bf16", s);
  if (q8)
    tree_attend_kernel<true><<<grid, threads<true>(), kSmemBytes, s>>>(p);
  else
    tree_attend_kernel<false><<<grid, threads<false>(), kSmemBytes, s>>>(p);
  return cudaGetLastError();
}

// One block per (entry, query row, 128 dims): the partials of a split chunk
// range, combined as merge_core.cuh does, written as bf16.
__global__ void tree_merge_kernel(uint16_t *out, float *lse, const float *part_o, const float *part_lse,
                                  const TreeMerge *entries) {
  const int row = blockIdx.y;
  const TreeMerge e = entries[blockIdx.x];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= e.nn * kHeads) return;
  const MergeSlice r = merge_slice(MergeEntry{0, e.first, e.count, 1}, row, blockIdx.z, part_o, part_lse, kTreeRows,
                                   kLatent, 1, static_cast<long long>(kTreeRows) * kLatent, kTreeRows, true);
  const size_t orow = static_cast<size_t>(e.node0) * kHeads + row;
  const bool none = r.m == -INFINITY;  // no part has seen a row
  if (lse && blockIdx.z == 0 && threadIdx.x == 0) lse[orow] = none ? -INFINITY : r.m + logf(r.sum);
  if (threadIdx.x < 32) {
    const float inv = 1.0f / r.sum;
    uint2 v = make_uint2(pack_bf16(r.t.x * inv, r.t.y * inv), pack_bf16(r.t.z * inv, r.t.w * inv));
    if (none) v = make_uint2(0u, 0u);
    *reinterpret_cast<uint2 *>(out + orow * kLatent + r.d0) = v;
  }
}

cudaError_t launch_tree_merge(const TreeParams &p, const TreeMerge *entries, int n, int max_count, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  ProfScope ps("tree_merge", s);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n, kTreeRows, kLatent / 128);
  cfg.blockDim = dim3(32 * merge_warps(max_count));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_merge_kernel, p.out, p.lse, (const float *)p.part_o, (const float *)p.part_lse,
                            entries);
}

}  // namespace kvl
