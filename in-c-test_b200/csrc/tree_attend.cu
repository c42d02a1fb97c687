// tree_attend.cu -- attention of a tree of drafted tokens over the latent
// cache (tree_attend.cuh has the formula and the work decomposition).
#include <algorithm>
#include <cmath>
#include <queue>

#include "merge_core.cuh"
#include "prof.cuh"
#include "sm100.cuh"
#include "tree_attend.cuh"

namespace kvl {

// ------------------------------------------------------------------ plan
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

}  // namespace kvl
